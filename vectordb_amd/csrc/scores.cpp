// C entry points of the 8-bit rows and of the score rows (contract: include/vdbmi.h).
#include <vector>

#include "guard.hpp"
#include "index.hpp"
#include "q8.hpp"
#include "scores_on.hpp"

using namespace vdb;

namespace {

constexpr size_t MAX_Q8_DIM = 1u << 24;

// [first, last) of a buffer of n rows, `row` bytes each, `stride` bytes apart.
struct Range { uintptr_t first, last; };
Range range_of(const void* p, size_t n, size_t row, size_t stride, const char* what) {
    size_t bytes;
    if (__builtin_mul_overflow(n - 1, stride, &bytes) || __builtin_add_overflow(bytes, row, &bytes) || __builtin_add_overflow((uintptr_t)p, bytes, &bytes))
        throw Failure(err_arg(std::string(what) + " does not fit the address space"));
    return {(uintptr_t)p, (uintptr_t)bytes};
}
bool meet(const Range& a, const Range& b) { return a.first < b.last && b.first < a.last; }

// The device that owns every buffer of a call; the thread's current device is put back at the end.  A caller that knows the device names
// it, and the runtime is not asked about each buffer (60 ns each).
class OnDevice {
public:
    explicit OnDevice(int known) : dev(known), ask(known < 0) {
        int n = 0;
        if (ask && (hipGetDeviceCount(&n) != hipSuccess || n <= 0)) { (void)hipGetLastError(); throw Failure(err_device("no HIP device available; libvdbmi has no CPU path")); }
        VDB_HIP(hipGetDevice(&before));
    }
    ~OnDevice() { if (at >= 0 && at != before) (void)hipSetDevice(before); }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    void add(const void* p, const char* what) {
        if (!ask) return;
        hipPointerAttribute_t a{};
        if (hipPointerGetAttributes(&a, p) != hipSuccess) { (void)hipGetLastError(); throw Failure(err_arg(std::string(what) + " is not device memory")); }
        if (a.type == hipMemoryTypeUnregistered) throw Failure(err_arg(std::string(what) + " is not device memory"));
        if (a.type == hipMemoryTypeHost) return;               // pinned: any device reads it
        if (dev >= 0 && a.device != dev) throw Failure(err_arg(std::string(what) + " lies on another device than the buffers before it"));
        dev = a.device;
    }
    void enter() { if (dev >= 0 && dev != before) { VDB_HIP(hipSetDevice(dev)); at = dev; } }
private:
    int before = 0, dev, at = -1;
    bool ask;
};

void check_rows(const vdb_q8_rows* r, const char* who) {
    const std::string w(who);
    if (!r) throw Failure(err_arg(w + " is NULL"));
    if (r->dim == 0) throw Failure(err_arg(w + ": dim must be positive"));
    if (r->dim > MAX_Q8_DIM) throw Failure(err_arg(w + ": more than 2^24 columns"));
    if (r->n > 0xFFFFFFFFull) throw Failure(err_arg(w + ": more than 2^32 - 1 rows"));
    if (r->code_stride % 16 || r->code_stride < r->dim) throw Failure(err_arg(w + ": code_stride is not a multiple of 16 that holds a row"));
    if (r->scale_stride % 4 || r->scale_stride < (r->dim + Q8_BLOCK - 1) / Q8_BLOCK) throw Failure(err_arg(w + ": scale_stride is not a multiple of 4 that holds a row's scales"));
    if (r->n == 0) return;
    if (!r->codes || !r->scales) throw Failure(err_arg(w + ": codes or scales are NULL"));
    if ((uintptr_t)r->codes % 16 || (uintptr_t)r->scales % 4 || (uintptr_t)r->norms2 % 4) throw Failure(err_arg(w + ": codes, scales or norms2 are misaligned"));
}
Range codes_of(const vdb_q8_rows& r, const char* who) { return range_of(r.codes, r.n, (r.dim + 15) & ~size_t(15), r.code_stride, who); }
Range scales_of(const vdb_q8_rows& r, const char* who) { return range_of(r.scales, r.n, ((r.dim + Q8_BLOCK - 1) / Q8_BLOCK + 3) & ~size_t(3), r.scale_stride, who); }
Range norms_of(const vdb_q8_rows& r, const char* who) { return r.norms2 ? range_of(r.norms2, r.n, 4, 4, who) : Range{0, 0}; }
void add_rows(OnDevice& d, const vdb_q8_rows& r, bool norms) {
    d.add(r.codes, "codes"); d.add(r.scales, "scales");
    if (norms) d.add(r.norms2, "norms2");
}
Q8View view(const vdb_q8_rows& r) { return {r.codes, r.scales, r.norms2, r.code_stride, r.scale_stride, (uint32_t)r.n, (uint32_t)r.dim}; }
void check_metric(int m) { if (m < VDB_COSINE || m > VDB_EUCLIDEAN) throw Failure(err_arg("unknown metric")); }

}  // namespace

extern "C" {

vdb_status vdb_q8_strides(size_t dim, size_t* code_stride, size_t* scale_stride) {
    return guard([&] {
        need(code_stride, "code_stride"); need(scale_stride, "scale_stride");
        if (dim == 0 || dim > MAX_Q8_DIM) throw Failure(err_arg("dim must be 1 .. 2^24"));
        *code_stride = (dim + 15) & ~size_t(15);
        *scale_stride = ((dim + Q8_BLOCK - 1) / Q8_BLOCK + 3) & ~size_t(3);
    });
}

vdb_status vdb_q8_quantize_on(int device, const void* d_rows, vdb_dtype dtype, size_t stride, const vdb_q8_rows* out, void* stream) {
    return guard([&] {
        check_rows(out, "out");
        if (dtype < VDB_F32 || dtype > VDB_BF16) throw Failure(err_arg("unknown element type"));
        if (stride < out->dim) throw Failure(err_arg("the row stride is shorter than the rows"));
        if (out->n == 0) return;
        need(d_rows, "d_rows");
        const size_t size = dtype == VDB_F32 ? 4 : 2;
        if ((uintptr_t)d_rows % size) throw Failure(err_arg("d_rows is not aligned to its element type"));
        size_t bytes;
        if (__builtin_mul_overflow(stride, size, &bytes)) throw Failure(err_arg("d_rows does not fit the address space"));
        const Range in = range_of(d_rows, out->n, out->dim * size, bytes, "d_rows"), c = codes_of(*out, "out"), s = scales_of(*out, "out"), m = norms_of(*out, "out");
        if (meet(in, c) || meet(in, s) || meet(in, m) || meet(c, s) || meet(c, m) || meet(s, m)) throw Failure(err_arg("the buffers overlap"));
        OnDevice dev(device);
        dev.add(d_rows, "d_rows"); add_rows(dev, *out, out->norms2 != nullptr);
        dev.enter();
        launch_q8_quantize(d_rows, dtype, stride, *out, (hipStream_t)stream);
    });
}

vdb_status vdb_q8_score_on(int device, const vdb_q8_rows* queries, const vdb_q8_rows* base, vdb_metric metric, float* d_out, size_t out_stride, void* stream) {
    return guard([&] {
        check_rows(queries, "queries"); check_rows(base, "base"); check_metric(metric);
        if (queries->dim != base->dim) throw Failure(err_length_mismatch(base->dim, queries->dim));
        if (out_stride < base->n) throw Failure(err_arg("out_stride is shorter than a row of scores"));
        if (queries->n == 0 || base->n == 0) return;
        need(d_out, "d_out");
        if ((uintptr_t)d_out % 4) throw Failure(err_arg("d_out is misaligned"));
        const bool norms = metric != VDB_DOT;
        if (norms && (!queries->norms2 || !base->norms2)) throw Failure(err_arg("cosine and Euclidean scores need norms2"));
        size_t bytes;
        if (__builtin_mul_overflow(out_stride, size_t(4), &bytes)) throw Failure(err_arg("d_out does not fit the address space"));
        const Range o = range_of(d_out, queries->n, base->n * 4, bytes, "d_out");
        for (const vdb_q8_rows* r : {queries, base})
            if (meet(o, codes_of(*r, "rows")) || meet(o, scales_of(*r, "rows")) || (norms && meet(o, norms_of(*r, "rows")))) throw Failure(err_arg("d_out overlaps the rows"));
        OnDevice dev(device);
        add_rows(dev, *queries, norms); add_rows(dev, *base, norms); dev.add(d_out, "d_out");
        dev.enter();
        launch_q8_score(view(*queries), view(*base), metric, d_out, out_stride, (hipStream_t)stream);
    });
}

vdb_status vdb_q8_quantize_dev(const void* d_rows, vdb_dtype dtype, size_t stride, const vdb_q8_rows* out, void* stream) {
    return vdb_q8_quantize_on(-1, d_rows, dtype, stride, out, stream);
}

vdb_status vdb_q8_score_dev(const vdb_q8_rows* queries, const vdb_q8_rows* base, vdb_metric metric, float* d_out, size_t out_stride, void* stream) {
    return vdb_q8_score_on(-1, queries, base, metric, d_out, out_stride, stream);
}

vdb_status vdb_score_adjust_dev(const float* d_scores, size_t stride, size_t nq, size_t n, vdb_metric metric, const vdb_score_adjust* how,
                                float* d_out, size_t out_stride, void* stream) {
    return vdb_score_adjust_on(-1, d_scores, stride, nq, n, metric, how, d_out, out_stride, stream);
}

vdb_status vdb_q8_score_scan(const float* queries, size_t nq, const float* base, size_t n, size_t dim, vdb_metric metric, int device, float* out) {
    return guard([&] {
        check_metric(metric);
        if (dim == 0 || dim > MAX_Q8_DIM) throw Failure(err_arg("dim must be 1 .. 2^24"));
        if (n > 0xFFFFFFFFull || nq > 0xFFFFFFFFull) throw Failure(err_arg("more than 2^32 - 1 rows or queries in one scan"));
        if (nq == 0 || n == 0) return;
        need(queries, "queries"); need(base, "base"); need(out, "out");
        for (const auto& [p, rows, row] : {std::tuple<const void*, size_t, size_t>{queries, nq, dim}, {base, n, dim}, {out, nq, n}})
            (void)range_of(p, rows, row * 4, row * 4, "a buffer");
        int ndev = 0, before = 0;
        if (hipGetDeviceCount(&ndev) != hipSuccess || ndev <= 0) { (void)hipGetLastError(); throw Failure(err_device("no HIP device available; libvdbmi has no CPU path")); }
        if (device < 0 || device >= ndev) throw Failure(err_device("no such device"));
        VDB_HIP(hipGetDevice(&before));
        VDB_HIP(hipSetDevice(device));
        struct Back { int d; ~Back() { (void)hipSetDevice(d); } } back{before};
        vdb_q8_rows side[2];
        DevBuf<float> f, norms[2], dout; DevBuf<uint8_t> codes[2], scales[2];
        hipStream_t s = nullptr;
        f.reserve(std::max(nq, n) * dim, s, false);
        for (int i = 0; i < 2; ++i) {
            vdb_q8_rows& r = side[i];
            r.n = i ? n : nq; r.dim = dim;
            r.code_stride = (dim + 15) & ~size_t(15); r.scale_stride = ((dim + Q8_BLOCK - 1) / Q8_BLOCK + 3) & ~size_t(3);
            codes[i].reserve(r.n * r.code_stride, s, false); scales[i].reserve(r.n * r.scale_stride, s, false); norms[i].reserve(r.n, s, false);
            r.codes = codes[i].p; r.scales = scales[i].p; r.norms2 = norms[i].p;
            VDB_HIP(hipMemcpy(f.p, i ? base : queries, r.n * dim * 4, hipMemcpyHostToDevice));   // ordered behind the first side's quantiser: one stream
            launch_q8_quantize(f.p, VDB_F32, dim, r, s);
        }
        dout.reserve(nq * n, s, false);
        launch_q8_score(view(side[0]), view(side[1]), metric, dout.p, n, s);
        VDB_HIP(hipMemcpy(out, dout.p, nq * n * 4, hipMemcpyDeviceToHost));
    });
}

vdb_status vdb_score_adjust_on(int device, const float* d_scores, size_t stride, size_t nq, size_t n, vdb_metric metric, const vdb_score_adjust* how,
                               float* d_out, size_t out_stride, void* stream) {
    return guard([&] {
        check_metric(metric); need(how, "how");
        if (n > 0xFFFFFFFFull || nq > 0xFFFFFFFFull) throw Failure(err_arg("more than 2^32 - 1 columns or queries"));
        if (stride < n || out_stride < n) throw Failure(err_arg("a row stride is shorter than a row of scores"));
        const size_t words = (n + 31) / 32;
        if (how->pass && how->pass_stride && how->pass_stride < words) throw Failure(err_arg("pass_stride is shorter than a bitmap"));
        if (how->boost && how->boost_stride && how->boost_stride < n) throw Failure(err_arg("boost_stride is shorter than a row"));
        if (how->n_seen && (!how->seen || !how->seen_offsets)) throw Failure(err_arg("seen or seen_offsets is NULL"));
        if (nq == 0 || n == 0) return;
        need(d_scores, "d_scores"); need(d_out, "d_out");
        if ((uintptr_t)d_scores % 4 || (uintptr_t)d_out % 4 || (uintptr_t)how->pass % 4 || (uintptr_t)how->boost % 4 || (uintptr_t)how->seen % 4 ||
            (uintptr_t)how->seen_offsets % 8 || (uintptr_t)how->repeat % 4 || (uintptr_t)how->frequency % 4 || (uintptr_t)how->presence % 4)
            throw Failure(err_arg("a buffer is misaligned"));
        AdjustArgs a{d_scores, d_out, stride, out_stride, (uint32_t)nq, (uint32_t)n, metric != VDB_DOT, *how};
        if (!a.how.n_seen) a.how.seen = nullptr;
        if (!a.how.seen) { a.how.seen_offsets = nullptr; a.how.repeat = a.how.frequency = a.how.presence = nullptr; }
        for (size_t v : {stride, out_stride, how->pass_stride, how->boost_stride, how->n_seen}) if (v >> 60) throw Failure(err_arg("a stride or n_seen does not fit the address space"));
        const Range o = range_of(d_out, nq, n * 4, out_stride * 4, "d_out"), in = range_of(d_scores, nq, n * 4, stride * 4, "d_scores");
        if (meet(o, in) && !(d_out == d_scores && out_stride == stride)) throw Failure(err_arg("d_out overlaps d_scores"));
        const size_t each = nq, one = 1;
        const struct { const void* p; size_t rows, row, stride; const char* what; } side[] = {
            {a.how.pass, how->pass_stride ? each : one, words * 4, how->pass_stride * 4, "pass"}, {a.how.boost, how->boost_stride ? each : one, n * 4, how->boost_stride * 4, "boost"},
            {a.how.seen, 1, how->n_seen * 4, 0, "seen"}, {a.how.seen_offsets, 1, (nq + 1) * 8, 0, "seen_offsets"},
            {a.how.repeat, 1, nq * 4, 0, "repeat"}, {a.how.frequency, 1, nq * 4, 0, "frequency"}, {a.how.presence, 1, nq * 4, 0, "presence"}};
        for (const auto& b : side) if (b.p && meet(o, range_of(b.p, b.rows, b.row, b.stride, b.what))) throw Failure(err_arg(std::string("d_out overlaps ") + b.what));
        OnDevice dev(device);
        dev.add(d_scores, "d_scores"); dev.add(d_out, "d_out");
        for (const auto& b : side) if (b.p) dev.add(b.p, b.what);
        dev.enter();
        launch_score_adjust(a, (hipStream_t)stream);
    });
}

}  // extern "C"
