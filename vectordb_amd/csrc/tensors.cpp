// vectordb_amd._tensors: the calls of scores.py on torch tensors, as a module of the interpreter.  A call reads addresses, sizes and
// strides from the tensors that it is given, checks them, allocates its result and calls the entry point on the tensors' device and its current
// stream.  In Python the same steps took 4 us of an 8 us call, more than the launch and the kernel of a small one.
// Nothing of a tensor is kept; the interpreter's lock is free while the entry point runs.
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>

#include <cstdint>
#include <string>
#include <utility>

#include "scores_on.hpp"

namespace {

// ---------------------------------------------------------------- Python's side

struct Ref {                                                   // a counted reference
    PyObject* p = nullptr;
    Ref() = default;
    explicit Ref(PyObject* o) : p(o) {}
    Ref(Ref&& o) noexcept : p(std::exchange(o.p, nullptr)) {}
    Ref(const Ref&) = delete;
    Ref& operator=(Ref&& o) noexcept { std::swap(p, o.p); return *this; }
    Ref& operator=(const Ref&) = delete;
    ~Ref() { Py_XDECREF(p); }
    PyObject* take() { return std::exchange(p, nullptr); }
};
struct Raised {};                                              // a Python exception is set
struct Refusal { std::string why; };                           // becomes an ArgumentError
[[noreturn]] void refuse(std::string why) { throw Refusal{std::move(why)}; }
template <class T> T* got(T* p) { if (!p) throw Raised{}; return p; }

// What bind() hands over, for the life of the process.
decltype(&vdb_q8_quantize_on) quantize_on;
decltype(&vdb_q8_score_on) score_on;
decltype(&vdb_score_adjust_on) adjust_on;
PyObject *rows_class, *check, *argument_error, *length_mismatch, *out_of_memory, *raw_stream, *metrics;
PyObject *name_codes, *name_scales, *name_norms2, *name_dim, *no_arguments;

PyObject* set_error() {                                        // the exception that is being handled, as Python's
    try { throw; }
    catch (const Raised&) {}
    catch (const Refusal& r) { PyErr_SetString(argument_error ? argument_error : PyExc_RuntimeError, r.why.c_str()); }
    catch (python_error& e) { e.restore(); }
    catch (const c10::OutOfMemoryError& e) { PyErr_SetString(out_of_memory ? out_of_memory : PyExc_RuntimeError, e.what_without_backtrace()); }
    catch (const c10::Error& e) { PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace()); }
    catch (const std::bad_alloc&) { PyErr_NoMemory(); }
    catch (const std::exception& e) { PyErr_SetString(PyExc_RuntimeError, e.what()); }
    return nullptr;
}

// Arguments by place (the first `by_place` of `names`) and by name; those left out are None.
template <int N> struct Arguments {
    PyObject* v[N];
    Arguments(const char* call, const char* const (&names)[N], PyObject* (&interned)[N], int needed, int by_place, PyObject* const* args, Py_ssize_t n, PyObject* kwnames) {
        if (!rows_class) { PyErr_SetString(PyExc_RuntimeError, "vectordb_amd.scores has to be imported first"); throw Raised{}; }
        if (n > by_place) { PyErr_Format(PyExc_TypeError, "%s() takes at most %d positional arguments (%zd given)", call, by_place, n); throw Raised{}; }
        for (int i = 0; i < N; ++i) v[i] = i < n ? args[i] : nullptr;
        const Py_ssize_t named = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
        for (Py_ssize_t k = 0; k < named; ++k) {
            PyObject* name = PyTuple_GET_ITEM(kwnames, k);
            int at = 0;
            while (at < N && interned[at] != name) ++at;
            if (at == N) for (at = 0; at < N && PyUnicode_CompareWithASCIIString(name, names[at]); ++at) {}
            if (at == N) { PyErr_Format(PyExc_TypeError, "%s() got an unexpected keyword argument '%U'", call, name); throw Raised{}; }
            if (v[at]) { PyErr_Format(PyExc_TypeError, "%s() got multiple values for argument '%s'", call, names[at]); throw Raised{}; }
            v[at] = args[n + k];
        }
        for (int i = 0; i < N; ++i) {
            if (!v[i] && i < needed) { PyErr_Format(PyExc_TypeError, "%s() missing required argument '%s'", call, names[i]); throw Raised{}; }
            if (!v[i]) v[i] = Py_None;
        }
    }
};
template <int N> void intern(const char* const (&names)[N], PyObject* (&to)[N]) {
    for (int i = 0; i < N; ++i) to[i] = got(PyUnicode_InternFromString(names[i]));
}

int metric_of(PyObject* o) {
    long m = -1;
    if (PyLong_Check(o)) {
        m = PyLong_AsLong(o);
        if (m == -1 && PyErr_Occurred()) PyErr_Clear();
    } else {                                                   // what equals a metric and hashes as it does, as in a set of them
        const int in = PySet_Contains(metrics, o);
        if (in < 0) PyErr_Clear();
        if (in > 0) {
            const double d = PyFloat_AsDouble(o);
            if (d == -1 && PyErr_Occurred()) PyErr_Clear();
            m = (long)d;
        }
    }
    if (m < VDB_COSINE || m > VDB_EUCLIDEAN) refuse("unknown metric");
    return (int)m;
}

// ---------------------------------------------------------------- tensors

std::string text(const c10::Device& d) { return d.str(); }
const char* text(at::ScalarType t) {
    switch (t) {
        case at::kByte: return "torch.uint8";
        case at::kFloat: return "torch.float32";
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        default: return "f32, f16 or bf16";
    }
}
bool is_tensor(PyObject* o) { return THPVariable_Check(o); }
const at::Tensor& on_gpu(PyObject* o, const char* what) {
    if (!is_tensor(o) || !THPVariable_Unpack(o).is_cuda()) refuse(std::string(what) + " must be a tensor on the GPU");
    return THPVariable_Unpack(o);
}

// A tensor whose last axis is dense: its memory, sizes, and elements from row to row.
struct Seen {
    void* p = nullptr;
    int64_t rows = 1, width = 0, stride = 0;
};
Seen seen(const at::Tensor& t, const char* what, at::ScalarType type, int axes, const c10::Device* device) {
    const std::string w(what);
    if (t.scalar_type() != type || t.dim() != axes || t.layout() != at::kStrided) refuse(w + ": expected a " + std::to_string(axes) + "-d " + text(type) + " tensor");
    if (device && t.device() != *device) refuse(w + " is on " + text(t.device()) + ", not on " + text(*device));
    if (!t.has_storage()) refuse(w + ": a tensor without memory");
    if (t.is_neg()) refuse(w + ": the memory of a negated view holds other values; resolve_neg() gives its own");
    // No gradient goes through these calls: a tensor that asks for one is not passed by without a word.
    if (t.requires_grad() && c10::GradMode::is_enabled()) refuse(w + " requires a gradient, and the call has none: pass " + w + ".detach(), or call under torch.no_grad()");
    if (t._fw_grad(0).defined()) refuse(w + " carries a tangent, and the call has none: pass its primal value");
    Seen s;
    s.width = t.size(axes - 1);
    s.rows = axes == 2 ? t.size(0) : 1;
    s.stride = s.width;
    if (!t.is_contiguous()) {
        if (s.width > 1 && t.stride(axes - 1) != 1) refuse(w + ": the last axis must be dense");
        if (axes == 2 && s.rows > 1) {
            s.stride = t.stride(0);
            if (s.stride < s.width) refuse(w + ": rows overlap");
        }
    }
    try { s.p = t.data_ptr(); }
    catch (const c10::Error&) { refuse(w + ": a tensor without memory"); }
    return s;
}
Seen seen(PyObject* o, const char* what, at::ScalarType type, int axes, const c10::Device* device) {
    if (!is_tensor(o)) refuse(std::string(what) + ": expected a " + std::to_string(axes) + "-d " + text(type) + " tensor");
    return seen(THPVariable_Unpack(o), what, type, axes, device);
}

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
constexpr int64_t BLOCK = 128;                                 // columns that share one scale

struct Rows {
    Ref codes, scales, norms2;                                 // alive during the call, whatever becomes of the Q8Rows meanwhile
    vdb_q8_rows c{};
    c10::Device device{c10::kCPU};
    void fill(int64_t dim) {
        const at::Tensor& t = on_gpu(codes.p, "codes");
        device = t.device();
        const Seen a = seen(t, "codes", at::kByte, 2, nullptr), b = seen(scales.p, "scales", at::kByte, 2, &device);
        if (dim < 1 || a.width < dim || a.width < up(dim, 16) || b.width < up(dim, 4 * BLOCK) / BLOCK) refuse("codes or scales are narrower than a row");
        if (a.rows != b.rows) refuse("codes and scales hold different numbers of rows");
        Seen n;
        if (norms2.p != Py_None) {
            n = seen(norms2.p, "norms2", at::kFloat, 1, &device);
            if (n.width != a.rows) refuse("codes and norms2 hold different numbers of rows");
        }
        c = {(uint8_t*)a.p, (uint8_t*)b.p, (float*)n.p, (size_t)a.rows, (size_t)dim, (size_t)a.stride, (size_t)b.stride};
    }
};
int64_t dim_of(PyObject* o) {
    const int64_t dim = PyLong_Check(o) ? PyLong_AsLongLong(o) : -1;
    if (dim == -1 && PyErr_Occurred()) PyErr_Clear();
    return dim;                                                // -1: refused by fill()
}
void rows_of(Rows& r, PyObject* o) {
    r.codes = Ref(got(PyObject_GetAttr(o, name_codes)));
    r.scales = Ref(got(PyObject_GetAttr(o, name_scales)));
    r.norms2 = Ref(got(PyObject_GetAttr(o, name_norms2)));
    const Ref dim(got(PyObject_GetAttr(o, name_dim)));
    r.fill(dim_of(dim.p));
}
bool is_rows(PyObject* o) { return (PyObject*)Py_TYPE(o) == rows_class || PyObject_IsInstance(o, rows_class) == 1; }

at::Tensor room(at::IntArrayRef shape, at::ScalarType type, const c10::Device& device) { return at::empty(shape, at::TensorOptions().dtype(type).device(device)); }
// The result: a tensor of its own, or `out`.
struct Result { Ref o; Seen s; };
Result result(PyObject* out, int64_t nq, int64_t n, const c10::Device& device) {
    Result r;
    if (out == Py_None) {
        const at::Tensor t = room({nq, n}, at::kFloat, device);
        r.s = {t.data_ptr(), nq, n, n};
        r.o = Ref(got(THPVariable_Wrap(t)));
        return r;
    }
    r.s = seen(out, "out", at::kFloat, 2, &device);
    if (r.s.rows != nq || r.s.width != n) refuse("out: expected shape (" + std::to_string(nq) + ", " + std::to_string(n) + ")");
    Py_INCREF(out);
    r.o = Ref(out);
    return r;
}
// Written past autograd: a backward pass that saved the tensor has to learn of it.
void written(PyObject* o) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
template <class F> void call(const c10::Device& device, F&& entry) {
    const Ref index(got(PyLong_FromLong(device.index())));
    const Ref stream(got(PyObject_CallOneArg(raw_stream, index.p)));
    void* s = PyLong_AsVoidPtr(stream.p);
    if (!s && PyErr_Occurred()) throw Raised{};
    vdb_status status;
    Py_BEGIN_ALLOW_THREADS
    status = entry(s);
    Py_END_ALLOW_THREADS
    if (status == VDB_OK) return;
    const Ref code(got(PyLong_FromLong(status)));
    const Ref none(got(PyObject_CallOneArg(check, code.p)));   // raises what belongs to the code, with the entry point's message
    PyErr_SetString(PyExc_RuntimeError, "an entry point failed");
    throw Raised{};
}

// ---------------------------------------------------------------- the calls

const char* const quantize_names[] = {"rows", "out"};
PyObject* quantize_interned[2];
PyObject* quantize_rows(PyObject*, PyObject* const* args, Py_ssize_t n_args, PyObject* kwnames) {
    try {
        const Arguments<2> a("quantize_rows", quantize_names, quantize_interned, 1, 2, args, n_args, kwnames);
        const at::Tensor& t = on_gpu(a.v[0], "rows");
        const at::ScalarType type = t.scalar_type();
        const int kind = type == at::kFloat ? VDB_F32 : type == at::kHalf ? VDB_F16 : type == at::kBFloat16 ? VDB_BF16 : -1;
        if (kind < 0) refuse("rows: expected f32, f16 or bf16");
        const Seen x = seen(t, "rows", type, 2, nullptr);
        const c10::Device device = t.device();
        Ref out;
        Rows r;
        if (a.v[1] == Py_None) {
            if (x.width < 1) refuse("empty rows");
            r.codes = Ref(got(THPVariable_Wrap(room({x.rows, up(x.width, 16)}, at::kByte, device))));
            r.scales = Ref(got(THPVariable_Wrap(room({x.rows, up(x.width, 4 * BLOCK) / BLOCK}, at::kByte, device))));
            r.norms2 = Ref(got(THPVariable_Wrap(room({x.rows}, at::kFloat, device))));
            r.fill(x.width);
            const Ref dim(got(PyLong_FromLongLong(x.width)));
            PyTypeObject* cls = (PyTypeObject*)rows_class;
            out = Ref(got(cls->tp_new(cls, no_arguments, nullptr)));
            if (PyObject_SetAttr(out.p, name_codes, r.codes.p) || PyObject_SetAttr(out.p, name_scales, r.scales.p) || PyObject_SetAttr(out.p, name_norms2, r.norms2.p) ||
                PyObject_SetAttr(out.p, name_dim, dim.p))
                throw Raised{};
        } else {
            if (!is_rows(a.v[1])) refuse("out is a Q8Rows");
            Py_INCREF(a.v[1]);
            out = Ref(a.v[1]);
            rows_of(r, out.p);
            if (r.c.n != (size_t)x.rows || r.c.dim != (size_t)x.width || r.device != device)
                refuse("out: expected " + std::to_string(x.rows) + " rows of " + std::to_string(x.width) + " columns on " + text(device));
        }
        call(device, [&](void* stream) { return quantize_on(device.index(), x.p, (vdb_dtype)kind, (size_t)x.stride, &r.c, stream); });
        if (a.v[1] != Py_None)
            for (PyObject* o : {r.codes.p, r.scales.p, r.norms2.p}) if (o != Py_None) written(o);
        return out.take();
    } catch (...) { return set_error(); }
}

const char* const score_names[] = {"queries", "base", "metric", "out"};
PyObject* score_interned[4];
PyObject* score_rows(PyObject*, PyObject* const* args, Py_ssize_t n_args, PyObject* kwnames) {
    try {
        const Arguments<4> a("score_rows", score_names, score_interned, 3, 4, args, n_args, kwnames);
        if (!is_rows(a.v[0]) || !is_rows(a.v[1])) refuse("queries and base are Q8Rows");
        Rows q, b;
        rows_of(q, a.v[0]);
        rows_of(b, a.v[1]);
        if (q.device != b.device) refuse("queries are on " + text(q.device) + ", not on " + text(b.device));
        if (q.c.dim != b.c.dim) {
            PyErr_Format(length_mismatch, "Vector length mismatch: expected %zu, got %zu", b.c.dim, q.c.dim);
            throw Raised{};
        }
        const int metric = metric_of(a.v[2]);
        Result out = result(a.v[3], (int64_t)q.c.n, (int64_t)b.c.n, b.device);
        call(b.device, [&](void* stream) { return score_on(b.device.index(), &q.c, &b.c, (vdb_metric)metric, (float*)out.s.p, (size_t)out.s.stride, stream); });
        if (a.v[3] != Py_None) written(out.o.p);
        return out.o.take();
    } catch (...) { return set_error(); }
}

enum { SCORES, METRIC, PASS_BITS, BOOST, SEEN, SEEN_OFFSETS, REPEAT, FREQUENCY, PRESENCE, OUT, N_ADJUST };
const char* const adjust_names[] = {"scores", "metric", "pass_bits", "boost", "seen", "seen_offsets", "repeat", "frequency", "presence", "out"};
PyObject* adjust_interned[N_ADJUST];
PyObject* adjust_scores(PyObject*, PyObject* const* args, Py_ssize_t n_args, PyObject* kwnames) {
    try {
        const Arguments<N_ADJUST> a("adjust_scores", adjust_names, adjust_interned, 2, 2, args, n_args, kwnames);
        const at::Tensor& t = on_gpu(a.v[SCORES], "scores");
        const c10::Device device = t.device();
        const Seen s = seen(t, "scores", at::kFloat, 2, nullptr);
        const int64_t nq = s.rows, n = s.width;
        const int metric = metric_of(a.v[METRIC]);
        vdb_score_adjust how{};
        // one row for all queries or one for each
        auto per_query = [&](int at, at::ScalarType type, int64_t width, size_t& stride) {
            PyObject* o = a.v[at];
            const bool one_axis = is_tensor(o) && THPVariable_Unpack(o).dim() == 1;
            const Seen r = seen(o, adjust_names[at], type, one_axis ? 1 : 2, &device);
            if (r.width < width || (r.rows != 1 && r.rows != nq)) refuse(std::string(adjust_names[at]) + ": expected 1 or " + std::to_string(nq) + " rows of " + std::to_string(width));
            stride = r.rows > 1 ? (size_t)r.stride : 0;
            return r.p;
        };
        if (a.v[PASS_BITS] != Py_None) how.pass = (const uint32_t*)per_query(PASS_BITS, at::kInt, up(n, 32) / 32, how.pass_stride);
        if (a.v[BOOST] != Py_None) how.boost = (const float*)per_query(BOOST, at::kFloat, n, how.boost_stride);
        const bool lists = a.v[SEEN] != Py_None;
        if (lists != (a.v[SEEN_OFFSETS] != Py_None)) refuse("seen and seen_offsets come together");
        if (lists) {
            const Seen l = seen(a.v[SEEN], "seen", at::kInt, 1, &device), o = seen(a.v[SEEN_OFFSETS], "seen_offsets", at::kLong, 1, &device);
            if (o.width != nq + 1) refuse("seen_offsets: expected " + std::to_string(nq + 1));
            how.n_seen = (size_t)l.width;
            if (how.n_seen) { how.seen = (const uint32_t*)l.p; how.seen_offsets = (const uint64_t*)o.p; }
        }
        auto each = [&](int at) -> const float* {
            if (a.v[at] == Py_None) return nullptr;
            const Seen v = seen(a.v[at], adjust_names[at], at::kFloat, 1, &device);
            if (!lists) refuse(std::string(adjust_names[at]) + " without seen");
            if (v.width != nq) refuse(std::string(adjust_names[at]) + ": expected " + std::to_string(nq));
            return (const float*)v.p;
        };
        how.repeat = each(REPEAT);
        how.frequency = each(FREQUENCY);
        how.presence = each(PRESENCE);
        Result out = result(a.v[OUT], nq, n, device);
        call(device, [&](void* stream) { return adjust_on(device.index(), (const float*)s.p, (size_t)s.stride, (size_t)nq, (size_t)n, (vdb_metric)metric, &how, (float*)out.s.p, (size_t)out.s.stride, stream); });
        if (a.v[OUT] != Py_None) written(out.o.p);
        return out.o.take();
    } catch (...) { return set_error(); }
}

// (codes, scales, norms2, dim) -> the members of vdb_q8_rows, checked
PyObject* rows_struct(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    try {
        if (n_args != 4) { PyErr_SetString(PyExc_TypeError, "rows_struct() takes 4 arguments"); throw Raised{}; }
        Rows r;
        for (int i = 0; i < 3; ++i) Py_INCREF(args[i]);
        r.codes = Ref(args[0]); r.scales = Ref(args[1]); r.norms2 = Ref(args[2]);
        r.fill(dim_of(args[3]));
        return Py_BuildValue("KKKnnnn", (unsigned long long)(uintptr_t)r.c.codes, (unsigned long long)(uintptr_t)r.c.scales, (unsigned long long)(uintptr_t)r.c.norms2, (Py_ssize_t)r.c.n,
                             (Py_ssize_t)r.c.dim, (Py_ssize_t)r.c.code_stride, (Py_ssize_t)r.c.scale_stride);
    } catch (...) { return set_error(); }
}
// the same without making anything of it
PyObject* check_rows(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    try {
        if (n_args != 4) { PyErr_SetString(PyExc_TypeError, "check_rows() takes 4 arguments"); throw Raised{}; }
        Rows r;
        for (int i = 0; i < 3; ++i) Py_INCREF(args[i]);
        r.codes = Ref(args[0]); r.scales = Ref(args[1]); r.norms2 = Ref(args[2]);
        r.fill(dim_of(args[3]));
        Py_RETURN_NONE;
    } catch (...) { return set_error(); }
}

PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long q, s, a;
    PyObject *rows, *chk, *refused, *mismatch, *oom, *stream, *m;
    if (!PyArg_ParseTuple(args, "KKKOOOOOOO", &q, &s, &a, &rows, &chk, &refused, &mismatch, &oom, &stream, &m)) return nullptr;
    quantize_on = (decltype(quantize_on))(uintptr_t)q; score_on = (decltype(score_on))(uintptr_t)s; adjust_on = (decltype(adjust_on))(uintptr_t)a;
    rows_class = Py_NewRef(rows); check = Py_NewRef(chk); argument_error = Py_NewRef(refused); length_mismatch = Py_NewRef(mismatch); out_of_memory = Py_NewRef(oom); raw_stream = Py_NewRef(stream); metrics = Py_NewRef(m);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"quantize_rows", (PyCFunction)(void (*)(void))quantize_rows, METH_FASTCALL | METH_KEYWORDS,
     "quantize_rows($module, rows, out=None)\n--\n\n"
     "f32 / f16 / bf16 rows [n, dim] -> Q8Rows (into `out` where given: appending is quantize_rows(new, out=room[n:n + k])).\n"
     "Not differentiable: rows that require a gradient are refused while gradients are recorded."},
    {"score_rows", (PyCFunction)(void (*)(void))score_rows, METH_FASTCALL | METH_KEYWORDS,
     "score_rows($module, queries, base, metric, out=None)\n--\n\n"
     "Scores [nq, n] of every query (Q8Rows) against every row (Q8Rows).  Not differentiable."},
    {"adjust_scores", (PyCFunction)(void (*)(void))adjust_scores, METH_FASTCALL | METH_KEYWORDS,
     "adjust_scores($module, scores, metric, *, pass_bits=None, boost=None, seen=None, seen_offsets=None, repeat=None, frequency=None, presence=None, out=None)\n--\n\n"
     "What vdb_score_adjust describes, over scores [nq, n] f32 (a tensor of its own, or `out`; out=scores works in place).\n\n"
     "pass_bits: int32 [words] or [1 or nq, words], words = ceil(n / 32); boost: f32 [n] or [1 or nq, n]; seen: int32 columns of all\n"
     "queries behind each other (read as unsigned; those >= n are passed over), seen_offsets: int64 [nq + 1]; repeat / frequency / presence: f32 [nq].\n"
     "Not differentiable: tensors that require a gradient are refused while gradients are recorded."},
    {"rows_struct", (PyCFunction)(void (*)(void))rows_struct, METH_FASTCALL, "rows_struct($module, codes, scales, norms2, dim, /)\n--\n\nThe members of vdb_q8_rows for these tensors."},
    {"check_rows", (PyCFunction)(void (*)(void))check_rows, METH_FASTCALL, "check_rows($module, codes, scales, norms2, dim, /)\n--\n\nRefuses tensors that do not hold rows of `dim` columns."},
    {"bind", bind, METH_VARARGS, "bind($module, quantize, score, adjust, rows_class, check, refusal, length_mismatch, out_of_memory, raw_stream, metrics, /)\n--\n\nThe entry points' addresses and what belongs to them."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "vectordb_amd._tensors", "The calls of vectordb_amd.scores.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() {
    try {
        name_codes = got(PyUnicode_InternFromString("codes")); name_scales = got(PyUnicode_InternFromString("scales"));
        name_norms2 = got(PyUnicode_InternFromString("norms2")); name_dim = got(PyUnicode_InternFromString("dim"));
        no_arguments = got(PyTuple_New(0));
        intern(quantize_names, quantize_interned);
        intern(score_names, score_interned);
        intern(adjust_names, adjust_interned);
    } catch (const Raised&) { return nullptr; }
    return PyModule_Create(&module);
}
