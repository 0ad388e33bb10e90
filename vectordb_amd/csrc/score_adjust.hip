// Filter bitmaps, boosts and the demotion of columns already seen, laid over dense score rows (formula: vdb_score_adjust in vdbmi.h).
#include <algorithm>

#include "q8.hpp"

namespace vdb {
namespace {

// A workgroup takes a span of columns of one query, four consecutive columns per thread and piece.  The scores are on their way while
// the span's columns of the query's list are counted in LDS (integer atomics: the same counts in any order); then every score is
// written once.  Bound by HBM: 8 bytes per column, 4 more for boosts.  Rows need no more than the alignment of a float.
// Workgroups are dealt to the eight dies in turn: each die takes an eighth of the spans of all queries, the queries of a span one behind
// the other, so that a bitmap or a row of boosts that they share is read once (16 x 1000003 with both: 22.4 us, query by query 28.3).
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef floatx4 floatx4_u __attribute__((aligned(4)));

template <int SPAN, int THREADS, bool SEEN>
__global__ void __launch_bounds__(THREADS) adjust_kernel(AdjustArgs a, uint64_t tasks) {
    constexpr int PIECES = SPAN / (4 * THREADS);
    __shared__ uint4 count[SEEN ? SPAN / 4 : 1];
    const uint64_t per = (tasks + 7) / 8, end_task = min((blockIdx.x % 8 + 1) * per, tasks);
    for (uint64_t t = blockIdx.x % 8 * per + blockIdx.x / 8; t < end_task; t += gridDim.x / 8) {
        const uint32_t q = (uint32_t)(t % a.nq), lo = (uint32_t)(t / a.nq) * SPAN, m = min((uint32_t)SPAN, a.n - lo);
        const float* scores = a.scores + q * a.stride + lo;
        floatx4 g[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const uint32_t i = (p * THREADS + threadIdx.x) * 4;
            if (i + 4 <= m) g[p] = *reinterpret_cast<const floatx4_u*>(scores + i);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) g[p][e] = i + e < m ? scores[i + e] : 0.f;
        }
        float repeat = 1.f, frequency = 0.f, presence = 0.f;
        if (SEEN) {
            __syncthreads();                                   // the last span's counts are read
#pragma unroll
            for (int p = 0; p < PIECES; ++p) count[p * THREADS + threadIdx.x] = uint4{0, 0, 0, 0};
            __syncthreads();
            const uint64_t end = min(a.how.seen_offsets[q + 1], (uint64_t)a.how.n_seen);
            for (uint64_t i = a.how.seen_offsets[q] + threadIdx.x; i < end; i += 4 * THREADS) {
                uint32_t c[4];                                 // four loads on their way; columns before lo wrap far beyond m
#pragma unroll
                for (int e = 0; e < 4; ++e) c[e] = i + e * THREADS < end ? a.how.seen[i + e * THREADS] - lo : m;
#pragma unroll
                for (int e = 0; e < 4; ++e) if (c[e] < m) atomicAdd(reinterpret_cast<uint32_t*>(count) + c[e], 1u);
            }
            if (a.how.repeat) repeat = a.how.repeat[q];
            if (a.how.frequency) frequency = a.how.frequency[q];
            if (a.how.presence) presence = a.how.presence[q];
            __syncthreads();
        }
        const float sign = a.negate ? -1.f : 1.f;
        const float* boost = a.how.boost ? a.how.boost + q * a.how.boost_stride + lo : nullptr;
        const uint32_t* pass = a.how.pass ? a.how.pass + q * a.how.pass_stride + lo / 32 : nullptr;
        float* out = a.out + q * a.out_stride + lo;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const uint32_t i = (p * THREADS + threadIdx.x) * 4;
            if (i >= m) break;
            const bool whole = i + 4 <= m;
            floatx4 v = g[p] * sign;
            if (SEEN) {
                const uint4 n4 = count[i / 4];
                const uint32_t n[4] = {n4.x, n4.y, n4.z, n4.w};
                if (n[0] | n[1] | n[2] | n[3])
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (n[e]) {
                        const float x = v[e] > 0.f ? v[e] / repeat : v[e] * repeat;
                        v[e] = x - __builtin_fmaf(frequency, (float)n[e], presence);
                    }
            }
            if (boost) {
                if (whole) v += *reinterpret_cast<const floatx4_u*>(boost + i);
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (i + e < m) v[e] += boost[i + e];
            }
            if (pass) {
                const uint32_t bits = pass[i / 32] >> (i % 32);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = bits >> e & 1 ? v[e] : -INFINITY;
            }
            v *= sign;
            if (whole) *reinterpret_cast<floatx4_u*>(out + i) = v;
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) if (i + e < m) out[i + e] = v[e];
        }
    }
}

}  // namespace

template <int SPAN, int THREADS>
static void launch(const AdjustArgs& a, hipStream_t s) {
    const uint64_t tasks = ((uint64_t)a.n + SPAN - 1) / SPAN * a.nq;
    const dim3 grid((uint32_t)std::min<uint64_t>((tasks + 7) / 8, 1u << 17) * 8);
    if (a.how.seen) hipLaunchKernelGGL((adjust_kernel<SPAN, THREADS, true>), grid, dim3(THREADS), 0, s, a, tasks);
    else hipLaunchKernelGGL((adjust_kernel<SPAN, THREADS, false>), grid, dim3(THREADS), 0, s, a, tasks);
    VDB_HIP(hipGetLastError());
}

void launch_score_adjust(const AdjustArgs& a, hipStream_t s) {
    // Every span reads its query's whole list again, so long lists want long spans while they fill the chip (64 x 128000, lists of 3000:
    // 14.4 us, spans of 4096 16.9; of 30000: 29.3 and 60.6); short lists want many workgroups (16 x 1000003, lists of 300: spans of 4096
    // 26.7 us, of 16384 31.8).
    // Without lists one piece per thread.  With boosts in spans of 4096 / 2048 / 1024 (torch's addition): 145 x 30088 8.1 / 7.8 / 7.3 us (7.6), 256 x 60000
    // 26.4 / 24.2 / 23.7 (22.2), 16 x 1000003 27.9 / 27.1 / 25.6 (30.2), 4 x 3000000 21.8 / 20.5 / 20.0 (23.2), but 64 x 128000 10.8 / 11.7 / 11.4 (11.8).
    if (!a.how.seen) launch<1024, 256>(a, s);
    else if (a.how.n_seen / a.nq >= 1024 && ((uint64_t)a.n + 16383) / 16384 * a.nq >= 256) launch<16384, 512>(a, s);
    else launch<4096, 512>(a, s);
}

}  // namespace vdb
