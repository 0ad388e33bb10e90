// Filter bitmaps, boosts and the demotion of columns already seen, laid over dense score rows (formula: vdb_score_adjust in vdbmi.h).
#include <algorithm>

#include "q8.hpp"

namespace vdb {
namespace {

// One workgroup takes a span of columns of one query.  How often the query has seen each of them is counted in LDS first (integer
// atomics: the same counts in any order); then the span is read and written once.  Bound by HBM: 8 bytes per column.
constexpr uint32_t SPAN = 4096;

__global__ void __launch_bounds__(256) adjust_kernel(AdjustArgs a, uint32_t spans, uint64_t tasks) {
    __shared__ uint32_t count[SPAN];
    for (uint64_t t = blockIdx.x; t < tasks; t += gridDim.x) {
        const uint32_t q = (uint32_t)(t / spans), lo = (uint32_t)(t % spans) * SPAN, m = min(SPAN, a.n - lo);
        float repeat = 1.f, frequency = 0.f, presence = 0.f;
        if (a.how.seen) {
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < m; i += 256) count[i] = 0;
            __syncthreads();
            const uint64_t end = min(a.how.seen_offsets[q + 1], (uint64_t)a.how.n_seen);
            for (uint64_t i = a.how.seen_offsets[q] + threadIdx.x; i < end; i += 256) {
                const uint32_t c = a.how.seen[i] - lo;         // columns before lo wrap far beyond m
                if (c < m) atomicAdd(&count[c], 1u);
            }
            __syncthreads();
            if (a.how.repeat) repeat = a.how.repeat[q];
            if (a.how.frequency) frequency = a.how.frequency[q];
            if (a.how.presence) presence = a.how.presence[q];
        }
        for (uint32_t i = threadIdx.x; i < m; i += 256) {
            const uint32_t c = lo + i;
            float g = a.scores[q * a.stride + c];
            if (a.negate) g = -g;
            if (a.how.seen && count[i]) {
                g = g > 0.f ? g / repeat : g * repeat;
                g -= __builtin_fmaf(frequency, (float)count[i], presence);
            }
            if (a.how.boost) g += a.how.boost[q * a.how.boost_stride + c];
            if (a.how.pass && !(a.how.pass[q * a.how.pass_stride + c / 32] >> (c % 32) & 1)) g = -INFINITY;
            a.out[q * a.out_stride + c] = a.negate ? -g : g;
        }
    }
}

}  // namespace

void launch_score_adjust(const AdjustArgs& a, hipStream_t s) {
    const uint32_t spans = (uint32_t)(((uint64_t)a.n + SPAN - 1) / SPAN);
    const uint64_t tasks = (uint64_t)spans * a.nq;
    hipLaunchKernelGGL(adjust_kernel, dim3((uint32_t)std::min<uint64_t>(tasks, 1u << 20)), dim3(256), 0, s, a, spans, tasks);
    VDB_HIP(hipGetLastError());
}

}  // namespace vdb
