// Host-visible launchers of the kernels on 8-bit rows (q8_kernels.hip) and on dense score rows (score_adjust.hip).
#pragma once
#include "common.hpp"

namespace vdb {

constexpr uint32_t Q8_BLOCK = 128;         // columns that share one scale

// n rows of dim columns as the kernels see them (layout: vdb_q8_rows in vdbmi.h).
struct Q8View {
    const uint8_t* codes; const uint8_t* scales; const float* norms2;
    size_t cs, ss;                         // bytes from row to row
    uint32_t n, dim;
    __host__ __device__ uint32_t blocks() const { return (dim + Q8_BLOCK - 1) / Q8_BLOCK; }
    __host__ __device__ uint32_t width() const { return (dim + 15u) & ~15u; }   // code bytes of a row that are read
};

void launch_q8_quantize(const void* rows, int dtype, size_t stride, const vdb_q8_rows& out, hipStream_t s);
void launch_q8_score(const Q8View& q, const Q8View& b, int metric, float* out, size_t out_stride, hipStream_t s);

struct AdjustArgs {
    const float* scores; float* out;
    size_t stride, out_stride;
    uint32_t nq, n;
    int negate;                            // distances: lower is better
    vdb_score_adjust how;
};
void launch_score_adjust(const AdjustArgs& a, hipStream_t s);

}  // namespace vdb
