// Rows held as e4m3 codes with one power-of-two scale per block of 128 columns: the quantiser and the block-scaled product.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>

#include "q8.hpp"

namespace vdb {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- quantiser
// Block of 128 columns, a = max |x| over its finite values: e = the smallest exponent from -100 on with a <= 448 * 2^e, code =
// e4m3(x * 2^-e) (v_cvt_pk_fp8_f32: nearest, ties to even; x * 2^-e is never beyond 448).  The smallest code is 2^-9: with e >= -100
// every value held is an ordinary bf16 and f32 number; at e = 120 codes end at 240, so that no value rounds up to 2^128.  Half a wavefront holds a block, four columns per lane: the row is read once, codes leave 128 bytes at a time.
// Bound by HBM: 4 (2) bytes read, 1 + 1/128 written per column.

__device__ inline float to_float(float v) { return v; }
__device__ inline float to_float(_Float16 v) { return (float)v; }
__device__ inline float to_float(__bf16 v) { return (float)v; }

template <class T> struct alignas(4 * sizeof(T)) Four { T v[4]; };

// `VEC`: row starts are aligned to four elements.
template <class T, bool VEC> __device__ inline void load_four(const T* row, uint32_t k, uint32_t dim, float (&x)[4]) {
    if (VEC && k + 4 <= dim) {
        const Four<T> f = *reinterpret_cast<const Four<T>*>(row + k);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = to_float(f.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = k + i < dim ? to_float(row[k + i]) : 0.f;
    }
}

constexpr int MIN_EXP = -100, TOP_EXP = 120;

template <class T, bool VEC>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ rows, size_t stride, vdb_q8_rows out) {
    const uint32_t lane = threadIdx.x & 31, dim = (uint32_t)out.dim;
    const uint32_t nb = (dim + Q8_BLOCK - 1) / Q8_BLOCK, width = (dim + 15u) & ~15u;
    for (size_t r = (size_t)blockIdx.x * 8 + threadIdx.x / 32; r < out.n; r += (size_t)gridDim.x * 8) {
        const T* row = rows + r * stride;
        uint8_t* codes = out.codes + r * out.code_stride;
        uint8_t* scales = out.scales + r * out.scale_stride;
        float norm = 0.f;
        for (uint32_t b = 0; b < nb; ++b) {
            const uint32_t k = b * Q8_BLOCK + lane * 4;
            float x[4];
            load_four<T, VEC>(row, k, dim, x);
            uint32_t a = 0;                                    // ordered as the absolute values are
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t u = __float_as_uint(x[i]) & 0x7FFFFFFFu;
                if (u < 0x7F800000u) a = max(a, u);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) a = max(a, (uint32_t)__shfl_xor((int)a, o, 64));
            // a = m * 2^E with 1 <= m < 2, 448 = 1.75 * 2^8
            int e = (int)(a >> 23) - 127 - 8 + ((a & 0x7FFFFFu) > 0x600000u);
            e = a == 0 ? 0 : max(e, MIN_EXP);
            const float up = __uint_as_float((uint32_t)(127 - e) << 23), down = __uint_as_float((uint32_t)(127 + e) << 23);
            const float top = e == TOP_EXP ? 240.f : 448.f;
            uint32_t c = 0;
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i] * up, -top, top);
            c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], c, false);
            c = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
#pragma unroll
            for (int i = 0; i < 4; ++i) if ((__float_as_uint(x[i]) & 0x7FFFFFFFu) >= 0x7F800000u) c = (c & ~(0xFFu << (8 * i))) | (0x7Fu << (8 * i));
            const float v0 = __builtin_amdgcn_cvt_f32_fp8(c, 0) * down, v1 = __builtin_amdgcn_cvt_f32_fp8(c, 1) * down;
            const float v2 = __builtin_amdgcn_cvt_f32_fp8(c, 2) * down, v3 = __builtin_amdgcn_cvt_f32_fp8(c, 3) * down;
            norm = __builtin_fmaf(v0, v0, norm); norm = __builtin_fmaf(v1, v1, norm);
            norm = __builtin_fmaf(v2, v2, norm); norm = __builtin_fmaf(v3, v3, norm);
            if (k < width) *reinterpret_cast<uint32_t*>(codes + k) = c;
            if (lane == 0) scales[b] = (uint8_t)(e + 127);
        }
        if (lane < ((nb + 3) & ~3u) - nb) scales[nb + lane] = 127;
        if (out.norms2) {
#pragma unroll
            for (int o = 16; o; o >>= 1) norm += __shfl_xor(norm, o, 64);
            if (lane == 0) out.norms2[r] = norm;
        }
    }
}

// ---------------------------------------------------------------- block-scaled product
// dot(q, r) = sum over blocks b of 2^(eq + er) * sum over k in b of cq[k] * cr[k].
// The matrix instructions on 8-bit operands add the products of eight columns in a window of 13 bits below the largest of them
// (one product of 2^14 and one of 1: the 1 is lost; sums of random positive products come out 2^-16 off), so codes become bf16
// first: four significant bits fit, the block's power of two goes into the exponent, and the conversion takes both
// (v_cvt_scalef32_pk_bf16_fp8, two codes per instruction at the rate of an addition).  Products of bf16 are exact in f32 and so is
// their window: the sums are ordinary 32-bit sums.
// The order of the columns inside a block is free as long as both sides use the same: lane (r, g) of v_mfma_f32_16x16x32_bf16
// takes the 16 bytes at 16 g and at 64 + 16 g of row r, so that a load reads 64 consecutive bytes of each row.  The result's lane
// (r, g) holds query r against rows 4 g .. 4 g + 3.

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ inline uint4 load16(const uint8_t* row, uint32_t k, uint32_t width) {
    return k < width ? *reinterpret_cast<const uint4*>(row + k) : uint4{0, 0, 0, 0};
}
__device__ inline float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ inline bf16x8 widen(uint32_t lo, uint32_t hi, float scale) {          // eight codes to bf16 values
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ inline float finish(float dot, float nq, float nb, int metric) {
    if (metric == VDB_DOT) return dot;
    if (metric == VDB_COSINE) return 1.0f - dot / (__builtin_sqrtf(nq) * __builtin_sqrtf(nb) + 1e-10f);
    const float d = __builtin_fmaf(-2.f, dot, nq + nb);
    return __builtin_sqrtf(d < 0.f ? 0.f : d);                 // NaN stays
}

// A wavefront scores 16 rows against 16 queries.
__global__ void __launch_bounds__(256) score_kernel(Q8View q, Q8View b, int metric, float* __restrict__ out, size_t out_stride, uint32_t row_tiles, uint64_t tiles) {
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const uint32_t nb = b.blocks(), width = b.width();
    for (uint64_t t = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64; t < tiles; t += (uint64_t)gridDim.x * 4) {
        const uint32_t row0 = (uint32_t)(t % row_tiles) * 16, q0 = (uint32_t)(t / row_tiles) * 16;
        const size_t row = min(row0 + r, b.n - 1), qu = min(q0 + r, q.n - 1);          // a tile's end repeats the last row; what it gives is not stored
        const uint8_t* rc = b.codes + row * b.cs; const uint8_t* qc = q.codes + qu * q.cs;
        const uint8_t* rs = b.scales + row * b.ss; const uint8_t* qs = q.scales + qu * q.ss;
        floatx4 acc{0.f, 0.f, 0.f, 0.f};
        for (uint32_t k = 0; k < nb; ++k) {
            const float xs = scale_of(rs[k]), ys = scale_of(qs[k]);
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint4 x = load16(rc, k * Q8_BLOCK + 64 * h + 16 * g, width), y = load16(qc, k * Q8_BLOCK + 64 * h + 16 * g, width);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(x.x, x.y, xs), widen(y.x, y.y, ys), acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(x.z, x.w, xs), widen(y.z, y.w, ys), acc, 0, 0, 0);
            }
        }
        if (q0 + r >= q.n) continue;
        const float nq = metric == VDB_DOT ? 0.f : q.norms2[qu];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t c = row0 + 4 * g + i;
            if (c < b.n) out[(size_t)qu * out_stride + c] = finish(acc[i], nq, metric == VDB_DOT ? 0.f : b.norms2[c], metric);
        }
    }
}

}  // namespace

void launch_q8_quantize(const void* rows, int dtype, size_t stride, const vdb_q8_rows& out, hipStream_t s) {
    const uint32_t blocks = (uint32_t)std::min<size_t>((out.n + 7) / 8, 1u << 20);
    const size_t size = dtype == VDB_F32 ? 4 : 2;
    const bool vec = (uintptr_t)rows % (4 * size) == 0 && stride % 4 == 0;
#define VDB_QUANT(T) do { if (vec) hipLaunchKernelGGL((quantize_kernel<T, true>), dim3(blocks), dim3(256), 0, s, (const T*)rows, stride, out); \
                          else hipLaunchKernelGGL((quantize_kernel<T, false>), dim3(blocks), dim3(256), 0, s, (const T*)rows, stride, out); } while (0)
    if (dtype == VDB_F32) VDB_QUANT(float); else if (dtype == VDB_F16) VDB_QUANT(_Float16); else VDB_QUANT(__bf16);
#undef VDB_QUANT
    VDB_HIP(hipGetLastError());
}

void launch_q8_score(const Q8View& q, const Q8View& b, int metric, float* out, size_t out_stride, hipStream_t s) {
    const uint32_t row_tiles = (uint32_t)(((uint64_t)b.n + 15) / 16);
    const uint64_t tiles = (((uint64_t)q.n + 15) / 16) * row_tiles;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((tiles + 3) / 4, 1u << 20);
    hipLaunchKernelGGL(score_kernel, dim3(blocks), dim3(256), 0, s, q, b, metric, out, out_stride, row_tiles, tiles);
    VDB_HIP(hipGetLastError());
}

}  // namespace vdb
