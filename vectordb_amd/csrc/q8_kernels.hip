// Rows held as e4m3 codes with one power-of-two scale per block of 128 columns: the quantiser and the block-scaled product.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

#include "q8.hpp"

namespace vdb {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------- quantiser
// Block of 128 columns, a = max |x| over its finite values: e = the smallest exponent from -100 on with a <= 448 * 2^e, code =
// e4m3(x * 2^-e) (v_cvt_scalef32_pk_fp8: nearest, ties to even; x * 2^-e is never beyond 448).  The smallest code is 2^-9: with e >= -100
// every value held is an ordinary bf16 and f32 number; at e = 120 codes end at 240, so that no value rounds up to 2^128.
// A lane reads 16 bytes, so 32 (16) lanes hold a block.  A row belongs to a group of that many lanes or fewer, to a wavefront or to a
// workgroup, by its length and the number of rows; the next 16 bytes are on their way while some are converted.
// Bound by HBM: 4 (2) bytes read, 1 + 1/128 written per column.  1M x 960 f32 841 us = 5.7 TB/s, 300007 x 100 bf16 18 us = 5.1 TB/s (rows
// of 100 columns leave lanes without work and lines in parts).  Few instructions count for short rows: with every value tested for
// being finite and scaled by a multiplication of its own, 300007 x 128 bf16 took 27 us, 1M x 128 f16 75 instead of 64.

constexpr size_t MAX_STRIDE = 1u << 24;     // of the rows that the tiled kernel takes: its offsets have 32 bits
constexpr int MIN_EXP = -100, TOP_EXP = 120;

template <int CTRL> __device__ inline uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true); }
// Over the 16 lanes of a row: exchanges of neighbours, pairs, and two mirrors; over 32 across two rows.
template <int LANES> __device__ inline uint32_t max_over(uint32_t v) {
    v = max(v, dpp<0xB1>(v)); v = max(v, dpp<0x4E>(v));
    if (LANES == 4) return v;
    v = max(v, dpp<0x141>(v));
    if (LANES == 8) return v;
    v = max(v, dpp<0x140>(v));
    if (LANES == 16) return v;
    const auto w = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(w[0], w[1]);
}
template <int LANES> __device__ inline float sum_over(float v) {
    v += __uint_as_float(dpp<0xB1>(__float_as_uint(v))); v += __uint_as_float(dpp<0x4E>(__float_as_uint(v)));
    if (LANES == 4) return v;
    v += __uint_as_float(dpp<0x141>(__float_as_uint(v)));
    if (LANES == 8) return v;
    v += __uint_as_float(dpp<0x140>(__float_as_uint(v)));
    if (LANES == 16) return v;
    const auto w = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(w[0]) + __uint_as_float(w[1]);
}

__device__ inline float sum_of_wave(float v) {
    v = sum_over<32>(v);
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(w[0]) + __uint_as_float(w[1]);
}

__device__ inline float to_float(float v) { return v; }
__device__ inline float to_float(_Float16 v) { return (float)v; }
__device__ inline float to_float(__bf16 v) { return (float)v; }

// 16 bytes of a row, which need no more than the alignment of an element; zeros behind its end.
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Piece { T v[16 / sizeof(T)]; };
template <class T> __device__ inline Piece<T> load_piece(const T* row, uint32_t k, uint32_t dim) {
    constexpr int E = 16 / sizeof(T);
    if (k + E <= dim) return *reinterpret_cast<const Piece<T>*>(row + k);
    Piece<T> f;
#pragma unroll
    for (int i = 0; i < E; ++i) f.v[i] = k + i < dim ? row[k + i] : (T)0.f;
    return f;
}

// Of a piece that was read at dim - E the values from k on, zeros behind them.
template <class T> __device__ inline Piece<T> shifted(const Piece<T>& in, uint32_t k, uint32_t dim) {
    constexpr int E = 16 / sizeof(T);
    const uint32_t at = dim - E, by = k > at ? min(k - at, (uint32_t)E) * (uint32_t)sizeof(T) : 0u;     // bytes
    uint4 w = __builtin_bit_cast(uint4, in);
    if (by & 16) w = uint4{0, 0, 0, 0};
    if (by & 8) w = uint4{w.z, w.w, 0, 0};
    if (by & 4) w = uint4{w.y, w.z, w.w, 0};
    if (by & 2) w = uint4{w.x >> 16 | w.y << 16, w.y >> 16 | w.z << 16, w.z >> 16 | w.w << 16, w.w >> 16};
    return __builtin_bit_cast(Piece<T>, w);
}

// The largest |x| as the bits of its f32: bits without the sign are ordered as the absolute values are, infinities and NaN above all.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ inline uint32_t largest(const Piece<float>& in) {
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) a = max(a, __float_as_uint(in.v[i]) & 0x7FFFFFFFu);
    return a;
}
template <class T> __device__ inline uint32_t largest(const Piece<T>& in) {
    u16x2 a{0, 0};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const T two[2] = {in.v[i], in.v[i + 1]};
        a = __builtin_elementwise_max(a, __builtin_bit_cast(u16x2, two) & (unsigned short)0x7FFF);
    }
    return __float_as_uint(to_float(__builtin_bit_cast(T, max(a[0], a[1]))));
}
// Two values / scale as codes in half HI of w.
template <bool HI> __device__ inline void code_pair(s16x2& w, const float* x, float scale) { w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[0], x[1], scale, HI); }
template <bool HI> __device__ inline void code_pair(s16x2& w, const _Float16* x, float scale) { w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, f16x2{x[0], x[1]}, scale, HI); }
template <bool HI> __device__ inline void code_pair(s16x2& w, const __bf16* x, float scale) { w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, bf16x2{x[0], x[1]}, scale, HI); }

// What a group of lanes makes of a block: a lane's codes, the exponent, and the lane's share of the squared norm.
template <class T, int LANES> struct Coded {
    static constexpr int E = 16 / sizeof(T);
    typedef uint32_t Codes __attribute__((ext_vector_type(E / 4)));
    Codes c;
    int e;
    __device__ void scale_by(uint32_t a) {                     // a = m * 2^E with 1 <= m < 2, 448 = 1.75 * 2^8
        e = (int)(a >> 23) - 127 - 8 + ((a & 0x7FFFFFu) > 0x600000u);
        e = a == 0 ? 0 : max(e, MIN_EXP);
    }
    __device__ Coded(const Piece<T>& in, float& norm) {
        const uint32_t a = max_over<LANES>(largest(in));
        scale_by(a);
        // Infinities, NaN and the codes that end at 240 are asked for once per wavefront.
        if (__builtin_expect(__any(a > 0x7F600000u), 0)) with_care(in);
        else {
            const float scale = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (int h = 0; h < E / 4; ++h) {
                s16x2 w{0, 0};
                code_pair<false>(w, in.v + 4 * h, scale);
                code_pair<true>(w, in.v + 4 * h + 2, scale);
                c[h] = __builtin_bit_cast(uint32_t, w);
            }
        }
        float sum = 0.f;                                       // of the squared codes
#pragma unroll
        for (int h = 0; h < E / 4; ++h) {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(c[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c[h], true);
            sum = __builtin_fmaf(lo[0], lo[0], sum); sum = __builtin_fmaf(lo[1], lo[1], sum);
            sum = __builtin_fmaf(hi[0], hi[0], sum); sum = __builtin_fmaf(hi[1], hi[1], sum);
        }
        const float down = __uint_as_float((uint32_t)(127 + e) << 23);
        norm = __builtin_fmaf(sum * down, down, norm);         // 2^240 is no f32: one factor at a time
    }
    __device__ void with_care(const Piece<T>& in) {
        float x[E];
        uint32_t a = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            x[i] = to_float(in.v[i]);
            const uint32_t v = __float_as_uint(x[i]) & 0x7FFFFFFFu;
            a = max(a, v < 0x7F800000u ? v : 0u);
        }
        scale_by(max_over<LANES>(a));
        const float up = __uint_as_float((uint32_t)(127 - e) << 23), top = e == TOP_EXP ? 240.f : 448.f;
#pragma unroll
        for (int h = 0; h < E / 4; ++h) {
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_fmed3f(x[4 * h + i] * up, -top, top);
            uint32_t w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
#pragma unroll
            for (int i = 0; i < 4; ++i) if ((__float_as_uint(x[4 * h + i]) & 0x7FFFFFFFu) >= 0x7F800000u) w = (w & ~(0xFFu << (8 * i))) | (0x7Fu << (8 * i));
            c[h] = w;
        }
    }
};

template <class T> constexpr int BLOCK_LANES = Q8_BLOCK * sizeof(T) / 16;

template <class T, int LANES, bool STREAMING>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ rows, size_t stride, vdb_q8_rows out) {
    constexpr int E = 16 / sizeof(T), GROUPS = 256 / LANES;
    const uint32_t lane = threadIdx.x % LANES, dim = (uint32_t)out.dim;
    const uint32_t nb = (dim + Q8_BLOCK - 1) / Q8_BLOCK, width = (dim + 15u) & ~15u;
    const size_t all = (size_t)gridDim.x * GROUPS;
    size_t r = (size_t)blockIdx.x * GROUPS + threadIdx.x / LANES, next_r = r;
    if (r >= out.n) return;                                    // whole groups of lanes: the exchanges below stay within one
    uint32_t b = 0, next_b = 0, scales = 0;
    float norm = 0.f;
    constexpr bool SHORT = LANES == 4;                         // rows that may be shorter than a load
    auto load = [&] {
        const uint32_t k = next_b * Q8_BLOCK + lane * E;
        const T* row = rows + next_r * stride;
        const Piece<T> x = SHORT ? load_piece(row, k, dim) : *reinterpret_cast<const Piece<T>*>(row + min(k, dim - E));
        if (++next_b < nb) return x;
        next_b = 0;
        if (out.n - next_r > all) next_r += all;               // behind the last row it comes again and is not used
        return x;
    };
    Piece<T> next = load();
    while (true) {
        Piece<T> x = next;
        next = load();
        if (!SHORT && (b + 1) * Q8_BLOCK > dim) x = shifted(x, b * Q8_BLOCK + lane * E, dim);
        const Coded<T, LANES> coded(x, norm);
        const uint32_t k = b * Q8_BLOCK + lane * E;
        if (k < width) {
            auto* to = reinterpret_cast<typename Coded<T, LANES>::Codes*>(out.codes + r * out.code_stride + k);
            if (STREAMING) __builtin_nontemporal_store(coded.c, to);
            else *to = coded.c;
        }
        if (b % 4 == 0) scales = 0x7F7F7F7Fu;                  // blocks behind the last: 127
        scales = (scales & ~(0xFFu << (8 * (b % 4)))) | (uint32_t)(coded.e + 127) << (8 * (b % 4));
        const bool last = b + 1 == nb;
        if (lane == 0 && (last || b % 4 == 3)) *reinterpret_cast<uint32_t*>(out.scales + r * out.scale_stride + b / 4 * 4) = scales;
        ++b;
        if (!last) continue;
        if (out.norms2) {
            norm = sum_over<LANES>(norm);
            if (lane == 0) out.norms2[r] = norm;
        }
        b = 0; norm = 0.f;
        if (out.n - r <= all) return;
        r += all;
    }
}

// Few rows: a workgroup per row, its blocks side by side.
template <class T>
__global__ void __launch_bounds__(256) quantize_row_kernel(const T* __restrict__ rows, size_t stride, vdb_q8_rows out) {
    constexpr int E = 16 / sizeof(T), LANES = BLOCK_LANES<T>, GROUPS = 256 / LANES;
    __shared__ float part[GROUPS];
    const uint32_t lane = threadIdx.x % LANES, group = threadIdx.x / LANES, dim = (uint32_t)out.dim;
    const uint32_t nb = (dim + Q8_BLOCK - 1) / Q8_BLOCK, width = (dim + 15u) & ~15u;
    const size_t r = blockIdx.x;
    float norm = 0.f;
    for (uint32_t b = group; b < ((nb + 3) & ~3u); b += GROUPS) {
        if (b >= nb) {                                         // blocks behind the last: 127
            if (lane == 0) out.scales[r * out.scale_stride + b] = 127;
            continue;
        }
        const uint32_t k = b * Q8_BLOCK + lane * E;
        const Coded<T, LANES> coded(load_piece(rows + r * stride, k, dim), norm);
        if (k < width) *reinterpret_cast<typename Coded<T, LANES>::Codes*>(out.codes + r * out.code_stride + k) = coded.c;
        if (lane == 0) out.scales[r * out.scale_stride + b] = (uint8_t)(coded.e + 127);
    }
    norm = sum_over<LANES>(norm);
    if (lane == 0) part[group] = norm;
    __syncthreads();
    if (threadIdx.x || !out.norms2) return;
    norm = 0.f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) norm += part[i];
    out.norms2[r] = norm;
}

// Long rows: a wavefront per row, 1024 bytes of it a step.
template <class T, bool STREAMING>
__global__ void __launch_bounds__(256) quantize_wave_kernel(const T* __restrict__ rows, size_t stride, vdb_q8_rows out) {
    constexpr uint32_t E = 16 / sizeof(T), LANES = BLOCK_LANES<T>, BLOCKS = 64 / LANES, SPAN = 64 * E;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), dim = (uint32_t)out.dim;
    const uint32_t nb = (dim + Q8_BLOCK - 1) / Q8_BLOCK, width = (dim + 15u) & ~15u, steps = (dim + SPAN - 1) / SPAN;
    for (size_t r = (size_t)blockIdx.x * 4 + wave; r < out.n; r += (size_t)gridDim.x * 4) {
        const T* row = rows + r * stride;
        auto load = [&](uint32_t i) { return *reinterpret_cast<const Piece<T>*>(row + min(i * SPAN + lane * E, dim - E)); };
        Piece<T> next = load(0);
        float norm = 0.f;
        int mine = 0;                                          // lane l: exponent of block l of 64
        for (uint32_t i = 0; i < steps; ++i) {
            const uint32_t k = i * SPAN + lane * E;
            Piece<T> x = next;
            next = load(min(i + 1, steps - 1));
            if ((i + 1) * SPAN > dim) x = shifted(x, k, dim);  // blocks behind the last are zeros, with the scale that belongs there
            const Coded<T, LANES> coded(x, norm);
            if (k < width) {
                auto* to = reinterpret_cast<typename Coded<T, LANES>::Codes*>(out.codes + r * out.code_stride + k);
                if (STREAMING) __builtin_nontemporal_store(coded.c, to);
                else *to = coded.c;
            }
            const uint32_t first = i * BLOCKS % 64;
#pragma unroll
            for (uint32_t g = 0; g < BLOCKS; ++g) {
                const int e = __builtin_amdgcn_readlane(coded.e, g * LANES);
                mine = lane == first + g ? e : mine;
            }
            if (first + BLOCKS < 64 && i + 1 < steps) continue;
            const uint32_t b = i * BLOCKS / 64 * 64 + lane;
            if (b < ((nb + 3) & ~3u)) out.scales[r * out.scale_stride + b] = (uint8_t)(mine + 127);
            mine = 0;
        }
        if (!out.norms2) continue;
        norm = sum_of_wave(norm);
        if (lane == 0) out.norms2[r] = norm;
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

// Roots and reciprocals are the hardware's (one step off at most): the scores are FAST arithmetic.
__device__ inline float root(float x) {                        // the instruction takes subnormals for zero
    const bool tiny = x < 0x1p-96f;
    const float y = __builtin_amdgcn_sqrtf(tiny ? x * 0x1p64f : x);
    return tiny ? y * 0x1p-32f : y;
}
__device__ inline float inverse(float x) { return __builtin_amdgcn_rcpf(x); }
// What a row's (query's) squared norm is used as.
__device__ inline float norm_of(const float* norms2, size_t i, int metric) {
    return metric == VDB_DOT ? 0.f : metric == VDB_COSINE ? root(norms2[i]) : norms2[i];
}
__device__ inline float finish(float dot, float nq, float nb, int metric) {
    if (metric == VDB_DOT) return dot;
    if (metric == VDB_COSINE) {
        // The reciprocal of a product beyond 2^126 is too small for the instruction (and 1e-10 vanishes long before): one factor at a time.
        const float both = nq * nb;
        const bool far = both > 0x1p60f;
        const float part = dot * inverse(far ? nq : both + 1e-10f);
        return 1.0f - (far ? part * inverse(nb) : part);
    }
    const float d = __builtin_fmaf(-2.f, dot, nq + nb);
    return root(d < 0.f ? 0.f : d);                            // NaN stays
}

// Many queries: a workgroup scores BM rows against BN queries at a time, a wavefront WM x WN of them in 32 x 32 tiles; the grid is
// what the chip holds and every workgroup walks through its tiles.  Both sides' codes go through a ring of S buffers in LDS, 64
// columns a step.  While a step is multiplied, the next one has arrived and the S - 2 behind it are on their way (straight to LDS, 16
// bytes per lane), those of the next tile too, so that a tile's first step waits for nothing; one barrier per step hands a buffer on,
// and the first fragments of a step are read before it.  A row's 16-byte chunk c lies at place c ^ (row / 4 mod 4): the eight rows
// that an LDS read serves at a time fall on different banks.
// v_mfma_f32_32x32x16_bf16: lane (r, g) holds eight columns of query (row) r; one 16-byte chunk makes two such operands (chunk
// 2 h + g in half h of the step).  Codes are widened when they are read: per 32 columns 8 conversions for each of the WM / 32 + WN / 32
// fragments, and WM WN / 512 matrix instructions of eight times their length.  The queries are the left operand: a result register
// holds 32 rows of two queries.  Slot 32 i + r of WM holds row MT r + i (MT = WM / 32), so that MT registers of a lane are consecutive
// rows: a store writes 128 MT bytes in a row for each of two queries.
// The scales of four blocks are one word per row, which comes with every step.
// Bound by power where products prevail (4096 x 32000 x 4096: 875 .. 940 us by card and warmth = 1.14 .. 1.23 PFLOP/s, the matrix pipes busy 64 % of the time at 1.9 GHz; 766 us with
// codes that are all equal), by the scores that leave where rows are short (1000 x 1M x 960: 2.07 .. 2.2 ms, 4 GB of them).  On the first of these 16 x 16
// instructions spill, and two workgroups of 256 x 128 per compute unit are slower; rings of 6, 9 and 12 buffers gain nothing on smaller tiles,
// nor does letting a tile's stores go on through the next tile's first two steps.
__device__ const uint4 zero16[1] = {};

// A wavefront's load straight to LDS: lane i's BYTES bytes at base + off (p) go to dst + i * BYTES.  Written as assembly because the
// compiler makes every LDS read behind such a load wait for it, whatever buffer it goes to; step_barrier() waits for the right ones.
// m0 holds the LDS address: an operand, so the compiler puts it there and knows that it did.  It sees no instruction in here, so the waits are
// written out: one state between m0 and the load, and five before a load that takes its base from scalar registers, which a vector
// instruction (v_readfirstlane) may have written last.
__device__ inline void load16_to_lds(const uint8_t* base, uint32_t off, uint32_t dst) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "{m0}"(dst) : "memory");
}
__device__ inline void load16_to_lds(const void* p, uint32_t dst) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(p), "{m0}"(dst) : "memory");
}
__device__ inline void load4_to_lds(const void* p, uint32_t dst) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" :: "v"(p), "{m0}"(dst) : "memory");
}
__device__ inline uint32_t lds_address(const void* p) {        // the same for the whole wavefront
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
}
// All but the wavefront's last N loads have arrived and its LDS reads are done; then everyone's.
template <int N> __device__ inline void step_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The tiles of a launch.  Workgroups are dealt to the eight dies in turn: each die takes one contiguous run of tiles, queries fastest
// within a group, so that the tiles it works on at one time share rows and queries in its L2.
struct TileOrder {
    uint32_t row_tiles, q_tiles, q_group;
    __device__ void at(uint64_t t, uint32_t& row_tile, uint32_t& q_tile) const {
        const uint64_t whole = (uint64_t)row_tiles * q_group;
        const uint32_t grp = (uint32_t)(t / whole), in_grp = min(q_group, q_tiles - grp * q_group);
        const uint32_t left = (uint32_t)(t - grp * whole);
        row_tile = left / in_grp; q_tile = grp * q_group + left % in_grp;
    }
};

template <int BM, int BN, int WM, int WN, int S>
__global__ void __launch_bounds__(64 * (BM / WM) * (BN / WN))
gemm_kernel(Q8View q, Q8View b, int metric, float* __restrict__ out, size_t out_stride, TileOrder order, bool streaming) {
    constexpr int WAVES = (BM / WM) * (BN / WN), ROWS = BM + BN;
    constexpr int KS = 64, CH = KS / 16, RPI = 64 / CH;        // columns per step, chunks per row, rows per load instruction of a wavefront
    constexpr int LOADS = ROWS / (RPI * WAVES);                // load instructions per wavefront and step
    constexpr int SLOADS = (ROWS / 64 + WAVES - 1) / WAVES;    // the same for the scales (a wavefront too many repeats the last one's)
    constexpr int MT = WM / 32, NT = WN / 32;
    typedef float Run __attribute__((ext_vector_type(MT)));
    typedef Run UnalignedRun __attribute__((aligned(4)));
    static_assert(ROWS % (RPI * WAVES) == 0 && BM % 64 == 0 && BN % 64 == 0 && S >= 3, "whole instructions");
    __shared__ uint4 tile[S][ROWS * CH];
    __shared__ uint32_t scale[S][ROWS];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), r = lane & 31, g = lane >> 5;

    const uint64_t tiles = (uint64_t)order.row_tiles * order.q_tiles, per = (tiles + 7) / 8;
    const uint64_t end = min((blockIdx.x % 8 + 1) * per, tiles);
    uint64_t t = blockIdx.x % 8 * per + blockIdx.x / 8;        // the tile that is multiplied
    if (t >= end) return;

    // what this lane loads: chunk c of one row per instruction; rows behind the last repeat it (their results are not stored).
    // Offsets count from the tile's first row: a tile is at most 256 rows of 2^24 bytes.
    const uint32_t lr = lane / CH, c = (lane % CH) ^ (lr >> 2 & 3);
    auto row_of = [](uint32_t slot) { return slot / WM * WM + MT * (slot % 32) + slot % WM / 32; };      // of the rows; a query's slot is its place
    const uint32_t width = b.width(), steps = (width + KS - 1) / KS;
    const uint32_t tile_dst = lds_address(&tile[0][wave * 64]);
    uint32_t scale_dst[SLOADS];
#pragma unroll
    for (int i = 0; i < SLOADS; ++i) scale_dst[i] = lds_address(scale[0] + min(i * WAVES + wave, (uint32_t)ROWS / 64 - 1) * 64);
    const uint8_t* row_base; const uint8_t* q_base;
    uint32_t off[LOADS];
    const uint8_t* scale_src[SLOADS];
    auto load_from = [&](uint64_t at) {
        uint32_t rt, qt;
        order.at(at, rt, qt);
        const uint32_t row0 = rt * BM, q0 = qt * BN;
        row_base = b.codes + (size_t)row0 * b.cs; q_base = q.codes + (size_t)q0 * q.cs;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t first = (i * WAVES + wave) * RPI;
            off[i] = (first < BM ? min(row_of(first + lr), b.n - 1 - row0) * (uint32_t)b.cs : min(first - BM + lr, q.n - 1 - q0) * (uint32_t)q.cs) + c * 16;
        }
#pragma unroll
        for (int i = 0; i < SLOADS; ++i) {
            const uint32_t first = min(i * WAVES + wave, (uint32_t)ROWS / 64 - 1) * 64;
            scale_src[i] = first < BM ? b.scales + (size_t)(row0 + min(row_of(first + lane), b.n - 1 - row0)) * b.ss : q.scales + (size_t)(q0 + min(first - BM + lane, q.n - 1 - q0)) * q.ss;
        }
    };
    // The step that is loaded: fs of tile ft.  Behind the last tile its first steps come again and are not used: every step has the same
    // number of loads.
    uint64_t ft = t;
    uint32_t fs = 0;
    load_from(t);
    auto fetch_tile = [&](uint32_t buf, int i) {
        const uint32_t dst = tile_dst + buf * (ROWS * CH * 16) + i * (WAVES * 1024);
        const uint8_t* base = ((i * WAVES + wave) * RPI < BM ? row_base : q_base) + (size_t)fs * KS;
        if ((fs + 1) * KS <= width) load16_to_lds(base, off[i], dst);
        else load16_to_lds(fs * KS + c * 16 < width ? (const void*)(base + off[i]) : (const void*)zero16, dst);      // zeros behind the rows' end
    };
    auto fetch_scales = [&](uint32_t buf) {
#pragma unroll
        for (int i = 0; i < SLOADS; ++i) load4_to_lds(scale_src[i] + (size_t)(fs / 8) * 4, scale_dst[i] + buf * (ROWS * 4));
    };
    auto fetched = [&] {
        if (++fs < steps) return;
        fs = 0;
        ft += gridDim.x / 8;
        if (ft < end) load_from(ft);
    };

    const uint32_t wm = wave % (BM / WM) * WM, wn = wave / (BM / WM) * WN;
    floatx16 acc[MT][NT] = {};
    struct Fragments { uint4 x[MT], y[NT]; };
    Fragments f0, f1;
    uint32_t xs[MT], ys[NT];
    auto read = [&](Fragments& f, uint32_t buf, uint32_t h) {
        const uint4* cur = tile[buf];
        const uint32_t place = (2 * h + g) ^ (r >> 2 & 3);
#pragma unroll
        for (int j = 0; j < NT; ++j) f.y[j] = cur[(BM + wn + 32 * j + r) * CH + place];
#pragma unroll
        for (int i = 0; i < MT; ++i) f.x[i] = cur[(wm + 32 * i + r) * CH + place];
    };
    auto read_scales = [&](uint32_t buf) {
#pragma unroll
        for (int j = 0; j < NT; ++j) ys[j] = scale[buf][BM + wn + 32 * j + r];
#pragma unroll
        for (int i = 0; i < MT; ++i) xs[i] = scale[buf][wm + 32 * i + r];
    };
    float xf[MT], yf[NT];
    // One half step.  `slot(i)` comes between the products of row tiles i and i + 1: loads are spread over the step, because the
    // wavefronts leave the barrier together and would otherwise queue for the memory pipe while the matrix pipe stands still.
    auto multiply = [&](const Fragments& f, auto&& slot) {
        bf16x8 y[NT][2], x[2][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) { y[j][0] = widen(f.y[j].x, f.y[j].y, yf[j]); y[j][1] = widen(f.y[j].z, f.y[j].w, yf[j]); }
        x[0][0] = widen(f.x[0].x, f.x[0].y, xf[0]); x[0][1] = widen(f.x[0].z, f.x[0].w, xf[0]);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if (i + 1 < MT) { x[(i + 1) & 1][0] = widen(f.x[i + 1].x, f.x[i + 1].y, xf[i + 1]); x[(i + 1) & 1][1] = widen(f.x[i + 1].z, f.x[i + 1].w, xf[i + 1]); }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[j][h], x[i & 1][h], acc[i][j], 0, 0, 0);
            slot(i);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Register e of tiles (0 .. MT - 1, j): rows row0 + MT r + 0 .. MT - 1 of query 32 j + 8 (e / 4) + 4 g + e mod 4.  Rows are asked
    // for one by one only where the tile holds the last.  The stores need no more than the alignment of a float.
    auto store_as = [&](auto kind, uint32_t row0, uint32_t q0) {
        constexpr int METRIC = decltype(kind)::value;
        const uint64_t row = (uint64_t)row0 + MT * r;
        float nb[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) nb[i] = norm_of(b.norms2, min(row + i, (uint64_t)b.n - 1), METRIC);
        float* lane_base = out + ((size_t)q0 + 4 * g) * out_stride + row;
        const uint32_t left = q.n - 1 - q0;                    // the last query's place
        // Lane l holds the norm of query l of the tile; a register's two queries are read from there.
        static_assert(WN <= 64, "a lane per query");
        float lane_nq = norm_of(q.norms2, (size_t)q0 + min(lane % WN, left), METRIC), least = lane_nq;
#pragma unroll
        for (int i = 0; i < MT; ++i) least = min(least, nb[i]);
        // `easy`: norms of 2^-4 and more: 1e-10 is less than half a step of their products, and the reciprocals may be taken apart;
        // squared norms of 2^-60 and more: their sum less twice the product is zero or a multiple of 2^-84, so no subnormal meets the root.
        enum { EDGE, WHOLE, STREAMING };                       // whole: every row and query of the tile is there
        auto put = [&](auto how, auto easy) {
            constexpr int HOW = decltype(how)::value;
            constexpr bool EASY = decltype(easy)::value;
            float* o = lane_base;
#pragma unroll
            for (int e = 0; e < 16 * NT; ++e) {
                const uint32_t at = e / 4 * 8 + e % 4;         // and at + 4 in the upper half of the lanes
                if (e) o += (e % 4 ? 1 : 5) * out_stride;
                if (HOW == EDGE && at + 4 * g > left) continue;
                float nq = 0.f;
                if (METRIC != VDB_DOT) {
                    const float low = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lane_nq), at)), high = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lane_nq), at + 4));
                    nq = g ? high : low;
                }
                Run v;
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const float dot = acc[i][e / 16][e % 16];
                    if (EASY && METRIC == VDB_COSINE) v[i] = __builtin_fmaf(dot * nq, -nb[i], 1.f);       // norms hold their reciprocals
                    else if (EASY && METRIC == VDB_EUCLIDEAN) {
                        const float d = __builtin_fmaf(-2.f, dot, nq + nb[i]);
                        v[i] = __builtin_amdgcn_sqrtf(d < 0.f ? 0.f : d);
                    } else v[i] = finish(dot, nq, nb[i], METRIC);
                }
                if (HOW == STREAMING) {
                    asm volatile("" ::: );                     // or the compiler makes one store of this and the one below, without the hint
                    __builtin_nontemporal_store(v, reinterpret_cast<UnalignedRun*>(o));
                } else if (HOW == WHOLE) *reinterpret_cast<UnalignedRun*>(o) = v;
                else
#pragma unroll
                    for (int i = 0; i < MT; ++i) if (row + i < b.n) o[i] = v[i];
            }
        };
        const std::integral_constant<int, EDGE> edge; const std::integral_constant<int, WHOLE> whole; const std::integral_constant<int, STREAMING> stream;
        if ((uint64_t)row0 + WM > b.n || left < WN - 1) put(edge, std::false_type{});
        else if (METRIC != VDB_DOT && !__all(least >= (METRIC == VDB_COSINE ? 0.0625f : 0x1p-60f))) put(whole, std::false_type{});
        else {
            if (METRIC == VDB_COSINE) {
                lane_nq = inverse(lane_nq);
#pragma unroll
                for (int i = 0; i < MT; ++i) nb[i] = inverse(nb[i]);
            }
            if (streaming) put(stream, std::true_type{}); else put(whole, std::true_type{});
        }
    };
    auto store = [&] {
        uint32_t rt, qt;
        order.at(t, rt, qt);
        const uint32_t row0 = rt * BM + wm, q0 = qt * BN + wn;
        if (row0 < b.n && q0 < q.n) {
            if (metric == VDB_DOT) store_as(std::integral_constant<int, VDB_DOT>{}, row0, q0);
            else if (metric == VDB_COSINE) store_as(std::integral_constant<int, VDB_COSINE>{}, row0, q0);
            else store_as(std::integral_constant<int, VDB_EUCLIDEAN>{}, row0, q0);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = floatx16{};
    };

    constexpr int PER = LOADS + SLOADS;
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) fetch_tile(s, i);
        fetch_scales(s);
        fetched();
    }
    step_barrier<(S - 2) * PER>();                             // the first step is there
    read(f0, 0, 0); read_scales(0);
    uint32_t buf = 0, s = 0;
    while (true) {
        step_barrier<(S - 3) * PER>();                         // the next step is there, and nobody reads the buffer of the last one any more
        const uint32_t next = buf + 1 == S ? 0 : buf + 1, last = buf == 0 ? S - 1 : buf - 1, shift = 8 * (s >> 1 & 3);
#pragma unroll
        for (int j = 0; j < NT; ++j) yf[j] = scale_of(ys[j] >> shift & 255u);
#pragma unroll
        for (int i = 0; i < MT; ++i) xf[i] = scale_of(xs[i] >> shift & 255u);
        read(f1, buf, 1);
        __builtin_amdgcn_sched_barrier(0);                     // the reads stay ahead of the products that hide them
        // 2 MT places for LOADS loads and the scales
        constexpr int PLACES = 2 * MT, EACH = (LOADS + PLACES - 1) / PLACES;
        multiply(f0, [&](int i) {
#pragma unroll
            for (int e = i * EACH; e < (i + 1) * EACH && e < LOADS; ++e) fetch_tile(last, e);
        });
        read(f0, next, 0); read_scales(next);
        __builtin_amdgcn_sched_barrier(0);
        multiply(f1, [&](int i) {
#pragma unroll
            for (int e = (MT + i) * EACH; e < (MT + i + 1) * EACH && e < LOADS; ++e) fetch_tile(last, e);
            if (i == MT - 1) fetch_scales(last);
        });
        fetched();
        buf = next;
        if (++s < steps) continue;
        s = 0;
        store();
        t += gridDim.x / 8;
        if (t >= end) break;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");           // nothing lands in LDS behind the workgroup's end
}

// Too few tiles for the kernel above: a workgroup scores 32 rows against 32 queries, its four wavefronts take a quarter of the columns
// each, straight from memory to registers with the next block on its way, and add up in LDS, in one order.
// It takes rows of any stride.  Bound by what one compute unit can fetch (64 x 64 x 4096: 256 KB each on four of them in 12 us; 8 wavefronts
// with an eighth of the columns 12.9, three blocks ahead 13.3, operands of 16 x 32 14.5).
__global__ void __launch_bounds__(256) narrow_kernel(Q8View q, Q8View b, int metric, float* __restrict__ out, size_t out_stride, uint32_t row_tiles, uint64_t tiles) {
    __shared__ float part[4][16][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), r = lane & 31, g = lane >> 5;
    for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const uint32_t row0 = (uint32_t)(t % row_tiles) * 32, q0 = (uint32_t)(t / row_tiles) * 32;
        const uint32_t nb = b.blocks(), width = b.width(), lo = nb * wave / 4, hi = nb * (wave + 1) / 4;
        const size_t row = row0 + min(r, b.n - 1 - row0), qu = q0 + min(r, q.n - 1 - q0);      // those behind the last repeat it and are not stored
        const uint8_t* xc = b.codes + row * b.cs; const uint8_t* xs = b.scales + row * b.ss;
        const uint8_t* yc = q.codes + qu * q.cs; const uint8_t* ys = q.scales + qu * q.ss;
        floatx16 acc = {};
        struct Block { uint4 x[4], y[4]; uint32_t xs, ys; };
        auto load = [&](Block& to, uint32_t k) {               // on no condition: chunks behind a row's end repeat its last
            to.xs = xs[k]; to.ys = ys[k];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const uint32_t at = min(k * Q8_BLOCK + 32 * h + 16 * g, width - 16);
                to.x[h] = *reinterpret_cast<const uint4*>(xc + at); to.y[h] = *reinterpret_cast<const uint4*>(yc + at);
            }
        };
        auto multiply = [&](Block& v, uint32_t k) {
            const float xf = scale_of(v.xs), yf = scale_of(v.ys);
            if ((k + 1) * Q8_BLOCK > width)
#pragma unroll
                for (int h = 0; h < 4; ++h) if (k * Q8_BLOCK + 32 * h + 16 * g >= width) v.x[h] = v.y[h] = uint4{0, 0, 0, 0};
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen(v.y[h].x, v.y[h].y, yf), widen(v.x[h].x, v.x[h].y, xf), acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen(v.y[h].z, v.y[h].w, yf), widen(v.x[h].z, v.x[h].w, xf), acc, 0, 0, 0);
            }
        };
        Block u, v;
        if (lo < hi) load(u, lo);
        for (uint32_t k = lo; k < hi; k += 2) {
            load(v, min(k + 1, hi - 1));
            multiply(u, k);
            if (k + 1 >= hi) break;
            load(u, min(k + 2, hi - 1));
            multiply(v, k + 1);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) part[wave][e][lane] = acc[e];
        __syncthreads();
        // register 4 wave + e: row r of query 8 wave + 4 g + e
        const uint64_t i = (uint64_t)row0 + r;
        const float norm = norm_of(b.norms2, row, metric);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint64_t at = (uint64_t)q0 + 8 * wave + 4 * g + e;
            if (at >= q.n || i >= b.n) continue;
            float dot = part[0][4 * wave + e][lane];
#pragma unroll
            for (int w = 1; w < 4; ++w) dot += part[w][4 * wave + e][lane];
            out[at * out_stride + i] = finish(dot, norm_of(q.norms2, at, metric), norm, metric);
        }
        __syncthreads();                                       // the parts are read
    }
}

// Up to 16 or 32 queries (QT = 1, 2): bound by the pass over the rows, which go from memory to registers.  The queries' codes lie in LDS, 16-byte chunk
// by chunk.  A wavefront takes 16 rows at a time, a block of 128 columns a step, and has DEPTH - 1 steps' codes on their way while it
// multiplies one.  The queries are the left operand: a result register holds 16 rows of four queries.
// Measured on 1 x 1M x 960: 162 us = 6.0 TB/s, 8 queries 195 (with rows staged through LDS, 4 wavefronts and 16 rows of 256 columns a step,
// 160 and 188, but 45 instead of 23 on 1M x 128); 64 rows at a time 190 .. 212 us; with the streaming hint 190 us (the second half of a line
// is fetched again).
// SPLIT: the four wavefronts of a workgroup take a quarter of the columns each of the same rows and add up in LDS, in one order.
template <int METRIC, bool SPLIT, int DEPTH, int QT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) stream_kernel(Q8View q, Q8View b, float* __restrict__ out, size_t out_stride, uint32_t groups) {
    constexpr uint32_t THREADS = 64 * WAVES;
    static_assert(!SPLIT || (QT == 1 && WAVES == 4), "one part per wavefront");
    extern __shared__ uint4 query[];                           // [8 chunks per block][queries], then the scales [4 blocks][queries]
    __shared__ floatx4 part[3][SPLIT ? 64 : 1];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), r = lane & 15, g = lane >> 4;
    const uint32_t nb = b.blocks(), width = b.width();
    uint32_t* query_scale = reinterpret_cast<uint32_t*>(query + nb * 8 * q.n);
    for (uint32_t i = threadIdx.x; i < nb * 8 * q.n; i += THREADS) query[i] = load16(q.codes + (size_t)(i % q.n) * q.cs, i / q.n * 16, width);
    for (uint32_t i = threadIdx.x; i < (nb + 3) / 4 * q.n; i += THREADS) query_scale[i] = *reinterpret_cast<const uint32_t*>(q.scales + (size_t)(i % q.n) * q.ss + i / q.n * 4);
    __syncthreads();
    uint32_t mine[QT];                                         // this lane's query of each tile; those behind the last repeat it and are not stored
#pragma unroll
    for (int j = 0; j < QT; ++j) mine[j] = min(16 * j + r, q.n - 1);
    float nq[4 * QT];                                          // register e of tile j: query 16 j + 4 g + e
#pragma unroll
    for (int e = 0; e < 4 * QT; ++e) nq[e] = norm_of(q.norms2, min(e / 4 * 16 + 4 * g + e % 4, q.n - 1), METRIC);

    const uint32_t first_group = SPLIT ? blockIdx.x : blockIdx.x * WAVES + wave, stride = SPLIT ? gridDim.x : gridDim.x * WAVES;
    if (first_group >= groups) return;                         // SPLIT: of the whole workgroup
    // Loads are on no condition, or the compiler could not tell how many are on their way and would wait for all of them: rows behind the
    // last repeat it and are not stored, chunks behind a row's end repeat its last and meet zeros of the query.
    struct Step { uint4 v[2]; uint32_t scale; };
    const uint8_t* row; const uint8_t* row_scales;
    auto row_at = [&](uint32_t group) { return (size_t)min((uint64_t)group * 16 + r, (uint64_t)b.n - 1); };
    auto go_to = [&](uint32_t group) {
        const size_t i = row_at(group);
        row = b.codes + i * b.cs;
        row_scales = b.scales + i * b.ss;
    };
    auto load = [&](Step& to, uint32_t k) {
        to.scale = row_scales[k];
#pragma unroll
        for (int h = 0; h < 2; ++h) to.v[h] = *reinterpret_cast<const uint4*>(row + min(k * Q8_BLOCK + 64 * h + 16 * g, width - 16));
    };
    floatx4 acc[QT] = {};
    float norm;
    auto multiply = [&](const Step& x, uint32_t k) {
        float qs[QT];
        const float rs = scale_of(x.scale);
#pragma unroll
        for (int j = 0; j < QT; ++j) qs[j] = scale_of(query_scale[k / 4 * q.n + mine[j]] >> (8 * (k & 3)) & 255u);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4 w = x.v[h];
            const bf16x8 lo = widen(w.x, w.y, rs), hi = widen(w.z, w.w, rs);
#pragma unroll
            for (int j = 0; j < QT; ++j) {
                const uint4 v = query[(k * 8 + 4 * h + g) * q.n + mine[j]];
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(v.x, v.y, qs[j]), lo, acc[j], 0, 0, 0);
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(v.z, v.w, qs[j]), hi, acc[j], 0, 0, 0);
            }
        }
    };
    auto clear = [&] {
#pragma unroll
        for (int j = 0; j < QT; ++j) acc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
    };
    auto store = [&](uint32_t group) {
        const uint64_t i = (uint64_t)group * 16 + r;
        if (i >= b.n) return;
#pragma unroll
        for (int e = 0; e < 4 * QT; ++e) {
            const uint32_t at = e / 4 * 16 + 4 * g + e % 4;
            if (at < q.n) out[(size_t)at * out_stride + i] = finish(acc[e / 4][e % 4], nq[e], METRIC == VDB_COSINE ? root(norm) : norm, METRIC);
        }
    };
    auto load_norm = [&](uint32_t group) { norm = METRIC == VDB_DOT ? 0.f : b.norms2[row_at(group)]; };
    Step step[DEPTH];

    if (SPLIT) {
        const uint32_t lo = nb * wave / 4, hi = nb * (wave + 1) / 4;
        for (uint32_t group = first_group; group < groups; group += stride) {
            go_to(group);
            load_norm(group);
            clear();
            if (lo < hi) {
#pragma unroll
                for (int i = 0; i < DEPTH - 1; ++i) load(step[i], min(lo + i, hi - 1));
                for (uint32_t k = lo; k < hi; k += DEPTH) {
#pragma unroll
                    for (int i = 0; i < DEPTH; ++i) {
                        if (k + i >= hi) break;
                        load(step[(i + DEPTH - 1) % DEPTH], min(k + i + DEPTH - 1, hi - 1));
                        multiply(step[i], k + i);
                    }
                }
            }
            __syncthreads();                                   // the parts of the last group are read
            if (wave) part[wave - 1][lane] = acc[0];
            __syncthreads();
            if (wave) continue;
#pragma unroll
            for (int w = 0; w < 3; ++w) acc[0] += part[w][lane];
            store(group);
        }
        return;
    }
    // the blocks of all groups in one sequence
    uint32_t group = first_group, k = 0, next_group = first_group, next_k = 0;
    auto load_next = [&](Step& to) {
        load(to, next_k);
        if (++next_k < nb) return;
        next_k = 0;
        if (groups - next_group > stride) { next_group += stride; go_to(next_group); }     // behind the last group it comes again and is not used
    };
    auto take = [&](const Step& x) {                           // -> whether the last group is done
        multiply(x, k);
        if (++k < nb) return false;
        k = 0;
        store(group);
        clear();
        if (groups - group <= stride) return true;
        group += stride;
        load_norm(group);
        return false;
    };
    go_to(group);
    load_norm(group);
#pragma unroll
    for (int i = 0; i < DEPTH - 1; ++i) load_next(step[i]);
    while (true)
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            load_next(step[(i + DEPTH - 1) % DEPTH]);
            if (take(step[i])) return;
        }
}

}  // namespace

template <class T, int LANES> static void launch_quantize_groups(const T* rows, size_t stride, const vdb_q8_rows& out, bool streaming, hipStream_t s) {
    // A group per row while the grid allows, but rows of one or two blocks are over too soon for that.  In 2^16 / 2^17 / 2^18 / 2^21 groups that
    // walk on: 1M x 128 124 / 120 / 115 / 126 us, 300007 x 100 bf16 19.4 / 19.2 / 20.1 / 20.8, 1M x 16 16.4 / 16.2 / 16.3 / 17.2; 771379 x 135 f32 128 / 127 /
    // 128 / 139, 1M x 300 325 / 314 / 304 / 297.
    constexpr size_t per = 256 / LANES;
    const size_t groups = out.dim <= Q8_BLOCK ? 1u << 17 : out.dim <= 2 * Q8_BLOCK ? 1u << 19 : 1u << 22;
    const uint32_t blocks = (uint32_t)std::min((out.n + per - 1) / per, groups / per);
    if (streaming) hipLaunchKernelGGL((quantize_kernel<T, LANES, true>), dim3(blocks), dim3(256), 0, s, rows, stride, out);
    else hipLaunchKernelGGL((quantize_kernel<T, LANES, false>), dim3(blocks), dim3(256), 0, s, rows, stride, out);
    VDB_HIP(hipGetLastError());
}

template <class T> static void launch_quantize(const T* rows, size_t stride, const vdb_q8_rows& out, hipStream_t s) {
    // Times for 1 / 500 / 2000 / 8000 rows of 960: 2.2 / 2.8 / 3.6 / 8.0 us a workgroup per row, 2.9 / 3.5 / 3.7 / 6.6 a wavefront, 4.3 / 5.0
    // / 5.3 / 7.9 a group of lanes; 4000 x 256: 4.1 a workgroup, 3.3 a group.
    if (out.n <= 2048 && out.dim > Q8_BLOCK) {
        hipLaunchKernelGGL(quantize_row_kernel<T>, dim3((uint32_t)out.n), dim3(256), 0, s, rows, stride, out);
        VDB_HIP(hipGetLastError());
        return;
    }
    // Codes leave with the streaming hint unless rows begin inside half a line, whose parts have to be joined (400000 x 720 360 against 302 us,
    // 744931 x 726 f16 460 against 397, but 1M x 128 132 against 137, 97895 x 1664 162 against 168).
    const bool streaming = out.code_stride % 64 == 0 && (uintptr_t)out.codes % 64 == 0;
    // A wavefront per row and a group of lanes per row: 1M x 960 837 and 959 us, 744931 x 726 f16 303 and 391, 1M x 512 417 and 432, f16 266 and
    // 271, but 1M x 384 384 and 326, f16 254 and 194 (a million wavefronts take 250 us to start; fewer that walk on are slower on long
    // rows: 65536 workgroups 860 us on 1M x 960, 2048 939).
    if (out.dim >= 512) {
        const uint32_t blocks = (uint32_t)std::min<size_t>((out.n + 3) / 4, 1u << 20);
        if (streaming) hipLaunchKernelGGL((quantize_wave_kernel<T, true>), dim3(blocks), dim3(256), 0, s, rows, stride, out);
        else hipLaunchKernelGGL((quantize_wave_kernel<T, false>), dim3(blocks), dim3(256), 0, s, rows, stride, out);
        VDB_HIP(hipGetLastError());
        return;
    }
    // Short rows take as many lanes as they fill, so that a wavefront holds more of them: 1M x 16 17 us (32 lanes a row: 111), 1M x 64 bf16 33 (80).
    constexpr int E = 16 / sizeof(T);
    if (out.dim <= 4 * E) return launch_quantize_groups<T, 4>(rows, stride, out, streaming, s);
    if (out.dim <= 8 * E) return launch_quantize_groups<T, 8>(rows, stride, out, streaming, s);
    if (out.dim <= 16 * E) return launch_quantize_groups<T, 16>(rows, stride, out, streaming, s);
    launch_quantize_groups<T, BLOCK_LANES<T>>(rows, stride, out, streaming, s);
}

void launch_q8_quantize(const void* rows, int dtype, size_t stride, const vdb_q8_rows& out, hipStream_t s) {
    if (dtype == VDB_F32) launch_quantize((const float*)rows, stride, out, s);
    else if (dtype == VDB_F16) launch_quantize((const _Float16*)rows, stride, out, s);
    else launch_quantize((const __bf16*)rows, stride, out, s);
}

static uint64_t tiles_of(uint32_t n, uint32_t size) { return ((uint64_t)n + size - 1) / size; }

template <int BM, int BN, int WM, int WN, int S>
static void launch_gemm(const Q8View& q, const Q8View& b, int metric, float* out, size_t out_stride, hipStream_t s) {
    const uint32_t rt = (uint32_t)tiles_of(b.n, BM), qt = (uint32_t)tiles_of(q.n, BN);
    constexpr int THREADS = 64 * (BM / WM) * (BN / WN);
    static const int resident = [] {                           // workgroups the chip holds: every gfx950 device alike
        int dev = 0, cus = 0, per_cu = 0;
        VDB_HIP(hipGetDevice(&dev));
        VDB_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
        VDB_HIP(hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, gemm_kernel<BM, BN, WM, WN, S>, THREADS, 0));
        return std::max(cus * std::max(per_cu, 1), 8);
    }();
    const uint32_t grid = (uint32_t)std::min<uint64_t>(((uint64_t)rt * qt + 7) / 8, resident / 8) * 8;
    // Scores that the last-level cache (256 MB) cannot keep leave with the streaming hint: they would drive the codes out of the L2 (1000 x 1M x
    // 64: 784 against 853 us, 8000 x 125000 x 960 1837 against 2327, 64 x 1M x 64 54 against 71; but 3860 x 12928 x 84, 200 MB, 49 against 42).
    // Score rows that share lines cost more that way, since their parts are not joined on the way, so there must be products enough to hide it
    // (more than four steps of columns) and codes that are read again: by the next queries' tiles, or from the cache if they fit there.
    // us without and with the hint, rows of 154113, 300007 and 729766 scores:
    //    154113 columns  100        256        320        960    |  729766 columns  100        256        320        512        960
    //      500      88   105   102   109   117   113   191   175 |    300       226   309   314   306   401   392   449   446   723   734
    //      768     136   168   145   172   166   175   280   261 |    512                                531   507   578   575   876   897
    //     1024     196   224   212   229   242   233   385   332 |    678       538   642   547   660   700   669   768   762  1223  1197
    //     4000     745   845   819   848   945   855  1516  1212 |   2000      1781  1950  1930  1947  2279  1972
    //    300007 columns  320        512        960       2000
    //      200     100    92   115   108   175   190   337   338
    //      384     196   187   206   180   328   349   608   630
    //      512     227   224   250   240   374   386   658   667
    const bool lines = out_stride % 32 == 0 && (uintptr_t)out % 128 == 0;
    const bool streaming = 4.0 * q.n * b.n > 235e6 && (lines || (b.width() > 256 && (q.n > 512 || (double)b.width() * b.n < 235e6)));
    hipLaunchKernelGGL((gemm_kernel<BM, BN, WM, WN, S>), dim3(grid), dim3(THREADS), 0, s, q, b, metric, out, out_stride, TileOrder{rt, qt, std::min<uint32_t>(qt, 2048 / BN)},
                       streaming);
    VDB_HIP(hipGetLastError());
}

template <int METRIC>
static void launch_stream(const Q8View& q, const Q8View& b, float* out, size_t out_stride, hipStream_t s) {
    const uint32_t nb = b.blocks(), groups = (uint32_t)tiles_of(b.n, 16);
    const size_t lds = ((size_t)nb * 128 + (nb + 3) / 4 * 4) * q.n;
    // Few rows: a workgroup per 16 of them with split columns (16 x 2000 x 4096 8.8 us, 16 on 512 workgroups that walk on, 25 on 256; 1 x 5000 x 8192
    // 14, 25 and 44; but 16 x 30000 x 2048 22.7, 15.6 and 13.7, 4 x 30000 x 960 7.4, 5.8 and 5.3).
    // Workgroups that walk through the rows, and the blocks that each wavefront has on its way or in work: 1M rows of 960 columns 162 us on
    // 512 workgroups with 3, 176 on 1024, 174 on 768, 211 on 256 (fewer walks keep to fewer pages of memory; 2 blocks 167 / 178 / 170);
    // 16 x 100000 x 4096 107 / 115 / 114; rows of one block 4 x 1M x 100 22 us on 1024 with 2, 27 on 512, 22 on 2048.  Many queries of
    // many columns leave room for one workgroup on a compute unit: 28 x 88422 x 3302 66 us on 256 of eight wavefronts, 86 on 512 of four.
#define STREAM(SPLIT, DEPTH, QT, WAVES, MOST) \
    hipLaunchKernelGGL((stream_kernel<METRIC, SPLIT, DEPTH, QT, WAVES>), dim3(std::min(SPLIT ? groups : (groups + WAVES - 1) / WAVES, MOST)), dim3(64 * WAVES), lds, s, q, b, out, out_stride, groups)
    if (q.n > 16) {
        if (nb == 1) STREAM(false, 2, 2, 4, 1024u);
        else STREAM(false, 2, 2, 8, 256u);
    } else if (groups <= 768 && nb >= 4) STREAM(true, 2, 1, 4, 768u);
    else if (nb == 1) STREAM(false, 2, 1, 4, 1024u);
    else if (groups <= 4096 || lds > (80u << 10)) STREAM(false, 2, 1, 8, 256u);
    else STREAM(false, 3, 1, 4, 512u);
#undef STREAM
    VDB_HIP(hipGetLastError());
}

void launch_q8_score(const Q8View& q, const Q8View& b, int metric, float* out, size_t out_stride, hipStream_t s) {
    const uint32_t rt = (uint32_t)tiles_of(b.n, 32);
    const uint64_t narrow = rt * tiles_of(q.n, 32);
    // Queries for 128 KiB of LDS (1 x 100000 x 8192 188 us, in tiles of 64 x 64 259); where that is much for the few rows, and for 17 to 32 queries
    // of few rows, the kernel below (16 x 10000 x 8192 56 against 34, 32 x 5000 x 4096 27 against 13, 17 x 10000 x 960 5.7 against 5.6; but 31 x 26096 x
    // 3242 20 us and 37 in tiles, 20 x 20000 x 768 6.1 and 8.9, 32 x 1M x 960 229 and 258).
    const uint64_t kib = (uint64_t)b.blocks() * q.n / 8;
    if (kib <= 128 && q.n <= 32 && (narrow > 448 || (q.n <= 16 && kib <= 64))) {
        if (metric == VDB_DOT) launch_stream<VDB_DOT>(q, b, out, out_stride, s);
        else if (metric == VDB_COSINE) launch_stream<VDB_COSINE>(q, b, out, out_stride, s);
        else launch_stream<VDB_EUCLIDEAN>(q, b, out, out_stride, s);
        return;
    }
    if (q.cs > MAX_STRIDE || b.cs > MAX_STRIDE || narrow <= 448) {
        // Times in tiles of 32 x 32 with split columns and of 64 x 64: 256 x 1000 x 4096 (256 of them) 13.1 and 26.0 us, 600 x 600 x 960 (361)
        // 6.7 and 8.6, but 100 x 4000 x 2048 (500) 14.4 and 14.5, 200 x 8000 x 768 (1750) 26 and 10.
        hipLaunchKernelGGL(narrow_kernel, dim3((uint32_t)std::min<uint64_t>(narrow, 1u << 20)), dim3(256), 0, s, q, b, metric, out, out_stride, rt, narrow);
        VDB_HIP(hipGetLastError());
        return;
    }
    // The larger the tile, the fewer conversions and LDS reads per product; the smaller, the more evenly tiles fall on the compute units
    // and the sooner one is done.  With k tiles for the fullest of 256 compute units and s steps of 64 columns a size takes about
    // once + k (ends + s step) us; the figures are fitted to 126 shapes and pick a size that is 0.9 % behind the fastest on average and 13 % at
    // most (1000 x 60000 x 100).  In tiles of 256 x 256, 256 x 128, 128 x 128, 128 x 64 and 64 x 64, us:
    //    678 x 729766 x  392   805   952  1088  1263  1423          64 x 1M     x 960   455  332  344  294  341
    //   1093 x 121956 x   77   145   137   167   178   204          20 x 100000 x 384    25   18   17   14   13
    //   1243 x   2485 x 3194    79    55    38    46    44         332 x 2060  x 1091    31   21   13   14   10
    const double steps = (b.width() + 63) / 64;
    auto cost = [&](int bm, int bn, double once, double ends, double step) { return once + (double)((tiles_of(b.n, bm) * tiles_of(q.n, bn) + 255) / 256) * (ends + steps * step); };
    const double costs[] = {cost(256, 256, 3.1, 4.9, 1.75), cost(256, 128, 2.8, 2.6, 1.04), cost(128, 128, 1.2, 1.35, 0.54), cost(128, 64, 4.4, 1.07, 0.32), cost(64, 64, 1.2, 0.66, 0.2)};
    switch (std::min_element(costs, costs + 5) - costs) {
        case 0: return launch_gemm<256, 256, 128, 64, 4>(q, b, metric, out, out_stride, s);
        case 1: return launch_gemm<256, 128, 64, 64, 4>(q, b, metric, out, out_stride, s);
        case 2: return launch_gemm<128, 128, 64, 32, 4>(q, b, metric, out, out_stride, s);
        case 3: return launch_gemm<128, 64, 64, 32, 4>(q, b, metric, out, out_stride, s);
        default: return launch_gemm<64, 64, 32, 32, 4>(q, b, metric, out, out_stride, s);
    }
}

}  // namespace vdb
