// Diagnostic for the 8-bit product (vectordb_amd/csrc/q8_kernels.hip), gfx950: (1) how many bits below the largest product the matrix
// instructions on e4m3 operands keep, against those on bf16; (2) whether v_cvt_scalef32_pk_bf16_fp8 is exact, code by code, for scale
// bytes 27, 127 and 247; (3) its rate beside an addition's.  Build: hipcc --offload-arch=gfx950 -O3 (and no packed f32 instructions).
// One wavefront or 512 workgroups of 256; every index is the thread's own place in a buffer of that size.
#include <hip/hip_runtime.h>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>
typedef int int8v __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
#define CHECK(x) do { hipError_t e = (x); if (e != hipSuccess) { printf("%s: %s\n", #x, hipGetErrorString(e)); exit(1); } } while (0)

// Each lane holds `per` consecutive columns of its row, lane group l / 16 the next ones; all rows alike: every result is the same sum.
__global__ void scaled_fp8(const int8v* a, const int8v* b, float* o) {         // 16 x 16 x 128, 32 codes a lane
    floatx4 x = {};
    x = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a[threadIdx.x], b[threadIdx.x], x, 0, 0, 0, 127, 0, 127);
    o[threadIdx.x] = x[0];
}
__global__ void plain_fp8(const long* a, const long* b, float* o) {            // 16 x 16 x 32, 8 codes a lane
    floatx4 x = {};
    x = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(a[threadIdx.x], b[threadIdx.x], x, 0, 0, 0);
    o[threadIdx.x] = x[0];
}
__global__ void bf16(const bf16x8* a, const bf16x8* b, float* o) {             // 16 x 16 x 32, 8 values a lane
    floatx4 x = {};
    x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[threadIdx.x], b[threadIdx.x], x, 0, 0, 0);
    o[threadIdx.x] = x[0];
}
__global__ void convert(uint32_t* o, uint32_t scale_byte) {                    // one code per thread of 256, twice in a word
    const bf16x2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(threadIdx.x | threadIdx.x << 8, __uint_as_float(scale_byte << 23), false);
    o[threadIdx.x] = __builtin_bit_cast(uint32_t, v);
}
template <bool CONVERT> __global__ void __launch_bounds__(256) rate(float* o, int n, float seed) {
    float x[8];
    for (int i = 0; i < 8; ++i) x[i] = seed + threadIdx.x * 8 + i;
    for (int t = 0; t < n; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (CONVERT) x[i] = __builtin_bit_cast(float, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(__float_as_uint(x[i]), seed, false));
            else x[i] += seed;
        }
    float s = 0.f;
    for (int i = 0; i < 8; ++i) s += x[i];
    o[blockIdx.x * 256 + threadIdx.x] = s;
}

static float value(int c) {                                                    // of a non-negative code below NaN
    const int e = c >> 3, f = c & 7;
    return e ? ldexpf(8 + f, e - 10) : ldexpf(f, -9);
}
static uint8_t code(float v) {
    for (int c = 0; c < 127; ++c) if (value(c) == v) return (uint8_t)c;
    printf("no code for %g\n", v);
    exit(1);
}
enum Kind { SCALED, PLAIN, BF16 };
static uint8_t *da, *db;
static float* dout;
static float sum(Kind k, const std::vector<float>& a, const std::vector<float>& b) {
    const int per = k == SCALED ? 32 : 8;
    std::vector<uint8_t> A(64 * 32, 0), B(64 * 32, 0);
    for (int l = 0; l < 64; ++l)
        for (int j = 0; j < per; ++j) {
            const size_t i = l / 16 * per + j;
            const float x = i < a.size() ? a[i] : 0, y = i < b.size() ? b[i] : 0;
            if (k == BF16) {
                uint32_t p, q;
                memcpy(&p, &x, 4); memcpy(&q, &y, 4);
                const uint16_t hp = p >> 16, hq = q >> 16;                     // four significant bits: exact
                memcpy(&A[l * 16 + 2 * j], &hp, 2); memcpy(&B[l * 16 + 2 * j], &hq, 2);
            } else { A[l * per + j] = code(x); B[l * per + j] = code(y); }
        }
    CHECK(hipMemcpy(da, A.data(), A.size(), hipMemcpyHostToDevice)); CHECK(hipMemcpy(db, B.data(), B.size(), hipMemcpyHostToDevice));
    if (k == SCALED) scaled_fp8<<<1, 64>>>((int8v*)da, (int8v*)db, dout);
    else if (k == PLAIN) plain_fp8<<<1, 64>>>((long*)da, (long*)db, dout);
    else bf16<<<1, 64>>>((bf16x8*)da, (bf16x8*)db, dout);
    CHECK(hipGetLastError());
    float o[64];
    CHECK(hipMemcpy(o, dout, sizeof o, hipMemcpyDeviceToHost));
    return o[0];
}

int main() {
    CHECK(hipMalloc(&da, 64 * 32)); CHECK(hipMalloc(&db, 64 * 32)); CHECK(hipMalloc(&dout, 512 * 256 * 4));
    const char* names[] = {"e4m3, scaled, 16x16x128", "e4m3, 16x16x32", "bf16, 16x16x32"};
    for (Kind k : {SCALED, PLAIN, BF16}) {
        const int columns = k == SCALED ? 128 : 32;
        printf("%s\n", names[k]);
        for (int at : {1, 4, 7, 8, 16, 31}) {
            printf("  2^m at column 0 beside 1 at column %2d, m for which the 1 is lost:", at);
            bool none = true;
            for (int m = 8; m <= 16; ++m) {                                    // 2^(m/2) * 2^(m - m/2), codes up to 2^8
                std::vector<float> a(columns, 0), b(columns, 0);
                a[0] = ldexpf(1, m / 2); b[0] = ldexpf(1, m - m / 2); a[at] = b[at] = 1;
                if (sum(k, a, b) != ldexpf(1, m) + 1) { printf(" %d", m); none = false; }
            }
            printf(none ? " none of 8 .. 16\n" : "\n");
        }
        srand(1);
        double worst = 0;
        for (int t = 0; t < 200; ++t) {
            std::vector<float> a(columns), b(columns);
            double want = 0;
            for (int i = 0; i < columns; ++i) { a[i] = ldexpf(8 + rand() % 8, rand() % 6 - 6); b[i] = ldexpf(8 + rand() % 8, rand() % 6 - 6); want += (double)a[i] * b[i]; }
            worst = fmax(worst, fabs(sum(k, a, b) - want) / want);
        }
        if (worst > 0) printf("  200 sums of random positive products: up to 2^%.1f of the sum off\n", log2(worst));
        else printf("  200 sums of random positive products: exact\n");
    }
    uint32_t* words = (uint32_t*)dout;
    for (uint32_t byte : {27u, 127u, 247u}) {
        convert<<<1, 256>>>(words, byte);
        CHECK(hipGetLastError());
        uint32_t got[256];
        CHECK(hipMemcpy(got, words, sizeof got, hipMemcpyDeviceToHost));
        int wrong = 0, beyond = 0;
        for (int c = 0; c < 256; ++c) {
            float g;
            const uint32_t w = got[c] << 16;
            memcpy(&g, &w, 4);
            if ((c & 127) == 127) { wrong += g == g; continue; }
            const double v = ldexp(value(c & 127), (int)byte - 127) * (c & 128 ? -1 : 1);
            if (fabs(v) >= 0x1p128) { ++beyond; continue; }
            wrong += (double)g != v;
        }
        printf("conversion at scale byte %u: %d codes of 256 wrong (%d are beyond f32 there)\n", byte, wrong, beyond);
    }
    hipEvent_t from, to;
    CHECK(hipEventCreate(&from)); CHECK(hipEventCreate(&to));
    auto time = [&](auto kernel, const char* what) {
        float ms = 0;
        for (int r = 0; r < 2; ++r) {
            CHECK(hipEventRecord(from));
            kernel<<<512, 256>>>(dout, 20000, 1.f);
            CHECK(hipEventRecord(to)); CHECK(hipEventSynchronize(to)); CHECK(hipEventElapsedTime(&ms, from, to));
        }
        printf("%s: %.3f ms for 512 workgroups of 160000\n", what, ms);
    };
    time(rate<true>, "conversions of two codes");
    time(rate<false>, "additions");
    return 0;
}
