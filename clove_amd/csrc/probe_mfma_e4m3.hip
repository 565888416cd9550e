// probe_mfma_e4m3 -- how the matrix cores add products of e4m3 codes, and at what
// rate, beside the same codes widened to bf16 (not part of the library;
// `make -C clove_amd/csrc probe` builds it).
//
// Part 1: one wave multiplies 32 x K by K x 32 codes by v_mfma_f32_32x32x64_f8f6f4, by
// v_mfma_f32_32x32x16_fp8_fp8 and, widened, by v_mfma_f32_32x32x16_bf16; printed is
// how far each is from sums in 64 bits: in the 2-norm, and on the average with its sign
// as a share of the sum of magnitudes.
// Part 2: a product of 2^14 at one place of K = 64 and one of 2^(14 - e) at each other:
// the largest e up to which their sum is exact.
// Part 3: register-only loops of each instruction on all CUs.
// Operands hold 32 * K bytes and a lane reads 32 of them from row lane % 32 at most 64
// before the row's end; every loop has a fixed trip count.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

enum Kind { F8F6F4, FP8, BF16 };
const char *const kNames[] = {"f8f6f4 ", "fp8_fp8", "bf16   "};

#define CHECK(x)                                                       \
    do {                                                               \
        const hipError_t e_ = (x);                                     \
        if (e_ != hipSuccess) {                                        \
            std::printf("%s: %s\n", #x, hipGetErrorString(e_));        \
            std::exit(1);                                              \
        }                                                              \
    } while (0)

// 64 codes of a row and of a column (a, b: this lane's, of which it holds half).
template <Kind KIND>
__device__ v16f step(const uint8_t *a, const uint8_t *b, v16f c, int h) {
    if constexpr (KIND == F8F6F4) {
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
            *reinterpret_cast<const v8i *>(a + 32 * h), *reinterpret_cast<const v8i *>(b + 32 * h),
            c, 0, 0, 0, 127, 0, 127);
    } else {
        for (int i = 0; i < 4; ++i) {
            const uint8_t *pa = a + 16 * i + 8 * h, *pb = b + 16 * i + 8 * h;
            if constexpr (KIND == FP8) {
                c = __builtin_amdgcn_mfma_f32_32x32x16_fp8_fp8(*reinterpret_cast<const long *>(pa),
                                                               *reinterpret_cast<const long *>(pb),
                                                               c, 0, 0, 0);
            } else {
                v8b x, y;
                for (int j = 0; j < 8; ++j) {
                    x[j] = (__bf16)__builtin_amdgcn_cvt_f32_fp8((int)pa[j], 0);
                    y[j] = (__bf16)__builtin_amdgcn_cvt_f32_fp8((int)pb[j], 0);
                }
                c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
            }
        }
        return c;
    }
}

template <Kind KIND>
__global__ void __launch_bounds__(64) product(const uint8_t *A, const uint8_t *B, float *C, int K) {
    const int r = threadIdx.x % 32, h = threadIdx.x / 32;
    v16f c = {0};
    for (int k = 0; k < K; k += 64) c = step<KIND>(A + r * K + k, B + r * K + k, c, h);
    for (int i = 0; i < 16; ++i) C[(i % 4 + 8 * (i / 4) + 4 * h) * 32 + r] = c[i];
}

// Four independent sums a wave, n rounds of 4 x 32 x 32 x 64.
template <Kind KIND>
__global__ void __launch_bounds__(256) rate(const uint8_t *A, float *C, int n) {
    v16f c[4] = {};
    v8i a[4];
    for (int i = 0; i < 4; ++i)
        a[i] = *reinterpret_cast<const v8i *>(A + threadIdx.x * 128 + 32 * i);
    for (int t = 0; t < n; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            union {
                v8i v;
                long q[4];
                v8b b[2];
            } x, y;
            x.v = a[i];
            y.v = a[(i + 1) & 3];
            if constexpr (KIND == F8F6F4)
                c[i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x.v, y.v, c[i], 0, 0, 0, 120,
                                                                       0, 120);
            else
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if constexpr (KIND == FP8)
                        c[i] = __builtin_amdgcn_mfma_f32_32x32x16_fp8_fp8(x.q[j], y.q[j], c[i], 0,
                                                                          0, 0);
                    else
                        c[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.b[j & 1], y.b[j >> 1],
                                                                       c[i], 0, 0, 0);
        }
    }
    float s = 0;
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 16; ++j) s += c[i][j];
    C[blockIdx.x * 256 + threadIdx.x] = s;
}

double value(uint8_t c) {
    const int f = (c >> 3) & 15, m = c & 7;
    const double v = f ? std::ldexp(8 + m, f - 10) : std::ldexp(m, -9);
    return c >> 7 ? -v : v;
}
uint8_t nearest(double x) {
    int best = 0;
    for (int c = 1; c < 127; ++c)
        if (std::fabs(value(c) - std::fabs(x)) < std::fabs(value(best) - std::fabs(x))) best = c;
    return (uint8_t)(best | (x < 0 ? 128 : 0));
}
uint8_t power(int e) { return (uint8_t)(e >= -6 ? (e + 7) << 3 : 1 << (e + 9)); }  // e in [-9, 8]

constexpr int kMaxK = 16384, kRateBlocks = 512;
uint8_t *dA, *dB;
float *dC;

std::vector<float> run(Kind kind, const std::vector<uint8_t> &A, const std::vector<uint8_t> &B) {
    CHECK(hipMemcpy(dA, A.data(), A.size(), hipMemcpyHostToDevice));
    CHECK(hipMemcpy(dB, B.data(), B.size(), hipMemcpyHostToDevice));
    const int K = (int)(A.size() / 32);
    if (kind == F8F6F4) product<F8F6F4><<<1, 64>>>(dA, dB, dC, K);
    if (kind == FP8) product<FP8><<<1, 64>>>(dA, dB, dC, K);
    if (kind == BF16) product<BF16><<<1, 64>>>(dA, dB, dC, K);
    std::vector<float> C(1024);
    CHECK(hipMemcpy(C.data(), dC, 4096, hipMemcpyDeviceToHost));
    return C;
}

int main() {
    CHECK(hipMalloc(&dA, 32 * kMaxK));
    CHECK(hipMalloc(&dB, 32 * kMaxK));
    CHECK(hipMalloc(&dC, kRateBlocks * 256 * 4));
    std::mt19937 g(1);
    std::normal_distribution<double> normal;
    for (int positive = 0; positive < 2; ++positive)
        for (int K : {128, 4096, kMaxK}) {
            std::vector<uint8_t> A(32 * K), B(32 * K);
            for (auto *v : {&A, &B})
                for (auto &c : *v) c = positive ? g() % 127 : nearest(normal(g) * 100);
            for (Kind kind : {F8F6F4, FP8, BF16}) {
                const std::vector<float> C = run(kind, A, B);
                double off = 0, all = 0, lean = 0;
                for (int i = 0; i < 32; ++i)
                    for (int j = 0; j < 32; ++j) {
                        double s = 0, mag = 0;
                        for (int k = 0; k < K; ++k) {
                            const double t = value(A[i * K + k]) * value(B[j * K + k]);
                            s += t;
                            mag += std::fabs(t);
                        }
                        const double d = C[i * 32 + j] - s;
                        off += d * d;
                        all += s * s;
                        lean += d / mag / 1024;
                    }
                std::printf("%s %s K %5d: %.2e off, on the average %+.1e\n", kNames[kind],
                            positive ? "positive" : "normal  ", K, std::sqrt(off / all), lean);
                std::fflush(stdout);
            }
        }
    for (Kind kind : {F8F6F4, FP8, BF16})
        for (int at : {0, 5, 40}) {
            int low[2] = {99, 99}, high[2] = {-1, -1};  // in its group of eight places, elsewhere
            for (int j = 0; j < 64; ++j) {
                if (j == at) continue;
                int best = -1;
                for (int e = 0; e <= 31; ++e) {
                    const int s = 14 - e, x = s >= 0 ? s / 2 : -(-s / 2), y = s - x;
                    if (y < -9) break;
                    std::vector<uint8_t> A(32 * 64, 0), B(32 * 64, 0);
                    for (int i = 0; i < 32; ++i) {
                        A[i * 64 + at] = B[i * 64 + at] = power(7);
                        A[i * 64 + j] = power(x);
                        B[i * 64 + j] = power(y);
                    }
                    if (run(kind, A, B)[0] != std::ldexp(1, 14) + std::ldexp(1, s)) break;
                    best = e;
                }
                const int where = j / 8 != at / 8;
                low[where] = std::min(low[where], best);
                high[where] = std::max(high[where], best);
            }
            std::printf("%s 2^14 at %2d beside 2^(14 - e): exact up to e %d..%d among its eight places, "
                        "%d..%d elsewhere\n", kNames[kind], at, low[0], high[0], low[1], high[1]);
            std::fflush(stdout);
        }
    std::vector<uint8_t> A(32 * kMaxK);
    for (auto &c : A) c = (uint8_t)(g() % 120 | (g() % 2 ? 128 : 0));
    CHECK(hipMemcpy(dA, A.data(), A.size(), hipMemcpyHostToDevice));
    hipEvent_t from, to;
    CHECK(hipEventCreate(&from));
    CHECK(hipEventCreate(&to));
    for (int again = 0; again < 2; ++again)
        for (Kind kind : {F8F6F4, FP8, BF16}) {
            const int n = 4000;
            CHECK(hipEventRecord(from));
            if (kind == F8F6F4) rate<F8F6F4><<<kRateBlocks, 256>>>(dA, dC, n);
            if (kind == FP8) rate<FP8><<<kRateBlocks, 256>>>(dA, dC, n);
            if (kind == BF16) rate<BF16><<<kRateBlocks, 256>>>(dA, dC, n);
            CHECK(hipEventRecord(to));
            CHECK(hipEventSynchronize(to));
            float ms;
            CHECK(hipEventElapsedTime(&ms, from, to));
            std::printf("%s registers only: %.0f TFLOP/s\n", kNames[kind],
                        kRateBlocks * 4.0 * n * 4 * 2 * 32 * 32 * 64 / ms / 1e9);
            std::fflush(stdout);
        }
    return 0;
}
