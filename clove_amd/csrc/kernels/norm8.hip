// norm8.hip -- the root-mean-square norm with the residual's addition, its
// output in 32 or 8 bits, and its gradient.
//
//   h = x + residual, r = 1 / sqrt(mean(h^2) + eps), y = h r gamma
//
// y is computed in 64 bits and rounded once to 32; the 8-bit output is the code of
// that 32-bit value.  So exponents and codes, which jump at borders, do not depend
// on the order of a sum, and equal quantize8's of the 32-bit output bit for bit.
//
//   g = grad_out gamma, grad_h = r (g - h r^2 mean(g h)) + grad_sum,
//   grad_gamma = sum over rows of grad_out h r
//
// with the two sums of a row in 64 bits (h^2 leaves f32's range from 2^64 on).
#include <algorithm>

#include "linear8.h"

namespace clove {
namespace k {

namespace {

__device__ __forceinline__ double shfl_sum(double v, int width) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        if (o < width) v += __shfl_xor(v, o, 64);
    return v;
}

// Sums over the TR threads that share a row; every one of them gets the result.
// N values at once; `red` holds N * T / 64 doubles.
template <int T, int TR, int N>
__device__ __forceinline__ void row_sum(double (&v)[N], double *red) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = shfl_sum(v[i], TR < 64 ? TR : 64);
    if constexpr (TR > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) red[i * (T / 64) + wave] = v[i];
        __syncthreads();
        const int first = threadIdx.x / TR * (TR / 64);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = red[i * (T / 64) + first];
#pragma unroll
            for (int w = 1; w < TR / 64; ++w) v[i] += red[i * (T / 64) + first + w];
        }
        __syncthreads();  // red may be written again
    }
}

__device__ __forceinline__ double square_sum(cl_f4 h, double s) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s = __builtin_fma((double)h[e], (double)h[e], s);
    return s;
}

__device__ __forceinline__ cl_f4 normed(cl_f4 h, cl_f4 g, double r) {
    cl_f4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (float)((double)h[e] * r * (double)g[e]);
    return y;
}

__device__ __forceinline__ double inv_rms(double sum, int cols, float eps) {
    return 1.0 / sqrt(sum / (double)cols + (double)eps);
}

// Writes chunk c (four columns) of row `row` of the output.
template <bool ODD, bool OUT8>
__device__ __forceinline__ void emit(const RmsNormArgs &a, size_t row, int c, cl_f4 y) {
    if constexpr (OUT8) {
        const int kp = (a.cols + 127) / 128 * 128;
        // (a row that is not finite makes NaN of the zeros behind it)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * c + i >= a.cols) y[i] = 0.0f;
        const int e = lin8_exp_of(half_umax(lin8_mag4(y)));
        if (4 * c >= kp) return;
        reinterpret_cast<unsigned *>(a.codes + row * kp)[c] = lin8_encode4(y, lin8_pow2(-e));
        if ((c & 31) == 0) a.exps[row * (kp / 128) + c / 32] = e;
    } else {
        lin8_store4<ODD>(a.out + row * a.cols, c, a.cols, y);
    }
}

// TR threads a row, NV chunks of four columns each, the row in registers.
template <int T, int TR, int NV, bool ODD, bool OUT8>
__global__ void __launch_bounds__(T) norm_kernel(RmsNormArgs a, size_t row0) {
    __shared__ double red[T / 64];
    const size_t row = row0 + (size_t)blockIdx.x * (T / TR) + threadIdx.x / TR;
    const int t = threadIdx.x % TR;
    const bool in = row < a.rows;
    const float *x = a.x + (in ? row : 0) * a.cols;
    cl_f4 h[NV], g[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) h[i] = lin8_load4<ODD>(x, t + TR * i, a.cols);
    if (a.residual) {
        const float *res = a.residual + (in ? row : 0) * a.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) h[i] += lin8_load4<ODD>(res, t + TR * i, a.cols);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) g[i] = lin8_load4<ODD>(a.gamma, t + TR * i, a.cols);
    double s[1] = {0.0};
#pragma unroll
    for (int i = 0; i < NV; ++i) s[0] = square_sum(h[i], s[0]);
    row_sum<T, TR>(s, red);
    if (!in) return;
    const double r = inv_rms(s[0], a.cols, a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = t + TR * i;
        if (a.sum) lin8_store4<ODD>(a.sum + row * a.cols, c, a.cols, h[i]);
        emit<ODD, OUT8>(a, row, c, normed(h[i], g[i], r));
    }
}

// Rows that registers do not hold: stats[row] = r first, a workgroup a row...
constexpr int kWide = 16384;
template <bool ODD>
__global__ void __launch_bounds__(1024) norm_stats_kernel(RmsNormArgs a, size_t row0) {
    __shared__ double red[16];
    const size_t row = row0 + blockIdx.x;
    double s[1] = {0.0};
    for (int c = threadIdx.x; 4 * (int64_t)c < a.cols; c += 1024) {
        cl_f4 h = lin8_load4<ODD>(a.x + row * a.cols, c, a.cols);
        if (a.residual) h += lin8_load4<ODD>(a.residual + row * a.cols, c, a.cols);
        s[0] = square_sum(h, s[0]);
    }
    row_sum<1024, 1024>(s, red);
    if (threadIdx.x == 0) a.stats[row] = inv_rms(s[0], a.cols, a.eps);
}
// ...and then the columns, 1024 of a row to a workgroup.
template <bool ODD, bool OUT8>
__global__ void __launch_bounds__(256) norm_apply_kernel(RmsNormArgs a, unsigned parts,
                                                         size_t done) {
    const size_t at = done + blockIdx.x;
    const size_t row = at / parts;
    const int c = (int)(at % parts) * 256 + threadIdx.x;
    cl_f4 h = lin8_load4<ODD>(a.x + row * a.cols, c, a.cols);
    if (a.residual) h += lin8_load4<ODD>(a.residual + row * a.cols, c, a.cols);
    const cl_f4 g = lin8_load4<ODD>(a.gamma, c, a.cols);
    if (a.sum) lin8_store4<ODD>(a.sum + row * a.cols, c, a.cols, h);
    emit<ODD, OUT8>(a, row, c, normed(h, g, a.stats[row]));
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A grid holds 2^32 threads: more workgroups go in several launches.
constexpr size_t kGrid = size_t(1) << 21;
template <class F>
void in_grids(size_t n, F launch) {
    for (size_t done = 0; done < n; done += kGrid)
        launch((unsigned)std::min(kGrid, n - done), done);
}

template <bool ODD, bool OUT8>
void norm_any(const RmsNormArgs &a, hipStream_t s) {
    // (with an 8-bit output the lanes behind the row write its padding)
    const int64_t cols = OUT8 ? ((int64_t)a.cols + 127) / 128 * 128 : a.cols;
    auto go = [&](auto kernel, int t, int tr) {
        const size_t per = t / tr;
        in_grids((a.rows + per - 1) / per, [&](unsigned n, size_t done) {
            kernel<<<n, t, 0, s>>>(a, done * per);
        });
    };
    if (cols <= 128) return go(norm_kernel<256, 32, 1, ODD, OUT8>, 256, 32);
    if (cols <= 256) return go(norm_kernel<256, 64, 1, ODD, OUT8>, 256, 64);
    if (cols <= 512) return go(norm_kernel<256, 64, 2, ODD, OUT8>, 256, 64);
    if (cols <= 1024) return go(norm_kernel<256, 64, 4, ODD, OUT8>, 256, 64);
    if (cols <= 2048) return go(norm_kernel<256, 256, 2, ODD, OUT8>, 256, 256);
    if (cols <= 4096) return go(norm_kernel<256, 256, 4, ODD, OUT8>, 256, 256);
    if (cols <= 8192) return go(norm_kernel<256, 256, 8, ODD, OUT8>, 256, 256);
    if (cols <= kWide) return go(norm_kernel<1024, 1024, 4, ODD, OUT8>, 1024, 1024);
    in_grids(a.rows, [&](unsigned n, size_t done) {
        norm_stats_kernel<ODD><<<n, 1024, 0, s>>>(a, done);
    });
    const unsigned parts = (unsigned)((cols + 1023) / 1024);
    in_grids(a.rows * parts, [&](unsigned n, size_t done) {
        norm_apply_kernel<ODD, OUT8><<<n, 256, 0, s>>>(a, parts, done);
    });
}

// ---- the gradient ------------------------------------------------------------

__device__ __forceinline__ double dot(cl_f4 a, cl_f4 b, double s) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s = __builtin_fma((double)a[e], (double)b[e], s);
    return s;
}

// What a row's two sums come to: r, and r^3 mean(g h).
__device__ __forceinline__ void coefficients(double sq, double gh, int cols, float eps, double *r,
                                             double *m) {
    *r = inv_rms(sq, cols, eps);
    *m = *r * *r * *r * (gh / (double)cols);
}

// Chunk c of row `row`: grad_h out, grad_out h r added to *acc.
template <bool ODD>
__device__ __forceinline__ void grad_chunk(const RmsNormGradArgs &a, size_t row, int c, cl_f4 h,
                                           cl_f4 gy, cl_f4 gamma, double r, double m, cl_f4 *acc) {
    cl_f4 ds = {0.f, 0.f, 0.f, 0.f}, dh;
    if (a.grad_sum) ds = lin8_load4<ODD>(a.grad_sum + row * a.cols, c, a.cols);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        (*acc)[e] += gy[e] * (float)((double)h[e] * r);
        // in 64 bits where the two terms meet: they can cancel
        dh[e] = (float)((double)(gy[e] * gamma[e]) * r - (double)h[e] * m + (double)ds[e]);
    }
    if (a.grad_h) lin8_store4<ODD>(a.grad_h + row * a.cols, c, a.cols, dh);
}

// A workgroup walks the rows blockIdx.x, + gridDim.x, ...; its threads keep the
// sums of their columns and write them as one row of `part`.
template <int T, int NV, bool ODD>
__global__ void __launch_bounds__(T) grad_kernel(RmsNormGradArgs a) {
    __shared__ double red[2 * T / 64];
    const int t = threadIdx.x;
    cl_f4 gamma[NV], acc[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        gamma[i] = lin8_load4<ODD>(a.gamma, t + T * i, a.cols);
        acc[i] = (cl_f4){0.f, 0.f, 0.f, 0.f};
    }
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        cl_f4 h[NV], gy[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            h[i] = lin8_load4<ODD>(a.h + row * a.cols, t + T * i, a.cols);
            gy[i] = lin8_load4<ODD>(a.grad_out + row * a.cols, t + T * i, a.cols);
        }
        double s[2] = {0.0, 0.0};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            s[0] = square_sum(h[i], s[0]);
            s[1] = dot(gy[i] * gamma[i], h[i], s[1]);
        }
        row_sum<T, T>(s, red);
        double r, m;
        coefficients(s[0], s[1], a.cols, a.eps, &r, &m);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            grad_chunk<ODD>(a, row, t + T * i, h[i], gy[i], gamma[i], r, m, &acc[i]);
    }
    if (a.part)
#pragma unroll
        for (int i = 0; i < NV; ++i)
            lin8_store4<ODD>(a.part + (size_t)blockIdx.x * a.cols, t + T * i, a.cols, acc[i]);
}

// Rows that registers do not hold (sixteen columns a thread and four arrays of them
// leave 1024 threads no room): the sums first...
constexpr int kWideGrad = 8192;
template <bool ODD>
__global__ void __launch_bounds__(1024) grad_stats_kernel(RmsNormGradArgs a, size_t row0) {
    __shared__ double red[32];
    const size_t row = row0 + blockIdx.x;
    double s[2] = {0.0, 0.0};
    for (int c = threadIdx.x; 4 * (int64_t)c < a.cols; c += 1024) {
        const cl_f4 h = lin8_load4<ODD>(a.h + row * a.cols, c, a.cols);
        const cl_f4 gy = lin8_load4<ODD>(a.grad_out + row * a.cols, c, a.cols);
        s[0] = square_sum(h, s[0]);
        s[1] = dot(gy * lin8_load4<ODD>(a.gamma, c, a.cols), h, s[1]);
    }
    row_sum<1024, 1024>(s, red);
    if (threadIdx.x == 0)
        coefficients(s[0], s[1], a.cols, a.eps, &a.stats[2 * row], &a.stats[2 * row + 1]);
}
// ...then the columns, 1024 to a workgroup, which walks the rows of its share.
template <bool ODD>
__global__ void __launch_bounds__(256) grad_apply_kernel(RmsNormGradArgs a, unsigned parts,
                                                         unsigned shares) {
    const unsigned share = blockIdx.x / parts;
    const int c = (int)(blockIdx.x % parts) * 256 + threadIdx.x;
    const cl_f4 gamma = lin8_load4<ODD>(a.gamma, c, a.cols);
    cl_f4 acc = {0.f, 0.f, 0.f, 0.f};
    for (size_t row = share; row < a.rows; row += shares) {
        const cl_f4 h = lin8_load4<ODD>(a.h + row * a.cols, c, a.cols);
        const cl_f4 gy = lin8_load4<ODD>(a.grad_out + row * a.cols, c, a.cols);
        grad_chunk<ODD>(a, row, c, h, gy, gamma, a.stats[2 * row], a.stats[2 * row + 1], &acc);
    }
    if (a.part) lin8_store4<ODD>(a.part + (size_t)share * a.cols, c, a.cols, acc);
}

template <bool ODD>
void grad_any(const RmsNormGradArgs &a, int num_cus, hipStream_t s) {
    const unsigned n = (unsigned)rms_norm_grad_parts(a.rows, a.cols, num_cus);
    if (a.cols <= 256) return (void)(grad_kernel<64, 1, ODD><<<n, 64, 0, s>>>(a));
    if (a.cols <= 1024) return (void)(grad_kernel<256, 1, ODD><<<n, 256, 0, s>>>(a));
    if (a.cols <= 2048) return (void)(grad_kernel<256, 2, ODD><<<n, 256, 0, s>>>(a));
    if (a.cols <= 4096) return (void)(grad_kernel<256, 4, ODD><<<n, 256, 0, s>>>(a));
    if (a.cols <= 8192) return (void)(grad_kernel<512, 4, ODD><<<n, 512, 0, s>>>(a));
    in_grids(a.rows, [&](unsigned g, size_t done) {
        grad_stats_kernel<ODD><<<g, 1024, 0, s>>>(a, done);
    });
    const unsigned parts = (unsigned)(((size_t)a.cols + 1023) / 1024);
    grad_apply_kernel<ODD><<<n * parts, 256, 0, s>>>(a, parts, n);
}

}  // namespace

size_t rms_norm_stats(size_t rows, int cols) { return cols > kWide ? rows : 0; }

void rms_norm(const RmsNormArgs &a, hipStream_t s) {
    if (a.rows == 0 || a.cols == 0) return;
    const bool odd = a.cols % 4 || !aligned16(a.x) || !aligned16(a.residual) ||
                     !aligned16(a.gamma) || !aligned16(a.sum) || !aligned16(a.out);
    if (a.out)
        odd ? norm_any<true, false>(a, s) : norm_any<false, false>(a, s);
    else
        odd ? norm_any<true, true>(a, s) : norm_any<false, true>(a, s);
}

size_t rms_norm_grad_parts(size_t rows, int cols, int num_cus) {
    // (wide rows: so many shares for each group of 1024 columns)
    const size_t groups = cols > kWideGrad ? ((size_t)cols + 1023) / 1024 : 1;
    const size_t per_cu = cols <= 256 ? 16 : cols <= 1024 ? 8 : cols <= 4096 ? 4 : 2;
    return std::min(rows, std::max((size_t)num_cus * per_cu / groups, (size_t)1));
}
size_t rms_norm_grad_stats(size_t rows, int cols) { return cols > kWideGrad ? 2 * rows : 0; }

void rms_norm_grad(const RmsNormGradArgs &a, int num_cus, hipStream_t s) {
    if (a.rows == 0 || a.cols == 0) return;
    const bool odd = a.cols % 4 || !aligned16(a.h) || !aligned16(a.gamma) ||
                     !aligned16(a.grad_out) || !aligned16(a.grad_sum) || !aligned16(a.grad_h) ||
                     !aligned16(a.part);
    odd ? grad_any<true>(a, num_cus, s) : grad_any<false>(a, num_cus, s);
}

}  // namespace k
}  // namespace clove
