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
// with g and the two sums of a row in 64 bits (h^2 leaves f32's range from 2^64 on, and g
// can where r brings grad_h back into it).
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
        const auto write = [&](auto plain) {
            constexpr bool P = decltype(plain)::value;
            const int e = lin8_exp_of(half_umax(lin8_mag4<P>(y)));
            if (4 * c >= kp) return;
            reinterpret_cast<unsigned *>(a.codes + row * kp)[c] =
                lin8_encode4<P>(y, lin8_pow2(-e));
            if ((c & 31) == 0) a.exps[row * (kp / 128) + c / 32] = e;
        };
        lin8_plain(lin8_bits4(y)) ? write(std::true_type()) : write(std::false_type());
    } else {
        lin8_store4<ODD>(a.out + row * a.cols, c, a.cols, y);
    }
}

// TR threads a row, NV chunks of four columns each, the row in registers: one pass over
// x and the residual.  Memory bounds it: 8192 x 4096 with a residual into sum and 8 bits
// 77 us, 5.6 TB/s; one row of 4096 3.3 us, most of it the launch.
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

// Rows that registers do not hold: stats[row] = r first, a workgroup a row, so that x and
// the residual are read twice: [2000, 16400] in 32 bits 77 us, 150 with the residual (3.4
// and 3.5 TB/s of what has to move), [2000, 16384] in one pass 57 and 102...
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

template <bool ODD, bool OUT8>
void norm_any(const RmsNormArgs &a, hipStream_t s) {
    // (with an 8-bit output the lanes behind the row write its padding)
    const int64_t cols = OUT8 ? ((int64_t)a.cols + 127) / 128 * 128 : a.cols;
    auto go = [&](auto kernel, int t, int tr) {
        const size_t per = t / tr;
        lin8_grids((a.rows + per - 1) / per, [&](unsigned n, size_t done) {
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
    lin8_grids(a.rows, [&](unsigned n, size_t done) {
        norm_stats_kernel<ODD><<<n, 1024, 0, s>>>(a, done);
    });
    const unsigned parts = (unsigned)((cols + 1023) / 1024);
    lin8_grids(a.rows * parts, [&](unsigned n, size_t done) {
        norm_apply_kernel<ODD, OUT8><<<n, 256, 0, s>>>(a, parts, done);
    });
}

// ---- the gradient ------------------------------------------------------------

// s + the sum of gy gamma h, gy gamma as the exact product: in 32 bits it leaves the
// range, or loses its bits below 2^-126, where r brings the gradient back.
__device__ __forceinline__ double dot(cl_f4 gy, cl_f4 gamma, cl_f4 h, double s) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        s = __builtin_fma((double)gy[e] * (double)gamma[e], (double)h[e], s);
    return s;
}

// What a row's two sums come to: r, and r^3 mean(g h).
__device__ __forceinline__ void coefficients(double sq, double gh, int cols, float eps, double *r,
                                             double *m) {
    *r = inv_rms(sq, cols, eps);
    *m = *r * *r * *r * (gh / (double)cols);
}

// Chunk c of row `row`: grad_h out, grad_out h r added to *acc; ds: grad_sum's chunk.
template <bool ODD>
__device__ __forceinline__ void grad_chunk(const RmsNormGradArgs &a, size_t row, int c, cl_f4 h,
                                           cl_f4 gy, cl_f4 ds, cl_f4 gamma, double r, double m,
                                           cl_f4 *acc) {
    cl_f4 dh;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        // (h r is at most sqrt(cols): a rounding here and one in the product)
        (*acc)[e] += gy[e] * (float)((double)h[e] * r);
        // in 64 bits where the terms meet, since they can cancel, and rounded once
        dh[e] = (float)__builtin_fma((double)gy[e] * (double)gamma[e], r,
                                     __builtin_fma(-(double)h[e], m, (double)ds[e]));
    }
    if (a.grad_h) lin8_store4<ODD>(a.grad_h + row * a.cols, c, a.cols, dh);
}

// Floats of a row of `part`: whole vectors.
__host__ __device__ __forceinline__ size_t part_pitch(int cols) {
    return ((size_t)cols + 3) / 4 * 4;
}
// Where the sums of a share of the rows go: a row of `part`, the gradient itself if
// there is one share, null if it is not wanted.
__device__ __forceinline__ float *gamma_sums(const RmsNormGradArgs &a, size_t share) {
    return a.part ? a.part + share * part_pitch(a.cols) : a.grad_gamma;
}

// TR threads a row.  A workgroup walks the rows from blockIdx.x * T / TR on, the
// next one on its way while one is reduced; its threads keep the sums of their
// columns and write them, those of its T / TR rows added up, as one row of `part`.
template <int T, int TR, int NV, bool ODD>
__global__ void __launch_bounds__(T) grad_kernel(RmsNormGradArgs a) {
    constexpr int PER = T / TR;
    __shared__ double red[2 * T / 64];
    __shared__ cl_f4 sums[PER > 1 ? PER - 1 : 1][PER > 1 ? NV * TR : 1];
    const int t = threadIdx.x % TR, mine = threadIdx.x / TR;
    cl_f4 gamma[NV], acc[NV], h[2][NV], gy[2][NV], ds[2][NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        gamma[i] = lin8_load4<ODD>(a.gamma, t + TR * i, a.cols);
        acc[i] = (cl_f4){0.f, 0.f, 0.f, 0.f};
    }
    const auto load = [&](size_t row, int s) {
        const bool in = row < a.rows;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int cols = in ? a.cols : 0, c = t + TR * i;
            h[s][i] = lin8_load4<ODD>(a.h + row * a.cols, c, cols);
            gy[s][i] = lin8_load4<ODD>(a.grad_out + row * a.cols, c, cols);
            ds[s][i] = lin8_load4<ODD>(a.grad_sum + row * a.cols, c, a.grad_sum ? cols : 0);
        }
    };
    // Long rows are widened again behind their sums: kept in 64 bits, four chunks a thread
    // spill, and of two [5000, 2100] takes 46.7 us for 45.2, [8192, 4096] 104.0 for 103.3.
    // Short rows stay as they are: [5000, 400] 11.5 for 12.2, [4000, 1500] 21.6 for 22.7.
    const auto widen_again = [&](cl_f4 (&v)[NV]) {
        if constexpr (NV > 2 || TR > 256)
#pragma unroll
            for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(v[i]));
    };
    const auto work = [&](size_t row, int s) {
        double v[2] = {0.0, 0.0};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[0] = square_sum(h[s][i], v[0]);
            v[1] = dot(gy[s][i], gamma[i], h[s][i], v[1]);
        }
        row_sum<T, TR>(v, red);
        double r, m;
        coefficients(v[0], v[1], a.cols, a.eps, &r, &m);
        widen_again(gamma);
        widen_again(gy[s]);
        widen_again(h[s]);
        if (row < a.rows)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                grad_chunk<ODD>(a, row, t + TR * i, h[s][i], gy[s][i], ds[s][i], gamma[i], r, m,
                                &acc[i]);
    };
    // (whole workgroups walk together: their barriers are in row_sum)
    const size_t step = (size_t)gridDim.x * PER;
    size_t row0 = (size_t)blockIdx.x * PER;
    load(row0 + mine, 0);
    while (true) {
        if (row0 + step < a.rows) load(row0 + step + mine, 1);
        work(row0 + mine, 0);
        if ((row0 += step) >= a.rows) break;
        if (row0 + step < a.rows) load(row0 + step + mine, 0);
        work(row0 + mine, 1);
        if ((row0 += step) >= a.rows) break;
    }
    float *const out = gamma_sums(a, blockIdx.x);
    if (!out) return;
    if constexpr (PER > 1) {
        if (mine)
#pragma unroll
            for (int i = 0; i < NV; ++i) sums[mine - 1][t + TR * i] = acc[i];
        __syncthreads();
        if (mine) return;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int w = 1; w < PER; ++w) acc[i] += sums[w - 1][t + TR * i];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) lin8_store4<ODD>(out, t + TR * i, a.cols, acc[i]);
}

// grad_gamma: the rows of `part` added up, 32 columns to a workgroup, every 128th
// row to a thread and then those in halves, in one order.  It follows the kernel whose
// rows it adds: with it a call takes 13.5 us for 8.75 at [1001, 2049] (256 rows) and 83.3
// for 79.6 at [8192, 4096]; 4.0 and 4.9 of kernel in a trace.  Launched behind itself it
// takes 2.7 for 256 or 512 rows of 2049, 2.65 and 2.9 with 64 columns to a workgroup.
__global__ void __launch_bounds__(1024) grad_join_kernel(RmsNormGradArgs a, int parts,
                                                          size_t done) {
    __shared__ cl_f4 sums[128][8];
    const size_t pitch = part_pitch(a.cols);
    const int q = threadIdx.x & 7, group = threadIdx.x >> 3;
    const size_t col0 = (done + blockIdx.x) * 32, at = col0 + 4 * q;
    cl_f4 s = {0.f, 0.f, 0.f, 0.f};
    if (at < pitch)
#pragma unroll 4
        for (int p = group; p < parts; p += 128)
            s += *reinterpret_cast<const cl_f4 *>(a.part + p * pitch + at);
    sums[group][q] = s;
    __syncthreads();
#pragma unroll
    for (int w = 64; w >= 16; w /= 2) {
        if (group < w) sums[group][q] += sums[group + w][q];
        __syncthreads();
    }
    if (threadIdx.x >= 32) return;
    const size_t col = col0 + threadIdx.x;
    float total = 0.0f;
#pragma unroll
    for (int g = 0; g < 16; ++g) total += sums[g][threadIdx.x / 4][threadIdx.x % 4];
    if (col < (size_t)a.cols) a.grad_gamma[col] = total;
}

// Rows that registers do not hold: the sums first ([2000, 16384] 131-134 us; 118 in one
// pass of 512 threads that spill, which takes 140 where these take 124 for [3000, 9001]
// and 33 where they take 27 for [300, 16380]; rows kept in LDS are not tried)...
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
        s[1] = dot(gy, lin8_load4<ODD>(a.gamma, c, a.cols), h, s[1]);
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
        const cl_f4 ds =
            lin8_load4<ODD>(a.grad_sum + row * a.cols, c, a.grad_sum ? a.cols : 0);
        grad_chunk<ODD>(a, row, c, h, gy, ds, gamma, a.stats[2 * row], a.stats[2 * row + 1], &acc);
    }
    if (float *out = gamma_sums(a, share)) lin8_store4<ODD>(out, c, a.cols, acc);
}

// Rows that a workgroup of grad_kernel takes at once, and workgroups, each a row of
// `part`.  With the next row on its way one workgroup a CU keeps the memory busy, and
// one that takes several rows leaves the join fewer to add: [1001, 2049] 12.6 us with
// two rows in 512 threads, 13.3 with one in twice the workgroups; [32768, 200] 23 with
// sixteen, 25 with four; [1554, 768] 8.0 with eight, 8.8 with four.  Many long rows go
// one by one ([8192, 4096] 101 us, 104 with two), and so do those of up to 2048
// columns, in two workgroups a CU ([4000, 1500] 23.6, 24.5).
size_t grad_rows(size_t rows, int cols, int num_cus) {
    return cols <= 128    ? 32
           : cols <= 256  ? 16
           : cols <= 1024 ? 8
           : cols > 2048 && cols <= 4096 && rows < 16 * (size_t)num_cus ? 2
                                                                        : 1;
}
size_t grad_parts(size_t rows, int cols, int num_cus) {
    const size_t cus = (size_t)num_cus, per = grad_rows(rows, cols, num_cus);
    // few rows are one share, with no join: [20, 100] and [2, 1500] 4.9 us a call for
    // 7.8, but with four turns of the workgroup [31, 1000] 9.2 and [8, 4000] 10.4
    if (rows <= 2 * per) return 1;
    if (cols > kWideGrad) {  // so many shares for each group of 1024 columns
        const size_t groups = ((size_t)cols + 1023) / 1024;
        return std::min(rows, std::max(cus * 4 / groups, (size_t)1));
    }
    return std::min((rows + per - 1) / per, cols > 1024 && cols <= 2048 ? 2 * cus : cus);
}

template <bool ODD>
void grad_any(const RmsNormGradArgs &a, size_t per, unsigned n, hipStream_t s) {
    const auto go = [&](auto kernel, int t) { kernel<<<n, t, 0, s>>>(a); };
    if (a.cols <= 128) return go(grad_kernel<1024, 32, 1, ODD>, 1024);
    if (a.cols <= 256) return go(grad_kernel<1024, 64, 1, ODD>, 1024);
    if (a.cols <= 512) return go(grad_kernel<512, 64, 2, ODD>, 512);
    if (a.cols <= 1024) return go(grad_kernel<512, 64, 4, ODD>, 512);
    if (a.cols <= 2048) return go(grad_kernel<256, 256, 2, ODD>, 256);
    if (a.cols <= 4096 && per == 2) return go(grad_kernel<512, 256, 4, ODD>, 512);
    if (a.cols <= 4096) return go(grad_kernel<512, 512, 2, ODD>, 512);
    if (a.cols <= kWideGrad) return go(grad_kernel<512, 512, 4, ODD>, 512);
    lin8_grids(a.rows, [&](unsigned g, size_t done) {
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

size_t rms_norm_grad_floats(size_t rows, int cols, int num_cus) {
    const size_t parts = grad_parts(rows, cols, num_cus);
    return parts > 1 ? parts * part_pitch(cols) : 0;
}
size_t rms_norm_grad_stats(size_t rows, int cols) { return cols > kWideGrad ? 2 * rows : 0; }

void rms_norm_grad(const RmsNormGradArgs &a, int num_cus, hipStream_t s) {
    if (a.rows == 0 || a.cols == 0) return;
    const bool odd = a.cols % 4 || !aligned16(a.h) || !aligned16(a.gamma) ||
                     !aligned16(a.grad_out) || !aligned16(a.grad_sum) || !aligned16(a.grad_h);
    const size_t per = grad_rows(a.rows, a.cols, num_cus);
    const unsigned parts = (unsigned)grad_parts(a.rows, a.cols, num_cus);
    odd ? grad_any<true>(a, per, parts, s) : grad_any<false>(a, per, parts, s);
    if (a.part)
        lin8_grids(((size_t)a.cols + 31) / 32, [&](unsigned n, size_t done) {
            grad_join_kernel<<<n, 1024, 0, s>>>(a, (int)parts, done);
        });
}

}  // namespace k
}  // namespace clove
