// quant8.hip -- f32 matrices as e4m3 codes with power-of-two block scales.
//
//   e = the smallest exponent in [-100, 119] with amax <= 448 * 2^e over the
//       block's finite elements, code = round_e4m3(x * 2^-e)
//
// Scaling by a power of two is exact, so every element is rounded once and codes
// and exponents are determined to the bit.
//
// A workgroup takes a tile of 128 x 128 elements: thread t holds four columns of
// RPT consecutive rows, so that a row of the tile is 512 consecutive bytes of a half
// wave, its codes 128, and a column's RPT codes one piece of the transposed tile,
// which goes through LDS to leave in lines: x is read once for both ways.
//
// What bounds it: memory, 4096 x 14336 in 128 x 128 blocks both ways 67.4 us, 5.2 TB/s;
// 16384 x 8192 in rows both ways 157 us, 5.2 TB/s, transposed alone 134, 5.05; 2050 x 3000
// in rows both ways 11-12 us for 7.8 of bytes, 408 tiles on 256 CUs.
#include "linear8.h"

namespace clove {
namespace k {

namespace {

typedef unsigned lin8_u4 __attribute__((ext_vector_type(4)));

// Columns 4l .. 4l + 3 of rows r0 .. r0 + RPT - 1 of a tile of `rows` x `left`, zeros
// past its edges, where the addresses stay within it: with loads behind branches the
// compiler waits for some before it sends the next.
template <int RPT, bool ODD>
__device__ __forceinline__ void load_tile(const float *src, size_t cols, int l, int left, int r0,
                                          int rows, cl_f4 *x) {
    if (rows == 128 && left == 128) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const float *p = src + (size_t)(r0 + i) * cols + 4 * l;
            x[i] = ODD ? (cl_f4)*reinterpret_cast<const lin8_f4u *>(p)
                       : *reinterpret_cast<const cl_f4 *>(p);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const float *p = src + (size_t)min(r0 + i, rows - 1) * cols;
        if constexpr (ODD) {
#pragma unroll
            for (int c = 0; c < 4; ++c) x[i][c] = p[min(4 * l + c, left - 1)];
        } else {
            x[i] = *reinterpret_cast<const cl_f4 *>(p + min(4 * l, left - 4));
        }
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (r0 + i >= rows || 4 * l + c >= left) x[i][c] = 0.0f;
}

template <int T, bool ODD, bool TILES>
__global__ void __launch_bounds__(T) quantize_kernel(Quant8Args a, size_t col_tiles,
                                                     size_t done) {
    constexpr int GROUPS = T / 32, RPT = 128 / GROUPS, WORDS = RPT / 4;
    __shared__ unsigned tops[GROUPS][128];
    // column c's piece p (16 rows) lies in slot p ^ (c / 4 % 8)
    __shared__ __attribute__((aligned(16))) unsigned codes_t[128][32];
    const size_t tile = done + blockIdx.x;
    const size_t row0 = tile / col_tiles * 128, col0 = tile % col_tiles * 128;
    const int t = threadIdx.x, l = t & 31, group = t >> 5;
    const size_t kp = (a.cols + 127) / 128 * 128, rp = (a.rows + 127) / 128 * 128;
    const int left = (int)min((size_t)128, a.cols - col0);       // columns of the tile
    const int rows = (int)min((size_t)128, a.rows - row0);       // and its rows
    cl_f4 x[RPT];
    load_tile<RPT, ODD>(a.x + row0 * a.cols + col0, a.cols, l, left, group * RPT, rows, x);
    // the maxima of this thread's columns, then its rows' codes on their way while the
    // other threads' maxima arrive
    int e_tile = 0;
    lin8_u4 top = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < RPT; ++i) top[c] = max(top[c], lin8_bits(x[i][c]));
    const bool plain = lin8_plain(max(max(top[0], top[1]), max(top[2], top[3])));
    if (!plain) {
        top = (lin8_u4){0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < RPT; ++i) top[c] = max(top[c], lin8_mag(x[i][c]));
    }
    if constexpr (TILES) {
        unsigned all = half_umax(max(max(top[0], top[1]), max(top[2], top[3])));
        if (l == 0) tops[group][0] = all;
        __syncthreads();
#pragma unroll 8
        for (int g = 0; g < GROUPS; ++g) all = max(all, tops[g][0]);
        e_tile = lin8_exp_of(all);
        if (t == 0 && a.codes) a.exps[row0 / 128 * (kp / 128) + col0 / 128] = e_tile;
        if (t == 0 && a.codes_t) a.exps_t[col0 / 128 * (rp / 128) + row0 / 128] = e_tile;
    } else {
        *reinterpret_cast<lin8_u4 *>(&tops[group][4 * l]) = top;
    }
    const auto straight = [&](auto p) {
        constexpr bool P = decltype(p)::value;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int r = group * RPT + i;
            const int e = TILES ? e_tile : lin8_exp_of(half_umax(lin8_mag4<P>(x[i])));
            if (r >= rows) continue;
            reinterpret_cast<unsigned *>(a.codes + (row0 + r) * kp + col0)[l] =
                lin8_encode4<P>(x[i], lin8_pow2(-e));
            if (!TILES && l == 0) a.exps[(row0 + r) * (kp / 128) + col0 / 128] = e;
        }
    };
    if (a.codes) plain ? straight(std::true_type()) : straight(std::false_type());
    if (!a.codes_t) return;
    int e[4] = {e_tile, e_tile, e_tile, e_tile};
    if constexpr (!TILES) {
        __syncthreads();
#pragma unroll 4
        for (int g = 0; g < GROUPS; ++g) {
            const lin8_u4 other = *reinterpret_cast<const lin8_u4 *>(&tops[g][4 * l]);
#pragma unroll
            for (int c = 0; c < 4; ++c) top[c] = max(top[c], other[c]);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            e[c] = lin8_exp_of(top[c]);
            if (group == 0 && 4 * l + c < left)
                a.exps_t[(col0 + 4 * l + c) * (rp / 128) + row0 / 128] = e[c];
        }
    }
    const auto transposed = [&](auto p) {
        typedef unsigned piece __attribute__((ext_vector_type(WORDS)));
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float inv = lin8_pow2(-e[c]);
            piece w;
#pragma unroll
            for (int i = 0; i < WORDS; ++i)
                w[i] = lin8_encode4<decltype(p)::value>(
                    (cl_f4){x[4 * i][c], x[4 * i + 1][c], x[4 * i + 2][c], x[4 * i + 3][c]}, inv);
            const int word = group * WORDS;  // of the column's 32
            *reinterpret_cast<piece *>(&codes_t[4 * l + c][(word / 4 ^ (l & 7)) * 4 + word % 4]) =
                w;
        }
    };
    plain ? transposed(std::true_type()) : transposed(std::false_type());
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 1024 / T; ++i) {
        const int c = i * (T / 8) + t / 8, piece = t & 7;
        if (c < left)
            *reinterpret_cast<lin8_u4 *>(a.codes_t + (col0 + c) * rp + row0 + 16 * piece) =
                *reinterpret_cast<const lin8_u4 *>(&codes_t[c][(piece ^ (c / 4 % 8)) * 4]);
    }
}

// Blocks of one row as they stand: a half wave a block, four each, 2^lx blocks of
// a row side by side in a workgroup's 32.
template <bool ODD>
__global__ void __launch_bounds__(256) quantize_rows_kernel(Quant8Args a, size_t col_parts, int lx,
                                                            size_t done) {
    const size_t at = done + blockIdx.x;
    const size_t row0 = at / col_parts * (32 >> lx), block0 = at % col_parts << lx;
    const size_t kb = (a.cols + 127) / 128;
    const int l = threadIdx.x & 31, group = threadIdx.x >> 5;
    cl_f4 x[4];
    size_t row[4], block[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int b = group + 8 * u;
        row[u] = row0 + (b >> lx);
        block[u] = block0 + (b & ((1 << lx) - 1));
        x[u] = (cl_f4){0.f, 0.f, 0.f, 0.f};
        if (row[u] < a.rows && block[u] < kb)
            x[u] = lin8_load4<ODD>(a.x + row[u] * a.cols + block[u] * 128, l,
                                   (int)min((size_t)128, a.cols - block[u] * 128));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const auto write = [&](auto p) {
            constexpr bool P = decltype(p)::value;
            const int e = lin8_exp_of(half_umax(lin8_mag4<P>(x[u])));
            if (row[u] >= a.rows || block[u] >= kb) return;
            const size_t i = row[u] * kb + block[u];
            reinterpret_cast<unsigned *>(a.codes + i * 128)[l] =
                lin8_encode4<P>(x[u], lin8_pow2(-e));
            if (l == 0) a.exps[i] = e;
        };
        lin8_plain(lin8_bits4(x[u])) ? write(std::true_type()) : write(std::false_type());
    }
}

}  // namespace

void quantize8(const Quant8Args &a, hipStream_t s) {
    if (a.rows == 0 || a.cols == 0 || (!a.codes && !a.codes_t)) return;
    const bool odd = a.cols % 4 || !aligned16(a.x);
    const size_t col_tiles = (a.cols + 127) / 128, n = (a.rows + 127) / 128 * col_tiles;
    if (a.block_rows == 1 && !a.codes_t) {
        // [2050, 3000] 7 us, 9.6 as tiles; [16384, 8192] 5.7 TB/s
        int lx = 0;
        while (lx < 5 && (size_t(1) << lx) < col_tiles) ++lx;
        const size_t parts = (col_tiles + (1 << lx) - 1) >> lx, per = 32 >> lx;
        const auto kernel = odd ? quantize_rows_kernel<true> : quantize_rows_kernel<false>;
        lin8_grids((a.rows + per - 1) / per * parts, [&](unsigned wgs, size_t done) {
            kernel<<<wgs, 256, 0, s>>>(a, parts, lx, done);
        });
        return;
    }
    const auto kernel = a.block_rows == 1
                            ? (odd ? quantize_kernel<512, true, false> : quantize_kernel<512, false, false>)
                            : (odd ? quantize_kernel<512, true, true> : quantize_kernel<512, false, true>);
    lin8_grids(n, [&](unsigned wgs, size_t done) {
        kernel<<<wgs, 512, 0, s>>>(a, col_tiles, done);
    });
}

}  // namespace k
}  // namespace clove
