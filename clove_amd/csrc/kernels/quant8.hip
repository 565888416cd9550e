// quant8.hip -- f32 matrices as e4m3 codes with power-of-two block scales.
//
//   e = the smallest exponent in [-100, 119] with amax <= 448 * 2^e over the
//       block's finite elements, code = round_e4m3(x * 2^-e)
//
// Scaling by a power of two is exact, so every element is rounded once and codes
// and exponents are determined to the bit.
//
// A workgroup takes a tile of 128 x 128 elements: thread t holds four columns of
// sixteen consecutive rows (64 floats), so that a row of the tile is 512
// consecutive bytes of a half wave, its codes 128, and a column's sixteen codes one
// 16-byte piece of the transposed tile, which goes through LDS to leave in lines.
#include <algorithm>

#include "linear8.h"

namespace clove {
namespace k {

namespace {

typedef unsigned lin8_u4 __attribute__((ext_vector_type(4)));

template <bool ODD, bool TILES>
__global__ void __launch_bounds__(256) quantize_kernel(Quant8Args a, size_t col_tiles,
                                                       size_t done) {
    __shared__ unsigned tops[8][128];
    __shared__ lin8_u4 codes_t[128][8];
    const size_t tile = done + blockIdx.x;
    const size_t row0 = tile / col_tiles * 128, col0 = tile % col_tiles * 128;
    const int t = threadIdx.x, l = t & 31, group = t >> 5;
    const size_t kp = (a.cols + 127) / 128 * 128, rp = (a.rows + 127) / 128 * 128;
    const int left = (int)min((size_t)128, a.cols - col0);       // columns of the tile
    const int rows = (int)min((size_t)128, a.rows - row0);       // and its rows
    cl_f4 x[16];
    const float *src = a.x + row0 * a.cols + col0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = group * 16 + i;
        x[i] = (cl_f4){0.f, 0.f, 0.f, 0.f};
        if (r < rows) x[i] = lin8_load4<ODD>(src + (size_t)r * a.cols, l, left);
    }
    int e_tile = 0;
    if constexpr (TILES) {
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, lin8_mag4(x[i]));
        top = half_umax(top);
        if (l == 0) tops[group][0] = top;
        __syncthreads();
#pragma unroll
        for (int g = 0; g < 8; ++g) top = max(top, tops[g][0]);
        e_tile = lin8_exp_of(top);
    }
    if (a.codes) {
        if (TILES && t == 0) a.exps[row0 / 128 * (kp / 128) + col0 / 128] = e_tile;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = group * 16 + i;
            const int e = TILES ? e_tile : lin8_exp_of(half_umax(lin8_mag4(x[i])));
            if (r >= rows) continue;
            reinterpret_cast<unsigned *>(a.codes + (row0 + r) * kp + col0)[l] =
                lin8_encode4(x[i], lin8_pow2(-e));
            if (!TILES && l == 0) a.exps[(row0 + r) * (kp / 128) + col0 / 128] = e;
        }
    }
    if (!a.codes_t) return;
    int e[4] = {e_tile, e_tile, e_tile, e_tile};
    if constexpr (!TILES) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) top = max(top, lin8_mag(x[i][c]));
            tops[group][4 * l + c] = top;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            unsigned top = 0;
#pragma unroll
            for (int g = 0; g < 8; ++g) top = max(top, tops[g][4 * l + c]);
            e[c] = lin8_exp_of(top);
            if (group == 0 && 4 * l + c < left)
                a.exps_t[(col0 + 4 * l + c) * (rp / 128) + row0 / 128] = e[c];
        }
    } else if (t == 0) {
        a.exps_t[col0 / 128 * (rp / 128) + row0 / 128] = e_tile;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const float inv = lin8_pow2(-e[c]);
        lin8_u4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = lin8_encode4((cl_f4){x[4 * i][c], x[4 * i + 1][c], x[4 * i + 2][c],
                                        x[4 * i + 3][c]}, inv);
        codes_t[4 * l + c][group ^ (l & 7)] = w;  // (piece `group` of the column)
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = i * 32 + t / 8, piece = t & 7;
        if (c < left)
            *reinterpret_cast<lin8_u4 *>(a.codes_t + (col0 + c) * rp + row0 + 16 * piece) =
                codes_t[c][piece ^ ((c >> 2) & 7)];
    }
}

constexpr size_t kGrid = size_t(1) << 21;  // a grid holds 2^32 threads

}  // namespace

void quantize8(const Quant8Args &a, hipStream_t s) {
    if (a.rows == 0 || a.cols == 0 || (!a.codes && !a.codes_t)) return;
    const bool odd = a.cols % 4 || (reinterpret_cast<uintptr_t>(a.x) & 15);
    const size_t col_tiles = (a.cols + 127) / 128, n = (a.rows + 127) / 128 * col_tiles;
    const auto kernel = a.block_rows == 1 ? (odd ? quantize_kernel<true, false> : quantize_kernel<false, false>)
                                          : (odd ? quantize_kernel<true, true> : quantize_kernel<false, true>);
    for (size_t done = 0; done < n; done += kGrid)
        kernel<<<(unsigned)std::min(kGrid, n - done), 256, 0, s>>>(a, col_tiles, done);
}

}  // namespace k
}  // namespace clove
