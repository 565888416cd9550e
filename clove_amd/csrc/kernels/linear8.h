// linear8.h -- what the kernels of 8-bit linear layers share: the format's
// exponents and codes (norm8.hip, quant8.hip, gemm8.hip).
//
// A matrix in 8 bits is codes [rows, Kp] (e4m3 bytes, Kp the next multiple of 128,
// zeros behind K) and exps: one exponent for each block of 128 elements of a row,
// or of 128 rows by 128 elements.  An element stands for its code times 2^exp.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "launch.hpp"
#include "wave.h"

namespace clove {
namespace k {

constexpr int kLin8MinExp = -100, kLin8MaxExp = 119;

// 2^e for e in [-126, 127].
__device__ __forceinline__ float lin8_pow2(int e) {
    return __uint_as_float((unsigned)(e + 127) << 23);
}

// |x|'s bits if x is finite, else 0: what a block's maximum is taken of.
__device__ __forceinline__ unsigned lin8_mag(float x) {
    const unsigned u = __float_as_uint(x) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}

// Most waves hold nothing past 448 * 2^119, no infinity and no NaN.  There |x|'s
// bits are lin8_mag and a code needs no clamp (PLAIN): rows of [2050, 3000] both ways
// 11.0 us a call, 12.1 where every element takes the longer way; of [4096, 11008] 55.1, 57.6.
constexpr unsigned kLin8Plain = 0x7f600000u;
__device__ __forceinline__ unsigned lin8_bits(float x) {
    return __float_as_uint(x) & 0x7fffffffu;
}
__device__ __forceinline__ unsigned lin8_bits4(cl_f4 x) {
    return max(max(lin8_bits(x.x), lin8_bits(x.y)), max(lin8_bits(x.z), lin8_bits(x.w)));
}
// Whether that holds for the whole wave, `bits` being the largest of a lane's.
__device__ __forceinline__ bool lin8_plain(unsigned bits) { return __all(bits <= kLin8Plain); }

// The smallest e in [-100, 119] with amax <= 448 * 2^e, amax >= 0 given by its
// bits.  448 = 1.75 * 2^8, so the fraction decides between exponent - 8 and - 7.
__device__ __forceinline__ int lin8_exp_of(unsigned amax) {
    const int e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, kLin8MinExp), kLin8MaxExp);
}

// x * 2^-exp (inv) on its way into a code: saturated at +-448 (which only
// magnitudes past 448 * 2^119 reach); an infinity or NaN becomes NaN by x * 0.
__device__ __forceinline__ float lin8_scaled(float x, float inv) {
    return __builtin_fmaf(x, 0.0f, __builtin_amdgcn_fmed3f(x * inv, -448.0f, 448.0f));
}

// Four elements as four codes, rounded to nearest, ties to even.
template <bool PLAIN>
__device__ __forceinline__ unsigned lin8_encode4(cl_f4 x, float inv) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = PLAIN ? x[i] * inv : lin8_scaled(x[i], inv);
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
}

template <bool PLAIN>
__device__ __forceinline__ unsigned lin8_mag4(cl_f4 x) {
    if constexpr (PLAIN) return lin8_bits4(x);
    return max(max(lin8_mag(x.x), lin8_mag(x.y)), max(lin8_mag(x.z), lin8_mag(x.w)));
}

// The maximum over the 32 lanes of each half of the wave: four rotations of 16
// lanes (row_ror 8, 4, 2, 1), then the two rows of a half against each other.
__device__ __forceinline__ unsigned half_umax(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x122, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x121, 0xf, 0xf, false));
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max((unsigned)r[0], (unsigned)r[1]);
}

// Elements 4c .. 4c + 3 of a row of `cols`, zeros past its end.  ODD: the row
// starts at any 4 bytes and ends anywhere.
typedef float lin8_f4u __attribute__((ext_vector_type(4), aligned(4)));
template <bool ODD>
__device__ __forceinline__ cl_f4 lin8_load4(const float *row, int c, int cols) {
    cl_f4 v = {0.f, 0.f, 0.f, 0.f};
    if constexpr (!ODD) {
        if (4 * c < cols) v = *reinterpret_cast<const cl_f4 *>(row + 4 * (size_t)c);
    } else {
        const float *p = row + 4 * (size_t)c;
        const int left = cols - 4 * c;
        if (left >= 4) {
            v = *reinterpret_cast<const lin8_f4u *>(p);
        } else if (left > 0) {
            v.x = p[0];
            if (left > 1) v.y = p[1];
            if (left > 2) v.z = p[2];
        }
    }
    return v;
}
template <bool ODD>
__device__ __forceinline__ void lin8_store4(float *row, int c, int cols, cl_f4 v) {
    float *p = row + 4 * (size_t)c;
    if constexpr (!ODD) {
        if (4 * c < cols) *reinterpret_cast<cl_f4 *>(p) = v;
    } else {
        const int left = cols - 4 * c;
        if (left >= 4) {
            *reinterpret_cast<lin8_f4u *>(p) = v;
        } else if (left > 0) {
            p[0] = v.x;
            if (left > 1) p[1] = v.y;
            if (left > 2) p[2] = v.z;
        }
    }
}

// A grid holds 2^32 threads: launch(workgroups, workgroups before) for n of them,
// 2^21 (of up to 1024 threads) at a time.
template <class F>
void lin8_grids(size_t n, F launch) {
    constexpr size_t most = size_t(1) << 21;
    for (size_t done = 0; done < n; done += most)
        launch((unsigned)std::min(most, n - done), done);
}

}  // namespace k
}  // namespace clove
