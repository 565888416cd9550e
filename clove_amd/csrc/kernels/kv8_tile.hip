// kv8_tile.hip -- attention of many query rows over the 8-bit paged cache:
// prompts, chunks of prompts, and the weights of their blocks.
//
// A workgroup takes a tile of 64 * NR query rows of one kv head (a wave 16 * NR
// of them) and walks the tokens they see in steps.  A step's codes are widened
// to bf16 once for the whole tile, on their way to LDS: the keys as rows, the
// values as columns of eight tokens; the next step's codes are on their way from
// memory meanwhile.  The products are those of kv8_stream.hip (S^T = K Q^T with
// q, O^T = V^T P^T with P, as three bf16 pieces each), and an operand read from
// LDS feeds 3 * NR MFMAs.  Where the exponents of the keys' tiles and the magnitudes
// within each row of q lie close enough together, which is nearly always, the
// scores take f16 in the place of bf16: two pieces of 11 bits hold q to 2^-23 of
// itself, two thirds of the MFMAs.  P stays in bf16: f16 ends at 2^-24, and a weight
// that far below the largest is all there is where the tokens ahead have no value.
//
// A prompt of 4096 rows, 32 heads of 128, takes 69 GFLOP for the scores and as many
// for the sums over V, in two and three pieces: 270 us at the 1271 TFLOP/s of a large
// bf16 product; 313 to 322 us measured, from box to box (all in bf16 pieces 333).  The
// MFMAs take 47% of the SIMDs' cycles there, and the time has followed their number
// (five pieces for four: 1.19 times the time).  Scores and weights stay in registers:
// S^T leaves the MFMA in the layout that P^T enters it.  What the vector units do
// between (the exponentials, the pieces of P, the widening of codes) runs beside the
// other workgroup's MFMAs.
#include <algorithm>
#include <type_traits>

#include "bf16x3.h"
#include "kv8.h"
#include "wave.h"

namespace clove {
namespace k {

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ cl_f4 mfma(u4 a, u4 b, cl_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a),
                                                   __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

// Eight dims of a query row times `scale`, in pieces.
__device__ __forceinline__ void split_q(const cl_f4 (&x)[2], float scale, u4 (&w)[3]) {
    const cl_f4 lo = x[0] * scale, hi = x[1] * scale;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        unsigned w1, w2, w3;
        split_pair<false>(e < 2 ? lo[2 * e] : hi[2 * e - 4], e < 2 ? lo[2 * e + 1] : hi[2 * e - 3],
                          &w1, &w2, &w3);
        w[0][e] = w1;
        w[1][e] = w2;
        w[2][e] = w3;
    }
}

__device__ __forceinline__ cl_f4 mfma_half(u4 a, u4 b, cl_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a),
                                                  __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
template <bool HALF>
__device__ __forceinline__ cl_f4 product(u4 a, u4 b, cl_f4 c) {
    return HALF ? mfma_half(a, b, c) : mfma(a, b, c);
}

// Two codes times a power of two: as two bf16, or as two f16 (exact where the
// result's bits are 2^-24 or more).
template <bool HALF, bool HIGH>
__device__ __forceinline__ unsigned widen(unsigned codes, float scale) {
    if constexpr (HALF)
        return __builtin_bit_cast(unsigned,
                                  __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HIGH));
    else
        return kv8_widen<HIGH>(codes, scale);
}

// Two floats as f16 and the rest of each as f16: off by at most 2^-23 of it, and
// by 2^-25 where that is more.
__device__ __forceinline__ void split_half(float a, float b, unsigned *w1, unsigned *w2) {
    const unsigned h = __builtin_bit_cast(unsigned, __builtin_convertvector((f2){a, b}, h2));
    float ra, rb;  // a - the low half of h, b - the high half
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(h), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=v"(rb)
        : "v"(h), "v"(b));
    *w1 = h;
    *w2 = __builtin_bit_cast(unsigned, __builtin_convertvector((f2){ra, rb}, h2));
}

// The table of tokens [c0, c1), rounded up to whole steps: the row of each four
// tokens' first and the scales of its key and value tile as bf16, 0 outside the
// pool.  Tokens behind the end take the first place.  True: some are outside.
// range (-1000s before): the keys' largest exponent and their least one's
// negative.
__device__ __forceinline__ int fill_table(const Kv8Args &c, int b, int h, int c0, int c1,
                                          int step, uint2 *table, int *range = nullptr) {
    int bad = 0, ends[2] = {-1000, -1000};
    for (int i = threadIdx.x; i < (c1 - c0 + step - 1) / step * (step / 4); i += 256) {
        const int t = c0 + 4 * i < c1 ? c0 + 4 * i : c0;
        const int64_t id = kv8_block(c, b, t / c.block_size, h == 0);
        uint2 e = {0, 0};
        if (id >= 0) {
            e.x = (unsigned)((id * c.num_heads + h) * c.block_size + t % c.block_size);
            e.y = __float_as_uint(kv8_scale(c.exps[kv8_tile(c, 0, id, h)])) |
                  __float_as_uint(kv8_scale(c.exps[kv8_tile(c, 1, id, h)])) >> 16;
            const int ke = (int)(e.y >> 23) - 127;
            ends[0] = max(ends[0], ke);
            ends[1] = max(ends[1], -ke);
        }
        bad |= id < 0;
        table[i] = e;
    }
    if (range) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) ends[j] = max(ends[j], __shfl_xor(ends[j], o, 64));
            if ((threadIdx.x & 63) == 0) atomicMax(&range[j], ends[j]);
        }
    }
    return bad;
}

// FULL: head_dim = DP; else MFMA steps and blocks past it are left out.
// HALF: q in two f16 pieces; a workgroup whose keys or rows do not let it leaves
// its run to the bf16 form (p.declined), which otherwise finds nothing to do.
// SUMS: the weights of every 16 tokens go out, for kv8_late_weights.
template <int DP, int NR, bool FULL, bool HALF, bool SUMS>
__global__ void __launch_bounds__(256, 2) tile_kernel(Kv8Attention a, Kv8Split p) {
    constexpr int KI = DP / 32;               // MFMA steps of q . k
    constexpr int KB = DP > 128 ? 32 : 64;    // tokens of a step
    constexpr int JB = DP / 16;               // 16-dim blocks of O^T
    constexpr int JG = FULL ? 4 : 2;          // of them at a time
    // (rows of operands start four banks apart; what conflicts remain take 12% of the
    // CUs' cycles in that prompt)
    constexpr int PK = 2 * DP + 16, PV = 2 * KB + 16;  // LDS pitches
    constexpr int NK = KB * DP / 16 / 256;    // 16-byte pieces of keys a thread stages
    constexpr int JV = DP * KB / 4 / 256;     // dims of four tokens' values a thread stages
    // tokens whose rows the table holds (two workgroups to a CU in any case)
    constexpr int kChunk = DP > 128 ? 2048 : 4096;
    static_assert(NK >= 1 && (JV == 4 || JV == 8), "256 threads stage a step");
    const Kv8Args &c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int H = c.num_heads, G = a.q_heads / H, D = c.head_dim, bs = c.block_size;
    __shared__ uint2 table[kChunk / 4];
    __shared__ __attribute__((aligned(16))) uint8_t sK[2][KB * PK], sV[2][DP * PV];
    __shared__ int s_wave[4], s_range[4];  // (the last two: bad; lost, as a float's bits)
    __shared__ Kv8Place s_place;

    if ((int)blockIdx.x >= p.grid) {
        kv8_zero_rows(a, blockIdx.x - p.grid);
        return;
    }
    int *declined = reinterpret_cast<int *>(a.ws + p.declined_at) + blockIdx.x;
    if (HALF) {
        if (tid == 0) *declined = 0;
    } else if (*declined == 0) {
        return;
    }
    Kv8Place at;
    int left, run = 0;
    if (p.join) {
        at = kv8_find_place(c, G, H, p.tile, p.step, p.extra, p.grid, blockIdx.x, s_wave, &s_place);
        run = min(at.share, at.total - at.share * (int)blockIdx.x);
        left = run;
        if (blockIdx.x == 0 && tid == 0)
            reinterpret_cast<int *>(a.ws + p.start_at)[0] = at.share;
    } else {
        // a tile to a workgroup; a sequence's last tiles, the longest, first
        at.h = blockIdx.x % H;
        at.b = kv8_slot(c, p.grid / H - 1 - blockIdx.x / H, p.tile, G, 1, &at.item);
        at.step = 0;
        at.share = 0;
        left = 1;
    }
    while (left > 0) {
        Kv8Tile T;
        if (p.join) {
            if (!kv8_next_tile(c, G, H, p.tile, &at, &T)) return;
        } else if (!kv8_tile_of(c, G, at.b, at.item, p.tile, &T) || T.high <= 0) {
            return;
        }
        const int h = at.h, all = kv8_steps(T.high, KB);
        if (p.join && at.step < p.extra) {
            left -= p.extra - at.step;
            if (left <= 0) return;
            at.step = p.extra;
        }
        const int s0 = p.join ? at.step - p.extra : 0, s1 = p.join ? min(all, s0 + left) : all;
        const int t_end = min(s1 * KB, T.high);
        if (p.join && s0 == 0 && tid == 0)
            reinterpret_cast<int *>(a.ws + p.start_at)
                [1 + (size_t)(kv8_first_slot(c, at.b, p.tile, G, 1) + at.item) * H + h] =
                    at.share * (int)blockIdx.x + (run - left);

        // this wave's rows, and the tokens each sees
        int lim[NR], lift[NR];
        size_t rowhead[NR];
        auto load_q = [&](int cc, int i, cl_f4 (&x)[2]) {
            const int d = 32 * i + 8 * q;
            x[0] = x[1] = (cl_f4){0.f, 0.f, 0.f, 0.f};
            if (16 * (NR * wave + cc) + r < T.rows && d < D) {
                const cl_f4 *from = reinterpret_cast<const cl_f4 *>(a.q + rowhead[cc] * D + d);
                x[0] = from[0];
                x[1] = from[1];
            }
        };
#pragma unroll
        for (int cc = 0; cc < NR; ++cc) {
            const int u = 16 * (NR * wave + cc) + r;
            const bool ok = u < T.rows;
            const int tok = (T.r0 + (ok ? u : 0)) / G, g = (T.r0 + (ok ? u : 0)) % G;
            lim[cc] = ok ? min(t_end, T.ctx - T.n + tok + 1) : 0;
            rowhead[cc] = (size_t)(T.first + tok) * a.q_heads + h * G + g;
        }
        const int u0 = 16 * NR * wave;  // tokens that all the wave's rows see, and that any does
        const int low = u0 < T.rows ? T.ctx - T.n + (T.r0 + u0) / G + 1 : 0;
        const int high =
            u0 < T.rows ? min(t_end, T.ctx - T.n + (T.r0 + min(u0 + 16 * NR, T.rows) - 1) / G + 1) : 0;

        // [kv head][16 tokens][(row, query head) pair of the call]
        const size_t pairs = (size_t)c.rows * G;
        float2 *sums = reinterpret_cast<float2 *>(a.ws + p.sums_at) +
                       (size_t)h * p.groups * pairs + (size_t)T.first * G + T.r0 + u0 + r;
        float m[NR], l[NR];
        cl_f4 o[NR][JB];
#pragma unroll
        for (int cc = 0; cc < NR; ++cc) {
            m[cc] = -INFINITY;
            l[cc] = 0.0f;
#pragma unroll
            for (int jb = 0; jb < JB; ++jb) o[cc][jb] = (cl_f4){0.f, 0.f, 0.f, 0.f};
        }

        // what this thread stages: NK pieces of keys, JV dims of a quad's values
        const int vquad = tid % (KB / 4), vdim = tid / (KB / 4) * JV;
        const uint8_t *vbase =
            c.codes + (size_t)c.num_blocks * H * bs * D + (vdim < D ? vdim : 0);
        // tokens 4 * (vquad % 4) + i of half (vquad / 4) % 2 of 32 tokens: the
        // order of S^T's elements in a lane, twice four of them
        const int vpos = vquad / 8 * 32 + vquad % 4 * 8 + vquad / 4 % 2 * 4;

        // the table of the chunk from c0 on, whole at the next barrier
        auto next_table = [&](int c0) {
            if (tid < 4) s_range[tid] = tid < 2 ? -1000 : 0;
            __syncthreads();  // the table and tiles before are done with
            const int c1 = min(c0 + kChunk, t_end);
            if (__any(fill_table(c, at.b, h, c0, c1, KB, table, s_range)) && lane == 0)
                s_range[2] = 1;
        };
        // the rows' loads run beside the table's
        u4 qf[NR][KI][HALF ? 2 : 3];
        {
            cl_f4 raw[NR][KI][2];
#pragma unroll
            for (int cc = 0; cc < NR; ++cc)
#pragma unroll
                for (int i = 0; i < KI; ++i) load_q(cc, i, raw[cc][i]);
            next_table(s0 * KB);
#pragma unroll
            for (int cc = 0; cc < NR; ++cc) {
                if constexpr (!HALF) {
#pragma unroll
                    for (int i = 0; i < KI; ++i)
                        split_q(raw[cc][i], a.scale * kLog2e, qf[cc][i]);
                } else {
                    // A row is lifted to 2^14 .. 2^15.  Elements below 2^-17 of its
                    // largest then lose bits: each is off by up to 2^-39 of the
                    // largest, `lost` times 2^-39 together.
                    float most = 0.0f;
#pragma unroll
                    for (int i = 0; i < KI; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            raw[cc][i][e / 4][e & 3] *= a.scale * kLog2e;  // (weights: powers of 2)
                            const float y = fabsf(raw[cc][i][e / 4][e & 3]);
                            if (kv8_finite(y)) most = fmaxf(most, y);
                        }
                    most = fmaxf(most, __shfl_xor(most, 16, 64));
                    most = fmaxf(most, __shfl_xor(most, 32, 64));
                    int small = 0;
#pragma unroll
                    for (int i = 0; i < KI; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float y = fabsf(raw[cc][i][e / 4][e & 3]);
                            small += y > 0.0f && y < most * 0x1p-17f;
                        }
                    small += __shfl_xor(small, 16, 64);
                    small += __shfl_xor(small, 32, 64);
                    lift[cc] = min(14 + 127 - (int)(__float_as_uint(most) >> 23), 100);
                    if (q == 0)
                        atomicMax(&s_range[3],
                                  __float_as_int(lift[cc] < -60 ? INFINITY : small * most));
                    const float up = kv8_pow2(max(lift[cc], -126));
#pragma unroll
                    for (int i = 0; i < KI; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            unsigned w1, w2;
                            split_half(raw[cc][i][e / 2][2 * (e & 1)] * up,
                                       raw[cc][i][e / 2][2 * (e & 1) + 1] * up, &w1, &w2);
                            qf[cc][i][0][e] = w1;
                            qf[cc][i][1][e] = w2;
                        }
                }
            }
        }
        __syncthreads();
        const float lost = HALF ? __int_as_float(s_range[3]) : 0.0f;

        for (int c0 = s0 * KB; c0 < t_end; c0 += kChunk) {
            const int c1 = min(c0 + kChunk, t_end);
            if (c0 != s0 * KB) {
                next_table(c0);
                __syncthreads();
            }
            const bool bad = s_range[2];
            // f16 holds codes times 2^(exponent - the largest + 7) exactly over 22
            // octaves of the tiles' exponents; with rows lifted likewise, two pieces
            // do what three bf16 ones do, if what the rows lost moves no score
            // (base 2) by more than 2^-22, a quarter of a weight's ulp.
            const int ke = s_range[0];
            if (HALF && (ke == -1000 || ke > 60 || ke + s_range[1] > 22 ||
                         lost * (0x1p-17f * kE4m3Max) * kv8_pow2(ke) > 1.0f)) {
                if (tid == 0) *declined = 1;
                return;
            }
            const float k_down = HALF ? kv8_pow2(7 - ke) : 1.0f;
            // A score's factor.  Never 0, which a masked score's -infinity would make
            // NaN: below 2^-126 (rows of zeros over keys of zeros) the sums, 2^39 at
            // most, come to nothing under either factor.
            float down[NR];
#pragma unroll
            for (int cc = 0; cc < NR; ++cc)
                down[cc] = HALF ? fmaxf(kv8_pow2(ke - 7) * kv8_pow2(-lift[cc]), 0x1p-126f) : 1.0f;
            u4 rk[NK];
            unsigned rv[4][JV / 4];
            float ksc[NK], vsc;
            auto load = [&](int kb) {
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    const int x = tid + 256 * i, key = x / (DP / 16), d = x % (DP / 16) * 16;
                    const uint2 e = table[(kb - c0 + key) >> 2];
                    ksc[i] = __uint_as_float(e.y & 0xffff0000u);
                    if (HALF) ksc[i] *= k_down;
                    // (past D, where q is 0, the row's first dims stand in)
                    rk[i] = *reinterpret_cast<const u4 *>(
                        c.codes + (size_t)(e.x + (key & 3)) * D + (d < D ? d : 0));
                }
                const uint2 e = table[((kb - c0) >> 2) + vquad];
                vsc = __uint_as_float(e.y << 16);
                const uint8_t *row = vbase + (size_t)e.x * D;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (JV == 8) {
                        const uint2 w = *reinterpret_cast<const uint2 *>(row + i * D);
                        rv[i][0] = w.x;
                        rv[i][1] = w.y;
                    } else {
                        rv[i][0] = *reinterpret_cast<const unsigned *>(row + i * D);
                    }
                }
            };
            auto store = [&](int kb, int buf) {
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    const int x = tid + 256 * i, key = x / (DP / 16), d = x % (DP / 16) * 16;
                    u4 w[2];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        w[e / 2][2 * (e & 1)] = widen<HALF, false>(rk[i][e], ksc[i]);
                        w[e / 2][2 * (e & 1) + 1] = widen<HALF, true>(rk[i][e], ksc[i]);
                    }
                    u4 *to = reinterpret_cast<u4 *>(&sK[buf][key * PK + 2 * d]);
                    to[0] = w[0];
                    to[1] = w[1];
                }
                if (bad || kb + KB > c1) {
                    // codes that nothing wrote may be NaN: 0 * NaN would stay
                    asm volatile("");
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (vsc == 0.0f || kb + 4 * vquad + i >= c1)
#pragma unroll
                            for (int e = 0; e < JV / 4; ++e) rv[i][e] = 0;
                }
#pragma unroll
                for (int e = 0; e < JV / 4; ++e)
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        unsigned w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            w[i] = hi ? kv8_widen<true>(rv[i][e], vsc) : kv8_widen<false>(rv[i][e], vsc);
                        uint8_t *to = &sV[buf][(vdim + 4 * e + 2 * hi) * PV + 2 * vpos];
                        *reinterpret_cast<uint2 *>(to) =
                            make_uint2(__builtin_amdgcn_perm(w[1], w[0], 0x05040100u),
                                       __builtin_amdgcn_perm(w[3], w[2], 0x05040100u));
                        *reinterpret_cast<uint2 *>(to + PV) =
                            make_uint2(__builtin_amdgcn_perm(w[1], w[0], 0x07060302u),
                                       __builtin_amdgcn_perm(w[3], w[2], 0x07060302u));
                    }
            };

            load(c0);
            store(c0, 0);
            __syncthreads();
            int buf = 0;
            for (int kb = c0; kb < c1; kb += KB, buf ^= 1) {
                const bool more = kb + KB < c1;
                if (more) load(kb + KB);
#pragma unroll 1
                for (int sub = 0; sub < KB / 32; ++sub) {
                    const int t0 = kb + 32 * sub;
                    if (t0 >= high) break;
                    cl_f4 s[NR][2];
#pragma unroll
                    for (int cc = 0; cc < NR; ++cc)
#pragma unroll
                        for (int u = 0; u < 2; ++u) s[cc][u] = (cl_f4){0.f, 0.f, 0.f, 0.f};
                    // raised priority over the MFMAs: the other wave of the SIMD does
                    // its softmax, conversions and loads in the gaps
                    __builtin_amdgcn_s_setprio(1);
#pragma unroll
                    for (int i = 0; i < KI; ++i) {
                        if (!FULL && 32 * i >= D) break;
                        u4 kf[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            kf[u] = *reinterpret_cast<const u4 *>(
                                &sK[buf][(32 * sub + 16 * u + r) * PK + 64 * i + 16 * q]);
#pragma unroll
                        for (int x = HALF ? 1 : 2; x >= 0; --x)
#pragma unroll
                            for (int cc = 0; cc < NR; ++cc)
#pragma unroll
                                for (int u = 0; u < 2; ++u)
                                    s[cc][u] = product<HALF>(kf[u], qf[cc][i][x], s[cc][u]);
                    }
                    __builtin_amdgcn_s_setprio(0);
                    if (bad || t0 + 32 > min(low, c1)) {
                        asm volatile("");  // (a branch, not selects that every step pays for)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const bool in = table[((t0 - c0) >> 2) + 4 * u + q].y != 0;
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int cc = 0; cc < NR; ++cc)
                                    if (!in || t0 + 16 * u + 4 * q + i >= lim[cc])
                                        s[cc][u][i] = -INFINITY;
                        }
                    }
                    u4 pf[NR][3];
#pragma unroll
                    for (int cc = 0; cc < NR; ++cc) {
                        float top = -INFINITY;
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int i = 0; i < 4; ++i) top = fmaxf(top, s[cc][u][i]);
                        if (HALF) top *= down[cc];
                        if (__any(top > m[cc] + kKv8Slack)) {
                            // a row moves its maximum by its own scores alone, so
                            // that its bits do not depend on the rows beside it
                            top = fmaxf(top, __shfl_xor(top, 16, 64));
                            top = fmaxf(top, __shfl_xor(top, 32, 64));
                            const float m_new = top > m[cc] + kKv8Slack ? top : m[cc];
                            const float f0 =
                                m_new == m[cc] ? 1.0f : __builtin_amdgcn_exp2f(m[cc] - m_new);
                            l[cc] *= f0;
#pragma unroll
                            for (int jb = 0; jb < JB; ++jb) o[cc][jb] *= f0;
                            m[cc] = m_new;
                        }
                        const float mz = m[cc] == -INFINITY ? 0.0f : m[cc];
                        float part_sum[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                s[cc][u][i] = __builtin_amdgcn_exp2f(
                                    HALF ? fmaf(s[cc][u][i], down[cc], -mz) : s[cc][u][i] - mz);
                            part_sum[u] = hsum4(s[cc][u]);
                            l[cc] += part_sum[u];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                unsigned w1, w2, w3;
                                split_pair<false>(s[cc][u][2 * e], s[cc][u][2 * e + 1], &w1, &w2,
                                                  &w3);
                                pf[cc][0][2 * u + e] = w1;
                                pf[cc][1][2 * u + e] = w2;
                                pf[cc][2][2 * u + e] = w3;
                            }
                        }
                        if constexpr (SUMS) {
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                part_sum[u] += __shfl_xor(part_sum[u], 16, 64);
                                part_sum[u] += __shfl_xor(part_sum[u], 32, 64);
                            }
                            if (q < 2 && t0 + 16 * q < lim[cc])
                                sums[(size_t)(t0 / 16 + q) * pairs + 16 * cc] =
                                    make_float2(part_sum[q], m[cc]);
                        }
                    }
                    __builtin_amdgcn_s_setprio(1);
#pragma unroll
                    for (int jb = 0; jb < JB; jb += JG) {
                        if (!FULL && 16 * jb >= D) break;
                        u4 v[JG];
#pragma unroll
                        for (int i = 0; i < JG; ++i)
                            v[i] = *reinterpret_cast<const u4 *>(
                                &sV[buf][(16 * (jb + i) + r) * PV + 64 * sub + 16 * q]);
#pragma unroll
                        for (int x = 2; x >= 0; --x)
#pragma unroll
                            for (int cc = 0; cc < NR; ++cc)
#pragma unroll
                                for (int i = 0; i < JG; ++i)
                                    o[cc][jb + i] = mfma(v[i], pf[cc][x], o[cc][jb + i]);
                    }
                }
                __builtin_amdgcn_s_setprio(0);
                if (more) store(kb + KB, buf ^ 1);
                __syncthreads();
            }
        }

        const bool whole = s0 == 0 && s1 == all;
        const size_t piece = (size_t)(2 * blockIdx.x + (s0 == 0 ? 1 : 0)) * p.stored;
#pragma unroll
        for (int cc = 0; cc < NR; ++cc) {
            float ls = l[cc];
            ls += __shfl_xor(ls, 16, 64);
            ls += __shfl_xor(ls, 32, 64);
            const int u = 16 * (NR * wave + cc) + r;
            if (u >= T.rows) continue;
            const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
            float *to = whole ? a.out + rowhead[cc] * D : a.ws + p.o_at + (piece + u) * D;
            const float f = whole ? inv : 1.0f;
#pragma unroll
            for (int jb = 0; jb < JB; ++jb)
                if (DP == 64 ? 16 * jb < D : 16 * jb + 4 * q < D)
                    *reinterpret_cast<cl_f4 *>(to + 16 * jb + 4 * q) = o[cc][jb] * f;
            if (q == 0) {
                if (!whole)
                    reinterpret_cast<float2 *>(a.ws + p.ml_at)[piece + u] = make_float2(m[cc], ls);
                else if (a.w_out)
                    reinterpret_cast<float2 *>(a.ws + p.row_ml_at)[rowhead[cc]] =
                        make_float2(m[cc], inv);
            }
        }
        left -= p.join ? s1 - s0 : 1;
        at.step = 0;
        ++at.h;
    }
}

// The attention weight of every four tokens, summed over the rows and the heads
// of a group: a workgroup takes 256 tokens of one kv head, a wave 64 of them as
// MFMA operands in registers, and walks the rows that see them, 32 at a time, in
// pieces through LDS (the next 32 on their way meanwhile).  A row's weights are
// 2^(s - m) / sum.  Long runs of rows are cut into parts of kPart pairs, each with
// sums of its own.  One launch is for tokens [t0, t1), a range of whole blocks.
constexpr int kPart = kKv8WeightPart;
template <int DP>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2)
    tile_weights_kernel(Kv8Attention a, Kv8Split p, int t0, int t1) {
    constexpr int KI = DP / 32;
    const Kv8Args &c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int H = c.num_heads, G = a.q_heads / H, D = c.head_dim;
    const int h = blockIdx.y, slot = blockIdx.z, c0 = t0 + blockIdx.x * 256;
    constexpr int NQ = (2 * KI * 64 + 255) / 256;  // eight dims of a row each
    __shared__ uint2 table[64];
    __shared__ u4 sq[2][2 * KI * 3 * 64];
    __shared__ float2 s_ml[2][32];
    __shared__ int s_lim[2][32];
    int part;
    const int b = kv8_slot(c, slot, kPart, G, 1, &part);
    int first, n;
    kv8_rows(c, b, &first, &n);
    const int ctx = kv8_context(c, b), c1 = min(c0 + 256, min(t1, ctx));
    if (part < 0 || part * kPart >= n * G || c0 >= c1) return;
    const int bad = __syncthreads_or(fill_table(c, b, 0, c0, c1, 256, table));
    // the keys: token 16u + r of the wave's, dims 32i + 8q .. + 7
    u4 kf[4][KI];
    bool in[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int t = 64 * wave + 16 * u + r;
        const uint2 e0 = table[t >> 2];
        // (the table is head 0's)
        const uint8_t *row =
            c.codes + ((size_t)e0.x + (size_t)h * c.block_size + (t & 3)) * D;
        const int tt = c0 + t < c1 ? c0 + t : c0;
        const int64_t id = kv8_block(c, b, tt / c.block_size, false);
        const float sc = id >= 0 ? kv8_scale(c.exps[kv8_tile(c, 0, id, h)]) : 0.0f;
#pragma unroll
        for (int i = 0; i < KI; ++i) {
            const int d = 32 * i + 8 * q;
            const uint2 w = *reinterpret_cast<const uint2 *>((id >= 0 ? row : c.codes) + (d < D ? d : 0));
            kf[u][i] = (u4){kv8_widen<false>(w.x, sc), kv8_widen<true>(w.x, sc),
                            kv8_widen<false>(w.y, sc), kv8_widen<true>(w.y, sc)};
        }
        in[u] = table[(64 * wave + 16 * u + 4 * q) >> 2].y != 0;
    }
    cl_f4 sum[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) sum[u] = (cl_f4){0.f, 0.f, 0.f, 0.f};
    // from the first row that sees the tokens' first
    const int u_end = min((part + 1) * kPart, n * G);
    int u0 = max(part * kPart, max(c0 - (ctx - n), 0) * G);
    cl_f4 raw[NQ][2];
    float2 ml_next;
    int lim_next;
    auto load = [&](int u0) {
#pragma unroll
        for (int y = 0; y < NQ; ++y) {
            const int x = tid + 256 * y;
            const int lr = x & 15, lq = x >> 4 & 3, i = (x >> 6) % KI, cc = x / (64 * KI);
            const int u = u0 + 16 * cc + lr, d = 32 * i + 8 * lq;
            raw[y][0] = raw[y][1] = (cl_f4){0.f, 0.f, 0.f, 0.f};
            if (x < 2 * KI * 64 && u < u_end && d < D) {
                const cl_f4 *qr = reinterpret_cast<const cl_f4 *>(
                    a.q + ((size_t)(first + u / G) * a.q_heads + h * G + u % G) * D + d);
                raw[y][0] = qr[0];
                raw[y][1] = qr[1];
            }
        }
        const int u = u0 + tid;
        lim_next = tid < 32 && u < u_end ? min(c1, ctx - n + u / G + 1) : 0;
        ml_next = make_float2(0.f, 0.f);
        if (lim_next > 0)
            ml_next = reinterpret_cast<const float2 *>(
                a.ws + p.row_ml_at)[(size_t)(first + u / G) * a.q_heads + h * G + u % G];
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int y = 0; y < NQ; ++y) {
            const int x = tid + 256 * y;
            if (x >= 2 * KI * 64) continue;
            u4 w[3];
            split_q(raw[y], a.scale * kLog2e, w);
#pragma unroll
            for (int z = 0; z < 3; ++z) sq[buf][((x >> 6) * 3 + z) * 64 + (x & 63)] = w[z];
        }
        if (tid < 32) {
            s_lim[buf][tid] = lim_next;
            s_ml[buf][tid] = ml_next;
        }
    };
    if (u0 < u_end) {
        load(u0);
        store(0);
    }
    __syncthreads();
    for (int buf = 0; u0 < u_end; u0 += 32, buf ^= 1) {
        if (u0 + 32 < u_end) load(u0 + 32);
        cl_f4 s[2][4];
#pragma unroll
        for (int cc = 0; cc < 2; ++cc)
#pragma unroll
            for (int u = 0; u < 4; ++u) s[cc][u] = (cl_f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KI; ++i) {
            if (32 * i >= D) break;
#pragma unroll
            for (int x = 2; x >= 0; --x)
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                    const u4 qf = sq[buf][((cc * KI + i) * 3 + x) * 64 + lane];
#pragma unroll
                    for (int u = 0; u < 4; ++u) s[cc][u] = mfma(kf[u][i], qf, s[cc][u]);
                }
        }
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
            const float2 ml = s_ml[buf][16 * cc + r];
            const float mz = ml.x == -INFINITY ? 0.0f : ml.x;
            const int lim = s_lim[buf][16 * cc + r];
            // (rows that no query is count nothing by their 0)
            if (bad || c0 + 64 * wave + 64 > min(c1, ctx - n + u0 / G + 1)) {
                asm volatile("");  // (a branch, not selects that every step pays for)
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!in[u] || c0 + 64 * wave + 16 * u + 4 * q + i >= lim)
                            s[cc][u][i] = -INFINITY;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sum[u][i] = fmaf(__builtin_amdgcn_exp2f(s[cc][u][i] - mz), ml.y, sum[u][i]);
        }
        if (u0 + 32 < u_end) store(buf ^ 1);
        __syncthreads();
    }
    float *out = a.ws + p.sums_at + ((size_t)slot * H + h) * p.groups;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        float x = hsum4(sum[u]);
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) x += __shfl_xor(x, o, 64);
        const int t = c0 + 64 * wave + 16 * u + 4 * q;
        if (r == 0 && t < c1) out[(t - t0) >> 2] = x;
    }
}

// The quads' sums of all parts and heads into the weights of blocks [j0, j1); lanes
// take 64 blocks, the sixteen waves the parts and heads in turn.
__global__ void __launch_bounds__(1024)
    block_weights_kernel(Kv8Attention a, Kv8Split p, int j0, int j1) {
    const Kv8Args &c = a.c;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int j = j0 + blockIdx.x * 64 + lane, b = blockIdx.y, per = c.block_size / 4;
    __shared__ float part[16][64];
    const int ctx = kv8_context(c, b);
    int first, n;
    kv8_rows(c, b, &first, &n);
    float w = 0.0f;
    if (n > 0 && j < j1 && j * c.block_size < ctx) {
        const int G = a.q_heads / c.num_heads, quads = min(per, (ctx - j * c.block_size + 3) / 4);
        const int parts = (n * G + kPart - 1) / kPart;
        const size_t slot = kv8_first_slot(c, b, kPart, G, 1);
        for (int x = wave; x < parts * c.num_heads; x += 16) {
            const float *y = a.ws + p.sums_at + (slot * c.num_heads + x) * p.groups + (size_t)(j - j0) * per;
#pragma unroll 4
            for (int i = 0; i < quads; ++i) w += y[i];
        }
    }
    part[wave][lane] = w;
    __syncthreads();
    if (wave == 0 && j < j1) {
        const size_t at = (size_t)b * c.max_blocks + j;
        for (int x = 1; x < 16; ++x) w += part[x][lane];
        a.w_out[at] = a.w_in[at] + w;
    }
}

// The weights of the blocks from the sums that the tiles stored: a workgroup takes
// the blocks of about 64 tokens, four sums of 16 tokens at a time; the lanes take
// pairs of rows and heads, the waves 64 pairs of one kv head in turn.
__global__ void __launch_bounds__(1024) sums_weights_kernel(Kv8Attention a, Kv8Split p, int blocks) {
    const Kv8Args &c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int H = c.num_heads, G = a.q_heads / H, per = c.block_size / 16;
    const int b = blockIdx.y, j0 = blockIdx.x * blocks, g1 = min(j0 + blocks, c.max_blocks) * per;
    __shared__ float part[16][4], total;
    const int ctx = kv8_context(c, b);
    int first, n;
    kv8_rows(c, b, &first, &n);
    const size_t pairs = (size_t)c.rows * G;
    const float2 *row_ml = reinterpret_cast<const float2 *>(a.ws + p.row_ml_at);
    const float2 *sums = reinterpret_cast<const float2 *>(a.ws + p.sums_at) + (size_t)first * G;
    if (tid == 0) total = 0.0f;
    for (int g0 = j0 * per; g0 < g1; g0 += 4) {
        // from the first row that sees any of the tokens
        const int past = ctx - n, R = n * G, low = max(16 * g0 - past, 0) * G / 64;
        const int chunks = 16 * g0 < ctx ? (R + 63) / 64 - low : 0;
        float w[4] = {};
        for (int x0 = wave; x0 < chunks * H; x0 += 64) {  // four at a time on their way
            float2 ml[4], v[4][4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int x = x0 + 16 * y, h = x / chunks, u = 64 * (low + x % chunks) + lane;
                const int see = x < chunks * H && u < R ? past + u / G + 1 : 0;
                if (see > 16 * g0)
                    ml[y] = row_ml[(size_t)(first + u / G) * a.q_heads + h * G + u % G];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[y][i] = make_float2(0.0f, -INFINITY);
                    if (g0 + i < g1 && 16 * (g0 + i) < see)
                        v[y][i] = sums[((size_t)h * p.groups + g0 + i) * pairs + u];
                }
            }
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!kv8_empty(make_float2(v[y][i].y, v[y][i].x)))
                        w[i] = fmaf(v[y][i].x, __builtin_amdgcn_exp2f(v[y][i].y - ml[y].x) * ml[y].y,
                                    w[i]);
        }
        __syncthreads();  // the four before are done with
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) w[i] += __shfl_xor(w[i], o, 64);
            if (lane == 0) part[wave][i] = w[i];
        }
        __syncthreads();
        if (tid == 0)
            for (int i = 0; i < 4 && g0 + i < g1; ++i) {
                for (int x = 0; x < 16; ++x) total += part[x][i];
                if ((g0 + i + 1) % per == 0) {
                    const size_t at = (size_t)b * c.max_blocks + (g0 + i) / per;
                    a.w_out[at] = a.w_in[at] + total;
                    total = 0.0f;
                }
            }
    }
}

}  // namespace

void kv8_tiles(const Kv8Attention &a, const Kv8Split &p, hipStream_t s) {
    auto launch = [&](auto full, auto half, auto sums) {
        constexpr bool F = decltype(full)::value, HALF = decltype(half)::value;
        constexpr bool S = decltype(sums)::value;
        const unsigned grid = p.grid + (HALF ? kv8_zero_grid(a.c) : 0);
        if (p.dp == 256)
            tile_kernel<256, 1, F, HALF, S><<<grid, 256, 0, s>>>(a, p);
        else if (p.dp == 128 && p.tile == 128)
            tile_kernel<128, 2, F, HALF, S><<<grid, 256, 0, s>>>(a, p);
        else if (p.dp == 128)
            tile_kernel<128, 1, F, HALF, S><<<grid, 256, 0, s>>>(a, p);
        else if (p.tile == 128)
            tile_kernel<64, 2, F, HALF, S><<<grid, 256, 0, s>>>(a, p);
        else
            tile_kernel<64, 1, F, HALF, S><<<grid, 256, 0, s>>>(a, p);
    };
    auto go = [&](auto full, auto half) {
        if (p.sums)
            launch(full, half, std::true_type{});
        else
            launch(full, half, std::false_type{});
    };
    if (a.c.head_dim == p.dp) {
        go(std::true_type{}, std::true_type{});
        go(std::true_type{}, std::false_type{});
    } else {
        go(std::false_type{}, std::true_type{});
        go(std::false_type{}, std::false_type{});
    }
}

void kv8_late_weights(const Kv8Attention &a, const Kv8Split &p, hipStream_t s) {
    const Kv8Args &c = a.c;
    if (p.sums) {
        const int blocks = std::max(1, 64 / c.block_size);
        sums_weights_kernel<<<dim3((c.max_blocks + blocks - 1) / blocks, c.num_seqs), 1024, 0, s>>>(
            a, p, blocks);
        return;
    }
    const int per = p.range / c.block_size;
    const unsigned parts = (unsigned)kv8_slots(c, kPart, a.q_heads / c.num_heads, 1);
    for (int j0 = 0; j0 < c.max_blocks; j0 += per) {
        const int n = std::min(per, c.max_blocks - j0), t0 = j0 * c.block_size;
        const int t1 = t0 + n * c.block_size;
        const dim3 grid((n * c.block_size + 255) / 256, c.num_heads, parts);
        if (p.dp == 64) tile_weights_kernel<64><<<grid, 256, 0, s>>>(a, p, t0, t1);
        if (p.dp == 128) tile_weights_kernel<128><<<grid, 256, 0, s>>>(a, p, t0, t1);
        if (p.dp == 256) tile_weights_kernel<256><<<grid, 256, 0, s>>>(a, p, t0, t1);
        block_weights_kernel<<<dim3((n + 63) / 64, c.num_seqs), 1024, 0, s>>>(a, p, j0, j0 + n);
    }
}

}  // namespace k
}  // namespace clove
