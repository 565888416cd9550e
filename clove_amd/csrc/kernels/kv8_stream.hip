// kv8_stream.hip -- attention of a few query rows over the 8-bit paged cache:
// decode steps, grouped heads, a handful of speculated tokens.
//
// Tiles of up to 16 * NC query rows of one kv head, their contexts in steps of
// 128 tokens, and every workgroup an equal run of all steps (Kv8Split): ragged
// batches keep every CU busy to the end.  Of a step each of the four waves takes
// 32 tokens and streams their codes from memory into the operands of
// v_mfma_f32_16x16x32_bf16:
//   S^T = K Q^T    A: lane (r, q) holds token r's dims 64s + 16q .. + 15 (one
//                  16-byte load, two MFMA steps; q is laid out alike),
//                  B: the 16 rows' q as three bf16 pieces, which hold all 24 bits;
//   O^T += V^T P^T A: lane (r, q) holds dims (DP/16) r .. of the eight tokens
//                  4q + i and 16 + 4q + i, paired up by byte permutes; these are
//                  the tokens of the lane's own S^T elements, so P^T needs no
//                  exchange between lanes; P in three bf16 pieces.
// A code times its tile's power of two is exact in bf16, so the conversion
// applies the scale, and products are those of 32-bit values with f32 sums.
#include "bf16x3.h"
#include "kv8.h"
#include "wave.h"

namespace clove {
namespace k {

namespace {

constexpr int kChunk = 4096;    // tokens whose rows a workgroup's table holds
constexpr int kMaxGrid = 1024;   // workgroups that share the steps
constexpr float kSlack = 8.0f;  // a maximum moves when a score exceeds it by this (base 2)

template <int BYTES>
struct Row {
    unsigned w[BYTES / 4];
};

__device__ __forceinline__ u4 load16(const uint8_t *p) {
    return __builtin_nontemporal_load(reinterpret_cast<const u4 *>(p));
}
template <int BYTES>
__device__ __forceinline__ Row<BYTES> load_row(const uint8_t *p) {
    if constexpr (BYTES == 4)
        return {{__builtin_nontemporal_load(reinterpret_cast<const unsigned *>(p))}};
    else if constexpr (BYTES == 8) {
        typedef unsigned u2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(Row<8>,
                                  __builtin_nontemporal_load(reinterpret_cast<const u2 *>(p)));
    } else
        return __builtin_bit_cast(Row<16>, load16(p));
}

template <bool HIGH>
__device__ __forceinline__ unsigned widen(unsigned codes, float scale) {
    return __builtin_bit_cast(unsigned,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
}

__device__ __forceinline__ cl_f4 mfma(u4 a, u4 b, cl_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a),
                                                   __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

// Steps of a tile whose last row sees `high` tokens.
__device__ __forceinline__ int steps_of(int high) { return (max(high, 0) + kKv8Step - 1) / kKv8Step; }

// Where a workgroup's run of steps begins.
struct Place {
    int b, item, h, step;
    int64_t share, total;
};

// All 256 threads: the steps before each sequence are summed up (in one order
// everywhere), and step `share * w` is looked up in them.
__device__ __forceinline__ Place find_place(const Kv8Args &c, int G, int tile, int grid, int w,
                                            int64_t *s_wave, Place *s_place) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, H = c.num_heads;
    const int per = (c.num_seqs + 255) / 256;
    auto steps = [&](int b) {
        int64_t sum = 0;
        Kv8Tile t;
        for (int item = 0; kv8_tile_of(c, G, b, item, tile, &t); ++item) sum += steps_of(t.high);
        return sum * H;
    };
    int64_t mine = 0;
    for (int b = tid * per; b < min((tid + 1) * per, c.num_seqs); ++b) mine += steps(b);
    int64_t inc = mine;
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t up = __shfl_up(inc, o, 64);
        if (lane >= o) inc += up;
    }
    if (lane == 63) s_wave[wave] = inc;
    if (tid == 0) s_place->b = -1;
    __syncthreads();
    const int64_t total = s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
    int64_t at = inc - mine;
    for (int i = 0; i < wave; ++i) at += s_wave[i];
    const int64_t share = max((total + grid - 1) / grid, (int64_t)1);
    const int64_t want = share * w;
    if (want >= at && want < at + mine) {
        for (int b = tid * per; b < min((tid + 1) * per, c.num_seqs); ++b) {
            Kv8Tile t;
            for (int item = 0; kv8_tile_of(c, G, b, item, tile, &t); ++item) {
                const int n = steps_of(t.high);
                if (want >= at && want < at + (int64_t)n * H) {
                    s_place->b = b;
                    s_place->item = item;
                    s_place->h = (int)((want - at) / n);
                    s_place->step = (int)((want - at) % n);
                }
                at += (int64_t)n * H;
            }
        }
    }
    __syncthreads();
    Place p = *s_place;
    p.share = share;
    p.total = total;
    return p;
}

template <int DP, int NC, int SUMS>
__global__ void __launch_bounds__(256, DP * NC > 128 ? 2 : 3)
    stream_kernel(Kv8Attention a, Kv8Split p) {
    constexpr int KS = DP / 64;  // 16-byte loads of a token's key
    constexpr int JB = DP / 16;  // dims a lane holds of a token's value
    constexpr int kPitch = DP + 4;
    const Kv8Args &c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int H = c.num_heads, G = a.q_heads / H, D = c.head_dim, bs = c.block_size;
    __shared__ union {
        struct {
            // four tokens: the row of the first ((block * H + h) * bs + slot) and
            // the scales of its key and value tile as bf16, 0 outside the pool
            uint2 table[kChunk / 4];
            u4 q[NC * 2 * KS * 3 * 64];
        } t;
        float o[4][16][kPitch];
    } sh;
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ int64_t s_wave[4];
    __shared__ Place s_place;

    if ((int)blockIdx.x >= p.grid) {
        // rows of no sequence, or without a token to see
        const int r0 = ((int)blockIdx.x - p.grid) * 4 + wave;
        if (blockIdx.x == (unsigned)p.grid && wave == 0) kv8_check(c);
        if (r0 >= c.rows) return;
        const int b = kv8_seq_of_row(c, r0);
        int see = 0;
        if (b >= 0) {
            int first, n;
            kv8_rows(c, b, &first, &n);
            see = kv8_context(c, b) - n + (r0 - first) + 1;
        }
        if (see <= 0)
            for (int d = lane; d < a.q_heads * D; d += 64)
                a.out[(size_t)r0 * a.q_heads * D + d] = 0.0f;
        return;
    }
    Place at = find_place(c, G, p.tile, p.grid, blockIdx.x, s_wave, &s_place);
    int64_t *starts = reinterpret_cast<int64_t *>(a.ws + p.start_at);
    if (p.join && blockIdx.x == 0 && tid == 0) starts[0] = at.share;
    int64_t left = min(at.share, at.total - at.share * blockIdx.x);
    bool front = true;

    while (left > 0) {
        // the next tile with steps
        Kv8Tile T;
        if (at.h >= H) {
            at.h = 0;
            ++at.item;
        }
        while (at.b < c.num_seqs) {
            if (!kv8_tile_of(c, G, at.b, at.item, p.tile, &T)) {
                ++at.b;
                at.item = 0;
            } else if (T.high <= 0) {
                ++at.item;
            } else {
                break;
            }
        }
        if (at.b >= c.num_seqs) return;  // (there are as many steps as were counted)
        const int h = at.h, all = steps_of(T.high);
        const int s0 = at.step, s1 = (int)min((int64_t)all, s0 + left);
        const int t_end = min(s1 * kKv8Step, T.high);
        const int64_t run0 = at.share * blockIdx.x + (min(at.share, at.total - at.share * blockIdx.x) - left);
        if (p.join && s0 == 0 && tid == 0)
            starts[1 + (size_t)(kv8_first_slot(c, at.b, p.tile, G, 1) + at.item) * H + h] = run0;

        // q times scale * log2(e) (weights are powers of two), in pieces
        __syncthreads();
        for (int x = tid; x < NC * 2 * KS * 64; x += 256) {
            const int lr = x & 15, lq = x >> 4 & 3, s = (x >> 6) % (2 * KS), cc = x / (128 * KS);
            const int u = 16 * cc + lr, d = 64 * (s / 2) + 16 * lq + 8 * (s & 1);
            cl_f4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
            if (u < T.rows && d < D) {
                const int tok = (T.r0 + u) / G, g = (T.r0 + u) % G;
                const cl_f4 *qr = reinterpret_cast<const cl_f4 *>(
                    a.q + ((size_t)(T.first + tok) * a.q_heads + h * G + g) * D + d);
                lo = qr[0] * (a.scale * 1.44269504088896341f);
                hi = qr[1] * (a.scale * 1.44269504088896341f);
            }
            u4 w[3];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                unsigned w1, w2, w3;
                split_pair<false>(e < 2 ? lo[2 * e] : hi[2 * e - 4],
                                  e < 2 ? lo[2 * e + 1] : hi[2 * e - 3], &w1, &w2, &w3);
                w[0][e] = w1;
                w[1][e] = w2;
                w[2][e] = w3;
            }
#pragma unroll
            for (int i = 0; i < 3; ++i)
                sh.t.q[((cc * 2 * KS + s) * 3 + i) * 64 + (x & 63)] = w[i];
        }
        int lim[NC];           // tokens each row sees
        unsigned rowhead[NC];
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) {
            const int u = 16 * cc + r;
            const bool ok = u < T.rows;
            const int tok = (T.r0 + (ok ? u : 0)) / G, g = (T.r0 + (ok ? u : 0)) % G;
            lim[cc] = ok ? min(t_end, T.ctx - T.n + tok + 1) : 0;
            rowhead[cc] = (T.first + tok) * a.q_heads + h * G + g;
        }

        float m[NC], l[NC];
        cl_f4 o[NC][JB];
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) {
            m[cc] = -INFINITY;
            l[cc] = 0.0f;
#pragma unroll
            for (int jb = 0; jb < JB; ++jb) o[cc][jb] = (cl_f4){0.f, 0.f, 0.f, 0.f};
        }
        float2 *sums = reinterpret_cast<float2 *>(a.ws + p.sums_at);
        const uint8_t *kbase = c.codes;
        int koff[KS];  // (q is 0 past D, where the row's first dims stand in)
#pragma unroll
        for (int i = 0; i < KS; ++i) koff[i] = 64 * i + 16 * q < D ? 64 * i + 16 * q : 0;
        const uint8_t *vbase = c.codes + (size_t)c.num_blocks * H * bs * D + (JB * r < D ? JB * r : 0);

        for (int c0 = s0 * kKv8Step; c0 < t_end; c0 += kChunk) {
            const int c1 = min(c0 + kChunk, t_end);
            if (c0 > s0 * kKv8Step) __syncthreads();  // the chunk before is done with
            // tokens behind the end take the chunk's first place (and no part in
            // what follows), so that every load lies in the pool
            int bad = 0;
            for (int i = tid; i < (c1 - c0 + kKv8Step - 1) / kKv8Step * (kKv8Step / 4); i += 256) {
                const int t = c0 + 4 * i < c1 ? c0 + 4 * i : c0;
                const int64_t id = kv8_block(c, at.b, t / bs, h == 0);
                uint2 e = {0, 0};
                if (id >= 0) {
                    e.x = (unsigned)((id * H + h) * bs + t % bs);
                    e.y = __float_as_uint(kv8_scale(c.exps[kv8_tile(c, 0, id, h)])) |
                          __float_as_uint(kv8_scale(c.exps[kv8_tile(c, 1, id, h)])) >> 16;
                }
                bad |= id < 0;
                sh.t.table[i] = e;
            }
            bad = __syncthreads_or(bad);

            u4 kk[2][KS];
            Row<JB> vv[8];
            float ks[2], vs[2];
            bool in[2];
            auto load_k = [&](int kb) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint2 e = sh.t.table[(kb - c0 + 16 * u + r) >> 2];
                    ks[u] = __uint_as_float(e.y & 0xffff0000u);
                    const uint8_t *row = kbase + (size_t)(e.x + (r & 3)) * D;
#pragma unroll
                    for (int i = 0; i < KS; ++i) kk[u][i] = load16(row + koff[i]);
                }
            };
            auto load_v = [&](int kb) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint2 e = sh.t.table[((kb - c0) >> 2) + 4 * u + q];
                    vs[u] = __uint_as_float(e.y << 16);
                    in[u] = e.y != 0;
                    const uint8_t *row = vbase + (size_t)e.x * D;
#pragma unroll
                    for (int i = 0; i < 4; ++i) vv[4 * u + i] = load_row<JB>(row + i * D);
                }
            };
            int kb = c0 + 32 * wave;
            if (kb < c1) {
                load_k(kb);
                load_v(kb);
            }
            for (; kb < c1; kb += kKv8Step) {
                const bool more = kb + kKv8Step < c1;
                cl_f4 s[NC][2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int cc = 0; cc < NC; ++cc) s[cc][u] = (cl_f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 2 * KS; ++i) {
                    u4 kf[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const unsigned w0 = kk[u][i / 2][2 * (i & 1)], w1 = kk[u][i / 2][2 * (i & 1) + 1];
                        kf[u] = (u4){widen<false>(w0, ks[u]), widen<true>(w0, ks[u]),
                                     widen<false>(w1, ks[u]), widen<true>(w1, ks[u])};
                    }
#pragma unroll
                    for (int cc = 0; cc < NC; ++cc)
#pragma unroll
                        for (int x = 2; x >= 0; --x) {
                            const u4 qf = sh.t.q[((cc * 2 * KS + i) * 3 + x) * 64 + lane];
#pragma unroll
                            for (int u = 0; u < 2; ++u) s[cc][u] = mfma(kf[u], qf, s[cc][u]);
                        }
                }
                if (more) load_k(kb + kKv8Step);
                if (bad || kb + 32 > min(T.low, c1)) {
                    asm volatile("");  // (a branch, not selects that every step pays for)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int t = kb + 16 * u + 4 * q + i;
#pragma unroll
                            for (int cc = 0; cc < NC; ++cc)
                                if (!in[u] || t >= lim[cc]) s[cc][u][i] = -INFINITY;
                            // codes that nothing wrote may be NaN: 0 * NaN would stay
                            if (!in[u] || t >= c1) vv[4 * u + i] = Row<JB>{};
                        }
                }
                u4 pf[NC][3];
#pragma unroll
                for (int cc = 0; cc < NC; ++cc) {
                    float top = -INFINITY;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[cc][u][i]);
                    if (__any(top > m[cc] + kSlack)) {
                        // a row moves its maximum by its own scores alone, so that
                        // its bits do not depend on the rows beside it
                        top = fmaxf(top, __shfl_xor(top, 16, 64));
                        top = fmaxf(top, __shfl_xor(top, 32, 64));
                        const float m_new = top > m[cc] + kSlack ? top : m[cc];
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
                            s[cc][u][i] = __builtin_amdgcn_exp2f(s[cc][u][i] - mz);
                        part_sum[u] = hsum4(s[cc][u]);
                        l[cc] += part_sum[u];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            unsigned w1, w2, w3;
                            split_pair<false>(s[cc][u][2 * e], s[cc][u][2 * e + 1], &w1, &w2, &w3);
                            pf[cc][0][2 * u + e] = w1;
                            pf[cc][1][2 * u + e] = w2;
                            pf[cc][2][2 * u + e] = w3;
                        }
                    }
                    if constexpr (SUMS != 0) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            float x = part_sum[u];
                            if (SUMS == 16) {
                                x += __shfl_xor(x, 16, 64);
                                x += __shfl_xor(x, 32, 64);
                            }
                            const int t = kb + 16 * u + (SUMS == 4 ? 4 * q : 0);
                            if ((SUMS == 4 || q == 0) && t < lim[cc])
                                sums[(size_t)rowhead[cc] * p.groups + t / SUMS] =
                                    make_float2(x, m[cc]);
                        }
                    }
                }
                // four dims of the eight tokens at a time
#pragma unroll
                for (int jb = 0; jb < JB; jb += 4) {
                    u4 v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float sc = vs[e / 2];
                        const unsigned wa = vv[2 * e].w[jb / 4], wb = vv[2 * e + 1].w[jb / 4];
                        const unsigned xa = widen<false>(wa, sc), xb = widen<false>(wb, sc);
                        const unsigned ya = widen<true>(wa, sc), yb = widen<true>(wb, sc);
                        v[0][e] = __builtin_amdgcn_perm(xb, xa, 0x05040100u);
                        v[1][e] = __builtin_amdgcn_perm(xb, xa, 0x07060302u);
                        v[2][e] = __builtin_amdgcn_perm(yb, ya, 0x05040100u);
                        v[3][e] = __builtin_amdgcn_perm(yb, ya, 0x07060302u);
                    }
#pragma unroll
                    for (int cc = 0; cc < NC; ++cc)
#pragma unroll
                        for (int x = 2; x >= 0; --x)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                o[cc][jb + i] = mfma(v[i], pf[cc][x], o[cc][jb + i]);
                }
                if (more) load_v(kb + kKv8Step);
            }
        }

        // join the four waves
        const bool whole = s0 == 0 && s1 == all;
        const size_t piece = (size_t)(2 * blockIdx.x + (front ? 0 : 1)) * p.stored;
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) {
            float ls = l[cc];
            ls += __shfl_xor(ls, 16, 64);
            ls += __shfl_xor(ls, 32, 64);
            __syncthreads();  // the tables, or the rows before, are done with
            if (q == 0) {
                s_m[wave][r] = m[cc];
                s_l[wave][r] = ls;
            }
            __syncthreads();
            const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
            const float f0 = m[cc] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[cc] - top);
            // element i of block jb is dim JB * (4q + i) + jb of row r
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int jb = 0; jb < JB; jb += 4) {
                    const cl_f4 x = {o[cc][jb][i] * f0, o[cc][jb + 1][i] * f0,
                                     o[cc][jb + 2][i] * f0, o[cc][jb + 3][i] * f0};
                    *reinterpret_cast<cl_f4 *>(&sh.o[wave][r][JB * (4 * q + i) + jb]) = x;
                }
            __syncthreads();
            const int D4 = D / 4;
            for (int x = tid; x < 16 * D4; x += 256) {
                const int row = x / D4, d = 4 * (x - row * D4);
                const int u = 16 * cc + row;
                if (u >= T.rows) break;
                cl_f4 sum = {0.f, 0.f, 0.f, 0.f};
                float mm = -INFINITY, ll = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) mm = fmaxf(mm, s_m[w][row]);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    sum += *reinterpret_cast<const cl_f4 *>(&sh.o[w][row][d]);
                    const float fw = s_m[w][row] == -INFINITY
                                         ? 0.0f
                                         : __builtin_amdgcn_exp2f(s_m[w][row] - mm);
                    ll += s_l[w][row] * fw;
                }
                if (whole) {
                    const int tok = (T.r0 + u) / G, g = (T.r0 + u) % G;
                    const size_t rh = (size_t)(T.first + tok) * a.q_heads + h * G + g;
                    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
                    *reinterpret_cast<cl_f4 *>(a.out + rh * D + d) = sum * inv;
                    if (SUMS && d == 0)
                        reinterpret_cast<float2 *>(a.ws + p.row_ml_at)[rh] = make_float2(mm, inv);
                } else {
                    *reinterpret_cast<cl_f4 *>(a.ws + p.o_at + (piece + u) * D + d) = sum;
                    if (d == 0)
                        reinterpret_cast<float2 *>(a.ws + p.ml_at)[piece + u] = make_float2(mm, ll);
                }
            }
        }
        left -= s1 - s0;
        front = false;
        at.step = 0;
        ++at.h;
    }
}

// Joins the pieces of one row and query head, the workgroup's waves in turn, a
// lane up to four dims.
__global__ void __launch_bounds__(1024) join_kernel(Kv8Attention a, Kv8Split p) {
    const Kv8Args &c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    const int hq = blockIdx.x % a.q_heads, row = blockIdx.x / a.q_heads;
    const int D = c.head_dim, H = c.num_heads, G = a.q_heads / H, h = hq / G;
    __shared__ float s_o[16][kKv8MaxHeadDim], s_f[kMaxGrid], s_l[16], s_top[16];
    const int b = kv8_seq_of_row(c, row);
    if (b < 0) return;
    int first, n;
    kv8_rows(c, b, &first, &n);
    const int u = (row - first) * G + hq % G;
    Kv8Tile T;
    if (!kv8_tile_of(c, G, b, u / p.tile, p.tile, &T) || T.high <= 0) return;
    const int64_t *starts = reinterpret_cast<const int64_t *>(a.ws + p.start_at);
    const int64_t share = starts[0];
    const size_t slot = kv8_first_slot(c, b, p.tile, G, 1) + u / p.tile;
    const int64_t start = starts[1 + slot * H + h], end = start + steps_of(T.high);
    const int64_t w0 = start / share;
    const int np = (int)((end - 1) / share - w0) + 1;
    if (np == 1) return;  // written whole
    // the first piece ends its workgroup's run unless the run begins with it
    auto place = [&](int i) {
        const int64_t w = w0 + i;
        return (size_t)(2 * w + (i == 0 && start != w * share ? 1 : 0)) * p.stored + u % p.tile;
    };
    const float2 *ml = reinterpret_cast<const float2 *>(a.ws + p.ml_at);
    float top = -INFINITY, x[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.0f;
    for (int i = tid; i < np; i += blockDim.x) {
        s_f[i] = ml[place(i)].x;
        top = fmaxf(top, s_f[i]);
    }
    top = wave_max(top);
    if (lane == 0) s_top[wave] = top;
    __syncthreads();
    for (int w = 0; w < waves; ++w) top = fmaxf(top, s_top[w]);
    for (int i = tid; i < np; i += blockDim.x) {
        const float f = s_f[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_f[i] - top);
        l += ml[place(i)].y * f;
        s_f[i] = f;
    }
    l = wave_sum(l);
    __syncthreads();
    const float *o = a.ws + p.o_at;
#pragma unroll 4
    for (int i = wave; i < np; i += waves) {
        const float f = s_f[i], *oi = o + place(i) * D;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (lane + 64 * e < D) x[e] = fmaf(oi[lane + 64 * e], f, x[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < D) s_o[wave][lane + 64 * e] = x[e];
    if (lane == 0) s_l[wave] = l;
    __syncthreads();
    l = 0.0f;
    for (int w = 0; w < waves; ++w) l += s_l[w];
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const size_t rh = (size_t)row * a.q_heads + hq;
    for (int d = tid; d < D; d += blockDim.x) {
        float sum = 0.0f;
        for (int w = 0; w < waves; ++w) sum += s_o[w][d];
        a.out[rh * D + d] = sum * inv;
    }
    if (tid == 0 && p.sums) reinterpret_cast<float2 *>(a.ws + p.row_ml_at)[rh] = make_float2(top, inv);
}

template <int DP, int NC>
void launch(const Kv8Attention &a, const Kv8Split &p, unsigned grid, hipStream_t s) {
    switch (p.sums) {
    case 0: stream_kernel<DP, NC, 0><<<grid, 256, 0, s>>>(a, p); break;
    case 4: stream_kernel<DP, NC, 4><<<grid, 256, 0, s>>>(a, p); break;
    default: stream_kernel<DP, NC, 16><<<grid, 256, 0, s>>>(a, p);
    }
}

}  // namespace

int kv8_stream_residents(int dp, int tile) { return dp * tile > 128 * 16 ? 2 : 3; }

void kv8_stream(const Kv8Attention &a, const Kv8Split &p, hipStream_t s) {
    const unsigned grid = p.grid + (a.c.rows + 3) / 4;
    if (p.tile == 16) {
        if (p.dp == 64) launch<64, 1>(a, p, grid, s);
        if (p.dp == 128) launch<128, 1>(a, p, grid, s);
        if (p.dp == 256) launch<256, 1>(a, p, grid, s);
    } else {
        if (p.dp == 64) launch<64, 2>(a, p, grid, s);
        if (p.dp == 128) launch<128, 2>(a, p, grid, s);
    }
    if (p.join) {
        // one workgroup a row and head; many waves where few rows have many pieces
        const unsigned n = (unsigned)a.c.rows * a.q_heads;
        join_kernel<<<n, n <= 64 ? 1024 : n <= 1024 ? 256 : 64, 0, s>>>(a, p);
    }
}

}  // namespace k
}  // namespace clove
