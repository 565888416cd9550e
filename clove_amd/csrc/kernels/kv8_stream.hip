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
constexpr int kStep = kKv8StreamStep;

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

__device__ __forceinline__ cl_f4 mfma(u4 a, u4 b, cl_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a),
                                                   __builtin_bit_cast(bf8, b), c, 0, 0, 0);
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
    __shared__ int s_wave[4];
    __shared__ Kv8Place s_place;

    if ((int)blockIdx.x >= p.grid) {
        kv8_zero_rows(a, blockIdx.x - p.grid);
        return;
    }
    Kv8Place at =
        kv8_find_place(c, G, p.tile, p.step, p.grid, blockIdx.x, s_wave, &s_place);
    int *starts = reinterpret_cast<int *>(a.ws + p.start_at);
    if (p.join && blockIdx.x == 0 && tid == 0) starts[0] = at.share;
    int left = min(at.share, at.total - at.share * (int)blockIdx.x);
    bool front = true;

    while (left > 0) {
        Kv8Tile T;
        if (!kv8_next_tile(c, G, p.tile, &at, &T)) return;
        const int h = at.h, all = kv8_steps(T.high, kStep);
        const int s0 = at.step, s1 = min(all, s0 + left);
        const int t_end = min(s1 * kStep, T.high);
        const int run0 = at.share * (int)blockIdx.x + (min(at.share, at.total - at.share * (int)blockIdx.x) - left);
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
                lo = qr[0] * (a.scale * kLog2e);
                hi = qr[1] * (a.scale * kLog2e);
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

        for (int c0 = s0 * kStep; c0 < t_end; c0 += kChunk) {
            const int c1 = min(c0 + kChunk, t_end);
            if (c0 > s0 * kStep) __syncthreads();  // the chunk before is done with
            // tokens behind the end take the chunk's first place (and no part in
            // what follows), so that every load lies in the pool
            int bad = 0;
            for (int i = tid; i < (c1 - c0 + kStep - 1) / kStep * (kStep / 4); i += 256) {
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
            for (; kb < c1; kb += kStep) {
                const bool more = kb + kStep < c1;
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
                        kf[u] = (u4){kv8_widen<false>(w0, ks[u]), kv8_widen<true>(w0, ks[u]),
                                     kv8_widen<false>(w1, ks[u]), kv8_widen<true>(w1, ks[u])};
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
                if (more) load_k(kb + kStep);
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
                    if (__any(top > m[cc] + kKv8Slack)) {
                        // a row moves its maximum by its own scores alone, so that
                        // its bits do not depend on the rows beside it
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
                        const unsigned xa = kv8_widen<false>(wa, sc), xb = kv8_widen<false>(wb, sc);
                        const unsigned ya = kv8_widen<true>(wa, sc), yb = kv8_widen<true>(wb, sc);
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
                if (more) load_v(kb + kStep);
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
    const unsigned grid = p.grid + kv8_zero_grid(a.c);
    if (p.tile == 16) {
        if (p.dp == 64) launch<64, 1>(a, p, grid, s);
        if (p.dp == 128) launch<128, 1>(a, p, grid, s);
        if (p.dp == 256) launch<256, 1>(a, p, grid, s);
    } else {
        if (p.dp == 64) launch<64, 2>(a, p, grid, s);
        if (p.dp == 128) launch<128, 2>(a, p, grid, s);
    }
}

}  // namespace k
}  // namespace clove
