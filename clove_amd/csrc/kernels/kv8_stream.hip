// kv8_stream.hip -- attention of a few query rows over the 8-bit paged cache:
// decode steps, grouped heads, a handful of speculated tokens.
//
// A workgroup takes one tile of up to 16 * NC query rows of one kv head and one
// part of their context; its four waves take steps of 32 tokens in turn and each
// streams its codes straight from memory into the operands of
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

constexpr int kEntries = 1024;  // tiles of a part (kv8_plan keeps to it)
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

template <int DP, int NC, int SUMS>
__global__ void __launch_bounds__(256, DP * NC > 128 ? 1 : 2)
    stream_kernel(Kv8Attention a, Kv8Split p, unsigned main) {
    constexpr int KS = DP / 64;  // 16-byte loads of a token's key
    constexpr int JB = DP / 16;  // dims a lane holds of a token's value
    const Kv8Args &c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int H = c.num_heads, G = a.q_heads / H, D = c.head_dim, bs = c.block_size;
    constexpr int kPitch = DP + 4;
    __shared__ union {
        struct {
            int id[kEntries];
            float ks[kEntries], vs[kEntries];
        } t;
        float o[4][16][kPitch];
    } sh;
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ int s_none[256];

    if (blockIdx.x == 0 && wave == 0) kv8_check(c);
    if (blockIdx.x >= main) {  // rows of no sequence
        const int r0 = (blockIdx.x - main) * 256;
        s_none[tid] = r0 + tid < c.rows && kv8_seq_of_row(c, r0 + tid) < 0;
        __syncthreads();
        const int X = a.q_heads * D;
        for (int i = 0; i < 256; ++i)
            if (s_none[i])
                for (int d = tid; d < X; d += 256) a.out[(size_t)(r0 + i) * X + d] = 0.0f;
        return;
    }
    const int h = blockIdx.x % H, part = blockIdx.x / H % p.parts;
    const int slot = blockIdx.x / H / p.parts;
    int b;
    Kv8Tile T;
    if (!kv8_tile_of(c, G, slot, 16 * NC, &b, &T)) return;
    const int t0 = part * p.part_tokens;
    const int t1 = min(t0 + p.part_tokens, T.high);
    if (t0 >= t1 && p.parts > 1) return;

    // the part's blocks: ids (-1 outside the pool) and scales
    const int j0 = t0 / bs, nblk = t1 > t0 ? (t1 - 1) / bs - j0 + 1 : 0;
    int bad = 0;
    for (int j = tid; j < nblk; j += 256) {
        const int64_t id = kv8_block(c, b, j0 + j, h == 0);
        sh.t.id[j] = (int)id;
        bad |= id < 0;
        if (id >= 0) {
            sh.t.ks[j] = kv8_scale(c.exps[kv8_tile(c, 0, id, h)]);
            sh.t.vs[j] = kv8_scale(c.exps[kv8_tile(c, 1, id, h)]);
        } else {
            sh.t.ks[j] = sh.t.vs[j] = 1.0f;
        }
    }

    // q times scale * log2(e) (weights are powers of two), in pieces; lim: the
    // tokens each row sees of the part
    u4 qf[NC][2 * KS][3];
    int lim[NC], rowhead[NC];
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
        const int u = 16 * cc + r;
        const bool ok = u < T.rows;
        const int tok = (T.r0 + (ok ? u : 0)) / G, g = (T.r0 + (ok ? u : 0)) % G;
        lim[cc] = ok ? min(t1, T.ctx - T.n + tok + 1) : 0;
        rowhead[cc] = (T.first + tok) * a.q_heads + h * G + g;
        const float *qr = a.q + (size_t)rowhead[cc] * D;
#pragma unroll
        for (int s = 0; s < 2 * KS; ++s) {
            const int d = 64 * (s / 2) + 16 * q + 8 * (s & 1);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = 0.0f, y = 0.0f;
                if (ok && d < D) {
                    x = qr[d + 2 * e] * (a.scale * 1.44269504088896341f);
                    y = qr[d + 2 * e + 1] * (a.scale * 1.44269504088896341f);
                }
                unsigned w1, w2, w3;
                split_pair<false>(x, y, &w1, &w2, &w3);
                qf[cc][s][0][e] = w1;
                qf[cc][s][1][e] = w2;
                qf[cc][s][2][e] = w3;
            }
        }
    }
    bad = __syncthreads_or(bad);

    struct Buf {
        u4 k[2][KS];
        Row<JB> v[8];
        float ks[2], vs[2];
        bool in[2];  // the value tokens' block lies in the pool
    };
    const size_t block_bytes = (size_t)H * bs * D;
    const uint8_t *kbase = c.codes + (size_t)h * bs * D;
    const uint8_t *vbase = kbase + (size_t)c.num_blocks * block_bytes;
    const unsigned magic = (unsigned)(((1ull << 32) + bs - 1) / bs);  // bs >= 4
    const int origin = j0 * bs;
    auto load = [&](int kb, Buf &f) {
        // tokens past the part take its first token's place (and no part in
        // what follows), so that every load lies in the pool
        auto place = [&](int t, int *j, int *s) {
            const int rel = (t < t1 ? t : t0) - origin;
            *j = __umulhi(rel, magic);
            *s = rel - *j * bs;
        };
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            int j, s;
            place(kb + 16 * u + r, &j, &s);
            f.ks[u] = sh.t.ks[j];
            const uint8_t *row = kbase + (size_t)max(sh.t.id[j], 0) * block_bytes + s * D;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const int d = 64 * i + 16 * q;
                f.k[u][i] = load16(row + (d < D ? d : 0));  // (q is 0 past D)
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            int j, s;
            place(kb + 16 * u + 4 * q, &j, &s);
            const int id = sh.t.id[j];
            f.vs[u] = sh.t.vs[j];
            f.in[u] = id >= 0;
            const uint8_t *row =
                vbase + (size_t)max(id, 0) * block_bytes + (s & ~3) * D + (JB * r < D ? JB * r : 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) f.v[4 * u + i] = load_row<JB>(row + i * D);
        }
    };

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

    auto fold = [&](int kb, Buf &f) {
        cl_f4 s[NC][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int cc = 0; cc < NC; ++cc) s[cc][u] = (cl_f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 2 * KS; ++i) {
                const unsigned w0 = f.k[u][i / 2][2 * (i & 1)], w1 = f.k[u][i / 2][2 * (i & 1) + 1];
                const u4 kf = {widen<false>(w0, f.ks[u]), widen<true>(w0, f.ks[u]),
                               widen<false>(w1, f.ks[u]), widen<true>(w1, f.ks[u])};
#pragma unroll
                for (int cc = 0; cc < NC; ++cc)
#pragma unroll
                    for (int x = 2; x >= 0; --x) s[cc][u] = mfma(kf, qf[cc][i][x], s[cc][u]);
            }
        }
        if (bad || kb + 32 > min(T.low, t1)) {
            asm volatile("");  // (a branch, not selects that every step pays for)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = kb + 16 * u + 4 * q + i;
#pragma unroll
                    for (int cc = 0; cc < NC; ++cc)
                        if (!f.in[u] || t >= lim[cc]) s[cc][u][i] = -INFINITY;
                    // codes that nothing wrote may be NaN: 0 * NaN would stay
                    if (!f.in[u] || t >= t1) f.v[4 * u + i] = Row<JB>{};
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
                // a row moves its maximum by its own scores alone, so that its
                // bits do not depend on the rows beside it
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float m_new = top > m[cc] + kSlack ? top : m[cc];
                const float f0 = m_new == m[cc] ? 1.0f : __builtin_amdgcn_exp2f(m[cc] - m_new);
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
                for (int i = 0; i < 4; ++i) s[cc][u][i] = __builtin_amdgcn_exp2f(s[cc][u][i] - mz);
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
                        sums[(size_t)rowhead[cc] * p.groups + t / SUMS] = make_float2(x, m[cc]);
                }
            }
        }
        // two dims of the eight tokens at a time
#pragma unroll
        for (int jb = 0; jb < JB; jb += 2) {
            u4 v0, v1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float sc = f.vs[e / 2];
                const unsigned wa = f.v[2 * e].w[jb / 4], wb = f.v[2 * e + 1].w[jb / 4];
                const unsigned xa = jb & 2 ? widen<true>(wa, sc) : widen<false>(wa, sc);
                const unsigned xb = jb & 2 ? widen<true>(wb, sc) : widen<false>(wb, sc);
                v0[e] = __builtin_amdgcn_perm(xb, xa, 0x05040100u);
                v1[e] = __builtin_amdgcn_perm(xb, xa, 0x07060302u);
            }
#pragma unroll
            for (int cc = 0; cc < NC; ++cc)
#pragma unroll
                for (int x = 2; x >= 0; --x) {
                    o[cc][jb] = mfma(v0, pf[cc][x], o[cc][jb]);
                    o[cc][jb + 1] = mfma(v1, pf[cc][x], o[cc][jb + 1]);
                }
        }
    };

    {   // two steps of loads in flight
        Buf A, B;
        int kb = t0 + 32 * wave;
        if (kb < t1) {
            load(kb, A);
            for (;;) {
                if (kb + 128 < t1) load(kb + 128, B);
                fold(kb, A);
                kb += 128;
                if (kb >= t1) break;
                if (kb + 128 < t1) load(kb + 128, A);
                fold(kb, B);
                kb += 128;
                if (kb >= t1) break;
            }
        }
    }

    // join the four waves
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
                const cl_f4 x = {o[cc][jb][i] * f0, o[cc][jb + 1][i] * f0, o[cc][jb + 2][i] * f0,
                                 o[cc][jb + 3][i] * f0};
                *reinterpret_cast<cl_f4 *>(&sh.o[wave][r][JB * (4 * q + i) + jb]) = x;
            }
        __syncthreads();
        const int D4 = D / 4;
        const size_t base =
            (((size_t)slot * H + h) * p.parts + part) * p.stored + 16 * cc;
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
            if (p.parts == 1) {
                const int tok = (T.r0 + u) / G, g = (T.r0 + u) % G;
                const size_t rh = (size_t)(T.first + tok) * a.q_heads + h * G + g;
                const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
                *reinterpret_cast<cl_f4 *>(a.out + rh * D + d) = sum * inv;
                if (SUMS && d == 0)
                    reinterpret_cast<float2 *>(a.ws + p.row_ml_at)[rh] = make_float2(mm, inv);
            } else {
                *reinterpret_cast<cl_f4 *>(a.ws + p.o_at + (base + row) * D + d) = sum;
                if (d == 0)
                    reinterpret_cast<float2 *>(a.ws + p.ml_at)[base + row] = make_float2(mm, ll);
            }
        }
    }
}

template <int DP, int NC>
void launch(const Kv8Attention &a, const Kv8Split &p, unsigned main, unsigned grid, hipStream_t s) {
    switch (p.sums) {
    case 0: stream_kernel<DP, NC, 0><<<grid, 256, 0, s>>>(a, p, main); break;
    case 4: stream_kernel<DP, NC, 4><<<grid, 256, 0, s>>>(a, p, main); break;
    default: stream_kernel<DP, NC, 16><<<grid, 256, 0, s>>>(a, p, main);
    }
}

}  // namespace

void kv8_stream(const Kv8Attention &a, const Kv8Split &p, hipStream_t s) {
    const unsigned main = p.slots * (unsigned)p.parts * (unsigned)a.c.num_heads;
    const unsigned none = a.c.row_starts && p.parts == 1 ? (a.c.rows + 255) / 256 : 0;
    const unsigned grid = main + none;
    if (p.tile == 16) {
        if (p.dp == 64) launch<64, 1>(a, p, main, grid, s);
        if (p.dp == 128) launch<128, 1>(a, p, main, grid, s);
        if (p.dp == 256) launch<256, 1>(a, p, main, grid, s);
    } else {
        if (p.dp == 64) launch<64, 2>(a, p, main, grid, s);
        if (p.dp == 128) launch<128, 2>(a, p, main, grid, s);
    }
}

}  // namespace k
}  // namespace clove
