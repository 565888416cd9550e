// kv8_stream.hip -- attention of a few query rows over the 8-bit paged cache:
// decode steps, grouped heads, a handful of speculated tokens.
//
// Tiles of up to 16 * NC query rows of HW neighbouring kv heads, their contexts in
// steps of 32 * 4 / HW tokens, and every workgroup an equal run of all steps
// (Kv8Split): ragged batches keep every CU busy to the end.  Of a step each of the
// four waves takes 32 tokens of a head and streams their codes from memory into the
// operands of v_mfma_f32_16x16x32_bf16:
//   S^T = K Q^T    A: lane (r, q) holds token r's dims 64s + 16q .. + 15 (one
//                  16-byte load, two MFMA steps; q is laid out alike),
//                  B: the 16 rows' q as three bf16 pieces, which hold all 24 bits;
//   O^T += V^T P^T A: lane (r, q) holds dims (DP/16) r .. of the eight tokens
//                  4q + i and 16 + 4q + i, paired up by byte permutes; these are
//                  the tokens of the lane's own S^T elements, so P^T needs no
//                  exchange between lanes; P in three bf16 pieces.
// A code times its tile's power of two is exact in bf16, so the conversion
// applies the scale, and products are those of 32-bit values with f32 sums.
//
// Bound by memory, two bytes a dim of a token, once the contexts are long: 32
// sequences of 511 to 4095 tokens, 32 heads of 128, 99 us with the join at 5.4
// TB/s; a form that only loads the codes runs 5% faster.  64 of 500 to 8191, 8 kv
// heads for 32: 103 us.  Few tiles are bound by latency besides: finding the
// place, the tables and the first codes, and the join are dependent trips to
// memory, some 15 of the 40 us of one context of 131000 tokens (3.3 TB/s).  The
// table of an item's tokens is therefore fetched while the one before runs, and the
// segment before goes out while the first codes are on their way.  Two workgroups
// to a CU: a third would take registers that spill.
#include "bf16x3.h"
#include "kv8.h"
#include "wave.h"

namespace clove {
namespace k {

namespace {

constexpr int kChunk = 2048;  // tokens whose rows a workgroup's table holds

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

// What a workgroup streams at a time: tokens [c0, c1) of a tile's segment, steps
// s0 .. s1 of it.
struct Item {
    Kv8Tile T;
    int b, h, c0, c1, t_end;
    int start;          // first token of the segment
    bool whole;         // the segment is the whole tile
    size_t piece;       // where it goes if not
};

template <int DP, int NC, int SUMS, int HW>
__global__ void __launch_bounds__(256, 2) stream_kernel(Kv8Attention a, Kv8Split p) {
    constexpr int KS = DP / 64;  // 16-byte loads of a token's key
    constexpr int JB = DP / 16;  // dims a lane holds of a token's value
    constexpr int TG = 4 / HW;   // waves that share a head
    constexpr int kStep = 32 * TG;
    constexpr int kPitch = DP + 4;
    constexpr int NE = kChunk / 4 / 256;              // table entries of a thread
    constexpr int NQ = (HW * NC * 2 * KS * 64 + 255) / 256;  // eights of a row's q of a thread
    const Kv8Args &c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, q = lane >> 4, hh = wave % HW;
    const int H = c.num_heads, G = a.q_heads / H, D = c.head_dim, bs = c.block_size;
    // four tokens: the row of the first in the first head's tile, ((block * H + h)
    // * bs + slot), and each head's scales of keys and values as bf16, 0 outside
    // the pool
    __shared__ unsigned s_row[kChunk / 4], s_scale[HW][kChunk / 4];
    __shared__ u4 s_q[HW * NC * 2 * KS * 3 * 64];
    __shared__ __attribute__((aligned(16))) float s_o[TG > 1 ? 2 : 1][TG > 1 ? 16 : 1][kPitch];
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ int s_wave[4];
    __shared__ Kv8Place s_place;

    if ((int)blockIdx.x >= p.grid) {
        kv8_zero_rows(a, blockIdx.x - p.grid);
        return;
    }
    const int w = (int)blockIdx.x;
    Kv8Place at = kv8_find_place(c, G, H / HW, p.tile, p.step, p.extra, p.grid, w, s_wave, &s_place);
    int *starts = reinterpret_cast<int *>(a.ws + p.start_at);
    if (p.join && w == 0 && tid == 0) starts[0] = at.share;
    const int run = min(at.share, at.total - at.share * w);
    int left = run;

    // The item behind `it` (the first one when it.b < 0); false at the end.
    auto next = [&](Item &it) {
        if (it.b >= 0) {
            if (it.c1 < it.t_end) {
                it.c0 = it.c1;
                it.c1 = min(it.c0 + kChunk, it.t_end);
                return true;
            }
            at.step = 0;
            ++at.h;
        }
        if (left <= 0 || !kv8_next_tile(c, G, H / HW, p.tile, &at, &it.T)) return false;
        const int all = kv8_steps(it.T.high, kStep), s1 = min(all, at.step + left);
        if (p.join && at.step == 0 && tid == 0)
            starts[1 + (size_t)(kv8_first_slot(c, at.b, p.tile, G, 1) + at.item) * (H / HW) + at.h] =
                at.share * w + (run - left);
        it.b = at.b;
        it.h = at.h * HW;
        it.start = it.c0 = at.step * kStep;
        it.t_end = min(s1 * kStep, it.T.high);
        it.c1 = min(it.c0 + kChunk, it.t_end);
        it.whole = at.step == 0 && s1 == all;
        it.piece = (size_t)(2 * w + (at.step == 0 ? 1 : 0)) * HW * p.stored;
        left -= s1 - at.step;
        return true;
    };

    // An item's table and q on their way: the block ids first, then what depends
    // on them, so that no step waits for either.
    int id[NE];
    unsigned kexp[NE][HW], vexp[NE][HW];
    cl_f4 qraw[NQ][2];
    constexpr bool kEarlyQ = HW * NC * DP <= 128;  // (where registers are left for it)
    const int shift = __builtin_ctz(bs);
    const bool pow2 = (bs & (bs - 1)) == 0;
    // tokens behind the end take the chunk's first place (and no part in what
    // follows), so that every load lies in the pool
    auto token = [&](const Item &it, int i) {
        const int t = it.c0 + 4 * i;
        return t < it.c1 ? t : it.c0;
    };
    auto fetch_ids = [&](const Item &it) {
#pragma unroll
        for (int y = 0; y < NE; ++y) {
            const int t = token(it, tid + 256 * y);
            const int j = pow2 ? t >> shift : t / bs;
            id[y] = -1;
            if (it.c0 + 4 * (tid + 256 * y) < it.c1 || y == 0)
                id[y] = c.block_tables[(size_t)it.b * c.max_blocks + j];
        }
    };
    auto fetch_q = [&](const Item &it) {
        if (it.c0 != it.start) return;
#pragma unroll
        for (int y = 0; y < NQ; ++y) {
            const int x = tid + 256 * y;
            const int lr = x & 15, lq = x >> 4 & 3, s = (x >> 6) % (2 * KS);
            const int cc = x / (128 * KS) % NC, head = x / (128 * KS * NC);
            const int u = 16 * cc + lr, d = 64 * (s / 2) + 16 * lq + 8 * (s & 1);
            qraw[y][0] = qraw[y][1] = (cl_f4){0.f, 0.f, 0.f, 0.f};
            if (head < HW && u < it.T.rows && d < D) {
                const int g = it.T.r0 + u;
                const cl_f4 *qr = reinterpret_cast<const cl_f4 *>(
                    a.q + ((size_t)(it.T.first + g / G) * a.q_heads + (it.h + head) * G + g % G) * D + d);
                qraw[y][0] = qr[0];
                qraw[y][1] = qr[1];
            }
        }
    };
    auto fetch_rest = [&](const Item &it) {
#pragma unroll
        for (int y = 0; y < NE; ++y) {
            if (id[y] >= 0 && id[y] < c.num_blocks)
#pragma unroll
                for (int i = 0; i < HW; ++i) {
                    kexp[y][i] = c.exps[kv8_tile(c, 0, id[y], it.h) + i];
                    vexp[y][i] = c.exps[kv8_tile(c, 1, id[y], it.h) + i];
                }
        }
        if (kEarlyQ) fetch_q(it);
    };
    // ... and into LDS; the entries outside the pool are reported.
    auto publish = [&](const Item &it) {
        int bad = 0;
#pragma unroll
        for (int y = 0; y < NE; ++y) {
            const int i = tid + 256 * y, t = token(it, i);
            if (i >= (it.c1 - it.c0 + kStep - 1) / kStep * (kStep / 4)) continue;
            unsigned row = 0;  // of the pool, where nothing is to be read
            const bool in = id[y] >= 0 && id[y] < c.num_blocks, behind = it.c0 + 4 * i >= it.c1;
            if (in && !behind)
                row = ((unsigned)id[y] * H + it.h) * bs + (pow2 ? t & (bs - 1) : t % bs);
            if (!in && !behind) {
                bad = 1;
                if (it.h == 0) atomicOr(c.err_flag, kErrPagedRange);
            }
            s_row[i] = row;
#pragma unroll
            for (int g = 0; g < HW; ++g)
                s_scale[g][i] = behind ? 0x00010001u
                                : in   ? __float_as_uint(kv8_scale(kexp[y][g])) |
                                           __float_as_uint(kv8_scale(vexp[y][g])) >> 16
                                       : 0;
        }
        if (it.c0 == it.start) {
            if (!kEarlyQ) fetch_q(it);
            // q times scale * log2(e) (weights are powers of two), in pieces
#pragma unroll
            for (int y = 0; y < NQ; ++y) {
                const int x = tid + 256 * y;
                if (x >= HW * NC * 2 * KS * 64) continue;
                const cl_f4 lo = qraw[y][0] * (a.scale * kLog2e), hi = qraw[y][1] * (a.scale * kLog2e);
                u4 v[3];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    unsigned w1, w2, w3;
                    split_pair<false>(e < 2 ? lo[2 * e] : hi[2 * e - 4],
                                      e < 2 ? lo[2 * e + 1] : hi[2 * e - 3], &w1, &w2, &w3);
                    v[0][e] = w1;
                    v[1][e] = w2;
                    v[2][e] = w3;
                }
#pragma unroll
                for (int i = 0; i < 3; ++i) s_q[((x >> 6) * 3 + i) * 64 + (x & 63)] = v[i];
            }
        }
        return bad;
    };

    float m[NC], l[NC];
    cl_f4 o[NC][JB];
    auto reset = [&] {
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) {
            m[cc] = -INFINITY;
            l[cc] = 0.0f;
#pragma unroll
            for (int jb = 0; jb < JB; ++jb) o[cc][jb] = (cl_f4){0.f, 0.f, 0.f, 0.f};
        }
    };
    // Row r of this wave's head, `f` times what the lanes hold.
    auto emit = [&](const Item &it, int cc, float f, float mm, float ll) {
        const int u = 16 * cc + r, g = it.T.r0 + u;
        if (u >= it.T.rows) return;
        const size_t rh = (size_t)(it.T.first + g / G) * a.q_heads + (it.h + hh) * G + g % G;
        const size_t piece = it.piece + (size_t)hh * p.stored + u;
        const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
        float *to = it.whole ? a.out + rh * D : a.ws + p.o_at + piece * D;
        if (it.whole) f *= inv;
        // element i of block jb is dim JB * (4q + i) + jb
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int jb = 0; jb < JB; jb += 4)
                if (JB * (4 * q + i) < D)
                    *reinterpret_cast<cl_f4 *>(to + JB * (4 * q + i) + jb) =
                        (cl_f4){o[cc][jb][i] * f, o[cc][jb + 1][i] * f, o[cc][jb + 2][i] * f,
                                o[cc][jb + 3][i] * f};
        if (q == 0) {
            if (!it.whole)
                reinterpret_cast<float2 *>(a.ws + p.ml_at)[piece] = make_float2(mm, ll);
            else if (a.w_out)
                reinterpret_cast<float2 *>(a.ws + p.row_ml_at)[rh] = make_float2(mm, inv);
        }
    };
    // The sums of a segment: the waves of a head together, and out.
    auto finish = [&](const Item &it) {
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) {
            float ls = l[cc];
            ls += __shfl_xor(ls, 16, 64);
            ls += __shfl_xor(ls, 32, 64);
            if constexpr (TG == 1) {
                emit(it, cc, 1.0f, m[cc], ls);
                continue;
            }
            lds_barrier();  // the rows before are done with
            if (q == 0) {
                s_m[wave][r] = m[cc];
                s_l[wave][r] = ls;
            }
            lds_barrier();
            float top = -INFINITY, all = 0.0f;
#pragma unroll
            for (int v = hh; v < 4; v += HW) top = fmaxf(top, s_m[v][r]);
#pragma unroll
            for (int v = hh; v < 4; v += HW)
                all += s_l[v][r] *
                       (s_m[v][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[v][r] - top));
            const float f0 = m[cc] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[cc] - top);
            // wave by wave (two at a time) into LDS; the last ones have the sum
            // (for one head: waves 0 and 1, 2 onto 0 and 3 onto 1, then 3 takes 2's)
            cl_f4 *buf = reinterpret_cast<cl_f4 *>(&s_o[wave & 1][r][0]);
            auto each = [&](auto f) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int jb = 0; jb < JB; jb += 4) f(i, jb, (JB * (4 * q + i) + jb) / 4);
            };
            auto put = [&](cl_f4 *to) {
                each([&](int i, int jb, int at) {
                    to[at] = (cl_f4){o[cc][jb][i], o[cc][jb + 1][i], o[cc][jb + 2][i], o[cc][jb + 3][i]};
                });
            };
            auto add = [&](const cl_f4 *from) {
                each([&](int i, int jb, int at) {
                    const cl_f4 x = from[at];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[cc][jb + e][i] += x[e];
                });
            };
#pragma unroll
            for (int jb = 0; jb < JB; ++jb) o[cc][jb] *= f0;
            if (wave < 2) put(buf);
            lds_barrier();
            if (wave >= 2) add(buf);
            if constexpr (TG == 4) {
                lds_barrier();
                if (wave == 2) put(buf);
                lds_barrier();
                if (wave == 3) {
                    add(reinterpret_cast<const cl_f4 *>(&s_o[0][r][0]));
                    emit(it, cc, 1.0f, top, all);
                }
            } else if (wave >= 2) {
                emit(it, cc, 1.0f, top, all);
            }
        }
    };

    float2 *sums = reinterpret_cast<float2 *>(a.ws + p.sums_at);
    const uint8_t *kbase = c.codes;
    int koff[KS];  // (q is 0 past D, where the row's first dims stand in)
#pragma unroll
    for (int i = 0; i < KS; ++i) koff[i] = 64 * i + 16 * q < D ? 64 * i + 16 * q : 0;
    const uint8_t *vbase =
        c.codes + (size_t)c.num_blocks * H * bs * D + (JB * r < D ? JB * r : 0);

    Item cur, done;
    cur.b = -1;
    if (!next(cur)) return;
    fetch_ids(cur);
    fetch_rest(cur);
    reset();
    bool pending = false, more_items = true;
    while (more_items) {
        lds_barrier();  // the item before is done with
        const int bad = __syncthreads_or(publish(cur));
        const int c0 = cur.c0, c1 = cur.c1;
        u4 kk[2][KS];
        Row<JB> vv[8];
        auto load_k = [&](int kb) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const unsigned e = s_row[(kb - c0 + 16 * u + r) >> 2] + hh * bs;
                const uint8_t *row = kbase + (size_t)(e + (r & 3)) * D;
#pragma unroll
                for (int i = 0; i < KS; ++i) kk[u][i] = load16(row + koff[i]);
            }
        };
        auto load_v = [&](int kb) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const unsigned e = s_row[((kb - c0) >> 2) + 4 * u + q] + hh * bs;
                const uint8_t *row = vbase + (size_t)e * D;
#pragma unroll
                for (int i = 0; i < 4; ++i) vv[4 * u + i] = load_row<JB>(row + i * D);
            }
        };
        int kb = c0 + 32 * (wave / HW);
        if (kb < c1) {
            load_k(kb);
            load_v(kb);
        }
        // the segment before goes out while the first codes are on their way
        if (pending) {
            finish(done);
            reset();
        }
        const Kv8Tile T = cur.T;
        const int h = cur.h + hh, low = T.low;
        int lim[NC];  // tokens each row sees
        unsigned rowhead[NC];
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) {
            const int u = 16 * cc + r;
            const bool ok = u < T.rows;
            const int g = T.r0 + (ok ? u : 0);
            lim[cc] = ok ? min(cur.t_end, T.ctx - T.n + g / G + 1) : 0;
            rowhead[cc] = (T.first + g / G) * a.q_heads + h * G + g % G;
        }
        done = cur;
        more_items = next(cur);
        if (more_items) fetch_ids(cur);
        const int kb0 = kb;
        for (; kb < c1; kb += kStep) {
            const bool more = kb + kStep < c1;
            float ks[2], vs[2];
            bool in[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                ks[u] = __uint_as_float(s_scale[hh][(kb - c0 + 16 * u + r) >> 2] & 0xffff0000u);
                const unsigned e = s_scale[hh][((kb - c0) >> 2) + 4 * u + q];
                vs[u] = __uint_as_float(e << 16);
                in[u] = e != 0;
            }
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
                        const u4 qf = s_q[(((hh * NC + cc) * 2 * KS + i) * 3 + x) * 64 + lane];
#pragma unroll
                        for (int u = 0; u < 2; ++u) s[cc][u] = mfma(kf[u], qf, s[cc][u]);
                    }
            }
            if (more) load_k(kb + kStep);
            if (bad || kb + 32 > min(low, c1)) {
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
            if (kb == kb0 && more_items) fetch_rest(cur);
        }
        if (kb0 >= c1 && more_items) fetch_rest(cur);
        pending = done.c1 == done.t_end;
    }
    finish(done);
}

template <int DP, int NC, int HW>
void launch(const Kv8Attention &a, const Kv8Split &p, unsigned grid, hipStream_t s) {
    switch (p.sums) {
    case 0: stream_kernel<DP, NC, 0, HW><<<grid, 256, 0, s>>>(a, p); break;
    case 4: stream_kernel<DP, NC, 4, HW><<<grid, 256, 0, s>>>(a, p); break;
    default: stream_kernel<DP, NC, 16, HW><<<grid, 256, 0, s>>>(a, p);
    }
}
template <int DP, int NC>
void launch(const Kv8Attention &a, const Kv8Split &p, unsigned grid, hipStream_t s) {
    if (p.hw == 1)
        launch<DP, NC, 1>(a, p, grid, s);
    else
        launch<DP, NC, kv8_stream_heads(DP, 16 * NC)>(a, p, grid, s);
}

}  // namespace

int kv8_stream_residents() { return 2; }

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
