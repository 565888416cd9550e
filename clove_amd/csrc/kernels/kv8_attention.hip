// kv8_attention.hip -- attention over the 8-bit paged cache: per row i of a
// sequence (position p) and query head h, with kv head g = h / (Hq / H),
//   s_t = scale * q . K_t,  out = sum_t softmax_t(s) V_t,  t = 0 .. p.
// Here: the kernels for shapes that the matrix cores' do not take, the joins of
// contexts cut over workgroups, the blocks' weights, and the choice between them.
// Weights are 2^(s log2 e - m) with m the row's maximum or less than it by the
// slack; sums over parts with maxima m_i join as 2^(m_i - m) times each.
#include <algorithm>

#include "kv8.h"
#include "wave.h"

namespace clove {
namespace k {

namespace {

__device__ __forceinline__ float fast_exp(float x) {
    return __builtin_amdgcn_exp2f(x * 1.44269504088896341f);
}

// Any head_dim, block size and alignment: one wave for each (row, query head),
// 64 tokens a step, a lane a token for the scores and a lane up to four dims
// for the sum over V.  ml (or null) receives the row's maximum and sum.  Bound by
// its byte loads: 2.6 ms for 32 sequences of 511 to 4095 tokens, 32 heads of 128,
// which the stream kernel takes 99 us for.
__global__ void __launch_bounds__(64) kv8_attention_any_kernel(Kv8Attention a, float2 *ml) {
    const Kv8Args &c = a.c;
    const int lane = threadIdx.x, r = blockIdx.x, hq = blockIdx.y;
    const int D = c.head_dim, bs = c.block_size, h = hq / (a.q_heads / c.num_heads);
    __shared__ float sq[kKv8MaxHeadDim], sp[64], sv[64];
    __shared__ size_t srow[64];
    if (r == 0 && hq == 0) kv8_check(c);
    const int b = kv8_seq_of_row(c, r);
    int visible = 0;
    if (b >= 0) {
        int first, n;
        kv8_rows(c, b, &first, &n);
        visible = kv8_context(c, b) - n + (r - first) + 1;
    }
    const size_t qo = ((size_t)r * a.q_heads + hq) * D;
    for (int d = lane; d < D; d += 64) sq[d] = a.q[qo + d];
    float m = -INFINITY, l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int t0 = 0; t0 < visible; t0 += 64) {
        __syncthreads();
        const int t = t0 + lane;
        float s = -INFINITY;
        int64_t id = -1;
        if (t < visible) id = kv8_block(c, b, t / bs, h == 0);
        if (id >= 0) {
            const size_t kt = kv8_tile(c, 0, id, h), vt = kv8_tile(c, 1, id, h);
            const uint8_t *kr = c.codes + kv8_tile_offset(c, kt) + (size_t)(t % bs) * D;
            float dot = 0.0f;
            for (int d = 0; d < D; ++d) dot = fmaf(sq[d], kv8_decode(kr[d]), dot);
            s = dot * kv8_scale(c.exps[kt]) * a.scale;
            srow[lane] = kv8_tile_offset(c, vt) + (size_t)(t % bs) * D;
            sv[lane] = kv8_scale(c.exps[vt]);
        }
        const float m_new = fmaxf(m, wave_max(s));
        const float mz = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = fast_exp(m - mz);
        const float p = id >= 0 ? fast_exp(s - mz) : 0.0f;
        l = l * alpha + wave_sum(p);
        m = m_new;
        sp[lane] = p;
        const uint64_t live = __ballot(id >= 0);
        __syncthreads();
        for (int i = 0; i < 4; ++i) o[i] *= alpha;
        for (int u = 0; u < 64; ++u) {
            if (!((live >> u) & 1)) continue;
            const float w = sp[u] * sv[u];
            for (int i = 0; i < 4; ++i) {
                const int d = lane + 64 * i;
                if (d < D) o[i] = fmaf(w, kv8_decode(c.codes[srow[u] + d]), o[i]);
            }
        }
    }
    // NaN scores stay NaN
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < D) a.out[qo + lane + 64 * i] = o[i] * inv;
    if (ml && lane == 0) ml[(size_t)r * a.q_heads + hq] = make_float2(m, inv);
}

// The weight of each block, the scores computed again: one workgroup for
// each (sequence, block), its sums in a fixed order.
__global__ void __launch_bounds__(256) kv8_weights_any_kernel(Kv8Attention a, const float2 *ml) {
    const Kv8Args &c = a.c;
    const int j = blockIdx.x, b = blockIdx.y;
    const int D = c.head_dim, bs = c.block_size, G = a.q_heads / c.num_heads;
    __shared__ float part[256];
    const size_t at = (size_t)b * c.max_blocks + j;
    const int ctx = kv8_context(c, b);
    const int tokens = min(bs, ctx - j * bs);
    float sum = 0.0f;
    int64_t id = -1;
    if (tokens > 0) id = kv8_block(c, b, j, false);
    if (id >= 0) {
        int first, n;
        kv8_rows(c, b, &first, &n);
        for (int64_t u = threadIdx.x; u < (int64_t)n * a.q_heads * tokens; u += 256) {
            const int tok = (int)(u % tokens);
            const int hq = (int)(u / tokens % a.q_heads), i = (int)(u / tokens / a.q_heads);
            if (j * bs + tok > ctx - n + i) continue;
            const size_t rh = (size_t)(first + i) * a.q_heads + hq;
            const size_t kt = kv8_tile(c, 0, id, hq / G);
            const uint8_t *kr = c.codes + kv8_tile_offset(c, kt) + (size_t)tok * D;
            float dot = 0.0f;
            for (int d = 0; d < D; ++d) dot = fmaf(a.q[rh * D + d], kv8_decode(kr[d]), dot);
            const float s = dot * kv8_scale(c.exps[kt]) * a.scale;
            sum += fast_exp(s - ml[rh].x) * ml[rh].y;
        }
    }
    part[threadIdx.x] = sum;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if (threadIdx.x < o) part[threadIdx.x] += part[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) a.w_out[at] = a.w_in[at] + part[0];
}

// The pieces of a tile and the first workgroup that has one.  Where row_starts
// decrease, tiles may share a slot and its start: the pieces stay those there are.
__device__ __forceinline__ int kv8_pieces(const Kv8Split &p, int share, int start, int steps,
                                          int *w0) {
    *w0 = min(max(start / share, 0), p.grid - 1);
    return min((int)(((unsigned)start + steps - 1) / (unsigned)share), p.grid - 1) - *w0 + 1;
}

// Blocks behind a join's others: the weights of 64 blocks of a sequence from the
// sums that the stream kernel stored.  Lanes take blocks, the waves the sequence's
// rows and heads in turn, 64 of them at a time, whose maxima and sums are put
// together here once more, so that no launch has to wait for the join.
__device__ void kv8_block_weights(const Kv8Attention &a, const Kv8Split &p, int block) {
    const Kv8Args &c = a.c;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int across = (c.max_blocks + 63) / 64, b = block / across;
    const int j = block % across * 64 + lane;
    const int per = c.block_size / p.sums, G = a.q_heads / c.num_heads;
    __shared__ float part[16][64];
    __shared__ float2 s_ml[64];
    int first, n;
    kv8_rows(c, b, &first, &n);
    const int ctx = kv8_context(c, b);
    const int slot = kv8_first_slot(c, b, p.tile, G, 1);
    const int *starts = reinterpret_cast<const int *>(a.ws + p.start_at);
    const float2 *row_ml = reinterpret_cast<const float2 *>(a.ws + p.row_ml_at);
    const float2 *piece_ml = reinterpret_cast<const float2 *>(a.ws + p.ml_at);
    const float2 *sums = reinterpret_cast<const float2 *>(a.ws + p.sums_at);
    float w = 0.0f;
    if ((int64_t)(j - lane) * c.block_size >= ctx) n = 0;  // (none of the blocks holds a token)
    for (int x0 = 0; x0 < n * a.q_heads; x0 += 64) {
        const int xs = min(64, n * a.q_heads - x0);
        __syncthreads();  // the rows before are done with
        for (int x = 4 * wave + lane / 16; x < xs; x += 4 * waves) {  // 16 lanes to a row
            const int i = (x0 + x) / a.q_heads, hq = (x0 + x) % a.q_heads, h = hq / G;
            const int u = i * G + hq % G, item = u / p.tile;
            Kv8Tile T;
            int w0 = 0, np = 1;
            if (p.join && kv8_tile_of(c, G, b, item, p.tile, &T) && T.high > 0) {
                const int start = starts[1 + (size_t)(slot + item) * (c.num_heads / p.hw) + h / p.hw];
                np = kv8_pieces(p, starts[0], start, kv8_steps(T.high, p.step), &w0);
            }
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (np <= 1) {
                ml = row_ml[(size_t)first * a.q_heads + x0 + x];
            } else {
                const size_t row = (size_t)(h % p.hw) * p.stored + u - T.r0;
                const size_t per_piece = (size_t)p.hw * p.stored;
                for (int y0 = lane & 15; y0 < np; y0 += 64) {
                    float2 v[4];
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const int y = y0 + 16 * z;
                        v[z] = make_float2(-INFINITY, 0.0f);
                        if (y < np)
                            v[z] = piece_ml[(size_t)(2 * (w0 + y) + (y == 0 ? 1 : 0)) * per_piece +
                                            row];
                    }
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        if (kv8_empty(v[z])) continue;
                        const float t = fmaxf(ml.x, v[z].x);
                        ml.y = ml.y * __builtin_amdgcn_exp2f(ml.x - t) +
                               v[z].y * __builtin_amdgcn_exp2f(v[z].x - t);
                        ml.x = t;
                    }
                }
                float top = ml.x;
#pragma unroll
                for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
                float l = kv8_empty(ml) ? 0.0f : ml.y * __builtin_amdgcn_exp2f(ml.x - top);
#pragma unroll
                for (int o = 1; o < 16; o <<= 1) l += __shfl_xor(l, o, 64);
                ml = make_float2(top, l == 0.0f ? 0.0f : 1.0f / l);
            }
            if ((lane & 15) == 0) s_ml[x] = ml;
        }
        __syncthreads();
        if (j < c.max_blocks && (int64_t)j * c.block_size < ctx) {
#pragma unroll 4
            for (int x = wave; x < xs; x += waves) {
                const int see = ctx - n + (x0 + x) / a.q_heads + 1 - j * c.block_size;
                const float2 ml = s_ml[x];
                const float2 *from = sums + ((size_t)first * a.q_heads + x0 + x) * p.groups + (size_t)j * per;
                for (int i = 0; i < per && i * p.sums < see; ++i) {
                    const float2 v = from[i];
                    const float f = v.y == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(v.y - ml.x);
                    w += v.x * f * ml.y;
                }
            }
        }
    }
    part[wave][lane] = w;
    __syncthreads();
    if (wave == 0 && j < c.max_blocks) {
        const size_t at = (size_t)b * c.max_blocks + j;
        for (int x = 1; x < waves; ++x) w += part[x][lane];
        a.w_out[at] = a.w_in[at] + w;
    }
}
__global__ void __launch_bounds__(256) kv8_weights_kernel(Kv8Attention a, Kv8Split p) {
    kv8_block_weights(a, p, blockIdx.x);
}

// Joins the pieces of the tiles that were cut: `per` waves take the pieces of a
// row in turn, eight on their way at a time, and a lane holds up to four dims.
// Bound by latency: 8 us for 32 rows of 129 pieces each.
__global__ void __launch_bounds__(1024) kv8_join_kernel(Kv8Attention a, Kv8Split p, int per,
                                                        int grid) {
    if ((int)blockIdx.x >= grid) {
        kv8_block_weights(a, p, blockIdx.x - grid);
        return;
    }
    const Kv8Args &c = a.c;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int D = c.head_dim, H = c.num_heads, G = a.q_heads / H;
    const int h = blockIdx.x % H, slot = blockIdx.x / H / p.stored;
    const int u = blockIdx.x / H % p.stored;
    __shared__ float s_o[16][kKv8MaxHeadDim], s_l[16], s_top[16];
    const int *starts = reinterpret_cast<const int *>(a.ws + p.start_at);
    const int share = starts[0], start = starts[1 + (size_t)slot * (H / p.hw) + h / p.hw];
    int item;
    const int b = kv8_slot(c, slot, p.tile, G, 1, &item);
    Kv8Tile T;
    if (!kv8_tile_of(c, G, b, item, p.tile, &T) || T.high <= 0) return;
    int w0;
    const int np = kv8_pieces(p, share, start, kv8_steps(T.high, p.step), &w0);
    if (np <= 1) return;  // written whole
    if (u >= T.rows) return;
    float top = -INFINITY, l = 0.0f, x[4] = {0.f, 0.f, 0.f, 0.f};
    const size_t row = (size_t)(h % p.hw) * p.stored + u, per_piece = (size_t)p.hw * p.stored;
    const size_t first = (2 * w0 + 1) * per_piece + row;
    const float2 *ml = reinterpret_cast<const float2 *>(a.ws + p.ml_at);
    const float *o = a.ws + p.o_at;
    for (int i0 = wave; i0 < np; i0 += 8 * per) {
        float2 v[8];
        float y[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = i0 + j * per;
            v[j] = make_float2(-INFINITY, 0.0f);
            if (i < np) {
                const size_t at = i == 0 ? first : 2 * (w0 + i) * per_piece + row;
                v[j] = ml[at];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    y[j][e] = lane + 64 * e < D ? o[at * D + lane + 64 * e] : 0.0f;
            }
        }
        float t = top;
#pragma unroll
        for (int j = 0; j < 8; ++j) t = fmaxf(t, v[j].x);
        const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - t);
        l *= f;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= f;
        top = t;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (!kv8_empty(v[j])) {
                const float fj = __builtin_amdgcn_exp2f(v[j].x - t);
                l = fmaf(v[j].y, fj, l);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = fmaf(y[j][e], fj, x[e]);
            }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < D) s_o[wave][lane + 64 * e] = x[e];
    if (lane == 0) {
        s_l[wave] = l;
        s_top[wave] = top;
    }
    __syncthreads();
    if (wave) return;
    const float mine = lane < per ? s_top[lane] : -INFINITY;
    top = wave_max(mine);
    const float f = mine == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mine - top);
    l = wave_sum(lane < per ? s_l[lane] * f : 0.0f);
    x[0] = x[1] = x[2] = x[3] = 0.0f;
#pragma unroll 4
    for (int w = 0; w < per; ++w) {
        const float fw = __shfl(f, w, 64);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (lane + 64 * e < D) x[e] = fmaf(s_o[w][lane + 64 * e], fw, x[e]);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const size_t rh = (size_t)(T.first + (T.r0 + u) / G) * a.q_heads + h * G + (T.r0 + u) % G;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < D) a.out[rh * D + lane + 64 * e] = x[e] * inv;
    if (lane == 0 && p.late)
        reinterpret_cast<float2 *>(a.ws + p.row_ml_at)[rh] = make_float2(top, inv);
}

// The same for tiles of many rows with few pieces: a thread joins four dims of a
// row, all the loads of a workgroup run along the rows.  5 us where 1024 rows of
// 128 are cut in two; 16 us for the 2000 rows and 24 heads of ragged chunks.
__global__ void __launch_bounds__(256) kv8_join_rows_kernel(Kv8Attention a, Kv8Split p, int grid) {
    if ((int)blockIdx.x >= grid) {
        kv8_block_weights(a, p, blockIdx.x - grid);
        return;
    }
    const Kv8Args &c = a.c;
    const int D = c.head_dim, H = c.num_heads, G = a.q_heads / H, D4 = D / 4;
    const int groups = (p.stored * D4 + blockDim.x - 1) / blockDim.x;
    const int h = blockIdx.x % H, slot = blockIdx.x / H / groups;
    const int x = (int)(blockIdx.x / H % groups) * blockDim.x + threadIdx.x;
    const int *starts = reinterpret_cast<const int *>(a.ws + p.start_at);
    const int share = starts[0], start = starts[1 + (size_t)slot * (H / p.hw) + h / p.hw];
    int item;
    const int b = kv8_slot(c, slot, p.tile, G, 1, &item);
    Kv8Tile T;
    if (!kv8_tile_of(c, G, b, item, p.tile, &T) || T.high <= 0) return;
    int w0;
    const int np = kv8_pieces(p, share, start, kv8_steps(T.high, p.step), &w0);
    const int u = x / D4, d4 = x - u * D4;
    if (np <= 1 || u >= T.rows) return;  // written whole, or no row
    const size_t row = (size_t)(h % p.hw) * p.stored + u, per_piece = (size_t)p.hw * p.stored;
    const size_t first = (2 * w0 + 1) * per_piece + row;
    const float2 *ml = reinterpret_cast<const float2 *>(a.ws + p.ml_at);
    const cl_f4 *o = reinterpret_cast<const cl_f4 *>(a.ws + p.o_at);
    float top = -INFINITY, l = 0.0f;
    cl_f4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < np; i0 += 2) {
        float2 v[2];
        cl_f4 y[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = min(i0 + j, np - 1);
            const size_t at = i == 0 ? first : 2 * (w0 + i) * per_piece + row;
            v[j] = ml[at];
            y[j] = o[at * D4 + d4];
        }
        if (i0 + 1 >= np) v[1] = make_float2(-INFINITY, 0.0f);
        const float t = fmaxf(top, fmaxf(v[0].x, v[1].x));
        const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - t);
        l *= f;
        sum *= f;
        top = t;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (!kv8_empty(v[j])) {
                const float fj = __builtin_amdgcn_exp2f(v[j].x - t);
                l = fmaf(v[j].y, fj, l);
                sum += y[j] * fj;
            }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const size_t rh = (size_t)(T.first + (T.r0 + u) / G) * a.q_heads + h * G + (T.r0 + u) % G;
    reinterpret_cast<cl_f4 *>(a.out)[rh * D4 + d4] = sum * inv;
    if (d4 == 0 && p.late)
        reinterpret_cast<float2 *>(a.ws + p.row_ml_at)[rh] = make_float2(top, inv);
}

// Tokens to a stored sum of weights: of one block.
int kv8_sum_tokens(int block_size) { return block_size % 16 == 0 ? 16 : 4; }

Kv8Split kv8_split(const Kv8Attention &a, int cus) {
    const Kv8Args &c = a.c;
    Kv8Split p{};
    const int D = c.head_dim, bs = c.block_size, G = a.q_heads / c.num_heads;
    const int sums = kv8_sum_tokens(bs);
    const int64_t rh = (int64_t)c.rows * a.q_heads;
    auto take = [&](int64_t n) {  // n floats, 16-byte aligned
        const size_t at = p.floats;
        p.floats += (size_t)((n + 3) / 4 * 4);
        return at;
    };
    // 16-byte pieces of every row, four tokens to a block, rows of the pool
    // numbered in 32 bits, grids within theirs
    const bool fast = D % 16 == 0 && bs % 4 == 0 && c.num_seqs > 0 && c.rows > 0 &&
                      c.num_blocks > 0 && c.max_blocks > 0 && rh < (1 << 24) &&
                      c.num_blocks * c.num_heads * bs < (1ll << 32) &&
                      ((reinterpret_cast<uintptr_t>(c.codes) | reinterpret_cast<uintptr_t>(a.q)) & 15) == 0;
    auto plain = [&] {
        p = Kv8Split{};
        if (a.w_out) p.row_ml_at = take(2 * rh);
        return p;
    };
    if (!fast) return plain();
    p.dp = D <= 64 ? 64 : D <= 128 ? 128 : 256;
    // rows of one sequence and kv head, on the average
    const int64_t units = ((int64_t)c.rows * G + c.num_seqs - 1) / c.num_seqs;
    const int64_t cap = (int64_t)c.max_blocks * bs;
    int residents;
    // (16 speculating sequences of 22 rows and heads each: 54 us, as tiles 59)
    if (units <= (p.dp == 256 ? 16 : 32)) {
        p.kind = KV8_STREAM;
        p.tile = units <= 16 || p.dp == 256 ? 16 : 32;
        // Four heads of the same tokens side by side are 8 KB in a row to the memory
        // (32 x 4096 tokens, 32 heads of 128: 98 against 109 us; 24 x 600 to 3000
        // tokens, 16 heads of 96, 96 tiles of four heads: 49 against 51) but cut a
        // tile into four times the pieces, which costs more than it gives where the
        // tiles are few (one context of 131000 tokens, one tile: 57 against 47
        // us), and two heads gain less (speculated tokens, 104 tiles: 60
        // against 53).
        p.hw = kv8_stream_heads(p.dp, p.tile);
        if (c.num_heads % p.hw ||
            kv8_slots(c, p.tile, G, 1) * c.num_heads / p.hw < (p.hw == 4 ? cus / 4 : cus))
            p.hw = 1;
        p.step = 32 * 4 / p.hw;
        residents = kv8_stream_residents();
    } else {
        p.kind = KV8_TILE;
        p.tile = units <= 64 || p.dp == 256 ? 64 : 128;
        p.hw = 1;
        p.step = p.dp == 256 ? 32 : 64;
        // A tile's table, rows, first codes and stores take the time of some four
        // steps: 2048 rows of 32 heads of 80, 180 us when runs are equal in steps
        // alone, 120 / 114 / 120 with 2 / 4 / 7 more a tile; chunks 170, 154 / 155 / 162.
        p.extra = 4;
        residents = 2;
    }
    p.stored = !c.row_starts && G < p.tile ? G : p.tile;
    const int64_t tiles = kv8_slots(c, p.tile, G, 1) * c.num_heads / p.hw;
    if (tiles >= (1 << 20) || kv8_slots(c, kKv8WeightPart, G, 1) > 65535) return plain();
    const int64_t steps = (cap + p.step - 1) / p.step;
    const int64_t room = std::min(kKv8MaxGrid, cus * residents);
    if (tiles * (steps + p.extra) >= (1ll << 30)) return plain();
    // (the weights' workgroups stand behind the join's, 2^32 threads to a grid)
    if (a.w_out && (int64_t)((c.max_blocks + 63) / 64) * c.num_seqs >= (1 << 21)) return plain();
    p.join = steps > 1 && (p.kind == KV8_STREAM || tiles < 2 * room);
    p.grid = (int)(p.join || p.kind == KV8_STREAM ? std::min<int64_t>(room, tiles * steps) : tiles);
    if (p.join) {
        p.o_at = take((int64_t)2 * p.grid * p.hw * p.stored * D);
        p.ml_at = take((int64_t)2 * p.grid * p.hw * p.stored * 2);
        p.start_at = take(1 + tiles);
    }
    if (p.kind == KV8_TILE) p.declined_at = take(p.grid);
    if (a.w_out) {
        p.row_ml_at = take(2 * rh);
        // Eight bytes for 16 tokens of a row, written on the way and read once,
        // against all scores computed again: 2000 rows in chunks, 24 query
        // heads of 80, contexts to 3700, 155 against 217 us.  They are stored up to a
        // GiB; a long prompt's are not, nor those of very wide tables.
        const int64_t pairs = kv8_slots(c, kKv8WeightPart, G, 1) * c.num_heads;
        if ((p.kind == KV8_STREAM || sums == 16) && 8 * rh * (cap / sums) <= kKv8MaxSums) {
            p.sums = sums;
            p.groups = (int)(cap / sums);
            p.sums_at = take(2 * rh * p.groups);
        } else {
            // four bytes for four tokens of a part of a sequence's rows
            const int64_t blocks = std::min<int64_t>(kKv8MaxSums / (pairs * bs), c.max_blocks);
            if (blocks == 0) return plain();
            p.range = (int)(blocks * bs);
            p.groups = p.range / 4;
            p.sums_at = take(pairs * p.groups);
        }
        p.late = p.kind == KV8_TILE || !p.sums;
    }
    return p;
}

// Sequences [b0, b0 + n) of a call with one row for each.
Kv8Attention kv8_some(Kv8Attention a, int b0, int n) {
    const size_t X = (size_t)a.q_heads * a.c.head_dim, entries = (size_t)b0 * a.c.max_blocks;
    a.c.block_tables += entries;
    a.c.context_lens += b0;
    a.c.num_seqs = a.c.rows = n;
    a.q += b0 * X;
    a.out += b0 * X;
    a.w_in += entries;
    a.w_out += entries;
    return a;
}

// Sequences of one row each go in several turns where their sums of weights would
// take more than kKv8MaxSums: 256 sequences, 64 heads, 131072-token tables, contexts
// of 500 to 4000, 563 us in five turns against 2191 with the scores computed again.
int kv8_at_once(const Kv8Attention &a, int cus) {
    const Kv8Args &c = a.c;
    const Kv8Split p = kv8_split(a, cus);
    if (p.kind != KV8_STREAM || !p.late || c.row_starts) return c.num_seqs;
    const int64_t cap = (int64_t)c.max_blocks * c.block_size;
    const int64_t most = kKv8MaxSums / (8 * a.q_heads * (cap / kv8_sum_tokens(c.block_size)));
    if (most == 0) return c.num_seqs;
    const int turns = (int)((c.num_seqs + most - 1) / most);
    return (c.num_seqs + turns - 1) / turns;
}

void kv8_turn(const Kv8Attention &a, int cus, hipStream_t s) {
    const Kv8Split p = kv8_split(a, cus);
    const Kv8Args &c = a.c;
    const bool weights = a.w_out && c.num_seqs > 0 && c.max_blocks > 0;
    if (p.kind == KV8_ANY) {
        float2 *ml = a.w_out ? reinterpret_cast<float2 *>(a.ws + p.row_ml_at) : nullptr;
        if (c.rows > 0) kv8_attention_any_kernel<<<dim3(c.rows, a.q_heads), 64, 0, s>>>(a, ml);
        if (weights)
            kv8_weights_any_kernel<<<dim3(c.max_blocks, c.num_seqs), 256, 0, s>>>(a, ml);
        return;
    }
    if (p.kind == KV8_STREAM)
        kv8_stream(a, p, s);
    else
        kv8_tiles(a, p, s);
    // the blocks' weights: with the join, or behind it
    const unsigned blocks =
        weights && !p.late ? (unsigned)((c.max_blocks + 63) / 64) * c.num_seqs : 0;
    if (p.join) {
        const unsigned tiles = (unsigned)kv8_slots(c, p.tile, a.q_heads / c.num_heads, 1) * c.num_heads;
        // pieces to a tile: 2 on the average where there are as many tiles as runs
        const int pieces = p.grid * p.hw / (int)tiles + 1;
        if (pieces <= 8) {
            const int n = p.stored * c.head_dim / 4;
            const int threads = blocks ? 256 : std::min(256, (n + 63) / 64 * 64);
            const unsigned grid = tiles * ((n + threads - 1) / threads);
            kv8_join_rows_kernel<<<grid + blocks, threads, 0, s>>>(a, p, (int)grid);
        } else {
            const int per = pieces <= 32 ? 4 : 16;
            const unsigned grid = tiles * p.stored;
            kv8_join_kernel<<<grid + blocks, 64 * per, 0, s>>>(a, p, per, (int)grid);
        }
    } else if (blocks) {
        kv8_weights_kernel<<<blocks, 256, 0, s>>>(a, p);
    }
    if (weights && p.late) kv8_late_weights(a, p, s);
}

}  // namespace

size_t kv8_attention_workspace(const Kv8Attention &a, int cus) {
    const int n = kv8_at_once(a, cus);
    if (n == a.c.num_seqs) return kv8_split(a, cus).floats * sizeof(float);
    const int last = (a.c.num_seqs - 1) % n + 1;
    return std::max(kv8_split(kv8_some(a, 0, n), cus).floats,
                    kv8_split(kv8_some(a, 0, last), cus).floats) * sizeof(float);
}

void kv8_attention(const Kv8Attention &a, int cus, hipStream_t s) {
    const int n = kv8_at_once(a, cus);
    if (n == a.c.num_seqs) return kv8_turn(a, cus, s);
    for (int b0 = 0; b0 < a.c.num_seqs; b0 += n)
        kv8_turn(kv8_some(a, b0, std::min(n, a.c.num_seqs - b0)), cus, s);
}

}  // namespace k
}  // namespace clove
