// kv8.h -- what the kernels over the 8-bit paged cache share: where a
// sequence's rows, context and tiles lie, and the e4m3 conversions.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "launch.hpp"

namespace clove {
namespace k {

constexpr int kKv8MinExp = -60, kKv8MaxExp = 119;
constexpr float kE4m3Max = 448.0f;

// Sequence b's context length inside its table's capacity.
__device__ __forceinline__ int kv8_context(const Kv8Args &a, int b) {
    return min(max(a.context_lens[b], 0), a.max_blocks * a.block_size);
}

// Sequence b's rows [*first, *first + *n), none where row_starts is not a
// range inside the rows.
__device__ __forceinline__ void kv8_rows(const Kv8Args &a, int b, int *first, int *n) {
    if (!a.row_starts) {
        *first = b;
        *n = 1;
        return;
    }
    const int s0 = a.row_starts[b], s1 = a.row_starts[b + 1];
    const bool ok = s0 >= 0 && s0 <= s1 && s1 <= a.rows;
    *first = ok ? s0 : 0;
    *n = ok ? s1 - s0 : 0;
}

// Reports contexts and row ranges that the two functions above clamped; one
// wave of a launch calls it.
__device__ __forceinline__ void kv8_check(const Kv8Args &a) {
    int bad = 0;
    for (int b = threadIdx.x & 63; b < a.num_seqs; b += 64) {
        if (a.context_lens[b] != kv8_context(a, b)) bad |= kErrPagedRange;
        if (a.row_starts) {
            const int s0 = a.row_starts[b], s1 = a.row_starts[b + 1];
            if (s0 < 0 || s0 > s1 || s1 > a.rows) bad |= kErrRowStarts;
        }
    }
    if (bad) atomicOr(a.err_flag, bad);
}

// How many of n ascending things come first for which f is true; the lanes of a
// wave look at 64 of them at a time (one round trip to memory for most batches,
// where a binary search takes one for each halving).
template <class F>
__device__ __forceinline__ int kv8_count(int n, F f) {
    const int lane = threadIdx.x & 63;
    int count = 0;
    for (int b = 0; b < n; b += 64) {
        const int hits = __popcll(__ballot(b + lane < n && f(b + lane)));
        count += hits;
        if (hits < 64) break;
    }
    return count;
}

// Work items of `per` units, `mul` units a row (`extra` more items than
// floor(units / per) at most).  Sequence b's items get the slots from
// floor(mul * row_starts[b] / per) + extra * b on: never more than the next
// sequence's first slot, so kv8_slots() slots serve any split of the rows
// without the host knowing it.  Returns the sequence that a slot (one for the
// wave) belongs to and the item's number within it.
__host__ __device__ __forceinline__ int64_t kv8_slots(const Kv8Args &a, int per, int mul,
                                                      int extra) {
    if (!a.row_starts) return (int64_t)a.num_seqs * ((mul + per - 1) / per);
    return (int64_t)a.rows * mul / per + (int64_t)extra * a.num_seqs;
}
__device__ __forceinline__ int kv8_slot(const Kv8Args &a, int slot, int per, int mul, int extra,
                                        int *item) {
    if (!a.row_starts) {
        const int each = (mul + per - 1) / per;
        *item = slot % each;
        return slot / each;
    }
    // the last b whose first slot is not behind this one
    const int lo = max(kv8_count(a.num_seqs, [&](int b) {
                           const int64_t s = min(max(a.row_starts[b], 0), a.rows);
                           return (int)(s * mul / per) + extra * b <= slot;
                       }) - 1, 0);
    const int64_t s = min(max(a.row_starts[lo], 0), a.rows);
    *item = slot - ((int)(s * mul / per) + extra * lo);
    return lo;
}

// The sequence that row r (one for the wave) belongs to, or -1.
__device__ __forceinline__ int kv8_seq_of_row(const Kv8Args &a, int r) {
    if (a.num_seqs == 0) return -1;
    if (!a.row_starts) return r;
    const int lo = max(kv8_count(a.num_seqs, [&](int b) { return a.row_starts[b] <= r; }) - 1, 0);
    int first, n;
    kv8_rows(a, lo, &first, &n);
    return r >= first && r < first + n ? lo : -1;
}

// Block j of sequence b, or -1 (reported) when its id lies outside the pool.
__device__ __forceinline__ int64_t kv8_block(const Kv8Args &a, int b, int j, bool report) {
    const int64_t id = a.block_tables[(size_t)b * a.max_blocks + j];
    if (id < 0 || id >= a.num_blocks) {
        if (report) atomicOr(a.err_flag, kErrPagedRange);
        return -1;
    }
    return id;
}

// Tile (plane, block, head): its number, and the offset of its first code.
__device__ __forceinline__ size_t kv8_tile(const Kv8Args &a, int plane, int64_t block, int h) {
    return ((size_t)plane * a.num_blocks + block) * a.num_heads + h;
}
__device__ __forceinline__ size_t kv8_tile_offset(const Kv8Args &a, size_t tile) {
    return tile * (size_t)(a.block_size * a.head_dim);
}

// 2^e for e in [-126, 127], and for an exponent as stored (what the append
// never writes is clamped).
__device__ __forceinline__ float kv8_pow2(int e) {
    return __uint_as_float((unsigned)(e + 127) << 23);
}
__device__ __forceinline__ float kv8_scale(int e) {
    return kv8_pow2(min(max(e, kKv8MinExp), kKv8MaxExp));
}

// The smallest e in [-60, 119] with amax <= 448 * 2^e; amax finite, >= 0.  448
// = 1.75 * 2^8, so the fraction bits decide between exponent - 8 and - 7.
__device__ __forceinline__ int kv8_exp_of(float amax) {
    const unsigned u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, kKv8MinExp), kKv8MaxExp);
}

__device__ __forceinline__ bool kv8_finite(float x) {
    return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}

// Four floats, already over their tile's scale, as four codes: nearest, ties
// to even; past +-448 (infinities, values over 448 * 2^119) saturates, NaN is 0.
__device__ __forceinline__ unsigned kv8_encode4(float a, float b, float c, float d) {
    auto in = [](float x) { return x != x ? 0.0f : fminf(fmaxf(x, -kE4m3Max), kE4m3Max); };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(in(a), in(b), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(in(c), in(d), w, true);
    return (unsigned)w;
}
__device__ __forceinline__ uint8_t kv8_encode(float x) {
    return (uint8_t)(kv8_encode4(x, 0.f, 0.f, 0.f) & 0xffu);
}
__device__ __forceinline__ float kv8_decode(uint8_t code) {
    return __builtin_amdgcn_cvt_f32_fp8((int)code, 0);
}

// ---- attention: how a call is cut into workgroups ---------------------------

// Query rows of one kv head are its sequence's (row, query head of the group)
// pairs, u = i * G + g; a tile is `tile` of them.
//
// All tiles' contexts are cut into steps of `step` tokens, numbered sequence by
// sequence, tile by tile, head by head, and each workgroup gets an equal run of
// them, whatever the lengths are: `share` steps, known on the device alone.  A
// tile that one workgroup holds whole is written by it; of a tile cut in pieces
// every workgroup stores its piece, and kv8_join puts them together: at most one
// that begins a tile, at the end of the run, and one that goes on with a tile, at
// its front.  `extra` steps that hold no tokens stand before each tile's own, for the
// time that a tile takes to begin and end.
struct Kv8Split {
    int kind;          // one of the KV8_ kernels
    int dp;            // head_dim the kernel is laid out for
    int tile;
    int step;
    int extra;
    int hw;            // heads that a workgroup takes together
    int grid;          // workgroups that share the steps, at most kKv8MaxGrid
    bool join;         // whether a tile may be cut
    int stored;        // rows of a piece
    int sums;          // tokens to a stored sum of weights, 0: none stored
    int groups;        // such sums a row
    int range;         // none stored: tokens whose scores are computed again at a time
    bool late;         // the blocks' weights come behind the join, which then leaves
                       // every row's maximum and sum
    // in the workspace, in floats
    size_t o_at, ml_at;      // piece 2w (+ 1: begins a tile) of workgroup w: of hw
                             // heads `stored` sums over V [D], and (maximum, sum) pairs
    size_t start_at;         // share, then [slot, head / hw] the tile's first step with tokens
    size_t declined_at;      // KV8_TILE: whether a workgroup leaves its run to the bf16 form
    size_t row_ml_at;        // (maximum, 1 / sum) of every row and query head
    size_t sums_at;          // [row, query head][groups] (sum, maximum) pairs
    size_t floats;
};
enum { KV8_ANY = 0, KV8_STREAM = 1, KV8_TILE = 2 };
constexpr int kKv8MaxGrid = 1024;
// Heads that a workgroup of the stream kernel takes together, where there are
// whole groups of them.
constexpr int kv8_stream_heads(int dp, int tile) { return dp * tile <= 128 * 16 ? 4 : 2; }

// The rows of a tile and the tokens they see.
struct Kv8Tile {
    int first, n, ctx;   // the sequence's rows and context
    int r0, rows;        // the tile's first (row, head) pair and how many it has
    int low, high;       // tokens its first row sees, and its last
};
// The slot of sequence b's first item.
__device__ __forceinline__ int kv8_first_slot(const Kv8Args &a, int b, int per, int mul,
                                              int extra) {
    if (!a.row_starts) return b * ((mul + per - 1) / per);
    const int64_t s = min(max(a.row_starts[b], 0), a.rows);
    return (int)(s * mul / per) + extra * b;
}
// Tile `item` of sequence b; false where there is none.
__device__ __forceinline__ bool kv8_tile_of(const Kv8Args &c, int G, int b, int item, int tile,
                                            Kv8Tile *t) {
    kv8_rows(c, b, &t->first, &t->n);
    t->ctx = kv8_context(c, b);
    const int R = t->n * G;
    t->r0 = item * tile;
    if (item < 0 || t->r0 >= R) return false;
    t->rows = min(tile, R - t->r0);
    t->low = t->ctx - t->n + t->r0 / G + 1;
    t->high = t->ctx - t->n + (t->r0 + t->rows - 1) / G + 1;
    return true;
}

// Steps of a tile whose last row sees `high` tokens.
__device__ __forceinline__ int kv8_steps(int high, int step) { return (max(high, 0) + step - 1) / step; }

// Where a workgroup's run of steps begins.
struct Kv8Place {
    int b, item, h, step;
    int share, total;
};

// All 256 threads: the steps before each sequence are summed up (in one order
// everywhere), and step `share * w` is looked up in them.
__device__ __forceinline__ Kv8Place kv8_find_place(const Kv8Args &c, int G, int H, int tile, int step,
                                                    int extra, int grid, int w, int *s_wave,
                                                    Kv8Place *s_place) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // a thread takes whole sequences, or (where there are few) part of one's tiles
    const int per = (c.num_seqs + 255) / 256, share_b = max(256 / max(c.num_seqs, 1), 1);
    const int b0 = tid / share_b * per, b1 = min(b0 + per, c.num_seqs), sub = tid % share_b;
    // f(item, steps) for the thread's tiles of sequence b
    auto tiles = [&](int b, auto f) {
        int first, n;
        kv8_rows(c, b, &first, &n);
        const int ctx = kv8_context(c, b), items = (n * G + tile - 1) / tile;
        const int each = (items + share_b - 1) / share_b;
        for (int item = sub * each; item < min((sub + 1) * each, items); ++item)
        {
            const int n_steps = kv8_steps(ctx - n + (min((item + 1) * tile, n * G) - 1) / G + 1, step);
            f(item, n_steps ? (n_steps + extra) * H : 0);
        }
    };
    int mine = 0;
    for (int b = b0; b < b1; ++b) tiles(b, [&](int, int n) { mine += n; });
    int inc = mine;
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(inc, o, 64);
        if (lane >= o) inc += up;
    }
    if (lane == 63) s_wave[wave] = inc;
    if (tid == 0) s_place->b = -1;
    __syncthreads();
    const int total = s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
    int at = inc - mine;
    for (int i = 0; i < wave; ++i) at += s_wave[i];
    const int share = max((total + grid - 1) / grid, 1);
    const int want = share * w;  // (the host keeps all steps below 2^30, and the grid)
    if (want >= at && want < at + mine) {
        for (int b = b0; b < b1; ++b)
            tiles(b, [&](int item, int n) {
                if (want >= at && want < at + n) {
                    s_place->b = b;
                    s_place->item = item;
                    s_place->h = (want - at) / (n / H);
                    s_place->step = (want - at) % (n / H);
                }
                at += n;
            });
    }
    __syncthreads();
    Kv8Place p = *s_place;
    p.share = share;
    p.total = total;
    return p;
}

// Moves `at` on to the next tile with steps; false behind the last.
__device__ __forceinline__ bool kv8_next_tile(const Kv8Args &c, int G, int H, int tile, Kv8Place *at,
                                              Kv8Tile *T) {
    if (at->h >= H) {
        at->h = 0;
        ++at->item;
    }
    while (at->b >= 0 && at->b < c.num_seqs) {
        if (!kv8_tile_of(c, G, at->b, at->item, tile, T)) {
            ++at->b;
            at->item = 0;
        } else if (T->high <= 0) {
            ++at->item;
        } else {
            return true;
        }
    }
    return false;
}

// A maximum and a sum of tokens that a row saw nothing of.  (Scores that are NaN
// leave a sum that is.)
__device__ __forceinline__ bool kv8_empty(float2 ml) { return ml.x == -INFINITY && ml.y == 0.0f; }

// Workgroups behind the others, of 256 threads, a wave a row: zeros for the rows
// of no sequence and those without a token to see.
inline unsigned kv8_zero_grid(const Kv8Args &c) { return (c.rows + 3) / 4; }
__device__ __forceinline__ void kv8_zero_rows(const Kv8Attention &a, int block) {
    const Kv8Args &c = a.c;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = block * 4 + wave;
    if (block == 0 && wave == 0) kv8_check(c);
    if (r >= c.rows) return;
    const int b = kv8_seq_of_row(c, r);
    int see = 0;
    if (b >= 0) {
        int first, n;
        kv8_rows(c, b, &first, &n);
        see = kv8_context(c, b) - n + (r - first) + 1;
    }
    if (see > 0) return;
    const int X = a.q_heads * c.head_dim;
    for (int d = lane; d < X; d += 64) a.out[(size_t)r * X + d] = 0.0f;
}

constexpr float kKv8Slack = 8.0f;  // a maximum moves when a score exceeds it by this (base 2)
constexpr float kLog2e = 1.44269504088896341f;

// Two e4m3 codes, times a power of two, as two bf16: exact.
template <bool HIGH>
__device__ __forceinline__ unsigned kv8_widen(unsigned codes, float scale) {
    return __builtin_bit_cast(unsigned,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
}

// Workgroups of the stream kernel that a CU holds.
int kv8_stream_residents();
void kv8_stream(const Kv8Attention &a, const Kv8Split &p, hipStream_t s);
void kv8_tiles(const Kv8Attention &a, const Kv8Split &p, hipStream_t s);
// The weights of the blocks, p.late: from sums that kv8_tiles stored, or the scores
// computed again.
constexpr int kKv8WeightPart = 512;
// Bytes of sums, however wide the tables are: where a sum for every 16 or 4 tokens of
// the tables and every row and head would take more, decode steps go in several turns,
// and others have the scores computed again, a range of the tables' blocks at a time.
constexpr int64_t kKv8MaxSums = 1ll << 30;
void kv8_late_weights(const Kv8Attention &a, const Kv8Split &p, hipStream_t s);

}  // namespace k
}  // namespace clove
