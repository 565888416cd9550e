// kv8_evict.hip -- eviction of the lightest blocks of long sequences.
//
// One workgroup a sequence.  Of its n = ceil(ctx / block_size) blocks the first
// and last ones stay; of those between them the (budget - first - last) heaviest
// do.  Weights are read once, as unsigned keys of the same order, into registers
// (K a thread).  The least key that stays is found bit by bit from the top: the
// largest x with at least `left` keys >= x, counted by ballots, which ends early
// once exactly `left` are.  One scan then gives every block its place: among equal
// weights the earlier blocks stay.  Only integers are counted, so results do not
// depend on timing.
//
// Bound by latency, a round over the workgroup for each of the keys' bits: 256
// sequences of 1250 to 4096 blocks down to 1024, 12.6 us (the weights and tables
// are 4 us of memory traffic; keys read again from memory for every bit, one thread a
// place: 44), 8 of 63 to 128 blocks 6 us.  The calls follow each other every 12.1 and
// 6.7 us: four allocations and the submission are 6.6 us of the host's time.
#include "kv8.h"

namespace clove {
namespace k {

namespace {

// Unsigned keys in the order of the weights; NaN lowest, -0 as 0.
__device__ __forceinline__ unsigned order_key(float w) {
    if (w != w) return 0;
    const unsigned u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Block tid + THREADS * i is thread tid's i-th.  K = 0: more blocks than registers
// hold; they are read again for every bit.
template <int THREADS, int K>
__global__ void __launch_bounds__(THREADS) evict_kernel(EvictArgs a) {
    constexpr int kWaves = THREADS / 64;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t at = (size_t)b * a.max_blocks;
    const int32_t *table = a.tables + at;
    const float *weights = a.weights + at;
    const int rounds = K ? K : (a.max_blocks + THREADS - 1) / THREADS;
    float w[K ? K : 1];
    int id[K ? K : 1];
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int j = tid + THREADS * i;
        w[i] = j < a.max_blocks ? weights[j] : 0.0f;
        id[i] = j < a.max_blocks ? table[j] : 0;
    }
    const int cap = a.max_blocks * a.block_size;
    int ctx = a.lens[b];
    if (ctx < 0 || ctx > cap) {
        if (tid == 0) atomicOr(a.err_flag, kErrPagedRange);
        ctx = ctx < 0 ? 0 : cap;
    }
    const int n = ctx / a.block_size + (ctx % a.block_size != 0);
    const int gone = max(n - a.budget, 0), mid_end = n - a.last;
    const int left = a.budget - a.first - a.last;  // places for blocks [first, mid_end)
    __shared__ int s_count[2][kWaves];

    // (a block that does not compete has the key 0, which no bit counts)
    auto mid = [&](int j) { return j >= a.first && j < mid_end; };
    unsigned keys[K ? K : 1];
#pragma unroll
    for (int i = 0; i < K; ++i) keys[i] = mid(tid + THREADS * i) ? order_key(w[i]) : 0;
    auto key = [&](int i) {
        const int j = tid + THREADS * i;
        return K ? keys[K ? i : 0] : mid(j) ? order_key(weights[j]) : 0u;
    };
    unsigned least = ~0u;  // kept: keys above it, and the first ones equal to it
    if (gone > 0 && left > 0) {
        least = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const unsigned x = least | 1u << bit;
            int count = 0;
            if constexpr (K > 0) {
#pragma unroll
                for (int i = 0; i < K; ++i) count += __popcll(__ballot(keys[i] >= x));
            } else {
                for (int i = 0; i < rounds; ++i) count += __popcll(__ballot(key(i) >= x));
            }
            if (lane == 0) s_count[bit & 1][wave] = count;
            __syncthreads();
            count = 0;
#pragma unroll
            for (int v = 0; v < kWaves; ++v) count += s_count[bit & 1][v];
            if (count >= left) least = x;
            if (count == left) break;
        }
    }
    auto sure = [&](int i) {  // stays whatever the ties
        const int j = tid + THREADS * i;
        return j < n && (gone == 0 || !mid(j) || key(i) > least);
    };
    auto tied = [&](int i) {
        return gone > 0 && left > 0 && mid(tid + THREADS * i) && key(i) == least;
    };
    // before a block: `x` that surely stay and `y` ties, of which the first stay
    auto put = [&](int i, int2 before, int ties, uint64_t bs, uint64_t bt) {
        const int j = tid + THREADS * i;
        if (j >= n) return;
        const uint64_t below = (1ull << lane) - 1;
        before.x += __popcll(bs & below);
        before.y += __popcll(bt & below);
        const int to = before.x + min(before.y, ties);
        const int block = K ? id[K ? i : 0] : table[j];
        if ((bs >> lane & 1) || ((bt >> lane & 1) && before.y < ties)) {
            a.tables_out[at + to] = block;
            a.weights_out[at + to] = K ? w[K ? i : 0] : weights[j];
        } else {
            a.evicted[at + j - to] = block;
        }
    };
    if constexpr (K > 0) {
        // one scan over what every wave counts in every round, in block order
        constexpr int E = K * kWaves, PER = (E + 63) / 64;
        __shared__ int2 s_before[PER * 64];
        __shared__ int s_sure;
        uint64_t bs[K], bt[K];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            bs[i] = __ballot(sure(i));
            bt[i] = __ballot(tied(i));
            if (lane == 0) s_before[i * kWaves + wave] = make_int2(__popcll(bs[i]), __popcll(bt[i]));
        }
        __syncthreads();
        if (wave == 0) {
            int2 mine = {0, 0}, each[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                each[i] = lane * PER + i < E ? s_before[lane * PER + i] : make_int2(0, 0);
                mine.x += each[i].x;
                mine.y += each[i].y;
            }
            int2 inc = mine;
            for (int o = 1; o < 64; o <<= 1) {
                const int x = __shfl_up(inc.x, o, 64), y = __shfl_up(inc.y, o, 64);
                if (lane >= o) {
                    inc.x += x;
                    inc.y += y;
                }
            }
            if (lane == 63) s_sure = inc.x;
            inc.x -= mine.x;
            inc.y -= mine.y;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                s_before[lane * PER + i] = inc;
                inc.x += each[i].x;
                inc.y += each[i].y;
            }
        }
        __syncthreads();
        const int ties = gone > 0 ? a.budget - s_sure : 0;
#pragma unroll
        for (int i = 0; i < K; ++i) put(i, s_before[i * kWaves + wave], ties, bs[i], bt[i]);
    } else {
        __shared__ int2 s_wave[2][kWaves];
        int all = 0;
        for (int i = 0; i < rounds; ++i) all += __popcll(__ballot(sure(i)));
        __syncthreads();  // (s_count is done with)
        if (lane == 0) s_count[0][wave] = all;
        __syncthreads();
        all = 0;
        for (int v = 0; v < kWaves; ++v) all += s_count[0][v];
        const int ties = gone > 0 ? a.budget - all : 0;
        int2 base = {0, 0};
        for (int i = 0; i < rounds; ++i) {
            const uint64_t bs = __ballot(sure(i)), bt = __ballot(tied(i));
            if (lane == 0) s_wave[i & 1][wave] = make_int2(__popcll(bs), __popcll(bt));
            __syncthreads();
            int2 before = base;
            for (int v = 0; v < kWaves; ++v) {
                const int2 x = s_wave[i & 1][v];
                if (v < wave) {
                    before.x += x.x;
                    before.y += x.y;
                }
                base.x += x.x;
                base.y += x.y;
            }
            put(i, before, ties, bs, bt);
        }
    }
    for (int i = n - gone + tid; i < a.max_blocks; i += THREADS) {
        a.tables_out[at + i] = -1;
        a.weights_out[at + i] = 0.0f;
    }
    for (int i = gone + tid; i < a.max_blocks; i += THREADS) a.evicted[at + i] = -1;
    if (tid == 0) a.lens_out[b] = ctx - gone * a.block_size;
}

}  // namespace

void paged_evict(const EvictArgs &a, hipStream_t s) {
    if (a.max_blocks <= 256 * 4)
        evict_kernel<256, 4><<<a.num_seqs, 256, 0, s>>>(a);
    else if (a.max_blocks <= 256 * 16)
        evict_kernel<512, 8><<<a.num_seqs, 512, 0, s>>>(a);
    else if (a.max_blocks <= 1024 * 16)
        evict_kernel<1024, 16><<<a.num_seqs, 1024, 0, s>>>(a);
    else
        evict_kernel<1024, 0><<<a.num_seqs, 1024, 0, s>>>(a);
}

}  // namespace k
}  // namespace clove
