// kv8_evict.hip -- eviction of the lightest blocks of long sequences.
//
// One workgroup a sequence.  Of its n = ceil(ctx / block_size) blocks the first
// and last ones stay; of the m between them the (budget - first - last) heaviest
// do.  The weight of the last one that stays is found by radix selection, a byte
// of the order-preserving key a pass (four histograms of 256 bins), then one
// ordered pass writes kept and evicted blocks: among equal weights the earlier
// blocks stay.  Only integers are counted, so results do not depend on timing.
#include "kv8.h"

namespace clove {
namespace k {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;

// Unsigned keys in the order of the weights; NaN lowest, -0 as 0.
__device__ __forceinline__ unsigned order_key(float w) {
    if (w != w) return 0;
    const unsigned u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum over the workgroup in thread order; *total gets the whole sum.
__device__ __forceinline__ int block_scan(int v, int *s_wave, int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int inc = v;
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(inc, o, 64);
        if (lane >= o) inc += up;
    }
    __syncthreads();
    if (lane == 63) s_wave[wave] = inc;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kWaves; ++w) {
        const int x = s_wave[w];
        if (w < wave) before += x;
        all += x;
    }
    *total = all;
    return before + inc - v;
}

__global__ void __launch_bounds__(kThreads) evict_kernel(EvictArgs a) {
    const int b = blockIdx.x, tid = threadIdx.x;
    const size_t at = (size_t)b * a.max_blocks;
    const int32_t *table = a.tables + at;
    const float *w = a.weights + at;
    const int cap = a.max_blocks * a.block_size;
    int ctx = a.lens[b];
    if (ctx < 0 || ctx > cap) {
        if (tid == 0) atomicOr(a.err_flag, kErrPagedRange);
        ctx = ctx < 0 ? 0 : cap;
    }
    const int n = ctx / a.block_size + (ctx % a.block_size != 0);
    const int gone_all = max(n - a.budget, 0);
    __shared__ int hist[256], s_wave[kWaves], s_byte, s_left;

    // blocks [first, n - last) compete for `left` places
    const int mid_end = n - a.last;
    unsigned prefix = 0, mask = 0;
    int left = a.budget - a.first - a.last;
    if (gone_all > 0 && left > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
            __syncthreads();
            for (int i = a.first + tid; i < mid_end; i += kThreads) {
                const unsigned key = order_key(w[i]);
                if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int byte = 255, need = left;
                while (byte > 0 && hist[byte] < need) need -= hist[byte--];
                s_byte = byte;
                s_left = need;
            }
            __syncthreads();
            prefix |= (unsigned)s_byte << shift;
            mask |= 255u << shift;
            left = s_left;
            __syncthreads();
        }
    }
    // kept: key above prefix, or equal to it and among the first `left` of those
    const bool some = a.budget - a.first - a.last > 0;
    const int per = (n + kThreads - 1) / kThreads;
    const int i0 = min(tid * per, n), i1 = min(i0 + per, n);
    int ties = 0;
    if (gone_all > 0 && some)
        for (int i = max(i0, a.first); i < min(i1, mid_end); ++i)
            ties += order_key(w[i]) == prefix;
    int total;
    int tie_at = block_scan(ties, s_wave, &total);
    auto keeps = [&](int i) {
        if (gone_all == 0 || i < a.first || i >= mid_end) return true;
        if (!some) return false;
        const unsigned key = order_key(w[i]);
        return key > prefix || (key == prefix && tie_at++ < left);
    };
    const int tie0 = tie_at;
    int kept = 0;
    for (int i = i0; i < i1; ++i) kept += keeps(i);
    const int kept_at = block_scan(kept, s_wave, &total);
    tie_at = tie0;
    int to = kept_at, out = i0 - kept_at;
    for (int i = i0; i < i1; ++i) {
        if (keeps(i)) {
            a.tables_out[at + to] = table[i];
            a.weights_out[at + to] = w[i];
            ++to;
        } else {
            a.evicted[at + out++] = table[i];
        }
    }
    for (int i = n - gone_all + tid; i < a.max_blocks; i += kThreads) {
        a.tables_out[at + i] = -1;
        a.weights_out[at + i] = 0.0f;
    }
    for (int i = gone_all + tid; i < a.max_blocks; i += kThreads) a.evicted[at + i] = -1;
    if (tid == 0) a.lens_out[b] = ctx - gone_all * a.block_size;
}

}  // namespace

void paged_evict(const EvictArgs &a, hipStream_t s) {
    evict_kernel<<<a.num_seqs, kThreads, 0, s>>>(a);
}

}  // namespace k
}  // namespace clove
