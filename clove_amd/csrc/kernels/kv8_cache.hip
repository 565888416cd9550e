// kv8_cache.hip -- storing rows in the 8-bit paged cache and reading them back.
//
// A tile (plane, block, head) is block_size * head_dim codes with one exponent.
// The append gives one wave to each tile that receives rows:
//   amax = max |x| over its new, finite elements,
//   e    = smallest exponent with amax <= 448 * 2^e; at least the tile's old one
//          when tokens stand before the new rows,
//   code = round_e4m3(x * 2^-e),
// and where e grew, the tokens before are rounded again, c * 2^(old - e).
// Scaling by a power of two is exact, so every element is rounded once.
#include "kv8.h"
#include "wave.h"

namespace clove {
namespace k {

namespace {

__global__ void __launch_bounds__(64) kv8_append_kernel(Kv8Args a, const float *k, const float *v) {
    const int lane = threadIdx.x, h = blockIdx.y, plane = blockIdx.z;
    if (blockIdx.x == 0 && h == 0 && plane == 0) kv8_check(a);
    int item;
    const int b = kv8_slot(a, blockIdx.x, a.block_size, 1, 2, &item);
    int first, n;
    kv8_rows(a, b, &first, &n);
    const int ctx = kv8_context(a, b);
    // rows at negative positions are skipped
    const int past = max(ctx - n, 0), skip = max(n - ctx, 0);
    const int bs = a.block_size, D = a.head_dim;
    const int64_t j = (int64_t)past / bs + item;
    const int64_t t0 = j * bs;
    if (item < 0 || t0 >= ctx || n - skip <= 0) return;
    const int64_t id = kv8_block(a, b, (int)j, h == 0 && plane == 0 && lane == 0);
    if (id < 0) return;
    // new slots [lo, hi) of the tile; slot s is row `row0 + s`
    const int lo = (int)max((int64_t)past - t0, (int64_t)0);
    const int hi = (int)min((int64_t)ctx - t0, (int64_t)bs);
    const int64_t row0 = first + skip + (t0 - past);
    const size_t tile = kv8_tile(a, plane, id, h);
    uint8_t *codes = a.codes + kv8_tile_offset(a, tile);
    const float *x = (plane ? v : k) + (size_t)h * D;
    const size_t X = (size_t)a.num_heads * D;

    const int count = (hi - lo) * D;
    float amax = 0.0f;
    bool bad = false;
    for (int i = lane; i < count; i += 64) {
        const int s = i / D, d = i - s * D;
        const float f = x[(size_t)(row0 + lo + s) * X + d];
        if (kv8_finite(f))
            amax = fmaxf(amax, fabsf(f));
        else
            bad = true;
    }
    amax = wave_max(amax);
    if (__any(bad) && lane == 0) atomicOr(a.err_flag, kErrNotFinite);
    int e = kv8_exp_of(amax);
    if (lo > 0) {
        const int old = min(max(a.exps[tile], kKv8MinExp), kKv8MaxExp);
        if (e > old) {
            const float r = kv8_pow2(max(old - e, -126));
            for (int i = lane; i < lo * D; i += 64) codes[i] = kv8_encode(kv8_decode(codes[i]) * r);
        }
        e = max(e, old);
    }
    const float inv = kv8_pow2(-e);
    for (int i = lane; i < count; i += 64) {
        const int s = i / D, d = i - s * D;
        codes[(size_t)(lo + s) * D + d] = kv8_encode(x[(size_t)(row0 + lo + s) * X + d] * inv);
    }
    if (lane == 0) a.exps[tile] = e;
}

__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8Args a, float *k, float *v) {
    const int r = blockIdx.x, plane = blockIdx.y;
    const int D = a.head_dim, bs = a.block_size;
    if (r == 0 && plane == 0 && threadIdx.x < 64) kv8_check(a);
    const int b = kv8_seq_of_row(a, r);
    int64_t id = -1;
    int slot = 0;
    if (b >= 0) {
        int first, n;
        kv8_rows(a, b, &first, &n);
        const int ctx = kv8_context(a, b);
        const int pos = ctx - n + (r - first);
        if (pos >= 0) {
            id = kv8_block(a, b, pos / bs, plane == 0 && threadIdx.x == 0);
            slot = pos % bs;
        }
    }
    const int X = a.num_heads * D;
    float *out = (plane ? v : k) + (size_t)r * X;
    for (int i = threadIdx.x; i < X; i += 256) {
        const int h = i / D, d = i - h * D;
        float f = 0.0f;
        if (id >= 0) {
            const size_t tile = kv8_tile(a, plane, id, h);
            f = kv8_decode(a.codes[kv8_tile_offset(a, tile) + (size_t)slot * D + d]) *
                kv8_scale(a.exps[tile]);
        }
        out[i] = f;
    }
}

}  // namespace

void kv8_append(const Kv8Args &a, const float *k, const float *v, hipStream_t s) {
    const unsigned slots = (unsigned)kv8_slots(a, a.block_size, 1, 2);
    kv8_append_kernel<<<dim3(slots, a.num_heads, 2), 64, 0, s>>>(a, k, v);
}

void kv8_read(const Kv8Args &a, float *k, float *v, hipStream_t s) {
    kv8_read_kernel<<<dim3(a.rows, 2), 256, 0, s>>>(a, k, v);
}

}  // namespace k
}  // namespace clove
