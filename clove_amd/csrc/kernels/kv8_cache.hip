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
//
// Bound by memory: five bytes an element.  Eight prompts of 200 to 2048 rows, 32
// heads of 128, stored and read back: 166 us for 10 bytes an element at 4.2 TB/s
// (a large copy: 4.9; one workgroup a tile, the rows read twice: 371).  A token for
// each of 32 sequences is two launches of 4 and 6 us, each a chain of dependent
// loads (row range, context, block, exponent, rows): 13 us with their submission.
#include <algorithm>

#include "kv8.h"
#include "wave.h"

namespace clove {
namespace k {

namespace {

// The tile that slot blockIdx.y of an append or read stands for: `item` blocks
// behind the one with the sequence's first row.
struct RowTile {
    int b, j;        // sequence and logical block
    int lo, hi;      // its slots among the rows
    int64_t row0;    // slot s is row row0 + s
};
__device__ __forceinline__ bool row_tile(const Kv8Args &a, int slot, RowTile *t) {
    int item, first, n;
    t->b = kv8_slot(a, slot, a.block_size, 1, 2, &item);
    kv8_rows(a, t->b, &first, &n);
    const int ctx = kv8_context(a, t->b);
    // rows at negative positions are skipped
    const int past = max(ctx - n, 0), skip = max(n - ctx, 0);
    const int64_t j = (int64_t)past / a.block_size + item, t0 = j * a.block_size;
    if (item < 0 || t0 >= ctx || n - skip <= 0) return false;
    t->j = (int)j;
    t->lo = (int)max((int64_t)past - t0, (int64_t)0);
    t->hi = (int)min((int64_t)ctx - t0, (int64_t)a.block_size);
    t->row0 = first + skip + (t0 - past);
    return true;
}

// Workgroups of four waves, a wave a head, neighbouring heads side by side: the
// rows are read and written in runs of whole lines.  NV > 0: a tile's new rows
// are at most 256 * NV elements and stay in registers between their maximum and
// their codes, four a lane (head_dim a multiple of 4, rows 16-byte aligned).
// NV = 0: any shape, the rows read twice.
template <int NV>
__global__ void __launch_bounds__(256) append_kernel(Kv8Args a, const float *k, const float *v,
                                                     unsigned done) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int groups = (a.num_heads + 3) / 4;
    const unsigned block = blockIdx.x + done;
    const int plane = block / groups % 2, slot = block / groups / 2;
    const int h = block % groups * 4 + wave;
    if (block == 0 && wave == 0) kv8_check(a);
    RowTile t;
    if (h >= a.num_heads || !row_tile(a, slot, &t)) return;
    const int D = a.head_dim;
    const size_t X = (size_t)a.num_heads * D;
    const float *x = (plane ? v : k) + (size_t)(t.row0 + t.lo) * X + (size_t)h * D;
    const int count = (t.hi - t.lo) * D;

    float amax = 0.0f;
    bool bad = false;
    auto look = [&](float f) {
        if (kv8_finite(f))
            amax = fmaxf(amax, fabsf(f));
        else
            bad = true;
    };
    cl_f4 y[NV > 0 ? NV : 1];
    const int D4 = D / 4;
    const unsigned magic = D4 > 1 ? (unsigned)(((1ull << 32) + D4 - 1) / D4) : 0;
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = lane + 64 * i;
            const int s = D4 > 1 ? __umulhi(e, magic) : e;
            y[i] = (cl_f4){0.f, 0.f, 0.f, 0.f};
            if (4 * e < count) y[i] = *reinterpret_cast<const cl_f4 *>(x + (size_t)s * X + 4 * (e - s * D4));
        }
    }
    const int64_t id = kv8_block(a, t.b, t.j, h == 0 && plane == 0 && lane == 0);
    if (id < 0) return;
    const size_t tile = kv8_tile(a, plane, id, h);
    uint8_t *codes = a.codes + kv8_tile_offset(a, tile);
    int old = kKv8MinExp;
    if (t.lo > 0) old = min(max(a.exps[tile], kKv8MinExp), kKv8MaxExp);
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) look(y[i][e]);
    } else {
        for (int i = lane; i < count; i += 64) look(x[(size_t)(i / D) * X + i % D]);
    }
    amax = wave_max(amax);
    if (__any(bad) && lane == 0) atomicOr(a.err_flag, kErrNotFinite);
    const int e = max(kv8_exp_of(amax), old);
    if (t.lo > 0 && e > old) {  // the tokens before, under the larger exponent
        const float r = kv8_pow2(max(old - e, -126));
        if constexpr (NV > 0) {
            unsigned *w = reinterpret_cast<unsigned *>(codes);
            for (int i = lane; i < t.lo * D4; i += 64) {
                const unsigned c = w[i];
                w[i] = kv8_encode4(__builtin_amdgcn_cvt_f32_fp8(c, 0) * r,
                                   __builtin_amdgcn_cvt_f32_fp8(c, 1) * r,
                                   __builtin_amdgcn_cvt_f32_fp8(c, 2) * r,
                                   __builtin_amdgcn_cvt_f32_fp8(c, 3) * r);
            }
        } else {
            for (int i = lane; i < t.lo * D; i += 64) codes[i] = kv8_encode(kv8_decode(codes[i]) * r);
        }
    }
    const float inv = kv8_pow2(-e);
    if constexpr (NV > 0) {
        unsigned *w = reinterpret_cast<unsigned *>(codes) + t.lo * D4;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (4 * (lane + 64 * i) < count)
                w[lane + 64 * i] = kv8_encode4(y[i].x * inv, y[i].y * inv, y[i].z * inv, y[i].w * inv);
    } else {
        for (int i = lane; i < count; i += 64)
            codes[(size_t)t.lo * D + i] = kv8_encode(x[(size_t)(i / D) * X + i % D] * inv);
    }
    if (lane == 0) a.exps[tile] = e;
}

// The same cut the other way round; VEC: four elements a lane.  Workgroups from
// `main` on write zeros for the rows that no tile holds.
template <bool VEC>
__global__ void __launch_bounds__(256) read_kernel(Kv8Args a, float *k, float *v, unsigned main,
                                                   unsigned done) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int D = a.head_dim;
    const size_t X = (size_t)a.num_heads * D;
    const unsigned block = blockIdx.x + done;
    if (block >= main) {
        const int r = (int)(block - main) * 4 + wave;
        if (block == main && wave == 0) kv8_check(a);
        if (r >= a.rows) return;
        const int b = kv8_seq_of_row(a, r);
        int pos = -1;
        if (b >= 0) {
            int first, n;
            kv8_rows(a, b, &first, &n);
            pos = kv8_context(a, b) - n + (r - first);
        }
        if (pos < 0)
            for (size_t d = lane; d < X; d += 64) k[r * X + d] = v[r * X + d] = 0.0f;
        return;
    }
    const int groups = (a.num_heads + 3) / 4;
    const int plane = block / groups % 2, slot = block / groups / 2;
    const int h = block % groups * 4 + wave;
    RowTile t;
    if (h >= a.num_heads || !row_tile(a, slot, &t)) return;
    const int64_t id = kv8_block(a, t.b, t.j, h == 0 && plane == 0 && lane == 0);
    float *x = (plane ? v : k) + (size_t)(t.row0 + t.lo) * X + (size_t)h * D;
    const int count = (t.hi - t.lo) * D;
    const size_t tile = kv8_tile(a, plane, max(id, (int64_t)0), h);
    // (outside the pool: zeros; nothing is read there)
    const float scale = id < 0 ? 0.0f : kv8_scale(a.exps[tile]);
    const uint8_t *codes = a.codes + kv8_tile_offset(a, tile) + (size_t)t.lo * D;
    if constexpr (VEC) {
        const int D4 = D / 4;
        const unsigned magic = D4 > 1 ? (unsigned)(((1ull << 32) + D4 - 1) / D4) : 0;
        for (int e0 = 0; 4 * e0 < count; e0 += 256) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = e0 + lane + 64 * i;
                if (4 * e >= count) continue;
                const int s = D4 > 1 ? __umulhi(e, magic) : e;
                const unsigned c = id < 0 ? 0 : reinterpret_cast<const unsigned *>(codes)[e];
                *reinterpret_cast<cl_f4 *>(x + (size_t)s * X + 4 * (e - s * D4)) =
                    (cl_f4){__builtin_amdgcn_cvt_f32_fp8(c, 0) * scale,
                            __builtin_amdgcn_cvt_f32_fp8(c, 1) * scale,
                            __builtin_amdgcn_cvt_f32_fp8(c, 2) * scale,
                            __builtin_amdgcn_cvt_f32_fp8(c, 3) * scale};
            }
        }
    } else {
        for (int i = lane; i < count; i += 64)
            x[(size_t)(i / D) * X + i % D] = id < 0 ? 0.0f : kv8_decode(codes[i]) * scale;
    }
}

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// A grid holds 2^32 threads: more workgroups of 256 go in several launches.
template <class F>
void in_grids(int64_t n, F launch) {
    constexpr int64_t kMost = 1 << 23;
    for (int64_t done = 0; done < n; done += kMost)
        launch((unsigned)std::min(n - done, kMost), (unsigned)done);
}

int64_t tile_groups(const Kv8Args &a) {
    return kv8_slots(a, a.block_size, 1, 2) * ((a.num_heads + 3) / 4) * 2;
}

}  // namespace

void kv8_append(const Kv8Args &a, const float *k, const float *v, hipStream_t s) {
    const bool vec = a.head_dim % 4 == 0 && aligned(k, 16) && aligned(v, 16) && aligned(a.codes, 4);
    // the most new elements of a tile
    const int64_t n = (int64_t)std::min(a.row_starts ? a.rows : 1, a.block_size) * a.head_dim;
    in_grids(tile_groups(a), [&](unsigned grid, unsigned done) {
        if (vec && n <= 256 * 2)
            append_kernel<2><<<grid, 256, 0, s>>>(a, k, v, done);
        else if (vec && n <= 256 * 8)
            append_kernel<8><<<grid, 256, 0, s>>>(a, k, v, done);
        else if (vec && n <= 256 * 32)
            append_kernel<32><<<grid, 256, 0, s>>>(a, k, v, done);
        else
            append_kernel<0><<<grid, 256, 0, s>>>(a, k, v, done);
    });
}

void kv8_read(const Kv8Args &a, float *k, float *v, hipStream_t s) {
    const int64_t main = a.num_seqs == 0 ? 0 : tile_groups(a);
    in_grids(main + (a.rows + 3) / 4, [&](unsigned grid, unsigned done) {
        if (a.head_dim % 4 == 0 && aligned(a.codes, 4))
            read_kernel<true><<<grid, 256, 0, s>>>(a, k, v, (unsigned)main, done);
        else
            read_kernel<false><<<grid, 256, 0, s>>>(a, k, v, (unsigned)main, done);
    });
}

}  // namespace k
}  // namespace clove
