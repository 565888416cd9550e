// kv8_attention.hip -- attention over the 8-bit paged cache: per row i of a
// sequence (position p) and query head h, with kv head g = h / (Hq / H),
//   s_t = scale * q . K_t,  out = sum_t softmax_t(s) V_t,  t = 0 .. p.
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
// for the sum over V.  ml (or null) receives the row's maximum and sum.
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

}  // namespace

size_t kv8_attention_workspace(const Kv8Attention &a, int) {
    return a.w_out ? (size_t)a.c.rows * a.q_heads * sizeof(float2) : 0;
}

void kv8_attention(const Kv8Attention &a, int, hipStream_t s) {
    float2 *ml = reinterpret_cast<float2 *>(a.ws);
    if (a.c.rows > 0)
        kv8_attention_any_kernel<<<dim3(a.c.rows, a.q_heads), 64, 0, s>>>(a, ml);
    if (a.w_out && a.c.num_seqs > 0 && a.c.max_blocks > 0)
        kv8_weights_any_kernel<<<dim3(a.c.max_blocks, a.c.num_seqs), 256, 0, s>>>(a, ml);
}

}  // namespace k
}  // namespace clove
