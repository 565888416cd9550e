// kv8.cpp -- host side of the paged KV cache in 8 bits and of block eviction:
// shape rules and launches (kernels/kv8_cache.hip, kv8_attention.hip,
// kv8_evict.hip).
#include <cmath>
#include <cstdint>

#include "common.hpp"
#include "kernels/launch.hpp"
#include "runtime.hpp"

namespace clove {

namespace {

void need_dtype(const Tensor &t, int dtype, const char *what) {
    static const char *names[] = {"f32", "int32", "e4m3"};
    CLOVE_REQUIRE(t.dtype == dtype, CLOVE_HIP_ERR_INVALID,
                  std::string(what) + " must be an " + names[dtype] + " tensor");
}

void tables_rule(const Tensor &bt, const Tensor &cl, size_t block_size) {
    need_dtype(bt, CLOVE_HIP_I32, "block_tables");
    need_dtype(cl, CLOVE_HIP_I32, "context_lens");
    CLOVE_REQUIRE(bt.shape.size() == 2 && bt.shape[0] == cl.numel, CLOVE_HIP_ERR_SHAPE,
                  "block_tables must be [num_seqs, max_blocks] with num_seqs = "
                  "numel(context_lens), got " + shape_str(bt.shape));
    CLOVE_REQUIRE(block_size >= 1 && block_size < (1ull << 31) && cl.numel < (1ull << 16) &&
                      bt.shape[1] < (1ull << 24) && bt.shape[1] * block_size < (1ull << 31),
                  CLOVE_HIP_ERR_SHAPE,
                  "block_size must be >= 1, a context's capacity below 2^31 tokens and 2^24 "
                  "blocks, and the sequences fewer than 2^16");
}

// The rules that every entry over the cache shares; `rows` rows in the call.
k::Kv8Args cache_args(const Tensor &codes, const Tensor &exps, const Tensor &bt,
                      const Tensor &cl, const Tensor *rs, size_t rows) {
    need_dtype(codes, CLOVE_HIP_E4M3, "codes");
    need_dtype(exps, CLOVE_HIP_I32, "exps");
    CLOVE_REQUIRE(codes.shape.size() == 5 && codes.shape[0] == 2, CLOVE_HIP_ERR_SHAPE,
                  "codes must be [2, num_blocks, heads, block_size, head_dim], got " +
                      shape_str(codes.shape));
    const size_t nb = codes.shape[1], H = codes.shape[2], bs = codes.shape[3], D = codes.shape[4];
    CLOVE_REQUIRE(exps.shape == (std::vector<size_t>{2, nb, H}), CLOVE_HIP_ERR_SHAPE,
                  "exps must be [2, num_blocks, heads] of codes " + shape_str(codes.shape) +
                      ", got " + shape_str(exps.shape));
    CLOVE_REQUIRE(D >= 1 && D <= (size_t)k::kKv8MaxHeadDim, CLOVE_HIP_ERR_SHAPE,
                  "the 8-bit cache supports head_dim 1.." + std::to_string(k::kKv8MaxHeadDim) +
                      ", got " + std::to_string(D));
    CLOVE_REQUIRE(H >= 1 && H <= 65535 && nb < (1ull << 31) && bs < (1ull << 20),
                  CLOVE_HIP_ERR_SHAPE,
                  "the 8-bit cache supports 1..65535 heads, blocks of fewer than 2^20 tokens and "
                  "fewer than 2^31 of them");
    tables_rule(bt, cl, bs);
    if (rs) {
        need_dtype(*rs, CLOVE_HIP_I32, "row_starts");
        CLOVE_REQUIRE(rs->numel == cl.numel + 1, CLOVE_HIP_ERR_SHAPE,
                      "row_starts must hold num_seqs + 1 = " + std::to_string(cl.numel + 1) +
                          " elements, got " + std::to_string(rs->numel));
    } else {
        CLOVE_REQUIRE(rows == cl.numel, CLOVE_HIP_ERR_SHAPE,
                      "without row_starts there is one row for each sequence: " +
                          std::to_string(cl.numel) + ", got " + std::to_string(rows));
    }
    // grids count threads in 32 bits, up to 256 a row
    CLOVE_REQUIRE(rows < (1ull << 24), CLOVE_HIP_ERR_SHAPE,
                  "the rows of a call must be fewer than 2^24");
    // (the append and the read cut the rows into tiles of a block and head)
    CLOVE_REQUIRE((rows / bs + 2 * cl.numel) * ((H + 3) / 4) * 2 + rows < (1ull << 32),
                  CLOVE_HIP_ERR_SHAPE, "too many rows and heads");
    k::Kv8Args a{};
    a.codes = codes.u8();
    a.exps = exps.i32();
    a.block_tables = bt.i32();
    a.context_lens = cl.i32();
    a.row_starts = rs ? rs->i32() : nullptr;
    a.err_flag = device_error_flag();
    a.num_blocks = (int64_t)nb;
    a.num_seqs = (int)cl.numel;
    a.max_blocks = (int)bt.shape[1];
    a.block_size = (int)bs;
    a.num_heads = (int)H;
    a.head_dim = (int)D;
    a.rows = (int)rows;
    return a;
}

size_t row_floats(const Tensor &codes) {
    return codes.shape.size() == 5 ? codes.shape[2] * codes.shape[4] : 0;
}

// Rows of an f32 tensor whose row holds `row` elements.
size_t rows_of(const Tensor &t, size_t row, const char *what) {
    need_dtype(t, CLOVE_HIP_F32, what);
    CLOVE_REQUIRE(row > 0 && t.numel % row == 0, CLOVE_HIP_ERR_SHAPE,
                  std::string(what) + " must hold whole rows of " + std::to_string(row) +
                      " elements, got " + shape_str(t.shape));
    return t.numel / row;
}

}  // namespace

void HipBackend::paged_kv8_append(const Tensor &codes, const Tensor &exps, const Tensor &k,
                                  const Tensor &v, const Tensor &bt, const Tensor &cl,
                                  const Tensor *rs) {
    const size_t row = row_floats(codes);
    const size_t rows = rows_of(k, row ? row : 1, "k");
    CLOVE_REQUIRE(rows_of(v, row ? row : 1, "v") == rows, CLOVE_HIP_ERR_SHAPE,
                  "k and v must have the same number of elements");
    const k::Kv8Args a = cache_args(codes, exps, bt, cl, rs, rows);
    if (a.num_seqs == 0 || a.rows == 0) return;
    k::kv8_append(a, k.f32(), v.f32(), ctx().stream);
}

void HipBackend::paged_kv8_read(const Tensor &codes, const Tensor &exps, const Tensor &bt,
                                const Tensor &cl, const Tensor *rs, size_t rows, TensorNode *k,
                                TensorNode *v) {
    const k::Kv8Args a = cache_args(codes, exps, bt, cl, rs, rows);
    *k = new_tensor({rows, row_floats(codes)}, CLOVE_HIP_F32);
    *v = new_tensor({rows, row_floats(codes)}, CLOVE_HIP_F32);
    if (a.rows == 0) return;
    k::kv8_read(a, (*k)->f32(), (*v)->f32(), ctx().stream);
}

TensorNode HipBackend::paged_kv8_attention(const Tensor &q, const Tensor &codes,
                                           const Tensor &exps, const Tensor &bt,
                                           const Tensor &cl, const Tensor *rs, float scale,
                                           const Tensor *weights, TensorNode *weights_out) {
    need_dtype(q, CLOVE_HIP_F32, "q");
    CLOVE_REQUIRE(q.shape.size() >= 2, CLOVE_HIP_ERR_SHAPE,
                  "q must be [rows, query heads * head_dim], got " + shape_str(q.shape));
    const size_t X = q.shape.back(), row = row_floats(codes);
    CLOVE_REQUIRE(row > 0 && X > 0 && X % row == 0 && X < (1ull << 31), CLOVE_HIP_ERR_SHAPE,
                  "q's last dimension must be a multiple of heads * head_dim = " +
                      std::to_string(row) + ", got " + std::to_string(X));
    k::Kv8Attention a{};
    a.c = cache_args(codes, exps, bt, cl, rs, q.numel / X);
    a.q_heads = (int)(X / (size_t)a.c.head_dim);
    // (the kernels number tokens in 31 bits, up to a table of 4096 past the last)
    CLOVE_REQUIRE(bt.shape[1] * (size_t)a.c.block_size <= (1ull << 31) - 8192, CLOVE_HIP_ERR_SHAPE,
                  "attention supports a capacity of up to 2^31 - 8192 tokens a context");
    CLOVE_REQUIRE((size_t)a.c.rows * (size_t)a.q_heads < (1ull << 31) && a.q_heads <= 65535,
                  CLOVE_HIP_ERR_SHAPE, "too many rows and query heads");
    if (weights) {
        need_dtype(*weights, CLOVE_HIP_F32, "weights");
        CLOVE_REQUIRE(weights->shape == bt.shape, CLOVE_HIP_ERR_SHAPE,
                      "weights must be [num_seqs, max_blocks] = " + shape_str(bt.shape) +
                          ", got " + shape_str(weights->shape));
        *weights_out = new_tensor(bt.shape, CLOVE_HIP_F32);
        a.w_in = weights->f32();
        a.w_out = (*weights_out)->f32();
    }
    TensorNode out = new_tensor(q.shape, CLOVE_HIP_F32);
    a.q = q.f32();
    a.out = out->f32();
    a.scale = scale > 0.0f ? scale : 1.0f / std::sqrt((float)a.c.head_dim);
    const int cus = ctx().num_cus;
    const size_t bytes = k::kv8_attention_workspace(a, cus);
    TensorNode ws;
    if (bytes) {
        ws = new_tensor({(bytes + 3) / 4}, CLOVE_HIP_F32);
        a.ws = ws->f32();
    }
    k::kv8_attention(a, cus, ctx().stream);
    return out;
}

void HipBackend::paged_evict(const Tensor &bt, const Tensor &cl, const Tensor &weights,
                             int block_size, int budget, int first, int last,
                             TensorNode out[4]) {
    CLOVE_REQUIRE(block_size >= 1, CLOVE_HIP_ERR_INVALID, "evict: block_size must be >= 1");
    tables_rule(bt, cl, (size_t)block_size);
    need_dtype(weights, CLOVE_HIP_F32, "weights");
    CLOVE_REQUIRE(weights.shape == bt.shape, CLOVE_HIP_ERR_SHAPE,
                  "evict: weights must be [num_seqs, max_blocks] = " + shape_str(bt.shape) +
                      ", got " + shape_str(weights.shape));
    CLOVE_REQUIRE(first >= 0 && last >= 1 && budget >= 1 && (int64_t)first + last <= budget,
                  CLOVE_HIP_ERR_INVALID,
                  "evict: first >= 0, last >= 1 and first + last <= budget are required");
    out[0] = new_tensor(bt.shape, CLOVE_HIP_I32);
    out[1] = new_tensor(cl.shape, CLOVE_HIP_I32);
    out[2] = new_tensor(bt.shape, CLOVE_HIP_F32);
    out[3] = new_tensor(bt.shape, CLOVE_HIP_I32);
    if (cl.numel == 0) return;
    k::EvictArgs a{};
    a.tables = bt.i32();
    a.lens = cl.i32();
    a.weights = weights.f32();
    a.tables_out = out[0]->i32();
    a.lens_out = out[1]->i32();
    a.weights_out = out[2]->f32();
    a.evicted = out[3]->i32();
    a.err_flag = device_error_flag();
    a.num_seqs = (int)cl.numel;
    a.max_blocks = (int)bt.shape[1];
    a.block_size = block_size;
    a.budget = budget;
    a.first = first;
    a.last = last;
    k::paged_evict(a, ctx().stream);
}

}  // namespace clove
