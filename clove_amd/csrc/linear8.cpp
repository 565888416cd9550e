// linear8.cpp -- host side of 8-bit linear layers and the root-mean-square norm:
// shape rules and launches (kernels/norm8.hip, quant8.hip, gemm8.hip).
#include <cmath>
#include <cstdint>

#include "common.hpp"
#include "kernels/launch.hpp"
#include "runtime.hpp"

namespace clove {

namespace {

// (the kernels count a row's columns in 31 bits, a little past its end)
constexpr size_t kMaxDim = (size_t(1) << 31) - 4096;

void rows_cols(const Tensor &t, const char *what, size_t *rows, size_t *cols) {
    CLOVE_REQUIRE(!t.shape.empty(), CLOVE_HIP_ERR_SHAPE,
                  std::string(what) + " needs at least 1 dimension");
    *cols = t.shape.back();
    *rows = 1;
    for (size_t i = 0; i + 1 < t.shape.size(); ++i) *rows *= t.shape[i];
    CLOVE_REQUIRE(*rows < kMaxDim && *cols < kMaxDim, CLOVE_HIP_ERR_SHAPE,
                  std::string(what) + " has dimensions of 2^31 - 4096 or more");
}

size_t blocks_of(size_t n) { return (n + 127) / 128; }

void same_shape(const Tensor &t, const Tensor &x, const char *what) {
    need_dtype(t, CLOVE_HIP_F32, what);
    CLOVE_REQUIRE(t.shape == x.shape, CLOVE_HIP_ERR_SHAPE,
                  std::string(what) + " must be " + shape_str(x.shape) + ", got " +
                      shape_str(t.shape));
}

void gamma_rule(const Tensor &gamma, size_t cols, float eps) {
    need_dtype(gamma, CLOVE_HIP_F32, "gamma");
    CLOVE_REQUIRE(gamma.numel == cols, CLOVE_HIP_ERR_SHAPE,
                  "gamma must hold " + std::to_string(cols) + " elements, got " +
                      shape_str(gamma.shape));
    CLOVE_REQUIRE(eps >= 0.0f && std::isfinite(eps), CLOVE_HIP_ERR_INVALID,
                  "eps must be finite and >= 0");
}

// x's shape with its last dimension replaced.
std::vector<size_t> with_last(const Tensor &x, size_t last) {
    std::vector<size_t> s = x.shape;
    s.back() = last;
    return s;
}

// The norm's arguments but for its output.
k::RmsNormArgs norm_args(const Tensor &x, const Tensor *residual, const Tensor &gamma, float eps,
                         TensorNode *sum, TensorNode *stats) {
    need_dtype(x, CLOVE_HIP_F32, "x");
    k::RmsNormArgs a{};
    size_t cols;
    rows_cols(x, "x", &a.rows, &cols);
    if (residual) same_shape(*residual, x, "residual");
    CLOVE_REQUIRE(residual || !sum, CLOVE_HIP_ERR_INVALID, "a sum needs a residual");
    gamma_rule(gamma, cols, eps);
    if (sum) *sum = new_tensor(x.shape, CLOVE_HIP_F32);
    a.x = x.f32();
    a.residual = residual ? residual->f32() : nullptr;
    a.gamma = gamma.f32();
    a.sum = sum ? (*sum)->f32() : nullptr;
    a.cols = (int)cols;
    a.eps = eps;
    if (const size_t n = k::rms_norm_stats(a.rows, a.cols)) {
        *stats = new_tensor({2 * n}, CLOVE_HIP_F32);
        a.stats = static_cast<double *>((*stats)->data);
    }
    return a;
}

// rows x blocks of a matrix in 8 bits, its exponents' kind.
void operand_rule(const Tensor &codes, const Tensor &exps, const char *what, size_t *rows,
                  size_t *blocks, bool *tiles) {
    const std::string name(what);
    need_dtype(codes, CLOVE_HIP_E4M3, what);
    need_dtype(exps, CLOVE_HIP_I32, (name + "_exps").c_str());
    size_t kp;
    rows_cols(codes, what, rows, &kp);
    CLOVE_REQUIRE(kp % 128 == 0 && kp < (size_t(1) << 23), CLOVE_HIP_ERR_SHAPE,
                  name + "'s last dimension must be a multiple of 128 below 2^23, got " +
                      std::to_string(kp));
    *blocks = kp / 128;
    const size_t last = exps.shape.empty() ? 0 : exps.shape.back();
    const size_t lines = last ? exps.numel / last : 0;
    CLOVE_REQUIRE(codes.numel == 0 ||
                      (last == *blocks && (lines == *rows || lines == blocks_of(*rows))),
                  CLOVE_HIP_ERR_SHAPE,
                  name + "_exps must hold an exponent for each 128 codes of " +
                      std::to_string(*rows) + " rows or of " +
                      std::to_string(blocks_of(*rows)) + " blocks of rows, [.., " +
                      std::to_string(*blocks) + "], got " + shape_str(exps.shape));
    *tiles = lines != *rows;
    CLOVE_REQUIRE(k::aligned16(codes.data), CLOVE_HIP_ERR_INVALID,
                  name + " must be 16-byte aligned");
}

}  // namespace

TensorNode HipBackend::rms_norm(const Tensor &x, const Tensor *residual, const Tensor &gamma,
                                float eps, TensorNode *sum) {
    TensorNode stats;
    k::RmsNormArgs a = norm_args(x, residual, gamma, eps, sum, &stats);
    TensorNode out = new_tensor(x.shape, CLOVE_HIP_F32);
    a.out = out->f32();
    k::rms_norm(a, ctx().stream);
    return out;
}

void HipBackend::rms_norm_e4m3(const Tensor &x, const Tensor *residual, const Tensor &gamma,
                               float eps, TensorNode *sum, TensorNode *codes, TensorNode *exps) {
    TensorNode stats;
    k::RmsNormArgs a = norm_args(x, residual, gamma, eps, sum, &stats);
    *codes = new_tensor(with_last(x, blocks_of((size_t)a.cols) * 128), CLOVE_HIP_E4M3);
    *exps = new_tensor(with_last(x, blocks_of((size_t)a.cols)), CLOVE_HIP_I32);
    a.codes = (*codes)->u8();
    a.exps = (*exps)->i32();
    k::rms_norm(a, ctx().stream);
}

void HipBackend::rms_norm_backward(const Tensor &h, const Tensor &gamma, const Tensor &grad_out,
                                   const Tensor *grad_sum, float eps, TensorNode *grad_h,
                                   TensorNode *grad_gamma) {
    need_dtype(h, CLOVE_HIP_F32, "h");
    k::RmsNormGradArgs a{};
    size_t cols;
    rows_cols(h, "h", &a.rows, &cols);
    same_shape(grad_out, h, "grad_out");
    if (grad_sum) same_shape(*grad_sum, h, "grad_sum");
    gamma_rule(gamma, cols, eps);
    a.h = h.f32();
    a.gamma = gamma.f32();
    a.grad_out = grad_out.f32();
    a.grad_sum = grad_sum ? grad_sum->f32() : nullptr;
    a.cols = (int)cols;
    a.eps = eps;
    const int cus = ctx().num_cus;
    hipStream_t s = ctx().stream;
    if (grad_h) {
        *grad_h = new_tensor(h.shape, CLOVE_HIP_F32);
        a.grad_h = (*grad_h)->f32();
    }
    TensorNode part, stats;
    if (grad_gamma) {
        *grad_gamma = new_tensor(gamma.shape, CLOVE_HIP_F32);
        a.grad_gamma = (*grad_gamma)->f32();
        if (a.rows == 0 && cols) k::fill_uniform(a.grad_gamma, cols, 0, 0.0f, 0.0f, s);
        if (const size_t n = k::rms_norm_grad_floats(a.rows, a.cols, cus)) {
            part = new_tensor({n}, CLOVE_HIP_F32);
            a.part = part->f32();
        }
    }
    if (a.rows == 0 || cols == 0) return;
    if (const size_t n = k::rms_norm_grad_stats(a.rows, a.cols)) {
        stats = new_tensor({2 * n}, CLOVE_HIP_F32);
        a.stats = static_cast<double *>(stats->data);
    }
    k::rms_norm_grad(a, cus, s);
}

void HipBackend::quantize_e4m3(const Tensor &x, int block_rows, TensorNode *codes,
                               TensorNode *exps, TensorNode *codes_t, TensorNode *exps_t) {
    need_dtype(x, CLOVE_HIP_F32, "x");
    CLOVE_REQUIRE(block_rows == 1 || block_rows == 128, CLOVE_HIP_ERR_INVALID,
                  "block_rows must be 1 or 128, got " + std::to_string(block_rows));
    k::Quant8Args a{};
    rows_cols(x, "x", &a.rows, &a.cols);
    const size_t kb = blocks_of(a.cols), rb = blocks_of(a.rows);
    if (codes) {
        *codes = new_tensor(with_last(x, kb * 128), CLOVE_HIP_E4M3);
        *exps = new_tensor(block_rows == 1 ? with_last(x, kb) : std::vector<size_t>{rb, kb},
                           CLOVE_HIP_I32);
        a.codes = (*codes)->u8();
        a.exps = (*exps)->i32();
    }
    if (codes_t) {
        *codes_t = new_tensor({a.cols, rb * 128}, CLOVE_HIP_E4M3);
        *exps_t = new_tensor({block_rows == 1 ? a.cols : kb, rb}, CLOVE_HIP_I32);
        a.codes_t = (*codes_t)->u8();
        a.exps_t = (*exps_t)->i32();
    }
    a.x = x.f32();
    a.block_rows = block_rows;
    k::quantize8(a, ctx().stream);
}

TensorNode HipBackend::matmul_e4m3(const Tensor &a, const Tensor &a_exps, const Tensor &b,
                                   const Tensor &b_exps, const Tensor *bias) {
    size_t m, n, ka, kb;
    k::Gemm8Args g{};
    operand_rule(a, a_exps, "a", &m, &ka, &g.a_tiles);
    operand_rule(b, b_exps, "b", &n, &kb, &g.b_tiles);
    CLOVE_REQUIRE(ka == kb, CLOVE_HIP_ERR_SHAPE,
                  "matmul_e4m3: the last dimensions differ, a " + shape_str(a.shape) + " b " +
                      shape_str(b.shape));
    if (bias) {
        need_dtype(*bias, CLOVE_HIP_F32, "bias");
        CLOVE_REQUIRE(bias->numel == n, CLOVE_HIP_ERR_SHAPE,
                      "bias must hold " + std::to_string(n) + " elements, got " +
                          shape_str(bias->shape));
    }
    // (a grid holds 2^32 threads: 2^22 tiles of 64 x 64 are 2^30, larger ones fewer, and 64
    // rows or less in the streaming kernel 2^31; tiles are counted in 31 bits)
    CLOVE_REQUIRE(((m + 63) / 64) * ((n + 63) / 64) < (size_t(1) << 22), CLOVE_HIP_ERR_SHAPE,
                  "matmul_e4m3: the result has 2^22 tiles of 64 x 64 or more");
    TensorNode out = new_tensor(with_last(a, n), CLOVE_HIP_F32);
    g.a = a.u8();
    g.b = b.u8();
    g.a_exps = a_exps.i32();
    g.b_exps = b_exps.i32();
    g.bias = bias ? bias->f32() : nullptr;
    g.out = out->f32();
    g.m = (int)m;
    g.n = (int)n;
    g.blocks = (int)ka;
    const int cus = ctx().num_cus;
    const k::Gemm8Plan plan = k::gemm8_plan(g, cus);
    TensorNode ws;
    if (const size_t floats = k::gemm8_workspace(g, plan)) {
        ws = new_tensor({floats}, CLOVE_HIP_F32);
        g.ws = ws->f32();
    }
    k::gemm8(g, plan, cus, ctx().stream);
    return out;
}

}  // namespace clove
