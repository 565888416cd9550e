"""Linear layers in 8 bits and the root-mean-square norm by their definitions, in
numpy: matrices as e4m3 codes and power-of-two exponents, the norm and its
gradient in 64 bits, and the bounds on what 32-bit arithmetic may be off."""
import numpy as np

from kv8_ref import VALUES, encode

MIN_EXP, MAX_EXP = -100, 119
NAN_CODE = 0x7F
U = 2.0 ** -24  # half a step of f32, relative


def up(n):
    return -(-n // 128) * 128


def exp_of(amax):
    """The smallest e in [MIN_EXP, MAX_EXP] with amax <= 448 * 2^e."""
    m, e = np.frexp(np.asarray(amax, np.float64))  # 448 = 0.875 * 2^9
    e = np.where(amax > 0, e - 9 + (m > 0.875), MIN_EXP)
    return np.clip(e, MIN_EXP, MAX_EXP).astype(np.int32)


def quantize(x, block_rows=1):
    """x f32 [rows, K] as (codes [rows, Kp], exps [ceil(rows / block_rows), Kp / 128])."""
    rows, cols = x.shape
    p = np.zeros((-(-rows // block_rows) * block_rows, up(cols)), np.float32)
    p[:rows, :cols] = x
    finite = np.where(np.isfinite(p), np.abs(p), 0)
    blocks = finite.reshape(-1, block_rows, up(cols) // 128, 128)
    e = exp_of(blocks.max((1, 3), initial=0))
    scale = np.repeat(np.repeat(np.exp2(e.astype(np.float64)), block_rows, 0), 128, 1)
    with np.errstate(invalid="ignore"):
        y = np.clip(np.where(np.isfinite(p), p, 0) / scale, -448, 448)
    codes = encode(y.astype(np.float32))
    codes = np.where(np.isfinite(p), codes, NAN_CODE).astype(np.uint8)
    return codes[:rows], e


def same_codes(got, want):
    """Equal codes, where a NaN is a NaN whatever its sign and zeros are zeros."""
    nan = (want & 0x7F) == NAN_CODE
    zero = (want & 0x7F) == 0
    np.testing.assert_array_equal((got & 0x7F)[nan | zero], want[nan | zero] & 0x7F)
    np.testing.assert_array_equal(np.where(nan | zero, 0, got), np.where(nan | zero, 0, want))


def values(codes, exps):
    """What a matrix in 8 bits stands for, in 64 bits."""
    v = np.where((codes & 0x7F) == NAN_CODE, np.nan, VALUES[np.where(
        (codes & 0x7F) == NAN_CODE, 0, codes)])
    e = np.exp2(exps.astype(np.float64))
    if exps.shape[0] != codes.shape[0]:
        e = np.repeat(e, 128, 0)[:codes.shape[0]]
    return v * np.repeat(e, 128, 1)


def matmul(a, a_exps, b, b_exps, bias=None):
    """(out, bound): sums of exact products in 64 bits, and how far 32-bit sums in
    any order may be off: each of up to K additions by a step (2 U) of its partial
    sum, at most sum |a b|; the bias's addition by half a step."""
    x, y = values(a, a_exps), values(b, b_exps)
    out = x @ y.T
    bound = (x.shape[1] + 16) * 2 * U * (np.abs(x) @ np.abs(y).T) + 2.0 ** -140
    if bias is not None:
        out = out + bias.astype(np.float64)
        bound = bound + 2 * U * np.abs(out)
    return out, bound


def rms_norm(x, gamma, residual=None, eps=1e-5):
    """(out in 64 bits, h f32)."""
    h = x if residual is None else x + residual
    h64 = h.astype(np.float64)
    r = 1 / np.sqrt((h64 * h64).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
    return h64 * r * gamma.astype(np.float64), h


def rms_norm_bound(out):
    """One rounding of what 64-bit arithmetic gives."""
    return U * 1.0001 * np.abs(out) + 2.0 ** -149


def rms_norm_backward(h, gamma, gy, grad_sum=None, eps=1e-5):
    """((grad_h, bound), (grad_gamma, bound)).  grad_out * gamma is rounded once, in
    the elements and in the row's sum; grad_h once at its end.  A column's terms
    take two roundings and their sum up to rows - 1 more, in any order."""
    h, gamma, gy = (v.astype(np.float64) for v in (h, gamma, gy))
    r = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
    g = gy * gamma
    dh = r * (g - h * r * r * (g * h).mean(-1, keepdims=True))
    off = U * r * (np.abs(g) + np.abs(h) * r * r * np.abs(g * h).mean(-1, keepdims=True))
    if grad_sum is not None:
        dh = dh + grad_sum
    terms = gy * h * r
    dg = terms.sum(0)
    n = h.shape[0]
    return ((dh, 1.01 * (off + U * np.abs(dh)) + 2.0 ** -148),
            (dg, (n + 8) * U * np.abs(terms).sum(0) + 2.0 ** -140))
