"""GPU: linear layers in 8 bits and the root-mean-square norm against their
definitions in numpy (linear8_ref): the norm in 32 and 8 bits and its gradient, the
quantiser both ways round, the product, and a run of them together as a layer is
trained and served.

Codes and exponents are determined to the bit and compared exactly; the rest within
the bounds that linear8_ref derives from the roundings.
"""
import ctypes as C

import numpy as np
import pytest

import linear8_ref as ref
from conftest import rng

pytestmark = pytest.mark.gpu


def within(got, want, tol, what=""):
    err = np.abs(np.asarray(got, np.float64) - want)
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {bad.sum()} of {err.size} out of tolerance, worst "
                           f"{(err / tol)[bad].max():.2f} times it, max abs err {err.max():.3e}")


def states(g, *shape):
    """Rows of very different size with a few strong channels."""
    x = g.standard_normal(shape) * 2.0 ** g.integers(-6, 7, shape[:-1] + (1,))
    x[..., 3::17] *= 20
    return x.astype(np.float32)


def off4(hip, a):
    """The same values four bytes off a 16-byte boundary; returns what must live."""
    room = hip.empty((a.size + 1,))
    room.write(1, a)
    return room, hip.wrap(room.device_ptr + 4, a.shape)


# ---- the quantiser -----------------------------------------------------------

def check_quantised(got, x, block_rows):
    codes, exps = ref.quantize(x, block_rows)
    np.testing.assert_array_equal(got[1].numpy().reshape(exps.shape), exps)
    ref.same_codes(got[0].numpy().reshape(codes.shape), codes)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 5), (2, 127), (127, 129), (128, 128),
                                       (129, 256), (300, 1000), (1000, 300), (257, 4099),
                                       (4099, 130), (16, 16384)])
def test_quantize(hip, rows, cols, block_rows):
    x = states(rng(rows * 31 + cols), rows, cols)
    t = hip.tensor(x)
    both = hip.quantize_e4m3(t, block_rows, True, True)
    check_quantised(both[:2], x, block_rows)
    check_quantised(both[2:], x.T, block_rows)
    for one, pair in ((hip.quantize_e4m3(t, block_rows), both[:2]),
                      (hip.quantize_e4m3(t, block_rows, False, True), both[2:])):
        for a, b in zip(one, pair):
            np.testing.assert_array_equal(a.numpy(), b.numpy())
    room, moved = off4(hip, x)
    for a, b in zip(hip.quantize_e4m3(moved, block_rows, True, True), both):
        np.testing.assert_array_equal(a.numpy(), b.numpy())


def test_quantize_borders_and_extremes(hip):
    """Maxima at and next to 448 * 2^e, ties between codes, zero blocks, subnormal
    and largest values, negative zeros."""
    x = np.zeros((40, 256), np.float32)
    for i, e in enumerate((-120, -100, -99, -30, 0, 1, 100, 118)):
        top = np.float32(448 * 2.0 ** e)
        x[4 * i, 7], x[4 * i + 1, 7] = top, np.nextafter(top, np.float32(np.inf))
        x[4 * i + 2, 7] = np.nextafter(top, np.float32(0))
        # halves between neighbouring codes, subnormal ones among them
        t = (ref.VALUES[:126] + ref.VALUES[1:127]) / 2 * 2.0 ** e
        x[4 * i + 3, :126], x[4 * i + 3, 127] = t, top
    x[32, :5] = 1e-45, -1e-40, 0.0, -0.0, 1e-38
    x[33, :2] = np.finfo(np.float32).max, -np.finfo(np.float32).max
    x[34, 130] = -1.0
    for block_rows in (1, 128):
        for y in (x, np.ascontiguousarray(x.T)):
            got = hip.quantize_e4m3(hip.tensor(y), block_rows, True, True)
            check_quantised(got[:2], y, block_rows)
            check_quantised(got[2:], y.T, block_rows)


def test_quantize_what_is_not_finite(hip):
    g = rng(5)
    x = states(g, 140, 300)
    x[3, 7], x[3, 8], x[5, 200], x[139, 299] = np.nan, np.inf, -np.inf, np.nan
    x[7] = np.nan
    for block_rows in (1, 128):
        got = hip.quantize_e4m3(hip.tensor(x), block_rows, True, True)
        check_quantised(got[:2], x, block_rows)
        check_quantised(got[2:], x.T, block_rows)


def test_quantize_keeps_leading_dimensions(hip):
    x = states(rng(6), 2, 3, 200)
    c, e, ct, et = hip.quantize_e4m3(hip.tensor(x), 1, True, True)
    assert c.shape == (2, 3, 256) and e.shape == (2, 3, 2)
    assert ct.shape == (200, 128) and et.shape == (200, 1)
    check_quantised((c, e), x.reshape(6, 200), 1)
    c, e, ct, et = hip.quantize_e4m3(hip.tensor(x), 128, True, True)
    assert c.shape == (2, 3, 256) and e.shape == (1, 2) and et.shape == (2, 1)


# ---- the norm ----------------------------------------------------------------

SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 128), (9, 130), (4, 256), (33, 500), (7, 513), (6, 1000),
          (5, 1024), (4, 1025), (3, 2049), (8, 4096), (3, 4099), (2, 8192), (2, 8196), (3, 16384),
          (2, 16385), (2, 40000), (300, 96)]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_rms_norm(hip, rows, cols, residual):
    g = rng(rows * 7 + cols)
    x = states(g, rows, cols)
    res = states(g, rows, cols) if residual else None
    gamma = g.uniform(-1.5, 1.5, cols).astype(np.float32)
    want, h = ref.rms_norm(x, gamma, res)

    def run(put):
        keep = [put(v) for v in (x, gamma) + ((res,) if residual else ())]
        t = [k[1] for k in keep]
        t += [None] * (3 - len(t))
        out, q = hip.rms_norm(*t), hip.rms_norm_e4m3(*t)
        if residual:
            out, total = out
            for s in (total, q[2]):
                np.testing.assert_array_equal(s.numpy(), h)
        o = out.numpy()
        within(o, want, ref.rms_norm_bound(want))
        codes, exps = ref.quantize(o)  # bit for bit those of the 32-bit norm
        np.testing.assert_array_equal(q[1].numpy(), exps)
        ref.same_codes(q[0].numpy(), codes)
        return o, q[0].numpy()

    first = run(lambda v: (None, hip.tensor(v)))
    for a, b in zip(first, run(lambda v: off4(hip, v))):
        np.testing.assert_array_equal(a, b)


def test_rms_norm_extremes(hip):
    """Rows whose squares leave f32's range, zero rows, eps 0 and large, and rows
    that are not finite, which stay apart from their neighbours."""
    g = rng(11)
    x = np.stack([g.standard_normal(300) * s for s in (1e30, 1e-30, 1e-42, 0.0, 1.0, 1.0, 1.0)])
    x = x.astype(np.float32)
    x[5, 17], x[6, 3] = np.inf, np.nan
    gamma = g.uniform(0.5, 2, 300).astype(np.float32)
    for eps in (1e-5, 0.0, 100.0):
        o = hip.rms_norm(hip.tensor(x), hip.tensor(gamma), eps=eps).numpy()
        with np.errstate(all="ignore"):
            want, _ = ref.rms_norm(x, gamma, eps=eps)
        good = [0, 1, 2, 4] + ([3] if eps else [])
        within(o[good], want[good], ref.rms_norm_bound(want[good]))
        assert np.isnan(o[6]).all() and np.isnan(o[5, 17]) and not o[5, :17].any()
        q, e = hip.rms_norm_e4m3(hip.tensor(x), hip.tensor(gamma), eps=eps)
        codes, exps = ref.quantize(o)
        np.testing.assert_array_equal(e.numpy(), exps)
        ref.same_codes(q.numpy(), codes)


@pytest.mark.parametrize("stream", [False, True])
@pytest.mark.parametrize("rows,cols", SHAPES + [(700, 64), (3000, 33), (1100, 1028), (600, 4100),
                                                (1030, 9000), (20000, 33), (9000, 130),
                                                (5000, 513), (5000, 700), (1000, 3001),
                                                (64, 100), (65, 100), (17, 800), (2, 3000),
                                                (4100, 2052)])
def test_rms_norm_backward(hip, rows, cols, stream):
    g = rng(rows * 13 + cols)
    h = states(g, rows, cols)
    gy = (g.standard_normal((rows, cols)) * 1e-3).astype(np.float32)
    gs = (g.standard_normal((rows, cols)) * 1e-3).astype(np.float32) if stream else None
    gamma = g.uniform(0.5, 1.5, cols).astype(np.float32)
    (dh, th), (dg, tg) = ref.rms_norm_backward(h, gamma, gy, gs)

    def run(put):
        keep = [put(v) for v in (h, gamma, gy) + ((gs,) if stream else ())]
        a, b = hip.rms_norm_backward(*[k[1] for k in keep])
        within(a.numpy(), dh, th, "grad_h")
        within(b.numpy(), dg, tg, "grad_gamma")
        return a.numpy(), b.numpy()

    first = run(lambda v: (None, hip.tensor(v)))
    for other in (run(lambda v: (None, hip.tensor(v))), run(lambda v: off4(hip, v))):
        for a, b in zip(first, other):  # sums in a fixed order
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("cols", [33, 200, 300, 700, 1500, 2100, 5000, 9000])
def test_rms_norm_backward_extremes(hip, cols):
    """Rows whose squares leave f32's range, a zero row, eps 0 and large, and grad_out
    times gamma past f32's range and under it, where r brings the gradient back."""
    g = rng(23 + cols)
    sizes = np.array([1e30, 1e25, 1e-30, 1e-42, 1.0, 0.0])[:, None]
    h = (g.standard_normal((6, cols)) * sizes).astype(np.float32)
    for size in (1e10, 1.0, 1e-10):
        gamma = (g.uniform(0.5, 2, cols) * size).astype(np.float32)
        # r times these is near 1 in the first rows, which eps does not reach
        gy = (g.standard_normal((6, cols)) * [[1e30], [1e20], [1e-32], [1e-35], [1e-3], [1e-3]]
              ).astype(np.float32)
        for eps in (1e-5, 0.0, 100.0):
            good = slice(0, 5 if eps == 0 else 6)
            args = h[good], gamma, gy[good]
            (dh, th), (dg, tg) = ref.rms_norm_backward(*args, eps=eps)
            a, b = (t.numpy() for t in hip.rms_norm_backward(*map(hip.tensor, args), eps=eps))
            within(a, dh, th, f"grad_h, gamma {size}, eps {eps}")
            within(b, dg, tg, f"grad_gamma, gamma {size}, eps {eps}")


def test_rms_norm_backward_keeps_what_is_not_finite_in_its_row(hip):
    g = rng(24)
    for rows, cols in ((9, 300), (900, 130), (40, 2100), (9, 9000)):
        h, gy = (g.standard_normal((rows, cols)).astype(np.float32) for _ in range(2))
        gamma = g.uniform(0.5, 2, cols).astype(np.float32)
        h[2, 7], h[5, cols - 1], gy[7, 3] = np.nan, np.inf, np.nan
        bad = [2, 5, 7]
        a, b = (t.numpy() for t in hip.rms_norm_backward(*map(hip.tensor, (h, gamma, gy))))
        assert np.isnan(a[bad]).all() and np.isnan(b[[3, cols - 1]]).all() and np.isnan(b).all()
        good = np.setdiff1d(np.arange(rows), bad)
        (dh, th), _ = ref.rms_norm_backward(h[good], gamma, gy[good])
        within(a[good], dh, th)


def test_rms_norm_backward_against_differences(hip):
    """The gradients are those of the forward pass: central differences of it, in
    32 bits, whose error is the outputs' rounding over the step."""
    g = rng(21)
    h, gy = (g.standard_normal((4, 40)).astype(np.float32) for _ in range(2))
    gamma = g.uniform(0.5, 1.5, 40).astype(np.float32)
    dh, dg = (v.numpy() for v in hip.rms_norm_backward(*map(hip.tensor, (h, gamma, gy))))
    d = np.float32(2.0 ** -7)

    def loss(h, gamma):
        return (hip.rms_norm(hip.tensor(h), hip.tensor(gamma)).numpy().astype(np.float64)
                * gy).sum()

    # the rounding of 160 outputs of at most 8 times gy, over 2 d; and the third
    # derivative's share, d^2 / 6 of some 10 times the loss's scale
    size = np.abs(gy).sum()
    tol = size * 8 * ref.U / (2 * d) + d * d / 6 * 10 * np.abs(gy).max() * 8
    for i in range(0, 160, 7):
        e = np.zeros_like(h)
        e.flat[i] = d
        assert abs((loss(h + e, gamma) - loss(h - e, gamma)) / (2 * d) - dh.flat[i]) <= tol
    for i in range(0, 40, 3):
        e = np.zeros_like(gamma)
        e[i] = d
        assert abs((loss(h, gamma + e) - loss(h, gamma - e)) / (2 * d) - dg[i]) <= tol


# every class of columns, a workgroup walking its rows in turns: an odd and an even number
# of them, the last one not full
@pytest.mark.parametrize("rows,cols", [(60001, 33), (17000, 128), (20001, 130), (9000, 256),
                                       (5000, 400), (7001, 512), (5000, 700), (4100, 1024),
                                       (2000, 1500), (1030, 2048), (1001, 2049), (3000, 3001),
                                       (4095, 2052), (5000, 2100), (1030, 5000), (700, 8192),
                                       (700, 9000), (2000, 8196), (65, 100), (64, 100), (3, 1500),
                                       (2, 20000)])
@pytest.mark.parametrize("wanted", ["both", "gamma"])
def test_rms_norm_backward_of_whole_numbers_is_exact(hip, rows, cols, wanted):
    """With h of +-1 and eps 0 every row's root mean square is 1 and grad_gamma a sum of
    whole numbers below 2^24 in magnitude, of which none is 0: a row lost or taken
    twice shows."""
    g = rng(rows + cols)
    h = g.choice(np.float32([-1, 1]), (rows, cols))
    gy = (g.integers(1, 9, (rows, cols)) * g.choice([-1, 1], (rows, cols))).astype(np.float32)
    assert 8 * rows < 1 << 24
    gamma = np.ones(cols, np.float32)
    t = [hip.tensor(v) for v in (h, gamma, gy)]
    if wanted == "both":
        a, b = (v.numpy() for v in hip.rms_norm_backward(*t, eps=0.0))
        # a row's sum of whole numbers is exact too: cols divides it with one rounding in 64
        # bits, and the difference is rounded to 32
        want = gy - h * ((gy * h).sum(1, keepdims=True, dtype=np.float64) / cols)
        within(a, want, ref.U * 1.0001 * np.abs(want) + 2.0 ** -48)
    else:
        out = C.c_void_p()
        assert hip.lib().clove_hip_rms_norm_backward(*[v.handle for v in t], None, 0.0, None,
                                                     C.byref(out)) == hip.OK
        b = hip.Tensor(out.value).numpy()
    np.testing.assert_array_equal(b, (gy * h).sum(0, dtype=np.float64))


def test_rms_norm_backward_skips_what_is_not_wanted(hip):
    g = rng(22)
    h, gamma, gy = (hip.tensor(g.standard_normal(s).astype(np.float32))
                    for s in ((37, 130), (130,), (37, 130)))
    both = [t.numpy() for t in hip.rms_norm_backward(h, gamma, gy)]
    lib = hip.lib()
    for i in range(2):
        out = C.c_void_p()
        p = [None, None]
        p[i] = C.byref(out)
        assert lib.clove_hip_rms_norm_backward(h.handle, gamma.handle, gy.handle, None, 1e-5,
                                               *p) == hip.OK
        np.testing.assert_array_equal(hip.Tensor(out.value).numpy(), both[i])
    out = C.c_void_p()
    res = hip.tensor(np.ones((37, 130), np.float32))
    p = lib.clove_hip_rms_norm(h.handle, res.handle, gamma.handle, 1e-5, None)  # no sum wanted
    np.testing.assert_array_equal(hip.Tensor(p).numpy(), hip.rms_norm(h, gamma, res)[0].numpy())


# ---- the product ---------------------------------------------------------------

def operands(g, m, n, k, a_tiles, b_tiles):
    a = ref.quantize(states(g, m, k), 128 if a_tiles else 1)
    b = ref.quantize((g.standard_normal((n, k)) * 2.0 ** g.integers(-3, 4, (n, 1))
                      ).astype(np.float32), 128 if b_tiles else 1)
    return a + b


def put(hip, a, ea, b, eb):
    return [hip.tensor(a, np.uint8), hip.tensor(ea), hip.tensor(b, np.uint8), hip.tensor(eb)]


# each side of the row counts and sizes at which the kernels change
PRODUCTS = [(1, 1, 1), (1, 16, 128), (1, 17, 129), (2, 300, 1000), (5, 4096, 512), (16, 100, 4096),
            (17, 64, 640), (32, 1000, 784), (33, 130, 300), (64, 256, 2048), (65, 64, 128),
            (65, 130, 257), (100, 10, 784), (128, 128, 384), (129, 257, 128), (200, 1000, 100),
            (257, 129, 1500), (300, 60, 4100), (512, 512, 1024), (777, 768, 768), (70, 5000, 256),
            (5000, 70, 256), (2100, 2100, 140), (130, 70, 16400)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("a_tiles,b_tiles", [(False, True), (False, False), (True, False)])
def test_matmul(hip, m, n, k, a_tiles, b_tiles):
    g = rng(m * 7 + n * 3 + k)
    ops = operands(g, m, n, k, a_tiles, b_tiles)
    bias = g.standard_normal(n).astype(np.float32) if (m + n) % 2 else None
    t = put(hip, *ops) + [None if bias is None else hip.tensor(bias)]
    got = hip.matmul_e4m3(*t)
    assert got.shape == (m, n)
    want, tol = ref.matmul(*ops, bias)
    within(got.numpy(), want, tol)
    np.testing.assert_array_equal(hip.matmul_e4m3(*t).numpy(), got.numpy())


# few rows against a long b, and results of many tiles, past every tile's edge
@pytest.mark.parametrize("m,n,k", [(1, 8200, 300), (32, 8225, 1200), (64, 1000, 1500),
                                   (48, 5000, 2100), (61, 16380, 700), (1930, 3970, 390),
                                   (1, 37, 9000), (32, 1001, 3000), (19, 4000, 8400),
                                   (3, 3900, 1000),
                                   (3841, 4000, 390)])
@pytest.mark.parametrize("a_tiles", [False, True])
def test_matmul_of_many(hip, m, n, k, a_tiles):
    g = rng(m + n * 5 + k)
    ops = operands(g, m, n, k, a_tiles, not a_tiles)
    bias = g.standard_normal(n).astype(np.float32) if a_tiles else None
    t = put(hip, *ops) + [None if bias is None else hip.tensor(bias)]
    want, tol = ref.matmul(*ops, bias)
    within(hip.matmul_e4m3(*t).numpy(), want, tol)


@pytest.mark.parametrize("m,n,k", [(1, 200, 700), (40, 100, 1300), (200, 300, 900),
                                   (600, 2000, 260), (130, 140, 9000)])
def test_matmul_of_small_whole_numbers_is_exact(hip, m, n, k):
    """Sums below 2^24 of whole numbers have one right answer in 32 bits."""
    g = rng(m + n + k)
    a, b = (g.integers(-8, 9, s).astype(np.float32) for s in ((m, k), (n, k)))
    bias = g.integers(-50, 50, n).astype(np.float32)
    qa, qb = ref.quantize(a), ref.quantize(b, 128)
    np.testing.assert_array_equal(ref.values(*qa)[:, :k], a)
    got = hip.matmul_e4m3(*put(hip, *qa, *qb), hip.tensor(bias)).numpy()
    np.testing.assert_array_equal(got, a.astype(np.float64) @ b.T.astype(np.float64) + bias)


# a size for every kernel, whole and cut along k, with ragged edges (which one takes which
# is checked on the CPU)
FORMS = [(32, 1001, 2900), (3, 3900, 1000), (3, 5000, 1000), (30, 8225, 1200), (40, 5000, 2100),
         (61, 16380, 700), (65, 130, 257), (70, 60, 4100), (3654, 133, 2435), (300, 700, 400),
         (70, 9596, 4290), (66, 50, 977), (1930, 3970, 390), (1880, 1608, 21156),
         (849, 1672, 15122), (840, 853, 31240), (3841, 4001, 390), (1927, 4065, 13493),
         (1967, 1928, 20452), (997, 1980, 25421)]


@pytest.mark.parametrize("m,n,k", FORMS)
def test_matmul_of_every_form_is_exact(hip, m, n, k):
    """Whole numbers of up to 8 with exponents of 0 and 1: sums below 2^24, exact in 32
    bits in any order, so a block lost, taken twice or scaled by another's exponent
    shows; a bias on top."""
    g = rng(m + n + k)
    code = ref.encode(np.arange(9, dtype=np.float32))

    def operand(rows, tiles):
        x = g.integers(0, 9, (rows, ref.up(k)), np.uint8)
        x[:, k:] = 0
        minus = g.integers(0, 2, x.shape, np.uint8)
        e = g.integers(0, 2, (-(-rows // 128) if tiles else rows, ref.up(k) // 128)).astype(np.int32)
        scale = np.repeat(e, 128, 0)[:rows] if tiles else e
        v = np.where(minus, -x.astype(np.float32), x).reshape(rows, -1, 128)
        v *= np.exp2(scale.astype(np.float32))[..., None]
        return code[x] | minus << 7, e, v.reshape(rows, -1)

    (a, ea, va), (b, eb, vb) = operand(m, False), operand(n, True)
    assert 256 * k < 1 << 24
    bias = g.integers(-50, 50, n).astype(np.float32)
    got = hip.matmul_e4m3(*put(hip, a, ea, b, eb), hip.tensor(bias)).numpy()
    np.testing.assert_array_equal(got, va @ vb.T + bias)


@pytest.mark.parametrize("m,n,k", [(8, 512, 1024), (512, 512, 1024), (300, 600, 4096)])
def test_matmul_sums_in_32_bits(hip, m, n, k):
    """K additions, each off by at most a step of a partial sum no larger than the
    result on the average: in the 2-norm sqrt(K) of them for terms of either sign.
    Positive terms all add up; they join the sum eight at a time at least (a matrix
    instruction takes sixteen), and the sum is half the result on the average."""
    g = rng(k)
    for positive in (False, True):
        a, b = (g.standard_normal(s).astype(np.float32) for s in ((m, k), (n, k)))
        if positive:
            a, b = np.exp(2 * a), np.exp(2 * b)
        ops = ref.quantize(a) + ref.quantize(b, 128)
        want, _ = ref.matmul(*ops)
        got = hip.matmul_e4m3(*put(hip, *ops)).numpy()
        rel = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert rel <= (2 * ref.U * k / 16 if positive else 2 * ref.U * np.sqrt(k)), rel


def test_matmul_extreme_exponents(hip):
    """Scales at both ends of the range, in every combination; products under
    f32's range vanish and those past it are infinite, as in f32."""
    g = rng(31)
    for m, n in ((20, 150), (100, 150)):
        for ea in (-100, -20, 119):
            for eb in (-100, 0, 119):
                a, b = ((g.standard_normal((r, 256)) * 40).astype(np.float32) for r in (m, n))
                qa, qb = ref.quantize(a), ref.quantize(b)
                qa, qb = (qa[0], np.full_like(qa[1], ea)), (qb[0], np.full_like(qb[1], eb))
                got = hip.matmul_e4m3(*put(hip, *qa, *qb)).numpy()
                want, tol = ref.matmul(*qa, *qb)
                if ea + eb > 100:
                    assert not np.isfinite(got).any()
                else:
                    within(got, want, tol)


@pytest.mark.parametrize("m,n", [(4, 40), (80, 200)])
@pytest.mark.parametrize("exps", [(-70, -66), (-70, -76), (-100, -52), (-59, -100)])
def test_matmul_keeps_subnormal_products(hip, m, n, exps):
    """Products of 448 * 448 * 2^(ea + eb), whole multiples of 2^-149, and their sums."""
    for count in (1, 100):
        x = [np.zeros((r, 256), np.float32) for r in (m, n)]
        for v in x:
            v[:, :count] = 448
        a, b = (ref.quantize(v)[0] for v in x)
        ea, eb = (np.full((r, 2), e, np.int32) for r, e in zip((m, n), exps))
        got = hip.matmul_e4m3(*put(hip, a, ea, b, eb)).numpy()
        want = count * 448.0 * 448.0 * 2.0 ** sum(exps)
        np.testing.assert_array_equal(got, np.full((m, n), want))


def test_matmul_carries_nan_to_its_row_and_column_alone(hip):
    g = rng(32)
    for m, n in ((10, 100), (150, 200)):
        x, w = states(g, m, 300), states(g, n, 300)
        x[3, 5], w[17, 299] = np.inf, np.nan
        t = hip.quantize_e4m3(hip.tensor(x)) + hip.quantize_e4m3(hip.tensor(w))
        got = hip.matmul_e4m3(*t).numpy()
        bad = np.zeros((m, n), bool)
        bad[3], bad[:, 17] = True, True
        np.testing.assert_array_equal(np.isnan(got), bad)
        x[3, 5], w[17, 299] = 0, 0
        want, tol = ref.matmul(*ref.quantize(x), *ref.quantize(w))
        within(got[~bad], want[~bad], tol[~bad])


def test_matmul_keeps_leading_dimensions(hip):
    g = rng(33)
    x, w = states(g, 2, 5, 200), states(g, 30, 200)
    out = hip.matmul_e4m3(*hip.quantize_e4m3(hip.tensor(x)),
                          *hip.quantize_e4m3(hip.tensor(w), 128))
    assert out.shape == (2, 5, 30)
    want, tol = ref.matmul(*ref.quantize(x.reshape(10, 200)), *ref.quantize(w, 128))
    within(out.numpy().reshape(10, 30), want, tol)


# ---- empty calls and refusals ----------------------------------------------------

def test_empty_calls(hip):
    gamma = hip.tensor(np.ones(5, np.float32))
    x = hip.empty((0, 5))
    assert hip.rms_norm(x, gamma).shape == (0, 5)
    q = hip.rms_norm_e4m3(x, gamma, x)
    assert [t.shape for t in q] == [(0, 128), (0, 1), (0, 5)]
    dh, dg = hip.rms_norm_backward(x, gamma, x)
    assert dh.shape == (0, 5)
    np.testing.assert_array_equal(dg.numpy(), np.zeros(5, np.float32))
    none = hip.empty((0,))
    assert hip.rms_norm(hip.empty((3, 0)), none).shape == (3, 0)
    assert hip.rms_norm_backward(hip.empty((3, 0)), none, hip.empty((3, 0)))[1].shape == (0,)
    c, e, ct, et = hip.quantize_e4m3(x, 1, True, True)
    assert [t.shape for t in (c, e, ct, et)] == [(0, 128), (0, 1), (5, 0), (5, 0)]
    w = hip.quantize_e4m3(hip.tensor(np.ones((7, 5), np.float32)), 128)
    assert hip.matmul_e4m3(c, e, *w).shape == (0, 7)
    assert hip.matmul_e4m3(*w, c, e).shape == (7, 0)
    # nothing along k: zeros, or the bias
    k0 = hip.quantize_e4m3(hip.empty((3, 0)))
    bias = np.arange(3, dtype=np.float32)
    np.testing.assert_array_equal(hip.matmul_e4m3(*k0, *k0).numpy(), np.zeros((3, 3)))
    np.testing.assert_array_equal(hip.matmul_e4m3(*k0, *k0, hip.tensor(bias)).numpy(),
                                  np.tile(bias, (3, 1)))
    big = hip.quantize_e4m3(hip.empty((70, 0)))
    np.testing.assert_array_equal(hip.matmul_e4m3(*big, *k0, hip.tensor(bias)).numpy(),
                                  np.tile(bias, (70, 1)))


def test_refusals(hip):
    def refused(code, f, *args, **kw):
        with pytest.raises(hip.CloveError) as e:
            f(*args, **kw)
        assert e.value.code == code, e.value

    x, gamma = hip.tensor(np.ones((3, 8), np.float32)), hip.tensor(np.ones(8, np.float32))
    ints = hip.tensor(np.ones((3, 8), np.int32))
    for f in (hip.rms_norm, hip.rms_norm_e4m3):
        refused(hip.ERR_INVALID, f, ints, gamma)
        refused(hip.ERR_SHAPE, f, x, hip.tensor(np.ones(7, np.float32)))
        refused(hip.ERR_SHAPE, f, x, gamma, hip.tensor(np.ones((2, 8), np.float32)))
        refused(hip.ERR_INVALID, f, x, gamma, ints)
        for eps in (-1e-5, float("nan"), float("inf")):
            refused(hip.ERR_INVALID, f, x, gamma, eps=eps)
    out = C.c_void_p()
    assert not hip.lib().clove_hip_rms_norm(x.handle, None, gamma.handle, 1e-5, C.byref(out))
    assert "residual" in hip.lib().clove_hip_last_error().decode() and out.value is None
    refused(hip.ERR_SHAPE, hip.rms_norm_backward, x, gamma, hip.tensor(np.ones((8, 3), np.float32)))
    refused(hip.ERR_SHAPE, hip.rms_norm_backward, x, gamma, x, gamma)
    refused(hip.ERR_INVALID, hip.rms_norm_backward, x, gamma, ints)
    refused(hip.ERR_INVALID, hip.quantize_e4m3, ints)
    for br in (0, 2, 64, 129, -1):
        refused(hip.ERR_INVALID, hip.quantize_e4m3, x, br)
    a = hip.quantize_e4m3(hip.tensor(np.ones((200, 300), np.float32)))
    b = hip.quantize_e4m3(hip.tensor(np.ones((50, 300), np.float32)), 128)
    c = hip.quantize_e4m3(hip.tensor(np.ones((50, 100), np.float32)), 128)
    refused(hip.ERR_SHAPE, hip.matmul_e4m3, *a, *c)
    refused(hip.ERR_INVALID, hip.matmul_e4m3, x, a[1], *b)
    refused(hip.ERR_INVALID, hip.matmul_e4m3, a[0], x, *b)
    refused(hip.ERR_SHAPE, hip.matmul_e4m3, a[0], b[1], *b)  # exponents of another matrix
    refused(hip.ERR_SHAPE, hip.matmul_e4m3, *a, *b, gamma)
    refused(hip.ERR_INVALID, hip.matmul_e4m3, *a, *b, hip.tensor(np.ones(50, np.int32)))
    odd = hip.tensor(np.zeros((4, 100), np.uint8), np.uint8)
    refused(hip.ERR_SHAPE, hip.matmul_e4m3, odd, hip.tensor(np.zeros((4, 1), np.int32)), *c)
    room = hip.empty((200 * 384 + 16,), np.uint8)
    moved = hip.wrap(room.device_ptr + 4, (200, 384), np.uint8)
    refused(hip.ERR_INVALID, hip.matmul_e4m3, moved, a[1], *b)


def test_freed_operands_are_refused(hip):
    """Not taken for operands that are left out."""
    ones = hip.tensor(np.ones((3, 8), np.float32))
    gamma = hip.tensor(np.ones(8, np.float32))
    q = hip.quantize_e4m3(ones)
    gone = hip.tensor(np.ones((3, 8), np.float32))
    gone.free()
    for f in (lambda: hip.matmul_e4m3(*q, *q, gone), lambda: hip.rms_norm(ones, gamma, gone),
              lambda: hip.rms_norm_e4m3(ones, gamma, gone),
              lambda: hip.rms_norm_backward(ones, gamma, ones, gone),
              lambda: hip.rms_norm(gone, gamma), lambda: hip.quantize_e4m3(gone)):
        with pytest.raises(hip.CloveError) as e:
            f()
        assert e.value.code == hip.ERR_INVALID


# ---- more workgroups than one launch holds ------------------------------------------

def test_many_rows(hip):
    """Rows past 2^21 workgroups equal the same rows in a call of their own."""
    rows = (1 << 24) + 1000
    x = hip.empty((rows, 3)).fill_normal(1)
    gamma = hip.tensor(np.array([0.5, 1, 2], np.float32))
    out = hip.rms_norm(x, gamma)
    for first in (0, (1 << 24) - 300, rows - 600):
        part = x.read(first * 3, 1800).reshape(600, 3)
        want = hip.rms_norm(hip.tensor(part), gamma).numpy()
        np.testing.assert_array_equal(out.read(first * 3, 1800).reshape(600, 3), want)


def test_many_rows_transposed(hip):
    rows = (1 << 28) + 300
    x = hip.empty((rows, 1)).fill_normal(2)
    codes, exps = hip.quantize_e4m3(x, 1, False, True)
    assert codes.shape == (1, (1 << 28) + 384) and exps.shape == (1, (1 << 21) + 3)
    for first in (0, (1 << 28) - 256, 1 << 28):
        part = x.read(first, min(512, rows - first)).reshape(1, -1)
        c, e = ref.quantize(part)
        np.testing.assert_array_equal(exps.read(first // 128, e.size), e[0])
        ref.same_codes(codes.read(first, c.size), c[0])


def test_a_row_of_many_columns(hip):
    cols = (1 << 27) + 70
    h = hip.empty((1, cols)).fill_uniform(3, 1.0, 1.0)
    gy, gamma = hip.empty((1, cols)).fill_normal(4), hip.empty((cols,)).fill_normal(5)
    r = np.float32(1 / np.sqrt(1 + np.float64(np.float32(1e-5))))
    dg = hip.rms_norm_backward(h, gamma, gy)[1]
    out = hip.rms_norm(h, gamma)
    for first in (0, cols - 200):
        np.testing.assert_array_equal(dg.read(first, 200), gy.read(first, 200) * r)
        want = gamma.read(first, 200) / np.sqrt(1 + np.float64(np.float32(1e-5)))
        within(out.read(first, 200), want, ref.rms_norm_bound(want))


# ---- together --------------------------------------------------------------------

def test_a_layer_trained_and_served(hip):
    """norm -> 8-bit product -> loss and back: every gradient against 64 bits on the
    same quantised operands, AdamW's step, and the updated weights serving single
    tokens and a prompt alike."""
    g = rng(41)
    T, K, N = 150, 200, 330
    x, res = states(g, T, K), states(g, T, K)
    gamma = g.uniform(0.5, 1.5, K).astype(np.float32)
    w = (g.standard_normal((K, N)) / np.sqrt(K)).astype(np.float32)
    target = g.standard_normal((T, N)).astype(np.float32)
    tw, tgamma = hip.tensor(w), hip.tensor(gamma)
    # forward: w's transposed pair multiplies the rows
    out, h = hip.rms_norm(hip.tensor(x), tgamma, hip.tensor(res))
    qx, ex, qxt, ext = hip.quantize_e4m3(out, 1, True, True)
    qw, ew, qwt, ewt = hip.quantize_e4m3(tw, 128, True, True)
    y = hip.matmul_e4m3(qx, ex, qwt, ewt)
    norm, _ = ref.rms_norm(x, gamma, res)
    pairs = {n: (q.numpy(), e.numpy()) for n, q, e in
             (("x", qx, ex), ("xt", qxt, ext), ("w", qw, ew), ("wt", qwt, ewt))}
    want, tol = ref.matmul(*pairs["x"], *pairs["wt"])
    within(y.numpy(), want, tol, "y")
    # the quantised layer is near the layer: each operand is off by 2^-4 at most
    true = norm @ w.astype(np.float64)
    assert (np.abs(want - true) <= (2.0 ** -3 + 2.0 ** -8) * (np.abs(norm) @ np.abs(w))
            + 2.0 ** -10 * 64 * np.abs(norm).max()).all()
    # backward
    one = hip.tensor(np.ones((1, 1), np.float32))
    gy = hip.mse_backward(y, hip.tensor(target), one)
    qg, eg, qgt, egt = hip.quantize_e4m3(gy, 1, True, True)
    dx = hip.matmul_e4m3(qg, eg, qw, ew)
    dw = hip.matmul_e4m3(qxt, ext, qgt, egt)
    assert dx.shape == (T, K) and dw.shape == (K, N)
    for got, a, b in ((dx, (qg, eg), pairs["w"]), (dw, pairs["xt"], (qgt, egt))):
        ops = [v if isinstance(v, np.ndarray) else v.numpy() for v in (*a, *b)]
        want, tol = ref.matmul(*ops)
        within(got.numpy(), want, tol)
    dh, dgamma = hip.rms_norm_backward(h, tgamma, dx)
    (wh, th), (wg, tg) = ref.rms_norm_backward(x + res, gamma, dx.numpy())
    within(dh.numpy(), wh, th, "grad_h")
    within(dgamma.numpy(), wg, tg, "grad_gamma")
    # the update, and the new weights at work: a row alone and among others
    zeros = [hip.tensor(np.zeros(s, np.float32)) for s in ((K, N), (K, N), (K,), (K,))]
    hip.adamw_step([tw, tgamma], [dw, dgamma], [zeros[0], zeros[2]], [zeros[1], zeros[3]],
                   step=1, loss_scale=1.0)
    assert not np.array_equal(tw.numpy(), w)
    new = hip.quantize_e4m3(tw, 128, False, True)
    rows = hip.rms_norm_e4m3(hip.tensor(x), tgamma, hip.tensor(res))[:2]
    many = hip.matmul_e4m3(*rows, *new).numpy()
    want, tol = ref.matmul(rows[0].numpy(), rows[1].numpy(), new[0].numpy(), new[1].numpy())
    within(many, want, tol)
    for t in (0, 77, 149):
        row = hip.rms_norm_e4m3(hip.tensor(x[t:t + 1]), tgamma, hip.tensor(res[t:t + 1]))[:2]
        single = hip.matmul_e4m3(*row, *new).numpy()
        within(single[0], want[t], tol[t])


def test_on_another_stream(hip):
    """The same calls on the backend's stream and on a caller's."""
    rt = C.CDLL("libamdhip64.so")
    g = rng(42)
    x, w = states(g, 300, 400), states(g, 500, 400)
    gamma = hip.tensor(np.ones(400, np.float32))

    def run():
        tx = hip.tensor(x)
        q = hip.rms_norm_e4m3(tx, gamma)
        y = hip.matmul_e4m3(*q, *hip.quantize_e4m3(hip.tensor(w), 128))
        return [y] + list(hip.rms_norm_backward(tx, gamma, tx))

    here = [t.numpy() for t in run()]
    other = C.c_void_p()
    assert rt.hipStreamCreate(C.byref(other)) == 0
    try:
        assert hip.lib().clove_hip_set_stream(other) == hip.OK
        there = [t.numpy() for t in run()]
    finally:
        assert hip.lib().clove_hip_set_stream(None) == hip.OK
        rt.hipStreamDestroy(other)
    for a, b in zip(here, there):
        np.testing.assert_array_equal(a, b)
