"""Linear layers in 8 bits on the CPU: the reference that the GPU tests compare
with, and the entries' refusal of missing handles and half pairs."""
import ctypes as C

import numpy as np
import pytest

import clove_amd as ca
import linear8_ref as ref
from conftest import rng


def test_reference_exponents():
    for x, e in ((448.0, 0), (448.00003, 1), (224.0, -1), (1.75, -8), (0.0, -100), (1e-38, -100),
                 (448 * 2.0 ** -100, -100), (449 * 2.0 ** -100, -99), (3.4e38, 119)):
        assert ref.exp_of(np.float32(x)) == e, x


def test_reference_codes_are_torchs():
    torch = pytest.importorskip("torch")
    g = rng(1)
    x = (g.standard_normal((5, 300)) * 2.0 ** g.integers(-20, 20, (5, 1))).astype(np.float32)
    codes, exps = ref.quantize(x)
    scale = np.repeat(np.exp2(exps.astype(np.float64)), 128, 1)[:, :300]
    want = torch.from_numpy((x / scale).astype(np.float32)).to(torch.float8_e4m3fn)
    np.testing.assert_array_equal(codes[:, :300], want.view(torch.uint8).numpy())
    assert not codes[:, 300:].any() and codes.shape == (5, 384) and exps.shape == (5, 3)
    got = ref.values(codes, exps)[:, :300]
    assert (np.abs(got - x) <= 2.0 ** -4 * np.abs(x) + 2.0 ** -10 * scale).all()


def test_reference_gradient_against_differences():
    g = rng(2)
    h, gy = (g.standard_normal((3, 7)) for _ in range(2))
    gamma = g.uniform(0.5, 1.5, 7)
    (dh, _), (dg, _) = ref.rms_norm_backward(h, gamma, gy)

    def loss(h, gamma):
        return (ref.rms_norm(h, gamma)[0] * gy).sum()

    d = 1e-6
    for i in np.ndindex(h.shape):
        e = np.zeros_like(h)
        e[i] = d
        np.testing.assert_allclose((loss(h + e, gamma) - loss(h - e, gamma)) / (2 * d), dh[i],
                                   rtol=0, atol=1e-8)
    for i in range(7):
        e = np.zeros(7)
        e[i] = d
        np.testing.assert_allclose((loss(h, gamma + e) - loss(h, gamma - e)) / (2 * d), dg[i],
                                   rtol=0, atol=1e-8)


def test_missing_handles_are_refused():
    lib = ca.lib()
    outs = [C.c_void_p(5) for _ in range(4)]
    p = [C.byref(o) for o in outs]
    assert not lib.clove_hip_rms_norm(None, None, None, 1e-5, p[0])
    assert lib.clove_hip_last_status() == ca.ERR_INVALID
    assert lib.clove_hip_rms_norm_e4m3(None, None, None, 1e-5, p[1], p[2], p[3]) == ca.ERR_INVALID
    assert all(o.value is None for o in outs)  # no stale handle on failure
    assert lib.clove_hip_rms_norm_e4m3(None, None, None, 1e-5, None, None,
                                       p[0]) == ca.ERR_INVALID
    assert "codes or exps" in ca.last_error()
    assert lib.clove_hip_rms_norm_backward(None, None, None, None, 1e-5, p[0],
                                           p[1]) == ca.ERR_INVALID
    assert lib.clove_hip_quantize_e4m3(None, 1, p[0], p[1], None, None) == ca.ERR_INVALID
    for half in ((p[0], None, None, None), (None, None, None, p[1])):
        assert lib.clove_hip_quantize_e4m3(None, 1, *half) == ca.ERR_INVALID
        assert "together" in ca.last_error()
    assert not lib.clove_hip_matmul_e4m3(None, None, None, None, None)
    assert lib.clove_hip_last_status() == ca.ERR_INVALID


class Gemm8Args(C.Structure):  # kernels/launch.hpp
    _fields_ = ([(n, C.c_void_p) for n in ("a", "b", "a_exps", "b_exps", "bias", "out", "ws")]
                + [(n, C.c_int) for n in ("m", "n", "blocks")]
                + [(n, C.c_bool) for n in ("a_tiles", "b_tiles")])


class Gemm8Plan(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("waves", "rows_a", "rows_b", "bm", "bn", "tiles_m",
                                       "tiles_n", "splits", "per_split")]


def test_the_products_tested_reach_every_form():
    """The kernel that a product takes is chosen by price: the sizes of the GPU test have
    to reach each, and each way of tiles that k is cut, whatever the prices become."""
    from test_gpu_linear8 import FORMS

    plan = ca.lib()["_ZN5clove1k10gemm8_planERKNS0_9Gemm8ArgsEi"]
    plan.restype, plan.argtypes = Gemm8Plan, [C.POINTER(Gemm8Args), C.c_int]
    seen = set()
    for m, n, k in FORMS:
        p = plan(C.byref(Gemm8Args(m=m, n=n, blocks=-(-k // 128))), 256)
        if p.waves:
            seen.add(("stream", p.rows_b, p.rows_a, p.waves))
        else:
            blocks = -(-k // 128)
            assert (p.splits - 1) * p.per_split < blocks <= p.splits * p.per_split
            seen.add(("tiles", p.bm, p.bn, "cut" if p.splits > 1 else "whole"))
    assert seen == {("stream", 16, 32, 8), ("stream", 32, 32, 8), ("stream", 32, 32, 4),
                    ("stream", 32, 64, 6), ("stream", 64, 64, 4)} | {
        ("tiles", bm, bn, how) for bm, bn in ((64, 64), (64, 128), (128, 128), (256, 256))
        for how in ("whole", "cut")}
