"""The 8-bit paged cache on the CPU: the reference the GPU tests compare with
against torch's own e4m3, the entries' refusal of missing handles, and the slot
arithmetic that spreads ragged rows over a grid of a size that the host knows."""
import ctypes as C

import numpy as np
import pytest

import clove_amd as ca
import kv8_ref as ref
from conftest import rng


def test_reference_codes_are_e4m3():
    torch = pytest.importorskip("torch")
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(t, ref.VALUES.astype(np.float32))
    g = rng(1)
    y = np.concatenate([g.uniform(-448, 448, 4000), g.standard_normal(4000) * 2.0 ** g.integers(
        -12, 6, 4000), (ref.VALUES[:126] + ref.VALUES[1:127]) / 2]).astype(np.float32)
    want = torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(ref.encode(y), want)


def test_reference_exponents():
    for x, e in ((448.0, 0), (448.00003, 1), (224.0, -1), (224.00002, 0), (1.0, -8), (1.75, -8),
                 (0.0, -60), (1e-30, -60), (3.4e38, 119)):
        assert ref.exp_of(np.float32(x)) == e, x
        if 1e-15 < x < 1e38:
            assert np.float32(x) <= 448 * 2.0 ** e and np.float32(x) > 448 * 2.0 ** (e - 1)


def test_missing_handles_are_refused():
    lib = ca.lib()
    null = C.c_void_p()
    assert lib.clove_hip_paged_kv8_append(*[None] * 7) == ca.ERR_INVALID
    assert lib.clove_hip_paged_kv8_read(None, None, None, None, None, 3, C.byref(null),
                                        C.byref(null)) == ca.ERR_INVALID
    assert lib.clove_hip_paged_kv8_read(None, None, None, None, None, 3, None,
                                        None) == ca.ERR_INVALID
    assert not lib.clove_hip_paged_kv8_attention(None, None, None, None, None, None, 0.0, None,
                                                 None)
    assert lib.clove_hip_last_status() == ca.ERR_INVALID
    one = C.c_void_p(1)  # never followed: the pair is checked first
    assert not lib.clove_hip_paged_kv8_attention(None, None, None, None, None, None, 0.0, one,
                                                 None)
    assert "both weights and weights_out" in ca.last_error()
    outs = [C.byref(C.c_void_p(5)) for _ in range(4)]
    assert lib.clove_hip_paged_evict(None, None, None, 16, 4, 1, 1, *outs) == ca.ERR_INVALID
    assert all(o._obj.value is None for o in outs)  # no stale handle on failure
    with pytest.raises(ValueError):
        ca.paged_kv8_read(None, None, None, None, row_starts=object())


@pytest.mark.parametrize("per,mul,extra,need", [
    # tiles that a sequence's rows may touch; row tiles of grouped heads
    (16, 1, 2, "tiles"), (1, 1, 2, "tiles"), (7, 1, 2, "tiles"), (128, 1, 1, "rows"),
    (16, 8, 1, "rows"), (64, 3, 1, "rows")])
def test_slots_hold_every_split(per, mul, extra, need):
    """floor(mul * start / per) + extra * b leaves each sequence room for its
    items, and the last ends inside the grid."""
    g = rng(per * 31 + mul)
    for _ in range(300):
        B = int(g.integers(1, 9))
        n = g.integers(0, int(g.choice([2, 5, 40, 300])), B)
        starts = ref.starts_of(n)
        base = [int(s) * mul // per + extra * b for b, s in enumerate(starts[:-1])]
        total = int(starts[-1]) * mul // per + extra * B
        for b in range(B):
            if need == "tiles":  # any position of the first row inside a block
                items = max(-(-(p + int(n[b])) // per) for p in range(per)) if n[b] else 0
            else:
                items = -(-int(n[b]) * mul // per)
            end = base[b + 1] if b + 1 < B else total
            assert base[b] + items <= end
