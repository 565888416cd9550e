"""GPU: the paged KV cache in 8 bits against its definition in numpy (kv8_ref):
the append that quantises, the read back, attention over the cache, and a run
of them together with the f32 prefill and the eviction.

Codes and exponents are bit-determined (scaling by powers of two is exact and
each element is rounded once), so they are compared exactly; attention within
the bounds that kv8_ref.attention derives from its 32-bit arithmetic.
"""
import ctypes as C

import numpy as np
import pytest

import kv8_ref as ref
from conftest import rng

pytestmark = pytest.mark.gpu


def up(hip, *arrays):
    return [None if a is None else hip.tensor(a, a.dtype.type) for a in arrays]


def within(got, want, tol, what=""):
    err = np.abs(np.asarray(got, np.float64) - want)
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {bad.sum()} of {err.size} out of tolerance, worst "
                           f"{(err / tol)[bad].max():.2f} times it, max abs err {err.max():.3e}")


def ragged(g, B, rows_hi, past_hi):
    rows = g.integers(0, rows_hi + 1, B)
    past = g.integers(0, past_hi + 1, B)
    return rows, (rows + past).astype(np.int32)


# ---- append and read --------------------------------------------------------

def check_append(hip, g, codes, exps, k, v, tables, lens, starts):
    tc, te = up(hip, codes, exps)
    hip.paged_kv8_append(tc, te, *up(hip, k, v, tables, lens, starts))
    hip.synchronize()
    ref.append(codes, exps, k, v, tables, lens, starts)
    np.testing.assert_array_equal(te.numpy(), exps)
    np.testing.assert_array_equal(tc.numpy(), codes)  # bytes behind the rows too
    rows = len(k)
    got = hip.paged_kv8_read(tc, te, *up(hip, tables, lens, starts), rows=rows)
    want = ref.read(codes, exps, tables, lens, rows, starts)
    for x, y in zip(got, want):
        np.testing.assert_array_equal(x.numpy(), y.astype(np.float32))


@pytest.mark.parametrize("D,bs,H", [(64, 16, 3), (128, 16, 2), (80, 8, 2), (256, 32, 1), (96, 64, 2),
                                    (1, 1, 1), (7, 5, 3), (33, 16, 2), (130, 3, 1), (16, 128, 2),
                                    (4, 16, 5), (255, 33, 1), (128, 128, 1)])
@pytest.mark.parametrize("rows_hi,past_hi", [(1, 70), (40, 0), (90, 50)])
def test_append_and_read(hip, D, bs, H, rows_hi, past_hi):
    g = rng(1000 + D * 31 + bs + rows_hi)
    rows, lens = ragged(g, 5, rows_hi, past_hi)
    width = max(1, -(-(rows_hi + past_hi) // bs))
    tables, nb = ref.pool(g, lens, bs, width)
    codes, exps = ref.cache(g, nb, H, bs, D)
    n = int(rows.sum())
    # rows of very different sizes, so that tiles grow or keep their exponents
    k, v = ((g.standard_normal((n, H * D)) * 2.0 ** g.integers(-8, 8, (n, 1))).astype(np.float32)
            for _ in range(2))
    check_append(hip, g, codes, exps, k, v, tables, lens, ref.starts_of(rows))


def test_append_one_row_each_and_growth(hip):
    """A token a call, as a decode loop stores them: each tile's exponent only
    grows while its block fills, and starts afresh in the next block."""
    g = rng(7)
    B, H, D, bs, width = 3, 2, 64, 4, 4
    tables, nb = ref.pool(g, [bs * width] * B, bs, width)
    codes, exps = ref.cache(g, nb, H, bs, D)
    for step in range(1, 12):
        lens = np.array([step, step + 3, 0 if step % 2 else step], np.int32)
        k, v = ((g.standard_normal((B, H * D)) * 2.0 ** g.integers(-6, 6)).astype(np.float32)
                for _ in range(2))
        check_append(hip, g, codes, exps, k, v, tables, lens, None)


@pytest.mark.parametrize("size", [0.0, 1e-45, 1e-20, 1.0, 448.0, 449.0, 3.4e38])
def test_append_sizes(hip, size):
    """From all zeros to the largest floats: the exponent's clamps at both ends."""
    g = rng(11)
    tables, lens = np.array([[1, 0]], np.int32), np.array([9], np.int32)
    codes, exps = ref.cache(g, 2, 1, 8, 16)
    k, v = ((g.uniform(-1, 1, (9, 16)) * size).astype(np.float32) for _ in range(2))
    k[0, 0] = v[0, 0] = np.float32(size)
    check_append(hip, g, codes, exps, k, v, tables, lens, np.array([0, 9], np.int32))


def test_every_rounding(hip):
    """Values on, beside and half way between codes, and every code back."""
    mags = ref.VALUES[:127]
    mid = (mags[1:] + mags[:-1]) / 2
    y = np.concatenate([mags, mid, np.nextafter(mid.astype(np.float32), np.float32(0)),
                        np.nextafter(mid.astype(np.float32), np.float32(1e9))])
    y = np.concatenate([y, -y, np.zeros(-2 * len(y) % 64)]).astype(np.float32).reshape(-1, 64)
    y[0, 0] = 448.0
    g = rng(5)
    n = len(y)
    codes, exps = ref.cache(g, 1, 1, n, 64)
    check_append(hip, g, codes, exps, y, y[::-1].copy(), np.array([[0]], np.int32),
                 np.array([n], np.int32), np.array([0, n], np.int32))


def test_append_not_finite(hip):
    """NaN as 0, infinities as their tile's largest, both reported once."""
    g = rng(13)
    tables, lens = np.array([[0], [1]], np.int32), np.array([3, 2], np.int32)
    codes, exps = ref.cache(g, 2, 2, 8, 16)
    k, v = (g.standard_normal((5, 32)).astype(np.float32) for _ in range(2))
    k[0, 3], k[1, 20], v[4, 0], v[2, 5] = np.nan, np.inf, -np.inf, np.nan
    v[3:, 16:] = np.inf  # a tile without a finite value
    starts = np.array([0, 3, 5], np.int32)
    tc, te = up(hip, codes, exps)
    hip.paged_kv8_append(tc, te, *up(hip, k, v, tables, lens, starts))
    with pytest.raises(hip.CloveError) as e:
        hip.synchronize()
    assert e.value.code == hip.ERR_RANGE and "not finite" in str(e.value)
    hip.synchronize()
    ref.append(codes, exps, k, v, tables, lens, starts)
    np.testing.assert_array_equal(te.numpy(), exps)
    np.testing.assert_array_equal(tc.numpy(), codes)


def test_rows_of_no_sequence_and_before_a_context(hip):
    """Rows in front of, behind and between nobody's sequences, more rows than
    context, empty contexts: skipped, and zeros when read or attended."""
    g = rng(17)
    H, D, bs = 2, 64, 8
    rows = [2, 0, 6, 1]
    starts = ref.starts_of(rows) + 3       # rows 0..2 belong to nobody
    lens = np.array([9, 20, 4, 0], np.int32)  # 6 rows in a context of 4, a row in none
    n = int(starts[-1]) + 5                # nor do the last five
    tables, nb = ref.pool(g, lens, bs, 3)
    codes, exps = ref.cache(g, nb, H, bs, D)
    k, v = (g.standard_normal((n, H * D)).astype(np.float32) for _ in range(2))
    check_append(hip, g, codes, exps, k, v, tables, lens, starts.astype(np.int32))
    q = g.standard_normal((n, H * D)).astype(np.float32)
    check_attention(hip, q, codes, exps, tables, lens, starts.astype(np.int32),
                    weights=g.random(tables.shape).astype(np.float32))


def test_bad_blocks_and_row_starts_are_reported(hip):
    g = rng(19)
    H, D, bs = 2, 32, 4
    lens = np.array([10, 7, 30], np.int32)    # the last one past its table
    tables, nb = ref.pool(g, [10, 7, 12], bs, 3)
    tables[0, 1], tables[1, 0] = nb, -5
    codes, exps = ref.cache(g, nb, H, bs, D)
    rows = np.array([10, 3, 12])
    starts = ref.starts_of(rows)
    k, v = (g.standard_normal((25, H * D)).astype(np.float32) for _ in range(2))
    q = g.standard_normal((25, H * D)).astype(np.float32)
    tc, te, tt, tl, ts = up(hip, codes, exps, tables, lens, starts)

    def reported(word):
        with pytest.raises(hip.CloveError) as e:
            hip.synchronize()
        assert e.value.code == hip.ERR_RANGE and word in str(e.value)

    hip.paged_kv8_append(tc, te, *up(hip, k, v), tt, tl, ts)
    reported("block-table")
    ref.append(codes, exps, k, v, tables, lens, starts)
    np.testing.assert_array_equal(tc.numpy(), codes)
    hip.paged_kv8_read(tc, te, tt, tl, ts, rows=25)
    reported("block-table")
    w = g.random(tables.shape).astype(np.float32)
    out, wo = hip.paged_kv8_attention(hip.tensor(q), tc, te, tt, tl, ts, weights=hip.tensor(w))
    reported("block-table")
    want, ww, tol, wtol = ref.attention(q, codes, exps, tables, lens, starts, weights=w)
    within(out.numpy(), want, tol, "out")
    within(wo.numpy(), ww, wtol + 1e-37, "weights")
    # ranges that decrease, start before the rows or end behind them: no rows
    good = np.array([4, 4, 4], np.int32)
    for bad in ([0, 30, 10, 25], [-1, 3, 5, 25], [0, 2, 3, 26], [2**31 - 1, -2**31, 7, 9]):
        hip.paged_kv8_append(tc, te, *up(hip, k, v, np.zeros((3, 1), np.int32) + np.arange(
            3, dtype=np.int32)[:, None], good, np.array(bad, np.int32)))
        reported("row_starts")
    hip.paged_evict(tt, tl, hip.tensor(w), bs, 2, 0, 1)
    reported("block-table")
    hip.synchronize()


# ---- attention ----------------------------------------------------------------

def check_attention(hip, q, codes, exps, tables, lens, starts=None, scale=None, weights=None):
    got = hip.paged_kv8_attention(*up(hip, q, codes, exps, tables, lens, starts),
                                  scale=scale or 0.0,
                                  weights=None if weights is None else hip.tensor(weights))
    want, w, tol, wtol = ref.attention(q, codes, exps, tables, lens, starts, scale, weights)
    out = got if weights is None else got[0]
    assert out.shape == q.shape
    within(out.numpy(), want, tol, "out")
    if weights is not None:
        within(got[1].numpy(), w, wtol + 1e-37, "weights")
    hip.synchronize()
    return out.numpy()


SHAPES = [  # head_dim, block size, kv heads, query heads
    (64, 16, 2, 2), (128, 16, 2, 2), (128, 16, 1, 4), (128, 16, 2, 16), (80, 8, 2, 6), (96, 32, 2, 4),
    (256, 16, 1, 2), (256, 64, 1, 8), (112, 16, 1, 7), (64, 32, 1, 20), (16, 16, 3, 3),
    (128, 128, 1, 1), (32, 4, 2, 2), (64, 24, 2, 4), (240, 16, 1, 3), (64, 16, 1, 40),
    # not whole 16-byte rows, block sizes of no power of two
    (1, 16, 1, 1), (7, 5, 2, 4), (50, 16, 1, 2), (100, 3, 1, 3), (255, 16, 1, 1), (64, 1, 2, 2),
]


@pytest.mark.parametrize("weighed", [False, True])
@pytest.mark.parametrize("D,bs,H,Hq", SHAPES)
def test_decode(hip, D, bs, H, Hq, weighed):
    g = rng(2000 + D + 7 * bs + Hq)
    # no context, one token, block and tile edges, partitions
    lens = np.array([1, 0, bs, bs + 1, 63, 64, 65, 300, 700], np.int32)
    width = -(-700 // bs) + 2
    tables, nb = ref.pool(g, lens, bs, width)
    codes, exps = ref.cache(g, nb, H, bs, D)
    q = g.standard_normal((len(lens), Hq * D)).astype(np.float32)
    check_attention(hip, q, codes, exps, tables, lens,
                    weights=g.random(tables.shape).astype(np.float32) if weighed else None)


@pytest.mark.parametrize("weighed", [False, True])
@pytest.mark.parametrize("D,bs,H,Hq", SHAPES)
def test_rows(hip, D, bs, H, Hq, weighed):
    """Chunks of prompts and single tokens in one call."""
    g = rng(3000 + D + 7 * bs + Hq)
    rows = np.array([1, 37, 0, 64, 5, 130])
    past = np.array([90, 0, 40, 17, 200, 3])
    lens = (rows + past).astype(np.int32)
    tables, nb = ref.pool(g, lens, bs, -(-int(lens.max()) // bs) + 1)
    codes, exps = ref.cache(g, nb, H, bs, D)
    q = g.standard_normal((int(rows.sum()), Hq * D)).astype(np.float32)
    check_attention(hip, q, codes, exps, tables, lens, ref.starts_of(rows),
                    scale=0.07 if D > 64 else None,
                    weights=g.random(tables.shape).astype(np.float32) if weighed else None)


@pytest.mark.parametrize("ctx,Hq", [(5000, 2), (20011, 8)])
def test_long_context(hip, ctx, Hq):
    """The context split over workgroups, for one row and for a few."""
    g = rng(ctx)
    H, D, bs = 1, 64, 16
    for rows in (1, 6):
        lens = np.array([ctx, 40], np.int32)
        tables, nb = ref.pool(g, lens, bs, -(-ctx // bs))
        codes, exps = ref.cache(g, nb, H, bs, D)
        q = g.standard_normal((2 * rows, Hq * D)).astype(np.float32)
        check_attention(hip, q, codes, exps, tables, lens,
                        None if rows == 1 else ref.starts_of([rows, rows]),
                        weights=g.random(tables.shape).astype(np.float32))


def test_scores_far_apart(hip):
    """One token far ahead of the rest, weights that underflow, values of very
    different sizes behind them, and query elements of very different sizes."""
    g = rng(23)
    H, D, bs, n = 1, 64, 16, 200
    lens = np.array([n], np.int32)
    tables, nb = ref.pool(g, lens, bs, 13)
    codes, exps = ref.cache(g, nb, H, bs, D)
    exps[1] = g.integers(-50, 60, exps[1].shape)
    q = (g.standard_normal((1, D)) * 2.0 ** g.integers(-20, 12, (1, D))).astype(np.float32)
    for scale in (1.0, 0.01, 1e-6):
        check_attention(hip, q, codes, exps, tables, lens, scale=scale)
        check_attention(hip, np.repeat(q, 40, 0), codes, exps, tables, lens,
                        np.array([0, 40], np.int32), scale=scale)


def test_codes_behind_a_context_do_not_count(hip):
    """NaN codes and wild exponents in slots and blocks that no row sees."""
    g = rng(29)
    H, D, bs = 2, 64, 16
    lens = np.array([21, 16, 3], np.int32)
    tables, nb = ref.pool(g, lens, bs, 4)
    codes, exps = ref.cache(g, nb, H, bs, D)
    used = np.zeros((nb, bs), bool)
    for b, n in enumerate(lens):
        for t in range(n):
            used[tables[b, t // bs], t % bs] = True
    codes.transpose(1, 3, 0, 2, 4)[~used] = 0x7F
    exps[:, ~used.any(1)] = 2**31 - 1
    q = g.standard_normal((3, 2 * H * D)).astype(np.float32)
    check_attention(hip, q, codes, exps, tables, lens,
                    weights=np.zeros(tables.shape, np.float32))
    rows = np.array([9, 16, 3])
    q = g.standard_normal((28, 2 * H * D)).astype(np.float32)
    check_attention(hip, q, codes, exps, tables, lens, ref.starts_of(rows),
                    weights=np.zeros(tables.shape, np.float32))


def test_not_finite_queries_stay_in_their_rows(hip):
    g = rng(31)
    H, D, bs = 2, 64, 16
    lens = np.array([50, 60], np.int32)
    tables, nb = ref.pool(g, lens, bs, 4)
    codes, exps = ref.cache(g, nb, H, bs, D)
    q = g.standard_normal((40, 2 * H * D)).astype(np.float32)
    starts = np.array([0, 25, 40], np.int32)
    clean = check_attention(hip, q, codes, exps, tables, lens, starts)
    q[3, 5], q[30, 70] = np.nan, np.nan
    got = hip.paged_kv8_attention(*up(hip, q, codes, exps, tables, lens, starts)).numpy()
    dirty = np.zeros((40, 2 * H), bool)
    dirty[3, 0] = dirty[30, 1] = True
    heads = got.reshape(40, 2 * H, D)
    assert np.isnan(heads[dirty]).all()
    np.testing.assert_array_equal(heads[~dirty], clean.reshape(40, 2 * H, D)[~dirty])


@pytest.mark.parametrize("rows,Hq", [(1, 4), (6, 4), (200, 2)])
def test_not_finite_queries_over_cut_contexts(hip, rows, Hq):
    """The same where a context is cut over workgroups and joined."""
    g = rng(rows)
    H, D, bs, n = 2, 64, 16, 6000
    lens = np.array([n], np.int32)
    tables, nb = ref.pool(g, lens, bs, n // bs)
    codes, exps = ref.cache(g, nb, H, bs, D)
    q = g.standard_normal((rows, Hq * D)).astype(np.float32)
    starts, w = np.array([0, rows], np.int32), np.zeros(tables.shape, np.float32)
    clean = check_attention(hip, q, codes, exps, tables, lens, starts, weights=w)
    q[0, 5] = np.nan
    out, wo = hip.paged_kv8_attention(*up(hip, q, codes, exps, tables, lens, starts),
                                      weights=hip.tensor(w))
    got = out.numpy().reshape(rows, Hq, D)
    assert np.isnan(got[0, 0]).all() and np.isnan(wo.numpy()[0, 0])
    dirty = np.zeros((rows, Hq), bool)
    dirty[0, 0] = True
    np.testing.assert_array_equal(got[~dirty], clean.reshape(rows, Hq, D)[~dirty])


def test_shared_blocks_and_repeats(hip):
    """Sequences that share a prefix's blocks, and the same bits twice."""
    g = rng(37)
    H, D, bs = 2, 128, 16
    lens = np.array([100, 90, 130], np.int32)
    tables, nb = ref.pool(g, lens, bs, 9)
    tables[1, :3] = tables[0, :3]
    tables[2, :5] = tables[0, :5]
    codes, exps = ref.cache(g, nb, H, bs, D)
    for rows in (None, np.array([3, 64, 20])):
        starts = None if rows is None else ref.starts_of(rows)
        n = 3 if rows is None else int(rows.sum())
        q = g.standard_normal((n, 2 * H * D)).astype(np.float32)
        w = g.random(tables.shape).astype(np.float32)
        args = up(hip, q, codes, exps, tables, lens, starts)
        first = [x.numpy() for x in hip.paged_kv8_attention(*args, weights=hip.tensor(w))]
        for _ in range(2):
            for x, y in zip(hip.paged_kv8_attention(*args, weights=hip.tensor(w)), first):
                np.testing.assert_array_equal(x.numpy(), y)
        want, ww, tol, wtol = ref.attention(q, codes, exps, tables, lens, starts, weights=w)
        within(first[0], want, tol, "out")
        within(first[1], ww, wtol, "weights")


@pytest.mark.parametrize("weighed", [False, True])
@pytest.mark.parametrize("D,bs,H,Hq,rows_hi", [
    # four heads to a workgroup
    (64, 16, 16, 16, 1), (128, 8, 16, 32, 1), (112, 4, 16, 16, 1), (128, 16, 16, 16, 12),
    (64, 16, 16, 16, 30),
    # two
    (256, 16, 8, 16, 1), (144, 16, 8, 8, 8), (128, 16, 8, 8, 40), (80, 32, 8, 16, 20)])
def test_many_sequences_and_heads(hip, D, bs, H, Hq, rows_hi, weighed):
    """Enough tiles that heads are taken together; one context in many pieces,
    whose table of tokens is filled twice."""
    g = rng(4000 + D + bs + Hq + rows_hi)
    B = 70
    rows = np.ones(B, np.int64) if rows_hi == 1 else g.integers(0, rows_hi + 1, B)
    if rows_hi > 1:
        rows[7] = rows_hi
    lens = (rows + g.integers(0, 70, B)).astype(np.int32)
    lens[3], lens[9] = 0, 2100 + bs
    rows[3] = min(rows[3], 1)
    tables, nb = ref.pool(g, lens, bs, -(-int(lens.max()) // bs))
    codes, exps = ref.cache(g, nb, H, bs, D)
    q = g.standard_normal((int(rows.sum()), Hq * D)).astype(np.float32)
    check_attention(hip, q, codes, exps, tables, lens, None if rows_hi == 1 else ref.starts_of(rows),
                    weights=g.random(tables.shape).astype(np.float32) if weighed else None)


@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_long_prompt_chunks(hip, D):
    """Chunks far into contexts: several tables of tokens to a tile, tiles cut
    over workgroups and joined."""
    g = rng(D)
    rows, past = np.array([70, 3, 41]), np.array([5000, 4096, 2040])
    lens = (rows + past).astype(np.int32)
    tables, nb = ref.pool(g, lens, 16, -(-5070 // 16))
    codes, exps = ref.cache(g, nb, 1, 16, D)
    q = g.standard_normal((int(rows.sum()), 2 * D)).astype(np.float32)
    check_attention(hip, q, codes, exps, tables, lens, ref.starts_of(rows),
                    weights=g.random(tables.shape).astype(np.float32))


@pytest.mark.parametrize("kspan,vspan,top", [(22, 22, -5), (23, 0, -5), (0, 23, -5), (3, 3, 60),
                                             (3, 3, 61), (3, 3, -57), (3, 3, 70)])
@pytest.mark.parametrize("small,gap,every", [(0, 0, 2), (1, 20, 2), (40, 20, 2), (63, 20, 2),
                                             (1, 24, 1), (1, 40, 1), (40, 40, 1)])
def test_sizes_of_tiles_and_query_elements(hip, kspan, vspan, top, small, gap, every):
    """Tiles whose exponents lie as far apart as 16-bit pieces hold and farther,
    the largest and smallest exponents, and rows of which `small` elements are
    2^gap below the others, with keys of zero at the large ones (in every other
    token, or in all of them, where the small ones alone make the scores)."""
    g = rng(100 * kspan + vspan + top + small + gap)
    H, D, bs, n = 2, 64, 16, 150
    lens = np.array([n], np.int32)
    tables, nb = ref.pool(g, lens, bs, 10)
    codes, exps = ref.cache(g, nb, H, bs, D)
    exps[0] = top - g.integers(0, kspan + 1, exps[0].shape)
    exps[1] = min(top, 100) - g.integers(0, vspan + 1, exps[1].shape)
    exps[0, tables[0, :2]] = np.array([[top], [max(top - kspan, -60)]])
    q = g.standard_normal((n, H * D)) * 2.0 ** (-9 - top + (gap if every == 1 else 0))
    at = g.permutation(D)[:small]
    q.reshape(n, H, D)[:, :, at] *= 2.0 ** -gap
    codes[0][:, :, ::every][..., np.setdiff1d(np.arange(D), at)] = 0
    check_attention(hip, q.astype(np.float32), codes, exps, tables, lens,
                    np.array([0, n], np.int32), weights=np.zeros(tables.shape, np.float32))


@pytest.mark.parametrize("rows", [1, 8, 60, 130])
def test_a_token_that_takes_all_the_weight(hip, rows):
    """A token 2^20 ahead of the others whose value is 0: what is left is the
    small weights' sum."""
    g = rng(43)
    H, D, bs, n = 2, 64, 16, 200
    lens = np.array([n], np.int32)
    tables, nb = ref.pool(g, lens, bs, 13)
    codes, exps = ref.cache(g, nb, H, bs, D)
    exps[0] = -10
    q = g.standard_normal((rows, H * D)).astype(np.float32)
    q.reshape(rows, H, D)[:, :, 0] = 5.0
    codes[0, :, :, :, 0] = 0
    codes[0, tables[0, 2]] = 0
    codes[1, tables[0, 2], :, 5] = 0
    codes[0, tables[0, 2], :, 5, 0] = ref.encode(np.array(20 * np.log(2) / 5 * 64))
    exps[0, tables[0, 2]] = -6
    out = check_attention(hip, q, codes, exps, tables, lens, np.array([0, rows], np.int32),
                          scale=1.0)
    assert np.abs(out).max() < 1e-2


@pytest.mark.parametrize("off", [4, 8, 16])
def test_wrapped_at_an_offset(hip, off):
    """Codes, exponents and rows that begin inside other allocations."""
    g = rng(off)
    H, D, bs = 2, 64, 16
    lens = np.array([40, 33, 90], np.int32)
    tables, nb = ref.pool(g, lens, bs, 6)
    codes, exps = ref.cache(g, nb, H, bs, D)
    hold = []

    def at(a, off=off):
        raw = np.concatenate([np.full(off, 0x55, np.uint8), a.reshape(-1).view(np.uint8),
                              np.full(32, 0x55, np.uint8)])
        hold.append(hip.tensor(raw, np.uint8))
        return hip.wrap(hold[-1].device_ptr + off, a.shape, a.dtype.type)

    for rows in ([1, 1, 1], [9, 0, 50]):
        starts = ref.starts_of(rows)
        n = int(starts[-1])
        k, v, q = (g.standard_normal((n, H * D)).astype(np.float32) for _ in range(3))
        for where in ((off, off), (off, 0), (0, off)):
            w = g.random(tables.shape).astype(np.float32)
            tc, te, tk, tv = at(codes, where[0]), at(exps), at(k), at(v)
            tt, tl, ts = at(tables), at(lens), at(starts)
            hip.paged_kv8_append(tc, te, tk, tv, tt, tl, ts)
            ref.append(codes, exps, k, v, tables, lens, starts)
            np.testing.assert_array_equal(tc.numpy(), codes)
            np.testing.assert_array_equal(te.numpy(), exps)
            for x, y in zip(hip.paged_kv8_read(tc, te, tt, tl, ts, rows=n),
                            ref.read(codes, exps, tables, lens, n, starts)):
                np.testing.assert_array_equal(x.numpy(), y.astype(np.float32))
            out, wo = hip.paged_kv8_attention(at(q, where[1]), tc, te, tt, tl, ts, weights=at(w))
            want, ww, tol, wtol = ref.attention(q, codes, exps, tables, lens, starts, weights=w)
            within(out.numpy(), want, tol, "out")
            within(wo.numpy(), ww, wtol, "weights")
            for x, y in zip(hip.paged_evict(tt, tl, at(w), bs, 3, 1, 1),
                            ref.evict(tables, lens, w, bs, 3, 1, 1)):
                np.testing.assert_array_equal(x.numpy(), y)
    for t in hold:  # nothing before or behind the tensors was touched
        raw = t.numpy()
        assert (raw[-32:] == 0x55).all()


@pytest.mark.parametrize("rows,D,Hq", [(25, 32, 2), (25, 128, 8), (400, 64, 2)])
def test_bad_row_starts_and_blocks_in_attention(hip, rows, D, Hq):
    """Starts that leave the rows: reported, and the other sequences get their
    answers.  Starts that decrease: reported (what the rows receive is not
    specified).  Then tables that leave the pool, in every kernel of the attention."""
    g = rng(rows + D)
    H, bs, ctx = 2, 16, 700
    lens = np.array([ctx, ctx - 5, 90], np.int32)
    tables, nb = ref.pool(g, lens, bs, 44)
    codes, exps = ref.cache(g, nb, H, bs, D)
    q = g.standard_normal((rows, Hq * D)).astype(np.float32)
    w = g.random(tables.shape).astype(np.float32)
    part = rows * 2 // 5
    for starts, whole in (([0, rows + 1, part, rows], []), ([0, 2 * part, part, rows], []),
                          ([-1, 3, 5, rows], [1, 2]), ([0, part, 2 * part, rows + 1], [0, 1]),
                          ([2**31 - 1, -2**31, 0, rows], [])):
        starts = np.array(starts, np.int32)
        args = up(hip, q, codes, exps, tables, lens, starts)
        out, wo = hip.paged_kv8_attention(*args, weights=hip.tensor(w))
        with pytest.raises(hip.CloveError) as e:
            hip.synchronize()
        assert e.value.code == hip.ERR_RANGE and "row_starts" in str(e.value)
        want, ww, tol, wtol = ref.attention(q, codes, exps, tables, lens, starts, weights=w)
        got, gw = out.numpy(), wo.numpy()
        for b in whole:
            at = slice(starts[b], starts[b + 1])
            within(got[at], want[at], tol[at], f"out of {b} of {starts}")
            within(gw[b], ww[b], wtol[b] + 1e-37, f"weights of {b} of {starts}")
    tables[0, [0, 3, 20]], tables[1, 43], tables[2, :] = [nb, -1, 2**31 - 1], -2**31, -7
    starts = np.array([0, part, 2 * part, rows], np.int32)
    out, wo = hip.paged_kv8_attention(*up(hip, q, codes, exps, tables, lens, starts),
                                      weights=hip.tensor(w))
    with pytest.raises(hip.CloveError) as e:
        hip.synchronize()
    assert e.value.code == hip.ERR_RANGE and "block-table" in str(e.value)
    want, ww, tol, wtol = ref.attention(q, codes, exps, tables, lens, starts, weights=w)
    within(out.numpy(), want, tol, "out")
    within(wo.numpy(), ww, wtol + 1e-37, "weights")


def test_on_another_stream(hip):
    """A step on the backend's stream, the next on a caller's: each waits for
    what it reads."""
    rt = C.CDLL("libamdhip64.so")
    g = rng(47)
    H, D, bs, B = 2, 64, 16, 3
    lens = np.array([40, 17, 64], np.int32)
    tables, nb = ref.pool(g, lens + 2, bs, 5)
    codes, exps = ref.cache(g, nb, H, bs, D)
    tc, te, tt = up(hip, codes, exps, tables)
    other = C.c_void_p()
    assert rt.hipStreamCreate(C.byref(other)) == 0
    try:
        for stream in (None, other, None):
            k, v, q = (g.standard_normal((B, H * D)).astype(np.float32) for _ in range(3))
            tl, tq = up(hip, lens, q)
            tk, tv = up(hip, k, v)
            assert hip.lib().clove_hip_set_stream(stream) == 0
            hip.paged_kv8_append(tc, te, tk, tv, tt, tl)
            ref.append(codes, exps, k, v, tables, lens)
            out = hip.paged_kv8_attention(tq, tc, te, tt, tl).numpy()
            want, _, tol, _ = ref.attention(q, codes, exps, tables, lens)
            within(out, want, tol, "out")
            lens = lens + 1
    finally:
        hip.lib().clove_hip_set_stream(None)
        rt.hipStreamDestroy(other)
    hip.synchronize()


def test_no_rows_and_no_sequences(hip):
    codes, exps = hip.paged_kv8_cache(2, 1, 4, 8)
    none, z = np.zeros((0, 8), np.float32), np.zeros(1, np.int32)
    tables, lens = up(hip, np.zeros((0, 3), np.int32), np.zeros(0, np.int32))
    hip.paged_kv8_append(codes, exps, *up(hip, none, none), tables, lens, hip.tensor(z))
    out, w = hip.paged_kv8_attention(hip.tensor(none), codes, exps, tables, lens, hip.tensor(z),
                                     weights=hip.tensor(np.zeros((0, 3), np.float32)))
    assert out.shape == (0, 8) and w.shape == (0, 3)
    # rows but no sequences; sequences but no rows: weights are copied
    x = hip.tensor(np.ones((4, 8), np.float32))
    out = hip.paged_kv8_attention(x, codes, exps, tables, lens, hip.tensor(z))
    np.testing.assert_array_equal(out.numpy(), 0)
    k, v = hip.paged_kv8_read(codes, exps, tables, lens, hip.tensor(z), rows=4)
    assert not k.numpy().any() and not v.numpy().any()
    w0 = np.arange(6, dtype=np.float32).reshape(2, 3)
    t2, l2, s2 = up(hip, np.zeros((2, 3), np.int32), np.array([5, 0], np.int32),
                    np.zeros(3, np.int32))
    out, w = hip.paged_kv8_attention(hip.tensor(none), codes, exps, t2, l2, s2,
                                     weights=hip.tensor(w0))
    np.testing.assert_array_equal(w.numpy(), w0)
    hip.synchronize()


# ---- eviction -----------------------------------------------------------------

@pytest.mark.parametrize("width,bs,budget,first,last", [
    (1, 16, 1, 0, 1), (5, 4, 3, 1, 1), (5, 4, 2, 1, 1), (40, 16, 16, 0, 1), (300, 16, 64, 4, 8),
    (1500, 8, 700, 2, 3), (3000, 1, 31, 0, 31), (2048, 16, 2047, 0, 1), (70, 3, 200, 5, 5),
    (9000, 2, 1000, 3, 2), (20000, 1, 15000, 1, 1)])
def test_evict(hip, width, bs, budget, first, last):
    g = rng(width + budget)
    lens = np.concatenate([[0, 1, width * bs, width * bs - bs + 1],
                           g.integers(0, width * bs + 1, 6)]).astype(np.int32)
    tables, _ = ref.pool(g, lens, bs, width)
    for kind in range(4):
        w = np.exp(g.standard_normal(tables.shape) * 3).astype(np.float32)
        if kind == 1:    # many equal ones
            w = g.integers(0, 3, tables.shape).astype(np.float32)
        elif kind == 2:  # what no sum of weights is, but a caller may pass
            w = g.choice(np.array([np.nan, np.inf, -np.inf, -0.0, 0.0, 1e-45, -3.0, 2.0],
                                  np.float32), tables.shape)
        elif kind == 3:
            w[:] = 0.5
        got = hip.paged_evict(*up(hip, tables, lens, w), bs, budget, first, last)
        for x, y, what in zip(got, ref.evict(tables, lens, w, bs, budget, first, last),
                              ("tables", "lens", "weights", "evicted")):
            np.testing.assert_array_equal(x.numpy(), y, what)


# ---- refusals -----------------------------------------------------------------

def test_refusals(hip):
    f = lambda *s: hip.tensor(np.zeros(s, np.float32))
    i = lambda *s: hip.tensor(np.zeros(s, np.int32))
    codes, exps = hip.paged_kv8_cache(4, 2, 8, 16)
    tables, lens, starts = i(3, 2), i(3), i(4)
    q = f(3, 64)

    def refused(code, fn, *args, **kw):
        with pytest.raises(hip.CloveError) as e:
            fn(*args, **kw)
        assert e.value.code == code, e.value

    att, app = hip.paged_kv8_attention, hip.paged_kv8_append
    SH, INV = hip.ERR_SHAPE, hip.ERR_INVALID
    refused(INV, att, q, f(2, 4, 2, 8, 16), exps, tables, lens)           # codes not e4m3
    refused(INV, att, q, codes, f(2, 4, 2), tables, lens)                 # exps not int32
    refused(SH, att, q, codes, i(2, 4, 3), tables, lens)
    refused(SH, att, q, hip.empty((2, 4, 2, 128), np.uint8), exps, tables, lens)
    refused(SH, att, q, hip.empty((3, 4, 2, 8, 16), np.uint8), exps, tables, lens)
    refused(SH, att, f(3, 48), codes, exps, tables, lens)                 # not whole groups
    refused(SH, att, f(4, 64), codes, exps, tables, lens)                 # rows != sequences
    refused(SH, att, f(64), codes, exps, tables, lens)
    refused(INV, att, i(3, 64), codes, exps, tables, lens)
    refused(SH, att, q, codes, exps, i(2, 2), lens)
    refused(INV, att, q, codes, exps, f(3, 2), lens)
    refused(INV, att, q, codes, exps, tables, f(3))
    refused(SH, att, q, codes, exps, tables, lens, i(3))                  # starts: B + 1
    refused(INV, att, q, codes, exps, tables, lens, f(4))
    refused(SH, att, q, codes, exps, tables, lens, weights=f(3, 3))
    refused(INV, att, q, codes, exps, tables, lens, weights=i(3, 2))
    refused(SH, att, f(3, 2 * 257), hip.empty((2, 4, 2, 8, 257), np.uint8), exps, tables, lens)
    refused(SH, app, codes, exps, f(3, 32), f(2, 32), tables, lens)
    refused(SH, app, codes, exps, f(3, 31), f(3, 31), tables, lens)
    refused(SH, app, codes, exps, f(4, 32), f(4, 32), tables, lens)
    refused(INV, app, codes, exps, f(3, 32), i(3, 32), tables, lens, starts)
    refused(SH, hip.paged_kv8_read, codes, exps, tables, lens, None, 5)
    refused(INV, hip.paged_evict, tables, lens, f(3, 2), 0, 2)
    refused(INV, hip.paged_evict, tables, lens, f(3, 2), 8, 2, 0, 0)
    refused(INV, hip.paged_evict, tables, lens, f(3, 2), 8, 2, 2, 1)
    refused(INV, hip.paged_evict, tables, lens, f(3, 2), 8, 2, -1, 1)
    refused(SH, hip.paged_evict, tables, lens, f(3, 3), 8, 2)
    refused(INV, hip.paged_evict, tables, lens, i(3, 2), 8, 2)
    # an e4m3 tensor in an f32 op
    for fn in (hip.relu, hip.softmax, hip.transpose):
        refused(INV, fn, hip.empty((4, 4), np.uint8))
    hip.synchronize()


def test_e4m3_tensors(hip):
    a = np.arange(256, dtype=np.uint8).reshape(4, 64)
    t = hip.tensor(a, np.uint8)
    assert t.dtype == np.uint8 and t.shape == (4, 64) and t.numel == 256
    np.testing.assert_array_equal(t.numpy(), a)
    np.testing.assert_array_equal(t.read(5, 7), a.ravel()[5:12])
    t.write(3, np.array([9, 8], np.uint8))
    assert t.numpy().ravel()[2:6].tolist() == [2, 9, 8, 5]
    # a graph's input handed through as an output: a copy of its bytes
    gr = hip.Graph()
    x = gr.input("4,64")
    np.testing.assert_array_equal(gr.compile([x]).execute([t])[0].numpy(), t.numpy())


# ---- together -------------------------------------------------------------------

def test_a_conversation(hip):
    """Two prompts in two chunks each, decode steps that keep the blocks'
    weights, an eviction, and more steps over what is left; every step against
    the same steps in numpy."""
    g = rng(41)
    B, H, G, D, bs, width = 2, 2, 2, 64, 8, 16
    tables, nb = ref.pool(g, [bs * width] * B, bs, width)
    codes, exps = ref.cache(g, nb, H, bs, D)
    tc, te, tt = up(hip, codes, exps, tables)
    lens = np.zeros(B, np.int32)
    tw, w = hip.tensor(np.zeros((B, width), np.float32)), np.zeros((B, width))
    wtol = np.zeros((B, width))

    def step(rows):
        nonlocal lens, tw, w, wtol
        lens = (lens + rows).astype(np.int32)
        n = int(np.sum(rows))
        starts = None if (np.asarray(rows) == 1).all() else ref.starts_of(rows)
        k, v = (g.standard_normal((n, H * D)).astype(np.float32) for _ in range(2))
        q = g.standard_normal((n, G * H * D)).astype(np.float32)
        tl, ts = up(hip, lens, starts)
        hip.paged_kv8_append(tc, te, *up(hip, k, v), tt, tl, ts)
        out, tw = hip.paged_kv8_attention(hip.tensor(q), tc, te, tt, tl, ts, weights=tw)
        ref.append(codes, exps, k, v, tables, lens, starts)
        want, nw, tol, _ = ref.attention(q, codes, exps, tables, lens, starts, weights=w)
        _, _, _, dw = ref.attention(q, codes, exps, tables, lens, starts,
                                    weights=np.zeros_like(w))
        w, wtol = nw, wtol + dw + np.abs(nw) * 2.0 ** -23
        within(out.numpy(), want, tol, f"out at {lens}")
        within(tw.numpy(), w, wtol + 1e-37, f"weights at {lens}")

    step([30, 19])
    step([21, 40])
    for _ in range(5):
        step([1, 1])
    got = hip.paged_evict(tt, hip.tensor(lens), tw, bs, 5, 1, 2)
    want = ref.evict(tables, lens, tw.numpy(), bs, 5, 1, 2)
    for x, y in zip(got, want):
        np.testing.assert_array_equal(x.numpy(), y)
    assert (want[1] < lens).all() and (want[3][:, 0] >= 0).all()
    tt, _, tw, _ = got
    tables, lens, w = want[0], want[1], want[2].astype(np.float64)
    # blocks for what comes next
    for b in range(B):
        tables[b, 5:8] = want[3][b, :3]
    tt = hip.tensor(tables)
    for _ in range(4):
        step([1, 1])
    step([7, 2])
    # the prompt's keys and values back in 32 bits, under the f32 prefill: the
    # same attention as the cache's own
    n = int(lens[0])
    k, v = hip.paged_kv8_read(tc, te, hip.tensor(tables[:1]), hip.tensor(lens[:1]),
                              hip.tensor(np.array([0, n], np.int32)), rows=n)
    q = g.standard_normal((n, H * D)).astype(np.float32)
    full = hip.flash_attention(hip.tensor(q), k, v, H, flags=hip.ATTN_CAUSAL).numpy()
    mine = hip.paged_kv8_attention(hip.tensor(q), tc, te, hip.tensor(tables[:1]),
                                   hip.tensor(lens[:1]),
                                   hip.tensor(np.array([0, n], np.int32))).numpy()
    _, _, tol, _ = ref.attention(q, codes, exps, tables[:1], lens[:1],
                                 np.array([0, n], np.int32))
    within(mine, full, 2 * tol, "prefill")
    hip.synchronize()
