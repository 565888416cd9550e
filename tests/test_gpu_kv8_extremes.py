"""GPU: attention over the 8-bit cache where magnitudes or sizes are extreme:
rows and keys of zero or nearly so, values whose exponents lie far apart along a
context, weights far below the largest, tables far wider than the contexts.
Bounds as kv8_ref.attention derives them."""
import numpy as np
import pytest

import kv8_ref as ref
from conftest import rng
from test_gpu_kv8 import check_attention, up, within

pytestmark = pytest.mark.gpu


# ---- zero rows over zero keys ---------------------------------------------------

# rows and earlier tokens of each sequence: a prompt; chunks cut over workgroups
PROMPT, CUT = ([150], [0]), ([130, 70], [5000, 40])


@pytest.mark.parametrize("rows,past", [PROMPT, CUT])
@pytest.mark.parametrize("D,H,Hq", [(64, 2, 2), (80, 2, 6), (128, 2, 2), (256, 1, 2)])
@pytest.mark.parametrize("what", ["all", "head", "rows", "tiny", "tinier"])
def test_zero_and_tiny_rows_over_zero_and_tiny_keys(hip, D, H, Hq, rows, past, what):
    """Scores that are all 0 (or too small to matter): a row's answer is the mean
    of the values that it sees, in whatever form the kernel holds rows and keys.
    all: a prompt of zeros; head: one kv head's rows and keys; rows: every third
    row over tiny keys; tiny, tinier: small rows over small keys."""
    g = rng(D + len(rows) + len(what))
    bs = 16
    lens = np.add(rows, past).astype(np.int32)
    tables, nb = ref.pool(g, lens, bs, -(-int(lens.max()) // bs))
    codes, exps = ref.cache(g, nb, H, bs, D)
    q = g.standard_normal((sum(rows), Hq * D)).astype(np.float32)
    heads = q.reshape(-1, H, Hq // H * D)
    if what == "all":
        codes[0], exps[0], q[:] = 0, -60, 0
    elif what == "head":
        codes[0, :, H - 1], exps[0, :, H - 1], heads[:, H - 1] = 0, -60, 0
    elif what == "rows":
        exps[0] -= 45
        q[::3] = 0
    elif what == "tiny":
        exps[0] -= 40
        q *= np.float32(2.0 ** -100)
    else:
        exps[0], codes[0, :, :, :, ::2] = -60, 0
        q *= np.float32(2.0 ** -120)
    check_attention(hip, q, codes, exps, tables, lens, ref.starts_of(rows),
                    weights=g.random(tables.shape).astype(np.float32))


def test_a_prompt_of_zeros_through_the_append(hip):
    """What a dummy pass of zeros stores and reads."""
    g = rng(61)
    H, D, bs, n = 2, 64, 16, 200
    lens, starts = np.array([n], np.int32), np.array([0, n], np.int32)
    tables, nb = ref.pool(g, lens, bs, 13)
    codes, exps = ref.cache(g, nb, H, bs, D)
    zero = np.zeros((n, H * D), np.float32)
    tc, te, tz, tt, tl, ts = up(hip, codes, exps, zero, tables, lens, starts)
    hip.paged_kv8_append(tc, te, tz, tz, tt, tl, ts)
    out, w = hip.paged_kv8_attention(tz, tc, te, tt, tl, ts,
                                     weights=hip.tensor(np.zeros(tables.shape, np.float32)))
    assert not out.numpy().any()
    # a row's weights add up to 1 for each of H heads; n + 16 roundings a row and head
    assert abs(float(w.numpy().astype(np.float64).sum()) - n * H) < n * H * (n + 16) * 2.0 ** -23


# ---- values of very different sizes along a context ----------------------------

def check_some_rows(hip, q, codes, exps, tables, ctx, past, heads, rows):
    """One sequence's attention; `rows` of `heads` against the definition, each
    as a sequence of its own that ends at the row's position."""
    H, D = codes.shape[2], codes.shape[4]
    n = len(q)
    got = hip.paged_kv8_attention(*up(hip, q, codes, exps, tables, np.array([ctx], np.int32),
                                      np.array([0, n], np.int32))).numpy().reshape(n, H, D)
    hip.synchronize()
    rows = np.array(rows)
    for h in heads:
        want, _, tol, _ = ref.attention(q.reshape(n, H, D)[rows, h], codes[:, :, h:h + 1],
                                        exps[:, :, h:h + 1], np.repeat(tables, len(rows), 0),
                                        past + rows + 1)
        within(got[rows, h], want, tol, f"head {h}")


@pytest.mark.parametrize("D,H,n,past", [(64, 64, 2048, 6000), (128, 64, 2048, 6000),
                                        (256, 16, 4096, 0)])
@pytest.mark.parametrize("first,then", [(45, None), (45, -55), (-55, 45), (None, 45), (60, -60)])
def test_values_of_different_sizes_along_a_context(hip, D, H, n, past, first, then):
    """Value exponents of a context's first tokens and of those behind them (None:
    zeros, as the append stores them), far apart; enough tiles that each workgroup
    walks a whole context and meets both."""
    g = rng(D + H)
    bs, ctx = 16, past + n
    tables, nb = ref.pool(g, [ctx], bs, -(-ctx // bs))
    codes = np.empty((2, nb, H, bs, D), np.uint8)
    some, _ = ref.cache(g, 40, 1, bs, D)  # (random codes, repeated: they are many)
    codes[:] = some[:, g.integers(0, 40, nb * H), 0].reshape(2, nb, H, bs, D)
    exps = np.full((2, nb, H), -8, np.int32)
    half = (2048 if D > 128 else 4096) // bs
    for ids, e in ((tables[0, :half], first), (tables[0, half:], then)):
        exps[1, ids] = -60 if e is None else e
        if e is None:
            codes[1, ids] = 0
    q = g.standard_normal((n, H * D), np.float32)
    check_some_rows(hip, q, codes, exps, tables, ctx, past, (0, H - 1),
                    (0, 1, n // 2 - 1, n // 2, n - 100, n - 1))


# ---- weights far below the largest ------------------------------------------------

@pytest.mark.parametrize("lead", [20, 24, 28, 33, 36, 40])
@pytest.mark.parametrize("rows,past", [(8, 192), (60, 140), (130, 70), (130, 5000)])
def test_small_weights_beside_a_token_without_value(hip, lead, rows, past):
    """A token 2^lead ahead of the others whose value is 0, in all dims or in every
    other: what the others' weights make has to keep its own precision."""
    g = rng(lead + rows)
    H, D, bs, n = 2, 64, 16, rows + past
    lens = np.array([n], np.int32)
    tables, nb = ref.pool(g, lens, bs, -(-n // bs))
    codes, exps = ref.cache(g, nb, H, bs, D)
    exps[0] = -10
    q = g.standard_normal((rows, H * D)).astype(np.float32)
    q.reshape(rows, H, D)[:, :, 0] = 5.0
    codes[0, :, :, :, 0] = 0
    codes[0, tables[0, 2]] = 0
    codes[1, tables[0, 2], 0, 5] = 0
    codes[1, tables[0, 2], 1, 5, ::2] = 0
    codes[0, tables[0, 2], :, 5, 0] = ref.encode(np.array(lead * np.log(2) / 5 * 64))
    exps[0, tables[0, 2]] = -6
    check_attention(hip, q, codes, exps, tables, lens, np.array([0, rows], np.int32), scale=1.0,
                    weights=np.zeros(tables.shape, np.float32))


# ---- tables far wider than the contexts -------------------------------------------

GIB = 1 << 30


@pytest.mark.parametrize("rows,H,Hq,bs,width,seqs,longest", [
    # decode in turns: sums of 16 tokens, of 4; joined contexts
    (1, 64, 64, 64, 256, 4096, 9000), (1, 64, 128, 8, 1024, 2048, 8100),
    # few rows each, scores computed again, 4096 tokens to a part of the tables
    (2, 64, 64, 64, 256, 4096, 9000),
    # a decode step of which one sequence's sums are too many
    (1, 8, 64, 4096, 9000, 2, 3000),
    # chunks whose sums are not stored (16 does not divide the block), 32768 to a part
    (40, 16, 16, 24, 4000, 2048, 70000)])
def test_weights_of_wide_tables(hip, rows, H, Hq, bs, width, seqs, longest):
    """The workspace of the blocks' weights stays below 1 GiB however wide the
    tables are, and weights in all parts of a table are right."""
    g = rng(seqs + width)
    D = 16
    n = np.full(seqs, rows)
    lens = np.zeros(seqs, np.int32)          # most rows stand before any token: zeros
    lens[::97] = g.integers(1, 3 * bs, len(lens[::97]))
    lens[seqs // 2], lens[-1] = longest, longest - min(2 * bs, 1000) - 1
    if rows > 2:
        n[seqs // 2], n[-1] = 3, 2
    tables, nb = ref.pool(g, lens, bs, width)
    codes, exps = ref.cache(g, nb, H, bs, D)
    starts = None if rows == 1 else ref.starts_of(n)
    q = g.standard_normal((int(n.sum()), Hq * D), np.float32)
    w = g.random(tables.shape, np.float32)
    args = up(hip, q, codes, exps, tables, lens, starts)
    tw = hip.tensor(w)
    hip.synchronize()
    before = hip.memory_reserved()
    out, wo = hip.paged_kv8_attention(*args, weights=tw)
    hip.synchronize()
    # the results, the pieces of contexts (at most 1024 x 2 x 128 rows of 16 and 2)
    # and the rows' maxima and sums come to less than a quarter of it
    assert hip.memory_reserved() - before < GIB + GIB // 4
    want, ww, tol, wtol = ref.attention(q, codes, exps, tables, lens, starts, weights=w)
    within(out.numpy(), want, tol, "out")
    within(wo.numpy(), ww, wtol + 1e-37, "weights")


# ---- capacities next to 2^31 tokens -------------------------------------------------

def test_capacities_next_to_2_31(hip):
    """Tables whose capacity a kernel's token numbers would leave are refused; the
    widest ones that are not hold a context to their last token."""
    g = rng(71)
    B, H, D, width, tokens = 1, 1, 16, 2048, 1 << 20
    q = g.standard_normal((B, H * D), np.float32)
    full = np.array([width * (tokens - 4)], np.int32)
    for bs, lens, code in ((tokens - 1, [100], "refused"), (tokens - 4, [100], None),
                           (tokens - 4, full, None)):
        tables, lens = np.zeros((1, width), np.int32), np.asarray(lens, np.int32)
        codes = ref.encode(g.standard_normal((2, 1, H, 1024, D)) * 120).repeat(1024, 3)[:, :, :, :bs]
        exps = np.full((2, 1, H), -7, np.int32)
        args = up(hip, q, np.ascontiguousarray(codes), exps, tables, lens)
        if code:
            with pytest.raises(hip.CloveError) as e:
                hip.paged_kv8_attention(*args)
            assert e.value.code == hip.ERR_SHAPE and "2^31" in str(e.value)
            continue
        out = hip.paged_kv8_attention(*args).numpy()
        hip.synchronize()
        # the block over and over: as over one of them
        one = np.minimum(lens, bs).astype(np.int32)
        want, _, _, _ = ref.attention(q, codes, exps, tables[:, :1], one)
        x, _ = ref.tokens(codes, exps, tables[:, :1], 0, int(one[0]))
        s = (x[0, :, 0] @ q[0].astype(np.float64)) / np.sqrt(D)
        p = np.exp(s - s.max())
        mag = (p / p.sum()) @ np.abs(x[1, :, 0])
        # every sum of a lane takes at most 2^17 tokens, then as many pieces again
        within(out, want, (2.0 ** 18 * 2.0 ** -24 + 2.0 ** -18) * mag[None], f"{bs} {lens}")
