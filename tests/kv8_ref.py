"""The 8-bit paged cache, its attention and the eviction in numpy, 64 bits,
written from their definitions (include/clove_hip.h); with makers of random
cases for the tests."""
import numpy as np

MIN_EXP, MAX_EXP, TOP = -60, 119, 448.0


def code_values():
    """The 256 e4m3 values; 0x7F and 0xFF are NaN."""
    v = np.empty(256)
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        x = f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
        v[c] = np.nan if c & 127 == 127 else (-x if c & 128 else x)
    return v


VALUES = code_values()
_MAGNITUDES = VALUES[:127]  # ascending


def encode(y):
    """Nearest e4m3 code, ties to the even one; NaN is 0, past 448 saturates."""
    y = np.asarray(y, np.float64)
    a = np.minimum(np.abs(np.nan_to_num(y, nan=0.0, posinf=TOP, neginf=-TOP)), TOP)
    hi = np.searchsorted(_MAGNITUDES, a)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _MAGNITUDES[lo], _MAGNITUDES[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (code | np.where(np.signbit(y) & ~np.isnan(y), 128, 0)).astype(np.uint8)


def exp_of(x):
    x = np.abs(np.asarray(x, np.float64))
    amax = x[np.isfinite(x)].max(initial=0.0)
    if amax == 0:
        return MIN_EXP
    _, e = np.frexp(amax / TOP)  # amax / 448 in [2^(e-1), 2^e)
    e = int(e) - 1 if amax / TOP == 2.0 ** (int(e) - 1) else int(e)
    return min(max(e, MIN_EXP), MAX_EXP)


def spans(lens, starts, rows, capacity):
    """(sequence, first row, rows, context) with clamped lengths."""
    out = []
    for b, ctx in enumerate(lens):
        s0, s1 = (b, b + 1) if starts is None else (int(starts[b]), int(starts[b + 1]))
        if not 0 <= s0 <= s1 <= rows:
            s0 = s1 = 0
        out.append((b, s0, s1 - s0, min(max(int(ctx), 0), capacity)))
    return out


def append(codes, exps, k, v, tables, lens, starts=None):
    """In place on numpy codes [2, nb, H, bs, D] and exps [2, nb, H]."""
    _, nb, H, bs, D = codes.shape
    for b, first, n, ctx in spans(lens, starts, len(k), tables.shape[1] * bs):
        past = ctx - n
        for j in range(max(past, 0) // bs, -(-ctx // bs)):
            blk = int(tables[b, j])
            lo, hi = max(past - j * bs, 0), min(ctx - j * bs, bs)
            if n == 0 or hi <= lo or not 0 <= blk < nb:
                continue
            r0 = first + j * bs + lo - past
            for plane, x in enumerate((k, v)):
                new = x[r0:r0 + hi - lo].reshape(hi - lo, H, D).astype(np.float64)
                for h in range(H):
                    e = exp_of(new[:, h])
                    if lo:
                        old = min(max(int(exps[plane, blk, h]), MIN_EXP), MAX_EXP)
                        if e > old:
                            t = codes[plane, blk, h, :lo]
                            t[:] = encode(VALUES[t] * 2.0 ** (old - e))
                        e = max(e, old)
                    exps[plane, blk, h] = e
                    codes[plane, blk, h, lo:hi] = encode(new[:, h] * 2.0 ** -e)


def tokens(codes, exps, tables, b, ctx):
    """Sequence b's keys and values [2, ctx, H, D] in 64 bits, and which tokens
    lie in the pool."""
    _, nb, H, bs, D = codes.shape
    ids = tables[b, :-(-ctx // bs)].astype(np.int64)
    ok = (ids >= 0) & (ids < nb)
    ids = np.where(ok, ids, 0)
    x = VALUES[codes[:, ids]] * 2.0 ** np.clip(exps[:, ids], MIN_EXP, MAX_EXP)[..., None, None]
    x = x.transpose(0, 1, 3, 2, 4).reshape(2, -1, H, D)[:, :ctx]
    return x, np.repeat(ok, bs)[:ctx]


def read(codes, exps, tables, lens, rows, starts=None):
    _, nb, H, bs, D = codes.shape
    out = np.zeros((2, rows, H * D))
    for b, first, n, ctx in spans(lens, starts, rows, tables.shape[1] * bs):
        x, ok = tokens(codes, exps, tables, b, ctx)
        x = np.where(ok[:, None, None], x, 0.0).reshape(2, ctx, H * D)
        take = min(n, ctx)
        if take:
            out[:, first + n - take:first + n] = x[:, ctx - take:]
    return out


def attention(q, codes, exps, tables, lens, starts=None, scale=None, weights=None):
    """(out, new weights, error bound of out, error bound of weights).  The
    bounds follow a 32-bit evaluation: a score off by at most
        ds = u * ((D + 16) * sum|q k| * scale + 8 * |s|) + 2^-21,  u = 2^-24,
    (the dot's roundings, the products by scale, log2 e and the maximum's
    subtraction; 2^-21 for the hardware's 2^x), weights then by ds of
    themselves on both sides of the quotient, and a sum over N tokens by
    (N + 16) u of its terms' magnitudes."""
    _, nb, H, bs, D = codes.shape
    rows, X = q.shape
    G = X // (H * D)
    u = 2.0 ** -24
    scale = 1 / np.sqrt(D) if scale is None else scale
    out, tol = np.zeros((rows, X)), np.zeros((rows, X))
    w = None if weights is None else weights.astype(np.float64)
    wtol = None if weights is None else np.abs(w) * 2 * u
    for b, first, n, ctx in spans(lens, starts, rows, tables.shape[1] * bs):
        x, ok = tokens(codes, exps, tables, b, ctx)
        for i in range(n):
            see = ctx - n + i + 1
            if see <= 0 or not ok[:see].any():
                continue
            at = np.flatnonzero(ok[:see])
            qr = q[first + i].astype(np.float64).reshape(H, G, D)
            kk, vv = x[0, at].transpose(1, 0, 2), x[1, at].transpose(1, 0, 2)
            s = qr @ kk.transpose(0, 2, 1) * scale
            mag = np.abs(qr) @ np.abs(kk).transpose(0, 2, 1) * abs(scale)
            ds = (u * ((D + 16) * mag + 8 * np.abs(s)) + 2.0 ** -21).max(-1, keepdims=True)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[first + i] = (p @ vv).reshape(-1)
            rel = 2 * ds + (2 * len(at) + 32) * u
            tol[first + i] = (rel * (p @ np.abs(vv))).reshape(-1)
            if w is not None:
                pe = np.zeros(-(-ctx // bs) * bs)
                pe[at] = p.sum((0, 1))
                w[b, :pe.size // bs] += pe.reshape(-1, bs).sum(1)
                te = np.zeros_like(pe)
                te[at] = (p * (rel + (n * H * G + bs) * u)).sum((0, 1))
                wtol[b, :pe.size // bs] += te.reshape(-1, bs).sum(1)
    return out, w, tol + 1e-37, wtol


def evict(tables, lens, weights, bs, budget, first, last):
    B, width = tables.shape
    t, e = np.full((B, width), -1, np.int32), np.full((B, width), -1, np.int32)
    w, n_out = np.zeros((B, width), np.float32), np.zeros(B, np.int32)
    for b in range(B):
        ctx = min(max(int(lens[b]), 0), width * bs)
        n = -(-ctx // bs)
        keep = list(range(n))
        if n > budget:
            key = [(-np.inf if np.isnan(x) else float(x), np.isnan(x)) for x in weights[b]]
            mid = sorted(range(first, n - last), key=lambda j: (-key[j][0], key[j][1], j))
            keep = sorted(list(range(first)) + list(range(n - last, n))
                          + mid[:budget - first - last])
        gone = sorted(set(range(n)) - set(keep))
        t[b, :len(keep)], w[b, :len(keep)] = tables[b, keep], weights[b, keep]
        e[b, :len(gone)] = tables[b, gone]
        n_out[b] = ctx - len(gone) * bs
    return t, n_out, w, e


def pool(g, lens, bs, width, spare=3):
    """Tables over a shuffled pool; -1 behind each sequence's blocks."""
    need = [-(-max(int(n), 0) // bs) for n in lens]
    ids = g.permutation(sum(need) + spare).astype(np.int32)
    t, at = np.full((len(lens), width), -1, np.int32), 0
    for b, n in enumerate(need):
        t[b, :n] = ids[at:at + n]
        at += n
    return t, sum(need) + spare


def cache(g, nb, H, bs, D):
    """A filled cache: normal data whose heads and blocks differ in size; all
    bytes but the NaN codes occur in real tiles, so slots behind a context hold
    what earlier sequences left."""
    codes = encode(g.standard_normal((2, nb, H, bs, D)) * 120)
    exps = g.integers(-9, -4, (2, nb, H)).astype(np.int32)
    return codes, exps


def starts_of(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
