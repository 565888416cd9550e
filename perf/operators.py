"""The paged KV cache in 8 bits and what serves from it, as cases to be timed:
the append that quantises, the read back, the attention over the cache (single
tokens and runs of tokens, grouped heads, with and without the attention
weight of each block) and the eviction of light blocks.

``run`` computes a case in elementary torch operations where ``own`` is false
and through clove_amd's entry points where it is true.

The cache: ``codes`` holds e4m3 bytes [2, num_blocks, heads, block, head_dim]
(keys, values), ``exps`` int32 [2, num_blocks, heads]; an element stands for
its code times 2^exp.  A tile (one block of one head) has the smallest exp in
[-60, 119] with amax <= 448 * 2^exp.  Sizes are those of the repository's
configurations (32 sequences of 512 to 4096 tokens, 32 heads of 128, 16-token
blocks, 4096-token prompts, 12 heads of 64) and generic ones around them.
"""
import math
import random

import torch

own = False

DEV = "cuda"
MIN_EXP, MAX_EXP = -60, 119


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _attention(name, seqs, rows, past, heads, kv_heads, head_dim, block, weights=False):
    c = dict(kind="attention", seqs=seqs, rows_lo=rows[0], rows_hi=rows[1], past_lo=past[0],
             past_hi=past[1], heads=heads, kv_heads=kv_heads, head_dim=head_dim, block=block,
             weights=weights)
    return dict(c, name=name) if name else c


def _append(name, seqs, rows, past, kv_heads, head_dim, block):
    c = dict(kind="append", seqs=seqs, rows_lo=rows[0], rows_hi=rows[1], past_lo=past[0],
             past_hi=past[1], kv_heads=kv_heads, head_dim=head_dim, block=block)
    return dict(c, name=name) if name else c


def _evict(name, seqs, ctx, block, budget, first, last):
    c = dict(kind="evict", seqs=seqs, ctx_lo=ctx[0], ctx_hi=ctx[1], block=block, budget=budget,
             first=first, last=last)
    return dict(c, name=name) if name else c


def listed():
    return [
        # every sequence of a decode batch stores the token it just made, and
        # its block is read back: launch latency and one partial tile a head
        _append("append_tokens", 32, (1, 1), (512, 4096), 8, 128, 16),
        # ragged prompts go into the cache behind what is there, and are read
        # back for a pass in 32 bits: bound by memory
        _append("append_prompts", 8, (200, 2048), (0, 100), 32, 128, 16),
        # one short conversation of a small model: the smallest decode call
        _attention("decode_one", 1, (1, 1), (100, 100), 12, 12, 64, 16),
        # a decode step of a full batch, a key head for every query head
        _attention("decode_batch", 32, (1, 1), (511, 4095), 32, 32, 128, 16),
        # a decode step of more and longer conversations, four query heads
        # to a key head
        _attention("decode_grouped", 64, (1, 1), (500, 8191), 32, 8, 128, 16),
        # one very long conversation, eight query heads to a key head, whose
        # blocks' weights are kept for eviction: few rows, a long axis
        _attention("decode_long", 1, (1, 1), (131000, 131000), 32, 4, 128, 32, True),
        # a decode step of a batch that keeps its blocks' weights
        _attention("decode_weighed", 24, (1, 1), (600, 3000), 16, 16, 96, 16, True),
        # speculated tokens, a few for each conversation, over what is cached
        _attention("speculate", 16, (2, 8), (300, 6000), 32, 8, 128, 16),
        # a whole prompt at once: bound by the matrix cores
        _attention("prompt", 1, (4096, 4096), (0, 0), 32, 32, 128, 16),
        # later chunks of ragged prompts with their blocks' weights
        _attention("prompt_chunks", 6, (1, 700), (0, 3000), 24, 8, 80, 32, True),
        # a few conversations give back what exceeds their budget
        _evict("evict_few", 8, (1000, 2048), 16, 64, 1, 4),
        # a large batch of long ones does
        _evict("evict_batch", 256, (20000, 65536), 16, 1024, 4, 16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    return rng.choice([(8, 8), (12, 12), (32, 32), (16, 16), (16, 8), (24, 8), (32, 8), (20, 4),
                       (28, 4), (32, 4), (8, 1), (16, 1)])


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "decode", "chunks", "chunks",
                       "evict"])
    block = rng.choice([8, 16, 16, 32, 64])
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 256])
    heads, kv_heads = _heads(rng)
    if kind == "append":
        seqs = _log(rng, 1, 32)
        per = 16000000 // (seqs * kv_heads * head_dim)
        rows_hi = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(4096, per)))
        past_hi = rng.choice([0, _log(rng, 1, 4096)])
        return _append(None, seqs, (rng.randint(1, rows_hi), rows_hi),
                       (rng.randint(0, past_hi), past_hi), kv_heads, head_dim, block)
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        past_hi = _log(rng, 16, min(65536, 400000000 // (2 * seqs * kv_heads * head_dim)))
        return _attention(None, seqs, (1, 1), (rng.randint(past_hi // 8, past_hi), past_hi),
                          heads, kv_heads, head_dim, block, rng.random() < 0.3)
    if kind == "chunks":
        seqs = rng.choice([1, 1, 2, 3, 6, 12])
        past_hi = 0 if rng.random() < 0.3 else _log(rng, 16, 6000)
        # the plain form holds every score of the padded batch at once
        scores = min(400000000, 60000000000 // (4 * head_dim)) // (seqs * heads)
        rows_hi = _log(rng, 2, 4000)
        while rows_hi > 2 and rows_hi * (rows_hi + past_hi) > scores:
            rows_hi = rows_hi * 3 // 4
        return _attention(None, seqs, (rng.randint(1, rows_hi), rows_hi),
                          (rng.randint(0, past_hi), past_hi), heads, kv_heads, head_dim, block,
                          rng.random() < 0.3)
    ctx_hi = _log(rng, 256, 65536)
    blocks = -(-ctx_hi // block)
    first, last = rng.randint(0, 4), rng.randint(1, 16)
    return _evict(None, _log(rng, 1, 256), (ctx_hi // 4, ctx_hi), block,
                  max(first + last, blocks // rng.randint(2, 16)), first, last)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _normal(g, shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _quantised(x):
    """Tiles [..., block, head_dim] as e4m3 bytes and exponents."""
    amax = x.abs().amax((-2, -1))
    exps = _exps_of(amax)
    codes = torch.ldexp(x, -exps[..., None, None]).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), exps


def _exps_of(amax):
    """The smallest e in [MIN_EXP, MAX_EXP] with amax <= 448 * 2^e."""
    mant, ex = torch.frexp(amax)  # 448 = 0.875 * 2^9
    e = ex - 9 + (mant > 0.875).int()
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP))
    return e.clamp(MIN_EXP, MAX_EXP).int()


def _lengths(case):
    """Each sequence's new rows and earlier tokens."""
    r = random.Random(17)
    return [(r.randint(case["rows_lo"], case["rows_hi"]), r.randint(case["past_lo"], case["past_hi"]))
            for _ in range(case["seqs"])]


def _starts(rows):
    s = [0]
    for n in rows:
        s.append(s[-1] + n)
    return s


def _tables(lens, block, width, seed):
    """Block tables over a pool a quarter larger than what is used, its blocks
    handed out in no order; -1 behind a sequence's blocks."""
    r = random.Random(seed + 1)
    need = [-(-n // block) for n in lens]
    pool = sum(need) + sum(need) // 4 + 1
    ids = list(range(pool))
    r.shuffle(ids)
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return table, pool


def _cache(g, pool, heads, block, dim):
    """A cache whose heads differ in magnitude, keys with a few strong channels."""
    codes = torch.empty((2, pool, heads, block, dim), dtype=torch.uint8, device=DEV)
    exps = torch.empty((2, pool, heads), dtype=torch.int32, device=DEV)
    for plane in range(2):
        size = torch.exp2(torch.rand((heads, 1, 1), generator=g, device=DEV) * 2 - 1)
        channel = torch.ones(dim, device=DEV)
        if plane == 0:
            channel[:: 29] = 3.0
        for at in range(0, pool, 16384):
            n = min(16384, pool - at)
            x = _normal(g, (n, heads, block, dim)).mul_(size).mul_(channel)
            codes[plane, at:at + n], exps[plane, at:at + n] = _quantised(x)
    return codes, exps


def _inputs(case, seed):
    """The case's tensors, and the lengths as the program's host side has them."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = case
    if c["kind"] == "evict":
        r = random.Random(seed)
        lens = [r.randint(c["ctx_lo"], c["ctx_hi"]) for _ in range(c["seqs"])]
        width = -(-c["ctx_hi"] // c["block"])
        table, _ = _tables(lens, c["block"], width, seed)
        # accumulated weights are heavy-tailed: few blocks hold most
        w = torch.exp(_normal(g, (c["seqs"], width)) * 2)
        return dict(tables=_ints(table), lens=_ints(lens), weights=w)
    lengths = _lengths(c)
    random.Random(seed).shuffle(lengths)  # which sequence has which
    rows, past = zip(*lengths)
    lens = [n + p for n, p in zip(rows, past)]
    width = -(-(c["rows_hi"] + c["past_hi"]) // c["block"])
    table, pool = _tables(lens, c["block"], width, seed)
    H, D = c["kv_heads"], c["head_dim"]
    codes, exps = _cache(g, pool, H, c["block"], D)
    d = dict(codes=codes, exps=exps, tables=_ints(table), lens=_ints(lens), host_rows=rows,
             host_past=past, host_table=table)
    if c["rows_hi"] > 1:
        d["starts"] = _ints(_starts(rows))
    if c["kind"] == "append":
        size = torch.exp2(torch.rand((1, H, 1), generator=g, device=DEV) * 2 - 1)
        for n in ("k", "v"):
            d[n] = _normal(g, (sum(rows), H, D)).mul_(size).view(sum(rows), H * D)
        # whole blocks are read back: the new rows and those before them in
        # the first block that is written
        back = [n + p % c["block"] for n, p in zip(rows, past)]
        d["host_back"] = back
        d["back_starts"] = _ints(_starts(back))
    else:
        d["q"] = _normal(g, (sum(rows), c["heads"] * D))
        if c["weights"]:  # of the steps before
            d["weights"] = torch.rand((c["seqs"], width), generator=g, device=DEV)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    st = dict(case=case, d=d)
    if own:
        import numpy as np

        import clove_amd as ca
        ca.init(0)
        kinds = {torch.float32: np.float32, torch.int32: np.int32, torch.uint8: np.uint8}
        torch.cuda.synchronize()  # the framework's stream does not wait for torch's
        st["ca"] = ca
        st["h"] = {n: ca.wrap(t.data_ptr(), tuple(t.shape), kinds[t.dtype])
                   for n, t in d.items() if isinstance(t, torch.Tensor)}
    elif case["kind"] != "evict":
        st["plan"] = _plan(case, d)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

class _Memory:
    """One output tensor's memory, for torch to view; it keeps the tensor."""

    def __init__(self, t, shape, kind):
        self.t = t
        self.__cuda_array_interface__ = dict(shape=shape, typestr=kind, version=2,
                                             data=(t.device_ptr, False))


def _view(t, shape, kind="<f4"):
    return torch.as_tensor(_Memory(t, tuple(shape), kind), device=DEV)


def run(state):
    c, d = state["case"], state["d"]
    if own:
        return _OWN[c["kind"]](state["ca"], c, d, state["h"])
    return _PLAIN[c["kind"]](c, d, state.get("plan"))


def _own_append(ca, c, d, h):
    ca.paged_kv8_append(h["codes"], h["exps"], h["k"], h["v"], h["tables"], h["lens"],
                        h.get("starts"))
    n, X = sum(d["host_back"]), c["kv_heads"] * c["head_dim"]
    k, v = ca.paged_kv8_read(h["codes"], h["exps"], h["tables"], h["lens"], h["back_starts"], n)
    return dict(k=_view(k, (n, X)), v=_view(v, (n, X)), exps=d["exps"])


def _own_attention(ca, c, d, h):
    o = ca.paged_kv8_attention(h["q"], h["codes"], h["exps"], h["tables"], h["lens"],
                               h.get("starts"), weights=h.get("weights"))
    if not c["weights"]:
        return _view(o, d["q"].shape)
    return dict(out=_view(o[0], d["q"].shape), weights=_view(o[1], d["weights"].shape))


def _own_evict(ca, c, d, h):
    t, n, w, e = ca.paged_evict(h["tables"], h["lens"], h["weights"], c["block"], c["budget"],
                                c["first"], c["last"])
    s = d["tables"].shape
    return dict(tables=_view(t, s, "<i4"), lens=_view(n, s[:1], "<i4"), weights=_view(w, s),
                evicted=_view(e, s, "<i4"))


_OWN = dict(append=_own_append, attention=_own_attention, evict=_own_evict)


# ---- the plain form --------------------------------------------------------

def _plan(c, d):
    """Where each row lies, as the program's host side knows it."""
    def places(rows, past):
        seq = [b for b, n in enumerate(rows) for _ in range(n)]
        pos = [p + i for n, p in zip(rows, past) for i in range(n)]
        return seq, pos

    def place_tensors(rows, past):
        seq, pos = places(rows, past)
        blk = [d["host_table"][b][p // c["block"]] for b, p in zip(seq, pos)]
        return [torch.tensor(x, device=DEV) for x in (seq, pos, blk, [p % c["block"] for p in pos])]

    rows, past = d["host_rows"], d["host_past"]
    if c["kind"] == "append":
        seq, pos = places(rows, past)
        tiles = {}
        row_tile = [tiles.setdefault((b, p // c["block"]), len(tiles)) for b, p in zip(seq, pos)]
        low = [past[b] - j * c["block"] if j * c["block"] < past[b] else 0 for b, j in tiles]
        blk = [d["host_table"][b][j] for b, j in tiles]
        back = d["host_back"]
        return dict(row_tile=torch.tensor(row_tile, device=DEV),
                    tile_low=torch.tensor(low, device=DEV), tile_blk=torch.tensor(blk, device=DEV),
                    rows=place_tensors(rows, past),
                    back=place_tensors(back, [p + n - m for p, n, m in zip(past, rows, back)]))
    seq, pos = places(rows, past)
    pad = torch.full((c["seqs"], max(rows)), sum(rows), dtype=torch.long)
    at = 0
    for b, n in enumerate(rows):
        pad[b, :n] = torch.arange(at, at + n)
        at += n
    local = [i for n in rows for i in range(n)]
    return dict(pad=pad.to(DEV), seq=torch.tensor(seq, device=DEV),
                local=torch.tensor(local, device=DEV), rows=torch.tensor(rows, device=DEV))


def _values(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _plain_append(c, d, plan):
    H, D = c["kv_heads"], c["head_dim"]
    low, blk = plan["tile_low"], plan["tile_blk"]
    _, _, row_blk, row_slot = plan["rows"]
    slots = torch.arange(c["block"], device=DEV)
    for plane, x in enumerate((d["k"], d["v"])):
        codes, exps = d["codes"][plane], d["exps"][plane]
        x = x.view(-1, H, D)
        amax = torch.zeros((low.numel(), H), device=DEV)
        amax.scatter_reduce_(0, plan["row_tile"][:, None].expand(-1, H), x.abs().amax(-1), "amax")
        e = _exps_of(amax)
        before = exps[blk]
        e = torch.where(low[:, None] > 0, torch.maximum(e, before), e)
        # what a tile held before its new rows, under its new exponent
        tile = _values(codes[blk])
        again = torch.ldexp(tile, (before - e)[..., None, None]).to(torch.float8_e4m3fn)
        old = (slots[None, :] < low[:, None])[:, None, :, None]
        codes[blk] = torch.where(old, again.view(torch.uint8), codes[blk])
        exps[blk] = e
        new = torch.ldexp(x, -e[plan["row_tile"]][..., None]).to(torch.float8_e4m3fn)
        codes[row_blk, :, row_slot] = new.view(torch.uint8)
    _, _, blk, slot = plan["back"]
    got = [torch.ldexp(_values(d["codes"][p][blk, :, slot]), d["exps"][p][blk][..., None])
           .view(-1, H * D) for p in range(2)]
    return dict(k=got[0], v=got[1], exps=d["exps"])


def _plain_attention(c, d, plan):
    B, H, D, bs = c["seqs"], c["kv_heads"], c["head_dim"], c["block"]
    G = c["heads"] // H
    tables = d["tables"].clamp(min=0).long()
    width = tables.shape[1]

    def plane(p):
        x = torch.ldexp(_values(d["codes"][p][tables]), d["exps"][p][tables][..., None, None])
        return x.permute(0, 2, 1, 3, 4).reshape(B, H, width * bs, D)

    q = torch.cat([d["q"], torch.zeros_like(d["q"][:1])])[plan["pad"]]  # [B, n, Hq*D]
    n = q.shape[1]
    q = q.view(B, n, H, G, D).transpose(1, 2).reshape(B, H, n * G, D)
    s = torch.matmul(q, plane(0).transpose(2, 3)) * (1.0 / math.sqrt(D))
    pos = (d["lens"] - plan["rows"])[:, None] + torch.arange(n, device=DEV)
    sees = torch.arange(width * bs, device=DEV) <= pos[..., None]
    sees = sees & (torch.arange(n, device=DEV) < plan["rows"][:, None])[..., None]
    s = s.view(B, H, n, G, -1).masked_fill_(~sees[:, None, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, torch.ones_like(total), total))
    o = torch.matmul(p.view(B, H, n * G, -1), plane(1))
    o = o.view(B, H, n, G, D).transpose(1, 2).reshape(B, n, H * G * D)
    o = o[plan["seq"], plan["local"]]
    if not c["weights"]:
        return o
    return dict(out=o, weights=d["weights"] + p.sum((1, 2, 3)).view(B, width, bs).sum(-1))


def _plain_evict(c, d, _):
    tables, lens, w = d["tables"], d["lens"], d["weights"]
    B, width = tables.shape
    blocks = (lens + c["block"] - 1) // c["block"]
    j = torch.arange(width, device=DEV).expand(B, width)
    held = j < blocks[:, None]
    must = (j < c["first"]) | (j >= blocks[:, None] - c["last"])
    key = torch.where(must, torch.full_like(w, math.inf), w)
    key = torch.where(held, key, torch.full_like(w, -math.inf))
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(1, order, j.contiguous())
    keep = held & (rank < c["budget"])
    gone = held & ~keep

    def packed(x, which, rest):
        to = torch.where(which, which.cumsum(1) - 1, torch.full_like(j, width))
        out = torch.full((B, width + 1), rest, dtype=x.dtype, device=DEV)
        return out.scatter_(1, to, x)[:, :width].contiguous()

    return dict(tables=packed(tables, keep, -1),
                lens=(lens - gone.sum(1) * c["block"]).int(),
                weights=packed(w, keep, 0.0), evicted=packed(tables, gone, -1))


_PLAIN = dict(append=_plain_append, attention=_plain_attention, evict=_plain_evict)


# ---------------------------------------------------------------------------
# the work of one pass
# ---------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "evict":
        n = c["seqs"] * -(-c["ctx_hi"] // c["block"])
        # table and weights in; tables, weights and the evicted blocks out
        return {"bytes": 20 * n + 8 * c["seqs"], "flops": 8 * n}
    H, D, bs = c["kv_heads"], c["head_dim"], c["block"]
    lengths = _lengths(c)
    if c["kind"] == "append":
        # rows in at 32 bits, out at 8; the same backwards for what is read
        rows = sum(n for n, _ in lengths)
        back = rows + sum(p % bs for _, p in lengths)
        tiles = sum(-(-(p % bs + n) // bs) for n, p in lengths)
        return {"bytes": 10 * H * D * (rows + back) + 16 * H * tiles,
                "flops": 8 * H * D * (rows + back)}
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in lengths)
    ctx = sum(n + p for n, p in lengths)
    blocks = sum(-(-(n + p) // bs) for n, p in lengths)
    got = 2 * H * D * ctx + (8 * H + 4) * blocks + 8 * sum(n for n, _ in lengths) * c["heads"] * D
    if c["weights"]:
        got += 8 * blocks
    return {"bytes": got, "flops": 4 * D * c["heads"] * pairs}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _code_values(codes):
    """What e4m3 bytes stand for, from their fields."""
    c = codes.to(torch.int64)
    field, frac = (c >> 3) & 15, (c & 7).double()
    v = torch.where(field == 0, frac * 2.0 ** -9, (8 + frac) * torch.exp2(field.double() - 10))
    return torch.where(c >= 128, -v, v)


def _to_e4m3(y):
    """|y| <= 448 rounded to the nearest e4m3 value, ties to even."""
    a = y.abs().clamp(min=2.0 ** -6)
    low = torch.floor(torch.log2(a))
    low = torch.where(torch.exp2(low) > a, low - 1, low)
    low = torch.where(torch.exp2(low + 1) <= a, low + 1, low)
    step = torch.exp2(low - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    d = _inputs(case, seed)
    return _EXACT[case["kind"]](case, d)


def _exact_append(c, d):
    H, D, bs = c["kv_heads"], c["head_dim"], c["block"]
    outs, exps = [], d["exps"].clone()
    for plane, x in enumerate((d["k"], d["v"])):
        x = x.double().view(-1, H, D)
        parts, at = [], 0
        for b, (n, past) in enumerate(zip(d["host_rows"], d["host_past"])):
            mine, at = x[at:at + n], at + n
            done = 0
            while done < n:
                j, low = divmod(past + done, bs)
                new = mine[done:done + bs - low]
                done += new.shape[0]
                blk = d["host_table"][b][j]
                top = new.abs().amax((0, 2)) / 448
                e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -1000)))
                e = torch.where(torch.exp2(e - 1) >= top, e - 1, e)
                e = torch.where(torch.exp2(e) < top, e + 1, e)
                e = e.clamp(MIN_EXP, MAX_EXP)
                if low:
                    was = exps[plane, blk].double()
                    e = torch.maximum(e, was)
                    kept = _code_values(d["codes"][plane, blk, :, :low])
                    kept = _to_e4m3(kept * torch.exp2(was - e)[:, None, None])
                    parts.append((kept * torch.exp2(e)[:, None, None]).transpose(0, 1))
                exps[plane, blk] = e.int()
                e = e[None, :, None]
                parts.append(_to_e4m3(new * torch.exp2(-e)) * torch.exp2(e))
        outs.append(torch.cat(parts).reshape(-1, H * D))
    return dict(k=outs[0], v=outs[1], exps=exps)


def _exact_attention(c, d):
    H, D, bs = c["kv_heads"], c["head_dim"], c["block"]
    G = c["heads"] // H
    q = d["q"].double().view(-1, H, G, D)
    out = torch.zeros_like(q)
    w = d["weights"].double() if c["weights"] else None
    at = 0
    for b, (n, past) in enumerate(zip(d["host_rows"], d["host_past"])):
        ctx = past + n
        blocks = torch.tensor(d["host_table"][b][:-(-ctx // bs)], device=DEV)
        for h in range(H):
            k, v = ((_code_values(d["codes"][p, blocks, h])
                     * torch.exp2(d["exps"][p, blocks, h].double())[:, None, None])
                    .reshape(-1, D)[:ctx] for p in range(2))
            for i in range(0, n, 512):
                part = q[at + i:at + min(n, i + 512), h]
                s = part.reshape(-1, D) @ k.t() / math.sqrt(D)
                pos = past + i + torch.arange(part.shape[0], device=DEV).repeat_interleave(G)
                s[torch.arange(ctx, device=DEV)[None] > pos[:, None]] = -math.inf
                p = torch.softmax(s, -1)
                out[at + i:at + i + part.shape[0], h] = (p @ v).view(-1, G, D)
                if w is not None:
                    sums = torch.zeros(blocks.numel() * bs, dtype=torch.float64, device=DEV)
                    sums[:ctx] = p.sum(0)
                    w[b, :blocks.numel()] += sums.view(-1, bs).sum(1)
        at += n
    out = out.view(-1, c["heads"] * D)
    return dict(out=out, weights=w) if c["weights"] else out


def _exact_evict(c, d):
    tables, lens, w = d["tables"].tolist(), d["lens"].tolist(), d["weights"].double().tolist()
    width = len(tables[0])
    got = dict(tables=[], lens=[], weights=[], evicted=[])
    for table, ctx, row in zip(tables, lens, w):
        n = -(-ctx // c["block"])
        must = [j for j in range(n) if j < c["first"] or j >= n - c["last"]]
        if n <= c["budget"]:
            keep = list(range(n))
        else:
            rest = sorted((j for j in range(c["first"], n - c["last"])), key=lambda j: (-row[j], j))
            keep = sorted(must + rest[:c["budget"] - len(must)])
        kept = set(keep)
        gone = [j for j in range(n) if j not in kept]
        got["tables"].append([table[j] for j in keep] + [-1] * (width - len(keep)))
        got["weights"].append([row[j] for j in keep] + [0.0] * (width - len(keep)))
        got["evicted"].append([table[j] for j in gone] + [-1] * (width - len(gone)))
        got["lens"].append(ctx - len(gone) * c["block"])
    out = {n: _ints(got[n]) for n in ("tables", "lens", "evicted")}
    return dict(out, weights=torch.tensor(got["weights"], dtype=torch.float64, device=DEV))


_EXACT = dict(append=_exact_append, attention=_exact_attention, evict=_exact_evict)
