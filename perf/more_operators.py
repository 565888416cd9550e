"""Linear layers in 8 bits and the norm before them, as cases to be timed: the
root-mean-square norm that adds the residual and writes 32 or 8 bits, its
gradient, the quantiser of activations, gradients and weights, and the matrix
product of two 8-bit operands with a scale for each block of 128.

``run`` computes a case in elementary torch operations where ``own`` is false
and through clove_amd's entry points where it is true.

The format: ``codes`` holds e4m3 bytes [rows, Kp], Kp being K rounded up to a
multiple of 128 (zeros behind K), and ``exps`` int32 [rows, Kp / 128] (a block is
128 elements of one row) or [ceil(rows / 128), Kp / 128] (a block is 128 rows by
128 elements); an element stands for its code times 2^exp.  A block has the
smallest exp in [-100, 119] with |x| <= 448 * 2^exp for all it holds.  A product
contracts the second axis of both operands.  Sizes are those of the repository's
configurations (4096-wide states and their products with 4096, 11008 and 14336,
blocks of 768 over 2 x 777 tokens, 2050 x 1028 x 3000) and generic ones.
"""
import math

import torch

own = False

DEV = "cuda"
MIN_EXP, MAX_EXP = -100, 119
EPS = 1e-5


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _norm(name, rows, cols, residual, out):
    c = dict(kind="norm", rows=rows, cols=cols, residual=residual, out=out)
    return dict(c, name=name) if name else c


def _grads(name, rows, cols, stream):
    c = dict(kind="grads", rows=rows, cols=cols, stream=stream)
    return dict(c, name=name) if name else c


def _quant(name, rows, cols, block_rows, ways):
    c = dict(kind="quant", rows=rows, cols=cols, block_rows=block_rows, ways=ways)
    return dict(c, name=name) if name else c


def _product(name, m, n, k, tiles, bias=False):
    c = dict(kind="product", m=m, n=n, k=k, tiles=tiles, bias=bias)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token between two layers of a decode step: launch latency
        _norm("norm_token", 1, 4096, True, "e4m3"),
        # the norm inside a block of a small model, in 32 bits
        _norm("norm_block", 1554, 768, True, "f32"),
        # the rows of long prompts on their way into an 8-bit product: memory
        _norm("norm_prompt", 8192, 4096, True, "e4m3"),
        # the same norm's gradient, with the gradient that the residual brings
        _grads("norm_grads", 8192, 4096, True),
        # a ragged batch of rows that are not whole vectors
        _grads("norm_grads_odd", 1001, 2049, False),
        # an output's gradient on its way into both products of a backward pass
        _quant("quant_grads", 2050, 3000, 1, "both"),
        # a weight matrix after its update, for the forward and the backward pass
        _quant("quant_weights", 4096, 14336, 128, "both"),
        # one token through a layer: latency, and the weights' bytes
        _product("product_token", 1, 4096, 4096, True),
        # a decode step's batch through a wide layer: the weights' bytes
        _product("product_decode", 32, 14336, 4096, True),
        # two sequences of 777 tokens into queries, keys and values, with the bias
        _product("product_block", 1554, 2304, 768, True, True),
        # a prompt through a square layer: bound by the matrix cores
        _product("product_prompt", 4096, 4096, 4096, True),
        # a weight's gradient: both operands transposed, blocks along the tokens
        _product("product_grads", 1028, 3000, 2050, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A size of any kind: as it comes, or a multiple of 16 or 128."""
    n, m = _log(rng, lo, hi), rng.choice([1, 1, 16, 128])
    return n if n < m else n // m * m


def draw(rng):
    kind = rng.choice(["norm", "norm", "grads", "quant", "quant", "product", "product", "product"])
    if kind == "product":
        thin = rng.random() < 0.45  # a decode step's rows
        m, n, k = _size(rng, 1, 64 if thin else 8192), _size(rng, 16, 16384), _size(rng, 16, 16384)
        while 2 * m * n * k > 130000000000 or n * k > 58000000:
            m, n, k = m if thin else -(-m * 3 // 4), -(-n * 3 // 4), -(-k * 3 // 4)
        return _product(None, m, n, k, rng.random() < 0.75, rng.random() < 0.3)
    cols = _size(rng, 16, 16384)
    most = 58000000 if kind == "quant" else 33000000
    rows = _size(rng, 1, max(1, min(32768, most // cols)))
    if kind == "norm":
        return _norm(None, rows, cols, rng.random() < 0.7, rng.choice(["f32", "e4m3"]))
    if kind == "grads":
        return _grads(None, rows, cols, rng.random() < 0.5)
    return _quant(None, rows, cols, rng.choice([1, 1, 128]),
                  rng.choice(["straight", "straight", "transposed", "both"]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _states(g, rows, cols):
    """Activations: tokens of different size, a few channels far stronger."""
    x = _normal(g, rows, cols)
    x[:, 7::61] *= 12.0
    return x.mul_(torch.exp2(torch.rand((rows, 1), generator=g, device=DEV) * 3 - 1))


def _gradients(g, rows, cols):
    """Gradients: small, and rows that differ by orders of magnitude."""
    return _normal(g, rows, cols).mul_(torch.exp(_normal(g, rows, 1) * 1.5 - 9))


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = case
    if c["kind"] == "quant":
        if c["block_rows"] == 1:
            return dict(x=_gradients(g, c["rows"], c["cols"]))
        return dict(x=_normal(g, c["rows"], c["cols"]).mul_(c["rows"] ** -0.5))
    if c["kind"] == "product":
        if c["tiles"]:  # states times weights
            a, b = _states(g, c["m"], c["k"]), _normal(g, c["n"], c["k"]).mul_(c["k"] ** -0.5)
        else:  # transposed states times transposed gradients
            a, b = (f(g, c["k"], w).t().contiguous()
                    for f, w in ((_states, c["m"]), (_gradients, c["n"])))
        d = {}
        d["a"], d["a_exps"] = _quantised(a, 1)
        d["b"], d["b_exps"] = _quantised(b, 128 if c["tiles"] else 1)
        if c["bias"]:
            d["bias"] = _normal(g, c["n"])
        return d
    d = dict(x=_states(g, c["rows"], c["cols"]),
             gamma=torch.rand(c["cols"], generator=g, device=DEV) + 0.5)
    if c["kind"] == "norm" and c["residual"]:
        d["residual"] = _states(g, c["rows"], c["cols"])
    if c["kind"] == "grads":
        d["grad"] = _gradients(g, c["rows"], c["cols"])
        if c["stream"]:
            d["grad_sum"] = _gradients(g, c["rows"], c["cols"])
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
                   for n, t in d.items()}
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    c, d = state["case"], state["d"]
    if own:
        return _OWN[c["kind"]](state["ca"], c, state["h"])
    return _PLAIN[c["kind"]](c, d)


def _up(n):
    return -(-n // 128) * 128


class _Memory:
    """One output tensor's memory, for torch to view; it keeps the tensor."""

    def __init__(self, t, shape, kind):
        self.t = t
        self.__cuda_array_interface__ = dict(shape=shape, typestr=kind, version=2,
                                             data=(t.device_ptr, False))


def _view(t, *shape):
    return torch.as_tensor(_Memory(t, shape, "<f4"), device=DEV)


def _view_codes(codes, exps, rows, cols, block_rows):
    """Codes as what they stand for beside their block's exponent."""
    kp = _up(cols)
    return dict(codes=torch.as_tensor(_Memory(codes, (rows, kp), "|u1"), device=DEV)
                .view(torch.float8_e4m3fn),
                exps=torch.as_tensor(_Memory(exps, (-(-rows // block_rows), kp // 128), "<i4"),
                                     device=DEV))


def _own_norm(ca, c, h):
    rows, cols = c["rows"], c["cols"]
    if c["out"] == "f32":
        o = ca.rms_norm(h["x"], h["gamma"], h.get("residual"), EPS)
        if not c["residual"]:
            return _view(o, rows, cols)
        return dict(out=_view(o[0], rows, cols), sum=_view(o[1], rows, cols))
    o = ca.rms_norm_e4m3(h["x"], h["gamma"], h.get("residual"), EPS)
    r = _view_codes(o[0], o[1], rows, cols, 1)
    return dict(r, sum=_view(o[2], rows, cols)) if c["residual"] else r


def _own_grads(ca, c, h):
    dx, dg = ca.rms_norm_backward(h["x"], h["gamma"], h["grad"], h.get("grad_sum"), EPS)
    return dict(x=_view(dx, c["rows"], c["cols"]), gamma=_view(dg, c["cols"]))


def _own_quant(ca, c, h):
    rows, cols, br, ways = c["rows"], c["cols"], c["block_rows"], c["ways"]
    o = ca.quantize_e4m3(h["x"], br, straight=ways != "transposed", transposed=ways != "straight")
    r = {}
    if ways != "transposed":
        r["straight"] = _view_codes(o[0], o[1], rows, cols, br)
    if ways != "straight":
        r["transposed"] = _view_codes(o[-2], o[-1], cols, rows, br)
    return r


def _own_product(ca, c, h):
    o = ca.matmul_e4m3(h["a"], h["a_exps"], h["b"], h["b_exps"], h.get("bias"))
    return _view(o, c["m"], c["n"])


_OWN = dict(norm=_own_norm, grads=_own_grads, quant=_own_quant, product=_own_product)


# ---- the plain form --------------------------------------------------------

def _two_to(e):
    """2^e in 32 bits, e int32 in [-126, 127]."""
    return ((e + 127) << 23).view(torch.float32)


def _blocks(x, block_rows):
    """x, zeros behind its edges, as [row blocks, block_rows, column blocks, 128]."""
    rows, cols = x.shape
    p = torch.zeros((-(-rows // block_rows) * block_rows, _up(cols)), dtype=x.dtype, device=x.device)
    p[:rows, :cols] = x
    return p.view(-1, block_rows, _up(cols) // 128, 128)


def _quantised(x, block_rows):
    """x [rows, cols] as e4m3 bytes [rows, Kp] and exponents."""
    p = _blocks(x, block_rows)
    amax = p.abs().amax((1, 3))
    mant, ex = torch.frexp(amax)  # 448 = 0.875 * 2^9
    e = ex - 9 + (mant > 0.875).int()
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)).clamp(MIN_EXP, MAX_EXP).int()
    codes = (p * _two_to(-e)[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.view(-1, _up(x.shape[1]))[:x.shape[0]].contiguous(), e


def _pair(x, block_rows):
    codes, exps = _quantised(x, block_rows)
    return dict(codes=codes.view(torch.float8_e4m3fn), exps=exps)


def _plain_norm(c, d):
    # in 64 bits: an 8-bit output's exponents and codes jump at borders
    h = d["x"] + d["residual"] if c["residual"] else d["x"]
    h64 = h.double()
    r = torch.rsqrt(h64.square().mean(-1, keepdim=True) + EPS)
    out = (h64 * r * d["gamma"].double()).float()
    if c["out"] == "f32":
        return dict(out=out, sum=h) if c["residual"] else out
    r = _pair(out, 1)
    return dict(r, sum=h) if c["residual"] else r


def _plain_grads(c, d):
    h, gy = d["x"], d["grad"]
    r = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    xhat = h * r
    t = gy * d["gamma"]
    dx = (t - xhat * (t * xhat).mean(-1, keepdim=True)) * r
    if c["stream"]:
        dx = dx + d["grad_sum"]
    return dict(x=dx, gamma=(gy * xhat).sum(0))


def _plain_quant(c, d):
    r = {}
    if c["ways"] != "transposed":
        r["straight"] = _pair(d["x"], c["block_rows"])
    if c["ways"] != "straight":
        r["transposed"] = _pair(d["x"].t(), c["block_rows"])
    return r


def _widened(codes, exps):
    v = codes.view(torch.float8_e4m3fn).float()
    scale = _two_to(exps)
    if exps.shape[0] < v.shape[0]:
        scale = scale.repeat_interleave(128, 0)[:v.shape[0]]
    return (v.view(v.shape[0], -1, 128) * scale[..., None]).view(v.shape)


def _plain_product(c, d):
    out = torch.matmul(_widened(d["a"], d["a_exps"]), _widened(d["b"], d["b_exps"]).t())
    return out + d["bias"] if c["bias"] else out


_PLAIN = dict(norm=_plain_norm, grads=_plain_grads, quant=_plain_quant, product=_plain_product)


# ---------------------------------------------------------------------------
# the work of one pass
# ---------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        kb = _up(k) // 128
        exps = 4 * kb * (m + (-(-n // 128) if c["tiles"] else n))
        return {"bytes": 128 * kb * (m + n) + exps + 4 * m * n + (4 * n if c["bias"] else 0),
                "flops": 2 * m * n * k}
    rows, cols = c["rows"], c["cols"]
    n = rows * cols
    held = rows * _up(cols) + rows * _up(cols) // 32  # codes, and an exponent for each 128
    if c["kind"] == "norm":
        out = held if c["out"] == "e4m3" else 4 * n
        return {"bytes": (12 if c["residual"] else 4) * n + out + 4 * cols, "flops": 6 * n}
    if c["kind"] == "grads":
        return {"bytes": (16 if c["stream"] else 12) * n + 8 * cols, "flops": 12 * n}
    got, br = 4 * n, c["block_rows"]
    if c["ways"] != "transposed":
        got += rows * _up(cols) + 4 * -(-rows // br) * (_up(cols) // 128)
    if c["ways"] != "straight":
        got += cols * _up(rows) + 4 * -(-cols // br) * (_up(rows) // 128)
    return {"bytes": got, "flops": 4 * n}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _power(e):
    return torch.exp2(e.double())


def _code_values(codes):
    """What e4m3 bytes stand for, from their fields."""
    c = codes.to(torch.int64)
    field, frac = (c >> 3) & 15, (c & 7).double()
    v = torch.where(field == 0, frac * 2.0 ** -9, (8 + frac) * _power(field - 10))
    return torch.where(c >= 128, -v, v)


def _to_e4m3(y):
    """|y| <= 448 rounded to the nearest e4m3 value, ties to even."""
    a = y.abs().clamp(min=2.0 ** -6)
    low = torch.floor(torch.log2(a))
    low = torch.where(_power(low) > a, low - 1, low)
    low = torch.where(_power(low + 1) <= a, low + 1, low)
    step = _power(low - 3)
    return torch.round(y / step) * step


def _exact_pair(x, block_rows):
    """The values of codes, and exponents, of x [rows, cols] in 64 bits."""
    rows, cols = x.shape
    codes = torch.zeros((rows, _up(cols)), dtype=torch.float64, device=x.device)
    exps = torch.empty((-(-rows // block_rows), _up(cols) // 128), dtype=torch.int32,
                       device=x.device)
    for j in range(exps.shape[1]):
        part = x[:, 128 * j:128 * (j + 1)]
        top = part.abs().amax(1)
        if block_rows > 1:
            tail = torch.zeros(exps.shape[0] * block_rows - rows, dtype=x.dtype, device=x.device)
            top = torch.cat([top, tail]).view(-1, block_rows).amax(1)
        e = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -200)))
        e = torch.where(448 * _power(e - 1) >= top, e - 1, e)
        e = torch.where(448 * _power(e) < top, e + 1, e)
        exps[:, j] = e.clamp(MIN_EXP, MAX_EXP).int()
        scale = _power(exps[:, j]).repeat_interleave(block_rows)[:rows, None]
        codes[:, 128 * j:128 * j + part.shape[1]] = _to_e4m3(part / scale)
    return dict(codes=codes, exps=exps)


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["kind"] == "quant":
        x, r = d["x"].double(), {}
        if c["ways"] != "transposed":
            r["straight"] = _exact_pair(x, c["block_rows"])
        if c["ways"] != "straight":
            r["transposed"] = _exact_pair(x.t(), c["block_rows"])
        return r
    if c["kind"] == "product":
        parts = []
        for n in ("a", "b"):
            v, e = _code_values(d[n]), d[n + "_exps"]
            row = torch.arange(v.shape[0], device=DEV)
            e = e[row] if e.shape[0] == v.shape[0] else e[row // 128]
            parts.append(v * _power(e).repeat_interleave(128, 1))
        out = parts[0] @ parts[1].t()
        return out + d["bias"].double() if c["bias"] else out
    gamma = d["gamma"].double()
    if c["kind"] == "grads":
        h, gy = d["x"].double(), d["grad"].double()
        n = (h * h).sum(-1, keepdim=True) / c["cols"] + EPS
        t = gy * gamma
        dx = t / n.sqrt() - h * (t * h).sum(-1, keepdim=True) / (c["cols"] * n * n.sqrt())
        if c["stream"]:
            dx = dx + d["grad_sum"].double()
        return dict(x=dx, gamma=(gy * h / n.sqrt()).sum(0))
    total = d["x"].double()
    if c["residual"]:
        total = total + d["residual"].double()
    h = total.float().double()  # the sum is kept, and normed, in 32 bits
    out = h / torch.sqrt((h * h).sum(-1, keepdim=True) / c["cols"] + EPS) * gamma
    if c["out"] == "f32":
        return dict(out=out, sum=total) if c["residual"] else out
    r = _exact_pair(out.float().double(), 1)  # the codes are those of the 32-bit norm
    return dict(r, sum=total) if c["residual"] else r
