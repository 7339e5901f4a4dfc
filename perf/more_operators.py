"""The operators of 8-bit language-model layers and how they are measured.

A transformer's products in 8-bit floating point (e4m3), a scale for each block
of 128 numbers, and what stands before them: the root-mean-square norm with the
residual's addition (``rms_norm``, differentiable), the same with its output in
8 bits (``rms_norm_quantized``), the quantising of activations and weights
(``quantize_rows``, ``quantize_tiles``), the product (``block_matmul``) and the
trainable layer made of them (``block_linear``).

``listed()`` names twelve calls, ``draw(rng)`` gives more of the same ranges,
``prepare`` makes what a program holds before the call, ``run`` is one pass:
the plain form from elementary torch operations in 32 bits, or, where ``own``
is true, the framework's operators.  ``work`` counts what a call cannot do
without, and ``exact`` is the definition in 64 bits.

An e4m3 number is returned as itself beside its block's scale; its exact value
is the quotient that it was rounded from.  A matrix comes in the layout that
the framework's quantisers give it.
"""

import math
import os
import sys

import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(REPO, "nl2cuda-kernel-agent_amd")
if PACKAGE not in sys.path:
    sys.path.insert(1, PACKAGE)

own = False

DEVICE = "cuda:0"
EPS = 1e-6
BLOCK = 128                    # numbers that share a scale, or the side of a tile that does
TOP = 448.0                    # largest e4m3 number
LEAST = 2.0 ** -126            # smallest scale
CODES = torch.float8_e4m3fn
SCALES = {"float32": torch.float32, "power2": torch.float8_e8m0fnu}

MAX_NORM = 1 << 25             # elements of the largest norm and of the largest matrix quantised
MAX_FLOPS = 2 * 8192 ** 3      # of the largest product


def listed():
    return [
        # One sequence decodes: the norm ahead of a layer, for one token; latency counts.
        {"name": "norm_quant_1x4096", "op": "rms_norm_quantized", "rows": 1, "d": 4096,
         "dtype": "bfloat16", "residual": True, "scale": "power2"},
        # A long prompt through the same.
        {"name": "norm_quant_8192x4096", "op": "rms_norm_quantized", "rows": 8192, "d": 4096,
         "dtype": "bfloat16", "residual": True, "scale": "float32"},
        # A training step's norm, forward and backward, the residual stream going on.
        {"name": "norm_train_4096x2048", "op": "rms_norm", "rows": 4096, "d": 2048,
         "dtype": "bfloat16", "residual": True},
        # The same in 32 bits, without a residual, of an odd width.
        {"name": "norm_train_999x5121", "op": "rms_norm", "rows": 999, "d": 5121,
         "dtype": "float32", "residual": False},
        # Activations for the forward and, transposed, for the weights' gradient.
        {"name": "quant_rows_4096x4096", "op": "quantize_rows", "rows": 4096, "d": 4096,
         "dtype": "bfloat16", "scale": "power2", "transposed": True},
        # A 32-bit master weight for both directions, after an update.
        {"name": "quant_tiles_8192x2048", "op": "quantize_tiles", "rows": 8192, "d": 2048,
         "dtype": "float32", "scale": "float32", "transposed": True},
        # One token times a projection: the weight is read once.
        {"name": "matmul_1x8192x4096", "op": "block_matmul", "m": 1, "n": 8192, "k": 4096,
         "scale": "float32", "out": "bfloat16"},
        # As many sequences decode together, from a wide layer back to the narrow one.
        {"name": "matmul_37x4096x14336", "op": "block_matmul", "m": 37, "n": 4096, "k": 14336,
         "scale": "power2", "out": "bfloat16"},
        # A prompt through a square projection, with 32-bit scales.
        {"name": "matmul_4096x4096x4096", "op": "block_matmul", "m": 4096, "n": 4096, "k": 4096,
         "scale": "float32", "out": "bfloat16"},
        # The largest product.
        {"name": "matmul_8192x8192x8192", "op": "block_matmul", "m": 8192, "n": 8192, "k": 8192,
         "scale": "power2", "out": "bfloat16"},
        # A layer's training step: quantised activations, weights and gradients, three products.
        {"name": "linear_4096x4096x2048", "op": "block_linear", "m": 4096, "n": 4096, "k": 2048,
         "dtype": "bfloat16", "weight": "bfloat16", "scale": "power2"},
        # The same of odd sizes, a 32-bit weight and 32-bit scales.
        {"name": "linear_1000x1111x2050", "op": "block_linear", "m": 1000, "n": 1111, "k": 2050,
         "dtype": "bfloat16", "weight": "float32", "scale": "float32"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm uniform."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _side(rng, lo, hi):
    """A matrix's side: half of them multiples of 64."""
    n = _log(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["rms_norm", "rms_norm_quantized", "quantize_rows", "quantize_tiles",
                     "block_matmul", "block_matmul", "block_linear"])
    scale = rng.choice(["float32", "power2"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    while True:
        if op in ("block_matmul", "block_linear"):
            m, n, k = _log(rng, 1, 8192), _side(rng, 64, 16384), _side(rng, 64, 16384)
            case = {"op": op, "m": m, "n": n, "k": k, "scale": scale}
            if op == "block_matmul":
                case["out"] = rng.choice(["bfloat16", "bfloat16", "float32"])
            else:
                case.update(dtype=rng.choice(["bfloat16", "bfloat16", "float32"]),
                            weight=rng.choice(["bfloat16", "float32"]))
            if max(m, n) * k <= MAX_NORM and work(case)["flops"] <= MAX_FLOPS:
                return case
            continue
        rows, d = _log(rng, 1, 16384), _side(rng, 64, 16384)
        if rows * d > MAX_NORM:
            continue
        case = {"op": op, "rows": rows, "d": d, "dtype": dtype}
        if op.startswith("rms_norm"):
            case["residual"] = rng.random() < 0.6
        if op != "rms_norm":
            case["scale"] = scale
        if op.startswith("quantize"):
            case["transposed"] = rng.random() < 0.6
        return case


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _hidden(g, rows, d):
    """Hidden states: channels of different sizes, a few far larger."""
    size = torch.exp(0.5 * _randn(g, d))
    size = torch.where(torch.rand(d, generator=g, device=DEVICE) < 0.004, 20 * size, size)
    return _randn(g, rows, d) * size


def _e4m3(g, rows, d, tiles, scale):
    """A matrix in 8 bits as the framework's quantisers lay it out: rows padded to 16 bytes; of
    rows' scales those of one block next to each other."""
    x = _randn(g, rows, d) * torch.exp(0.3 * _randn(g, rows, 1))
    q, s = _quantized(x, tiles, scale)
    codes = torch.zeros(rows, (d + 15) // 16 * 16, dtype=torch.uint8, device=DEVICE)
    codes[:, :d] = q.view(torch.uint8)
    s = s.view(torch.uint8) if scale == "power2" else s
    s = s if tiles else s.t().contiguous().t()
    return codes.view(CODES)[:, :d], s.view(SCALES[scale])


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    state = {"op": op, "case": case}
    if op.startswith("rms_norm"):
        rows, d, dtype = case["rows"], case["d"], getattr(torch, case["dtype"])
        state["x"] = _hidden(g, rows, d).to(dtype)
        state["residual"] = (2 * _hidden(g, rows, d)).to(dtype) if case["residual"] else None
        state["weight"] = (1 + 0.1 * _randn(g, d)).to(dtype)
        if op == "rms_norm":
            state["dy"] = (_randn(g, rows, d) * torch.exp(_randn(g, rows, 1))).to(dtype)
            state["dh"] = _randn(g, rows, d).to(dtype) if case["residual"] else None
            for t in ("x", "residual", "weight"):
                if state[t] is not None:
                    state[t].requires_grad_(True)
        return state
    if op.startswith("quantize"):
        x = _hidden(g, case["rows"], case["d"])
        if op == "quantize_tiles":
            x = 0.02 * x
        state["x"] = x.to(getattr(torch, case["dtype"]))
        return state
    m, n, k = case["m"], case["n"], case["k"]
    if op == "block_matmul":
        state["a"] = _e4m3(g, m, k, False, case["scale"])
        state["b"] = _e4m3(g, n, k, True, case["scale"])
        return state
    dtype = getattr(torch, case["dtype"])
    state["x"] = _hidden(g, m, k).to(dtype).requires_grad_(True)
    state["weight"] = (_randn(g, n, k) / math.sqrt(k)).to(getattr(torch, case["weight"]))
    state["weight"].requires_grad_(True)
    state["dy"] = (1e-4 * _randn(g, m, n) * torch.exp(_randn(g, m, 1))).to(dtype)
    return state


# -------------------------------------------------------------- plain forms
def _blocks(x, tiles):
    """x [m, k] as [m', p, k', 128], zeros past its ends; p is 128 where tiles share a scale."""
    m, k = x.shape
    p = BLOCK if tiles else 1
    x = torch.nn.functional.pad(x, (0, -k % BLOCK, 0, -m % p))
    return x.reshape(x.shape[0] // p, p, x.shape[1] // BLOCK, BLOCK)


def _quantized(x, tiles, scale):
    """(codes [m, k], scales) of x [m, k] in 32 bits.  Next to a border of the rounding of scales
    32 bits do not do: those are formed in 64 and rounded once."""
    m, k = x.shape
    b = _blocks(x, tiles)
    least = b.abs().amax((1, 3)).double() / TOP
    if scale == "power2":
        f, e = torch.frexp(least)
        s = torch.ldexp(torch.ones_like(least), torch.where(f == 0.5, e - 1, e)).clamp(min=LEAST)
    else:
        s = least.clamp(min=LEAST)
    s = s.float()
    inverse = (1.0 / s.double()).float()
    q = (b * inverse[:, None, :, None]).reshape(b.shape[0] * b.shape[1], -1)[:m, :k]
    return q.to(CODES).contiguous(), s.to(SCALES[scale])


def _values(codes, scales, tiles):
    """The numbers that codes and scales stand for, in 32 bits."""
    m, k = codes.shape
    b = _blocks(codes.float(), tiles) * scales.float()[:, None, :, None]
    return b.reshape(b.shape[0] * b.shape[1], -1)[:m, :k]


def _through(x, tiles, scale):
    """x as 8 bits hold it."""
    return _values(*_quantized(x, tiles, scale), tiles)


def _norm_plain(st):
    """(h, h in 32 bits, 1 / rms, y in 32 bits); the sum is h's type's, as all that follows reads
    it."""
    x = st["x"].detach().float()
    if st["residual"] is not None:
        h = (x + st["residual"].detach().float()).to(st["residual"].dtype)
        x = h.float()
    else:
        h = None
    rstd = 1.0 / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)
    return h, x, rstd, x * rstd * st["weight"].detach().float()


def _plain(st):
    op, case = st["op"], st["case"]
    if op == "rms_norm":
        h, x, rstd, y = _norm_plain(st)
        dy, u = st["dy"].float(), x * rstd
        g = dy * st["weight"].detach().float()
        dx = rstd * (g - u * ((g * u).sum(-1, keepdim=True) / x.shape[-1]))
        dw = (dy * u).sum(0).to(st["weight"].dtype)
        y = y.to(st["x"].dtype)
        if h is None:
            return {"y": y, "dx": dx.to(st["x"].dtype), "dw": dw}
        dx = dx + st["dh"].float()
        return {"y": y, "h": h, "dx": dx.to(st["x"].dtype), "dw": dw,
                "dresidual": dx.to(st["residual"].dtype)}
    if op == "rms_norm_quantized":
        h, _, _, y = _norm_plain(st)
        codes, scales = _quantized(y, False, case["scale"])
        return {"codes": codes, "scales": scales, "h": h}
    if op.startswith("quantize"):
        tiles, x = op == "quantize_tiles", st["x"].float()
        codes, scales = _quantized(x, tiles, case["scale"])
        got = {"codes": codes, "scales": scales}
        if case["transposed"]:
            if tiles:
                got["codes_t"] = codes.t().contiguous()
            else:
                got["codes_t"], got["scales_t"] = _quantized(x.t(), False, case["scale"])
        return got
    if op == "block_matmul":
        a, b = _values(*st["a"], False), _values(*st["b"], True)
        return (a @ b.t()).to(getattr(torch, case["out"]))
    x, w, dy, scale = st["x"].detach().float(), st["weight"].detach().float(), st["dy"].float(), \
        case["scale"]
    wq = _through(w, True, scale)
    y = _through(x, False, scale) @ wq.t()
    dx = _through(dy, False, scale) @ wq
    dw = _through(dy.t(), False, scale) @ _through(x.t(), False, scale).t()
    return {"y": y.to(st["x"].dtype), "dx": dx.to(st["x"].dtype), "dw": dw.to(st["weight"].dtype)}


# ---------------------------------------------------------------------- run
def _framework(st):
    op, case = st["op"], st["case"]
    if op == "rms_norm":
        from cases.rms_norm.op import rms_norm
        if st["residual"] is None:
            y = rms_norm(st["x"], st["weight"], eps=EPS)
            dx, dw = torch.autograd.grad(y, (st["x"], st["weight"]), st["dy"])
            return {"y": y.detach(), "dx": dx, "dw": dw}
        y, h = rms_norm(st["x"], st["weight"], st["residual"], eps=EPS)
        dx, dr, dw = torch.autograd.grad((y, h), (st["x"], st["residual"], st["weight"]),
                                         (st["dy"], st["dh"]))
        return {"y": y.detach(), "h": h.detach(), "dx": dx, "dresidual": dr, "dw": dw}
    if op == "rms_norm_quantized":
        from cases.rms_norm.op import rms_norm_quantized
        got = rms_norm_quantized(st["x"], st["weight"], st["residual"], eps=EPS,
                                 scale_dtype=SCALES[case["scale"]])
        return {"codes": got[0], "scales": got[1], "h": got[2] if len(got) > 2 else None}
    if op.startswith("quantize"):
        from cases.block_quant.op import quantize_rows, quantize_tiles
        call = quantize_tiles if op == "quantize_tiles" else quantize_rows
        got = call(st["x"], scale_dtype=SCALES[case["scale"]], transposed=case["transposed"])
        return dict(zip(("codes", "scales", "codes_t", "scales_t"),
                        got[:3] if op == "quantize_tiles" else got))
    if op == "block_matmul":
        from cases.block_matmul.op import block_matmul
        return block_matmul(*st["a"], *st["b"], out_dtype=getattr(torch, case["out"]))
    from cases.block_matmul.op import block_linear
    y = block_linear(st["x"], st["weight"], scale_dtype=SCALES[case["scale"]])
    dx, dw = torch.autograd.grad(y, (st["x"], st["weight"]), st["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


def run(state):
    if own:
        return _framework(state)
    with torch.no_grad():
        return _plain(state)


# --------------------------------------------------------------------- work
def _bytes_of(name):
    return torch.empty((), dtype=getattr(torch, name)).element_size()


def _scale_bytes(rows, d, scale):
    return rows * -(-d // BLOCK) * (1 if scale == "power2" else 4)


def work(case):
    """Each input read once, each output written once."""
    op = case["op"]
    if op in ("block_matmul", "block_linear"):
        m, n, k = case["m"], case["n"], case["k"]
        if op == "block_linear":
            e, w = _bytes_of(case["dtype"]), _bytes_of(case["weight"])
            return {"bytes": 2 * m * k * e + 2 * m * n * e + 2 * n * k * w, "flops": 6 * m * n * k}
        scales = _scale_bytes(m, k, case["scale"]) + _scale_bytes(-(-n // BLOCK), k, case["scale"])
        return {"bytes": (m + n) * k + scales + m * n * _bytes_of(case["out"]),
                "flops": 2 * m * n * k}
    rows, d, e = case["rows"], case["d"], _bytes_of(case["dtype"])
    if op == "rms_norm":
        # x, dy read, y, dx written; with a residual it and dh read, h and its gradient written
        return {"bytes": rows * d * e * (8 if case["residual"] else 4) + 2 * d * e,
                "flops": rows * d * 14}
    if op == "rms_norm_quantized":
        return {"bytes": rows * d * (1 + e * (3 if case["residual"] else 1)) + d * e
                + _scale_bytes(rows, d, case["scale"]), "flops": rows * d * 8}
    both = 2 if case["transposed"] else 1
    if op == "quantize_tiles":
        scales = _scale_bytes(-(-rows // BLOCK), d, case["scale"])
    else:
        scales = _scale_bytes(rows, d, case["scale"])
        if both == 2:
            scales += _scale_bytes(d, rows, case["scale"])
    return {"bytes": rows * d * (e + both) + scales, "flops": 3 * both * rows * d}


# -------------------------------------------------------------------- exact
def _scales_exact(x, tiles, scale):
    """A scale for every number of x [m, k] in 64 bits, and the scales themselves."""
    m, k = x.shape
    p = BLOCK if tiles else 1
    rows, cols = -(-m // p), -(-k // BLOCK)
    r, c = torch.arange(m, device=x.device) // p, torch.arange(k, device=x.device) // BLOCK
    top = torch.zeros(m, cols, dtype=x.dtype, device=x.device)
    top = top.scatter_reduce(1, c.expand(m, k), x.abs(), "amax")
    if tiles:
        top = torch.zeros(rows, cols, dtype=x.dtype, device=x.device).scatter_reduce(
            0, r[:, None].expand(m, cols), top, "amax")
    s = torch.maximum(top / TOP, torch.full_like(top, LEAST))
    if scale == "power2":
        # the exponent by halves of a step: a quotient that is a power of two is one exactly
        e = torch.round(torch.log2(s))
        s = torch.where(torch.exp2(e) >= s, torch.exp2(e), torch.exp2(e + 1))
    return s[r][:, c], s


def _rounded_exact(x, tiles, scale):
    """x as 8 bits hold it, in 64: scales and what a number is multiplied by to be rounded are 32-bit
    numbers."""
    each = _scales_exact(x, tiles, scale)[0].float().double()
    return (x * (1.0 / each).float().double()).float().to(CODES).double() * each


def exact(case, seed):
    st = prepare(case, seed)
    op, scale = st["op"], case.get("scale")
    if op.startswith("rms_norm"):
        h = None
        x = st["x"].detach().double()
        if st["residual"] is not None:
            h = x + st["residual"].detach().double()
            x = h.to(st["residual"].dtype).double()
        if op == "rms_norm_quantized":
            y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * st["weight"].double()
            each, s = _scales_exact(y, False, scale)
            return {"codes": y / each, "scales": s, "h": h}
        x.requires_grad_(True)
        w = st["weight"].detach().double().requires_grad_(True)
        y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w
        dx, dw = torch.autograd.grad(y, (x, w), st["dy"].double())
        if h is None:
            return {"y": y.detach(), "dx": dx, "dw": dw}
        dx = dx + st["dh"].double()
        return {"y": y.detach(), "h": h, "dx": dx, "dresidual": dx, "dw": dw}
    if op.startswith("quantize"):
        tiles, x = op == "quantize_tiles", st["x"].double()
        each, s = _scales_exact(x, tiles, scale)
        got = {"codes": x / each, "scales": s}
        if case["transposed"]:
            if tiles:
                got["codes_t"] = (x / each).t()
            else:
                each, got["scales_t"] = _scales_exact(x.t(), False, scale)
                got["codes_t"] = x.t() / each
        return got
    if op == "block_matmul":
        (a, sa), (b, sb) = st["a"], st["b"]
        a, b, sa, sb = a.double(), b.double(), sa.float().double(), sb.float().double()
        a = a * sa.repeat_interleave(BLOCK, 1)[:, :a.shape[1]]
        b = b * sb.repeat_interleave(BLOCK, 0)[:b.shape[0]].repeat_interleave(BLOCK, 1)[
            :, :b.shape[1]]
        return torch.mm(a, b.t().contiguous())
    x, w, dy = (st[t].detach().double() for t in ("x", "weight", "dy"))
    wq = _rounded_exact(w, True, scale)
    y = torch.mm(_rounded_exact(x, False, scale), wq.t().contiguous())
    dx = torch.mm(_rounded_exact(dy, False, scale), wq)
    dw = torch.mm(_rounded_exact(dy.t(), False, scale),
                  _rounded_exact(x.t(), False, scale).t().contiguous())
    return {"y": y, "dx": dx, "dw": dw}
