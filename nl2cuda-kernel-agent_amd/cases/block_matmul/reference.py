"""PyTorch reference of the layer in 8 bits, from basic operators: operands
rounded to e4m3 under a scale for each block of 128, gradients passed through
the roundings.  Inputs are drawn on the host CPU from one seeded generator:
X ~ N(0, 1), W ~ N(0, 1) / sqrt(K)."""

import torch

from cases.block_matmul import config

BLOCK, TOP, LEAST = 128, 448.0, 2.0 ** -126


def rounded(x, side, scale_dtype):
    """x [M, K] as 8 bits hold it, a scale for `side` rows by 128 columns."""
    M, K = x.shape
    b = torch.nn.functional.pad(x, (0, -K % BLOCK, 0, -M % side))
    b = b.reshape(-(-M // side), side, -(-K // BLOCK), BLOCK)
    least = b.abs().amax((1, 3), keepdim=True).double() / TOP
    if scale_dtype == torch.float32:
        s = least.clamp(min=LEAST).float()
    else:
        f, e = torch.frexp(least)
        s = torch.ldexp(torch.ones_like(f), torch.where(f == 0.5, e - 1, e))
        s = s.clamp(min=LEAST).float()
    q = (b * (1.0 / s.double()).float()).to(torch.float8_e4m3fn).to(x.dtype) * s
    return q.reshape(-(-M // side) * side, -1)[:M, :K].to(x.dtype)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, W, scale_dtype):
        w = rounded(W, BLOCK, scale_dtype)
        ctx.save_for_backward(rounded(X.t(), 1, scale_dtype), w)
        ctx.scale_dtype = scale_dtype
        return rounded(X, 1, scale_dtype) @ w.t()

    @staticmethod
    def backward(ctx, G):
        xt, w = ctx.saved_tensors
        return (rounded(G, 1, ctx.scale_dtype) @ w,
                rounded(G.t(), 1, ctx.scale_dtype) @ xt.t(), None)


def reference_forward(inputs, params):
    """inputs={"X":[M,K], "W":[N,K]} -> X W^T [M,N]."""
    return _Linear.apply(inputs["X"], inputs["W"],
                         params.get("scale_dtype", torch.float8_e8m0fnu))


def make_inputs_for(m, n, k):
    """Input generator for m rows and a weight of n rows, k numbers each."""

    def make_inputs(seed, dtype, device, requires_grad=False):
        gen = torch.Generator(device="cpu").manual_seed(seed)
        X = torch.randn(m, k, generator=gen)
        W = torch.randn(n, k, generator=gen) / k ** 0.5
        got = {"X": X.to(device=device, dtype=dtype), "W": W.to(device=device, dtype=dtype)}
        if requires_grad:
            for v in got.values():
                v.requires_grad_(True)
        return got

    return make_inputs


make_inputs = make_inputs_for(*config.SIZES)
