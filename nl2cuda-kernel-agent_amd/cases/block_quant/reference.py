"""PyTorch reference of the block quantisation, from basic operators.  Inputs
are drawn on the host CPU from one seeded generator: N(0, 1) times a size for
each row."""

import torch

from cases.block_quant import config

BLOCK, TOP, LEAST = 128, 448.0, 2.0 ** -126


def reference_forward(inputs, params):
    """inputs={"X":[M,K]} -> what its codes and scales stand for."""
    X = inputs["X"]
    M, K = X.shape
    x = torch.nn.functional.pad(X, (0, -K % BLOCK)).reshape(M, -1, BLOCK)
    least = x.abs().amax(-1, keepdim=True).double() / TOP
    if params.get("scale_dtype", torch.float8_e8m0fnu) == torch.float32:
        s = least.clamp(min=LEAST).float()
    else:
        f, e = torch.frexp(least)
        s = torch.ldexp(torch.ones_like(f), torch.where(f == 0.5, e - 1, e))
        s = s.clamp(min=LEAST).float()
    q = (x * (1.0 / s.double()).float()).to(torch.float8_e4m3fn).to(X.dtype) * s
    return q.reshape(M, -1)[:, :K].to(X.dtype)


def make_inputs_for(m, k):
    """Input generator for m x k numbers."""

    def make_inputs(seed, dtype, device, requires_grad=False):
        gen = torch.Generator(device="cpu").manual_seed(seed)
        X = torch.randn(m, k, generator=gen) * torch.exp(torch.randn(m, 1, generator=gen))
        return {"X": X.to(device=device, dtype=dtype)}

    return make_inputs


make_inputs = make_inputs_for(*config.SIZES)
