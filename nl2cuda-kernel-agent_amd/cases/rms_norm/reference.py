"""PyTorch reference of the root-mean-square norm with the residual's addition,
from basic operators; autograd gives the backward.  Inputs are drawn on the host
CPU from one seeded generator: X, R ~ N(0, 1), W = 1 + 0.1 N(0, 1)."""

import torch

from cases.rms_norm import config


def reference_forward(inputs, params):
    """inputs={"X":[B,D], "R":[B,D], "W":[D]} -> y [B,D]."""
    h = inputs["X"] + inputs["R"]
    rms = torch.sqrt(h.square().mean(-1, keepdim=True) + params.get("eps", 1e-6))
    return h / rms * inputs["W"]


def make_inputs_for(b, d):
    """Input generator for b rows of d numbers."""

    def make_inputs(seed, dtype, device, requires_grad=False):
        gen = torch.Generator(device="cpu").manual_seed(seed)
        X = torch.randn(b, d, generator=gen)
        R = torch.randn(b, d, generator=gen)
        W = 1 + 0.1 * torch.randn(d, generator=gen)
        got = {"X": X, "R": R, "W": W}
        got = {k: v.to(device=device, dtype=dtype) for k, v in got.items()}
        if requires_grad:
            for v in got.values():
                v.requires_grad_(True)
        return got

    return make_inputs


make_inputs = make_inputs_for(*config.SIZES)
