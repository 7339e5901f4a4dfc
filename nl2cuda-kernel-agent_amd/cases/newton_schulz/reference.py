"""PyTorch reference of the Newton-Schulz orthogonalisation, from basic
operators.  Inputs are drawn on the host CPU from one seeded generator."""

import torch

from cases.newton_schulz import config


def reference_forward(inputs, params):
    """inputs={"G":[count,m,n]} -> the orthogonalised matrices."""
    G = inputs["G"]
    a, b, c = params["coefficients"]
    tall = G.shape[-2] > G.shape[-1]
    X = G.mT if tall else G
    X = X / (torch.linalg.norm(X, dim=(-2, -1), keepdim=True) + params["eps"])
    for _ in range(params["steps"]):
        A = X @ X.mT
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.mT.contiguous() if tall else X


def make_inputs_for(count, m, n):
    """Input generator for `count` matrices m x n."""

    def make_inputs(seed, dtype, device, requires_grad=False):
        gen = torch.Generator(device="cpu").manual_seed(seed)
        return {"G": torch.randn(count, m, n, generator=gen).to(device=device, dtype=dtype)}

    return make_inputs


make_inputs = make_inputs_for(*config.SIZES)
