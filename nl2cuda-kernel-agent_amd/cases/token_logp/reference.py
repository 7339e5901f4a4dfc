"""PyTorch reference of the token log-probabilities, from basic operators;
autograd gives the backward.  Inputs are drawn on the host CPU from one seeded
generator: logits ~ N(0, 1), labels uniform, one token in eight ignored."""

import torch

from cases.token_logp import config

IGNORE = -100


def reference_forward(inputs, params):
    """inputs={"logits":[B,S,V], "labels":[B,S] int64} -> logp [B,S]."""
    x, labels = inputs["logits"] / params.get("temperature", 1.0), inputs["labels"]
    keep = labels != IGNORE
    at = torch.where(keep, labels, torch.zeros_like(labels)).unsqueeze(-1)
    logp = x.gather(-1, at).squeeze(-1) - torch.logsumexp(x, dim=-1)
    return torch.where(keep, logp, torch.zeros_like(logp))


def make_inputs_for(b, s, v):
    """Input generator for B x S tokens over V classes."""

    def make_inputs(seed, dtype, device, requires_grad=False):
        gen = torch.Generator(device="cpu").manual_seed(seed)
        logits = torch.randn(b, s, v, generator=gen).to(device=device, dtype=dtype)
        labels = torch.randint(0, v, (b, s), generator=gen)
        labels[torch.rand(b, s, generator=gen) < 0.125] = IGNORE
        if requires_grad:
            logits.requires_grad_(True)
        return {"logits": logits, "labels": labels.to(device)}

    return make_inputs


make_inputs = make_inputs_for(*config.SIZES)
