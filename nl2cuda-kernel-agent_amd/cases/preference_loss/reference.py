"""PyTorch reference of the preference loss, from basic operators; autograd
gives the backward.  Inputs are drawn on the host CPU from one seeded
generator: answers of different lengths, their prompts ignored."""

import torch

from cases.preference_loss import config
from cases.token_logp.reference import IGNORE, reference_forward as token_logp


def reference_forward(inputs, params):
    """inputs={"logits":[2N,S,V], "labels":[2N,S], "ref_seq_logp":[2N]} -> scalar loss."""
    seq = token_logp(inputs, {}).sum(1)
    if params["average"]:
        seq = seq / (inputs["labels"] != IGNORE).sum(1).clamp(min=1)
    h = params["beta"] * (seq - inputs["ref_seq_logp"])
    n = h.numel() // 2
    d = h[:n] - h[n:]
    eps = params["label_smoothing"]
    softplus = torch.nn.functional.softplus
    return ((1 - eps) * softplus(-d) + eps * softplus(d)).mean()


def make_inputs_for(n, s, v):
    """Input generator for N pairs of at most S tokens over V classes."""

    def make_inputs(seed, dtype, device, requires_grad=False):
        gen = torch.Generator(device="cpu").manual_seed(seed)
        logits = torch.randn(2 * n, s, v, generator=gen).to(dtype)
        labels = torch.randint(0, v, (2 * n, s), generator=gen)
        lengths = torch.randint(1, s + 1, (2 * n,), generator=gen)
        at = torch.arange(s)[None, :]
        labels[(at < s // 8) | (at >= lengths[:, None])] = IGNORE
        seq = token_logp({"logits": logits.float(), "labels": labels}, {}).sum(1)
        ref = seq + 3.0 * torch.randn(2 * n, generator=gen)
        logits = logits.to(device)
        if requires_grad:
            logits.requires_grad_(True)
        return {"logits": logits, "labels": labels.to(device), "ref_seq_logp": ref.to(device)}

    return make_inputs


make_inputs = make_inputs_for(*config.SIZES)
