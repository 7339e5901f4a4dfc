"""PyTorch reference of the clipped policy loss with a KL term, from basic
operators; autograd gives the backward.  Inputs are drawn on the host CPU from
one seeded generator: log ratios ~ N(0, 0.2), one advantage an answer, answers
of different lengths."""

import torch

from cases.policy_loss import config
from cases.token_logp.reference import reference_forward as token_logp


def reference_forward(inputs, params):
    """inputs={"logits":[B,S,V], "labels", "old_logp", "ref_logp":[B,S],
    "advantages":[B,1], "mask":[B,S] bool} -> scalar loss."""
    mask = inputs["mask"]
    logp = token_logp(inputs, params)
    ratio = torch.exp(logp - inputs["old_logp"])
    adv = inputs["advantages"]
    cut = torch.clamp(ratio, 1 - params["clip_low"], 1 + params["clip_high"])
    d = inputs["ref_logp"] - logp
    term = params["kl_coef"] * (torch.exp(d) - d - 1) - torch.minimum(ratio * adv, cut * adv)
    return (term * mask).sum() / mask.sum()


def make_inputs_for(b, s, v):
    """Input generator for B answers of S tokens over V classes."""

    def make_inputs(seed, dtype, device, requires_grad=False):
        gen = torch.Generator(device="cpu").manual_seed(seed)
        logits = torch.randn(b, s, v, generator=gen).to(dtype)
        labels = torch.randint(0, v, (b, s), generator=gen)
        logp = token_logp({"logits": logits.float(), "labels": labels}, {})
        lengths = torch.randint(1, s + 1, (b,), generator=gen)
        inputs = {"logits": logits.to(device), "labels": labels,
                  "old_logp": logp + 0.2 * torch.randn(b, s, generator=gen),
                  "ref_logp": logp + 0.2 * torch.randn(b, s, generator=gen),
                  "advantages": torch.randn(b, 1, generator=gen),
                  "mask": torch.arange(s)[None, :] < lengths[:, None]}
        inputs = {k: t.to(device) for k, t in inputs.items()}
        if requires_grad:
            inputs["logits"].requires_grad_(True)
        return inputs

    return make_inputs


make_inputs = make_inputs_for(*config.SIZES)
