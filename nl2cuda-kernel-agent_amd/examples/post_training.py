"""Post-training of a small language model with the framework's operators.

A model of two matrices between embeddings (layernorm's kernels in between)
learns to count: after token t comes t + 1.  First from rewards: it samples
answers, ``token_logp`` records what it chose, and ``policy_loss`` with a KL
term to the model it started from moves it; then from pairs of answers, one
right and one random, by ``preference_loss``.  The matrices are updated by
``Muon``, the embeddings by plain steps.

  python nl2cuda-kernel-agent_amd/examples/post_training.py
"""

import os
import sys

import torch

PKG = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if PKG not in sys.path:
    sys.path.insert(0, PKG)

from cases.layernorm import op as layernorm  # noqa: E402
from cases.newton_schulz.op import Muon  # noqa: E402
from cases.policy_loss.op import policy_loss  # noqa: E402
from cases.preference_loss.op import preference_loss  # noqa: E402
from cases.token_logp.op import token_logp  # noqa: E402

VOCABULARY, WIDTH, LENGTH, ANSWERS = 48, 96, 12, 64
IGNORE = -100


class Model(torch.nn.Module):
    """Logits of the next token from the present one."""

    def __init__(self, generator):
        super().__init__()

        def weight(*shape, scale=1.0):
            w = torch.randn(*shape, generator=generator) * scale
            return torch.nn.Parameter(w.cuda())

        self.embedding = weight(VOCABULARY, WIDTH)
        self.hidden = weight(WIDTH, WIDTH, scale=WIDTH ** -0.5)
        self.head = weight(WIDTH, VOCABULARY, scale=0.1 * WIDTH ** -0.5)
        self.gamma = torch.nn.Parameter(torch.ones(WIDTH, device="cuda"))
        self.beta = torch.nn.Parameter(torch.zeros(WIDTH, device="cuda"))

    def forward(self, tokens):
        x = self.embedding[tokens.reshape(-1)] @ self.hidden
        x = layernorm.candidate({"X": x, "gamma": self.gamma, "beta": self.beta}, {"eps": 1e-5})
        return (torch.relu(x) @ self.head).view(*tokens.shape, VOCABULARY)


def optimisers(model, lr):
    return (Muon([model.hidden, model.head], lr=lr),
            torch.optim.SGD([model.embedding, model.gamma, model.beta], lr=10 * lr))


def update(opts, loss):
    for o in opts:
        o.zero_grad()
    loss.backward()
    for o in opts:
        o.step()


@torch.no_grad()
def sample(model, generator):
    """(tokens [ANSWERS, LENGTH + 1], logp [ANSWERS, LENGTH]): a prompt of one
    token and an answer, with the log-probability of each token as chosen."""
    tokens = [torch.randint(0, VOCABULARY, (ANSWERS,), generator=generator, device="cuda")]
    logp = []
    for _ in range(LENGTH):
        logits = model(tokens[-1])
        choice = torch.multinomial(torch.softmax(logits, -1), 1, generator=generator)[:, 0]
        logp.append(token_logp(logits, choice))
        tokens.append(choice)
    return torch.stack(tokens, 1), torch.stack(logp, 1)


def reward(tokens):
    """Share of an answer's tokens that count on from the one before."""
    return (tokens[:, 1:] == (tokens[:, :-1] + 1) % VOCABULARY).float().mean(1)


def learn_from_rewards(model, steps, generator, lr=0.02):
    """Mean reward of each step's answers."""
    start = {k: v.clone() for k, v in model.state_dict().items()}
    opts, history = optimisers(model, lr), []
    for _ in range(steps):
        tokens, old = sample(model, generator)
        score = reward(tokens)
        history.append(score.mean().item())
        advantage = (score - score.mean()) / (score.std() + 1e-6)
        inputs, labels = tokens[:, :-1], tokens[:, 1:].contiguous()
        with torch.no_grad():
            ref = token_logp(torch.func.functional_call(model, start, (inputs,)), labels)
        for _ in range(2):
            loss, _ = policy_loss(model(inputs), labels, old, advantage, ref, kl_coef=1e-3,
                                  clip_low=0.2, clip_high=0.3)
            update(opts, loss)
    return history


def learn_from_pairs(model, steps, generator, lr=0.02):
    """Loss of each step."""
    opts, history = optimisers(model, lr), []
    start = {k: v.clone() for k, v in model.state_dict().items()}
    for _ in range(steps):
        first = torch.randint(0, VOCABULARY, (ANSWERS, 1), generator=generator, device="cuda")
        right = (first + torch.arange(LENGTH + 1, device="cuda")) % VOCABULARY
        wrong = torch.randint(0, VOCABULARY, right.shape, generator=generator, device="cuda")
        wrong[:, 0] = first[:, 0]
        tokens = torch.cat([right, wrong])
        inputs, labels = tokens[:, :-1], tokens[:, 1:].clone()
        lengths = torch.randint(1, LENGTH + 1, (2 * ANSWERS, 1), generator=generator,
                                device="cuda")
        labels[torch.arange(LENGTH, device="cuda") >= lengths] = IGNORE   # padding
        with torch.no_grad():
            ref = token_logp(torch.func.functional_call(model, start, (inputs,)), labels).sum(1)
        loss, _ = preference_loss(model(inputs), labels, ref, beta=0.1)
        update(opts, loss)
        history.append(loss.item())
    return history


def main():
    if not torch.cuda.is_available():
        print("post_training: needs an MI355X GPU", file=sys.stderr)
        return 2
    generator = torch.Generator(device="cuda").manual_seed(0)
    model = Model(torch.Generator().manual_seed(0))
    rewards = learn_from_rewards(model, 60, generator)
    print(f"rewards: {rewards[0]:.3f} -> {rewards[-1]:.3f}")
    model = Model(torch.Generator().manual_seed(1))
    losses = learn_from_pairs(model, 40, generator)
    print(f"preference loss: {losses[0]:.3f} -> {losses[-1]:.3f}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
