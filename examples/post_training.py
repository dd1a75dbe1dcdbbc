"""Three stages of post-training on one GPU with the objectives and MuonAdamW.

A small next-token model (embedding, two-layer MLP, output head) over a
synthetic language: the next token depends on the current one by a fixed table
with a few likely continuations.

1. Distillation: the student learns the table from its eight largest logits a
   token (``distill_loss``, with the mass of the others known).
2. Policy optimisation: sequences are sampled, scored by how often they take a
   wanted token, and the policy moves towards the better ones of each group
   (``token_logprobs`` for the policy's and the reference's log-probabilities,
   ``policy_loss`` with a KL term).
3. Preference optimisation: of two continuations the one from the table is
   preferred to one that is not (``preference_loss``).

    python examples/post_training.py
"""

from __future__ import annotations

import copy
import sys
from pathlib import Path

import torch
import torch.nn as nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "triton-muonadamw_amd"))

from triton_muon_adamw import (  # noqa: E402
    AdamConfig,
    MuonAdamW,
    MuonConfig,
    distill_loss,
    policy_loss,
    preference_loss,
    token_logprobs,
)

VOCAB, DIM, LENGTH, BATCH, TOP = 1003, 128, 24, 32, 8


class Model(nn.Module):
    def __init__(self):
        super().__init__()
        self.embed = nn.Embedding(VOCAB, DIM)
        self.up = nn.Linear(DIM, 4 * DIM)
        self.down = nn.Linear(4 * DIM, DIM)
        self.norm = nn.LayerNorm(DIM)
        self.head = nn.Linear(DIM, VOCAB, bias=False)

    def get_input_embeddings(self):
        return self.embed

    def get_output_embeddings(self):
        return self.head

    def forward(self, tokens):
        x = self.embed(tokens)
        x = x + self.down(torch.relu(self.up(x)))
        return self.head(self.norm(x))


def optimizer(model, lr):
    return MuonAdamW(model, muon_config=MuonConfig(lr=lr, weight_decay=0.0),
                     adam_config=AdamConfig(lr=lr / 4, weight_decay=0.0))


def sample(logits, gen):
    """Tokens drawn from softmax(logits)."""
    u = torch.rand(logits.shape, device=logits.device, generator=gen)
    return (logits - (-u.clamp(1e-20, 1 - 1e-7).log()).log()).argmax(-1)


def distill(model, table, gen, steps):
    """Losses of the student against the table's TOP first logits."""
    opt, losses = optimizer(model, 0.02), []
    values, index = table.topk(TOP, dim=-1)
    lse = torch.logsumexp(table, -1)
    for _ in range(steps):
        tokens = torch.randint(VOCAB, (BATCH, LENGTH), device=table.device, generator=gen)
        mask = torch.rand(tokens.shape, device=table.device, generator=gen) < 0.9  # the rest as padding
        loss = distill_loss(model(tokens), values[tokens], index[tokens], teacher_lse=lse[tokens], mask=mask)
        loss.backward()
        opt.step()
        opt.zero_grad()
        losses.append(loss.detach())
    return losses


def optimise_policy(model, wanted, gen, steps, group=8):
    """Mean rewards (share of wanted tokens) of the sampled sequences."""
    reference = copy.deepcopy(model).requires_grad_(False)
    opt, rewards = optimizer(model, 0.005), []
    for _ in range(steps):
        with torch.no_grad():  # BATCH / group prompts of one token, a group of continuations each
            start = torch.randint(VOCAB, (BATCH // group, 1), device=wanted.device, generator=gen)
            tokens = start.repeat_interleave(group, 0)
            for _ in range(LENGTH):
                tokens = torch.cat([tokens, sample(model(tokens[:, -1:])[:, -1], gen)[:, None]], 1)
            inputs, targets = tokens[:, :-1], tokens[:, 1:].clone()
            reward = wanted[targets].float().mean(1)
            better = reward.view(-1, group)
            advantage = ((better - better.mean(1, keepdim=True)) / (better.std(1, keepdim=True) + 1e-3)).view(-1, 1)
            old = token_logprobs(model(inputs), targets)
            ref = token_logprobs(reference(inputs), targets)
        for _ in range(2):  # the second step is off the policy that sampled
            out = policy_loss(model(inputs), targets, old, advantage, ref_logprobs=ref, kl_coef=0.01, clip=(0.2, 0.28))
            out.loss.backward()
            opt.step()
            opt.zero_grad()
        rewards.append(reward.mean())
    return rewards


def optimise_preference(model, table, gen, steps):
    """Margins (reward of the preferred sequence less that of the other) of each step's pairs."""
    reference = copy.deepcopy(model).requires_grad_(False)
    opt, margins = optimizer(model, 0.005), []
    for _ in range(steps):
        inputs = torch.randint(VOCAB, (BATCH, LENGTH), device=table.device, generator=gen)
        good = sample(table[inputs], gen)
        bad = torch.randint(VOCAB, inputs.shape, device=table.device, generator=gen)
        targets = torch.cat([good, bad])
        targets[:, :4] = -100  # the prompt
        both = torch.cat([inputs, inputs])
        with torch.no_grad():
            ref = token_logprobs(reference(both), targets).sum(1)
        out = preference_loss(model(both), targets, ref, beta=0.1)
        out.loss.backward()
        opt.step()
        opt.zero_grad()
        margins.append((out.rewards[:BATCH] - out.rewards[BATCH:]).mean())
    return margins


def main(steps=60, seed=0):
    """(distillation losses, policy rewards, preference margins), a number for each step."""
    torch.manual_seed(seed)
    device = torch.device("cuda:0")
    gen = torch.Generator(device=device).manual_seed(seed)
    table = 2.0 * torch.randn(VOCAB, VOCAB, device=device, generator=gen)
    table.scatter_add_(1, torch.randint(VOCAB, (VOCAB, 4), device=device, generator=gen),
                       torch.full((VOCAB, 4), 6.0, device=device))
    wanted = torch.arange(VOCAB, device=device) % 10 == 0
    model = Model().to(device)
    curves = (distill(model, table, gen, steps), optimise_policy(model, wanted, gen, steps),
              optimise_preference(model, table, gen, steps))
    return tuple(torch.stack(c).tolist() for c in curves)


if __name__ == "__main__":
    for name, curve in zip(("distillation loss", "policy reward", "preference margin"), main()):
        print(f"{name}: {curve[0]:.4f} -> {curve[-1]:.4f} in {len(curve)} steps", flush=True)
