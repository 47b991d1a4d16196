"""Policy fine-tuning of a small decoder with experts: the row operators of ``muonium_amd.kernels``
with the ``Muon`` step, as a training loop uses them.

    python examples/policy_experts.py [--steps 30]

A decoder of two layers (grouped heads, normalized and rotated queries and keys, eight experts of which
each token takes two) answers random prompts; an answer token is rewarded when it repeats the
token three places before it. Each step samples answers with the current weights
(``token_logprobs`` gives what they were sampled with, and what the frozen first model thinks of
them), then takes two steps on ``policy_loss`` with the balance and z losses of ``route``.
"""

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "dtensor-muon_amd"))

from muonium_amd import Muon  # noqa: E402
from muonium_amd.kernels import policy_loss, qk_norm_rope, route, token_logprobs  # noqa: E402

VOCAB, WIDTH, LAYERS, HEADS, KV_HEADS, DIM, EXPERTS, TOP, HIDDEN = 64, 128, 2, 4, 2, 32, 8, 2, 128


class Layer(nn.Module):
    def __init__(self):
        super().__init__()

        def weight(*shape):
            return nn.Parameter(torch.randn(*shape) * shape[-1] ** -0.5)

        self.qkv = weight((HEADS + 2 * KV_HEADS) * DIM, WIDTH)
        self.out = weight(WIDTH, HEADS * DIM)
        self.router = weight(EXPERTS, WIDTH)
        self.up = weight(EXPERTS, HIDDEN, WIDTH)
        self.down = weight(EXPERTS, WIDTH, HIDDEN)
        self.q_gain, self.k_gain = (nn.Parameter(torch.ones(DIM)) for _ in range(2))

    def attend(self, x, cos, sin):
        b, t, _ = x.shape
        q, k, v = (x @ self.qkv.T).view(b, t, -1, DIM).split([HEADS, KV_HEADS, KV_HEADS], 2)
        q, k = qk_norm_rope(q, k, self.q_gain, self.k_gain, cos, sin)
        k, v = (y.repeat_interleave(HEADS // KV_HEADS, 2).transpose(1, 2).contiguous() for y in (k, v))
        scores = q.transpose(1, 2) @ k.transpose(2, 3).contiguous() * DIM**-0.5
        later = torch.ones(t, t, dtype=torch.bool, device=x.device).triu(1)
        y = scores.masked_fill(later, float("-inf")).softmax(-1) @ v
        return y.transpose(1, 2).reshape(b, t, -1) @ self.out.T

    def experts(self, x):
        flat = x.flatten(0, 1)
        r = route(flat @ self.router.T, TOP)
        # every expert on every token: a small model can afford it
        share = torch.zeros(len(flat), EXPERTS, device=x.device).scatter(1, r.experts, r.gates)
        hidden = torch.relu(flat @ self.up.transpose(1, 2).contiguous()).square()
        y = (hidden @ self.down.transpose(1, 2).contiguous()).transpose(0, 1)
        return (share[:, :, None] * y).sum(1).view_as(x), r


def norm(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


class Decoder(nn.Module):
    def __init__(self, length):
        super().__init__()
        self.embed = nn.Parameter(torch.randn(VOCAB, WIDTH))
        self.head = nn.Parameter(torch.randn(VOCAB, WIDTH) * WIDTH**-0.5 * 0.1)
        self.layers = nn.ModuleList(Layer() for _ in range(LAYERS))
        angle = torch.arange(length)[:, None] * 1000.0 ** (-torch.arange(DIM // 2) / (DIM // 2))
        self.register_buffer("cos", angle.cos())
        self.register_buffer("sin", angle.sin())

    def forward(self, tokens):
        x, routings = self.embed[tokens], []
        for layer in self.layers:
            x = x + layer.attend(norm(x), self.cos, self.sin)
            y, r = layer.experts(norm(x))
            x = x + y
            routings.append(r)
        return norm(x) @ self.head.T, routings


@torch.no_grad()
def sample(model, prompts, length):
    """The prompts with ``length`` sampled tokens behind them."""
    tokens = prompts
    for _ in range(length):
        p = model(tokens)[0][:, -1].softmax(-1)
        tokens = torch.cat([tokens, torch.multinomial(p, 1)], 1)
    return tokens


def train(steps=30, batch=64, prompt=6, answer=10, seed=0, log=print):
    """Mean reward of each step's samples."""
    torch.manual_seed(seed)
    model = Decoder(prompt + answer).cuda()
    first = Decoder(prompt + answer).cuda()
    first.load_state_dict(model.state_dict())
    matrices = [p for layer in model.layers for n, p in layer.named_parameters() if p.ndim >= 2]
    rest = [model.embed, model.head, *(p for layer in model.layers for p in layer.parameters()
                                       if p.ndim < 2)]
    optimizers = [Muon(matrices, lr=0.01, wd=0.0), torch.optim.AdamW(rest, lr=0.01, weight_decay=0.0)]
    rewards = []
    for step in range(steps):
        prompts = torch.randint(VOCAB, (batch, prompt), device="cuda")
        tokens = sample(model, prompts, answer)
        seen, said = tokens[:, :-1], tokens[:, 1:].contiguous()
        place = torch.arange(said.shape[1], device="cuda")
        weights = (place >= prompt - 1).float().expand(said.shape) / (batch * answer)
        reward = (said == torch.roll(said, 3, 1)).float()
        advantages = reward - (reward * weights).sum()
        with torch.no_grad():
            old = token_logprobs(model(seen)[0], said)
            reference = token_logprobs(first(seen)[0], said)
        for _ in range(2):
            logits, routings = model(seen)
            out = policy_loss(logits, said, old, advantages, weights, reference, kl_coef=0.001)
            loss = out.loss + sum(0.01 * r.balance_loss + 0.001 * r.z_loss for r in routings)
            loss.backward()
            for optimizer in optimizers:
                optimizer.step()
                optimizer.zero_grad()
        rewards.append((reward * weights).sum().item())
        log(f"step {step}: reward {rewards[-1]:.3f}  loss {out.loss.item():+.4f}  tokens of the "
            f"busiest expert {max(r.counts.max().item() for r in routings)}")
    return rewards


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=30)
    train(parser.parse_args().steps)
