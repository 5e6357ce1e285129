"""Preference and policy tuning of the mHC-patched decoder mock.

The decoder of llama_mock.py with its MLP on FusedLinear (the gate's silu and
the block's residual in the matrix products' epilogues), the square projections
rewired by AutoPatcher, everything but the mHC parameters frozen.  A step runs
the model on pairs of answers (or on sampled ones with advantages), takes the
loss and the logits' gradient from one call, sends that through the model and
updates the mHC parameters, hundreds of small tensors, in one launch.

    python examples/tune_llama_mock.py [--steps N] [--loss preference|policy] [--state-bits 8]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import llama_mock  # noqa: E402

from mhc_b200 import (AdamW, AutoPatcher, FusedLinear, policy_loss_grad,  # noqa: E402
                      preference_loss_grad, token_logprobs)
from mhc_b200.dist import mhc_parameters  # noqa: E402

IGNORE = -100


class FusedMLP(nn.Module):
    def __init__(self, dims: int, mlp_dims: int, **kw):
        super().__init__()
        self.w1 = FusedLinear(dims, mlp_dims, bias=False, activation="silu", **kw)
        self.w3 = FusedLinear(dims, mlp_dims, bias=False, **kw)
        self.w2 = FusedLinear(mlp_dims, dims, bias=False, **kw)

    def forward(self, x, residual):
        return self.w2(self.w1(x) * self.w3(x), residual=residual)


class FusedBlock(llama_mock.MockBlock):
    def __init__(self, dims: int, num_heads: int, mlp_dims: int, **kw):
        super().__init__(dims, num_heads, mlp_dims, **kw)
        self.feed_forward = FusedMLP(dims, mlp_dims, **kw)

    def forward(self, x):
        h = x + self.attention(self.attention_norm(x))
        return self.feed_forward(self.ffn_norm(h), h)


def build(layers=2, dims=256, num_heads=4, mlp_dims=688, vocab=512, n_streams=4,
          dtype=torch.bfloat16, device="cuda", seed=0) -> llama_mock.LlamaMock:
    torch.manual_seed(seed)
    model = llama_mock.LlamaMock(0, dims, num_heads, mlp_dims, vocab, device=device, dtype=dtype)
    model.layers = nn.ModuleList(FusedBlock(dims, num_heads, mlp_dims, device=device, dtype=dtype)
                                 for _ in range(layers))
    for p in model.parameters():
        p.requires_grad_(False)
    AutoPatcher.patch(model, n_streams=n_streams, verbose=False, output_dtype="input",
                      identity_init=False)
    return model


def optimizer(model, lr: float = 1e-2, state_bits: int = 32) -> AdamW:
    return AdamW(mhc_parameters(model), lr=lr, weight_decay=0.0, state_bits=state_bits)


def shifted(tokens: torch.Tensor, prompt: int) -> torch.Tensor:
    """Targets of the logits at positions 0 .. S - 2; the prompt's take no part."""
    targets = tokens[:, 1:].clone()
    targets[:, :prompt - 1] = IGNORE
    return targets


@torch.no_grad()
def logprobs(model, tokens: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """The model's log probabilities of its tokens, for a reference or an old policy."""
    return token_logprobs(model(tokens)[:, :-1], targets, ignore_index=IGNORE)


def preference_step(model, opt: AdamW, tokens, targets, ref, beta: float = 0.5) -> torch.Tensor:
    """tokens [2 P, S]: answers in pairs (chosen, rejected).  Returns the loss."""
    opt.zero_grad()
    logits = model(tokens)[:, :-1]
    r = preference_loss_grad(logits.detach(), targets, ref, beta=beta, ignore_index=IGNORE)
    logits.backward(r.dlogits)
    opt.step()
    return r.loss


def policy_step(model, opt: AdamW, tokens, targets, old, ref, advantages) -> torch.Tensor:
    """tokens [B, S]: sampled answers with an advantage a token.  Returns the loss."""
    opt.zero_grad()
    logits = model(tokens)[:, :-1]
    r = policy_loss_grad(logits.detach(), targets, old, advantages, ref_logprobs=ref,
                         kl_coef=0.02, ignore_index=IGNORE)
    logits.backward(r.dlogits)
    opt.step()
    return r.loss


def main(argv=None) -> list[float]:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--loss", choices=("preference", "policy"), default="preference")
    ap.add_argument("--state-bits", type=int, choices=(8, 32), default=32)
    ap.add_argument("--pairs", type=int, default=4)
    ap.add_argument("--length", type=int, default=64)
    ap.add_argument("--prompt", type=int, default=12)
    a = ap.parse_args(argv)
    model = build()
    opt = optimizer(model, state_bits=a.state_bits)
    g = torch.Generator(device="cuda").manual_seed(1)
    vocab = model.head.out_features
    tokens = torch.randint(0, vocab, (2 * a.pairs, a.length), device="cuda", generator=g)
    tokens[1::2, :a.prompt] = tokens[::2, :a.prompt]  # a pair answers one prompt
    targets = shifted(tokens, a.prompt)
    start = logprobs(model, tokens, targets)  # the reference, and the policy that sampled
    advantages = torch.randn(2 * a.pairs, 1, device="cuda", generator=g).expand_as(start)
    losses = []
    for step in range(a.steps):
        if a.loss == "preference":
            loss = preference_step(model, opt, tokens, targets, start)
        else:
            loss = policy_step(model, opt, tokens, targets, start, start, advantages)
        losses.append(float(loss))
        print(f"step {step}: {a.loss} loss {losses[-1]:.4f}")
    return losses


if __name__ == "__main__":
    main()
