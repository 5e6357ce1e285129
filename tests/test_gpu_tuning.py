"""The tuning operators together, as the example runs them."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

from mhc_b200.dist import mhc_parameters

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "mhc-mlx_b200" / "examples"))
import tune_llama_mock as T  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("loss", ["preference", "policy"])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_few_steps_lower_the_loss(loss, bits):
    losses = T.main(["--steps", "6", "--loss", loss, "--state-bits", str(bits)])
    assert all(x == x for x in losses) and losses[-1] < losses[0]


def test_gradients_are_those_of_the_loss_on_logits():
    """The parameters' gradients from preference_loss_grad are those of the same loss
    written out on the same model's logits (bf16: the logits' gradient is rounded alike)."""
    model = T.build()
    tokens = torch.randint(0, 512, (4, 40), device="cuda",
                           generator=torch.Generator(device="cuda").manual_seed(2))
    targets = T.shifted(tokens, 8)
    ref = T.logprobs(model, tokens, targets) - 0.1
    params = [p for p in mhc_parameters(model) if p.requires_grad]
    logits = model(tokens)[:, :-1]
    r = T.preference_loss_grad(logits.detach(), targets, ref, beta=0.5, ignore_index=T.IGNORE)
    got = torch.autograd.grad(logits, params, r.dlogits, retain_graph=True, allow_unused=True)
    x = logits.float()
    keep = targets != T.IGNORE
    lp = torch.log_softmax(x, -1).gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    R = torch.where(keep, lp - ref, torch.zeros_like(lp)).sum(1)
    loss = F.softplus(-0.5 * (R[0::2] - R[1::2])).mean()
    want = torch.autograd.grad(loss, params, allow_unused=True)
    assert abs(float(loss) - float(r.loss)) < 1e-4
    for a, b in zip(got, want):
        assert (a is None) == (b is None)
        if a is not None:
            assert (a - b).norm() <= 0.05 * b.norm() + 1e-6
