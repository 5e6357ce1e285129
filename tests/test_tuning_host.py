"""Argument checks of the fine-tuning operators: they come before any CUDA call."""

from __future__ import annotations

import pytest
import torch

import mhc_b200
from mhc_b200 import _capi


def _rows(T=4, V=8, dtype=torch.float32):
    return torch.zeros(T, V, dtype=dtype), torch.zeros(T, dtype=torch.int64)


def test_losses_refuse_cpu_tensors():
    x, y = _rows()
    z = torch.zeros(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        mhc_b200.token_logprobs(x, y)
    with pytest.raises(RuntimeError, match="CUDA"):
        mhc_b200.policy_loss_grad(x, y, z, z)
    with pytest.raises(RuntimeError, match="CUDA"):
        mhc_b200.preference_loss(x, y, z, torch.tensor([0, 2, 4]))


def test_logits_refusals():
    x, y = _rows()
    for bad, t, match in [(x.double(), y, "dtype"), (x[0], y[0], r"\[T, V\]"), (x, y.int(), "int64"),
                          (x, y[:3], "targets"), (x[:, :0], y, "class")]:
        with pytest.raises(ValueError, match=match):
            mhc_b200.token_logprobs(bad, t)


def test_preference_refusals():
    x, y = _rows()
    z, cu = torch.zeros(4), torch.tensor([0, 2, 4])
    for args, kw, match in [((x, y, z[:3], cu), {}, "ref_logprobs"), ((x, y, y, cu), {}, "floating"),
                            ((x, y, z), {}, "cu_seqlens"), ((x, y, z, cu[:2]), {}, "pairs"),
                            ((x, y, z, cu[:0]), {}, "pairs"), ((x, y, z, cu.float()), {}, "int32"),
                            ((x, y, z, cu), dict(label_smoothing=1.0), "label_smoothing"),
                            ((x, y, z, cu), dict(denominator=0), "denominator"),
                            ((x[None], y[None], z[None]), {}, "pairs")]:
        for f in (mhc_b200.preference_loss, mhc_b200.preference_loss_grad):
            with pytest.raises(ValueError, match=match):
                f(*args, **kw)


def test_policy_refusals():
    x, y = _rows()
    z = torch.zeros(4)
    for args, kw, match in [((x, y, z[:3], z), {}, "old_logprobs"), ((x, y, z, y), {}, "floating"),
                            ((x, y, z, z), dict(kl_coef=0.1), "ref_logprobs"),
                            ((x, y, z, z), dict(clip_low=1.5), "clip_low"),
                            ((x, y, z, z), dict(clip_high=-0.1), "clip_high"),
                            ((x, y, z, z), dict(denominator=-1), "denominator")]:
        for f in (mhc_b200.policy_loss, mhc_b200.policy_loss_grad):
            with pytest.raises(ValueError, match=match):
                f(*args, **kw)


def test_loss_entry_points_check_their_arguments():
    rows = (None, 0, 0, 1, 0, 0)
    with pytest.raises(ValueError, match="V=0"):
        _capi.call("mhc_token_logprobs", *rows, 0, None, -100, None, None, None)
    with pytest.raises(ValueError, match="dtype"):
        _capi.call("mhc_token_logprobs", None, 9, 0, 1, 0, 0, 5, None, -100, None, None, None)
    with pytest.raises(ValueError, match="rows"):
        _capi.call("mhc_token_logprobs", None, 0, 1 << 28, 1, 0, 0, 5, None, -100, None, None, None)
    with pytest.raises(ValueError, match="NULL"):
        _capi.call("mhc_token_logprobs", None, 0, 3, 3, 0, 5, 5, None, -100, None, None, None)
    with pytest.raises(ValueError, match="unless_one"):
        _capi.call("mhc_logits_grad", *rows, 5, None, -100, None, None, 1.0, None, 1, None, None)
    with pytest.raises(ValueError, match="pairs"):
        _capi.call("mhc_preference_loss", *rows, 5, None, -100, None, 0, 0, 0, None, 0.1, 0.0, 1.0,
                   1.0, None, None, None, None, None, None, None)
    assert _capi.query("mhc_policy_workspace_bytes") >= 256 + 16 * 148
