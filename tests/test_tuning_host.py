"""Argument checks of the fine-tuning operators: they come before any CUDA call."""

from __future__ import annotations

import ctypes

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


def test_adamw_refusals():
    p = torch.nn.Parameter(torch.zeros(4, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        mhc_b200.AdamW([p])
    for kw, match in [(dict(state_bits=16), "state_bits"), (dict(lr=-1.0), "lr"),
                      (dict(lr=torch.tensor(0.1)), "lr"), (dict(betas=(1.0, 0.9)), "betas"),
                      (dict(eps=-1.0), "eps"), (dict(weight_decay=-0.1), "weight_decay")]:
        with pytest.raises(ValueError, match=match):
            mhc_b200.AdamW([p], **kw)
    with pytest.raises(ValueError, match="dtype"):
        mhc_b200.AdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))])
    with pytest.raises(ValueError, match="dense"):
        mhc_b200.AdamW([torch.zeros(4, 8)[:, ::2].requires_grad_(True)])


def test_adamw_entry_point_checks_its_arguments():
    tail = (0.9, 0.1, 0.9, 0.1, 1.0, 0.1, 1.0, 1e-8, None, 0, None)
    none = (None, None, None, None)
    with pytest.raises(ValueError, match="state_bits"):
        _capi.call("mhc_adamw_step", 0, *none, 0, 4, None, None, None, None, None, *tail)
    with pytest.raises(ValueError, match="master"):
        _capi.call("mhc_adamw_step", 0, *none, 0, 32, None, None, None, None, 256, *tail)
    with pytest.raises(ValueError, match="NULL"):
        _capi.call("mhc_adamw_step", 1, *none, 0, 32, None, None, None, None, None, *tail)
    one = (ctypes.c_uint64 * 1)(256)
    size, off = (ctypes.c_int64 * 1)(4), (ctypes.c_int64 * 1)(100)
    with pytest.raises(ValueError, match="multiple of 256"):
        _capi.call("mhc_adamw_step", 1, one, one, size, off, 0, 32, 256, None, 256, None, None, *tail)
    with pytest.raises(ValueError, match="scales"):
        _capi.call("mhc_adamw_step", 1, one, one, size, off, 0, 8, 256, None, 256, None, None, *tail)
    _capi.call("mhc_adamw_step", 0, *none, 0, 32, None, None, None, None, None, *tail)


def test_linear_refusals():
    x, w = torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    b, r = torch.zeros(4, dtype=torch.bfloat16), torch.zeros(3, 4, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        mhc_b200.linear_act(x, w, b, residual=r)
    for args, kw, match in [((x.float(), w.float()), {}, "float16 or bfloat16"),
                            ((x, w.half()), {}, "weight"), ((x, w[0]), {}, "weight"),
                            ((x, w[:0]), {}, "weight"), ((x[:, :7], w), {}, "x must"),
                            ((x, w, b[:3]), {}, "bias"), ((x, w, b.float()), {}, "bias"),
                            ((x, w), dict(residual=r[:2]), "residual"),
                            ((x, w), dict(residual=r.half()), "residual"),
                            ((x, w), dict(activation="tanh"), "activation")]:
        with pytest.raises(ValueError, match=match):
            mhc_b200.linear_act(*args, **kw)
    with pytest.raises(ValueError, match="activation"):
        mhc_b200.FusedLinear(8, 4, activation="swish")


def test_linear_entry_points_check_their_arguments():
    fwd = lambda x=256, ldx=8, dt=2, act=0, M=1, N=4, K=8: _capi.call(  # noqa: E731
        "mhc_linear_fwd", x, ldx, 256, 8, None, None, 0, dt, act, None, 0, 256, 4, M, N, K, None, 0,
        None)
    with pytest.raises(_capi.MHCError, match="dtype"):
        fwd(dt=0)
    for kw, match in [(dict(dt=9), "dtype"), (dict(act=4), "act"), (dict(M=-1), "M="),
                      (dict(N=0), "N="), (dict(K=0), "K="), (dict(x=None), "NULL x"),
                      (dict(x=257), "aligned"), (dict(ldx=7), "apart")]:
        with pytest.raises(ValueError, match=match):
            fwd(**kw)
    with pytest.raises(_capi.MHCError, match="workspace"):
        fwd(x=258, M=100)  # rows that have to be padded
    fwd(M=0)
    query = lambda *a: _capi.query("mhc_linear_bwd_workspace_bytes", *a)  # noqa: E731
    assert query(256, 64, 256, 64, 256, 64, 0, 1, 1, 0, 100, 64, 64) == 0
    assert query(256, 64, 256, 64, 256, 64, 2, 1, 0, 0, 100, 64, 64) >= 100 * 64 * 2
    with pytest.raises(ValueError, match="z"):
        _capi.call("mhc_linear_bwd", 256, 64, None, 0, 256, 64, 256, 64, 2, 1, 256, 64, None, 0, None,
                   100, 64, 64, None, 0, None)


def test_host_extension():
    """It is built from the source beside it, takes CUDA tensors only, and refuses bad calls."""
    import ctypes

    from mhc_b200 import _build

    host = _capi.host()
    assert host.build_id == _build.host_id()
    p = torch.nn.Parameter(torch.zeros(4))
    numel, out = (ctypes.c_int64 * 1)(4), (ctypes.c_uint64 * 1)(7)
    at = ctypes.addressof
    assert host.gather([p], at(numel), 0, 0, at(out), at(out)) is False and out[0] == 7
    assert host.gather([3], at(numel), 0, 0, at(out), at(out)) is False
    assert host.gather([], at(numel), 0, 0, at(out), at(out)) is True
    for bad in (((p,), at(numel), 0, 0, at(out), at(out)), ([p], at(numel), 0, 0, at(out))):
        with pytest.raises(TypeError):
            host.gather(*bad)
    for bad in (([p], 0, 0, 0, at(out), at(out)), ([p], at(numel), 9, 0, at(out), at(out)),
                ([p], at(numel), 0, -1, at(out), at(out))):
        with pytest.raises(ValueError):
            host.gather(*bad)


def test_host_calls_refuse_other_arguments():
    host = _capi.host()
    x, y = _rows()
    for call in (host.linear, host.token_logprobs, host.logits_grad, host.preference, host.policy,
                 host.bind):
        with pytest.raises(TypeError):
            call(x)
    with pytest.raises(TypeError):
        host.token_logprobs(x, 3, -100)
    with pytest.raises(TypeError):
        host.token_logprobs(x, y, "a")
    with pytest.raises(RuntimeError, match="CUDA"):
        host.token_logprobs(x, y, -100)
    with pytest.raises(RuntimeError, match="CUDA"):
        host.linear(x, x, None, None, 0)
