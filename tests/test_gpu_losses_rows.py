"""The losses where each group of blocks walks several rows that count, and their calls'
other duties.  Tolerances as in test_gpu_losses.py."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from test_gpu_losses import (IGN, _check_grad, _logits, _logp_tol, _policy_inputs, _policy_ref,
                             _policy_tol, _ref_logp)

import mhc_b200
from mhc_b200 import _capi

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


# (type, V, blocks that share a row, groups of blocks an SM holds): every thread count, whole
# and split rows, rows on and off 16-byte boundaries
SUMS = [(BF16, 512, 1, 12), (BF16, 12000, 1, 6), (BF16, 32000, 1, 3), (F32, 511, 1, 12),
        (F16, 50001, 2, 1.5), (F16, 50000, 2, 1.5), (F32, 50001, 4, 0.75), (F32, 50000, 4, 0.75)]
POLICY = [(BF16, 512, 1, 8), (BF16, 12000, 1, 4), (BF16, 32000, 1, 2), (F32, 511, 1, 8),
          (F16, 50001, 2, 1), (F16, 50000, 2, 1), (F32, 50001, 4, 0.5), (F32, 50000, 4, 0.5)]


def _rows_for(per_sm, counted):
    """Rows of which `counted` (a share) leave each group five or more."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return int(5.5 * per_sm * sms / counted) + 1


def _mask(y):
    """A third of the rows ignored: every fifth, and runs of them."""
    t = torch.arange(y.shape[0], device=DEV)
    y[(t % 5 == 1) | (t % 37 < 5)] = IGN
    keep = float((y != IGN).double().mean())
    assert 0.6 < keep < 0.8
    return y


def _chunks(T, V):
    step = max(1, (1 << 25) // V)
    return [slice(a, min(T, a + step)) for a in range(0, T, step)]


@pytest.mark.parametrize("dtype,V,share,per_sm", SUMS)
def test_sums_and_gradients_of_many_rows(dtype, V, share, per_sm):
    T = _rows_for(per_sm, 0.65)
    x, y = _logits((T, V), dtype, V + share)
    _mask(y)
    d = torch.randn(T, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5))
    x.requires_grad_(True)
    lp = mhc_b200.token_logprobs(x, y)
    lp.backward(d)
    for s in _chunks(T, V):
        x64 = x.detach()[s].double().requires_grad_(True)
        ref = _ref_logp(x64, y[s])
        ref.backward(d[s].double())
        assert ((lp[s].double() - ref).abs() <= _logp_tol(x.detach()[s], y[s])).all()
        _check_grad(x.grad[s], x64.grad, 0.0, dtype)
        ignored = y[s] == IGN
        assert not lp[s][ignored].any() and not x.grad[s][ignored].any()


@pytest.mark.parametrize("dtype,V,share,per_sm", POLICY)
def test_policy_loss_of_many_rows(dtype, V, share, per_sm):
    T = _rows_for(per_sm, 0.65)
    x, y = _logits((T, V), dtype, V + share + 1)
    parts = [_policy_inputs(x[s], y[s], i) for i, s in enumerate(_chunks(T, V))]
    old, ref, adv = (torch.cat([p[k] for p in parts]) for k in range(3))
    _mask(y)
    n = int((y != IGN).sum())
    r = mhc_b200.policy_loss_grad(x, y, old, adv, ref_logprobs=ref, clip_high=0.28, kl_coef=0.05,
                                  grad_scale=float(n))
    loss = kl = tol = 0.0
    for s in _chunks(T, V):
        x64 = x[s].double().requires_grad_(True)
        u, lp, k = _policy_ref(x64, y[s], old[s], adv[s], ref[s], 0.05, d=1.0)
        u.backward()
        t = _policy_tol(x[s], y[s], adv[s], old[s], ref[s])
        loss, kl, tol = loss + float(u), kl + float(k), max(tol, t)
        assert ((r.logprobs[s].double() - lp).abs() <= _logp_tol(x[s], y[s])).all()
        _check_grad(r.dlogits[s], x64.grad, t * 4, dtype)
    assert abs(float(r.loss) - loss / n) <= tol * (float(adv.abs().max()) * 4 + 1)
    assert abs(float(r.kl) - kl / n) <= tol * 4


@pytest.mark.parametrize("dtype,V", [(BF16, 32000), (F32, 12001), (F16, 511)])
def test_preference_loss_of_many_rows(dtype, V):
    per_sm = {32000: 3, 12001: 3, 511: 12}[V]
    T = _rows_for(per_sm, 0.65)
    x, y = _logits((T, V), dtype, V)
    ref = torch.cat([_ref_logp(x[s].double(), y[s]).float() for s in _chunks(T, V)])
    ref += 0.1 * torch.randn(T, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    _mask(y)
    cu = [0, T // 9, T // 3, T // 3 + 1, T // 2, T - 700, T]
    beta, pairs = 0.01, 3
    lp = torch.cat([_ref_logp(x[s].double(), y[s]) for s in _chunks(T, V)])
    delta = torch.where(y != IGN, lp - ref.double(), torch.zeros_like(lp))
    R = torch.stack([delta[a:b].sum() for a, b in zip(cu[:-1], cu[1:])])
    z = beta * (R[0::2] - R[1::2])
    tol = max(float(_logp_tol(x[s], y[s]).max()) for s in _chunks(T, V))
    dz = beta * max(b - a for a, b in zip(cu[:-1], cu[1:])) * 2 * tol + 2.0 ** -22
    r = mhc_b200.preference_loss_grad(x, y, ref, torch.tensor(cu, device=DEV), beta=beta)
    assert ((r.margins.double() - z).abs() <= dz * (1 + z.abs())).all()
    # loss and gradient follow from the margins
    z = r.margins.double()
    want = torch.nn.functional.softplus(-z).sum() / pairs
    assert abs(float(r.loss) - float(want)) <= 2.0 ** -22 * (1 + float(want))
    c = torch.zeros_like(lp)
    slope = (torch.sigmoid(z) - 1) * beta / pairs
    for k in range(6):
        c[cu[k]:cu[k + 1]] = slope[k // 2] * (1 if k % 2 == 0 else -1)
    for s in _chunks(T, V):
        x64 = x[s].double().requires_grad_(True)
        _ref_logp(x64, y[s]).backward(c[s])
        assert ((r.logprobs[s].double() - lp[s]).abs() <= _logp_tol(x[s], y[s])).all()
        _check_grad(r.dlogits[s], x64.grad, 2.0 ** -20, dtype)


@pytest.mark.parametrize("dtype,V", [(BF16, 8), (F32, 3), (F16, 512)])
def test_policy_workspace_is_large_enough(dtype, V):
    """More rows than blocks can be resident: nothing past the workspace is written."""
    T = 40000
    x, y = _logits((T, V), dtype, V)
    z = torch.zeros(T, device=DEV)
    logp, stats, coef = torch.empty(T, device=DEV), torch.empty(4 * T, device=DEV), torch.empty(T, device=DEV)
    loss, kl = torch.empty((), device=DEV), torch.empty((), device=DEV)
    size = _capi.query("mhc_policy_workspace_bytes")
    ws = torch.full((size + 65536,), 0xA5, dtype=torch.uint8, device=DEV)
    p = lambda t: t.data_ptr()  # noqa: E731
    _capi.call("mhc_policy_loss", p(x), _capi.dtype_code(dtype), T, T, 0, V, V, p(y), -100, p(z), p(z),
               None, 0.2, 0.2, 0.0, 0.0, 1.0, p(logp), p(stats), p(coef), p(loss), p(kl), None, p(ws),
               size, torch.cuda.current_stream().cuda_stream)
    assert (ws[size:] == 0xA5).all() and torch.isfinite(loss)


def test_forward_mode_is_refused():
    x, y = _logits((6, 40), F32, 1)
    z = torch.zeros(6, device=DEV)
    cu = torch.tensor([0, 3, 6], device=DEV)
    with fwAD.dual_level():
        d, e = (fwAD.make_dual(t, torch.ones_like(t)) for t in (x, z))
        for call in (lambda: mhc_b200.token_logprobs(d, y), lambda: mhc_b200.preference_loss(d, y, z, cu),
                     lambda: mhc_b200.preference_loss_grad(d, y, z, cu),
                     lambda: mhc_b200.preference_loss_grad(x, y, e, cu),
                     lambda: mhc_b200.policy_loss(d, y, z, z), lambda: mhc_b200.policy_loss_grad(d, y, z, z),
                     lambda: mhc_b200.policy_loss_grad(x, y, z, e)):
            with pytest.raises(RuntimeError, match="forward-mode|jvp"):
                call()


@pytest.mark.parametrize("V", [512, 32000, 131072])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sums_are_not_off_in_the_mean(dtype, V):
    """The hardware's exponential is low by 5e-8 in the mean, and a term meets up to three.
    That is taken out of the exponents: rows like a model's logits keep half of one at most,
    rows whose sum falls to a few terms or to one power of two, none of whose errors the
    correction was made for, two."""
    n = min(4096, (1 << 27) // V)
    g = torch.Generator(device=DEV).manual_seed(V)
    r = lambda m: torch.randn(n, m, device=DEV, generator=g)  # noqa: E731
    y = torch.zeros(n, dtype=torch.int64, device=DEV)
    rows = {"spread 2": (2 * r(V), 2.5e-8), "spread 1": (r(V), 1e-7), "spread 5": (5 * r(V), 1e-7),
            "flat": (torch.full((n, V), 1.25, device=DEV), 1e-7),
            "even": (-20 * torch.rand(n, V, device=DEV, generator=g), 1e-7),
            "one high": (torch.cat([r(V - 1), 12 + r(1)], 1), 1e-7)}
    for name, (x, most) in rows.items():
        x = x.to(dtype)
        logp, stats = _capi.host().token_logprobs(x, y, IGN)
        got = logp.double() + stats.view(n, 4)[:, 3].double()  # with its low part
        want = torch.cat([torch.log_softmax(x[s].double(), 1)[:, 0] for s in _chunks(n, V)])
        off = got - want
        # the mean's own spread, four times over
        spread = 4 * float(off.std()) / n ** 0.5
        assert abs(float(off.mean())) <= most + spread, (name, float(off.mean()))
