"""Calls of the linear layer that its kernels do not see, and its gradients' digits.
Tolerances as in test_gpu_linear.py, but for the slope: it comes from the pre-activation in
fp32, so nothing is allowed for a rounding of z."""

from __future__ import annotations

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from test_gpu_linear import ACT, EPS, TINY, U, _make, _within

from mhc_b200 import FusedLinear, _capi, linear_act, token_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 64), (13, 1500, 72), (17, 1501, 72), (40, 2050, 100),
                                   (300, 1000, 40), (1000, 777, 33)])
def test_slopes_come_from_the_pre_activation_in_fp32(dtype, act, M, N, K):
    """dbias is a sum of dz in fp32: u of itself, and the slope's own error.  A z rounded to
    the type would add 0.3 u |dy| a row, most of it where the slope goes through 0."""
    x, w, b, res, dy = _make(M, N, K, dtype, M + N)
    bias = b.clone().requires_grad_(True)
    y = linear_act(x, w, bias, residual=res, activation=act)
    (db,) = torch.autograd.grad(y, bias, dy)
    X, W, D = x.double(), w.double(), dy.double()
    z = (X @ W.t() + b.double()).requires_grad_(True)
    size = X.abs() @ W.abs().t() + b.double().abs()
    (slope,) = torch.autograd.grad(ACT[act](z).sum(), z)
    dz = D * slope
    noise = EPS * D.abs() * (1 + size)
    want = dz.sum(0)
    _within(db, want, noise.sum(0) + EPS * dz.abs().sum(0) + U[dtype] * want.abs() + TINY[dtype] + 1e-30, "db")


def test_forward_mode_is_refused():
    """An output without a tangent would be taken for a constant."""
    x, w, b, res, dy = _make(20, 24, 16, torch.bfloat16, 1)
    for i in range(4):
        for M in (1, 20):
            for grad in (False, True):
                with fwAD.dual_level(), torch.set_grad_enabled(grad):
                    ts = [x[:M], w, b, res[:M]]
                    ts[i] = fwAD.make_dual(ts[i], torch.ones_like(ts[i]))
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        linear_act(*ts[:3], residual=ts[3], activation="silu")
    with fwAD.dual_level():
        linear_act(x, w, b, residual=res)  # none of them dual
        leaf = x.clone().requires_grad_()
        y = linear_act(leaf, w)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, leaf, fwAD.make_dual(dy, torch.ones_like(dy)))


@pytest.mark.parametrize("dtype", list(U))
def test_autocast(dtype):
    """Under autocast the operands take its type, as nn.Linear's do."""
    torch.manual_seed(0)
    for own in (torch.float32, torch.bfloat16):
        lin = FusedLinear(48, 40, activation="gelu", device=DEV, dtype=own)
        x = torch.randn(6, 48, device=DEV, requires_grad=True)
        r = torch.randn(6, 40, device=DEV, requires_grad=True)
        with torch.autocast("cuda", dtype=dtype):
            y = lin(x, residual=r)
            like = torch.nn.Linear(48, 40, device=DEV)(x)
        assert y.dtype == like.dtype == dtype
        cast = [t.detach().to(dtype).requires_grad_() for t in (x, lin.weight, lin.bias, r)]
        z = linear_act(*cast[:3], residual=cast[3], activation="gelu")
        assert torch.equal(y, z)
        y.float().square().sum().backward()
        z.float().square().sum().backward()
        for a, c in zip((x, lin.weight, lin.bias, r), cast):
            assert a.grad.dtype == a.dtype and torch.equal(a.grad, c.grad.to(a.dtype))
    with torch.autocast("cuda", dtype=dtype, enabled=False), pytest.raises(ValueError, match="float16 or"):
        lin(x)
    with torch.autocast("cuda", dtype=dtype), pytest.raises(ValueError, match="dtype"):
        linear_act(x.double(), lin.weight)


def test_more_rows_than_a_grid_has():
    """8.4 million rows: more blocks of 128 rows than the second axis of a grid takes."""
    M, N, K = 65535 * 128 + 77, 8, 8
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g).to(torch.bfloat16)  # noqa: E731
    x, w, b, dy = (t.requires_grad_(i < 3) for i, t in enumerate((r(M, K), r(N, K), r(N), r(M, N))))
    y = linear_act(x, w, b, activation="relu")
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    with torch.no_grad():
        z = x.double() @ w.double().t() + b.double()
        size = x.double().abs() @ w.double().abs().t() + b.double().abs()
        dz = dy.double() * (z > 0)
        # a z that is 0 to within its error may fall on either side
        edge = torch.where(z.abs() <= 2 * EPS * size, dy.double().abs(), torch.zeros_like(z))
        u = U[torch.bfloat16]
        rounded = edge + u * dz.abs()
        for name, got, want, tol in (
                ("dx", dx, dz @ w.double(), rounded @ w.double().abs() + EPS * (dz.abs() @ w.double().abs())),
                ("dw", dw, dz.t() @ x.double(),
                 rounded.t() @ x.double().abs() + EPS * (dz.abs().t() @ x.double().abs())),
                ("db", db, dz.sum(0), edge.sum(0) + EPS * dz.abs().sum(0))):
            _within(got, want, tol + u * want.abs() + 1e-30, name)
    torch.cuda.empty_cache()


def test_a_call_that_fails_raises_the_packages_error():
    """In the forward, and in the backward on the autograd engine's thread; the entry points
    are replaced by ones that return a status, so no kernel runs."""
    host, lib = _capi.host(), _capi.load()
    names = ["mhc_linear_fwd_workspace_bytes", "mhc_linear_fwd", "mhc_linear_bwd_workspace_bytes",
             "mhc_linear_bwd", "mhc_token_logprobs", "mhc_logits_grad", "mhc_preference_loss",
             "mhc_policy_workspace_bytes", "mhc_policy_loss", "mhc_last_error"]
    real = [ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names]
    x, w, *_ = _make(20, 24, 16, torch.bfloat16, 1)
    x.requires_grad_(True)
    y = linear_act(x, w)
    logits, targets = torch.zeros(4, 8, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    fail = ctypes.CFUNCTYPE(ctypes.c_int)(lambda: _capi.MHC_ERR_UNSUPPORTED)
    fake = [ctypes.cast(fail, ctypes.c_void_p).value if "bytes" not in n and "error" not in n else a
            for n, a in zip(names, real)]
    host.bind(*fake, _capi.MHCError)
    try:
        for call, name in ((lambda: linear_act(x, w), "mhc_linear_fwd"), (y.sum().backward, "mhc_linear_bwd"),
                           (lambda: token_logprobs(logits, targets), "mhc_token_logprobs")):
            with pytest.raises(_capi.MHCError, match=name) as e:
                call()
            assert e.value.code == _capi.MHC_ERR_UNSUPPORTED
    finally:
        host.bind(*real, _capi.MHCError)
    linear_act(x, w).sum().backward()
