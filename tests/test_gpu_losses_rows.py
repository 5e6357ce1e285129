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
