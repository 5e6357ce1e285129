"""The losses where each group of blocks walks several rows that count, and their calls'
other duties.  Tolerances as in test_gpu_losses.py."""

from __future__ import annotations

import pytest
import torch
from test_gpu_losses import (IGN, _check_grad, _logits, _logp_tol, _policy_inputs, _policy_ref,
                             _policy_tol, _ref_logp)

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
