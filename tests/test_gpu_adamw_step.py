"""What a step of AdamW does beside its arithmetic, and the arithmetic at the ends of the
types' ranges.  Tolerances as in test_gpu_adamw.py."""

from __future__ import annotations


import pytest
import torch
from test_gpu_adamw import HYPER, _params, _set_grads

import mhc_b200

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("transposed", [False, True])
def test_a_step_is_an_in_place_change(bits, dtype, transposed):
    """A graph that saved a parameter cannot be differentiated once a step has changed it."""
    w = torch.randn(24, 16, device=DEV).to(dtype)
    p = torch.nn.Parameter(w.t() if transposed else w)
    opt = mhc_b200.AdamW([p], state_bits=bits, master_weights=True, **HYPER)
    loss = (p * p).sum()
    loss.backward(retain_graph=True)
    before = p._version, opt.state[p]["exp_avg"]._version
    opt.step()
    assert p._version > before[0] and opt.state[p]["exp_avg"]._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    q = torch.nn.Parameter(torch.ones(4, device=DEV))  # no gradient: left alone
    version = q._version
    mhc_b200.AdamW([q]).step()
    assert q._version == version


def test_a_step_between_two_backwards_of_a_linear_layer():
    lin = mhc_b200.FusedLinear(32, 48, activation="silu", device=DEV)
    x = torch.randn(20, 32, device=DEV).to(torch.bfloat16).requires_grad_()
    opt = mhc_b200.AdamW(lin.parameters())
    y = lin(x).float().sum()
    y.backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_capture_is_refused():
    """A captured step would repeat one step's bias corrections and rounding."""
    (p,) = _params([(300,)], torch.float32, 1)
    opt = mhc_b200.AdamW([p], state_bits=8, **HYPER)
    _set_grads([p], 2)
    opt.step()
    before = p.detach().clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captur"):
        with torch.cuda.graph(g):
            opt.step()
    assert opt.state_dict()["state"][0]["step"] == 1 and torch.equal(p.detach(), before)
    opt.step()
    assert not torch.equal(p.detach(), before)


def test_parameters_that_share_memory_are_refused():
    """Blocks of one launch would write the same values."""
    p = torch.nn.Parameter(torch.zeros(10, device=DEV))
    with pytest.warns(UserWarning, match="duplicate"), pytest.raises(ValueError, match="share memory"):
        mhc_b200.AdamW([p, p])
    flat = torch.zeros(100, device=DEV)
    part = lambda a, b: torch.nn.Parameter(flat[a:b])  # noqa: E731
    with pytest.raises(ValueError, match="share memory"):
        mhc_b200.AdamW([part(50, 100), part(0, 10), part(9, 20)])
    with pytest.raises(ValueError, match="share memory"):
        mhc_b200.AdamW([part(0, 100), part(10, 20), torch.nn.Parameter(flat[30:30])])
    mhc_b200.AdamW([part(50, 100), part(10, 50), part(0, 10), torch.nn.Parameter(flat[30:30])])
