"""Calls of the tuning operators, as far as they go without a GPU."""

from __future__ import annotations

import pytest
import torch

import mhc_b200
from mhc_b200 import FusedLinear, QuantizedLinear, _capi


@pytest.mark.parametrize("bad", [float("inf"), 1e39, 1e300, 1e-39, float("nan")])
def test_denominators_whose_inverse_is_no_fp32_number(bad):
    """The inverse goes to the kernels in fp32, where 0 stands for the number of tokens."""
    x, y, z = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    cu = torch.tensor([0, 2, 4])
    for f in (mhc_b200.policy_loss, mhc_b200.policy_loss_grad):
        with pytest.raises(ValueError, match="denominator"):
            f(x, y, z, z, denominator=bad)
    for f in (mhc_b200.preference_loss, mhc_b200.preference_loss_grad):
        with pytest.raises(ValueError, match="denominator"):
            f(x, y, z, cu, denominator=bad)


def test_a_quantized_layer_keeps_no_activation():
    """QuantizedLinear has no activation: a FusedLinear with one is refused, not stripped of it."""
    plain = FusedLinear(64, 64, dtype=torch.float32)
    QuantizedLinear.from_linear(plain)
    with pytest.raises(ValueError, match="activation"):
        QuantizedLinear.from_linear(FusedLinear(64, 64, activation="silu", dtype=torch.float32))


def test_versions_go_up():
    """What a kernel has written through its address counts as changed in place."""
    host = _capi.host()
    a, b = torch.zeros(4), torch.nn.Parameter(torch.zeros(3))
    view = b.detach()[1:]
    with torch.inference_mode():
        c = torch.zeros(2)  # has no version
    host.changed([a, b, a, c])
    assert (a._version, b._version, view._version) == (2, 1, 1)
    for bad in (((a,),), ([a, 3],), ([a], 1), (a,)):
        with pytest.raises(TypeError):
            host.changed(*bad)
