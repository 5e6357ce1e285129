"""Calls of the tuning operators, as far as they go without a GPU."""

from __future__ import annotations

import pytest
import torch

from mhc_b200 import FusedLinear, QuantizedLinear, _capi


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
