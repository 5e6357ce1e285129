"""What a step of AdamW does beside its arithmetic, and the arithmetic at the ends of the
types' ranges.  Tolerances as in test_gpu_adamw.py."""

from __future__ import annotations


import pytest
import torch

import mhc_b200

pytestmark = pytest.mark.gpu
DEV = "cuda"


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
