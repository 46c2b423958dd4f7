"""
The torch layers refuse inputs whose last dimension is not theirs, on any device.
"""

from __future__ import annotations

import pytest

import kt_ops
import tuned_modules as tm

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("shape", [(4, 128), (4, 32), (2, 2, 96), (64, 1)])
def test_last_dimension(shape):
    """Several rows' worth of columns in one row, or a part of a row's, are no rows."""
    layers = [tm.TunedLayerNorm(64), tm.TunedLayerNorm(64, checkpoint8=True),
              tm.TunedLinearW4(kt_ops.W4Weight(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 1), None, 64))]
    for layer in layers:
        for mode in (torch.no_grad, torch.enable_grad):
            with mode(), pytest.raises(ValueError, match="64 columns"):
                layer(torch.zeros(shape))
