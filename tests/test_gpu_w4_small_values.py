"""
Products of very small fp32 tokens with 4-bit weights. A token is split into three
bf16 numbers, exactly while its last bit is at least bf16's least, 2^-133 (so from
2^-110 on); below, it is off by less than 2^-133. The sums are kept over 64, where fp32's
least is 2^-149: each of at most 3 K / 16 + K / 32 + 16 additions may lose as much, and
comes back 64 times a scale.
"""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import kt_ops  # noqa: E402
from test_gpu_w4 import make, values  # noqa: E402


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("power", [-100, -109, -115, -120, -126, -132])
def test_small_tokens(dev, lib, power, group):
    x, w, _ = make(dev, 5, 70, 640, group, torch.float32)
    x = (x.double() * 2.0 ** power).float()
    y = kt_ops.w4_linear(x, w, lib=lib)
    v, xd, k = values(w), x.double(), x.shape[1]
    want = xd @ v.T
    tol = 2.0 ** -24 * want.abs() + (32 + k / 32) * 2.0 ** -22 * (xd.abs() @ v.abs().T)
    tol += (3 * k / 16 + k / 32 + 16) * 2.0 ** -143 * w.scales.double().amax(1) + 2.0 ** -149
    tol += 2.0 ** -133 * ((xd.abs() < 2.0 ** -110).double() @ v.abs().T)
    assert bool(((y.double() - want).abs() <= tol).all())
