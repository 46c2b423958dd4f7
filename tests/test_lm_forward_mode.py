"""
Forward-mode differentiation: the layers over the kernel library have no
tangents, so an input that carries one is refused instead of losing it.
"""

from __future__ import annotations

import pytest

import kt_ops
import tuned_modules as tm

torch = pytest.importorskip("torch")

fwd = torch.autograd.forward_ad


def dual(x):
    return fwd.make_dual(x, torch.ones_like(x))


def test_layers_without_a_gradient():
    lin = tm.TunedLinear(64, 8)
    w4 = tm.TunedLinearW4(kt_ops.W4Weight(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 1), None, 64))
    for layer in (lin, w4):
        with fwd.dual_level(), torch.no_grad():
            with pytest.raises(RuntimeError, match="forward-mode"):
                layer(dual(torch.zeros(2, 64)))
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # without a tangent: the device
            layer(torch.zeros(2, 64))


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_differentiable_layers(dev, lib, t):
    ln = tm.TunedLayerNorm(64).to(dev)
    x = torch.randn(6, 64, device=dev).to(t)
    target = torch.zeros(6, dtype=torch.int64, device=dev)
    calls = [lambda v: ln(v), lambda v: tm.token_log_probs(v, target).logprob, lambda v: tm.token_log_probs(v).entropy]
    for recording in (True, False):
        ln.requires_grad_(recording)
        for f in calls:
            for mode in (torch.enable_grad, torch.no_grad):
                with fwd.dual_level(), mode():
                    with pytest.raises(NotImplementedError):
                        f(dual(x))
                    assert f(x).isfinite().all()  # a plain input inside a level
            with pytest.raises((NotImplementedError, RuntimeError)):
                torch.func.jvp(f, (x,), (torch.ones_like(x),))
