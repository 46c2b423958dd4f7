"""
What the torch layers of a language model's output end give to autograd: the
gradients of lse and of targets that are no column, and forward mode, which they
do not have and refuse.
"""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import kt_ops  # noqa: E402
import tuned_modules as tm  # noqa: E402
from test_gpu_logprob_gradient import TYPES, case, check  # noqa: E402


@pytest.mark.parametrize("t", TYPES)
def test_impossible_targets_have_no_gradient_but_nan(dev, lib, t):
    """The log probability of a target that is no column is NaN, and so is what
    it gives the logits; with a gradient of 0 nothing is asked of it."""
    x, targets, g, h = case(dev, 8, 600)
    x = x.to(t)
    bad = targets.clone()
    bad[2], bad[5] = 600, -1
    wrong = torch.zeros(8, dtype=torch.bool, device=dev)
    wrong[2] = wrong[5] = True
    r = kt_ops.token_logprobs(x, bad, lib=lib)
    assert lib.device_error(reset=True) == 2 and torch.equal(r.logprob.isnan(), wrong)
    whole = kt_ops.token_logprobs(x, targets, lib=lib)
    for a, b in ((g, h), (g, None)):
        dx = kt_ops.token_logprobs_bwd(x, bad, r, a, b, lib=lib)
        assert dx[wrong].isnan().all()
        assert torch.equal(dx[~wrong], kt_ops.token_logprobs_bwd(x, targets, whole, a, b, lib=lib)[~wrong])
    off = torch.where(wrong, 0.0, g)
    assert kt_ops.token_logprobs_bwd(x, bad, r, off, None, lib=lib)[wrong].eq(0).all()
    dx = kt_ops.token_logprobs_bwd(x, bad, r, off, h, lib=lib)  # the entropy's part alone
    assert torch.equal(dx[wrong], kt_ops.token_logprobs_bwd(x, bad, r, None, h, lib=lib)[wrong])
    assert dx.isfinite().all()


@pytest.mark.parametrize("rows,V", [(24, 1003), (400, 1003), (3, 40000)])
@pytest.mark.parametrize("offset", [0.0, 1e4])
def test_gradient_of_lse(dev, lib, rows, V, offset):
    x, targets, g, h = case(dev, rows, V, offset)
    l = torch.linspace(-1, 1, rows, device=dev)
    for a, b in ((None, None), (g, None), (None, h), (g, h)):
        check(x, targets, 0.7, a, b, lib, l=l)
    with pytest.raises(ValueError):
        kt_ops.token_logprobs_bwd(x, targets, kt_ops.token_logprobs(x, targets, lib=lib), lib=lib, grad_lse=l[1:])


@pytest.mark.parametrize("t", TYPES)
def test_loss_with_a_term_of_lse(dev, lib, t):
    """A cross entropy with a squared lse beside it, as autograd runs it."""
    x, targets, _, _ = case(dev, 30, 500)
    x = x.to(t).view(5, 6, 500)
    targets = targets.view(5, 6).clone()
    targets[1, 2] = -100
    x.requires_grad_()
    r = tm.token_log_probs(x, targets, top_k=2)
    assert not r.top_logprob.requires_grad and not r.top_index.requires_grad
    (-r.logprob.mean() + 0.01 * r.lse.square().mean()).backward()
    xd = x.detach().double().requires_grad_()
    lse = torch.logsumexp(xd, -1)
    lp = torch.where(targets >= 0, xd.gather(-1, targets.clamp(min=0)[..., None])[..., 0] - lse, 0.0)
    (-lp.mean() + 0.01 * lse.square().mean()).backward()
    want, off = xd.grad, 2.0 ** -24 * 300 * (xd.grad.abs() + torch.softmax(xd.detach(), -1) / 30)
    # 300 steps: what L of the gradient's own tests comes to at 500 columns within 20 of the largest
    step = torch.finfo(t).eps / 2 * want.abs() + torch.finfo(t).tiny * torch.finfo(t).eps
    assert bool(((x.grad.double() - want).abs() <= off + step).all())
    x.grad = None
    tm.token_log_probs(x).lse.sum().backward()  # lse alone: the probabilities
    p = torch.softmax(x.detach().double(), -1)
    tol = (torch.finfo(t).eps / 2 + 300 * 2.0 ** -24) * p + torch.finfo(t).tiny * torch.finfo(t).eps
    assert bool(((x.grad.double() - p).abs() <= tol).all())


def test_lse_gradient_against_differences(dev, lib):
    x, targets, g, h = case(dev, 5, 60)
    l = torch.linspace(-1, 1, 5, device=dev)
    r = kt_ops.token_logprobs(x, targets, scale=0.7, lib=lib)
    dx = kt_ops.token_logprobs_bwd(x, targets, r, scale=0.7, lib=lib, grad_lse=l).double()
    gen = torch.Generator(device=dev).manual_seed(5)
    d = 1e-5
    for _ in range(4):
        step = torch.randn(5, 60, dtype=torch.float64, device=dev, generator=gen)
        up, down = (float((l.double() * torch.logsumexp(0.7 * (x.double() + s * step), 1)).sum()) for s in (d, -d))
        # differences: d^2 and 2^-52/d of values of order 50; fp32: 2^-16 of the magnitudes
        assert abs((up - down) / (2 * d) - float((dx * step).sum())) <= 2.0 ** -16 * float((dx * step).abs().sum()) + 1e-7
