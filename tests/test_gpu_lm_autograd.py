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
