"""
The gradient of token log probabilities and entropies where the logits lie far
from 0, and of rows masked by the type's lowest value, against the formulas in
64 bits.

Tolerances, with E = 2^-24, z = scale x, a = |z - zmax|, S the mean of a under p
and n = V/256 + 64 additions in a row: an exponent (x - m) scale log2 e has four
roundings (4 E a) and the exponential 2^-22 = 4 E, so the sum of exponentials is
off by E (n + 4 + 4 S) of itself, its logarithm by 2 E log V more, and a
probability, whose own exponent has the same roundings and that of the
logarithm's subtraction, by L = E (n + 12 + 4 S + 4 a + 4 |log p| + 4 log V) of
itself. No term goes with |z|: a common offset changes nothing. Each gradient is
then off by p times its factors times L, and rounded once to its type.
"""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import kt_ops  # noqa: E402

E = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def formula(x, targets, scale, g, h, l=None):
    """Gradient in 64 bits, and what it may be off by before it is rounded."""
    rows, V = x.shape
    z = x.double() * torch.tensor(scale, dtype=torch.float32).double().item()
    a = z.amax(1, keepdim=True) - z
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    far = torch.where(p > 0, logp.abs(), 0.0)
    a = torch.where(p > 0, a, 0.0)
    H = (p * far).sum(1, keepdim=True)
    S = (p * a).sum(1, keepdim=True)
    zero = torch.zeros(rows, device=x.device)
    G, K, L2 = ((v if v is not None else zero).double()[:, None] for v in (g, h, l))
    at = torch.arange(V, device=x.device) == targets[:, None]
    want = scale * (G * at - p * (G - L2 + K * (H - far)))
    n = V / 256 + 64
    L = E * (n + 12 + 4 * S + 4 * a + 4 * far + 4 * math.log(V))
    tol_h = E * (n + 16) * (2 + 2 * S)
    off = scale * p * ((G.abs() + L2.abs() + K.abs() * (far + H)) * (L + 8 * E) + K.abs() * (L + tol_h + 4 * E * (far + H)))
    off = off + scale * 4 * E * G.abs() * at
    # the exponential flushes p < 2^-126 to 0
    return want, off + scale * 2.0 ** -126 * (G.abs() + L2.abs() + K.abs() * (104 + H))


def check(x, targets, scale, g, h, lib, l=None):
    r = kt_ops.token_logprobs(x, targets, scale=scale, lib=lib)
    kw = {} if l is None else {"grad_lse": l}
    dx = kt_ops.token_logprobs_bwd(x, targets, r, g, h, scale=scale, lib=lib, **kw)
    want, off = formula(x, targets, scale, g, h, l)
    t = torch.finfo(x.dtype)
    step = t.eps / 2 * want.abs() + t.tiny * t.eps
    over = float(((dx.double() - want).abs() / (off + step)).max())
    assert over <= 1, over
    return dx, want, off + step


def case(dev, rows, V, offset=0.0, spread=2.5, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + rows * 31 + V)
    x = torch.randn(rows, V, device=dev, generator=gen) * spread
    targets = torch.randint(0, V, (rows,), device=dev, generator=gen)
    x[torch.arange(rows, device=dev), targets] += spread * torch.rand(rows, device=dev, generator=gen)
    g = torch.randn(rows, device=dev, generator=gen)
    h = torch.randn(rows, device=dev, generator=gen) * 0.3
    return x + offset, targets, g, h


@pytest.mark.parametrize("rows,V", [(24, 1003), (400, 1003), (3, 40000)])  # CTAs, single warps, clusters
@pytest.mark.parametrize("offset", [0.0, -30.0, 1e3, -1e4, 1e5, 3e30])
def test_common_offset(dev, lib, rows, V, offset):
    x, targets, g, h = case(dev, rows, V, offset)
    for a, b in ((g, None), (None, h), (g, h)):
        check(x, targets, 1.0, a, b, lib)


@pytest.mark.parametrize("offset", [0.0, 1e3, 1e5])
def test_rows_of_the_gradient_add_up_to_zero(dev, lib, offset):
    x, targets, g, _ = case(dev, 64, 2000, offset)
    dx, want, tol = check(x, targets, 1.0, g, None, lib)
    assert bool((dx.double().sum(1).abs() <= tol.sum(1)).all())


def test_large_scale(dev, lib):
    x, targets, g, h = case(dev, 24, 1003, offset=7.0, spread=2.5e-3)
    check(x, targets, 1e3, g, h, lib)
    check(x, targets, 1e6, g, h, lib)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,V", [(5, 1000), (500, 1000), (1, 50000)])
def test_rows_masked_by_the_lowest_value(dev, lib, rows, V, t):
    """A row of nothing but the type's lowest value is uniform; -inf alone has no distribution."""
    low = torch.finfo(t).min
    x = torch.full((rows, V), low, device=dev, dtype=t)
    targets = torch.arange(rows, device=dev) % V
    g = torch.linspace(0.5, 1.5, rows, device=dev)
    h = torch.linspace(-0.3, 0.3, rows, device=dev)
    for scale in (1.0, 2.0):  # 2: scale x is past fp32's range
        dx, _, _ = check(x, targets, scale, g, h, lib)
        assert dx[:, -1].ne(0).all()
    r = kt_ops.token_logprobs(x, targets, scale=2.0, lib=lib)
    assert bool(((r.logprob + math.log(V)).abs() <= E * (V / 256 + 96) * 8 + 4 * E * math.log(V)).all())


@pytest.mark.parametrize("t", TYPES)
def test_results_put_together_anew(dev, lib, t):
    """A result that lost its norm has it computed again; a wrong one is refused."""
    x, targets, g, h = case(dev, 12, 1003, offset=100.0)
    x = x.to(t)
    r = kt_ops.token_logprobs(x, targets, top_k=2, scale=0.9, lib=lib)
    logprob, entropy, lse, top, index = r
    want = kt_ops.token_logprobs_bwd(x, targets, r, g, h, scale=0.9, lib=lib)
    for again in (kt_ops.TokenLogprobs(*r), r._replace(lse=lse + 1), kt_ops.TokenLogprobs(None, entropy, lse, top, index)):
        assert again.norm is None
        assert torch.equal(kt_ops.token_logprobs_bwd(x, targets, again, g, h, scale=0.9, lib=lib), want)
    for norm in (r.norm.cpu(), r.norm.double(), r.norm[:5], r.norm.t()):
        again.norm = norm
        with pytest.raises(ValueError):
            kt_ops.token_logprobs_bwd(x, targets, again, g, h, scale=0.9, lib=lib)


def test_gradient_from_lse(dev, lib):
    """kt_token_logprobs and kt_token_logprobs_bwd, without the norm: near 0 the
    same but for 2^-24 of |lse|."""
    x, targets, g, h = case(dev, 40, 1003)
    rows, V = x.shape
    out = [torch.empty(rows, device=dev) for _ in range(3)]
    at = torch.cuda.current_stream().cuda_stream
    lib.token_logprobs(x.data_ptr(), V, targets.data_ptr(), rows, V, 1.0, -100, 0, *(v.data_ptr() for v in out), None,
                       None, 0, at)
    r = kt_ops.token_logprobs(x, targets, lib=lib)
    assert all(torch.equal(a, b) for a, b in zip(out, r))
    dx = torch.empty_like(x)
    lib.token_logprobs_bwd(x.data_ptr(), V, targets.data_ptr(), out[2].data_ptr(), out[1].data_ptr(), g.data_ptr(),
                           h.data_ptr(), rows, V, 1.0, -100, dx.data_ptr(), V, 0, at)
    want, off = formula(x, targets, 1.0, g, h)
    # a factor 1 + 2^-24 |lse| on each probability, and as much in the entropy's term
    z = x.double()
    lse = torch.logsumexp(z, 1, keepdim=True).abs()
    p = torch.softmax(z, 1)
    far = torch.log_softmax(z, 1).abs()
    H = (p * far).sum(1, keepdim=True)
    more = p * 2 * E * lse * (g.abs()[:, None] + h.abs()[:, None] * (far + H + 1))
    assert bool(((dx.double() - want).abs() <= off + more + E * want.abs() + 2.0 ** -149).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,V", [(8, 700), (400, 700), (8, 30000)])
def test_rows_that_are_not_finite(dev, lib, rows, V, t):
    """A NaN or +inf makes a row's gradient NaN, whatever else the row holds; a row
    of only -inf has none."""
    x, targets, g, h = case(dev, rows, V)
    x = x.to(t)
    whole = kt_ops.token_logprobs(x, targets, lib=lib)
    x[1] = float("nan")
    x[2], x[2, V - 1] = -math.inf, float("nan")
    x[3, 5] = math.inf
    x[4, 6], x[4, 7] = float("nan"), math.inf
    x[5] = -math.inf
    x[6] = math.inf
    r = kt_ops.token_logprobs(x, targets, lib=lib)
    l = torch.ones(rows, device=dev)
    rest = torch.ones(rows, dtype=torch.bool, device=dev)
    rest[1:7] = False
    for a, b, c in ((g, None, None), (None, h, None), (None, None, l), (g, h, l)):
        dx = kt_ops.token_logprobs_bwd(x, targets, r, a, b, lib=lib, grad_lse=c)
        assert dx[[1, 2, 3, 4, 6]].isnan().all() and dx[5].eq(0).all()
        assert torch.equal(dx[rest], kt_ops.token_logprobs_bwd(x, targets, whole, a, b, lib=lib, grad_lse=c)[rest])
    zero = torch.zeros(rows, device=dev)
    assert kt_ops.token_logprobs_bwd(x, targets, r, zero, zero, lib=lib, grad_lse=zero).eq(0).all()


@pytest.mark.parametrize("rows,V", [(24, 1003), (400, 1003), (3, 40000)])
@pytest.mark.parametrize("offset", [0.0, 1e3, -1e5, 3e30])
def test_values_at_a_common_offset(dev, lib, rows, V, offset):
    """Log probabilities and entropies are off by what goes with |z - zmax|, not with |z|."""
    x, targets, _, _ = case(dev, rows, V, offset)
    r = kt_ops.token_logprobs(x, targets, top_k=4, lib=lib)
    z = x.double()
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    a = z.amax(1, keepdim=True) - z
    S = torch.where(p > 0, p * a, 0.0).sum(1, keepdim=True)
    H = -torch.where(p > 0, p * logp, 0.0).sum(1)
    n = V / 256 + 64
    L = E * (n + 12 + 4 * S + 4 * a + 4 * logp.abs() + 4 * math.log(V))
    index = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(r.top_index, index)
    for got, at in ((r.logprob[:, None], targets[:, None]), (r.top_logprob, index)):
        assert bool(((got.double() - logp.gather(1, at)).abs() <= L.gather(1, at)).all())
    assert bool(((r.entropy.double() - H).abs() <= E * (n + 16) * (2 + 2 * S[:, 0])).all())
