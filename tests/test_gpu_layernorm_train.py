"""
LayerNorm for training on a GPU: forward and backward in three types, with and
without 8-bit checkpoints, against the formulas in 64 bits.

Tolerances. An output of type t is rounded once: eps(t)/2 of its size. Inside,
a sum of n fp32 terms by chains of at most c additions is off by at most
c 2^-24 of the sum of magnitudes. A row's sums are chains of at most
32 + cols/256 additions in a thread and 10 in the tree, and each term comes
from at most 8 roundings: K = 64 + cols/128 covers them. With
A = |xh| + rstd mean|x| the value xh is off by at most K 2^-24 A (the mean's
error is rstd mean|x| K 2^-24); the bounds below follow the formulas with that.
The weights' gradients are chains over rows/64 rows and at most 160 parts.
"""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import kt_lib  # noqa: E402
import kt_ops  # noqa: E402

E = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def rounded8(x):
    """(q, exponent codes, values) of the 8-bit checkpoint, in 64 bits."""
    r, c = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -c % 32)).view(r, -1, 32)
    top = b.abs().amax(-1)
    finite = torch.isfinite(b).all(-1)
    # frexp: 2^(e-1) <= top < 2^e, and the fp32 exponent field is e + 126
    code = (torch.frexp(torch.where(finite, top, 1.0)).exponent + 126).clamp(min=7)
    code = torch.where(top == 0, 7, code)
    step = torch.ldexp(torch.ones_like(top), code - 133).unsqueeze(-1)
    q = torch.where(finite.unsqueeze(-1), (b / step).round().clamp(-127, 127), 0.0)
    value = torch.where(finite.unsqueeze(-1), q * step, float("nan"))
    code = torch.where(finite, code, 255)
    return q.view(r, -1)[:, :c].to(torch.int8), code.to(torch.uint8), value.view(r, -1)[:, :c]


def check(x, dy, gamma, beta, eps=1e-5, ckpt8=False, lib=None):
    y, saved = kt_ops.layernorm_train(x, gamma, beta, eps, ckpt8=ckpt8, lib=lib)
    dx, dgamma, dbeta = kt_ops.layernorm_bwd(dy, saved, lib=lib)
    torch.cuda.synchronize()
    rows, cols = x.shape
    K = 64 + cols / 128
    xd, d = x.double(), dy.double()
    g = gamma.double() if gamma is not None else torch.ones(cols, dtype=torch.float64, device=x.device)
    b = beta.double() if beta is not None else torch.zeros(cols, dtype=torch.float64, device=x.device)
    mu = xd.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((xd - mu) ** 2).mean(1, keepdim=True) + eps)
    xh = (xd - mu) * r
    mag = r * xd.abs().mean(1, keepdim=True)

    def near(got, want, inner, name):
        assert got.dtype in TYPES
        tol = half_step(got.dtype) * want.abs() + inner + torch.finfo(got.dtype).tiny
        over = ((got.double() - want).abs() / tol).max()
        assert over <= 1, (name, float(over))

    near(saved.mean, mu[:, 0], K * E * xd.abs().mean(1), "mean")
    near(saved.rstd, r[:, 0], K * E * (r + r * mag * mag)[:, 0], "rstd")
    near(y, g * xh + b, K * E * ((xh.abs() + mag) * (1 + mag * mag) * g.abs() + b.abs()), "y")
    if ckpt8:
        q, code, xd = rounded8(x)
        assert torch.equal(saved.q8, q) and torch.equal(saved.q8_exp, code)
        assert saved.x is None
        xh = (xd - mu) * r
    A = xh.abs() + mag
    w = d * g
    c1, c2 = (w * xh).mean(1, keepdim=True), w.mean(1, keepdim=True)
    m1 = (w.abs() * A).mean(1, keepdim=True)
    near(dx, r * (w - c2 - xh * c1),
         K * E * r * (1 + mag * mag) * (w.abs() + w.abs().mean(1, keepdim=True) + 2 * A * m1), "dx")
    chain = K + rows / 64 + 160
    if gamma is not None:
        assert dgamma.dtype == gamma.dtype
        near(dgamma, (d * xh).sum(0), chain * E * (d.abs() * A * (1 + mag * mag)).sum(0), "dgamma")
    else:
        assert dgamma is None
    if beta is not None:
        assert dbeta.dtype == beta.dtype
        near(dbeta, d.sum(0), chain * E * d.abs().sum(0), "dbeta")
    else:
        assert dbeta is None
    return y, dx, dgamma, dbeta


def inputs(dev, rows, cols, t, wt=torch.float32, seed=0, offset=0):
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + rows * 31 + cols)

    def make(*shape):
        v = torch.randn(*shape, device=dev, generator=g)
        if offset == 0:
            return v.to(t)
        base = torch.empty(v.numel() + offset, dtype=t, device=dev)
        return base[offset:].view(shape).copy_(v)

    x, dy = make(rows, cols), make(rows, cols)
    gamma = (1 + 0.2 * torch.randn(cols, device=dev, generator=g)).to(wt)
    beta = (0.3 * torch.randn(cols, device=dev, generator=g)).to(wt)
    return x, dy, gamma, beta


SHAPES = [(1, 1), (1, 8), (2, 3), (3, 31), (5, 32), (7, 33), (9, 64), (17, 127), (64, 128), (3, 129), (40, 255),
          (33, 256), (19, 500), (11, 512), (13, 1023), (300, 1024), (21, 1025), (1500, 520), (8, 2047), (6, 2048),
          (5, 4096), (700, 4095), (4, 4097), (3, 8191), (2, 8192), (3, 8193), (2, 16384), (2, 16385), (1, 40000)]


@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_shapes(dev, lib, rows, cols, t, ckpt8):
    x, dy, gamma, beta = inputs(dev, rows, cols, t)
    check(x, dy, gamma, beta, ckpt8=ckpt8, lib=lib)
    assert lib.device_error() == 0


@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("t", TYPES[1:])
def test_weights_of_the_input_type(dev, lib, t, ckpt8):
    for rows, cols in ((37, 96), (5, 1000), (3, 4096)):
        x, dy, gamma, beta = inputs(dev, rows, cols, t, wt=t)
        check(x, dy, gamma, beta, ckpt8=ckpt8, lib=lib)


@pytest.mark.parametrize("t", TYPES)
def test_without_weights(dev, lib, t):
    x, dy, gamma, beta = inputs(dev, 70, 200, t)
    check(x, dy, None, None, lib=lib)
    check(x, dy, gamma, None, lib=lib)
    check(x, dy, None, beta, lib=lib)
    check(x, dy, None, beta.to(t), ckpt8=True, lib=lib)
    y, saved = kt_ops.layernorm_train(x, gamma, beta, lib=lib)
    dx, dgamma, dbeta = kt_ops.layernorm_bwd(dy, saved, weight_grads=False, lib=lib)
    assert dgamma is None and dbeta is None
    assert torch.equal(dx, kt_ops.layernorm_bwd(dy, saved, lib=lib)[0])


@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("offset", [1, 2, 3, 5])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_unaligned(dev, lib, offset, t, ckpt8):
    for rows, cols in ((9, 64), (50, 1000), (4, 4097)):
        check(*inputs(dev, rows, cols, t, offset=offset), ckpt8=ckpt8, lib=lib)
        # dy and x differ in their alignment
        x, dy, gamma, beta = inputs(dev, rows, cols, t, offset=offset)
        check(x.clone(), dy, gamma, beta, ckpt8=ckpt8, lib=lib)


@pytest.mark.parametrize("ckpt8", [False, True])
def test_large_offsets_and_outliers(dev, lib, ckpt8):
    x, dy, gamma, beta = inputs(dev, 64, 2048, torch.float32)
    x[:, 5] *= 500.0
    x[3] = 4.0  # a row of one value: variance 0
    x[4] = 0.0
    x[5] *= 1e-30
    x[6] *= 1e15
    x += 3.0 * torch.arange(64, device=dev).unsqueeze(1) / 64
    check(x, dy, gamma, beta, ckpt8=ckpt8, lib=lib)


@pytest.mark.parametrize("t", TYPES)
def test_non_finite_rows_stay_by_themselves(dev, lib, t):
    x, dy, gamma, beta = inputs(dev, 40, 300, t)
    x[7, 20], x[9, 299] = float("nan"), float("inf")
    for ckpt8 in (False, True):
        y, saved = kt_ops.layernorm_train(x, gamma, beta, ckpt8=ckpt8, lib=lib)
        dx, dgamma, dbeta = kt_ops.layernorm_bwd(dy, saved, lib=lib)
        bad = torch.zeros(40, dtype=torch.bool, device=dev)
        bad[7] = bad[9] = True
        assert y[bad].isnan().all() and dx[bad].isnan().all()
        assert y[~bad].isfinite().all() and dx[~bad].isfinite().all()
        assert dgamma.isnan().all() and dbeta.isfinite().all()
        if ckpt8:
            q, code, _ = rounded8(x)
            assert torch.equal(saved.q8, q) and torch.equal(saved.q8_exp, code)


@pytest.mark.parametrize("rows", [1, 23, 701])
@pytest.mark.parametrize("t", TYPES)
def test_checkpoints_of_odd_widths(dev, lib, rows, t):
    for cols in (1, 7, 33, 130, 257, 514, 1023, 2049, 4100, 8191, 8193, 12345, 16383, 16387):
        if rows * cols > 1 << 23:
            continue
        x, dy, gamma, beta = inputs(dev, rows, cols, t)
        a = check(x, dy, gamma, beta, ckpt8=True, lib=lib)
        # rows of q8 without a gap take another way to the same checkpoint and nearly the same gradients
        _, saved = kt_ops.layernorm_train(x, gamma, beta, ckpt8=True, lib=lib)
        b = kt_ops.layernorm_bwd(dy, saved._replace(q8=saved.q8.contiguous()), lib=lib)
        for u, v in zip(a[1:], b):
            assert (u.double() - v.double()).norm() <= 4 * (half_step(t) + 64 * E) * v.double().norm()


def test_empty(dev, lib):
    for t in TYPES:
        for rows, cols in ((0, 16), (16, 0)):
            x, dy, gamma, beta = inputs(dev, rows, cols, t)
            y, saved = kt_ops.layernorm_train(x, gamma, beta, ckpt8=True, lib=lib)
            dx, dgamma, dbeta = kt_ops.layernorm_bwd(dy, saved, lib=lib)
            assert y.shape == dx.shape == (rows, cols)
            assert dgamma.eq(0).all() and dbeta.eq(0).all() and dgamma.shape == (cols,)


@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("rows,cols,t", [(16384, 4096, torch.bfloat16), (4099, 1023, torch.float32),
                                         (20001, 96, torch.float16), (16384, 4096, torch.float32)])
def test_large_and_deterministic(dev, lib, rows, cols, t, ckpt8):
    x, dy, gamma, beta = inputs(dev, rows, cols, t)
    a = check(x, dy, gamma, beta, ckpt8=ckpt8, lib=lib)
    y, saved = kt_ops.layernorm_train(x, gamma, beta, ckpt8=ckpt8, lib=lib)
    b = (y, *kt_ops.layernorm_bwd(dy, saved, lib=lib))
    for u, v in zip(a, b):
        assert torch.equal(u, v)


def test_gradients_against_differences(dev, lib):
    """The formula's gradients against central differences of the 64-bit forward
    pass along random directions (error of order h^2), and the kernel's against the formula's."""
    x, dy, gamma, beta = inputs(dev, 6, 48, torch.float32)
    xd, d, g, b = x.double(), dy.double(), gamma.double(), beta.double()

    def loss(x, g, b):
        mu = x.mean(1, keepdim=True)
        xh = (x - mu) / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + 1e-5)
        return (d * (xh * g + b)).sum()

    _, dx, dgamma, dbeta = check(x, dy, gamma, beta, lib=lib)
    rng = torch.Generator(device=dev).manual_seed(3)
    h = 1e-5
    for i, (v, grad) in enumerate(((xd, dx), (g, dgamma), (b, dbeta))):
        step = torch.randn(v.shape, dtype=torch.float64, device=dev, generator=rng)
        args = [xd, g, b]
        args[i] = v + h * step
        up = loss(*args)
        args[i] = v - h * step
        slope = float((up - loss(*args)) / (2 * h))
        want = float((grad.double() * step).sum())
        # fp32 gradients: 2^-18 of the sum of magnitudes; differences: h^2 and 2^-52/h
        assert abs(slope - want) <= 2.0 ** -18 * float((grad.double() * step).abs().sum()) + 1e-6


def test_other_stream_and_graph(dev, lib):
    x, dy, gamma, beta = inputs(dev, 100, 768, torch.bfloat16)
    want = check(x, dy, gamma, beta, ckpt8=True, lib=lib)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, saved = kt_ops.layernorm_train(x, gamma, beta, ckpt8=True, lib=lib)
        got = (y, *kt_ops.layernorm_bwd(dy, saved, lib=lib))
    side.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(want, got))
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn: their workspaces are their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, saved = kt_ops.layernorm_train(x, gamma, beta, ckpt8=True, lib=lib)
            out = (y, *kt_ops.layernorm_bwd(dy, saved, lib=lib))
        graphs.append((g, out))
    x2, dy2, _, _ = inputs(dev, 100, 768, torch.bfloat16, seed=5)
    want2 = check(x2, dy2, gamma, beta, ckpt8=True, lib=lib)
    x.copy_(x2)
    dy.copy_(dy2)
    for g, out in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(u, v) for u, v in zip(want2, out))


def test_refusals(dev, lib):
    x, dy, gamma, beta = inputs(dev, 8, 64, torch.bfloat16)
    bad = [lambda: kt_ops.layernorm_train(x.double(), None, None, lib=lib),
           lambda: kt_ops.layernorm_train(x.t(), gamma, beta, lib=lib),
           lambda: kt_ops.layernorm_train(x[0], gamma, beta, lib=lib),
           lambda: kt_ops.layernorm_train(x, gamma[:-1], beta, lib=lib),
           lambda: kt_ops.layernorm_train(x, gamma.half(), beta.half(), lib=lib),
           lambda: kt_ops.layernorm_train(x, gamma.bfloat16(), beta, lib=lib),
           lambda: kt_ops.layernorm_train(x, gamma.cpu(), beta, lib=lib)]
    _, saved = kt_ops.layernorm_train(x, gamma, beta, lib=lib)
    bad += [lambda: kt_ops.layernorm_bwd(dy[:4], saved, lib=lib),
            lambda: kt_ops.layernorm_bwd(dy.float(), saved, lib=lib),
            lambda: kt_ops.layernorm_bwd(dy.cpu(), saved, lib=lib)]
    _, kept8 = kt_ops.layernorm_train(x, gamma, beta, ckpt8=True, lib=lib)
    bad.append(lambda: kt_ops.layernorm_bwd(dy, kept8._replace(q8=kept8.q8.t().contiguous().t()), lib=lib))
    for f in bad:
        with pytest.raises(ValueError):
            f()
    with pytest.raises(kt_lib.KtError):
        kt_ops.layernorm_train(x, gamma, beta, eps=-1.0, lib=lib)
