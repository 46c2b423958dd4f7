"""
LayerNorm for training: rows far from 0, in place, checkpoints between other
data, and every way that the dispatch takes with several rows per CTA.
"""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import kt_lib  # noqa: E402
import kt_ops  # noqa: E402
from test_gpu_layernorm_train import E, TYPES, check, half_step, inputs, rounded8  # noqa: E402


@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("rows,cols", [(40, 64), (9, 1024), (3, 8192), (700, 256), (2, 32768)])
@pytest.mark.parametrize("value", [1000.0, 2.0 ** 80, -2.0 ** 120])
def test_rows_of_one_value(dev, lib, rows, cols, value, ckpt8):
    """A constant row (of a value that 8 bits hold) whose mean is exact has xh = 0:
    y is beta, dgamma 0 and dx = r (w - mean w). The mean of w is off by K 2^-24 of
    the mean |w|, w and the difference by a step each, r by 2^-22 (rsqrtf) and the
    rounding of eps."""
    if abs(value) * cols > 2.0 ** 127:
        cols = 64
    x = torch.full((rows, cols), value, device=dev)
    _, dy, gamma, beta = inputs(dev, rows, cols, torch.float32)
    y, saved = kt_ops.layernorm_train(x, gamma, beta, ckpt8=ckpt8, lib=lib)
    assert torch.equal(saved.mean, x[:, 0]) and torch.equal(y, beta.expand(rows, cols))
    dx, dgamma, dbeta = kt_ops.layernorm_bwd(dy, saved, lib=lib)
    assert dgamma.eq(0).all()
    w = dy.double() * gamma.double()
    r = 1e-5 ** -0.5
    want = r * (w - w.mean(1, keepdim=True))
    K = 64 + cols / 128
    tol = E * r * (2 * w.abs() + K * w.abs().mean(1, keepdim=True)) + 8 * E * want.abs()
    assert bool(((dx.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols", [3, 48, 77, 300, 1000, 1021, 3000, 6999, 12344, 12345, 16387])
def test_means_are_those_of_a_division(dev, lib, cols, t, ckpt8):
    """1000 in every column: the sum (below 2^24 thousands) is exact and so is its
    quotient by the columns, though one over the columns is not. Then nothing is
    left of x - mean, and of dy = 1 less its mean."""
    for rows, offset in ((5, 0), (700, 0), (5, 1)):
        base = torch.full((rows * cols + offset,), 1000.0, device=dev).to(t)
        x = base[offset:].view(rows, cols)
        beta = torch.linspace(-1, 1, cols, device=dev)
        y, saved = kt_ops.layernorm_train(x, None, beta, ckpt8=ckpt8, lib=lib)
        assert saved.mean.eq(1000).all() and torch.equal(y, beta.to(t).expand(rows, cols))
        dx, _, dbeta = kt_ops.layernorm_bwd(torch.ones_like(x), saved, lib=lib)
        assert dx.eq(0).all() and dbeta.eq(rows).all()


@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(3, 16387), (700, 16387), (70, 20000), (300, 1000), (50, 1023), (9, 8192)])
def test_gradient_of_the_input_in_place(dev, lib, rows, cols, t, ckpt8):
    """dx over dy's memory, and over x's: the weights' gradients stay those of the inputs."""
    x, dy, gamma, beta = inputs(dev, rows, cols, t)
    _, saved = kt_ops.layernorm_train(x, gamma, beta, ckpt8=ckpt8, lib=lib)
    want = kt_ops.layernorm_bwd(dy, saved, lib=lib)
    for over in ("dy",) if ckpt8 else ("dy", "x"):
        dx, x2 = dy.clone(), x.clone()
        dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(beta)
        if over == "x":
            dx, src = x2, dy
        else:
            src = dx
        size = lib.layernorm_bwd_workspace_bytes(rows, cols)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        at = saved.stats.data_ptr()
        q = (None, saved.q8.data_ptr(), saved.q8_exp.data_ptr(), saved.q8.stride(0)) if ckpt8 else \
            (x2.data_ptr(), None, None, 0)
        lib.layernorm_train_bwd(src.data_ptr(), *q, gamma.data_ptr(), at, at + 4 * rows, dx.data_ptr(),
                                dgamma.data_ptr(), dbeta.data_ptr(), rows, cols, kt_ops._DTYPES[t], kt_lib.KT_F32,
                                ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for got, w in zip((dx, dgamma, dbeta), want):
            assert torch.equal(got, w), over


@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(700, 16387), (3000, 1000), (2000, 1023), (9, 8192), (2000, 77)])
def test_output_in_place(dev, lib, rows, cols, t, ckpt8):
    """y over x's memory."""
    x, _, gamma, beta = inputs(dev, rows, cols, t)
    y, saved = kt_ops.layernorm_train(x, gamma, beta, ckpt8=ckpt8, lib=lib)
    stats = torch.empty_like(saved.stats)
    q8, exp, ld = None, None, 0
    if ckpt8:
        ld = saved.q8.stride(0)
        q8, exp = torch.empty(rows, ld, dtype=torch.int8, device=dev), torch.empty_like(saved.q8_exp)
    at = stats.data_ptr()
    lib.layernorm_train_fwd(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), x.data_ptr(), at, at + 4 * rows,
                            q8.data_ptr() if ckpt8 else None, exp.data_ptr() if ckpt8 else None, ld, rows, cols, 1e-5,
                            kt_ops._DTYPES[t], kt_lib.KT_F32, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(x, y) and torch.equal(stats, saved.stats)
    if ckpt8:
        assert torch.equal(q8[:, :cols], saved.q8) and torch.equal(exp, saved.q8_exp)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols,ld", [(9, 12), (30, 36), (61, 68), (1001, 1004), (8191, 8196), (9, 9), (9, 10), (12, 12),
                                     (64, 68), (16, 24)])
def test_bytes_behind_a_checkpoint_row_stay(dev, lib, cols, ld, t):
    """Rows of q8 whose distance is no multiple of 8 are written up to their last
    column only, and rows of whole 8-byte words never behind the words' end."""
    rows = 5
    x, dy, gamma, beta = inputs(dev, rows, cols, t)
    _, want = kt_ops.layernorm_train(x, gamma, beta, ckpt8=True, lib=lib)
    buf = torch.full((rows + 1, ld), 77, dtype=torch.int8, device=dev)
    exp = torch.empty_like(want.q8_exp)
    y, stats = torch.empty_like(x), torch.empty_like(want.stats)
    at = stats.data_ptr()
    lib.layernorm_train_fwd(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), at, at + 4 * rows,
                            buf.data_ptr(), exp.data_ptr(), ld, rows, cols, 1e-5, kt_ops._DTYPES[t], kt_lib.KT_F32,
                            torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(buf[:rows, :cols], want.q8) and torch.equal(exp, want.q8_exp)
    end = min(ld, (cols + 7) // 8 * 8) if ld % 8 == 0 else cols
    assert buf[:rows, end:].eq(77).all() and buf[rows].eq(77).all()
    saved = want._replace(q8=buf[:rows, :cols])
    for u, v in zip(kt_ops.layernorm_bwd(dy, saved, lib=lib), kt_ops.layernorm_bwd(dy, want, lib=lib)):
        assert (u.double() - v.double()).norm() <= 4 * (half_step(u.dtype) + 64 * E) * v.double().norm()


# The shapes that the dispatch tells apart, with more rows than CTAs, so that each
# takes several: 32 threads a row of one piece and of 16 columns, 64, 128, 256 and 512 threads of
# 16 columns, 256 and 512 of 32, and the kernels without a limit of width; whole pieces and cut ones.
MANY = [(t, *shape) for shape in [(2000, 128), (2000, 300), (2000, 512), (3000, 1000), (2000, 1021), (1500, 2000),
                                  (1500, 3333), (900, 7000), (900, 6999), (700, 12345), (700, 16384), (700, 16383),
                                  (1300, 16387)] for t in TYPES]
MANY += [(t, 5000, cols) for cols in (8000, 4101) for t in TYPES[1:]]
MANY += [(torch.float32, 2500, cols) for cols in (6000, 4101)]


@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("t,rows,cols", MANY)
def test_several_rows_for_each_cta(dev, lib, t, rows, cols, ckpt8):
    x, dy, gamma, beta = inputs(dev, rows, cols, t)
    check(x, dy, gamma, beta, ckpt8=ckpt8, lib=lib)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("rows,cols", [(600000, 4096), (140000, 16387)])
def test_offsets_past_32_bits(dev, lib, rows, cols, ckpt8):
    """The same 40 rows again and again, over more than 2^31 elements: each row's
    results are those of the first."""
    few, dfew, gamma, beta = inputs(dev, 40, cols, torch.bfloat16)
    x, dy = few.repeat(rows // 40, 1), dfew.repeat(rows // 40, 1)
    assert x.numel() > 1 << 31
    y, saved = kt_ops.layernorm_train(x, gamma, beta, ckpt8=ckpt8, lib=lib)
    want, wsaved = kt_ops.layernorm_train(few, gamma, beta, ckpt8=ckpt8, lib=lib)
    for at in (0, rows // 80 * 40, rows - 40):
        assert torch.equal(y[at:at + 40], want) and torch.equal(saved.stats[:, at:at + 40], wsaved.stats)
        if ckpt8:
            assert torch.equal(saved.q8[at:at + 40], wsaved.q8) and torch.equal(saved.q8_exp[at:at + 40], wsaved.q8_exp)
    del x, y
    dx, dgamma, dbeta = kt_ops.layernorm_bwd(dy, saved, lib=lib)
    dwant, _, _ = kt_ops.layernorm_bwd(dfew, wsaved, lib=lib)
    for at in (0, rows // 80 * 40, rows - 40):
        assert torch.equal(dx[at:at + 40], dwant)
    # rows/64 + 160 additions in a chain, each off by 2^-24 of the magnitudes (a CTA, or a 64th of the rows, adds fewer)
    d, n = dfew.double(), rows // 40
    kept = rounded8(few)[2] if ckpt8 else few.double()
    xh = (kept - wsaved.mean.double()[:, None]) * wsaved.rstd.double()[:, None]
    tol = (rows / 64 + 160 + 64) * E * n * (d * xh).abs().sum(0) + 64 * E * n * d.abs().sum(0)
    assert bool(((dgamma.double() - n * (d * xh).sum(0)).abs() <= tol).all())
    assert bool(((dbeta.double() - n * d.sum(0)).abs() <= (rows / 64 + 160) * E * n * d.abs().sum(0)).all())
    del dx, dy, saved
    torch.cuda.empty_cache()
