"""
4-bit weights on a GPU: quantisation and products of few tokens against the
formulas in 64 bits.

Tolerances: the output is rounded once (eps/2 of its size). Inside, products
are exact; a group's sum is a chain of at most 8 tensor-core steps, each of
which may be off by 2^-22 of its magnitudes (16 products added with truncation),
and the groups, column-warps and CTAs are joined in at most K/32 + 16 fp32
additions: (32 + K/32) 2^-22 of the sum of the products' magnitudes.
"""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import kt_lib  # noqa: E402
import kt_ops  # noqa: E402

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def values(w):
    """The (N, K) matrix that 4-bit weights stand for, in 64 bits."""
    n, half = w.packed.shape
    q = torch.stack((w.packed & 15, w.packed >> 4), 2).view(n, -1, w.group).double()
    q = q - (8.0 if w.zeros is None else w.zeros.double().unsqueeze(-1))
    return (q * w.scales.double().unsqueeze(-1)).view(n, 2 * half)


def make(dev, m, n, k, group, t, zeros=True, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed * 131 + m * 17 + n * 3 + k)
    packed = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=dev, generator=g)
    scales = (torch.rand(n, k // group, device=dev, generator=g) * 0.1 + 0.01).to(t)
    z = torch.randint(0, 16, (n, k // group), dtype=torch.uint8, device=dev, generator=g) if zeros else None
    x = torch.randn(m, k, device=dev, generator=g).to(t)
    bias = torch.randn(n, device=dev, generator=g).to(t)
    return x, kt_ops.W4Weight(packed, scales, z, group), bias


def check(x, w, bias, lib):
    y = kt_ops.w4_linear(x, w, bias, lib=lib)
    v, xd = values(w), x.double()
    want = xd @ v.T + (bias.double() if bias is not None else 0.0)
    k = x.shape[1]
    mag = xd.abs() @ v.abs().T + (bias.double().abs() if bias is not None else 0.0)
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() + (32 + k / 32) * 2.0 ** -22 * mag
    over = ((y.double() - want).abs() / tol).max()
    assert y.shape == want.shape and y.dtype == x.dtype
    assert over <= 1, float(over)
    return y


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 1, 128), (1, 16, 128), (2, 17, 256), (7, 63, 384), (8, 64, 1024), (9, 65, 640),
                                   (16, 200, 2048), (17, 130, 1152), (40, 33, 256), (3, 1000, 4096), (5, 300, 16384),
                                   (16, 31, 32768)])
def test_shapes(dev, lib, m, n, k, group, t):
    for zeros in (False, True):
        check(*make(dev, m, n, k, group, t, zeros=zeros), lib)
    assert lib.device_error() == 0


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("group,k", [(32, 32), (32, 96), (32, 160), (64, 64), (64, 192), (64, 6080), (32, 4128)])
def test_columns_that_end_inside_a_segment(dev, lib, group, k, t):
    for m in (1, 4, 16):
        check(*make(dev, m, 70, k, group, t), lib)


@pytest.mark.parametrize("t", TYPES)
def test_no_bias_and_unaligned_scales(dev, lib, t):
    for group in (32, 64, 128):
        x, w, bias = make(dev, 3, 100, 512, group, t)
        want = check(x, w, None, lib)
        base = torch.empty(100 * 512 // group + 1, dtype=t, device=dev)
        scales = base[1:].view(100, -1).copy_(w.scales)
        zbase = torch.empty(100 * 512 // group + 1, dtype=torch.uint8, device=dev)
        zeros = zbase[1:].view(100, -1).copy_(w.zeros)
        assert torch.equal(kt_ops.w4_linear(x, w._replace(scales=scales), lib=lib), want)
        assert torch.equal(kt_ops.w4_linear(x, w._replace(zeros=zeros), lib=lib), want)


@pytest.mark.parametrize("t", TYPES)
def test_strided_and_unaligned_tokens(dev, lib, t):
    x, w, bias = make(dev, 4, 80, 256, 128, t)
    wide = torch.zeros(4, 300, dtype=t, device=dev)
    wide[:, 3:259] = x
    want = check(x, w, bias, lib)
    assert torch.equal(kt_ops.w4_linear(wide[:, 3:259], w, bias, lib=lib), want)
    one = x[:1].expand(4, 256)  # rows at distance 0
    assert torch.equal(kt_ops.w4_linear(one, w, bias, lib=lib), want[:1].expand(4, 80))


def test_rows_of_tokens_do_not_mix(dev, lib):
    for t in TYPES:
        x, w, bias = make(dev, 9, 80, 512, 64, t)
        want = kt_ops.w4_linear(x, w, bias, lib=lib)
        x[4, 100] = float("nan")
        x[2, 7] = float("inf")
        w = w._replace(zeros=None, packed=w.packed | 0x99)  # no weight is 0: inf stays inf
        want = kt_ops.w4_linear(torch.where(x.isfinite(), x, 0), w, bias, lib=lib)
        got = kt_ops.w4_linear(x, w, bias, lib=lib)
        rest = [0, 1, 3, 5, 6, 7, 8]
        assert torch.equal(got[rest], want[rest])
        assert got[4].isnan().all() and got[2].isinf().all()


def test_large_values_in_fp32(dev, lib):
    x, w, bias = make(dev, 2, 64, 256, 128, torch.float32)
    x *= 1e30
    # the products with q - z, up to 15 times these, stay within fp32
    x[0, :8] = torch.tensor([3e36, 1e-38, 1e36, 2e-39, -3e36, 1.0, 0.0, -0.0], device=dev)
    w = w._replace(scales=w.scales * 1e-6)
    check(x, w, bias, lib)


@pytest.mark.parametrize("m,n,k,t,group", [(1, 4096, 4096, torch.bfloat16, 128), (8, 50000, 8192, torch.float16, 64),
                                           (16, 8192, 8192, torch.bfloat16, 32), (1, 11008, 4096, torch.float32, 128)])
def test_large_and_deterministic(dev, lib, m, n, k, t, group):
    x, w, bias = make(dev, m, n, k, group, t)
    y = check(x, w, bias, lib)
    assert torch.equal(y, kt_ops.w4_linear(x, w, bias, lib=lib))


@pytest.mark.parametrize("m,k,group", [(1, 4096, 128), (8, 8192, 64), (16, 8192, 32), (13, 16384, 128)])
def test_many_calls_agree(dev, lib, m, k, group):
    """Bits of many calls, behind one another and on two streams at once."""
    x, w, bias = make(dev, m, 5000, k, group, torch.bfloat16)
    want = check(x, w, bias, lib)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(30):
        got.append(kt_ops.w4_linear(x, w, bias, lib=lib))
        with torch.cuda.stream(side):
            got.append(kt_ops.w4_linear(x, w, bias, lib=lib))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_offsets_past_32_bits(dev, lib):
    """9 billion weights: byte offsets need 33 bits, those of columns 34."""
    n, k = 1_100_000, 8192
    x, w, _ = make(dev, 1, 64, k, 128, torch.bfloat16, zeros=False)
    packed = w.packed.repeat(n // 64 + 1, 1)[:n]
    scales = w.scales.repeat(n // 64 + 1, 1)[:n]
    want = kt_ops.w4_linear(x, w, lib=lib)
    got = kt_ops.w4_linear(x, kt_ops.W4Weight(packed, scales, None, 128), lib=lib)
    assert torch.equal(got[0], want[0].repeat(n // 64 + 1)[:n])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize(dev, lib, group, t):
    g = torch.Generator(device=dev).manual_seed(group)
    w = torch.randn(37, 3 * 128, device=dev, generator=g).to(t)
    w[3, :group] = 0
    w[4, 1] = float("nan")
    for st in TYPES:
        q = kt_ops.w4_quantize(w, group, scale_dtype=st, lib=lib)
        blocks = w.float().view(37, -1, group)
        # (a quotient rounded to 53 and then to 24 bits is the fp32 quotient)
        s = (blocks.abs().amax(-1).double() / 7).float().to(st)
        bad = ~torch.isfinite(blocks).all(-1)
        assert q.scales.dtype == st and q.scales[bad].isnan().all()
        assert int((q.scales[~bad] != s[~bad]).sum()) == 0
        got = torch.stack((q.packed & 15, q.packed >> 4), 2).view(37, -1, group).float()
        sf = s.float().unsqueeze(-1)
        want = torch.where(sf > 0, (torch.round(blocks / sf) + 8).clamp(0, 15), 8.0)
        ok = ~bad & ~s.isnan()
        assert int((got[ok] != want[ok]).sum()) == 0
    empty = kt_ops.w4_quantize(torch.empty(0, 128, device=dev, dtype=t), group, lib=lib)
    assert empty.packed.shape == (0, 64)


def test_empty_and_refusals(dev, lib):
    x, w, bias = make(dev, 2, 48, 256, 128, torch.float16)
    assert kt_ops.w4_linear(x[:0], w, bias, lib=lib).shape == (0, 48)
    bad = [lambda: kt_ops.w4_linear(x.double(), w, bias, lib=lib),
           lambda: kt_ops.w4_linear(x[:, :128], w, bias, lib=lib),
           lambda: kt_ops.w4_linear(x.t(), w, bias, lib=lib),
           lambda: kt_ops.w4_linear(x, w, bias[:-1], lib=lib),
           lambda: kt_ops.w4_linear(x, w, bias.float(), lib=lib),
           lambda: kt_ops.w4_linear(x, w._replace(group=48), bias, lib=lib),
           lambda: kt_ops.w4_linear(x, w._replace(group=64), bias, lib=lib),
           lambda: kt_ops.w4_linear(x, w._replace(zeros=w.zeros[:-1]), bias, lib=lib),
           lambda: kt_ops.w4_linear(x, w._replace(scales=w.scales.double()), bias, lib=lib),
           lambda: kt_ops.w4_linear(x, w._replace(scales=w.scales.bfloat16()), bias, lib=lib),
           lambda: kt_ops.w4_linear(x, w._replace(packed=w.packed.cpu()), bias, lib=lib),
           lambda: kt_ops.w4_linear(x, w, bias, out=torch.empty(2, 47, dtype=x.dtype, device=dev), lib=lib),
           lambda: kt_ops.w4_quantize(x, 96, lib=lib),
           lambda: kt_ops.w4_quantize(x.double(), 128, lib=lib)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    base = torch.zeros(48 * 128 + 16, dtype=torch.uint8, device=dev)
    shifted = w._replace(packed=base[4:4 + 48 * 128].view(48, 128))
    with pytest.raises(kt_lib.KtError):
        kt_ops.w4_linear(x, shifted, bias, lib=lib)


def test_other_stream_and_graph(dev, lib):
    x, w, bias = make(dev, 5, 300, 2048, 64, torch.bfloat16)
    want = check(x, w, bias, lib)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kt_ops.w4_linear(x, w, bias, lib=lib)
    side.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kt_ops.w4_linear(x, w, bias, lib=lib)
    x.copy_(torch.randn_like(x))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, check(x, w, bias, lib))
