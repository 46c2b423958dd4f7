"""
The output end of a language model on a GPU, as a user runs it: the torch layers
over layer norm training, 8-bit checkpoints, token log probabilities and 4-bit
weights, alone and together, against the same in 64 bits.

Tolerances: a product of the library's TF32 GEMM is off by up to 2^-11 of its
operands (two of them: 2^-10, accumulated at random; 1e-3 normwise, as the
GEMM's own tests allow); what follows it inherits that. Where no GEMM takes part,
the operators' own tests hold the kernels to their types' steps, and here
normwise bounds of 1e-5 (fp32) and 2^-7 (bf16: two roundings of 2^-8 each) do.
"""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import kt_ops  # noqa: E402
import tuned_modules as tm  # noqa: E402


def normwise(got, want):
    return float((got.detach().double() - want.detach()).abs().max() / want.detach().abs().max())


def rounded8(x):
    """What the 8-bit checkpoint of x (rows, cols) stands for."""
    r, c = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -c % 32)).view(r, -1, 32)
    e = torch.frexp(b.abs().amax(-1, keepdim=True)).exponent
    step = torch.ldexp(torch.ones_like(e, dtype=torch.float64), e - 7)
    return ((b / step).round().clamp(-127, 127) * step).view(r, -1)[:, :c]


class _Norm8(torch.autograd.Function):
    """Layer norm in 64 bits whose backward pass sees the rounded input."""

    @staticmethod
    def forward(ctx, x, g, b):
        mu = x.mean(-1, keepdim=True)
        r = 1 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + 1e-5)
        ctx.save_for_backward(rounded8(x.reshape(-1, x.shape[-1])).view(x.shape), g, mu, r)
        return (x - mu) * r * g + b

    @staticmethod
    def backward(ctx, dy):
        x, g, mu, r = ctx.saved_tensors
        xh, w = (x - mu) * r, dy * g
        dx = r * (w - w.mean(-1, keepdim=True) - xh * (w * xh).mean(-1, keepdim=True))
        lead = tuple(range(dy.dim() - 1))
        return dx, (dy * xh).sum(lead), dy.sum(lead)


@pytest.mark.parametrize("checkpoint8", [False, True])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_layer_norm_autograd(dev, lib, t, checkpoint8):
    torch.manual_seed(0)
    ln = tm.TunedLayerNorm(200, checkpoint8=checkpoint8).to(dev)
    with torch.no_grad():
        ln.weight.uniform_(0.5, 1.5)
        ln.bias.uniform_(-0.5, 0.5)
    x = torch.randn(3, 70, 200, device=dev).to(t).requires_grad_()
    dy = torch.randn(3, 70, 200, device=dev).to(t)
    y = ln(x)
    y.backward(dy)
    xd = x.detach().double().requires_grad_()
    g, b = ln.weight.detach().double().requires_grad_(), ln.bias.detach().double().requires_grad_()
    if checkpoint8:
        want = _Norm8.apply(xd, g, b)
    else:
        want = torch.nn.functional.layer_norm(xd, (200,), g, b, 1e-5)
    want.backward(dy.double())
    tol = 1e-5 if t == torch.float32 else 2.0 ** -7
    assert y.dtype == t and x.grad.dtype == t and ln.weight.grad.dtype == torch.float32
    assert normwise(y, want.detach()) <= tol and normwise(x.grad, xd.grad) <= tol
    assert normwise(ln.weight.grad, g.grad) <= 1e-5 and normwise(ln.bias.grad, b.grad) <= 1e-5


def test_layer_norm_without_autograd_is_as_before(dev, lib):
    ln = tm.TunedLayerNorm(512).to(dev)
    x = torch.randn(40, 512, device=dev)
    with torch.no_grad():
        assert torch.equal(ln(x), kt_ops.layernorm(x, ln.weight, ln.bias, ln.eps, lib=lib))
        assert normwise(ln(x.half()), torch.nn.functional.layer_norm(x.half().double(), (512,))) <= 2.0 ** -10


def test_layer_norm_memory_of_checkpoints(dev, lib):
    """The 8-bit checkpoint takes the place of the input: 33/32 bytes a value."""
    x = torch.randn(1024, 4096, device=dev, dtype=torch.bfloat16)
    _, saved = kt_ops.layernorm_train(x, ckpt8=True, lib=lib)
    kept = sum(t.numel() * t.element_size() for t in saved[:3] if t is not None)
    assert kept == 1024 * 4096 * 33 // 32


def test_layer_norm_frozen_parts(dev, lib):
    ln = tm.TunedLayerNorm(64).to(dev)
    x = torch.randn(8, 64, device=dev)
    ln(x).sum().backward()  # weights only
    assert ln.weight.grad is not None and x.grad is None
    ln.requires_grad_(False)
    x.requires_grad_()
    ln(x).sum().backward()
    assert x.grad.abs().max() < 1e-5  # the sum of a normalised row does not change (up to rounding)
    dx, = torch.autograd.grad(ln(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):  # differentiable once
        dx.sum().backward()


def test_token_log_probs_autograd(dev, lib):
    torch.manual_seed(1)
    x = (3 * torch.randn(4, 9, 1003, device=dev)).requires_grad_()
    t = torch.randint(0, 1003, (4, 9), device=dev)
    t[1, 3] = -100
    r = tm.token_log_probs(x, t, top_k=3, scale=0.8)
    assert r.logprob.shape == r.entropy.shape == (4, 9) and r.top_index.shape == (4, 9, 3)
    w = torch.randn(4, 9, device=dev)
    (r.logprob * w).sum().add(r.entropy.sum() * 0.1).backward()
    xd = x.detach().double().requires_grad_()
    logp = torch.log_softmax(0.8 * xd, -1)
    lp = logp.gather(-1, t.clamp(min=0).unsqueeze(-1))[..., 0] * (t >= 0)
    H = -(logp.exp() * logp).sum(-1)
    ((lp * w).sum() + H.sum() * 0.1).backward()
    assert normwise(r.logprob.detach(), lp.detach()) <= 1e-5 and normwise(r.entropy.detach(), H.detach()) <= 1e-5
    assert normwise(x.grad, xd.grad) <= 1e-5
    assert torch.equal(r.top_index, logp.topk(3, -1).indices)
    x.grad = None
    tm.token_log_probs(x, t).logprob.mean().backward()  # a gradient that is expanded
    assert x.grad.isfinite().all()
    x.grad = None
    tm.token_log_probs(x).entropy.sum().backward()  # no targets
    xd.grad = None
    logp = torch.log_softmax(xd, -1)
    (-(logp.exp() * logp).sum()).backward()
    assert normwise(x.grad, xd.grad) <= 1e-5
    with pytest.raises(ValueError):
        tm.token_log_probs(x, t[:2])


def test_linear_w4_layer(dev, lib):
    torch.manual_seed(2)
    lin = torch.nn.Linear(384, 200).to(dev, torch.bfloat16)
    layer = tm.TunedLinearW4.from_linear(lin)
    x = torch.randn(2, 3, 384, device=dev, dtype=torch.bfloat16)
    with torch.no_grad():
        y = layer(x)
        q = torch.stack((layer.packed & 15, layer.packed >> 4), 2).view(200, -1, 128).double() - 8
        w = (q * layer.scales.double().unsqueeze(-1)).view(200, 384)
        # a weight is off by half a step of its group (and the scale's rounding of 7 steps by 2^-9)
        step = layer.scales.double().repeat_interleave(128, 1)
        assert bool(((w - lin.weight.double()).abs() <= step * (0.5 + 8 * 2.0 ** -8)).all())
        assert normwise(y, x.double() @ w.T + lin.bias.double()) <= 2.0 ** -8
        turned = x[0].t().contiguous().t()  # (3, 384), columns first
        assert torch.equal(layer(turned), y[0]) and torch.equal(layer(turned[:1]), y[0, :1])
    with pytest.raises(RuntimeError):
        layer(x.requires_grad_())
    model = torch.nn.Sequential(torch.nn.Linear(384, 96), torch.nn.Linear(96, 40), torch.nn.Linear(40, 8)).to(dev)
    tm.apply_tuned_layers(model, "w4")
    assert isinstance(model[0], tm.TunedLinearW4) and model[0].group == 128
    assert isinstance(model[1], tm.TunedLinearW4) and model[1].group == 32
    assert type(model[2]) is torch.nn.Linear  # 40 columns hold no whole group
    again = tm.TunedLinearW4(kt_ops.W4Weight(*(torch.empty_like(v) if v is not None else None
                                               for v in (layer.packed, layer.scales, layer.zeros)), 128),
                             torch.empty_like(layer.bias))
    again.load_state_dict(layer.state_dict())
    with torch.no_grad():
        assert torch.equal(again(x.detach()), y)


@pytest.mark.parametrize("checkpoint8", [False, True])
def test_training_step(dev, lib, checkpoint8):
    """Norm, head and token log probabilities, and their gradients: the head's
    products by the library's GEMM in both directions."""
    torch.manual_seed(3)
    N, C, V = 96, 256, 1500
    h = torch.randn(N, C, device=dev).requires_grad_()
    head = (torch.randn(V, C, device=dev) / C ** 0.5)
    targets = torch.randint(0, V, (N,), device=dev)
    ln = tm.TunedLayerNorm(C, checkpoint8=checkpoint8).to(dev)

    y = ln(h)
    logits = kt_ops.gemm(y.detach(), head, transpose_b=True).requires_grad_()
    r = tm.token_log_probs(logits, targets)
    loss = -(r.logprob.mean() + 0.01 * r.entropy.mean())
    loss.backward()
    dhead = kt_ops.gemm(logits.grad.t().contiguous(), y.detach())
    y.backward(kt_ops.gemm(logits.grad, head))

    hd = h.detach().double().requires_grad_()
    hw = head.double().requires_grad_()
    g = torch.ones(C, device=dev, dtype=torch.float64).requires_grad_()
    b = torch.zeros(C, device=dev, dtype=torch.float64).requires_grad_()
    yd = _Norm8.apply(hd, g, b) if checkpoint8 else torch.nn.functional.layer_norm(hd, (C,), g, b, 1e-5)
    logp = torch.log_softmax(yd @ hw.T, -1)
    lp = logp.gather(1, targets[:, None])[:, 0]
    want = -(lp.mean() - 0.01 * (logp.exp() * logp).sum(-1).mean())
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-3 * abs(want.item())
    assert normwise(h.grad, hd.grad) <= 4e-3 and normwise(dhead, hw.grad) <= 4e-3
    assert normwise(ln.weight.grad, g.grad) <= 4e-3 and normwise(ln.bias.grad, b.grad) <= 4e-3
    assert lib.device_error() == 0


def test_serving_step(dev, lib):
    """Norm, 4-bit head, log probability of the chosen token and its alternatives, captured and replayed."""
    torch.manual_seed(4)
    C, V = 512, 5000
    ln = tm.TunedLayerNorm(C, dtype=torch.bfloat16).to(dev)
    lin = torch.nn.Linear(C, V, bias=False).to(dev, torch.bfloat16)
    head = tm.TunedLinearW4.from_linear(lin, 64)
    h = torch.randn(2, C, device=dev, dtype=torch.bfloat16)
    chosen = torch.tensor([17, 4999], device=dev)

    @torch.no_grad()
    def step():
        return tm.token_log_probs(head(ln(h)), chosen, top_k=5)

    eager = step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = step()
    for seed in (5, 6):
        torch.manual_seed(seed)
        h.copy_(torch.randn_like(h))
        g.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(r, eager))
        with torch.no_grad():
            logp = torch.log_softmax(head(ln(h)).double(), -1)
        assert normwise(r.logprob, logp.gather(1, chosen[:, None])[:, 0]) <= 1e-5
        top = logp.topk(5, -1)
        assert normwise(r.top_logprob, top.values) <= 1e-5


def test_backward_captured_into_a_graph(dev, lib):
    """A whole step captured, after a warm-up on the capturing stream whose graph
    is gone (torch refuses a capture while an eager graph of the same leaves is
    alive on another stream, whatever the layers)."""
    torch.manual_seed(7)
    ln = tm.TunedLayerNorm(256, checkpoint8=True).to(dev)
    x = torch.randn(64, 256, device=dev).requires_grad_()
    t = torch.randint(0, 256, (64,), device=dev)
    leaves = [x, ln.weight, ln.bias]

    def step():
        return torch.autograd.grad(tm.token_log_probs(ln(x), t).logprob.sum(), leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        grads = step()
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(grads, step()):
        assert torch.equal(a, b)


def test_threads_call_at_once(dev, lib):
    """Calls from several threads, each on its own stream."""
    import threading
    x = torch.randn(300, 777, device=dev)
    t = torch.randint(0, 777, (300,), device=dev)
    w = kt_ops.w4_quantize(torch.randn(500, 768, device=dev), 128, lib=lib)

    def work():
        y, saved = kt_ops.layernorm_train(x, lib=lib)
        dx, _, _ = kt_ops.layernorm_bwd(x, saved, lib=lib)
        r = kt_ops.token_logprobs(x, t, top_k=4, lib=lib)
        return y, dx, r.logprob, r.top_index, kt_ops.w4_linear(x[:5, :768], w, lib=lib)

    want = work()
    torch.cuda.synchronize()
    bad = []

    def run():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = work()
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(want, got)):
                    bad.append(1)

    threads = [threading.Thread(target=run) for _ in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad
