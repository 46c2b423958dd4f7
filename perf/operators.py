"""
operators.py — cases of the operators at the output end of a language model:
its last layer norm (trained, with and without 8-bit checkpoints), its head
with 4-bit weights, and the log probabilities of its tokens.

Where `own` is false, `run` computes an operator from elementary torch
operations in 32 bits; where it is true, it calls the kernel library through
the framework's public wrappers (kt_ops).

Ranges: layer norm of 1 to 16384 rows and 32 to 16384 columns; logits of 1 to
2048 rows and 1000 to 131072 tokens; 4-bit products of 1 to 16 tokens with
matrices of 256 to 131072 rows and 256 to 16384 columns.
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_EPS = 1e-5

_MAX_NORM = 16384 * 4096
_MAX_LOGITS = 2048 * 131072
_MAX_W4 = 131072 * 8192


def listed():
    return [
        # one short prompt's tokens through a small model's norm: launch latency
        {"name": "norm_small", "op": "norm", "rows": 8, "cols": 512, "dtype": "fp32", "weights": "fp32"},
        # the repository's own LayerNorm configuration, trained in bf16 with fp32 weights
        {"name": "norm_large", "op": "norm", "rows": 16384, "cols": 4096, "dtype": "bf16", "weights": "fp32"},
        # a ragged batch and an odd width, everything in fp32
        {"name": "norm_odd", "op": "norm", "rows": 4099, "cols": 1023, "dtype": "fp32", "weights": "fp32"},
        # a long training batch whose norm inputs are kept in 8 bits
        {"name": "norm8_large", "op": "norm8", "rows": 16384, "cols": 4096, "dtype": "bf16", "weights": "bf16"},
        # a ragged batch of a wide model with 8-bit checkpoints, in fp16
        {"name": "norm8_wide", "op": "norm8", "rows": 1021, "cols": 8192, "dtype": "fp16", "weights": "fp32"},
        # one decoding step: the sampled token and its 5 best alternatives
        {"name": "logprob_decode", "op": "logprob", "rows": 1, "cols": 32768, "dtype": "fp32", "top": 5, "masked": False},
        # scoring a long text with a large vocabulary, 20 alternatives for each position
        {"name": "logprob_score", "op": "logprob", "rows": 2048, "cols": 131072, "dtype": "bf16", "top": 20, "masked": False},
        # a batch of constrained decoding: most tokens are masked out with -inf
        {"name": "logprob_masked", "op": "logprob", "rows": 61, "cols": 50001, "dtype": "fp16", "top": 8, "masked": True},
        # a policy-gradient step with an entropy term: values and the gradient of the logits
        {"name": "logprob_train", "op": "logprob_train", "rows": 2048, "cols": 50001, "dtype": "bf16"},
        # the same on a short fp32 batch
        {"name": "logprob_train_small", "op": "logprob_train", "rows": 96, "cols": 32768, "dtype": "fp32"},
        # one token through a square projection: the smallest serving call
        {"name": "w4_token", "op": "w4", "tokens": 1, "rows": 4096, "cols": 4096, "group": 128, "zeros": False,
         "dtype": "bf16"},
        # a small batch of tokens through the head of a large vocabulary
        {"name": "w4_head", "op": "w4", "tokens": 8, "rows": 131072, "cols": 8192, "group": 64, "zeros": True,
         "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm8", "logprob", "logprob_train", "w4"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op in ("norm", "norm8"):
        cols = _log(rng, 32, 16384)
        if rng.random() < 0.5:  # widths of models are mostly multiples of 64
            cols = max(64, cols // 64 * 64)
        rows = _log(rng, 1, min(16384, _MAX_NORM // cols // (2 if dtype == "fp32" else 1)))
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "weights": rng.choice(["fp32", dtype])}
    if op in ("logprob", "logprob_train"):
        cols = _log(rng, 1000, 131072)
        most = _MAX_LOGITS // cols // (4 if op == "logprob_train" else 2)
        rows = _log(rng, 1, min(2048, most))
        if op == "logprob_train":
            return {"op": op, "rows": rows, "cols": cols, "dtype": dtype}
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "top": rng.randint(0, 32),
                "masked": rng.random() < 0.25}
    group = rng.choice([32, 64, 128])
    cols = max(256, _log(rng, 256, 16384) // group * group)
    rows = _log(rng, 256, min(131072, _MAX_W4 // cols))
    return {"op": op, "tokens": rng.randint(1, 16), "rows": rows, "cols": cols, "group": group,
            "zeros": rng.random() < 0.5, "dtype": dtype}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = dict(case)
    if case["op"] in ("norm", "norm8"):
        r, c, wt = case["rows"], case["cols"], _DTYPES[case["weights"]]
        # a residual stream: some channels carry much larger values, and rows have a small common offset
        channel = torch.exp(0.5 * normal(c))
        s["x"] = (normal(r, c).mul_(channel).add_(0.2 * normal(r, 1))).to(dt)
        s["dy"] = normal(r, c).to(dt)
        s["gamma"] = (1.0 + 0.1 * normal(c)).to(wt)
        s["beta"] = (0.1 * normal(c)).to(wt)
    elif case["op"] in ("logprob", "logprob_train"):
        r, c = case["rows"], case["cols"]
        x = normal(r, c).mul_(2.5)
        s["targets"] = torch.randint(0, c, (r,), device="cuda", generator=g)
        # most tokens are likely ones: their logits stand out by 0 to 12
        x[torch.arange(r, device="cuda"), s["targets"]] += 12.0 * torch.rand(r, device="cuda", generator=g)
        if case.get("masked"):
            x.masked_fill_(torch.rand(r, c, device="cuda", generator=g) < 0.9, -math.inf)
        s["logits"] = x.to(dt)
        if case["op"] == "logprob_train":
            s["grad_logprob"] = normal(r) / r
            s["grad_entropy"] = torch.full((r,), 0.01 / r, device="cuda") * torch.rand(r, device="cuda", generator=g)
    else:
        m, n, k, grp = case["tokens"], case["rows"], case["cols"], case["group"]
        # two 4-bit values to a byte, the even column in the low half
        s["packed"] = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
        s["scales"] = ((0.5 + torch.rand(n, k // grp, device="cuda", generator=g)) / (6.0 * math.sqrt(k))).to(dt)
        s["zeros"] = None
        if case["zeros"]:
            s["zeros"] = torch.randint(5, 12, (n, k // grp), device="cuda", generator=g, dtype=torch.uint8)
        s["x"] = normal(m, k).to(dt)
        s["bias"] = (0.1 * normal(n)).to(dt)
    return s


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------

def _ops():
    try:
        return sys.modules["kt_ops"]
    except KeyError:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "cd-cuda-course-project_b200", "src"))
        import kt_ops
        return kt_ops


def _run_own(s):
    kt = _ops()
    op = s["op"]
    if op in ("norm", "norm8"):
        y, saved = kt.layernorm_train(s["x"], s["gamma"], s["beta"], _EPS, ckpt8=op == "norm8")
        dx, dgamma, dbeta = kt.layernorm_bwd(s["dy"], saved)
        return {"y": y, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if op == "logprob":
        r = kt.token_logprobs(s["logits"], s["targets"], top_k=s["top"])
        return {"logprob": r.logprob, "entropy": r.entropy, "top_logprob": r.top_logprob, "top_index": r.top_index}
    if op == "logprob_train":
        r = kt.token_logprobs(s["logits"], s["targets"])
        dx = kt.token_logprobs_bwd(s["logits"], s["targets"], r, s["grad_logprob"], s["grad_entropy"])
        return {"logprob": r.logprob, "entropy": r.entropy, "dlogits": dx}
    w = kt.W4Weight(s["packed"], s["scales"], s["zeros"], s["group"])
    return {"y": kt.w4_linear(s["x"], w, s["bias"])}


# ---------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------

def _rounded8(x):
    """fp32 values as blocks of 32 int8 numbers with a common power of two stand for them."""
    r, c = x.shape
    b = torch.nn.functional.pad(x, (0, -c % 32)).view(r, -1, 32)
    field = (b.abs().amax(-1, keepdim=True).view(torch.int32) >> 23).clamp(7, 254)
    up, down = ((260 - field) << 23).view(torch.float32), ((field - 6) << 23).view(torch.float32)
    q = torch.round(b * up).clamp(-127, 127)
    return (q * down).view(r, -1)[:, :c]


def _plain_norm(s):
    x, dy, gamma = s["x"].float(), s["dy"].float(), s["gamma"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + _EPS)
    y = centred * rstd * gamma + s["beta"].float()
    if s["op"] == "norm8":
        centred = _rounded8(x) - x.mean(1, keepdim=True)
    xhat = centred * rstd
    w = dy * gamma
    dx = rstd * (w - w.mean(1, keepdim=True) - xhat * (w * xhat).mean(1, keepdim=True))
    dt, wt = s["x"].dtype, s["gamma"].dtype
    return {"y": y.to(dt), "dx": dx.to(dt), "dgamma": (dy * xhat).sum(0).to(wt), "dbeta": dy.sum(0).to(wt)}


def _plain_logprob(s):
    x = s["logits"].float()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    logprob = x.gather(1, s["targets"][:, None]) - lse
    p = e / total
    entropy = lse - torch.where(p > 0, p * x, 0.0).sum(1, keepdim=True)
    out = {"logprob": logprob[:, 0], "entropy": entropy[:, 0]}
    if s["op"] == "logprob":
        value, index = torch.sort(x, dim=1, descending=True, stable=True)
        return out | {"top_logprob": value[:, :s["top"]] - lse, "top_index": index[:, :s["top"]].contiguous()}
    g, h = s["grad_logprob"][:, None], s["grad_entropy"][:, None]
    dx = -p * (g + h * (x - lse + entropy))
    dx.scatter_add_(1, s["targets"][:, None], g)
    return out | {"dlogits": dx.to(s["logits"].dtype)}


def _plain_w4(s):
    n, half = s["packed"].shape
    q = torch.stack((s["packed"] & 15, s["packed"] >> 4), dim=2).view(n, -1, s["group"]).float()
    q -= 8.0 if s["zeros"] is None else s["zeros"].float()[:, :, None]
    w = (q * s["scales"].float()[:, :, None]).view(n, 2 * half)
    return {"y": (s["x"].float() @ w.T + s["bias"].float()).to(s["x"].dtype)}


def run(state):
    if own:
        return _run_own(state)
    if state["op"] in ("norm", "norm8"):
        return _plain_norm(state)
    if state["op"] in ("logprob", "logprob_train"):
        return _plain_logprob(state)
    return _plain_w4(state)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_norm(s):
    x = s["x"].double()
    dy, gamma, beta = s["dy"].double(), s["gamma"].double(), s["beta"].double()
    var, mu = torch.var_mean(x, dim=1, keepdim=True, correction=0)
    r = 1.0 / torch.sqrt(var + _EPS)
    y = torch.addcmul(beta, (x - mu) * r, gamma)
    if s["op"] == "norm8":
        c = x.shape[1]
        whole = torch.cat((x, x.new_zeros(x.shape[0], -c % 32)), dim=1).unflatten(1, (-1, 32))
        # 2^(e-1) <= largest < 2^e: the block's values are multiples of 2^(e-7)
        e = torch.frexp(whole.abs().max(dim=2, keepdim=True).values).exponent.clamp(min=-119)
        step = torch.ldexp(torch.ones_like(e, dtype=torch.float64), e - 7)
        x = ((whole / step).round().clamp(-127, 127) * step).flatten(1)[:, :c]
    xh = (x - mu) * r
    n = x.shape[1]
    a = dy * gamma
    dx = (a - a.sum(1, keepdim=True) / n - xh * ((a * xh).sum(1, keepdim=True) / n)) * r
    return {"y": y, "dx": dx, "dgamma": torch.einsum("rc,rc->c", dy, xh), "dbeta": dy.sum(0)}


def _exact_logprob(s):
    z = s["logits"].double()
    lse = torch.logsumexp(z, dim=1, keepdim=True)
    logp = z - lse
    p = logp.exp()
    plogp = torch.nan_to_num(p * logp, nan=0.0)  # 0 log 0
    entropy = -plogp.sum(1)
    t = s["targets"]
    rows = torch.arange(z.shape[0], device=z.device)
    out = {"logprob": logp[rows, t], "entropy": entropy}
    if s["op"] == "logprob":
        k = s["top"]
        return out | {"top_logprob": torch.topk(logp, k, dim=1).values, "top_index": None}
    g, h = s["grad_logprob"].double()[:, None], s["grad_entropy"].double()[:, None]
    dx = -(g * p) - h * (plogp + p * entropy[:, None])
    dx[rows, t] += g[:, 0]
    return out | {"dlogits": dx}


def _exact_w4(s):
    n, half = s["packed"].shape
    grp = s["group"]
    x = s["x"].double()
    y = s["bias"].double().expand(x.shape[0], n).clone()
    step = max(1, (1 << 28) // (2 * half))
    for at in range(0, n, step):
        part = s["packed"][at:at + step].long()
        q = torch.empty(part.shape[0], 2 * half, dtype=torch.float64, device=x.device)
        q[:, 0::2] = (part % 16).double()
        q[:, 1::2] = (part // 16).double()
        zero = 8.0 if s["zeros"] is None else s["zeros"][at:at + step].double().repeat_interleave(grp, dim=1)
        w = (q - zero) * s["scales"][at:at + step].double().repeat_interleave(grp, dim=1)
        y[:, at:at + step] += x @ w.T
    return {"y": y}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "norm8"):
        return _exact_norm(s)
    if case["op"] in ("logprob", "logprob_train"):
        return _exact_logprob(s)
    return _exact_w4(s)


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] in ("norm", "norm8"):
        r, c, w = case["rows"], case["cols"], _SIZE[case["weights"]]
        values = r * c
        # forward: x in, y out, mean and rstd out; backward: dy and the saved input in, dx out
        saved = 1 + 1 / 32 if case["op"] == "norm8" else size
        extra = saved if case["op"] == "norm8" else 0
        return {"bytes": values * (2 * size + extra) + values * (2 * size + saved) + 16 * r + 5 * w * c,
                "flops": 20 * values}
    if case["op"] == "logprob":
        r, c = case["rows"], case["cols"]
        return {"bytes": r * c * size + r * (16 + 12 * case["top"]), "flops": 6 * r * c}
    if case["op"] == "logprob_train":
        r, c = case["rows"], case["cols"]
        return {"bytes": 3 * r * c * size + 28 * r, "flops": 12 * r * c}
    m, n, k = case["tokens"], case["rows"], case["cols"]
    groups = k // case["group"]
    return {"bytes": n * k // 2 + n * groups * (size + (1 if case["zeros"] else 0)) + (m * k + n + m * n) * size,
            "flops": 2 * m * n * k}
