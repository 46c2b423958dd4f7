"""
tuned_modules.py — PyTorch layers that run on the tuned B200 kernels.

The reference's `TunedLinear`, `TunedLayerNorm` and `TunedMultiheadAttention`
(src/pytorch_integration.py:314-378) only attach the tuner's best parameters
to the stock torch layers as metadata and compute with cuBLAS / SDPA. Here
the same three layers compute with the kernel library: each one loads the
variant library the tuner picked (results/{kernel}_tuning.json, field
`best.library`), or the default library when no tuning result exists, and
calls it through the C ABI on the current CUDA stream:

  TunedLinear             y = x·W^T (+ b): kt_gemm_f32 with transpose_b (the
                          nn.Linear weight is already the N×K "Bt" layout);
                          TF32 tensor cores by default, exact FFMA on request
                          or when the tuned winner is the FFMA variant
  TunedLayerNorm          kt_layernorm_f32 over the last dimension; under
                          autograd, or for bf16 and fp16 inputs, the training
                          kernels (kt_layernorm_train_fwd / _bwd), which can
                          keep the input in 8 bits for the backward pass
  TunedMultiheadAttention q/k/v/out projections as TunedLinear, the attention
                          core as kt_fa_fwd_bf16 (bf16 Q/K/V, fp32 softmax and
                          accumulation), optionally causal

  TunedLinearW4           y = x·W^T (+ b) with 4-bit weights for serving few
                          tokens (kt_w4_linear), made from an nn.Linear
  token_log_probs         log probabilities of given tokens, entropies and top
                          alternatives of logits, with their gradient
                          (kt_token_logprobs_train / _train_bwd)

The linear and attention layers are inference layers (they have forward
kernels only): a call with autograd recording raises instead of silently
computing something else. None of the layers has forward-mode tangents; inputs
that carry one are refused. `apply_tuned_layers` swaps layers into a model,
copying the weights (the reference's version builds fresh layers and drops the
trained weights).
`sdpa_comparison` checks and times the attention core against
torch.nn.functional.scaled_dot_product_attention (the reference's SDPA vs
manual-attention benchmark, src/pytorch_integration.py:120-192).
"""

from __future__ import annotations

import json
import math
import os
from pathlib import Path
from typing import Any, Dict, Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import forward_ad as _forward_ad

import kt_lib
import kt_ops


def _results_dir(results_dir: Optional[os.PathLike] = None) -> Path:
    if results_dir is not None:
        return Path(results_dir)
    env = os.environ.get("KT_RESULTS_DIR")
    return Path(env) if env else Path(__file__).resolve().parent.parent / "results"


def load_best_params(kernel: str, results_dir: Optional[os.PathLike] = None) -> Dict[str, Any]:
    """Parameters of the tuner's best variant of `kernel` ({} without a tuning result)."""
    f = _results_dir(results_dir) / f"{kernel}_tuning.json"
    if not f.exists():
        return {}
    best = json.loads(f.read_text()).get("best") or {}
    return dict(best.get("params") or {})


def tuned_library(kernel: str, results_dir: Optional[os.PathLike] = None) -> kt_lib.KtLibrary:
    """The library of the tuner's best variant of `kernel` if it exists, else the default library."""
    f = _results_dir(results_dir) / f"{kernel}_tuning.json"
    if f.exists():
        best = json.loads(f.read_text()).get("best") or {}
        so = best.get("library")
        if so and Path(so).exists():
            return kt_lib.load(so)
    return kt_lib.load()


def _tangents(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether forward-mode differentiation has given one of them a tangent."""
    if getattr(_forward_ad, "_current_level", 0) < 0:  # (asking a tensor takes 0.7 us)
        return False
    return any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _recording(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a result computed from them is to be differentiable. A tangent counts:
    the autograd functions below have none to give and torch refuses the call."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or _tangents(*tensors)


def _no_autograd(name: str, *tensors: Optional[torch.Tensor]) -> None:
    if _recording(*tensors):
        raise RuntimeError(f"{name} runs forward-only B200 kernels; call it under torch.no_grad() "
                           "or torch.inference_mode(), without forward-mode tangents")


def _columns(name: str, x: torch.Tensor, columns: int) -> None:
    if x.dim() < 1 or x.shape[-1] != columns:
        raise ValueError(f"{name}: rows of {columns} columns expected, got {tuple(x.shape)}")


class TunedLinear(nn.Linear):
    """nn.Linear computed by the library's GEMM (x·W^T with W as the transpose_b operand)."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, kernel: str = "matmul",
                 variant: Optional[str] = None, results_dir: Optional[os.PathLike] = None,
                 device=None, dtype=None) -> None:
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        self.tuned_params = load_best_params(kernel, results_dir)
        self._lib = tuned_library(kernel, results_dir)
        v = variant or self.tuned_params.get("variant", "tf32")
        self.gemm_variant = kt_lib.KT_GEMM_FFMA if v == "ffma" else kt_lib.KT_GEMM_TF32

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _no_autograd("TunedLinear", x, self.weight, self.bias)
        lead = x.shape[:-1]
        x2 = x.reshape(-1, self.in_features).contiguous()
        y = kt_ops.gemm(x2, self.weight.contiguous(), transpose_b=True, variant=self.gemm_variant, lib=self._lib)
        if self.bias is not None:
            y.add_(self.bias)
        return y.view(*lead, self.out_features)


class _LayerNormTrain(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, checkpoint8):
        y, saved = kt_ops.layernorm_train(x, weight, bias, eps, ckpt8=checkpoint8)
        ctx.save_for_backward(saved.x, saved.q8, saved.q8_exp, saved.gamma, saved.stats)
        ctx.beta_dtype = saved.beta_dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        saved = kt_ops.LayerNormSaved(*ctx.saved_tensors, ctx.beta_dtype)
        weights = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dx, dgamma, dbeta = kt_ops.layernorm_bwd(dy.contiguous(), saved, weight_grads=weights)
        return dx, dgamma, dbeta, None, None


class TunedLayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last dimension computed by the library's LayerNorm kernels.

    With autograd recording it is differentiable (once); checkpoint8 then keeps
    the input for the backward pass in 8 bits. Inputs are fp32, bf16 or fp16, the
    weights fp32 or of the input's type.
    """

    def __init__(self, normalized_shape: int, eps: float = 1e-5, results_dir: Optional[os.PathLike] = None,
                 device=None, dtype=None, checkpoint8: bool = False) -> None:
        super().__init__(normalized_shape, eps=eps, elementwise_affine=True, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError("TunedLayerNorm normalises the last dimension only")
        self.tuned_params = load_best_params("layernorm", results_dir)
        self._lib = tuned_library("layernorm", results_dir)
        self.checkpoint8 = checkpoint8

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        c = self.normalized_shape[0]
        _columns("TunedLayerNorm", x, c)
        x2 = x.reshape(-1, c).contiguous()
        if _recording(x, self.weight, self.bias):
            y = _LayerNormTrain.apply(x2, self.weight, self.bias, self.eps, self.checkpoint8)
        elif x.dtype == torch.float32:
            y = kt_ops.layernorm(x2, self.weight, self.bias, self.eps, lib=self._lib)
        else:
            y, _ = kt_ops.layernorm_train(x2, self.weight, self.bias, self.eps)
        return y.view(x.shape)


class TunedLinearW4(nn.Module):
    """A linear layer with 4-bit weights (kt_ops.W4Weight) for serving few tokens.

    The weights are buffers (packed, scales, zeros); inputs and bias are of the
    scales' type. Inference only.
    """

    def __init__(self, weight: kt_ops.W4Weight, bias: Optional[torch.Tensor] = None) -> None:
        super().__init__()
        self.group = weight.group
        self.in_features = 2 * weight.packed.shape[1]
        self.out_features = weight.packed.shape[0]
        self.register_buffer("packed", weight.packed)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("zeros", weight.zeros)
        self.register_buffer("bias", bias)

    @classmethod
    def from_linear(cls, linear: nn.Linear, group: int = 128) -> "TunedLinearW4":
        """Quantise a linear layer's weight (on a CUDA device) symmetrically in groups of `group` columns."""
        w = kt_ops.w4_quantize(linear.weight.detach().contiguous(), group)
        return cls(w, linear.bias.detach().clone() if linear.bias is not None else None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _columns("TunedLinearW4", x, self.in_features)
        _no_autograd("TunedLinearW4", x)
        w = kt_ops.W4Weight(self.packed, self.scales, self.zeros, self.group)
        x2 = x.reshape(-1, self.in_features)
        if x2.stride(1) != 1:
            x2 = x2.contiguous()
        y = kt_ops.w4_linear(x2, w, self.bias)
        return y.view(*x.shape[:-1], self.out_features)


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, scale, ignore_index):
        r = kt_ops.token_logprobs(logits, targets, top_k, scale, ignore_index)
        ctx.save_for_backward(logits, targets, r.entropy, r.norm)
        ctx.scale, ctx.ignore_index = scale, ignore_index
        ctx.mark_non_differentiable(r.top_logprob, r.top_index)
        ctx.set_materialize_grads(False)
        return tuple(r)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logprob, grad_entropy, grad_lse, *_):
        logits, targets, entropy, norm = ctx.saved_tensors
        grads = [g.contiguous() if g is not None else None for g in (grad_logprob, grad_entropy, grad_lse)]
        if all(g is None for g in grads):
            return None, None, None, None, None
        r = kt_ops.TokenLogprobs(None, entropy, None, None, None)
        r.norm = norm
        dx = kt_ops.token_logprobs_bwd(logits, targets, r, grads[0], grads[1], ctx.scale, ctx.ignore_index,
                                       grad_lse=grads[2])
        return dx, None, None, None, None


def token_log_probs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top_k: int = 0, scale: float = 1.0,
                    ignore_index: int = -100) -> kt_ops.TokenLogprobs:
    """kt_ops.token_logprobs over the last dimension of logits with any leading
    dimensions (those of targets), differentiable (once) through logprob, entropy
    and lse; the top alternatives carry no gradient."""
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    x = logits.reshape(-1, vocab)
    if x.shape[1] > 1 and x.stride(1) != 1:
        x = x.contiguous()
    if targets is not None:
        if targets.shape != lead:
            raise ValueError(f"targets must be {tuple(lead)}, got {tuple(targets.shape)}")
        targets = targets.reshape(-1).contiguous()
    if _recording(logits):
        r = kt_ops.TokenLogprobs(*_TokenLogProbs.apply(x, targets, top_k, scale, ignore_index))
    else:
        r = kt_ops.token_logprobs(x, targets, top_k, scale, ignore_index)
    return kt_ops.TokenLogprobs(r.logprob.view(lead) if r.logprob is not None else None, r.entropy.view(lead),
                                r.lse.view(lead), r.top_logprob.view(*lead, top_k), r.top_index.view(*lead, top_k))


class TunedMultiheadAttention(nn.Module):
    """Multi-head attention (batch_first) with the flash-attention kernel as its core."""

    def __init__(self, embed_dim: int, num_heads: int, dropout: float = 0.0, bias: bool = True,
                 results_dir: Optional[os.PathLike] = None, device=None, dtype=None) -> None:
        super().__init__()
        if embed_dim % num_heads:
            raise ValueError("embed_dim must be divisible by num_heads")
        self.embed_dim = embed_dim
        self.num_heads = num_heads
        self.head_dim = embed_dim // num_heads
        if self.head_dim not in (64, 128):
            raise ValueError(f"head dim {self.head_dim}: the attention kernel supports 64 and 128")
        self.scale = self.head_dim ** -0.5
        self.dropout = dropout
        self.tuned_params = load_best_params("attention", results_dir)
        self._lib = tuned_library("attention", results_dir)
        kw = dict(bias=bias, results_dir=results_dir, device=device, dtype=dtype)
        self.q_proj = TunedLinear(embed_dim, embed_dim, **kw)
        self.k_proj = TunedLinear(embed_dim, embed_dim, **kw)
        self.v_proj = TunedLinear(embed_dim, embed_dim, **kw)
        self.out_proj = TunedLinear(embed_dim, embed_dim, **kw)

    def _heads(self, t: torch.Tensor, B: int, S: int) -> torch.Tensor:
        return t.view(B, S, self.num_heads, self.head_dim).transpose(1, 2).contiguous().to(torch.bfloat16)

    def forward(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                key_padding_mask: Optional[torch.Tensor] = None, need_weights: bool = False,
                is_causal: bool = False) -> Tuple[torch.Tensor, None]:
        if key_padding_mask is not None:
            raise NotImplementedError("key_padding_mask is not supported by the attention kernel")
        if need_weights:
            raise NotImplementedError("the attention kernel does not form the weight matrix")
        if self.training and self.dropout > 0:
            raise NotImplementedError("attention dropout is not supported (inference layer)")
        B, S, _ = query.shape
        if key.shape[1] != S or value.shape[1] != S:
            raise NotImplementedError("query and key/value sequences of different lengths")
        q = self._heads(self.q_proj(query), B, S)
        k = self._heads(self.k_proj(key), B, S)
        v = self._heads(self.v_proj(value), B, S)
        o = kt_ops.fa_fwd(q, k, v, scale=self.scale, causal=is_causal, lib=self._lib)
        o = o.to(query.dtype).transpose(1, 2).reshape(B, S, self.embed_dim)
        return self.out_proj(o), None


def apply_tuned_layers(model: nn.Module, kernel: str = "matmul", results_dir: Optional[os.PathLike] = None) -> nn.Module:
    """Replace nn.Linear (kernel "matmul" or "all") and nn.LayerNorm ("layernorm" or "all")
    in `model` by their tuned versions, in place, keeping the weights; "w4" replaces
    nn.Linear by layers with 4-bit weights in groups of 128 (or else 64, 32) columns
    where one divides the input features."""
    for name, module in list(model.named_modules()):
        if not name:
            continue
        parent_name, _, child = name.rpartition(".")
        parent = model.get_submodule(parent_name) if parent_name else model
        new = None
        if kernel == "w4" and type(module) is nn.Linear:
            group = next((g for g in (128, 64, 32) if module.in_features % g == 0), None)
            if group is not None:
                setattr(parent, child, TunedLinearW4.from_linear(module, group))
            continue
        if kernel in ("matmul", "all") and type(module) is nn.Linear:
            new = TunedLinear(module.in_features, module.out_features, module.bias is not None,
                              results_dir=results_dir, device=module.weight.device, dtype=module.weight.dtype)
        elif kernel in ("layernorm", "all") and type(module) is nn.LayerNorm and module.elementwise_affine \
                and len(module.normalized_shape) == 1:
            new = TunedLayerNorm(module.normalized_shape[0], module.eps, results_dir=results_dir,
                                 device=module.weight.device, dtype=module.weight.dtype)
        if new is not None:
            new.load_state_dict(module.state_dict())
            setattr(parent, child, new)
    return model


@torch.no_grad()
def sdpa_comparison(batch: int = 4, heads: int = 8, seq_len: int = 1024, head_dim: int = 128, causal: bool = False,
                    warmup: int = 3, samples: int = 20, seed: int = 0, lib: Optional[kt_lib.KtLibrary] = None) -> dict:
    """The attention kernel against torch's scaled_dot_product_attention on the
    same bf16 inputs: normwise difference and mean CUDA-event times."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v = (torch.randn(batch, heads, seq_len, head_dim, device="cuda", dtype=torch.bfloat16, generator=g)
               for _ in range(3))
    scale = 1.0 / math.sqrt(head_dim)
    lib = lib or kt_lib.load()

    def ours():
        return kt_ops.fa_fwd(q, k, v, scale=scale, causal=causal, lib=lib)

    def sdpa():
        return F.scaled_dot_product_attention(q, k, v, is_causal=causal, scale=scale)

    def time_ms(fn) -> float:
        for _ in range(warmup):
            fn()
        ev = [(torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)) for _ in range(samples)]
        for a, b in ev:
            a.record()
            fn()
            b.record()
        torch.cuda.synchronize()
        return sum(a.elapsed_time(b) for a, b in ev) / samples

    a, b = ours().float(), sdpa().float()
    err = float((a - b).abs().max() / b.abs().max())
    t_ours, t_sdpa = time_ms(ours), time_ms(sdpa)
    pairs = seq_len * (seq_len + 1) // 2 if causal else seq_len * seq_len
    flops = 4 * batch * heads * pairs * head_dim
    return {"shape": [batch, heads, seq_len, head_dim], "causal": causal, "normwise_diff": err,
            "kt_ms": t_ours, "sdpa_ms": t_sdpa, "kt_tflops": flops / t_ours / 1e9, "sdpa_tflops": flops / t_sdpa / 1e9}
