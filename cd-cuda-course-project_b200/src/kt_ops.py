"""
kt_ops.py — torch-facing wrappers over the C ABI.

torch provides device memory and streams only; every computation goes
through the loaded kernel library. Each wrapper checks device, dtype and
contiguity, allocates the output, and launches on torch's current stream (the
training and serving operators: of their tensors' device).
There is no CPU or torch fallback: a missing library raises.
"""

from __future__ import annotations

import functools
import math
from typing import NamedTuple, Optional

import torch

import kt_lib


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _check(t: torch.Tensor, name: str, dtype: torch.dtype) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def softmax(x: torch.Tensor, out: Optional[torch.Tensor] = None, lib: Optional[kt_lib.KtLibrary] = None) -> torch.Tensor:
    """Row softmax over the last dim of a 2-D fp32 tensor."""
    _check(x, "x", torch.float32)
    if x.dim() != 2:
        raise ValueError("x must be 2-D (rows, cols)")
    lib = lib or kt_lib.load()
    y = out if out is not None else torch.empty_like(x)
    lib.softmax_f32(x.data_ptr(), y.data_ptr(), x.shape[0], x.shape[1], _stream())
    return y


def layernorm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-5,
              out: Optional[torch.Tensor] = None, lib: Optional[kt_lib.KtLibrary] = None) -> torch.Tensor:
    """LayerNorm over the last dim of a 2-D fp32 tensor (biased variance)."""
    for t, n in ((x, "x"), (gamma, "gamma"), (beta, "beta")):
        _check(t, n, torch.float32)
    if x.dim() != 2 or gamma.numel() != x.shape[1] or beta.numel() != x.shape[1]:
        raise ValueError("layernorm: x (rows, cols), gamma/beta (cols,)")
    lib = lib or kt_lib.load()
    y = out if out is not None else torch.empty_like(x)
    lib.layernorm_f32(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(),
                      x.shape[0], x.shape[1], float(eps), _stream())
    return y


class ReduceWorkspace:
    """Caller-owned scratch for kt_reduce_sum_f32, reusable across calls."""

    def __init__(self, n: int, device: torch.device | str = "cuda", lib: Optional[kt_lib.KtLibrary] = None):
        lib = lib or kt_lib.load()
        self.bytes = lib.reduce_workspace_bytes(n)
        self.buf = torch.empty(max(self.bytes, 16), dtype=torch.uint8, device=device)


def reduce_sum(x: torch.Tensor, out64: Optional[torch.Tensor] = None, out32: Optional[torch.Tensor] = None,
               workspace: Optional[ReduceWorkspace] = None,
               lib: Optional[kt_lib.KtLibrary] = None) -> torch.Tensor:
    """Sum of all elements of an fp32 tensor, accumulated in fp64 (returns a 1-element fp64 tensor)."""
    _check(x, "x", torch.float32)
    lib = lib or kt_lib.load()
    n = x.numel()
    if out64 is None:
        out64 = torch.empty(1, dtype=torch.float64, device=x.device)
    ws = workspace or ReduceWorkspace(n, x.device, lib)
    lib.reduce_sum_f32(x.data_ptr(), n, out64.data_ptr(), out32.data_ptr() if out32 is not None else None,
                       ws.buf.data_ptr(), ws.bytes, _stream())
    return out64


def gemm(A: torch.Tensor, B: torch.Tensor, transpose_b: bool = False, variant: int = kt_lib.KT_GEMM_TF32,
         out: Optional[torch.Tensor] = None, lib: Optional[kt_lib.KtLibrary] = None) -> torch.Tensor:
    """C = A·B, or A·Bt^T when transpose_b (B then holds Bt, shape N×K)."""
    _check(A, "A", torch.float32)
    _check(B, "B", torch.float32)
    M, K = A.shape
    if transpose_b:
        N, K2 = B.shape
    else:
        K2, N = B.shape
    if K2 != K:
        raise ValueError(f"gemm: inner dims differ ({K} vs {K2})")
    lib = lib or kt_lib.load()
    C = out if out is not None else torch.empty((M, N), dtype=torch.float32, device=A.device)
    lib.gemm_f32(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, transpose_b, variant, _stream())
    return C


def fa_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None,
           causal: bool = False, out: Optional[torch.Tensor] = None,
           lib: Optional[kt_lib.KtLibrary] = None) -> torch.Tensor:
    """Flash-attention forward on bf16 [B, H, S, D] tensors."""
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _check(t, n, torch.bfloat16)
    if q.dim() != 4 or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("fa_fwd: q, k, v must share shape [B, H, S, D]")
    B, H, S, D = q.shape
    lib = lib or kt_lib.load()
    o = out if out is not None else torch.empty_like(q)
    sc = float(scale) if scale is not None else 1.0 / math.sqrt(D)
    lib.fa_fwd_bf16(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), B, H, S, D, sc, causal, _stream())
    return o


# ---------------------------------------------------------------------------
# Training and serving operators (fp32, bf16, fp16)
# ---------------------------------------------------------------------------

_DTYPES = {torch.float32: kt_lib.KT_F32, torch.bfloat16: kt_lib.KT_BF16, torch.float16: kt_lib.KT_F16}


def _dtype(t: torch.Tensor, name: str) -> int:
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return dt


def _dense(t: torch.Tensor, name: str, dtype: torch.dtype, device: int) -> None:
    """A contiguous tensor of `dtype` on CUDA device `device`."""
    if not (t.dtype is dtype and t.get_device() == device and t.is_contiguous()):
        _check(t, name, dtype)
        raise ValueError(f"{name} is on {t.device}, not on cuda:{device}")


def _rows(t: torch.Tensor, name: str) -> int:
    """A 2-D CUDA tensor whose rows are dense and any distance apart; returns that distance in elements."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D")
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the elements of a row must be contiguous")
    return t.stride(0) if rows > 1 else cols


def _launch(device: int, fn, *args) -> None:
    """fn(*args, stream) on that device and its current stream."""
    if device == torch._C._cuda_getDevice():  # (torch.cuda.current_device takes twice as long)
        fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            fn(*args, torch._C._cuda_getCurrentRawStream(device))


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return t.data_ptr() if t is not None else None


class LayerNormSaved(NamedTuple):
    """What layernorm_train keeps for layernorm_bwd: the input x, or its 8-bit
    checkpoint (q8, q8_exp; include/kt_abi.h has the format), gamma, the rows'
    statistics (2, rows), and beta's type (None without beta)."""
    x: Optional[torch.Tensor]
    q8: Optional[torch.Tensor]
    q8_exp: Optional[torch.Tensor]
    gamma: Optional[torch.Tensor]
    stats: torch.Tensor
    beta_dtype: Optional[torch.dtype]

    @property
    def mean(self) -> torch.Tensor:
        return self.stats[0]

    @property
    def rstd(self) -> torch.Tensor:
        return self.stats[1]


def layernorm_train(x: torch.Tensor, gamma: Optional[torch.Tensor] = None, beta: Optional[torch.Tensor] = None,
                    eps: float = 1e-5, ckpt8: bool = False,
                    lib: Optional[kt_lib.KtLibrary] = None) -> tuple[torch.Tensor, LayerNormSaved]:
    """LayerNorm over the last dim of a 2-D fp32, bf16 or fp16 tensor, and what its backward pass needs.

    gamma and beta (None: 1 and 0) are fp32 or of x's type. With ckpt8 the
    backward pass gets x in 8 bits (blocks of 32 columns sharing a power of
    two), so that x itself need not be kept.
    """
    dt = _dtype(x, "x")
    _check(x, "x", x.dtype)
    if x.dim() != 2:
        raise ValueError("x must be 2-D (rows, cols)")
    rows, cols = x.shape
    dev = x.get_device()
    wdt = kt_lib.KT_F32
    beta_dtype = None
    if gamma is not None:
        wdt = _dtype(gamma, "gamma")
        _dense(gamma, "gamma", torch.float32 if wdt == kt_lib.KT_F32 else x.dtype, dev)
        if gamma.numel() != cols:
            raise ValueError(f"layernorm_train: gamma must have {cols} elements")
    if beta is not None:
        beta_dtype = beta.dtype
        wdt_beta = _dtype(beta, "beta")
        _dense(beta, "beta", torch.float32 if wdt_beta == kt_lib.KT_F32 else x.dtype, dev)
        if beta.numel() != cols:
            raise ValueError(f"layernorm_train: beta must have {cols} elements")
        if gamma is not None and wdt_beta != wdt:
            raise ValueError("layernorm_train: gamma and beta must be of one type")
        wdt = wdt_beta
    if lib is None:
        lib = kt_lib.load()
    y = torch.empty_like(x)
    stats = x.new_empty((2, rows), dtype=torch.float32)
    at = stats.data_ptr()
    q8 = q8_exp = None
    ld_q8 = 0
    if ckpt8:
        ld_q8 = (cols + 7) // 8 * 8  # rows of whole 8-byte words
        q8 = x.new_empty((rows, ld_q8), dtype=torch.int8)
        if ld_q8 != cols:
            q8 = q8[:, :cols]
        q8_exp = x.new_empty((rows, (cols + 31) // 32), dtype=torch.uint8)
    _launch(dev, lib.layernorm_train_fwd, x.data_ptr(), _ptr(gamma), _ptr(beta), y.data_ptr(), at, at + 4 * rows,
            _ptr(q8), _ptr(q8_exp), ld_q8, rows, cols, eps, dt, wdt)
    return y, LayerNormSaved(None if ckpt8 else x, q8, q8_exp, gamma, stats, beta_dtype)


@functools.lru_cache(maxsize=1024)
def _ln_workspace(lib: kt_lib.KtLibrary, rows: int, cols: int) -> int:
    """The workspace's size, a pure function of the shape; a call into the library takes 1 us."""
    return lib.layernorm_bwd_workspace_bytes(rows, cols)


def layernorm_bwd(dy: torch.Tensor, saved: LayerNormSaved, weight_grads: bool = True,
                  lib: Optional[kt_lib.KtLibrary] = None
                  ) -> tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dx, dgamma, dbeta) of layernorm_train from dy. dgamma and dbeta are of
    gamma's type and None where gamma or beta was None, or weight_grads is False."""
    x, q8, q8_exp, gamma, stats, beta_dtype = saved
    dt = _dtype(dy, "dy")
    _check(dy, "dy", dy.dtype if x is None else x.dtype)
    dev = dy.get_device()
    kept = q8 if x is None else x
    if kept is None or dy.shape != kept.shape or dy.dim() != 2:
        raise ValueError(f"layernorm_bwd: dy is {tuple(dy.shape)}, the input was "
                         f"{tuple(kept.shape) if kept is not None else 'not saved'}")
    rows, cols = dy.shape
    ld_q8 = 0
    if x is None:
        ld_q8 = q8.stride(0) if rows > 1 else max(q8.stride(0), cols)
        if not (q8.dtype is torch.int8 and q8.get_device() == dev and (q8.stride(1) == 1 or cols == 1) and ld_q8 >= cols):
            raise ValueError("q8 must be int8 on dy's device, the elements of a row contiguous")
        # the kernels read whole 8 bytes of rows that are a multiple of 8 apart; a copy's last row may end before
        if cols % 8 and ld_q8 % 8 == 0 and q8.untyped_storage().nbytes() < \
                q8.storage_offset() + (rows - 1) * ld_q8 + (cols + 7) // 8 * 8:
            q8 = q8.contiguous()
            ld_q8 = cols
        if q8_exp is None or not (q8_exp.dtype is torch.uint8 and q8_exp.get_device() == dev
                                  and q8_exp.is_contiguous() and q8_exp.numel() == rows * ((cols + 31) // 32)):
            raise ValueError(f"q8_exp must be uint8 on dy's device, contiguous and {(rows, (cols + 31) // 32)}")
    else:
        _dense(x, "x", dy.dtype, dev)
    if not (stats.dtype is torch.float32 and stats.get_device() == dev and stats.is_contiguous()
            and stats.numel() == 2 * rows):
        raise ValueError(f"stats must be float32 on dy's device, contiguous and {(2, rows)}")
    wt = gamma.dtype if gamma is not None else beta_dtype or torch.float32
    wdt = _DTYPES.get(wt)
    if wdt not in (kt_lib.KT_F32, dt) or (gamma is not None and beta_dtype not in (None, wt)):
        raise ValueError(f"dy and the weights must be of one type or the weights fp32, got {dy.dtype} and {wt}")
    if gamma is not None and not (gamma.get_device() == dev and gamma.is_contiguous() and gamma.numel() == cols):
        raise ValueError(f"gamma must be on dy's device, contiguous and have {cols} elements")
    if lib is None:
        lib = kt_lib.load()
    dx = torch.empty_like(dy)
    dgamma = dbeta = ws = None
    ws_bytes = 0
    if weight_grads and (gamma is not None or beta_dtype is not None):
        dgamma = torch.empty_like(gamma) if gamma is not None else None
        if beta_dtype is not None:
            dbeta = torch.empty_like(gamma) if gamma is not None and gamma.dim() == 1 else dy.new_empty(cols, dtype=wt)
        ws_bytes = _ln_workspace(lib, rows, cols)
        ws = stats.new_empty(ws_bytes // 4)
    at = stats.data_ptr()
    _launch(dev, lib.layernorm_train_bwd, dy.data_ptr(), _ptr(x), _ptr(q8), _ptr(q8_exp), ld_q8, _ptr(gamma), at,
            at + 4 * rows, dx.data_ptr(), _ptr(dgamma), _ptr(dbeta), rows, cols, dt, wdt, _ptr(ws), ws_bytes)
    return dx, dgamma, dbeta


class _TokenLogprobs(NamedTuple):
    logprob: Optional[torch.Tensor]
    entropy: torch.Tensor
    lse: torch.Tensor
    top_logprob: torch.Tensor
    top_index: torch.Tensor


class TokenLogprobs(_TokenLogprobs):
    """Per row of logits: the target's log probability (None without targets),
    the entropy (nats), log sum exp, and the top k log probabilities with their columns (int64).

    Beside these five, token_logprobs' result has `norm`, (rows, 2) fp32: what
    the gradient takes in lse's place, which is rounded (include/kt_abi.h)."""
    norm: Optional[torch.Tensor] = None


def _per_row(t: torch.Tensor, name: str, dtype: torch.dtype, rows: int, device: int) -> None:
    if not (t.dtype is dtype and t.get_device() == device and t.dim() == 1 and t.numel() == rows
            and t.is_contiguous()):
        _dense(t, name, dtype, device)
        raise ValueError(f"{name} must be ({rows},), got {tuple(t.shape)}")


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top_k: int = 0, scale: float = 1.0,
                   ignore_index: int = -100, lib: Optional[kt_lib.KtLibrary] = None) -> TokenLogprobs:
    """Log probabilities of `targets` under softmax(scale * logits), with the
    entropy and the top_k (up to 32) most likely columns of each row.

    logits: (rows, vocab) fp32, bf16 or fp16, rows any distance apart; targets:
    (rows,) int64. Rows whose target is ignore_index get log probability 0;
    other targets that are no column get NaN, in the gradient too, and set the
    library's device error.
    """
    dt = _dtype(logits, "logits")
    ld = _rows(logits, "logits")
    rows, vocab = logits.shape
    dev = logits.get_device()
    if targets is not None:
        _per_row(targets, "targets", torch.int64, rows, dev)
    if not 0 <= top_k <= 32 or (rows and top_k > vocab):
        raise ValueError(f"top_k must be between 0 and min(32, vocab), got {top_k}")
    if lib is None:
        lib = kt_lib.load()
    entropy = logits.new_empty(rows, dtype=torch.float32)
    logprob = torch.empty_like(entropy) if targets is not None else None
    lse = torch.empty_like(entropy)
    # (sizes one by one, and a tensor of the right type to start from, take a third less time)
    norm = entropy.new_empty(rows, 2)
    top_logprob = entropy.new_empty(rows, top_k)
    if targets is not None:
        top_index = targets.new_empty(rows, top_k)
    else:
        top_index = logits.new_empty(rows, top_k, dtype=torch.int64)
    _launch(dev, lib.token_logprobs_train, logits.data_ptr(), ld, _ptr(targets), rows, vocab, scale, ignore_index,
            top_k, _ptr(logprob), entropy.data_ptr(), lse.data_ptr(), norm.data_ptr(), top_logprob.data_ptr(),
            top_index.data_ptr(), dt)
    result = tuple.__new__(TokenLogprobs, (logprob, entropy, lse, top_logprob, top_index))
    result.norm = norm
    return result


def token_logprobs_bwd(logits: torch.Tensor, targets: Optional[torch.Tensor], result: TokenLogprobs,
                       grad_logprob: Optional[torch.Tensor] = None, grad_entropy: Optional[torch.Tensor] = None,
                       scale: float = 1.0, ignore_index: int = -100, out: Optional[torch.Tensor] = None,
                       lib: Optional[kt_lib.KtLibrary] = None,
                       grad_lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of the logits from those of the log probabilities, the entropies
    and lse (fp32, (rows,); None: 0); result, scale and ignore_index are those
    of token_logprobs. `out` may be the logits themselves, not a part of their memory.
    A result without its norm (put together anew) has it computed again from the logits."""
    dt = _dtype(logits, "logits")
    ld = _rows(logits, "logits")
    rows, vocab = logits.shape
    dev = logits.get_device()
    _per_row(result.entropy, "result.entropy", torch.float32, rows, dev)
    if grad_logprob is not None:
        _per_row(grad_logprob, "grad_logprob", torch.float32, rows, dev)
        if targets is None:
            raise ValueError("grad_logprob needs targets")
    if grad_entropy is not None:
        _per_row(grad_entropy, "grad_entropy", torch.float32, rows, dev)
    if grad_lse is not None:
        _per_row(grad_lse, "grad_lse", torch.float32, rows, dev)
    if targets is not None:
        _per_row(targets, "targets", torch.int64, rows, dev)
    if out is None:
        out = logits.new_empty((rows, vocab))
        ld_out = vocab
    else:
        ld_out = _rows(out, "out")
        if out.shape != logits.shape or out.dtype != logits.dtype or out.get_device() != dev:
            raise ValueError(f"out must be {tuple(logits.shape)} {logits.dtype} on {logits.device}")
        if rows > 1 and ld_out < vocab:
            raise ValueError("out: rows overlap")
        at, to, size = logits.data_ptr(), out.data_ptr(), logits.element_size()
        if rows and (at, ld) != (to, ld_out) and at < to + ((rows - 1) * ld_out + vocab) * size \
                and to < at + ((rows - 1) * ld + vocab) * size:
            raise ValueError("out overlaps the logits without being the same")
    if lib is None:
        lib = kt_lib.load()
    norm = getattr(result, "norm", None)
    if norm is None:
        norm = token_logprobs(logits, scale=scale, lib=lib).norm
    _dense(norm, "result.norm", torch.float32, dev)
    if norm.numel() != 2 * rows:
        raise ValueError(f"result.norm must be {(rows, 2)}, got {tuple(norm.shape)}")
    _launch(dev, lib.token_logprobs_train_bwd, logits.data_ptr(), ld, _ptr(targets), norm.data_ptr(),
            result.entropy.data_ptr(), _ptr(grad_logprob), _ptr(grad_entropy), _ptr(grad_lse), rows, vocab, scale, ignore_index,
            out.data_ptr(), ld_out, dt)
    return out


class W4Weight(NamedTuple):
    """An (N, K) matrix of 4-bit weights: packed (N, K/2) uint8, the even column
    in the low half of a byte; scales (N, K/group) of the tokens' type;
    zeros (N, K/group) uint8 with values of 0..15, or None for 8. A weight is
    scale * (q - zero)."""
    packed: torch.Tensor
    scales: torch.Tensor
    zeros: Optional[torch.Tensor] = None
    group: int = 128


def w4_quantize(weight: torch.Tensor, group: int = 128, scale_dtype: Optional[torch.dtype] = None,
                lib: Optional[kt_lib.KtLibrary] = None) -> W4Weight:
    """An (N, K) fp32, bf16 or fp16 matrix as symmetric 4-bit weights with one
    scale (of scale_dtype, default the matrix's type) per `group` (32, 64 or 128) columns."""
    dt = _dtype(weight, "weight")
    _check(weight, "weight", weight.dtype)
    if weight.dim() != 2:
        raise ValueError("weight must be 2-D (N, K)")
    N, K = weight.shape
    if group not in (32, 64, 128) or K % group:
        raise ValueError(f"group must be 32, 64 or 128 and divide K={K}, got {group}")
    lib = lib or kt_lib.load()
    packed = weight.new_empty((N, K // 2), dtype=torch.uint8)
    scales = weight.new_empty((N, K // group), dtype=scale_dtype or weight.dtype)
    _launch(weight.get_device(), lib.w4_quantize, weight.data_ptr(), N, K, group, dt, packed.data_ptr(),
            scales.data_ptr(), _dtype(scales, "scales"))
    return W4Weight(packed, scales, None, group)


def w4_linear(x: torch.Tensor, weight: W4Weight, bias: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None, lib: Optional[kt_lib.KtLibrary] = None) -> torch.Tensor:
    """y = x w^T + bias for a few tokens x (M, K), fp32, bf16 or fp16, with 4-bit weights."""
    packed, scales, zeros, group = weight
    dt = _dtype(x, "x")
    ldx = _rows(x, "x")
    M, K = x.shape
    dev = x.get_device()
    _dense(packed, "packed", torch.uint8, dev)
    _dense(scales, "scales", x.dtype, dev)
    if packed.dim() != 2 or packed.shape[1] * 2 != K:
        raise ValueError(f"w4_linear: packed must be (N, {K // 2}), got {tuple(packed.shape)}")
    N = packed.shape[0]
    if group not in (32, 64, 128) or K % group:
        raise ValueError(f"group must be 32, 64 or 128 and divide K={K}, got {group}")
    if scales.shape != (N, K // group):
        raise ValueError(f"w4_linear: scales must be {(N, K // group)}, got {tuple(scales.shape)}")
    if zeros is not None:
        _dense(zeros, "zeros", torch.uint8, dev)
        if zeros.shape != scales.shape:
            raise ValueError(f"w4_linear: zeros must be {(N, K // group)}, got {tuple(zeros.shape)}")
    if bias is not None:
        _dense(bias, "bias", x.dtype, dev)
        if bias.numel() != N:
            raise ValueError(f"w4_linear: bias must have {N} elements")
    if out is None:
        out = x.new_empty((M, N))
    else:
        _dense(out, "out", x.dtype, dev)
        if out.shape != (M, N):
            raise ValueError(f"out must be {(M, N)}, got {tuple(out.shape)}")
    if lib is None:
        lib = kt_lib.load()
    _launch(dev, lib.w4_linear, x.data_ptr(), ldx, packed.data_ptr(), scales.data_ptr(), _ptr(zeros), _ptr(bias),
            out.data_ptr(), N, M, N, K, group, dt)
    return out
