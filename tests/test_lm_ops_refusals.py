"""
The training and serving operators without a GPU: the C entry points refuse bad
arguments before any CUDA call, the torch wrappers refuse tensors that are not
on a CUDA device, and tuning variants do not build these operators.
"""

from __future__ import annotations

import pytest

import kt_lib
import kt_ops

torch = pytest.importorskip("torch")

P = 1 << 20  # an aligned address that is never read


def refused(fn, *statuses):
    with pytest.raises(kt_lib.KtError) as ei:
        fn()
    assert ei.value.status in (statuses or (kt_lib.KT_ERR_ARG,)), ei.value
    assert ei.value.message


def ln_fwd(lib, x=P, gamma=P, beta=P, y=P, mean=P, rstd=P, q8=None, q8_exp=None, rows=4, cols=64, eps=1e-5, dtype=0,
           wdtype=0, ld_q8=64):
    lib.layernorm_train_fwd(x, gamma, beta, y, mean, rstd, q8, q8_exp, ld_q8, rows, cols, eps, dtype, wdtype)


def ln_bwd(lib, dy=P, x=P, q8=None, q8_exp=None, gamma=P, mean=P, rstd=P, dx=P, dgamma=P, dbeta=P, rows=4, cols=64,
           dtype=0, wdtype=0, ws=P, ws_bytes=1 << 20, ld_q8=64):
    lib.layernorm_train_bwd(dy, x, q8, q8_exp, ld_q8, gamma, mean, rstd, dx, dgamma, dbeta, rows, cols, dtype, wdtype,
                            ws, ws_bytes)


@pytest.mark.parametrize("bad", [dict(x=0), dict(y=0), dict(mean=0), dict(rstd=0), dict(rows=-1), dict(cols=-1),
                                 dict(eps=-1.0), dict(eps=float("nan")), dict(dtype=3), dict(dtype=-1),
                                 dict(dtype=1, wdtype=2), dict(dtype=0, wdtype=1), dict(q8=P), dict(q8_exp=P),
                                 dict(q8=P, q8_exp=P, ld_q8=63), dict(x=P + 2), dict(gamma=P + 1), dict(dtype=1, x=P + 1)])
def test_layernorm_train_fwd(lib, bad):
    refused(lambda: ln_fwd(lib, **bad))


@pytest.mark.parametrize("bad", [dict(dy=0), dict(dx=0), dict(mean=0), dict(rstd=0), dict(x=None),
                                 dict(q8=P, q8_exp=P), dict(q8=P), dict(rows=-1), dict(dtype=9),
                                 dict(x=None, q8=P, q8_exp=P, ld_q8=63),
                                 dict(dtype=2, wdtype=1), dict(ws=0), dict(ws_bytes=16), dict(ws=P + 8),
                                 dict(dgamma=P + 2), dict(dy=P + 3)])
def test_layernorm_train_bwd(lib, bad):
    refused(lambda: ln_bwd(lib, **bad))


def test_layernorm_workspace(lib):
    f = lib.layernorm_bwd_workspace_bytes
    assert f(0, 10) == f(10, 0) == f(-1, 5) == 0
    assert f(1, 64) == 2 * 64 * 4
    assert f(10 ** 7, 64) == f(10 ** 6, 64) > f(100, 64)


def logprobs(lib, logits=P, ld=100, targets=P, rows=4, vocab=100, scale=1.0, top_k=0, logprob=P, entropy=P, lse=P,
             top_logprob=P, top_index=P, dtype=0):
    lib.token_logprobs(logits, ld, targets, rows, vocab, scale, -100, top_k, logprob, entropy, lse, top_logprob,
                       top_index, dtype)


@pytest.mark.parametrize("bad", [dict(logits=0), dict(lse=0), dict(logprob=None), dict(rows=-1), dict(vocab=-1),
                                 dict(vocab=0), dict(ld=-1), dict(scale=0.0), dict(scale=-2.0),
                                 dict(scale=float("inf")), dict(scale=float("nan")), dict(scale=3e38),
                                 dict(top_k=-1), dict(top_k=33),
                                 dict(vocab=3, top_k=4), dict(top_k=2, top_logprob=None),
                                 dict(top_k=2, top_index=None), dict(dtype=5), dict(logits=P + 2),
                                 dict(targets=P + 4)])
def test_token_logprobs(lib, bad):
    refused(lambda: logprobs(lib, **bad))


def logprobs_bwd(lib, logits=P, ld=100, targets=P, lse=P, entropy=P, g=P, h=P, rows=4, vocab=100, scale=1.0, dx=P,
                 ld_dx=100, dtype=0):
    lib.token_logprobs_bwd(logits, ld, targets, lse, entropy, g, h, rows, vocab, scale, -100, dx, ld_dx, dtype)


@pytest.mark.parametrize("bad", [dict(logits=0), dict(dx=0), dict(lse=0), dict(entropy=None), dict(targets=None),
                                 dict(rows=-1), dict(vocab=0), dict(scale=0.0), dict(ld_dx=99), dict(dtype=4),
                                 dict(dx=P + 1)])
def test_token_logprobs_bwd(lib, bad):
    refused(lambda: logprobs_bwd(lib, **bad))


def w4(lib, x=P, ldx=256, packed=P, scales=P, zeros=None, bias=None, y=P + (1 << 16), ldy=64, M=2, N=64, K=256,
       group=128, dtype=0):
    lib.w4_linear(x, ldx, packed, scales, zeros, bias, y, ldy, M, N, K, group, dtype)


@pytest.mark.parametrize("bad", [dict(x=0), dict(packed=0), dict(scales=0), dict(y=0), dict(M=-1), dict(N=-1),
                                 dict(K=-128), dict(K=0), dict(K=192), dict(group=48), dict(group=0), dict(dtype=3),
                                 dict(ldx=-1), dict(ldy=63), dict(packed=P + 8), dict(x=P + 2), dict(scales=P + 1),
                                 dict(K=1 << 18), dict(y=P), dict(y=P + 2 * 256 * 4 - 4), dict(y=P - 128 * 4 + 4)])
def test_w4_linear(lib, bad):
    refused(lambda: w4(lib, **bad), kt_lib.KT_ERR_ARG, kt_lib.KT_ERR_UNSUPPORTED)


@pytest.mark.parametrize("bad", [dict(w=0), dict(packed=0), dict(scales=0), dict(N=-1), dict(K=100), dict(group=16),
                                 dict(dtype=3), dict(scale_dtype=7)])
def test_w4_quantize(lib, bad):
    a = dict(w=P, N=8, K=128, group=64, dtype=0, packed=P, scales=P, scale_dtype=0) | bad
    refused(lambda: lib.w4_quantize(**a), kt_lib.KT_ERR_ARG, kt_lib.KT_ERR_UNSUPPORTED)


def test_empty_calls_reach_no_device(lib):
    ln_fwd(lib, x=0, y=0, rows=0)
    ln_fwd(lib, x=0, y=0, cols=0)
    ln_bwd(lib, dy=0, x=0, cols=0)
    logprobs(lib, logits=0, rows=0)
    logprobs_bwd(lib, logits=0, rows=0)
    w4(lib, x=0, M=0)
    w4(lib, x=0, N=0, ldy=0)
    lib.w4_quantize(0, 0, 128, 64, 0, 0, 0, 0)


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(4, 64)
    w = kt_ops.W4Weight(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 1), None, 64)
    for f in (lambda: kt_ops.layernorm_train(x), lambda: kt_ops.token_logprobs(x),
              lambda: kt_ops.w4_quantize(x, 32), lambda: kt_ops.w4_linear(x, w)):
        with pytest.raises(ValueError, match="CUDA"):
            f()


def test_tuning_variants_do_not_build_them(tmp_path, monkeypatch):
    monkeypatch.setenv("KT_RESULTS_DIR", str(tmp_path))
    import generator
    ok, log, so = generator.ensure_variant("layernorm", {"block_size": 128, "vec_per_thread": 8, "min_blocks": 1})
    assert ok, log
    v = kt_lib.KtLibrary(so)
    for f in (lambda: ln_fwd(v), lambda: ln_bwd(v), lambda: logprobs(v), lambda: logprobs_bwd(v), lambda: w4(v),
              lambda: v.w4_quantize(P, 8, 128, 64, 0, P, P, 0)):
        refused(f, kt_lib.KT_ERR_UNSUPPORTED)
    assert v.layernorm_bwd_workspace_bytes(10, 10) == 0
