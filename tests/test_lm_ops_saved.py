"""
The backward pass of LayerNorm takes what it reads from the tensors that the
forward pass left, so it refuses those that are not on dy's device, or whose type
or size is not what the forward pass leaves. Both refuse an output that shares a
part of an input's memory. The same for what token log probabilities leave.
"""

from __future__ import annotations

import pytest

import kt_lib
import kt_ops
from test_lm_ops_refusals import P, ln_bwd, ln_fwd, refused

torch = pytest.importorskip("torch")


def saved_like(rows, cols, ckpt8, device):
    q8 = torch.zeros(rows, (cols + 7) // 8 * 8, dtype=torch.int8, device=device)[:, :cols]
    exp = torch.zeros(rows, (cols + 31) // 32, dtype=torch.uint8, device=device)
    return kt_ops.LayerNormSaved(None if ckpt8 else torch.zeros(rows, cols, device=device),
                                 q8 if ckpt8 else None, exp if ckpt8 else None, torch.ones(cols, device=device),
                                 torch.ones(2, rows, device=device), torch.float32)


@pytest.mark.parametrize("ckpt8", [False, True])
def test_tensors_on_the_host_are_refused(ckpt8):
    with pytest.raises(ValueError, match="CUDA"):
        kt_ops.layernorm_bwd(torch.zeros(4, 64), saved_like(4, 64, ckpt8, "cpu"))


@pytest.mark.gpu
@pytest.mark.parametrize("ckpt8", [False, True])
def test_saved_tensors_that_do_not_fit_are_refused(dev, lib, ckpt8):
    rows, cols = 6, 100
    dy = torch.ones(rows, cols, device=dev)
    good = saved_like(rows, cols, ckpt8, dev)
    kt_ops.layernorm_bwd(dy, good, lib=lib)
    bad = [dict(stats=good.stats.cpu()), dict(stats=good.stats[:, :5].contiguous()), dict(stats=good.stats[0]),
           dict(stats=good.stats.double()), dict(stats=torch.ones(4, rows, device=dev)[::2]),
           dict(gamma=good.gamma.cpu()), dict(gamma=good.gamma[:99]), dict(gamma=good.gamma.double()),
           dict(gamma=torch.ones(200, device=dev)[::2]), dict(beta_dtype=torch.float64)]
    if ckpt8:
        bad += [dict(q8=good.q8.cpu()), dict(q8=good.q8.float()), dict(q8=good.q8[:5]), dict(q8=good.q8[:, :99]),
                dict(q8=good.q8.contiguous().view(-1)), dict(q8=None), dict(q8=good.q8[:1].expand(rows, cols)),
                dict(q8_exp=good.q8_exp.cpu()), dict(q8_exp=good.q8_exp[:, :3].contiguous()), dict(q8_exp=None),
                dict(q8_exp=good.q8_exp.float()), dict(q8_exp=torch.zeros(rows, 8, dtype=torch.uint8, device=dev)[:, ::2]),
                dict(q8_exp=good.q8_exp[:5])]
    else:
        bad += [dict(x=good.x.cpu()), dict(x=good.x.half()), dict(x=good.x[:5]), dict(x=good.x.t().contiguous().t()),
                dict(x=good.x.view(-1)), dict(x=None)]
    for change in bad:
        with pytest.raises(ValueError):
            kt_ops.layernorm_bwd(dy, good._replace(**change), lib=lib)
    with pytest.raises(ValueError):
        kt_ops.layernorm_bwd(dy.cpu(), good, lib=lib)


def test_outputs_that_overlap_a_part_of_an_input_are_refused(lib):
    size = 4 * 64 * 4  # of the tensors
    for shift in (4, -4, size - 4, 4 - size):
        refused(lambda: ln_fwd(lib, y=P + shift))
        refused(lambda: ln_bwd(lib, dx=P + shift))
        refused(lambda: ln_bwd(lib, dx=P + 2 * size, x=P + 2 * size + shift))
        refused(lambda: ln_bwd(lib, x=None, q8=P, q8_exp=P, dx=P + shift))
        refused(lambda: ln_fwd(lib, y=P + shift // 2, dtype=kt_lib.KT_BF16, wdtype=kt_lib.KT_BF16))


def train(lib, norm=P, logits=P, lse=P, rows=4, vocab=100, scale=1.0, top_k=0, targets=P, logprob=P):
    lib.token_logprobs_train(logits, vocab, targets, rows, vocab, scale, -100, top_k, logprob, P, lse, norm, None, None, 0)


def train_bwd(lib, norm=P, logits=P, dx=P, rows=4, vocab=100, scale=1.0, targets=P, entropy=P, ld_dx=100):
    lib.token_logprobs_train_bwd(logits, vocab, targets, norm, entropy, P, P, P, rows, vocab, scale, -100, dx, ld_dx, 0)


def test_token_logprobs_for_training_refuse(lib):
    for bad in (dict(norm=None), dict(norm=P + 4), dict(logits=0), dict(lse=0), dict(rows=-1), dict(scale=0.0),
                dict(top_k=2), dict(logprob=None)):
        refused(lambda: train(lib, **bad))
    for bad in (dict(norm=None), dict(norm=P + 4), dict(logits=0), dict(dx=0), dict(rows=-1), dict(scale=0.0),
                dict(targets=None), dict(entropy=None), dict(ld_dx=99)):
        refused(lambda: train_bwd(lib, **bad))
    train(lib, norm=None, logits=0, rows=0)
    train_bwd(lib, norm=None, logits=0, rows=0)


class Recorder:
    """Takes the library's place and launches nothing."""

    def layernorm_bwd_workspace_bytes(self, rows, cols):
        return 16

    def layernorm_train_bwd(self, dy, x, q8, q8_exp, ld_q8, *rest):
        self.q8, self.ld_q8 = q8, ld_q8


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(1, 13), (1, 16), (7, 13), (7, 16)])
def test_checkpoint_rows_are_read_within_their_memory(dev, rows, cols):
    """The kernels read rows whose distance is a multiple of 8 up to their next
    whole 8 bytes. A copy of a row has the distance and not the bytes."""
    dy, saved, lib = torch.ones(rows, cols, device=dev), saved_like(rows, cols, True, dev), Recorder()
    tight = torch.zeros((rows - 1) * 16 + cols, dtype=torch.int8, device=dev)
    copies = [saved.q8, saved.q8.clone(), saved.q8.contiguous(), torch.as_strided(tight, (rows, cols), (16, 1))]
    for q8 in copies:
        kt_ops.layernorm_bwd(dy, saved._replace(q8=q8), lib=lib)
        assert lib.ld_q8 >= cols
        if lib.q8 == q8.data_ptr():
            last = cols if lib.ld_q8 % 8 else (cols + 7) // 8 * 8
            assert q8.storage_offset() + (rows - 1) * lib.ld_q8 + last <= q8.untyped_storage().nbytes()
    kt_ops.layernorm_bwd(dy, saved, lib=lib)
    assert lib.ld_q8 == 16  # with its bytes behind the row, as the forward pass leaves it
