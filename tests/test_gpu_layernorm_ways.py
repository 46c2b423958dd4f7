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
from test_gpu_layernorm_train import E, TYPES, check, half_step, inputs  # noqa: E402


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
