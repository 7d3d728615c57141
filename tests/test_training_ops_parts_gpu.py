"""Backward calls of the gated feed-forward block that ask for part of the gradients: what they return has
the bits of the full call, for every family of kernels."""

import itertools

import pytest
import torch

from kfold_amd import ops
from tests.test_training_ops_gpu import BF, F32, ffn_inputs

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


# rows kept in registers at C = 64, 128, 256; tiles of 256 x 128 and 64 x 64; a contraction cut for dx; fp32
@pytest.mark.parametrize("M,C,F,dtype", [(16_400, 64, 32, BF), (16_500, 128, 64, BF), (16_390, 256, 32, BF), (33_000, 136, 40, BF),
                                         (45, 64, 72, BF), (37, 64, 768, BF), (700, 72, 40, F32), (45, 64, 384, F32)])
def test_gated_ffn_parts_of_the_gradients(M, C, F, dtype):
    print(f"case parts of the gradients {M} x {C} x {F} {dtype}", flush=True)
    x, w_in, w_out, dy = (t.to(DEV) for t in ffn_inputs(M, C, F, dtype, 50))
    full = ops.gated_ffn_backward(dy, x, w_in, w_out, dw_dtype=F32)
    assert all(torch.isfinite(t).all() and t.abs().max() > 0 for t in full)
    for want in itertools.product((False, True), repeat=3):
        got = ops.gated_ffn_backward(dy, x, w_in, w_out, need_dx=want[0], need_dw=want[1:], dw_dtype=F32)
        for g, f, w in zip(got, full, want):
            assert torch.equal(g, f) if w else g is None, want
    assert [t is not None for t in ops.gated_ffn_backward(dy, x, w_in, w_out, need_dw=False)] == [True, False, False]
