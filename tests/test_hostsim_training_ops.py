"""The training operators on the kernels' host build: their GPU tests (see test_hostsim_parity), walks over
the addresses of large shapes, and runs under other orders of the lanes."""

import pytest
import torch

import tests.test_training_ops_gpu as _mod
from kfold_amd import ops
from tests import hostsim
from tests.test_hostsim_address_walk import _untouched
from tests.test_hostsim_parity import _twin

# streams and graphs of a device; minutes of CPU time
SKIP = {"test_training_ops_streams_and_graphs", "test_training_ops_two_graphs", "test_gated_ffn_largest_tiles"}

for _attr, _fn in list(vars(_mod).items()):
    if _attr.startswith("test_") and callable(_fn) and _attr not in SKIP:
        globals()[f"test_host_training__{_attr[5:]}"] = _twin(_mod, _fn)

BF, F32 = torch.bfloat16, torch.float32

# offsets beyond 32 bits; every choice of tile; hidden widths at which one range of rows would do for the
# weight gradients (they take two)
FFN_WALKS = [(1_300_000, 128, 512, BF), (700_001, 256, 1024, BF), (16_385, 256, 16_544, BF), (16_384, 64, 32, BF),
             (70_001, 256, 32, BF), (250_000, 384, 1000, BF), (33_000, 136, 72, BF), (40_000, 8, 600, BF),
             (300_007, 64, 512, F32), (300, 16_384, 64, BF), (300, 64, 65_536, BF)]


@pytest.mark.parametrize("rows,C,F,dtype", FFN_WALKS)
def test_walk_gated_ffn(rows, C, F, dtype):
    hs = hostsim.load()
    with torch.no_grad(), hostsim.host_backend(block_stride=4099, block_edge=2, skip_math=True) as arena:
        hs.hostsim_set_fill(0)
        try:
            x, dy = _untouched(arena, (rows, C), dtype), _untouched(arena, (rows, C), dtype)
            w_in, w_out = _untouched(arena, (2 * F, C), dtype), _untouched(arena, (C, F), dtype)
            ops.gated_ffn_forward(x, w_in, w_out)
            ops.gated_ffn_backward(dy, x, w_in, w_out)
            ops.gated_ffn_backward(dy, x, w_in, w_out, need_dx=False, dw_dtype=F32)
        finally:
            hs.hostsim_set_fill(1)


@pytest.mark.parametrize("rows,C,dtype", [(20_000_003, 128, BF), (9_000_000, 256, F32), (3_000_001, 765, BF), (600_000, 5000, BF),
                                          (200_000_000, 8, F32)])
def test_walk_layer_norm(rows, C, dtype):
    hs = hostsim.load()
    with torch.no_grad(), hostsim.host_backend(block_stride=200_003, block_edge=2, skip_math=True) as arena:
        hs.hostsim_set_fill(0)
        try:
            x, dy = _untouched(arena, (rows, C), dtype), _untouched(arena, (rows, C), dtype)
            w = _untouched(arena, (C,), F32)
            ops.layer_norm_forward(x, w, w, stats=True)
            stat = _untouched(arena, (rows,), F32)
            ops.layer_norm_backward(dy, x, stat, stat, w, need_dparams=False)
        finally:
            hs.hostsim_set_fill(1)


@pytest.mark.parametrize("shape,shared", [((2_200_000_000,), None), ((3, 40_000, 20_000), 1), ((3, 40_000, 20_001), 1), ((2_200_000_003, 1), 0),
                                          ((1, 2_200_000_003), 1)])
def test_walk_dropout(shape, shared):
    hs = hostsim.load()
    with torch.no_grad(), hostsim.host_backend(block_stride=2_000_003, block_edge=2, skip_math=True) as arena:
        hs.hostsim_set_fill(0)
        try:
            x = _untouched(arena, shape, BF)
            ops.dropout_forward(x, 0.1, 3, shared_dim=shared, residual=x)
        finally:
            hs.hostsim_set_fill(1)


def _one_of_each():
    """Results of one call per kernel family on fixed inputs."""
    g = torch.Generator().manual_seed(77)
    r = []
    for dtype in (BF, F32):
        for rows, C in ((70, 128), (9, 765), (40, 2048), (5, 2500)):
            x, dy = _mod.rand(g, rows, C, dtype=dtype), _mod.rand(g, rows, C, dtype=dtype)
            y, mean, rstd = ops.layer_norm_forward(x, stats=True)
            r += [y, mean, rstd, *ops.layer_norm_backward(dy, x, mean, rstd)]
        for M, C, F in ((37, 64, 72), (600, 136, 64)):
            x, w_in, w_out, dy = _mod.ffn_inputs(M, C, F, dtype, 5)
            r += [ops.gated_ffn_forward(x, w_in, w_out), *ops.gated_ffn_backward(dy, x, w_in, w_out)]
    for M, C, F in ((33_000, 8, 16), (16_400, 128, 32), (16_390, 256, 32)):
        x, w_in, w_out, dy = _mod.ffn_inputs(M, C, F, BF, 6)
        r += [ops.gated_ffn_forward(x, w_in, w_out), *ops.gated_ffn_backward(dy, x, w_in, w_out)]
    x = _mod.rand(g, 4, 9, 24)
    r += [ops.dropout_forward(x, 0.3, 4), ops.dropout_forward(x, 0.3, 4, shared_dim=1), ops.dropout_forward(x[..., :5], 0.3, 4, shared_dim=1)]
    return [t.clone() for t in r]


def test_training_ops_under_other_lane_orders_and_poisoned_lds():
    """The order in which wavefronts reach their barriers changes nothing, and no kernel reads LDS that its
    own workgroup has not written."""
    hs = hostsim.load()
    with torch.no_grad(), hostsim.host_backend():
        want = _one_of_each()
    for schedule, poison in ((1, 0), (2, 0), (0, 1)):
        hs.hostsim_set_schedule(schedule)
        hs.hostsim_set_poison_lds(poison)
        try:
            with torch.no_grad(), hostsim.host_backend():
                got = _one_of_each()
        finally:
            hs.hostsim_set_schedule(0)
            hs.hostsim_set_poison_lds(0)
        assert all(torch.equal(p, q) for p, q in zip(got, want)), (schedule, poison)
