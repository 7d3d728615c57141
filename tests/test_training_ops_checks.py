"""The training operators' C entry points refuse malformed requests with a status code and a message,
before anything is enqueued; their size queries.  No GPU: the pointers are never used."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="runs on GPU-less hosts only")

EINVAL, EUNSUPPORTED = -1, -2


@pytest.fixture(scope="module")
def env():
    from kfold_amd import _lib

    buf = ctypes.create_string_buffer(1 << 16)
    base = (ctypes.addressof(buf) + 4095) // 4096 * 4096
    return _lib.lib(), [base + 4096 * i for i in range(12)], buf


def _expect(lib, rc, code, *words):
    msg = lib.kfh_last_error().decode()
    assert rc == code, (rc, msg)
    for w in words:
        assert w in msg, msg


def test_layer_norm_checks(env):
    lib, p, _ = env
    f = lib.kfh_layer_norm_forward
    _expect(lib, f(p[0], None, None, p[1], None, None, -1, 128, 1e-5, 0, None), EINVAL, "rows=-1")
    _expect(lib, f(p[0], None, None, p[1], None, None, 4, 0, 1e-5, 0, None), EUNSUPPORTED, "C=0")
    _expect(lib, f(p[0], None, None, p[1], None, None, 4, 65537, 1e-5, 0, None), EUNSUPPORTED, "C=65537")
    _expect(lib, f(p[0], None, None, p[1], None, None, 1 << 30, 8, 1e-5, 0, None), EUNSUPPORTED, "rows=1073741824")
    _expect(lib, f(p[0], None, None, p[1], None, None, 4, 128, 1e-5, 2, None), EINVAL, "io_dtype 2")
    _expect(lib, f(None, None, None, p[1], None, None, 4, 128, 1e-5, 0, None), EINVAL, "null")
    _expect(lib, f(p[0], None, None, p[1], p[2], None, 4, 128, 1e-5, 0, None), EINVAL, "together")
    assert f(None, None, None, None, None, None, 0, 128, 1e-5, 0, None) == 0
    b = lib.kfh_layer_norm_backward
    need = lib.kfh_layer_norm_backward_workspace_bytes(100, 128)
    assert need > 0 and need % 256 == 0 and lib.kfh_layer_norm_backward_workspace_bytes(100, 0) == 0
    assert lib.kfh_layer_norm_backward_workspace_bytes(-1, 128) == 0
    ok = [p[0], p[1], p[2], p[3], None, p[4], p[5], p[6]]
    _expect(lib, b(*ok, p[7], need - 1, 100, 128, 0, None), EINVAL, "workspace", str(need))
    _expect(lib, b(*ok, None, need, 100, 128, 0, None), EINVAL, "workspace")
    _expect(lib, b(*ok, p[7] + 16, need, 100, 128, 0, None), EINVAL, "aligned")
    _expect(lib, b(p[0], p[1], None, p[3], None, p[4], None, None, None, 0, 100, 128, 0, None), EINVAL, "null")
    _expect(lib, b(p[0], p[1], p[2], p[3], None, p[1], None, None, None, 0, 100, 128, 0, None), EINVAL, "alias")
    _expect(lib, b(*ok, p[7], need, 100, 128, 5, None), EINVAL, "io_dtype 5")
    _expect(lib, b(*ok, p[7], need, -2, 128, 0, None), EINVAL, "rows=-2")


def test_gated_ffn_checks(env):
    lib, p, _ = env
    f, b, ws = lib.kfh_gated_ffn_forward, lib.kfh_gated_ffn_backward, lib.kfh_gated_ffn_workspace_bytes
    for C, F in ((12, 16), (16, 12), (0, 16), (16, 0), (32768, 16)):
        assert ws(10, C, F, 0, 0) == 0
        _expect(lib, f(p[0], p[1], p[2], p[3], p[4], 1 << 20, 10, C, F, 0, None), EUNSUPPORTED, f"C={C}", f"F={F}")
        _expect(lib, b(p[0], p[1], p[2], p[3], p[4], p[5], p[6], 0, p[7], 1 << 20, 10, C, F, 0, None), EUNSUPPORTED, f"C={C}")
    _expect(lib, f(p[0], p[1], p[2], p[3], p[4], 1 << 20, -1, 64, 64, 0, None), EINVAL, "rows=-1")
    _expect(lib, f(p[0], p[1], p[2], p[3], p[4], 1 << 20, 1 << 30, 64, 64, 0, None), EUNSUPPORTED, "rows=1073741824")
    _expect(lib, f(p[0], p[1], p[2], p[3], p[4], 1 << 20, 10, 64, 64, 3, None), EINVAL, "io_dtype 3")
    _expect(lib, f(p[0], None, p[2], p[3], p[4], 1 << 20, 10, 64, 64, 0, None), EINVAL, "null")
    _expect(lib, f(p[0] + 2, p[1], p[2], p[3], p[4], 1 << 20, 10, 64, 64, 0, None), EINVAL, "16 bytes")
    _expect(lib, f(p[0], p[1], p[2], p[0], p[4], 1 << 20, 10, 64, 64, 0, None), EINVAL, "alias")
    need = ws(10, 72, 64, 0, 1)
    _expect(lib, f(p[0], p[1], p[2], p[3], p[4], need - 1, 10, 72, 64, 1, None), EINVAL, "workspace", str(need))
    _expect(lib, f(p[0], p[1], p[2], p[3], None, need, 10, 72, 64, 1, None), EINVAL, "workspace")
    assert f(None, None, None, None, None, 0, 0, 64, 64, 0, None) == 0
    need = ws(10, 64, 64, 1, 0)
    ok = [p[0], p[1], p[2], p[3], p[4], p[5], p[6]]
    _expect(lib, b(*ok, 0, p[7], need - 1, 10, 64, 64, 0, None), EINVAL, "workspace", str(need))
    _expect(lib, b(*ok, 7, p[7], need, 10, 64, 64, 0, None), EINVAL, "dw_dtype 7")
    _expect(lib, b(p[0], p[1], p[2], p[3], p[1], p[5], p[6], 0, p[7], need, 10, 64, 64, 0, None), EINVAL, "alias")
    _expect(lib, b(p[0], p[1], p[2], p[3], p[0], p[5], p[6], 0, p[7], need, 10, 64, 64, 0, None), EINVAL, "alias")
    _expect(lib, b(p[0], p[1], p[2], p[3], p[4], p[5] + 8, p[6], 0, p[7], need, 10, 64, 64, 0, None), EINVAL, "16 bytes")
    _expect(lib, b(None, p[1], p[2], p[3], p[4], p[5], p[6], 0, p[7], need, 10, 64, 64, 0, None), EINVAL, "null")
    assert ws(589824, 128, 256, 1, 0) < 16 << 30


def test_dropout_checks(env):
    lib, p, _ = env
    f = lib.kfh_dropout
    _expect(lib, f(p[0], None, p[1], -1, 1, 8, 0.1, None, 0, 0, 0, None), EINVAL, "[-1, 1, 8]")
    for bad in (-0.1, 1.1, float("nan")):
        _expect(lib, f(p[0], None, p[1], 1, 1, 8, bad, None, 0, 0, 0, None), EINVAL, "probability")
    _expect(lib, f(p[0], None, p[1], 1, 1, 8, 0.1, None, 0, 0, 9, None), EINVAL, "io_dtype 9")
    _expect(lib, f(None, None, p[1], 1, 1, 8, 0.1, None, 0, 0, 0, None), EINVAL, "null")
    _expect(lib, f(p[0], None, p[1], 1 << 31, 1 << 31, 1 << 31, 0.1, None, 0, 0, 0, None), EUNSUPPORTED, "elements")
    assert f(None, None, None, 0, 5, 8, 0.1, None, 0, 0, 0, None) == 0


def test_cpu_tensors_are_refused():
    from kfold_amd import ops

    x, w = torch.zeros(4, 64), torch.zeros(128, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.layer_norm_forward(x)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.gated_ffn_forward(x, w, w.t().contiguous())
    with pytest.raises(RuntimeError, match="GPU"):
        ops.dropout_forward(x, 0.1, 0)
