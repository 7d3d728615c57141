"""The training operators under autograd's and torch's other modes, on the kernels' host build (no GPU)."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from kfold_amd import functional, layers, ops, primitives
from tests import hostsim


def _rand(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_tangents_are_refused(grad):
    """A tangent on any argument raises, whether or not gradients are wanted; it is never dropped."""
    x, t = _rand(5, 64), _rand(5, 64, seed=1)
    w, tw = _rand(64, seed=2), _rand(64, seed=3)
    w_in, w_out = _rand(64, 64, seed=4, scale=0.1), _rand(64, 32, seed=5, scale=0.1)
    block = layers.Transition(64, 2).requires_grad_(False)
    with hostsim.host_backend(), fwad.dual_level(), torch.set_grad_enabled(grad):
        dx, dw = fwad.make_dual(x, t), fwad.make_dual(w, tw)
        dwi, dwo = fwad.make_dual(w_in, w_in), fwad.make_dual(w_out, w_out)
        calls = [lambda: functional.layer_norm(dx), lambda: functional.layer_norm(x, dw), lambda: functional.layer_norm(x, w, dw),
                 lambda: functional.gated_ffn(dx, w_in, w_out), lambda: functional.gated_ffn(x, dwi, w_out),
                 lambda: functional.gated_ffn(x, w_in, dwo), lambda: functional.dropout(dx, 0.3, 1),
                 lambda: functional.dropout(x, 0.3, 1, residual=dx), lambda: primitives.LayerNorm(64)(dx),
                 lambda: primitives.Dropout(0.3)(dx)]
        if grad:
            calls.append(lambda: block(dx))
        for k, call in enumerate(calls):
            with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward"):
                print(k, call())
        # without a tangent the same calls run; dropout that does nothing keeps the tangent
        assert functional.layer_norm(x, w, w).shape == functional.gated_ffn(x, w_in, w_out).shape == x.shape
        assert torch.equal(fwad.unpack_dual(primitives.Dropout(0.3).eval()(dx)).tangent, t)


def test_dropout_seed_comes_from_the_cpu_generator():
    """Under another default device too: there a drawn seed would belong to that device's generator, and
    reading it would wait for the device."""
    x = _rand(40, 64)
    drop = primitives.Dropout(0.3)
    with hostsim.host_backend():
        torch.manual_seed(1)
        want = drop(x)
        torch.manual_seed(1)
        with torch.device("meta"):
            got = drop(x)
        assert torch.equal(got, want)              # (the host build's memory ends with its context)


def test_frozen_weights_are_not_asked_for(monkeypatch):
    """The backward call computes the gradients that somebody wants, each weight by itself."""
    asked = []

    def backward(*args, _call=ops.gated_ffn_backward, **kwargs):
        got = _call(*args, **kwargs)
        asked.append(tuple(t is not None for t in got))
        return got
    monkeypatch.setattr(ops, "gated_ffn_backward", backward)
    args = (_rand(5, 64), _rand(64, 64, seed=4, scale=0.1), _rand(64, 32, seed=5, scale=0.1))
    with hostsim.host_backend(), torch.enable_grad():
        for k in range(1, 8):
            want = tuple(bool(k >> i & 1) for i in range(3))
            leaves = [t.clone().requires_grad_(w) for t, w in zip(args, want)]
            functional.gated_ffn(*leaves).sum().backward()
            assert asked.pop() == want
