"""Sums over rows (weight gradients of the gated feed-forward block, dgamma and dbeta of the layer norm)
to an accuracy at which one missing or doubled row shows.

A worst-case bound grows with the number of rows M, a sum of terms of either sign with sqrt(M), so at
many rows that bound cannot see a row.  Here the error of a whole result is held to the size its
roundings have together.  The roundings of different terms are independent, so the squared error,
summed over a result, is the sum of the squares of the single roundings (a sum over M rows and 10^2 to
10^5 values: it stays within some per cent of that, LIMIT leaves 15 % of the norm):
  - an operand rounded to bf16 (h, du, dv) is off by at most half a step of its binade, evenly between
    the ends: a third of the half step squared, times the other operand squared;
  - each of `adds` fp32 additions into a sum is off by at most U = 2^-24 of the partial sum, likewise:
    U^2 / 3 of its square, which is on average at most (sum of the squared terms) + (the sum)^2;
  - the terms themselves carry a few fp32 roundings (xh, the activation): TERM = 16 U of the term each, and
    for three-part products the dropped part products (2^-24 each) as much again, within TERM.
That the check sees a row is part of the test: against 64-bit sums without one row (the last, the middle
one, the one that adds least) or with row 0 twice, the same results fail it.
"""

import pytest
import torch

from kfold_amd import ops
from tests.test_training_ops_gpu import BF, F32, U, ffn64, ffn_inputs, rand

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
LIMIT, TERM = 1.15, 16 * U


def half_step(t):
    """Half the bf16 step at each value: 8 bits of mantissa, |t| = m 2^e with m in [1/2, 1)."""
    return torch.ldexp(torch.ones_like(t), torch.frexp(t).exponent - 9) * (t != 0)


def limit_of(rounded, sq_terms, total, adds):
    """rounded: the variance that rounded operands give each value; sq_terms: its squared terms' sum."""
    var = rounded + sq_terms * TERM ** 2 + U ** 2 / 3 * adds * (sq_terms + total ** 2)
    return LIMIT * var.sum().sqrt().item()


def check(got, want, limit, rows, what):
    """rows: f(r) = what row r adds to `want`; rows.norms: the norms of all of them."""
    got = got.detach().double().cpu()
    err = (got - want).norm().item()
    M, least = rows.norms.numel(), rows.norms.argmin().item()
    print(f"  {what}: error {err:.3e} limit {limit:.3e}; least row {rows.norms[least].item():.3e}", flush=True)
    assert err <= limit, (what, err, limit)
    for wrong in (want - rows(M - 1), want - rows(M // 2), want - rows(least), want + rows(0)):
        assert (got - wrong).norm().item() > limit, (what, "a missing row would pass", limit)


class Rows:
    """Row r adds a[r] (x) b[r] (b None: a[r] itself)."""

    def __init__(self, a, b=None):
        self.a, self.b = a, b
        self.norms = a.norm(dim=1) * (1 if b is None else b.norm(dim=1))

    def __call__(self, r):
        return self.a[r] if self.b is None else torch.outer(self.a[r], self.b[r])


# (rows kept in registers; 256 x 256, 256 x 128, 128 x 256, 128 x 128 and 64 x 64 tiles on row-major hidden values and on
# blocks of them; ragged last tiles and ranges of rows; fp32)
CASES = [(16_400, 64, 32, BF), (16_385, 64, 96, BF), (16_500, 128, 96, BF), (16_390, 256, 32, BF), (33_001, 24, 40, BF),
         (2500, 128, 256, BF), (4097, 72, 40, F32)]
LARGE = [(70_000, 256, 288, BF), (33_000, 136, 264, BF), (33_000, 264, 264, BF), (20_000, 264, 136, BF)]


def ffn_case(M, C, F, dtype):
    x, w_in, w_out, dy = ffn_inputs(M, C, F, dtype, 60)
    # rows of one size: no row adds much less than the others
    x, dy = ((t / t.double().norm(dim=1, keepdim=True) * C ** 0.5).to(dtype) for t in (x, dy))
    r = ffn64(x, w_in, w_out, dy)
    _, dwi, dwo = ops.gated_ffn_backward(dy.to(DEV), x.to(DEV), w_in.to(DEV), w_out.to(DEV), need_dx=False, dw_dtype=F32)
    d, x64, dy64 = torch.cat([r["du"], r["dv"]], 1), x.double(), dy.double()
    for got, name, a, b, hidden in ((dwi, "dw_in", d, x64, d), (dwo, "dw_out", dy64, r["h"], r["h"])):
        if dtype == BF:
            step = half_step(hidden).square() / 3
            rounded = (step if hidden is a else a.square()).t() @ (step if hidden is b else b.square())
        else:
            rounded = torch.zeros(())
        limit = limit_of(rounded, a.square().t() @ b.square(), r[name], M if dtype == BF else 6 * M)
        check(got, r[name], limit, Rows(a, b), name)


@pytest.mark.parametrize("M,C,F,dtype", CASES)
def test_weight_gradients_hold_every_row(M, C, F, dtype):
    print(f"case weight gradients hold every row {M} x {C} x {F} {dtype}", flush=True)
    ffn_case(M, C, F, dtype)


@pytest.mark.parametrize("M,C,F,dtype", LARGE)
def test_weight_gradients_hold_every_row_large(M, C, F, dtype):
    print(f"case weight gradients hold every row, large {M} x {C} x {F} {dtype}", flush=True)
    ffn_case(M, C, F, dtype)


@pytest.mark.parametrize("M,C,dtype", [(20_011, 128, BF), (20_011, 24, F32), (16_385, 765, F32), (9001, 768, BF), (5003, 2500, BF)])
def test_layer_norm_sums_hold_every_row(M, C, dtype):
    print(f"case layer norm sums hold every row {M} x {C} {dtype}", flush=True)
    g = torch.Generator().manual_seed(61)
    x, dy = rand(g, M, C, dtype=dtype), rand(g, M, C, dtype=dtype)
    _, mean, rstd = ops.layer_norm_forward(x.to(DEV), stats=True)
    _, dw, db = ops.layer_norm_backward(dy.to(DEV), x.to(DEV), mean, rstd, need_dx=False)
    xh = (x.double() - mean.double().cpu()[:, None]) * rstd.double().cpu()[:, None]
    dy64 = dy.double()
    t = dy64 * xh
    check(dw, t.sum(0), limit_of(0.0, t.square().sum(0), t.sum(0), M), Rows(t), "dweight")
    check(db, dy64.sum(0), limit_of(0.0, dy64.square().sum(0), dy64.sum(0), M), Rows(dy64), "dbias")
