"""Layer norm, gated feed-forward block and dropout, forward and backward, against the formulas in
64 bits.

Tolerances are worst-case bounds of the roundings a kernel makes, evaluated element by element from
the 64-bit intermediate values.  H is half a step of the output type (2^-8 of the value for bf16,
2^-24 for fp32), U = 2^-24 the half step of the fp32 arithmetic; a sum of K fp32 products in any order
is off by at most K * U * sum|terms| (to first order), written gamma(K) below.
"""

import math

import pytest
import torch

from kfold_amd import functional, layers, modules, ops, primitives, synthetic

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
BF, F32 = torch.bfloat16, torch.float32


def gamma(k):
    return (k + 8) * U


def within(got, want, tol, what):
    g, w = got.detach().double().cpu(), want.double()
    assert g.shape == w.shape, (what, g.shape, w.shape)
    assert torch.equal(torch.isfinite(g), torch.isfinite(w)), what
    d = torch.where(torch.isfinite(w), (g - w).abs(), torch.zeros_like(w))
    over = (d - tol).max().item() if d.numel() else 0.0
    worst = (d / (tol + 1e-300)).max().item() if d.numel() else 0.0
    print(f"  {what}: worst error / bound {worst:.3f}", flush=True)
    assert over <= 0, (what, over, worst)


def rand(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


# ---------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------
def ln64(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * rstd
    y = xh if w is None else xh * w.double()
    return (y if b is None else y + b.double()), mean, rstd, xh


def ln_forward_bound(x, w, b, y, mean, rstd, xh, dtype):
    """Row statistics: the mean is off by gamma(C) * mean|x| and each deviation by that and U * |x|; the
    relative error of rstd is half that of the variance, 2 * (deviation error * rstd) + gamma(C)."""
    C = x.shape[-1]
    ax = x.double().abs().mean(-1, keepdim=True)
    edev = gamma(C) * ax + U * x.double().abs().amax(-1, keepdim=True)
    rel = edev * rstd + gamma(C)
    wa = 1.0 if w is None else w.double().abs()
    exh = edev * rstd + xh.abs() * (2 * rel + 4 * U)
    ey = exh * wa + 4 * U * (xh.abs() * wa + (0 if b is None else b.double().abs()))
    return edev, rstd * (2 * rel + 4 * U), ey + HALF[dtype] * (y.abs() + ey)


LN_SHAPES = [(1, 1), (3, 2), (5, 7), (1, 128), (67, 128), (130, 64), (33, 96), (19, 256), (9, 384), (21, 765), (7, 768),
             (4, 1000), (3, 1024), (2, 2048), (2, 2049), (2, 5000), (300, 8), (70, 16), (41, 513), (11, 120)]


@pytest.mark.parametrize("rows,C", LN_SHAPES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_layer_norm_forward_and_backward(rows, C, dtype):
    print(f"case layer norm {rows} x {C} {dtype}", flush=True)
    g = torch.Generator().manual_seed(rows * 7919 + C)
    affine = (rows + C) % 3
    x = ((torch.randn(rows, C, generator=g) + 2.0) * (0.5 + torch.rand(rows, 1, generator=g))).to(dtype)
    w = None if affine == 0 else 1 + rand(g, C, scale=0.3)
    b = None if affine <= 1 else rand(g, C, scale=0.2)
    dy = rand(g, rows, C, dtype=dtype)
    eps = 1e-5
    y64, mean64, rstd64, xh = ln64(x, w, b, eps)
    dev = [None if t is None else t.to(DEV) for t in (x, w, b, dy)]
    y, mean, rstd = ops.layer_norm_forward(dev[0], dev[1], dev[2], eps, stats=True)
    em, er, ey = ln_forward_bound(x, w, b, y64, mean64, rstd64, xh, dtype)
    within(mean[:, None], mean64, em + U * mean64.abs(), "mean")
    within(rstd[:, None], rstd64, er, "rstd")
    within(y, y64, ey, "y")
    y2 = ops.layer_norm_forward(dev[0], dev[1], dev[2], eps)
    assert torch.equal(y2, y)
    # backward, with the statistics as computed (their error is part of the forward bound)
    m, r = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    xh = (x.double() - m) * r
    a = dy.double() * (1.0 if w is None else w.double())
    s1, s2 = a.mean(-1, keepdim=True), (a * xh).mean(-1, keepdim=True)
    dx64 = r * (a - s1 - xh * s2)
    exh = 4 * U * (x.double().abs() + m.abs()) * r
    e1 = gamma(C) * a.abs().mean(-1, keepdim=True)
    e2 = gamma(C) * (a * xh).abs().mean(-1, keepdim=True) + (a.abs() * exh).mean(-1, keepdim=True)
    edx = r * (e1 + xh.abs() * e2 + exh * s2.abs() + 8 * U * (a.abs() + s1.abs() + (xh * s2).abs()))
    dx, dw, db = ops.layer_norm_backward(dev[3], dev[0], mean, rstd, dev[1])
    within(dx, dx64, edx + HALF[dtype] * (dx64.abs() + edx), "dx")
    t = dy.double() * xh
    within(dw, t.sum(0), gamma(rows) * t.abs().sum(0) + (dy.double().abs() * exh).sum(0), "dweight")
    within(db, dy.double().sum(0), gamma(rows) * dy.double().abs().sum(0), "dbias")
    # the same call gives the same bits, in place on dy too; parts can be left out
    inplace = dev[3].clone()
    dx2, dw2, db2 = ops.layer_norm_backward(inplace, dev[0], mean, rstd, dev[1], out=inplace)
    assert torch.equal(dx2, dx) and torch.equal(dw2, dw) and torch.equal(db2, db)
    dx3, dw3, db3 = ops.layer_norm_backward(dev[3], dev[0], mean, rstd, dev[1], need_dparams=False)
    assert dw3 is None and db3 is None and torch.equal(dx3, dx)
    dx4, dw4, db4 = ops.layer_norm_backward(dev[3], dev[0], mean, rstd, dev[1], need_dx=False)
    assert dx4 is None and torch.equal(dw4, dw) and torch.equal(db4, db)
    xi = dev[0].clone()
    assert torch.equal(ops.layer_norm_forward(xi, dev[1], dev[2], eps, out=xi), y)


def test_layer_norm_many_rows_sum_in_order():
    """More rows than one round of workgroups takes: the sums over rows stay within the bound of a sum
    in any order, and repeat bit for bit."""
    print("case layer norm, 20011 rows", flush=True)
    g = torch.Generator().manual_seed(3)
    for C, dtype in ((128, BF), (24, F32)):
        rows = 20011
        x, dy = rand(g, rows, C, dtype=dtype), rand(g, rows, C, dtype=dtype)
        xd, dyd = x.to(DEV), dy.to(DEV)
        _, mean, rstd = ops.layer_norm_forward(xd, stats=True)
        dx, dw, db = ops.layer_norm_backward(dyd, xd, mean, rstd)
        xh = (x.double() - mean.double().cpu()[:, None]) * rstd.double().cpu()[:, None]
        t = dy.double() * xh
        exh = 4 * U * (x.double().abs() + mean.double().cpu().abs()[:, None]) * rstd.double().cpu()[:, None]
        within(dw, t.sum(0), gamma(rows) * t.abs().sum(0) + (dy.double().abs() * exh).sum(0), "dweight")
        within(db, dy.double().sum(0), gamma(rows) * dy.double().abs().sum(0), "dbias")
        again = ops.layer_norm_backward(dyd, xd, mean, rstd)
        assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db)))


@pytest.mark.parametrize("C", [128, 384, 77])
def test_layer_norm_hard_rows(C):
    """A constant row, rows far from zero, rows of huge and tiny values, and rows with inf and NaN, which
    leave the other rows alone."""
    print(f"case layer norm hard rows C={C}", flush=True)
    g = torch.Generator().manual_seed(C)
    x = rand(g, 12, C)
    x[1] = 3.25
    x[2] += 1e4
    x[3] *= 1e15
    x[4] *= 1e-12
    x[5, C // 2] = float("inf")
    x[6, 0] = float("nan")
    x[7] = 0.0
    y, mean, rstd = ops.layer_norm_forward(x.to(DEV), stats=True)
    keep = [i for i in range(12) if i not in (5, 6)]
    y64, mean64, rstd64, xh = ln64(x, None, None, 1e-5)
    em, er, ey = ln_forward_bound(x, None, None, y64, mean64, rstd64, xh, F32)
    within(y.cpu()[keep], y64[keep], ey[keep], "finite rows")
    assert torch.isnan(y[5]).all().item() and torch.isnan(y[6]).all().item()
    assert (y[1] == 0).all().item() and (y[7] == 0).all().item()


def test_layer_norm_strided_views_and_offsets():
    """Transposed, sliced and offset views give the bits of their contiguous copies; an output of the
    caller's is written."""
    print("case layer norm views", flush=True)
    g = torch.Generator().manual_seed(8)
    base = rand(g, 6, 9, 128, dtype=BF).to(DEV)
    flat = rand(g, 1 + 33 * 128, dtype=BF).to(DEV)
    for v in (base.transpose(0, 1), base[:, ::2], base[:, :, 8:72], base[..., 1:], flat[1:].view(33, 128)):
        c = v.contiguous().clone()
        y, mean, rstd = ops.layer_norm_forward(v, stats=True)
        yc, mc, rc = ops.layer_norm_forward(c, stats=True)
        # a row may go through another kernel where it does not start at a 16-byte boundary: rounding
        assert ((y.float() - yc.float()).abs() <= 2 ** -7 * yc.float().abs() + 1e-6).all()
        out = torch.empty_like(c)
        assert ops.layer_norm_forward(v, out=out) is out and torch.equal(out, y)
        dx, dw, db = ops.layer_norm_backward(v, v, mean, rstd)
        dxc, dwc, dbc = ops.layer_norm_backward(c, c, mc, rc)
        assert ((dx.float() - dxc.float()).abs() <= 2 ** -7 * dxc.float().abs() + 1e-5).all()
        assert (dw - dwc).abs().max() <= 1e-4 * dwc.abs().max() and torch.allclose(db, dbc, rtol=1e-5, atol=1e-4)


# ---------------------------------------------------------------------------------------------
# gated feed-forward block
# ---------------------------------------------------------------------------------------------
def ffn64(x, w_in, w_out, dy=None):
    x, w_in, w_out = x.double(), w_in.double(), w_out.double()
    F = w_out.shape[1]
    u, v = (x @ w_in.t()).split(F, dim=1)
    s = torch.sigmoid(u)
    h = u * s * v
    r = {"u": u, "v": v, "s": s, "h": h, "y": h @ w_out.t()}
    if dy is not None:
        dy = dy.double()
        dh = dy @ w_out
        du, dv = dh * v * s * (1 + u * (1 - s)), dh * u * s
        r.update(dh=dh, du=du, dv=dv, dx=torch.cat([du, dv], 1) @ w_in, dw_in=torch.cat([du, dv], 1).t() @ x,
                 dw_out=dy.t() @ h)
    return r


def ffn_bounds(x, w_in, w_out, r, dtype, dy=None, dw_dtype=None):
    """x, weights and dy are exact inputs.  u, v and dh are fp32 sums of products (six part products per
    term in fp32 arithmetic), the hidden values and their gradients are formed in fp32 with an exp2 and a
    reciprocal of a few U, and rounded to the type before the next product."""
    F, C = w_out.shape[1], w_out.shape[0]
    M = x.shape[0]
    mult = 6 if dtype == F32 else 1
    ax, awi, awo = x.double().abs(), w_in.double().abs(), w_out.double().abs()
    eu, ev = (gamma(mult * C) * (ax @ awi.t())).split(F, dim=1)
    u, v, s, h = r["u"].abs(), r["v"].abs(), r["s"], r["h"].abs()
    es = s * (1 - s) * eu + (16 + 2 * u) * U * s                  # sigmoid: slope, and its own evaluation
    ds = s * (1 + u * (1 - s))                                    # bounds |d silu / du|
    ehid = ds * v * eu + u * v * es + u * s * ev + 8 * U * h
    rnd = HALF[dtype]
    eh = ehid + rnd * (h + ehid)
    ey = eh @ awo.t() + gamma(mult * F) * (h @ awo.t())
    out = {"y": ey + rnd * (r["y"].abs() + ey)}
    if dy is None:
        return out
    ady = dy.double().abs()
    dh, du, dv = r["dh"].abs(), r["du"].abs(), r["dv"].abs()
    edh = gamma(mult * C) * (ady @ awo)
    eus = u * es + s * eu
    edv = dh * eus + u * s * edh + 8 * U * dv
    # du = dh v (s + u s (1 - s)): both terms to first order
    edu = (v * edh + dh * ev) * ds + dh * v * (es * (1 + 2 * u) + eus) + 16 * U * dh * v * ds
    edv, edu = edv + rnd * (dv + edv), edu + rnd * (du + edu)
    ed, d = torch.cat([edu, edv], 1), torch.cat([du, dv], 1)
    edx = ed @ awi + gamma(mult * 2 * F) * (d @ awi)
    edwi = ed.t() @ ax + gamma(mult * M) * (d.t() @ ax)
    edwo = ady.t() @ eh + gamma(mult * M) * (ady.t() @ h)
    rw = HALF[dw_dtype or dtype]
    out["dx"] = edx + rnd * (r["dx"].abs() + edx)
    out["dw_in"] = edwi + rw * (r["dw_in"].abs() + edwi)
    out["dw_out"] = edwo + rw * (r["dw_out"].abs() + edwo)
    return out


def ffn_inputs(M, C, F, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (rand(g, M, C, dtype=dtype), rand(g, 2 * F, C, dtype=dtype, scale=C ** -0.5),
            rand(g, C, F, dtype=dtype, scale=F ** -0.5), rand(g, M, C, dtype=dtype))


FFN_SHAPES = [(1, 8, 8), (1, 384, 768), (37, 384, 384), (63, 64, 72), (64, 128, 256), (65, 128, 256), (129, 128, 512),
              (200, 256, 512), (31, 136, 200), (300, 32, 64), (70, 40, 1000), (257, 256, 256), (96, 128, 128)]


@pytest.mark.parametrize("M,C,F", FFN_SHAPES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_gated_ffn_forward_and_backward(M, C, F, dtype):
    print(f"case gated ffn {M} x {C} x {F} {dtype}", flush=True)
    x, w_in, w_out, dy = ffn_inputs(M, C, F, dtype, M * 31 + C + F)
    r = ffn64(x, w_in, w_out, dy)
    e = ffn_bounds(x, w_in, w_out, r, dtype, dy)
    xd, wi, wo, dyd = (t.to(DEV) for t in (x, w_in, w_out, dy))
    y = ops.gated_ffn_forward(xd, wi, wo)
    within(y, r["y"], e["y"], "y")
    dx, dwi, dwo = ops.gated_ffn_backward(dyd, xd, wi, wo)
    within(dx, r["dx"], e["dx"], "dx")
    within(dwi, r["dw_in"], e["dw_in"], "dw_in")
    within(dwo, r["dw_out"], e["dw_out"], "dw_out")
    again = ops.gated_ffn_backward(dyd, xd, wi, wo)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dwi, dwo)))
    only = ops.gated_ffn_backward(dyd, xd, wi, wo, need_dw=False)
    assert torch.equal(only[0], dx) and only[1] is None and only[2] is None
    only = ops.gated_ffn_backward(dyd, xd, wi, wo, need_dx=False)
    assert only[0] is None and torch.equal(only[1], dwi) and torch.equal(only[2], dwo)


@pytest.mark.parametrize("M,C,F", [(33001, 24, 40), (32900, 8, 136), (16400, 64, 32), (16385, 64, 96), (16500, 128, 64),
                                   (16500, 128, 96), (16384, 256, 160), (16400, 256, 32)])
def test_gated_ffn_big_tiles(M, C, F):
    """Enough rows for every kernel to take its large tiles, or for the kernels that keep the rows in
    registers (C = 64, 128, 256), with ragged edges on all sides."""
    print(f"case gated ffn big tiles {M} x {C} x {F}", flush=True)
    x, w_in, w_out, dy = ffn_inputs(M, C, F, BF, 6)
    r = ffn64(x, w_in, w_out, dy)
    e = ffn_bounds(x, w_in, w_out, r, BF, dy)
    xd, wi, wo, dyd = (t.to(DEV) for t in (x, w_in, w_out, dy))
    within(ops.gated_ffn_forward(xd, wi, wo), r["y"], e["y"], "y")
    for got, name in zip(ops.gated_ffn_backward(dyd, xd, wi, wo), ("dx", "dw_in", "dw_out")):
        within(got, r[name], e[name], name)


@pytest.mark.parametrize("C", [5, 40, 72, 264, 765, 768, 1544])
def test_layer_norm_infinite_weight(C):
    """An infinite weight of the last channel: dx is infinite and NaN exactly where the formula is (a lane
    without channels of its own adds nothing)."""
    print(f"case layer norm infinite weight {C}", flush=True)
    g = torch.Generator().manual_seed(C)
    for dtype in (BF, F32):
        x, dy = rand(g, 7, C, dtype=dtype), rand(g, 7, C, dtype=dtype)
        w = torch.ones(C)
        w[-1] = float("inf")
        _, mean, rstd = ops.layer_norm_forward(x.to(DEV), w.to(DEV), stats=True)
        dx = ops.layer_norm_backward(dy.to(DEV), x.to(DEV), mean, rstd, w.to(DEV))[0].cpu().double()
        xd = x.double()
        xh = (xd - xd.mean(-1, keepdim=True)) / (xd.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
        a = dy.double() * w.double()
        want = a - a.mean(-1, keepdim=True) - xh * (a * xh).mean(-1, keepdim=True)
        assert torch.equal(torch.isnan(dx), torch.isnan(want)) and torch.equal(torch.isinf(dx), torch.isinf(want))
        assert torch.isinf(want).any()


@pytest.mark.parametrize("M,C,F", [(33_000, 136, 264), (33_000, 264, 264), (20_000, 264, 136), (70_000, 256, 288)])
def test_gated_ffn_largest_tiles(M, C, F):
    """The 256 x 256, 256 x 128 and 128 x 128 tiles on row-major hidden values and on blocks of them."""
    print(f"case gated ffn largest tiles {M} x {C} x {F}", flush=True)
    test_gated_ffn_big_tiles(M, C, F)


def test_gated_ffn_bad_rows_among_many():
    """As test_gated_ffn_saturated_and_bad_rows, for the kernels that keep the rows in registers."""
    print("case gated ffn bad rows among many", flush=True)
    for C, F in ((64, 32), (128, 32), (256, 32)):
        M = 16_390
        x, w_in, w_out, dy = (t.to(DEV) for t in ffn_inputs(M, C, F, BF, 13))
        y, dx = ops.gated_ffn_forward(x, w_in, w_out), ops.gated_ffn_backward(dy, x, w_in, w_out)[0]
        bad = x.clone()
        rows = (7, 4099, M - 1)
        for r in rows:
            bad[r, r % C] = float("nan")
        yb = ops.gated_ffn_forward(bad, w_in, w_out)
        dxb = ops.gated_ffn_backward(dy, bad, w_in, w_out)[0]
        for r in rows:
            assert torch.isnan(yb[r]).all() and torch.isnan(dxb[r]).all()
            yb[r], dxb[r] = y[r], dx[r]
        assert torch.equal(yb, y) and torch.equal(dxb, dx)


def test_gated_ffn_many_rows():
    """Rows beyond one range of the weight gradients' sums, a ragged end, gradients kept in fp32."""
    print("case gated ffn 2500 rows", flush=True)
    M, C, F = 2500, 128, 256
    x, w_in, w_out, dy = ffn_inputs(M, C, F, BF, 5)
    r = ffn64(x, w_in, w_out, dy)
    e = ffn_bounds(x, w_in, w_out, r, BF, dy, dw_dtype=F32)
    xd, wi, wo, dyd = (t.to(DEV) for t in (x, w_in, w_out, dy))
    within(ops.gated_ffn_forward(xd, wi, wo), r["y"], e["y"], "y")
    dx, dwi, dwo = ops.gated_ffn_backward(dyd, xd, wi, wo, dw_dtype=F32)
    assert dwi.dtype == F32 and dwo.dtype == F32
    for got, name in ((dx, "dx"), (dwi, "dw_in"), (dwo, "dw_out")):
        within(got, r[name], e[name], name)
    # a shorter call on the same rows may go through another kernel, which adds in another order: both are
    # within the bound e of the exact y, so |a - b| <= |a - y| + |b - y| <= 2 e
    part = ops.gated_ffn_forward(xd[:900], wi, wo)
    within(part, ops.gated_ffn_forward(xd, wi, wo)[:900].cpu(), 2 * e["y"][:900], "y of the first 900 rows")


def test_gated_ffn_leaves_what_is_not_its_own():
    """Memory behind the last row of every result stays as it was; a caller's workspace full of NaN
    changes nothing."""
    print("case gated ffn guards", flush=True)
    for dtype in (BF, F32):
        M, C, F = 45, 128, 256
        x, w_in, w_out, dy = (t.to(DEV) for t in ffn_inputs(M, C, F, dtype, 9))
        want = ops.gated_ffn_forward(x, w_in, w_out)
        big = torch.full((M + 40, C), 7.0, dtype=dtype, device=DEV if DEV != "cpu" else None)
        ops.gated_ffn_forward(x, w_in, w_out, out=big[:M])
        assert torch.equal(big[:M], want) and (big[M:] == 7).all()
        dx, dwi, dwo = ops.gated_ffn_backward(dy, x, w_in, w_out)
        need = ops.workspace_bytes("gated_ffn", rows=M, C=C, F=F, backward=True, dtype=dtype)
        ws = torch.full((need + 512,), 255, dtype=torch.uint8, device=DEV if DEV != "cpu" else None)
        ws = ws[(-ws.data_ptr()) % 256:][:need]
        big = torch.full((M + 40, C), 7.0, dtype=dtype, device=DEV if DEV != "cpu" else None)
        got = ops.gated_ffn_backward(dy, x, w_in, w_out, out=big[:M], workspace=ws)
        assert all(torch.equal(p, q) for p, q in zip(got, (dx, dwi, dwo))) and (big[M:] == 7).all()


def test_gated_ffn_saturated_and_bad_rows():
    """Gates far out on both sides stay finite; a row of NaN or inf spoils itself and the weight
    gradients, not the other rows."""
    print("case gated ffn saturation", flush=True)
    x, w_in, w_out, dy = ffn_inputs(40, 64, 64, F32, 11)
    w_in = w_in * 40
    r = ffn64(x, w_in, w_out, dy)
    e = ffn_bounds(x, w_in, w_out, r, F32, dy)
    xd, wi, wo, dyd = (t.to(DEV) for t in (x, w_in, w_out, dy))
    within(ops.gated_ffn_forward(xd, wi, wo), r["y"], e["y"], "y")
    for got, name in zip(ops.gated_ffn_backward(dyd, xd, wi, wo), ("dx", "dw_in", "dw_out")):
        within(got, r[name], e[name], name)
    for dtype in (BF, F32):
        x, w_in, w_out, dy = (t.to(DEV) for t in ffn_inputs(40, 64, 64, dtype, 12))
        y, dx = ops.gated_ffn_forward(x, w_in, w_out), ops.gated_ffn_backward(dy, x, w_in, w_out)[0]
        bad = x.clone()
        bad[7, 3] = float("nan")
        bad[9, 0] = float("inf")
        yb = ops.gated_ffn_forward(bad, w_in, w_out)
        dxb = ops.gated_ffn_backward(dy, bad, w_in, w_out)[0]
        keep = [i for i in range(40) if i not in (7, 9)]
        assert torch.equal(yb[keep], y[keep]) and torch.equal(dxb[keep], dx[keep])
        assert not torch.isfinite(yb[7]).any() and not torch.isfinite(yb[9]).all()


def test_gated_ffn_views():
    print("case gated ffn views", flush=True)
    g = torch.Generator().manual_seed(2)
    for dtype in (BF, F32):
        base = rand(g, 6, 7, 64, dtype=dtype).to(DEV)
        w_in, w_out = rand(g, 64, 128, dtype=dtype, scale=0.1).to(DEV), rand(g, 64, 64, dtype=dtype, scale=0.1).to(DEV)
        odd = rand(g, 1 + 13 * 64, dtype=dtype).to(DEV)[1:].view(13, 64)
        for v in (base.transpose(0, 1), base[:, ::3], odd):
            c = v.contiguous().clone()
            wt = w_in.t()                                           # [128, 64], transposed in memory
            wc = wt.contiguous()
            assert torch.equal(ops.gated_ffn_forward(v, wt, w_out), ops.gated_ffn_forward(c, wc, w_out))
            for p, q in zip(ops.gated_ffn_backward(v, v, wt, w_out), ops.gated_ffn_backward(c, c, wc, w_out)):
                assert torch.equal(p, q)


# ---------------------------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------------------------
M32 = 0xFFFFFFFF


def philox(counter, offset, seed):
    """Philox4x32-10 of the 2011 paper on Python integers."""
    c = [counter & M32, counter >> 32 & M32, offset & M32, offset >> 32 & M32]
    k = [seed & M32, seed >> 32 & M32]
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & M32, (a >> 32) ^ c[3] ^ k[1], a & M32]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return c


def keep_mask(shape, p, seed, offset, shared_dim):
    s = list(shape)
    if shared_dim is not None:
        s[shared_dim] = 1
    n = math.prod(s)
    t = math.floor(p * 65536 + 0.5)
    bits = []
    for g in range((n + 7) // 8):
        for w in philox(g, offset & (2 ** 64 - 1), seed & (2 ** 64 - 1)):
            bits += [w & 0xFFFF, w >> 16]
    return (torch.tensor(bits[:n]) >= t).view(s), t


def drop_ref(x, p, seed, offset, shared_dim, residual):
    keep, t = keep_mask(x.shape, p, seed, offset, shared_dim)
    scale = torch.tensor(65536 / (65536 - t) if t < 65536 else 0.0, dtype=F32)
    y = torch.where(keep, x.float() * scale, torch.zeros(()))
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype), keep


def test_dropout_known_answers():
    """Words of the generator for the zero counter and key, as its paper's implementation publishes."""
    assert philox(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


DROP_CASES = [((1,), None), ((7,), None), ((8,), 0), ((3, 5), 0), ((3, 5), 1), ((2, 9, 11), 1), ((2, 9, 16), 1), ((2, 9, 16), 0),
              ((2, 9, 16), 2), ((1, 6, 7, 32), 1), ((2, 6, 7, 32), 2), ((2, 4, 5, 24), None), ((2, 4, 5, 13), 2), ((260, 33), None),
              ((70, 128), None), ((1, 40, 3, 64), 1), ((1, 3, 40, 64), 2), ((5, 1, 128), 1)]


@pytest.mark.parametrize("shape,shared", DROP_CASES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_dropout_values(shape, shared, dtype):
    """Bit for bit: the products and sums are single fp32 operations, rounded once (the compiler may
    contract them into one fused operation, which then differs by at most half a step)."""
    print(f"case dropout {shape} shared={shared} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape))
    x, res = rand(g, *shape, dtype=dtype), rand(g, *shape, dtype=dtype)
    for p, seed, offset in ((0.1, 1234567890123456789, 0), (0.5, -1, 2 ** 40 + 3), (0.0, 5, 1), (1.0, 5, 1), (0.3, 77, 9)):
        want, keep = drop_ref(x, p, seed, offset, shared, None)
        got = ops.dropout_forward(x.to(DEV), p, seed, offset, shared)
        assert torch.equal(got.cpu(), want), (p, seed)
        assert torch.equal(ops.dropout_backward(x.to(DEV), p, seed, offset, shared).cpu(), want)
        want, _ = drop_ref(x, p, seed, offset, shared, res)
        got = ops.dropout_forward(x.to(DEV), p, seed, offset, shared, residual=res.to(DEV))
        scale = 1.0 if p == 1.0 else 1 / (1 - p)
        tol = 2 * HALF[dtype] * want.double().abs() + 2 * U * (scale * 1.001 * x.double().abs() + res.double().abs())
        within(got, want, tol, f"p={p} with residual")
        both = res.to(DEV)
        assert torch.equal(ops.dropout_forward(x.to(DEV), p, seed, offset, shared, residual=both, out=both), got)
        xi = x.to(DEV)
        alone = ops.dropout_forward(xi, p, seed, offset, shared)
        assert torch.equal(ops.dropout_forward(xi, p, seed, offset, shared, out=xi), alone)


def test_dropout_dropped_values_are_never_used():
    print("case dropout inf / nan", flush=True)
    x = torch.full((64, 24), float("nan"))
    x[::2] = float("inf")
    for dtype in (BF, F32):
        keep, _ = keep_mask(x.shape, 0.4, 3, 0, None)
        y = ops.dropout_forward(x.to(dtype).to(DEV), 0.4, 3).cpu()
        assert (y[~keep] == 0).all() and not torch.isfinite(y[keep].float()).any()
        res = torch.ones(64, 24, dtype=dtype)
        y = ops.dropout_forward(x.to(dtype).to(DEV), 0.4, 3, residual=res.to(DEV)).cpu()
        assert (y[~keep] == 1).all()


def test_dropout_seeds_offsets_and_device_seed():
    print("case dropout seeds", flush=True)
    x = torch.ones(1000, 16).to(DEV)
    base = ops.dropout_forward(x, 0.25, 11)
    assert torch.equal(base, ops.dropout_forward(x, 0.25, 11))
    n = x.numel()
    for other in (ops.dropout_forward(x, 0.25, 12), ops.dropout_forward(x, 0.25, 11, 1), ops.dropout_forward(x, 0.25, 11 + 2 ** 32)):
        # independent masks agree with probability 0.625: 16000 draws, six standard deviations
        same = ((other == 0) == (base == 0)).float().mean().item()
        assert abs(same - 0.625) < 6 * math.sqrt(0.625 * 0.375 / n)
    kept = (base != 0).float().mean().item()
    assert abs(kept - 0.75) < 6 * math.sqrt(0.75 * 0.25 / n)
    seed = torch.tensor([11]).to(DEV)
    assert torch.equal(ops.dropout_forward(x, 0.25, seed), base)
    big = torch.tensor(-5).to(DEV)
    assert torch.equal(ops.dropout_forward(x, 0.25, big), ops.dropout_forward(x, 0.25, -5))


def test_dropout_views_and_guards():
    print("case dropout views", flush=True)
    g = torch.Generator().manual_seed(4)
    flat = rand(g, 3 + 40 * 16, dtype=BF)
    for v in (flat[3:].view(40, 16), flat[:640].view(40, 16).t(), flat[:640].view(40, 16)[::2], flat[1:601].view(1, 20, 30)):
        for sd in (None, 0):
            want, _ = drop_ref(v.contiguous(), 0.2, 9, 4, sd, None)
            assert torch.equal(ops.dropout_forward(v.to(DEV) if DEV != "cpu" else v, 0.2, 9, 4, sd).cpu(), want)
    big = torch.full((600,), 7.0, device=DEV if DEV != "cpu" else None)
    x = torch.ones(589).to(DEV)
    ops.dropout_forward(x, 0.5, 1, out=big[:589])
    assert (big[589:] == 7).all() and ((big[:589] == 0) | (big[:589] == 2)).all()
    big = torch.full((600,), 7.0, device=DEV if DEV != "cpu" else None)
    ops.dropout_forward(x, 0.5, 1, out=big[3:592])                   # an output off its 16-byte boundary
    assert (big[:3] == 7).all() and (big[592:] == 7).all() and torch.equal(big[3:592], ops.dropout_forward(x, 0.5, 1))


# ---------------------------------------------------------------------------------------------
# empty inputs and refusals
# ---------------------------------------------------------------------------------------------
def test_training_ops_empty_inputs():
    print("case training ops, no rows", flush=True)
    for dtype in (BF, F32):
        x = torch.empty(0, 5, 64, dtype=dtype).to(DEV)
        y, mean, rstd = ops.layer_norm_forward(x, stats=True)
        assert y.shape == x.shape and mean.shape == (0, 5)
        dx, dw, db = ops.layer_norm_backward(x, x, mean, rstd)
        assert dx.shape == x.shape and (dw == 0).all() and (db == 0).all() and dw.shape == (64,)
        w_in, w_out = torch.ones(16, 64, dtype=dtype).to(DEV), torch.ones(64, 8, dtype=dtype).to(DEV)
        assert ops.gated_ffn_forward(x, w_in, w_out).shape == x.shape
        dx, dwi, dwo = ops.gated_ffn_backward(x, x, w_in, w_out)
        assert dx.shape == x.shape and dwi.shape == (16, 64) and (dwi == 0).all() and (dwo == 0).all()
        assert ops.dropout_forward(x, 0.1, 1, shared_dim=1).shape == x.shape
        assert ops.dropout_forward(torch.empty(3, 0, 4, dtype=dtype).to(DEV), 0.1, 1, shared_dim=1).numel() == 0


def test_training_ops_refusals():
    x = torch.zeros(4, 64).to(DEV)
    with pytest.raises(TypeError):
        ops.layer_norm_forward(x.half())
    with pytest.raises(ValueError):
        ops.layer_norm_forward(torch.zeros(4, 0).to(DEV))
    with pytest.raises(ValueError):
        ops.layer_norm_forward(torch.zeros(()).to(DEV))
    with pytest.raises(ValueError, match="weight"):
        ops.layer_norm_forward(x, torch.ones(63).to(DEV))
    with pytest.raises(ValueError, match="out"):
        ops.layer_norm_forward(x, out=torch.zeros(4, 64, dtype=BF).to(DEV))
    _, mean, rstd = ops.layer_norm_forward(x, stats=True)
    with pytest.raises(ValueError, match="dy"):
        ops.layer_norm_backward(x.bfloat16(), x, mean, rstd)
    with pytest.raises(ValueError, match="rstd"):
        ops.layer_norm_backward(x, x, mean, rstd[:3])
    with pytest.raises(Exception, match="alias"):
        ops.layer_norm_backward(x.clone(), x, mean, rstd, out=x)
    w_in, w_out = torch.zeros(32, 64).to(DEV), torch.zeros(64, 16).to(DEV)
    with pytest.raises(ValueError, match="w_in"):
        ops.gated_ffn_forward(x, w_out, w_in)
    with pytest.raises(TypeError, match="one dtype"):
        ops.gated_ffn_forward(x, w_in.bfloat16(), w_out)
    with pytest.raises(NotImplementedError, match="C=12"):
        ops.gated_ffn_forward(torch.zeros(4, 12).to(DEV), torch.zeros(16, 12).to(DEV), torch.zeros(12, 8).to(DEV))
    with pytest.raises(ValueError, match="dy"):
        ops.gated_ffn_backward(x[:3], x, w_in, w_out)
    with pytest.raises(TypeError, match="dw_dtype"):
        ops.gated_ffn_backward(x, x, w_in, w_out, dw_dtype=torch.float16)
    with pytest.raises(Exception, match="alias"):
        ops.gated_ffn_backward(x.clone(), x, w_in, w_out, out=x)
    with pytest.raises(Exception, match="alias"):
        dy = x.clone()
        ops.gated_ffn_backward(dy, x, w_in, w_out, out=dy)
    with pytest.raises(ValueError, match="probability"):
        ops.dropout_forward(x, 1.5, 0)
    with pytest.raises(ValueError, match="probability"):
        ops.dropout_forward(x, float("nan"), 0)
    with pytest.raises(ValueError, match="dimension"):
        ops.dropout_forward(x, 0.1, 0, shared_dim=2)
    with pytest.raises(ValueError, match="int64"):
        ops.dropout_forward(x, 0.1, torch.zeros(1, dtype=torch.int32).to(DEV))
    with pytest.raises(ValueError, match="residual"):
        ops.dropout_forward(x, 0.1, 0, residual=x[:2])
    with pytest.raises(ValueError, match="probability"):
        primitives.Dropout(-0.1)


# ---------------------------------------------------------------------------------------------
# gradients through autograd
# ---------------------------------------------------------------------------------------------
def test_functional_gradients_against_differences():
    """Directional derivatives of the whole step z + dropout(ffn(layer_norm(z))) in fp32 arithmetic:
    central differences of step e are off by e^2 / 6 of the third derivative and by the forward's
    rounding / e; with |z| = O(1), e = 2^-6 and forward errors of about 2^-20 of sums of n terms both
    stay under 2^-9 of |gradient| |direction|."""
    print("case differences", flush=True)
    g = torch.Generator().manual_seed(21)
    M, C, F = 24, 64, 128
    t = {"z": rand(g, M, C), "lw": 1 + rand(g, C, scale=0.2), "lb": rand(g, C, scale=0.1), "wi": rand(g, 2 * F, C, scale=C ** -0.5),
         "wo": rand(g, C, F, scale=F ** -0.5)}
    t = {k: v.to(DEV) for k, v in t.items()}
    probe = rand(g, M, C).to(DEV)

    def step(a):
        y = functional.gated_ffn(functional.layer_norm(a["z"], a["lw"], a["lb"]), a["wi"], a["wo"])
        return functional.dropout(y, 0.2, 5, 1, residual=a["z"])

    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    with torch.enable_grad():
        loss = (step(leaves) * probe).sum()
        grads = dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()))))
    e = 2.0 ** -6
    for k in t:
        d = rand(g, *t[k].shape).to(DEV) * t[k].abs().mean()
        up, dn = dict(t), dict(t)
        up[k], dn[k] = t[k] + e * d, t[k] - e * d
        with torch.no_grad():
            num = ((step(up).double() - step(dn).double()) * probe.double()).sum().item() / (2 * e)
        ana = (grads[k].double() * d.double()).sum().item()
        scale = (grads[k].double().norm() * d.double().norm()).item()
        print(f"  {k}: {num:.6f} {ana:.6f} scale {scale:.3f}", flush=True)
        assert abs(num - ana) <= 2.0 ** -9 * scale, (k, num, ana, scale)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_transition_training_step(dtype):
    """The module with gradients enabled: its value is the inference path's to bf16 accuracy, its
    gradients the formulas', parameters stay fp32 and get fp32 gradients."""
    print(f"case transition step {dtype}", flush=True)
    C, E = 64, 2
    mod = layers.Transition(C, E)
    synthetic.init_weights_(mod, 3, std=0.1)
    with torch.no_grad():
        mod.layernorm.weight.add_(0.1 * torch.randn(C, generator=torch.Generator().manual_seed(1)))
    mod = mod.to(DEV)
    g = torch.Generator().manual_seed(4)
    x, dy = rand(g, 3, 11, C, dtype=dtype), rand(g, 3, 11, C, dtype=dtype)
    xd = x.to(DEV).detach().requires_grad_()
    with torch.enable_grad():
        y = mod(xd)
        params = list(mod.parameters())
        grads = torch.autograd.grad(y, [xd] + params, dy.to(DEV))
    with torch.no_grad():
        inf = mod(x.to(DEV))
    assert y.dtype == dtype and all(q.dtype == F32 for q in grads[1:])
    # the same step in 64 bits, the parameters as they are
    x64 = x.double().requires_grad_()
    p64 = [q.detach().double().cpu().requires_grad_() for q in params]
    names = [n for n, _ in mod.named_parameters()]
    P = dict(zip(names, p64))
    with torch.enable_grad():
        xn = torch.nn.functional.layer_norm(x64, (C,), P["layernorm.weight"], P["layernorm.bias"], 1e-5)
        u, v = (xn @ P["swiglu.linear.weight"].t()).chunk(2, -1)
        want = (torch.nn.functional.silu(u) * v) @ P["linear_out.weight"].t()
        wg = torch.autograd.grad(want, [x64] + p64, dy.double())
    # bf16: about five roundings of 2^-9 rms each meet in a result; fp32: sums of up to 128 terms
    rel = 8 * 2.0 ** -9 if dtype == BF else 128 * 2.0 ** -24
    for got, ref, name in zip((y,) + tuple(grads), (want,) + wg, ["y", "dx"] + names):
        err = ((got.detach().double().cpu() - ref.detach()).norm() / ref.detach().norm()).item()
        print(f"  {name}: {err:.2e}", flush=True)
        assert err <= rel, (name, err, rel)
    err = ((inf.double().cpu() - want.detach()).norm() / want.detach().norm()).item()
    assert err <= 8 * 2.0 ** -9, err


def test_transition_training_under_autocast():
    """fp32 tensors under bf16 autocast: bf16 products on the rounded normalised rows, fp32 results and
    gradients; a forward pass inside and the backward pass outside of it."""
    print("case transition under autocast", flush=True)
    C = 64
    mod = layers.Transition(C, 2)
    synthetic.init_weights_(mod, 3, std=0.1)
    mod = mod.to(DEV)
    g = torch.Generator().manual_seed(14)
    x, dy = rand(g, 2, 9, C).to(DEV).requires_grad_(), rand(g, 2, 9, C).to(DEV)
    params = list(mod.parameters())
    with torch.enable_grad():
        with torch.autocast(x.device.type, dtype=BF):
            y = mod(x)
        grads = torch.autograd.grad(y, [x] + params, dy)
        xn = functional.layer_norm(x, mod.layernorm.weight, mod.layernorm.bias, mod.layernorm.eps)
        want = functional.gated_ffn(xn.to(BF), mod.swiglu.linear.weight, mod.linear_out.weight).float()
        wg = torch.autograd.grad(want, [x] + params, dy)
    assert y.dtype == F32 and torch.equal(y, want)
    assert all(p.dtype == F32 and torch.equal(p, q) for p, q in zip(grads, wg))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_functional_gradients_of_some_inputs(dtype):
    """Frozen inputs change nothing in the gradients of the others."""
    print(f"case gradients of some inputs {dtype}", flush=True)
    g = torch.Generator().manual_seed(15)
    x, w_in, w_out, dy = (t.to(DEV) for t in ffn_inputs(45, 64, 32, dtype, 15))
    lw, lb = (1 + rand(g, 64, scale=0.2)).to(DEV), rand(g, 64, scale=0.1).to(DEV)
    for f, args in ((functional.gated_ffn, (x, w_in, w_out)), (functional.layer_norm, (x, lw, lb))):
        def run(which):
            leaves = [t.clone().requires_grad_(k in which) for k, t in enumerate(args)]
            with torch.enable_grad():
                return torch.autograd.grad(f(*leaves), [leaves[k] for k in which], dy)
        full = run((0, 1, 2))
        for which in ((0,), (1,), (2,), (0, 2), (1, 2)):
            assert all(torch.equal(p, full[k]) for p, k in zip(run(which), which)), (f, which)


def test_modules_and_mixed_types():
    print("case modules", flush=True)
    g = torch.Generator().manual_seed(6)
    ln = primitives.LayerNorm(96, create_offset=False).to(DEV)
    x = rand(g, 5, 96, dtype=BF).to(DEV).requires_grad_()
    with torch.enable_grad():
        y = ln(x)
        gx, gw = torch.autograd.grad(y, [x, ln.weight], torch.ones_like(y))
    assert y.dtype == BF and gx.dtype == BF and gw.dtype == F32
    with torch.no_grad():
        assert torch.equal(ln(x.detach()), y.detach())
    drop = primitives.Dropout(0.3, shared_dim=-2)
    a, r = rand(g, 2, 6, 7, 32).to(DEV), rand(g, 2, 6, 7, 32).to(DEV)
    want = ops.dropout_forward(a, 0.3, 8, 2, 2, residual=r)
    assert torch.equal(drop(a, r, seed=8, offset=2), want)
    torch.manual_seed(1)
    one = drop(a)
    torch.manual_seed(1)
    assert torch.equal(drop(a), one) and not torch.equal(drop(a), one)
    drop.eval()
    assert torch.equal(drop(a, r), r + a) and drop(a) is a
    ar, rr = a.clone().requires_grad_(), r.clone().requires_grad_()
    drop.train()
    with torch.enable_grad():
        y = drop(ar, rr, seed=8)
        ga, gr = torch.autograd.grad(y, [ar, rr], torch.ones_like(y))
    assert torch.equal(gr, torch.ones_like(gr)) and torch.equal(ga, ops.dropout_backward(torch.ones_like(a), 0.3, 8, 0, 2))
    # weights of two types: each gradient in its own, rounded once
    x = rand(g, 9, 64, dtype=BF).to(DEV)
    wi, wo = rand(g, 64, 64, scale=0.1).to(DEV).double().requires_grad_(), rand(g, 64, 32, dtype=BF, scale=0.1).to(DEV).requires_grad_()
    with torch.enable_grad():
        y = functional.gated_ffn(x, wi, wo)
        gi, go = torch.autograd.grad(y, [wi, wo], torch.ones_like(y))
    _, ri, ro = ops.gated_ffn_backward(torch.ones_like(x), x, wi.detach().to(BF), wo.detach(), dw_dtype=F32)
    assert gi.dtype == torch.float64 and torch.equal(gi, ri.double()) and go.dtype == BF and torch.equal(go, ro.to(BF))
    # a device seed changed in place before the backward pass is an error, not another mask
    s = torch.tensor([8]).to(DEV)
    with torch.enable_grad():
        y = functional.dropout(ar, 0.3, s)
        s.add_(1)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, [ar], torch.ones_like(y))
    # second derivatives are refused
    with torch.enable_grad():
        z = a.clone().requires_grad_()
        (gz,) = torch.autograd.grad(functional.layer_norm(z).pow(2).sum(), [z], create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(gz.sum(), [z])


def test_parcae_trunk_lm_dropout():
    """The recurrence with its own dropout equals the one whose caller drops the embedding."""
    print("case parcae trunk with lm dropout", flush=True)
    C, n = 128, 6
    trunk = modules.ParcaeTrunk(C, lm_blocks=1, main_blocks=1).eval()
    synthetic.init_weights_(trunk, 5)
    trunk = trunk.to(DEV)
    g = torch.Generator().manual_seed(5)
    z0, zin, zlm = (rand(g, 1, n, n, C) for _ in range(3))
    pm = torch.ones(1, n, n, dtype=torch.bool)
    step = iter(range(10))

    def dropped():
        return ops.dropout_forward(zlm.to(DEV), 0.25, 99, next(step))
    with torch.no_grad():
        want = trunk(z0.to(DEV), zin.to(DEV), dropped, pm.to(DEV), num_recycles=1)
        got = trunk(z0.to(DEV), zin.to(DEV), zlm.to(DEV), pm.to(DEV), num_recycles=1, lm_dropout=0.25, lm_seed=99)
        plain = trunk(z0.to(DEV), zin.to(DEV), zlm.to(DEV), pm.to(DEV), num_recycles=1)
    assert torch.equal(got, want) and not torch.equal(got, plain)


def test_training_ops_streams_and_graphs():
    """Every operator on a side stream, and recorded into a graph that is replayed several times with new
    inputs and eager work between the replays: same bits as eager calls."""
    print("case streams and graphs", flush=True)
    g = torch.Generator().manual_seed(30)
    M, C, F = 333, 128, 256
    x, w_in, w_out, dy = (t.to(DEV) for t in ffn_inputs(M, C, F, BF, 31))
    lw, lb = (1 + rand(g, C, scale=0.2)).to(DEV), rand(g, C, scale=0.1).to(DEV)
    seed = torch.tensor([5]).to(DEV)
    z = x.clone()

    def step():
        xn, mean, rstd = ops.layer_norm_forward(z, lw, lb, stats=True)
        y = ops.gated_ffn_forward(xn, w_in, w_out)
        out = ops.dropout_forward(y, 0.25, seed, 3, residual=z)
        dyd = ops.dropout_backward(dy, 0.25, seed, 3)
        dxn, dwi, dwo = ops.gated_ffn_backward(dyd, xn, w_in, w_out)
        dz, dlw, dlb = ops.layer_norm_backward(dxn, z, mean, rstd, lw)
        return out, dz, dwi, dwo, dlw, dlb

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        z.copy_(rand(g, M, C, dtype=BF))
        seed.fill_(100 + k)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(replayed, want)), k
    # autograd on a side stream
    leaves = [t.clone().requires_grad_() for t in (z, lw, lb, w_in, w_out)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.enable_grad():
        y = functional.gated_ffn(functional.layer_norm(leaves[0], leaves[1], leaves[2]), leaves[3], leaves[4])
        y = functional.dropout(y, 0.25, 103, 3, residual=leaves[0])
        grads = torch.autograd.grad(y, leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(y.detach(), want[0])
    assert torch.equal(grads[3], want[2]) and torch.equal(grads[4], want[3]) and torch.equal(grads[1], want[4])
    assert torch.equal(grads[0], dy + want[1])


@pytest.mark.parametrize("M,C,F,dtype", [(16_390, 128, 64, BF), (16_390, 256, 64, BF), (12, 64, 32, BF), (3000, 136, 264, BF),
                                         (70, 128, 256, F32)])
def test_training_ops_two_graphs(M, C, F, dtype):
    """Two recorded steps of different inputs that live side by side, replayed in turn and on two streams
    at once with eager work between: same bits as eager calls."""
    print(f"case two graphs {M} x {C} x {F} {dtype}", flush=True)
    sets = [[t.to(DEV) for t in ffn_inputs(M, C, F, dtype, 40 + k)] for k in range(2)]

    def step(x, w_in, w_out, dy):
        xn, mean, rstd = ops.layer_norm_forward(x, stats=True)
        y = ops.gated_ffn_forward(xn, w_in, w_out)
        dxn, dwi, dwo = ops.gated_ffn_backward(dy, xn, w_in, w_out)
        return (y, dwi, dwo) + ops.layer_norm_backward(dxn, x, mean, rstd)

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    graphs, held = [torch.cuda.CUDAGraph() for _ in sets], []
    for graph, s in zip(graphs, sets):
        with torch.cuda.graph(graph):
            held.append(step(*s))
    streams = [torch.cuda.Stream() for _ in sets]
    for k in range(4):
        for t in (t for h in held for t in h):
            t.zero_()
        torch.cuda.synchronize()
        for i, graph in enumerate(graphs):
            if k % 2:
                with torch.cuda.stream(streams[i]):
                    graph.replay()
            else:
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for h, w in zip(held, want) for p, q in zip(h, w)), k
        assert all(torch.equal(p, q) for p, q in zip(step(*sets[k % 2]), want[k % 2])), k
        torch.cuda.synchronize()
