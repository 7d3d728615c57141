"""Timing cases of the training operators: layer norm, the gated feed-forward block and dropout.

``run`` computes a case in elementary torch operations, in 32 bits and rounded once at the end, or,
with ``own`` set, through ``kfold_amd.ops``.  ``exact`` restates the operators in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# --------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------
def _ln(name, direction, rows, C, dtype, affine=True):
    return {"name": name, "op": "layer_norm", "direction": direction, "rows": rows, "C": C, "dtype": dtype,
            "affine": affine}


def _ffn(name, direction, rows, C, F, dtype):
    return {"name": name, "op": "gated_ffn", "direction": direction, "rows": rows, "C": C, "F": F, "dtype": dtype}


def _drop(name, direction, B, I, J, C, dtype, p, shared, residual):
    """x [B, I, J, C]; shared: the dimension one mask value covers ("none", "rows" = 1, "columns" = 2)."""
    return {"name": name, "op": "dropout", "direction": direction, "B": B, "I": I, "J": J, "C": C, "dtype": dtype,
            "p": p, "shared": shared, "residual": residual}


def listed():
    return [
        # the single track of a short chain: a launch and little else
        _ln("ln_fwd_tokens", "forward", 64, 384, "f32"),
        # the pair representation of a training crop of 384 tokens
        _ln("ln_bwd_pair_crop", "backward", 384 * 384, 128, "bf16"),
        # the pair representation of 768 tokens at the shipping trunk's width
        _ln("ln_fwd_pair_large", "forward", 768 * 768, 256, "bf16"),
        # a ragged width, rows that are no multiple of anything
        _ln("ln_bwd_odd_width", "backward", 5001, 765, "f32"),
        # the single track of 37 tokens, one sample: weights are most of the traffic
        _ffn("ffn_fwd_tokens", "forward", 37, 384, 768, "bf16"),
        # transition of the pair track (expansion 2) at 768 tokens
        _ffn("ffn_fwd_pair", "forward", 768 * 768, 128, 256, "bf16"),
        # its backward pass on a training crop of 384 tokens
        _ffn("ffn_bwd_pair_crop", "backward", 384 * 384, 128, 256, "bf16"),
        # backward pass of the shipping trunk's transition (width 256, expansion 4), odd token count
        _ffn("ffn_bwd_trunk_crop", "backward", 383 * 383, 256, 1024, "bf16"),
        # the single track trained in fp32, two samples of 333 tokens
        _ffn("ffn_bwd_tokens_f32", "backward", 2 * 333, 384, 768, "f32"),
        # dropout of a single track's update
        _drop("drop_fwd_tokens", "forward", 1, 1, 80, 384, "bf16", 0.1, "none", False),
        # row-wise dropout of a triangle update with its residual, 768 tokens
        _drop("drop_fwd_pair_rows", "forward", 1, 768, 768, 128, "bf16", 0.25, "rows", True),
        # gradient of plain dropout on an odd pair grid and width
        _drop("drop_bwd_odd", "backward", 1, 765, 333, 129, "f32", 0.1, "none", False),
    ]


def _loguniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "gated_ffn", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    direction = rng.choice(["forward", "backward"])
    if op == "layer_norm":
        C = rng.choice([_loguniform(rng, 8, 2048), 32 * rng.randint(1, 64), rng.choice([64, 128, 256, 384, 768])])
        budget = 768 * 768 * 256 // (2 if dtype == "f32" else 1)
        if direction == "backward":
            budget = budget * 2 // 3
        c = _ln("", direction, _loguniform(rng, 1, budget // C), C, dtype, rng.random() < 0.85)
    elif op == "gated_ffn":
        C = rng.choice([64, 128, 128, 256, 384, 8 * rng.randint(2, 64)])
        F = rng.choice([C, 2 * C, 2 * C, 4 * C, 8 * rng.randint(2, 192)])
        budget = (383 * 383 * 256 * 1024) // (1 if dtype == "bf16" else 16)
        if direction == "forward":
            budget = budget * 2
        c = _ffn("", direction, _loguniform(rng, 1, max(2, min(768 * 768, budget // (C * F)))), C, F, dtype)
    else:
        C = rng.choice([64, 128, 256, 384, rng.randint(1, 400)])
        residual = direction == "forward" and rng.random() < 0.5
        budget = 768 * 768 * 128 // (2 if dtype == "f32" else 1)
        n = _loguniform(rng, 1, budget // C)
        I = _loguniform(rng, 1, n)
        J = max(1, n // I)
        B = rng.choice([1, 1, 2, 3])
        I = max(1, I // B)
        c = _drop("", direction, B, I, J, C, dtype, rng.choice([0.1, 0.15, 0.25, rng.random()]),
                  rng.choice(["none", "rows", "columns"]), residual)
    del c["name"]
    return c


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    back = case["direction"] == "backward"
    if case["op"] == "layer_norm":
        M, C = case["rows"], case["C"]
        par = 4 * C if case["affine"] else 0
        if back:
            return {"bytes": 3 * M * C * e + 8 * M + 3 * par, "flops": 13 * M * C}
        return {"bytes": 2 * M * C * e + 8 * M + 2 * par, "flops": 7 * M * C}
    if case["op"] == "gated_ffn":
        M, C, F = case["rows"], case["C"], case["F"]
        if back:        # three gradients' products and the two projections once more
            return {"bytes": (3 * M * C + 6 * C * F) * e, "flops": 16 * M * C * F + 12 * M * F}
        return {"bytes": (2 * M * C + 3 * C * F) * e, "flops": 6 * M * C * F + 5 * M * F}
    n = case["B"] * case["I"] * case["J"] * case["C"]
    return {"bytes": (3 if case["residual"] else 2) * n * e, "flops": (2 if case["residual"] else 1) * n}


# --------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def prepare(case, seed):
    g = _gen(seed)
    dt = _TYPES[case["dtype"]]

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    s = {"case": case}
    if case["op"] == "layer_norm":
        M, C = case["rows"], case["C"]
        # a residual stream: channels of unlike size, rows off zero
        s["x"] = ((torch.randn(M, C, generator=g, device=DEV) + 0.5) *
                  (0.5 + torch.rand(C, generator=g, device=DEV))).to(dt)
        s["weight"] = 1 + 0.2 * torch.randn(C, generator=g, device=DEV) if case["affine"] else None
        s["bias"] = 0.1 * torch.randn(C, generator=g, device=DEV) if case["affine"] else None
        s["eps"] = 1e-5
        if case["direction"] == "backward":
            s["dy"] = randn(M, C)
            xf = s["x"].float()
            s["mean"] = xf.mean(1)
            s["rstd"] = ((xf - s["mean"][:, None]).square().mean(1) + s["eps"]).rsqrt()
    elif case["op"] == "gated_ffn":
        M, C, F = case["rows"], case["C"], case["F"]
        s["x"] = randn(M, C)                                    # rows come out of a layer norm
        s["w_in"] = randn(2 * F, C, scale=C ** -0.5)
        s["w_out"] = randn(C, F, scale=F ** -0.5)
        if case["direction"] == "backward":
            s["dy"] = randn(M, C)
    else:
        shape = (case["B"], case["I"], case["J"], case["C"])
        s["x"] = randn(*shape)
        s["residual"] = randn(*shape) if case["residual"] else None
        s["seed"] = 0x5EED0000 + 7919 * seed
        s["offset"] = (seed % 1000) * 3 + 1
        s["shared_dim"] = {"none": None, "rows": 1, "columns": 2}[case["shared"]]
    return s


# --------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from kfold_amd import ops

    case = s["case"]
    back = case["direction"] == "backward"
    if case["op"] == "layer_norm":
        if back:
            grads = ops.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"],
                                            need_dparams=case["affine"])
            return grads if case["affine"] else grads[0]
        return ops.layer_norm_forward(s["x"], s["weight"], s["bias"], eps=s["eps"], stats=True)
    if case["op"] == "gated_ffn":
        if back:
            return ops.gated_ffn_backward(s["dy"], s["x"], s["w_in"], s["w_out"])
        return ops.gated_ffn_forward(s["x"], s["w_in"], s["w_out"])
    if back:
        return ops.dropout_backward(s["x"], case["p"], s["seed"], s["offset"], shared_dim=s["shared_dim"])
    return ops.dropout_forward(s["x"], case["p"], s["seed"], s["offset"], shared_dim=s["shared_dim"],
                               residual=s["residual"])


def _run_plain(s):
    case = s["case"]
    back = case["direction"] == "backward"
    if case["op"] == "layer_norm":
        return _plain_ln_backward(s) if back else _plain_ln_forward(s)
    if case["op"] == "gated_ffn":
        return _plain_ffn_backward(s) if back else _plain_ffn_forward(s)
    return _plain_dropout(s)


def _plain_ln_forward(s):
    x = s["x"].float()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = (d.square().mean(1) + s["eps"]).rsqrt()
    y = d * rstd[:, None]
    if s["weight"] is not None:
        y = y * s["weight"] + s["bias"]
    return y.to(s["x"].dtype), mean, rstd


def _plain_ln_backward(s):
    dy = s["dy"].float()
    xh = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    a = dy if s["weight"] is None else dy * s["weight"]
    dx = (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True)) * s["rstd"][:, None]
    if s["weight"] is None:
        return dx.to(s["x"].dtype)
    # sums over all rows: in 64 bits
    dw = (dy * xh).sum(0, dtype=torch.float64).float()
    db = dy.sum(0, dtype=torch.float64).float()
    return dx.to(s["x"].dtype), dw, db


def _plain_ffn_forward(s):
    F = s["w_out"].shape[1]
    t = s["x"].float() @ s["w_in"].float().t()
    u, v = t[:, :F], t[:, F:]
    h = u / (1 + torch.exp(-u)) * v
    return (h @ s["w_out"].float().t()).to(s["x"].dtype)


def _plain_ffn_backward(s):
    F = s["w_out"].shape[1]
    dt = s["x"].dtype
    x, dy = s["x"].float(), s["dy"].float()
    w_in, w_out = s["w_in"].float(), s["w_out"].float()
    t = x @ w_in.t()
    u, v = t[:, :F], t[:, F:]
    sig = 1 / (1 + torch.exp(-u))
    dh = dy @ w_out
    dw_out = dy.t() @ (u * sig * v)
    dt_ = torch.cat([dh * v * sig * (1 + u * (1 - sig)), dh * u * sig], dim=1)
    return (dt_ @ w_in).to(dt), (dt_.t() @ x).to(dt), dw_out.to(dt)


_LO = 0xFFFFFFFF


def _philox_words(n, seed, offset):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011):
    the four words of the counters (0..n-1, offset) under the key ``seed``, as int64."""
    i = torch.arange(n, device=DEV, dtype=torch.int64)
    c0, c1 = i & _LO, i >> 32
    c2 = torch.full_like(i, offset & _LO)
    c3 = torch.full_like(i, (offset >> 32) & _LO)
    k0, k1 = seed & _LO, (seed >> 32) & _LO
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57              # 64-bit products, wrapping
        c0, c1, c2, c3 = (((p1 >> 32) & _LO) ^ c1 ^ k0, p1 & _LO, ((p0 >> 32) & _LO) ^ c3 ^ k1, p0 & _LO)
        k0, k1 = (k0 + 0x9E3779B9) & _LO, (k1 + 0xBB67AE85) & _LO
    return c0, c1, c2, c3


def _keep(shape, p, seed, offset):
    n = math.prod(shape)
    words = torch.stack(_philox_words((n + 7) // 8, seed, offset), 1)
    r16 = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]
    return (r16 >= _threshold(p)).reshape(shape)


def _threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def _plain_dropout(s):
    case = s["case"]
    x = s["x"].float()
    shape = list(x.shape)
    if s["shared_dim"] is not None:
        shape[s["shared_dim"]] = 1
    t = _threshold(case["p"])
    keep = _keep(shape, case["p"], s["seed"], s["offset"])
    y = torch.where(keep, x * (65536 / (65536 - t) if t < 65536 else 0.0), torch.zeros((), device=DEV))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


# --------------------------------------------------------------------------------------------
# 64-bit restatement
# --------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    back = case["direction"] == "backward"
    x = s["x"].double()
    if case["op"] == "layer_norm":
        C = case["C"]
        w = torch.ones(C, device=DEV, dtype=torch.float64) if s["weight"] is None else s["weight"].double()
        if not back:
            mean = x.sum(1) / C
            var = (x - mean[:, None]).pow(2).sum(1) / C
            rstd = 1 / torch.sqrt(var + s["eps"])
            y = (x - mean[:, None]) * rstd[:, None] * w
            return (y if s["bias"] is None else y + s["bias"].double()), mean, rstd
        # the vector-Jacobian product with the statistics the pass is given
        rstd = s["rstd"].double()[:, None]
        n = (x - s["mean"].double()[:, None]) * rstd
        d = s["dy"].double()
        a = d * w
        dx = rstd / C * (C * a - a.sum(1, keepdim=True) - n * (a * n).sum(1, keepdim=True))
        if s["weight"] is None:
            return dx
        return dx, (d * n).sum(0), d.sum(0)
    if case["op"] == "gated_ffn":
        F = case["F"]
        wu, wv, wo = s["w_in"][:F].double(), s["w_in"][F:].double(), s["w_out"].double()
        # rows in pieces: the hidden values of all rows at once would not fit comfortably
        step = max(1, (1 << 26) // F)
        ys, dxs = [], []
        dwu, dwv, dwo = torch.zeros_like(wu), torch.zeros_like(wv), torch.zeros_like(wo)
        for r in range(0, case["rows"], step):
            xr = x[r:r + step]
            u, v = torch.matmul(xr, wu.t()), torch.matmul(xr, wv.t())
            sg = torch.sigmoid(u)
            if not back:
                ys.append(torch.matmul(u * sg * v, wo.t()))
                continue
            d = s["dy"][r:r + step].double()
            gh = torch.matmul(d, wo)
            gv = gh * (u * sg)
            gu = gh * v * (sg + u * sg * (1 - sg))
            dxs.append(torch.matmul(gu, wu) + torch.matmul(gv, wv))
            dwu += torch.matmul(gu.t(), xr)
            dwv += torch.matmul(gv.t(), xr)
            dwo += torch.matmul(d.t(), u * sg * v)
        if not back:
            return torch.cat(ys)
        return torch.cat(dxs), torch.cat([dwu, dwv]), dwo
    # dropout: the mask element by element, straight from the counters
    shape = [case["B"], case["I"], case["J"], case["C"]]
    if s["shared_dim"] is not None:
        shape[s["shared_dim"]] = 1
    count = math.prod(shape)
    bits = torch.empty(count, device=DEV, dtype=torch.int64)
    words = _philox_by_halves((count + 7) // 8, s["seed"], s["offset"])
    for e in range(8):
        half = (words[e // 2] >> (16 * (e % 2))) & 0xFFFF
        part = bits[e::8]
        part.copy_(half[:part.numel()])
    t = round(case["p"] * 65536)
    if t >= 65536:
        y = torch.zeros_like(x)
    else:
        y = x * (bits.reshape(shape) >= t).double() * (65536.0 / (65536 - t))
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return y


def _philox_by_halves(n, seed, offset):
    """The same generator with its 32 x 32-bit products put together from 16-bit halves."""
    def mul(a, c):
        al, ah, cl, ch = a & 0xFFFF, a >> 16, c & 0xFFFF, c >> 16
        mid = al * ch + ((al * cl) >> 16)
        mid2 = ah * cl + (mid & 0xFFFF)
        return (ah * ch + (mid >> 16) + (mid2 >> 16)), ((mid2 & 0xFFFF) << 16) | ((al * cl) & 0xFFFF)

    idx = torch.arange(n, device=DEV, dtype=torch.int64)
    zero = torch.zeros_like(idx)
    w = [idx % (1 << 32), idx // (1 << 32), zero + offset % (1 << 32), zero + (offset >> 32) % (1 << 32)]
    keys = [seed % (1 << 32), (seed >> 32) % (1 << 32)]
    for r in range(10):
        ka, kb = (keys[0] + r * 0x9E3779B9) % (1 << 32), (keys[1] + r * 0xBB67AE85) % (1 << 32)
        ha, la = mul(w[0], 0xD2511F53)
        hb, lb = mul(w[2], 0xCD9E8D57)
        w = [hb ^ w[1] ^ ka, lb, ha ^ w[3] ^ kb, la]
    return w
