"""Layers of any width on the GPU against their formulas in 64 bits.

Tolerances are bounds, element by element: a product's fp32 sum of K terms is off by at most (K + 4) 2^-23 times the sum of
their magnitudes (each addition half a step of a partial sum, doubled for matrix cores that cut instead of rounding); an
activation passes that on with its steepest slope and adds U.ACT_TOL; a rounding to the output's type adds half a step.
"""
import ctypes as C

import pytest
import torch

import layers_util as U
import ngp_abi as A

pytestmark = pytest.mark.gpu

STEEPEST = {"none": 1.0, "relu": 1.0, "logistic": 0.25, "gelu": 1.13, "silu": 1.1}  # exponential: its own value
CURVE = {"none": 0.0, "relu": 0.0, "logistic": 0.1, "gelu": 0.8, "silu": 0.5}       # the largest second derivative


def normal(seed, *shape, scale=1.0, t=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)


def close(got, want, tol, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.numel(), float(err[bad].max()), float(tol[bad].max()) if tol.dim() else float(tol))


def sum_tol(magnitudes, k):
    return (k + 4) * 2.0 ** -23 * magnitudes


def check_checkpoint(c8, want, tol, kind):
    """A checkpoint of values that are `want` up to `tol`: the block's power of two, and every value within its step."""
    width = want.shape[1]
    q, e = c8[0][:, :width], c8[1][:, :U.blocks(width)]
    got = U.load(q, e)
    step = torch.exp2(e.double() - 133)
    top = torch.zeros(want.shape[0], U.blocks(width) * 32, dtype=torch.float64, device=want.device)
    top[:, :width] = want.abs()
    slack = torch.zeros_like(top)
    slack[:, :width] = tol
    top, slack = top.view(want.shape[0], -1, 32).amax(-1), slack.view(want.shape[0], -1, 32).amax(-1)
    low = 2.0 ** -24 if kind == "f16" else 2.0 ** -133
    assert (128 * step >= top - slack).all()
    assert ((64 * step <= top + slack) | (step <= low)).all()
    each = step.repeat_interleave(32, 1)[:, :width]
    near_end = want.abs() + tol >= 127 * each
    close(got, want, torch.where(near_end, each, each / 2) + tol, "checkpoint")


# n, n_in, n_out: a row, tiles' edges on both sides, odd widths, few and many rows
SHAPES = [(1, 1, 1), (1, 64, 64), (1, 1024, 520), (2, 33, 65), (5, 7, 3), (16, 256, 48), (17, 40, 130), (33, 8, 31), (63, 65, 127),
          (64, 64, 64), (65, 72, 136), (129, 257, 255), (200, 512, 264), (257, 96, 1), (300, 1, 300), (1000, 333, 77),
          (127, 2048, 64), (513, 128, 640), (2049, 64, 16), (1, 4096, 4500), (3, 2500, 40), (16, 16384, 96), (13, 2111, 36),
          (3, 65536, 40), (40, 24, 65536)]


def forward_reference(x, w, b, name, r):
    z = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    ztol = sum_tol(mag, x.shape[1])
    v = U.act(name, z)
    tol = (STEEPEST[name] if name in STEEPEST else v * 1.01) * ztol + U.ACT_TOL * (0.0 if name in ("none", "relu") else v.abs().clamp(min=1))
    return z, ztol, (v + r.double() if r is not None else v), tol


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n, n_in, n_out", SHAPES)
def test_forward(n, n_in, n_out, kind):
    t = U.TYPES[kind][1]
    for seed, name in enumerate(U.ACTS):
        x, w = normal(seed, n, n_in, t=t), normal(seed + 10, n_out, n_in, scale=n_in ** -0.5, t=t)
        b = normal(seed + 20, n_out) if seed % 3 else None
        r = normal(seed + 30, n, n_out, t=t) if seed % 2 else None
        z, z8 = torch.empty(n, n_out, dtype=t, device="cuda"), U.new8(n, n_out)
        y = U.call_linear(kind, x, w, b, name, r, z=z if seed != 2 else None, z8=z8 if seed != 3 else None)
        ze, ztol, ye, ytol = forward_reference(x, w, b, name, r)
        close(y, ye, ytol + U.rounding(ye.abs() + ytol, t), name)
        if seed != 2:
            close(z, ze, ztol + U.rounding(ze.abs() + ztol, t), "z")
        if seed != 3:
            check_checkpoint(z8, ze, ztol, kind)


# enough output tiles of 256 x 256 for one per CU, with edges on both sides: each product of the passes in turn, over a K of
# less than a stage, of whole stages, and with an odd rest
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n, n_in, n_out", [(3700, 40, 3990), (4100, 256, 3601), (3650, 3700, 16), (4001, 3520, 264), (32, 3900, 3700),
                                            (167, 4096, 4000), (1000, 3601, 3601)])
def test_large_products(n, n_in, n_out, kind):
    t = U.TYPES[kind][1]
    x, w, r = normal(1, n, n_in, t=t), normal(2, n_out, n_in, scale=n_in ** -0.5, t=t), normal(3, n, n_out, t=t)
    z8 = U.new8(n, n_out)
    y = U.call_linear(kind, x, w, None, "silu", r, z8=z8)
    ze, ztol, ye, ytol = forward_reference(x, w, None, "silu", r)
    close(y, ye, ytol + U.rounding(ye.abs() + ytol, t))
    check_checkpoint(z8, ze, ztol, kind)
    dy, xk, zk, w, x, z = backward_inputs(kind, n, n_in, n_out, 5, True, True)
    check_backward(kind, U.call_linear_backward(kind, dy, xk, w, "gelu", zk, "silu"), dy, x, z, w, "gelu", "silu")


@pytest.mark.parametrize("pad, offset", [(0, 0), (8, 0), (3, 0), (0, 1), (8, 8), (5, 3)])
@pytest.mark.parametrize("n, n_in, n_out", [(1, 72, 40), (37, 40, 88), (70, 33, 67), (300, 200, 264)])
def test_forward_strides_and_frames(n, n_in, n_out, pad, offset):
    t = torch.float16
    mats = {k: U.Framed(*s, t, pad, offset, value=float("nan"), init=v) for k, s, v in (
        ("x", (n, n_in), normal(1, n, n_in)), ("w", (n_out, n_in), normal(2, n_out, n_in, scale=n_in ** -0.5)),
        ("r", (n, n_out), normal(3, n, n_out)), ("y", (n, n_out), None), ("z", (n, n_out), None))}
    z8 = U.new8(n, n_out, pad)
    x, w, r = (mats[k].t.clone() for k in "xwr")
    U.call_linear("f16", mats["x"].t, mats["w"].t, None, "silu", mats["r"].t, y=mats["y"].t, z=mats["z"].t, z8=z8)
    ze, ztol, ye, ytol = forward_reference(x, w, None, "silu", r)
    close(mats["y"].t, ye, ytol + U.rounding(ye.abs() + ytol, t))
    close(mats["z"].t, ze, ztol + U.rounding(ze.abs() + ztol, t))
    check_checkpoint(z8, ze, ztol, "f16")
    for k, m in mats.items():
        assert m.untouched_outside(), k
    assert (z8[0][:, n_out:] == 85).all() and (z8[1][:, U.blocks(n_out):] == 170).all()


def test_forward_in_the_place_of_the_residual():
    for n, n_out in ((3, 64), (130, 200), (400, 256)):
        x, w, r = normal(1, n, 64, t=torch.bfloat16), normal(2, n_out, 64, scale=0.1, t=torch.bfloat16), normal(3, n, n_out, t=torch.bfloat16)
        want = U.call_linear("bf16", x, w, None, "gelu", r)
        U.call_linear("bf16", x, w, None, "gelu", r, y=r)
        assert torch.equal(r, want)


@pytest.mark.parametrize("n", [1, 40, 300])
def test_forward_keeps_non_finite_rows_to_themselves(n):
    x, w = normal(1, n, 96, t=torch.float16), normal(2, 80, 96, scale=0.1, t=torch.float16)
    want = U.call_linear("f16", x, w, None, "relu")
    x[n // 2, 17] = float("nan")
    y, z8 = torch.empty_like(want), U.new8(n, 80)
    U.call_linear("f16", x, w, None, "relu", y=y, z8=z8)
    assert torch.isnan(y[n // 2]).all() and (z8[1][n // 2, :3] == 255).all()
    keep = torch.arange(n, device="cuda") != n // 2
    assert torch.equal(y[keep], want[keep]) and (z8[1][keep, :3] != 255).all()


def backward_inputs(kind, n, n_in, n_out, seed, z8, x8):
    t = U.TYPES[kind][1]
    dy, x, z = normal(seed, n, n_out, scale=0.1, t=t), normal(seed + 1, n, n_in, t=t), normal(seed + 2, n, n_out, t=t)
    w = normal(seed + 3, n_out, n_in, scale=n_in ** -0.5, t=t)
    xk, zk = U.call_store(kind, x) if x8 else x, U.call_store(kind, z) if z8 else z
    return dy, xk, zk, w, U.load(*xk) if x8 else x.double(), U.load(*zk) if z8 else z.double()


def check_backward(kind, got, dy, x, z, w, name, x_name, dw_kind=None, base=None):
    t = U.TYPES[kind][1]
    dy, w = dy.double(), w.double()
    dx, dw, db = U.linear_backward(dy, z, x, w, name, x_name, t)
    s = U.act_slope(name, z) if name != "none" else torch.ones_like(dy)
    dz = dy * s
    # the slope, and dz's rounding to the operands' type
    slope_err = dy.abs() * U.ACT_TOL * s.abs().clamp(min=1) if name not in ("none", "relu") else torch.zeros_like(dy)
    dz_err = slope_err + (0.0 if name in ("none", "relu") else U.rounding(dz.abs() + slope_err, t))
    a = U.act(x_name, x)
    a = a.to(t).double() if x_name != "none" else a
    # an activation recomputed within ACT_TOL may round to the other side
    a_err = U.ACT_TOL * a.abs().clamp(min=1) + 2 * U.rounding(a, t) if x_name not in ("none", "relu") else torch.zeros_like(a)
    p, n_out, n = dz.abs() + dz_err, w.shape[0], dy.shape[0]
    if got[0] is not None:
        pre = dz @ w
        tol = dz_err @ w.abs() + sum_tol(p @ w.abs(), n_out)
        xs = U.act_slope(x_name, x) if x_name != "none" else torch.ones_like(pre)
        tol = tol * xs.abs() + (0.0 if x_name in ("none", "relu") else (pre.abs() + tol) * U.ACT_TOL * xs.abs().clamp(min=1))
        close(got[0], dx, tol + U.rounding(dx.abs() + tol, t), "dx")
    if got[1] is not None:
        tol = dz_err.t() @ a.abs() + p.t() @ a_err + sum_tol(p.t() @ (a.abs() + a_err), n)
        dw_t = U.TYPES[dw_kind or kind][1]
        if base is not None:
            dw, tol = dw + base[0].double(), tol + 2.0 ** -23 * (dw + base[0].double()).abs()
        close(got[1], dw, tol + U.rounding(dw.abs() + tol, dw_t), "dw")
    if got[2] is not None:
        tol = slope_err.sum(0) + sum_tol(dz.abs().sum(0), n)
        if base is not None:
            db, tol = db + base[1].double(), tol + 2.0 ** -23 * (db + base[1].double()).abs()
        close(got[2], db, tol, "db")


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n, n_in, n_out", SHAPES)
def test_backward(n, n_in, n_out, kind):
    for seed, (name, x_name, z8, x8) in enumerate((("none", "none", False, False), ("relu", "none", False, True),
                                                   ("gelu", "none", True, False), ("silu", "relu", True, True),
                                                   ("none", "gelu", False, True), ("logistic", "silu", False, False),
                                                   ("exponential", "logistic", False, False), ("none", "exponential", False, True))):
        dy, xk, zk, w, x, z = backward_inputs(kind, n, n_in, n_out, seed, z8, x8)
        got = U.call_linear_backward(kind, dy, xk, w, name, zk if name != "none" else None, x_name)
        check_backward(kind, got, dy, x, z, w, name, x_name)


# layers of up to 128 x 128 over many rows: every pair of padded widths, rows that end inside a workgroup's turn
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n, n_in, n_out", [(16384, 64, 64), (16385, 16, 16), (20011, 128, 128), (40001, 33, 67), (17000, 100, 64), (16500, 3, 120),
                                            (16999, 128, 8), (100003, 1, 1)])
def test_narrow_layers(n, n_in, n_out, kind):
    t = U.TYPES[kind][1]
    for seed, name in enumerate(("relu", "gelu")):
        x, w, b, r = normal(seed, n, n_in, t=t), normal(seed + 1, n_out, n_in, scale=n_in ** -0.5, t=t), normal(seed + 2, n_out), normal(seed + 3, n, n_out, t=t)
        z, z8 = torch.empty(n, n_out, dtype=t, device="cuda"), U.new8(n, n_out)
        y = U.call_linear(kind, x, w, b, name, r if seed else None, z=z, z8=z8 if seed else None)
        ze, ztol, ye, ytol = forward_reference(x, w, b, name, r if seed else None)
        close(y, ye, ytol + U.rounding(ye.abs() + ytol, t), name)
        close(z, ze, ztol + U.rounding(ze.abs() + ztol, t), "z")
        if seed:
            check_checkpoint(z8, ze, ztol, kind)
    for seed, (name, x_name, z8, x8) in enumerate((("relu", "none", False, False), ("silu", "gelu", True, True), ("none", "relu", False, True))):
        dy, xk, zk, w, x, z = backward_inputs(kind, n, n_in, n_out, seed, z8, x8)
        every = U.call_linear_backward(kind, dy, xk, w, name, zk if name != "none" else None, x_name)
        check_backward(kind, every, dy, x, z, w, name, x_name)
    for k in range(3):
        some = U.call_linear_backward(kind, dy, xk, w, name, None, x_name, dx=k == 0 or None, dw=k == 1 or None, db=k == 2 or None)
        if k < 2:
            assert torch.equal(some[k], every[k])
        else:
            check_backward(kind, some, dy, x, z, w, name, x_name)
    base = normal(9, n_out, n_in), normal(10, n_out)
    got = U.call_linear_backward(kind, dy, xk, w, name, None, x_name, dw_kind="f32", accumulate=True, dw=base[0].clone(), db=base[1].clone())
    check_backward(kind, got, dy, x, z, w, name, x_name, "f32", base)


def test_narrow_layers_strides_and_frames():
    t, nan = torch.float16, float("nan")
    for n, n_in, n_out, pad, offset in ((16400, 64, 40, 8, 0), (16400, 72, 64, 3, 1), (17001, 45, 91, 0, 1)):
        dy, x, z, w, dx, dw = (U.Framed(*s, t, pad, offset, value=nan, init=normal(k, *s, scale=0.2)) for k, s in enumerate(
            ((n, n_out), (n, n_in), (n, n_out), (n_out, n_in), (n, n_in), (n_out, n_in))))
        got = U.call_linear_backward("f16", dy.t, x.t, w.t, "gelu", z.t, "silu", dx=dx.t, dw=dw.t)
        check_backward("f16", got, dy.t, x.t.double(), z.t.double(), w.t, "gelu", "silu")
        y = U.Framed(n, n_out, t, pad, offset)
        U.call_linear("f16", x.t, w.t, None, "silu", z.t, y=y.t)
        ze, ztol, ye, ytol = forward_reference(x.t, w.t, None, "silu", z.t)
        close(y.t, ye, ytol + U.rounding(ye.abs() + ytol, t))
        for m in (dy, x, z, w, dx, dw, y):
            assert m.untouched_outside()


@pytest.mark.parametrize("n, n_in, n_out", [(1, 72, 40), (37, 40, 88), (70, 33, 67), (700, 200, 264)])
def test_backward_accumulates_in_32_bits(n, n_in, n_out):
    dy, xk, zk, w, x, z = backward_inputs("f16", n, n_in, n_out, 5, True, False)
    base = normal(9, n_out, n_in), normal(10, n_out)
    got = U.call_linear_backward("f16", dy, xk, w, "gelu", zk, dw_kind="f32", accumulate=True, dw=base[0].clone(), db=base[1].clone())
    check_backward("f16", got, dy, x, z, w, "gelu", "none", "f32", base)
    got = U.call_linear_backward("f16", dy, xk, w, "gelu", zk, dw_kind="f32")
    check_backward("f16", got, dy, x, z, w, "gelu", "none", "f32")


@pytest.mark.parametrize("pad, offset", [(8, 0), (3, 0), (0, 1), (8, 8), (5, 3)])
@pytest.mark.parametrize("x_name", ["none", "gelu"])
def test_backward_strides_and_frames(pad, offset, x_name):
    t = torch.bfloat16
    for n, n_in, n_out in ((1, 72, 40), (70, 33, 67), (300, 200, 264)):
        nan = float("nan")
        dy, x, z, w, dx, dw = (U.Framed(*s, t, pad, offset, value=nan, init=normal(k, *s, scale=0.2)) for k, s in enumerate(
            ((n, n_out), (n, n_in), (n, n_out), (n_out, n_in), (n, n_in), (n_out, n_in))))
        got = U.call_linear_backward("bf16", dy.t, x.t, w.t, "silu", z.t, x_name, dx=dx.t, dw=dw.t)
        check_backward("bf16", got, dy.t, x.t.double(), z.t.double(), w.t, "silu", x_name)
        for m in (dy, x, z, w, dx, dw):
            assert m.untouched_outside()


def test_backward_of_some_gradients_only():
    dy, xk, zk, w, x, z = backward_inputs("f16", 150, 88, 40, 3, False, True)
    every = U.call_linear_backward("f16", dy, xk, w, "relu", zk)
    for k in range(3):
        some = U.call_linear_backward("f16", dy, xk if k == 1 else None, w, "relu", zk, dx=k == 0 or None, dw=k == 1 or None, db=k == 2 or None)
        assert torch.equal(some[k], every[k]) and all(v is None for i, v in enumerate(some) if i != k)


# what a call does not need may be absent, what it has no use for may be there
@pytest.mark.parametrize("n, n_in, n_out", [(150, 88, 40), (16400, 64, 40), (16401, 45, 91), (4100, 3600, 264)])
def test_backward_with_as_little_and_as_much_as_is_allowed(n, n_in, n_out):
    dy, xk, zk, w, x, z = backward_inputs("f16", n, n_in, n_out, 4, False, False)
    every = U.call_linear_backward("f16", dy, xk, w, "none", None)
    check_backward("f16", every, dy, x, z, w, "none", "none")
    for got in (U.call_linear_backward("f16", dy, xk, w, "none", zk), U.call_linear_backward("f16", dy, xk, w, "none", U.call_store("f16", zk))):
        assert all(torch.equal(g, e) for g, e in zip(got, every))
    got = U.call_linear_backward("f16", dy, None, w, "none", None, dw=None)
    assert got[1] is None
    check_backward("f16", got, dy, x, z, w, "none", "none")  # (one product alone may take other tiles than two together)
    got = U.call_linear_backward("f16", dy, xk, None, "none", None, dx=None, db=None, n_in=n_in)
    assert got[0] is None and got[2] is None
    check_backward("f16", got, dy, x, z, w, "none", "none")


def test_no_rows():
    for kind in ("f16", "bf16"):
        t = U.TYPES[kind][1]
        x, w = torch.empty(0, 40, dtype=t, device="cuda"), normal(1, 24, 40, t=t)
        assert U.call_linear(kind, x, w).shape == (0, 24)
        dx, dw, db = U.call_linear_backward(kind, torch.empty(0, 24, dtype=t, device="cuda"), x, w)
        assert (dw == 0).all() and (db == 0).all()
        dw = normal(2, 24, 40)
        got = U.call_linear_backward(kind, torch.empty(0, 24, dtype=t, device="cuda"), x, w, dw_kind="f32", accumulate=True,
                                     dw=dw.clone(), db=torch.ones(24, device="cuda"))
        assert torch.equal(got[1], dw) and (got[2] == 1).all()
        y, mean, rstd = U.call_layer_norm(kind, x)
        dx, dg, db = U.call_layer_norm_backward(kind, x, x, mean, rstd)
        assert y.shape == (0, 40) and (dg == 0).all() and (db == 0).all()
        q, e = U.call_store(kind, x)
        assert U.call_load(kind, (q, e), 40).shape == (0, 40)


# ---- layer norm ------------------------------------------------------------------------------------------------------
NORMS = [(1, 1), (1, 4096), (3, 33), (2, 8), (7, 31), (5, 64), (130, 100), (65, 255), (64, 256), (33, 777), (9, 1024), (4, 1025), (300, 2048),
         (17, 4097), (3, 8192), (2, 12345), (2, 65536), (1000, 40), (5000, 16)]


def norm_tol(x, mean, rstd, width, gain):
    """How far a row's normalised values times `gain` may be off before they are rounded: sums over `width` values of which
    each is at most (width / 32 + 40) additions long, doubled; the mean's error times rstd and rstd's relative error."""
    adds = (width / 32 + 40) * 2.0 ** -23
    dmean = adds * x.abs().mean(-1, keepdim=True)
    r = rstd[:, None]
    centred = (x - mean[:, None]).abs()
    drel = adds + 2 * dmean * r * (1 + centred.mean(-1, keepdim=True) * r)  # of the variance, halved by the root
    return ((dmean + centred * (drel + 2.0 ** -21)) * r) * gain, dmean[:, 0], (drel + 2.0 ** -21)[:, 0] * rstd


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, width", NORMS)
def test_layer_norm(n, width, kind):
    t = U.TYPES[kind][1]
    x = (normal(1, n, width, scale=2.0) + normal(2, n, 1)).to(t)
    gamma, beta = normal(3, width, scale=0.3) + 1, normal(4, width)
    for g, b in ((gamma, beta), (None, None)):
        y8 = U.new8(n, width)
        y, mean, rstd = U.call_layer_norm(kind, x, g, b, y8=y8)
        ge, be = (torch.ones_like(gamma), torch.zeros_like(beta)) if g is None else (g, b)
        ye, me, re = U.layer_norm(x.double(), ge.double(), be.double(), 1e-5)
        tol, dmean, drstd = norm_tol(x.double(), me, re, width, ge.double().abs())
        tol = tol + 2.0 ** -22 * (ye.abs() + be.double().abs())
        close(y, ye, tol + U.rounding(ye.abs() + tol, t), "y")
        close(mean, me, dmean + 2.0 ** -24 * me.abs() + 1e-37, "mean")
        close(rstd, re, drstd, "rstd")
        check_checkpoint(y8, ye, tol, kind)


def test_layer_norm_of_rows_far_from_zero_and_of_equal_values():
    x = normal(1, 50, 700) + 10000.0
    y, mean, rstd = U.call_layer_norm("f32", x)
    ye, me, re = U.layer_norm(x.double(), torch.ones(700, device="cuda").double(), 0.0, 1e-5)
    tol, dmean, drstd = norm_tol(x.double(), me, re, 700, 1.0)
    close(y, ye, tol + 2.0 ** -22 * ye.abs()), close(mean, me, dmean), close(rstd, re, drstd)
    y, mean, rstd = U.call_layer_norm("f32", torch.full((3, 96), 5.0, device="cuda"), eps=0.25)
    assert (y == 0).all() and (mean == 5).all() and (rstd == 2).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, width", NORMS)
def test_layer_norm_backward(n, width, kind):
    t = U.TYPES[kind][1]
    x = (normal(1, n, width, scale=2.0) + normal(2, n, 1)).to(t)
    dy, add, gamma = normal(3, n, width, scale=0.1, t=t), normal(4, n, width, scale=0.1, t=t), normal(5, width, scale=0.3) + 1
    _, mean, rstd = U.call_layer_norm(kind, x)
    for x8, a, g in ((False, add, gamma), (True, None, gamma), (True, add, None)):
        xk = U.call_store(kind, x) if x8 else x
        xe = U.load(*xk) if x8 else x.double()
        got = U.call_layer_norm_backward(kind, dy, xk, mean, rstd, g, a)
        ge = gamma.double() if g is not None else torch.ones(width, dtype=torch.float64, device="cuda")
        m, r = mean.double(), rstd.double()
        dx, dg, db = U.layer_norm_backward(dy.double(), xe, m, r, ge)
        xh, gr = (xe - m[:, None]) * r[:, None], dy.double() * ge
        adds = (width / 32 + 40) * 2.0 ** -23
        xh_err = 2.0 ** -22 * xh.abs() + 2.0 ** -23 * (xe.abs() + m.abs()[:, None]) * r[:, None]
        s0, s1 = gr.abs().mean(-1, keepdim=True), (gr.abs() * (xh.abs() + xh_err)).mean(-1, keepdim=True)
        tol = r[:, None] * (adds * s0 + xh.abs() * (adds * s1 + (gr.abs() * xh_err).mean(-1, keepdim=True)) + xh_err * s1
                            + 2.0 ** -21 * (gr.abs() + s0 + xh.abs() * s1))
        if a is not None:
            dx = dx + a.double()
            tol = tol + 2.0 ** -23 * (dx.abs() + a.double().abs())
        close(got[0], dx, tol + U.rounding(dx.abs() + tol, t), "dx")
        close(got[1], dg, sum_tol((dy.double().abs() * (xh.abs() + xh_err)).sum(0), n) + (dy.double().abs() * xh_err).sum(0), "dgamma")
        close(got[2], db, sum_tol(dy.double().abs().sum(0), n), "dbeta")


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("pad, offset", [(8, 0), (3, 0), (0, 1), (5, 3)])
def test_norm_strides_and_frames(kind, pad, offset):
    t, nan = U.TYPES[kind][1], float("nan")
    for n, width in ((1, 40), (130, 100), (20, 777), (6, 4096)):
        x, dy, add, y, dx = (U.Framed(n, width, t, pad, offset, value=nan, init=normal(k, n, width)) for k in range(5))
        y8 = U.new8(n, width, pad)
        plain_y, mean, rstd = U.call_layer_norm(kind, x.t.contiguous())
        plain_dx = U.call_layer_norm_backward(kind, dy.t.contiguous(), x.t.contiguous(), mean, rstd, add=add.t.contiguous())
        U.call_layer_norm(kind, x.t, y=y.t, y8=y8)
        got = U.call_layer_norm_backward(kind, dy.t, x.t, mean, rstd, add=add.t, dx=dx.t)
        want8 = U.new8(n, width)
        U.call_layer_norm(kind, x.t.contiguous(), y8=want8)
        for u, v in ((y.t, plain_y), (dx.t, plain_dx[0])):  # another alignment may sum in another order
            close(u, v.double(), 2 * U.rounding(v.double(), t) + 1e-5)
        for k in (1, 2):
            close(got[k], plain_dx[k].double(), torch.tensor(1e-4, device="cuda").double())
        assert (y8[0][:, width:] == 85).all() and (y8[1][:, U.blocks(width):] == 170).all()
        close(U.load(y8[0][:, :width], y8[1][:, :U.blocks(width)]), U.load(*want8), torch.tensor(0.126, device="cuda").double())  # a step below 8
        assert all(m.untouched_outside() for m in (x, dy, add, y, dx))


def test_norm_backward_in_the_place_of_the_other_branch_and_accumulating():
    x, dy, add = (normal(k, 90, 256, t=torch.float16) for k in range(3))
    _, mean, rstd = U.call_layer_norm("f16", x)
    want = U.call_layer_norm_backward("f16", dy, x, mean, rstd, add=add)
    g0, b0 = normal(8, 256), normal(9, 256)
    got = U.call_layer_norm_backward("f16", dy, x, mean, rstd, add=add, dx=add, dgamma=g0.clone(), dbeta=b0.clone(), accumulate=True)
    assert torch.equal(got[0], want[0])
    assert torch.equal(got[1], g0 + want[1]) and torch.equal(got[2], b0 + want[2])
    only = U.call_layer_norm_backward("f16", dy, x, mean, rstd, dx=None, dbeta=None)
    assert only[0] is None and only[2] is None and torch.equal(only[1], want[1])


# ---- checkpoints -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, width", [(1, 1), (1, 32), (3, 31), (2, 33), (77, 333), (64, 64), (5, 4096), (300, 2040), (40, 65536)])
def test_checkpoints_are_the_definition(n, width, kind):
    t = U.TYPES[kind][1]
    v = (normal(1, n, width) * torch.exp2(normal(2, n, width, scale=2.0))).to(t)
    v[0, 0] = 0.0
    c8 = U.call_store(kind, v)
    q, e = U.store(v.double(), kind)
    assert torch.equal(c8[0], q) and torch.equal(c8[1], e)
    assert torch.equal(U.call_load(kind, c8, width).double(), U.load(q, e))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_checkpoints_of_extreme_values(kind):
    t = U.TYPES[kind][1]
    info = torch.finfo(t)
    v = torch.zeros(6, 70, dtype=t, device="cuda")
    v[0] = info.max
    v[1, ::3] = -info.max
    v[2] = info.smallest_normal * info.eps  # the smallest number
    v[2, 40] = 3 * info.smallest_normal * info.eps
    v[3, 5], v[4, 69], v[4, 3] = float("nan"), float("-inf"), 1.0
    c8 = U.call_store(kind, v)
    q, e = U.store(v.double(), kind) if kind != "f32" else (None, None)
    if kind != "f32":  # (32-bit subnormals lie below the definition's smallest step)
        assert torch.equal(c8[0], q) and torch.equal(c8[1], e)
    got = U.call_load(kind, c8, 70)
    assert torch.isfinite(got[:3]).all() and (got[0] > info.max * 0.98).all()
    if kind == "f16":
        assert torch.equal(got[2], v[2])
    assert torch.isnan(got[3, :32]).all() and (got[3, 32:] == 0).all()
    assert torch.isnan(got[4, 64:]).all() and (got[4, 3] == 1).all() and (got[5] == 0).all()


@pytest.mark.parametrize("pad, offset", [(3, 0), (0, 1), (8, 8), (5, 3)])
def test_checkpoint_strides_and_frames(pad, offset):
    for kind in ("f32", "bf16"):
        t = U.TYPES[kind][1]
        for n, width in ((1, 7), (30, 100), (9, 512)):
            v = U.Framed(n, width, t, pad, offset, value=float("nan"), init=normal(1, n, width))
            c8 = U.new8(n, width, pad)
            U.call_store(kind, v.t, c8)
            q, e = U.store(v.t.double(), kind)
            assert torch.equal(c8[0][:, :width], q) and torch.equal(c8[1][:, :U.blocks(width)], e)
            assert (c8[0][:, width:] == 85).all() and (c8[1][:, U.blocks(width):] == 170).all()
            out = U.Framed(n, width, t, pad, offset)
            U.call_load(kind, c8, width, out.t)
            assert torch.equal(out.t.double(), U.load(q, e)) and out.untouched_outside() and v.untouched_outside()


# ---- together, as they are used --------------------------------------------------------------------------------------
def residual_block(kind, s):
    """x + W2 gelu(W1 norm(x) + b1) + b2 and its gradients; norm(x) and W1's pre-activation are kept in 8 bits."""
    n, d = s["x"].shape
    hidden = s["w1"].shape[0]
    h8, z8, x8 = U.new8(n, d), U.new8(n, hidden), U.call_store(kind, s["x"])
    h, mean, rstd = U.call_layer_norm(kind, s["x"], s["gamma"], s["beta"], y8=h8)
    a = U.call_linear(kind, h, s["w1"], s["b1"], "gelu", z8=z8)
    y = U.call_linear(kind, a, s["w2"], s["b2"], residual=s["x"])
    dz, dw2, db2 = U.call_linear_backward(kind, s["dy"], z8, s["w2"], x_activation="gelu")
    dh, dw1, db1 = U.call_linear_backward(kind, dz, h8, s["w1"])
    dx, dgamma, dbeta = U.call_layer_norm_backward(kind, dh, x8, mean, rstd, s["gamma"], s["dy"])
    return dict(y=y, dx=dx, dw1=dw1, db1=db1, dw2=dw2, db2=db2, dgamma=dgamma, dbeta=dbeta)


def block_state(kind, n, d, hidden, seed=0):
    t = U.TYPES[kind][1]
    return dict(x=normal(seed, n, d, t=t), gamma=normal(seed + 1, d, scale=0.2) + 1, beta=normal(seed + 2, d, scale=0.2),
                w1=normal(seed + 3, hidden, d, scale=d ** -0.5, t=t), b1=normal(seed + 4, hidden, scale=0.2),
                w2=normal(seed + 5, d, hidden, scale=hidden ** -0.5, t=t), b2=normal(seed + 6, d, scale=0.2),
                dy=normal(seed + 7, n, d, scale=0.1, t=t))


@pytest.mark.parametrize("kind, n, d, hidden", [("f16", 600, 64, 256), ("bf16", 257, 136, 520), ("f16", 33, 45, 91)])
def test_a_residual_block_learns_what_its_formula_says(kind, n, d, hidden):
    s = block_state(kind, n, d, hidden)
    got = residual_block(kind, s)
    v = {k: u.double().requires_grad_() for k, u in s.items() if k != "dy"}
    h, _, _ = U.layer_norm(v["x"], v["gamma"], v["beta"], 1e-5)
    y = U.act("gelu", h @ v["w1"].t() + v["b1"]) @ v["w2"].t() + v["b2"] + v["x"]
    g = torch.autograd.grad(y, [v[k] for k in ("x", "w1", "b1", "w2", "b2", "gamma", "beta")], s["dy"].double())
    want = dict(zip(("dx", "dw1", "db1", "dw2", "db2", "dgamma", "dbeta"), g), y=y.detach())
    # In the 2-norm: a checkpoint's value is at most half a step off, 2^-7 of a block's largest, which is within 4.5 times
    # the root mean square for 32 normal values (and the gelu's slope's slope is at most 0.8): at most 2^-7 4.5 = 0.035,
    # uniform over the step 0.035 / sqrt(3) = 0.02; two checkpoints meet in a gradient, and a few roundings of 2^-8 pass
    # through: 0.04.  The output meets no checkpoint: five roundings of 2^-8 at most.
    for k, w in want.items():
        err = (got[k].double() - w).norm() / w.norm()
        assert err < (5 * U.half_step(U.TYPES[kind][1]) if k == "y" else 0.04), (k, float(err))


@pytest.mark.parametrize("n, d, hidden", [(3000, 256, 512), (4200, 520, 4400), (20000, 64, 128), (9, 130, 200)])
def test_the_same_result_every_time_on_any_stream_and_in_graphs(n, d, hidden):
    s = block_state("f16", n, d, hidden)
    want = {k: v.clone() for k, v in residual_block("f16", s).items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        residual_block("f16", s)
        other = residual_block("f16", s)
    side.synchronize()
    assert all(torch.equal(other[k], want[k]) for k in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = residual_block_without_checks("f16", s)
    fresh = block_state("f16", n, d, hidden, seed=50)
    old = {k: v.clone() for k, v in s.items()}
    for step in range(4):
        source = old if step % 2 else fresh
        for k in s:
            s[k].copy_(source[k])
        eager = residual_block("f16", s)
        torch.cuda.synchronize()
        for v in held[0].values():
            v.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(held[0][k], eager[k]), (step, k)
            if step % 2:
                assert torch.equal(eager[k], want[k])


def test_two_streams_at_once():
    states = [block_state("bf16", n, d, hidden, seed) for n, d, hidden, seed in ((5000, 256, 1024, 0), (4000, 264, 1000, 40))]
    want = [{k: v.clone() for k, v in residual_block("bf16", s).items()} for s in states]
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, stream in zip(states, streams):  # nothing waits in between; every call has a workspace of its own
            with torch.cuda.stream(stream):
                got.append(residual_block_without_checks("bf16", s))
        torch.cuda.synchronize()
        for (out, rooms), w in zip(got, want):
            assert all(U.guards_hold(r) for r in rooms)
            assert all(torch.equal(out[k], w[k]) for k in w)


@pytest.mark.parametrize("n, n_in, n_out", [(40, 70, 50), (20000, 64, 48), (3700, 3600, 48)])
def test_a_row_that_is_not_finite_reaches_what_it_enters_and_no_more(n, n_in, n_out):
    dy, xk, zk, w, x, z = backward_inputs("f16", n, n_in, n_out, 3, True, False)
    want = U.call_linear_backward("f16", dy, xk, w, "silu", zk)
    dy[n // 3, 5] = float("inf")
    dx, dw, db = U.call_linear_backward("f16", dy, xk, w, "silu", zk)
    keep = torch.arange(n, device="cuda") != n // 3
    assert torch.equal(dx[keep], want[0][keep]) and not torch.isfinite(dx[n // 3]).any()
    cols = torch.arange(n_out, device="cuda") != 5
    assert torch.equal(dw[cols], want[1][cols]) and not torch.isfinite(dw[5]).any()
    assert torch.equal(db[cols], want[2][cols]) and not torch.isfinite(db[5])


def residual_block_without_checks(kind, s):
    """The block for a capture: guards are not looked at (that waits for the GPU), and every buffer stays held."""
    held, asked = [], U.guards_hold
    U.guards_hold = lambda room: held.append(room) or True
    try:
        return residual_block(kind, s), held
    finally:
        U.guards_hold = asked


def test_many_rows():
    n = 1 << 27  # more rows of a few values than a launch's threads
    x = torch.full((n, 5), 2.0, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = -2.0
    row = x[:1].double()
    want, _, _ = U.layer_norm(row, torch.ones(5, device="cuda").double(), 0.0, 1e-5)
    y, mean, rstd = U.call_layer_norm("bf16", x)
    for i in (0, n // 2 + 1, n - 1):
        close(y[i:i + 1], want, U.rounding(want, torch.bfloat16) * 1.01 + 1e-5)
    assert torch.equal(y.amin(0), y.amax(0))
    dx, dg, db = U.call_layer_norm_backward("bf16", x, x, mean, rstd, dx=y)
    assert torch.equal(dx.amin(0), dx.amax(0))
    # 2^27 equal terms: sums of 2^27 / 2^14 = 2^13 at most by one thread, then of their sums, each within half a step
    close(dg, n * (row * want)[0], 2.0 ** -10 * n * (row * want)[0].abs() + 1)
    close(db, n * row[0], 2.0 ** -10 * n * row[0].abs() + 1)
    w = normal(1, 3, 5, t=torch.bfloat16)
    out = U.call_linear("bf16", x, w)
    close(out[n - 1:], row @ w.double().t(), U.rounding(row @ w.double().t(), torch.bfloat16) * 1.01 + 1e-5)
    assert torch.equal(out.amin(0), out.amax(0))
    c8 = U.call_store("bf16", x)
    assert torch.equal(U.call_load("bf16", c8, 5, y), x)


def test_offsets_past_32_bits():
    n, width = 70000, 33000  # 2.3e9 values: past 2^31 elements, 4.6e9 bytes
    v = torch.empty(n, width, dtype=torch.float16, device="cuda")
    v.fill_(0.25)
    v[-1] = normal(1, width, t=torch.float16)
    c8 = torch.empty(n, width, dtype=torch.int8, device="cuda"), torch.empty(n, U.blocks(width), dtype=torch.uint8, device="cuda")
    U.call_store("f16", v, c8)
    q, e = U.store(v[-1:].double(), "f16")
    assert torch.equal(c8[0][-1:], q) and torch.equal(c8[1][-1:], e) and (c8[0][-2] == 64).all() and (c8[0][n // 2] == 64).all()
    out = torch.empty_like(v)
    U.call_load("f16", c8, width, out)
    assert torch.equal(out[-1:].double(), U.load(q, e)) and (out[n // 2] == 0.25).all()
    y, mean, rstd = U.call_layer_norm("f16", v, y=out)
    want, _, _ = U.layer_norm(v[-1:].double(), torch.ones(width, device="cuda").double(), 0.0, 1e-5)
    close(y[-1:], want, U.rounding(want, torch.float16) * 1.01 + 1e-5)
    dx, dg, db = U.call_layer_norm_backward("f16", v, c8, mean, rstd, dx=out)
    xe = U.load(q, e)
    want = U.layer_norm_backward(v[-1:].double(), xe, mean[-1:].double(), rstd[-1:].double(), torch.ones(width, device="cuda").double())[0]
    close(dx[-1:], want, U.rounding(want, torch.float16) * 1.01 + 1e-5)
    del out, dx, y
    w = normal(2, 24, width, scale=0.01, t=torch.float16)
    y = U.call_linear("f16", v, w)
    ze, ztol, ye, ytol = forward_reference(v[-1:], w, None, "none", None)
    close(y[-1:], ye, ytol + U.rounding(ye.abs() + ytol, torch.float16))
    dy = torch.zeros(n, 24, dtype=torch.float16, device="cuda")
    dy[-1] = normal(3, 24, t=torch.float16)
    dx, dw, db = U.call_linear_backward("f16", dy, c8, w, x_activation="relu")
    check_backward("f16", (dx[-1:], dw, db), dy[-1:], xe, None, w, "none", "relu")
    assert (dx[:-1] == 0).all()
