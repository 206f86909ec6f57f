"""Layers of any width: sums over rows that fp32 holds exactly, so that a row that is lost or taken twice shows, and rows that
are not finite."""
import math

import pytest
import torch

import layers_util as U

pytestmark = pytest.mark.gpu


# ---- sums over rows that every partial sum holds exactly ----------------------------------------------------------------
def small(seed, *shape, t, most=2):
    """Whole numbers of 1 .. most and their negatives."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randint(1, most + 1, shape, generator=g, device="cuda") * (torch.randint(0, 2, shape, generator=g, device="cuda") * 2 - 1)
    return v.to(t)


def products(a, b):
    """a^T b of whole numbers, exact, in pieces that fit."""
    out = torch.zeros(a.shape[1], b.shape[1], dtype=torch.float64, device="cuda")
    for i in range(0, a.shape[0], 1 << 16):
        out += a[i:i + (1 << 16)].double().t() @ b[i:i + (1 << 16)].double()
    return out


def equal(got, want, what):
    assert torch.equal(got.double(), want.to(got.dtype).double()), (what, int((got.double() != want.to(got.dtype).double()).sum()))


# the one-pass kernel: both padded widths of either side, even and odd, no rest, one row, a row less than a chunk of 64, several
# turns of its 256 or 512 workgroups; then the other tiles, with and without splits of the rows
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n, n_in, n_out", [
    (16384, 64, 64), (16385, 16, 16), (16447, 64, 128), (32769, 128, 64), (16385, 128, 128), (40001, 33, 67), (32831, 67, 33), (16447, 99, 101),
    (65537, 1, 1), (100003, 5, 8), (16384, 7, 3), (33000, 128, 127),
    (1, 64, 64), (17, 40, 130), (3001, 77, 130), (5000, 256, 256), (16385, 200, 40), (20001, 40, 513), (70001, 136, 24), (4099, 3600, 264)])
def test_sums_over_rows_are_exact(n, n_in, n_out, kind):
    t = U.TYPES[kind][1]
    dy, x, w, z = small(1, n, n_out, t=t), small(2, n, n_in, t=t), small(3, n_out, n_in, t=t, most=1), small(4, n, n_out, t=t)
    z[-64:] = 1.0  # the rest's rows count whatever the activation
    x8, z8 = U.call_store(kind, x), U.call_store(kind, z)
    for name, x_name, zk, xk in (("none", "none", None, x), ("none", "relu", None, x8), ("relu", "none", z, x8), ("relu", "relu", z8, x)):
        dz = torch.where(z > 0, dy, torch.zeros_like(dy)) if name == "relu" else dy
        a = x.clamp(min=0) if x_name == "relu" else x
        dw = products(dz, a)
        got = U.call_linear_backward(kind, dy, xk, w, name, zk, x_name, dw_kind="f32")
        equal(got[1], dw, ("dw", name, x_name))
        equal(got[2], dz.double().sum(0), ("db", name, x_name))
        dx = dz.float() @ w.float()  # at most 2 x 513, exact
        equal(got[0], torch.where(x > 0, dx, torch.zeros_like(dx)) if x_name == "relu" else dx, ("dx", name, x_name))
    got = U.call_linear_backward(kind, dy, x, w, dx=None, dw_kind="f32", accumulate=True, dw=torch.full((n_out, n_in), 3.0, device="cuda"),
                                 db=torch.full((n_out,), -5.0, device="cuda"))
    equal(got[1], products(dy, x) + 3.0, "dw added to")
    equal(got[2], dy.double().sum(0) - 5.0, "db added to")
    got = U.call_linear_backward(kind, dy, None, w, dw=None)
    equal(got[2], dy.double().sum(0), "db without dw")
    equal(U.call_linear_backward(kind, dy, x, w, dx=None, db=None)[1], products(dy, x), "dw in 16 bits")


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n, n_in, n_out", [(16, 777, 100), (17, 40, 130), (16385, 64, 64), (300, 333, 777), (32, 3900, 3700), (4100, 256, 3601), (3001, 777, 1030)])
def test_forward_sums_are_exact(n, n_in, n_out, kind):
    t = U.TYPES[kind][1]
    x, w, b, r = small(1, n, n_in, t=t), small(2, n_out, n_in, t=t), small(3, n_out, t=torch.float32), small(4, n, n_out, t=t)
    want = x.float() @ w.float().t() + b  # at most 4 x 3900, exact in any order
    z, z8 = torch.empty(n, n_out, dtype=t, device="cuda"), U.new8(n, n_out)
    y = U.call_linear(kind, x, w, b, "relu", r, z=z, z8=z8)
    equal(z, want, "z")
    equal(y, want.clamp(min=0) + r, "y")
    q, e = U.store(want.double(), kind)
    assert torch.equal(z8[0], q) and torch.equal(z8[1], e)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, width", [(1, 8), (5000, 16), (5003, 777), (4097, 64), (6145, 2048), (2049, 4097), (513, 8192), (257, 8200), (300, 9001),
                                      ((1 << 24) + 5, 3)])
def test_norm_sums_over_rows_are_exact(n, width, kind):
    t = U.TYPES[kind][1]
    x, dy = small(1, n, width, t=t), small(2, n, width, t=t, most=1)
    mean, rstd = torch.zeros(n, device="cuda"), torch.full((n,), 2.0, device="cuda")  # xh = 2 x
    dg = torch.stack([2 * (dy[:, j].double() * x[:, j].double()).sum() for j in range(width)]) if width < 16 else 2 * (dy.float() * x.float()).sum(0, dtype=torch.float64)
    db = dy.sum(0, dtype=torch.float64)
    for xk in (x, U.call_store(kind, x)):
        for dx in (True, None):
            got = U.call_layer_norm_backward(kind, dy, xk, mean, rstd, dx=dx)
            equal(got[1], dg, "dgamma")
            equal(got[2], db, "dbeta")
    got = U.call_layer_norm_backward(kind, dy, x, mean, rstd, dx=None, dgamma=None, dbeta=torch.full((width,), 3.0, device="cuda"), accumulate=True)
    equal(got[2], db + 3.0, "dbeta added to")


# ---- rows that are not finite --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, width", [(1, 33), (5, 64), (130, 100), (3000, 256), (70, 4100), (40, 9000), (2100, 9000)])
def test_norms_keep_rows_that_are_not_finite_to_themselves(n, width, kind):
    t = U.TYPES[kind][1]
    g = torch.Generator(device="cuda").manual_seed(7)
    x, dy = (torch.randn(n, width, generator=g, device="cuda").to(t) for _ in range(2))
    want8, at, keep = U.new8(n, width), n // 2, torch.arange(n, device="cuda") != n // 2
    want = U.call_layer_norm(kind, x, y8=want8)
    x8 = U.call_store(kind, x)
    back, back8 = (U.call_layer_norm_backward(kind, dy, v, *want[1:]) for v in (x, x8))
    cols = torch.arange(width, device="cuda")
    for bad in (math.nan, math.inf, -math.inf):
        xb = x.clone()
        xb[at, width - 1] = bad
        y8 = U.new8(n, width)
        y, mean, rstd = U.call_layer_norm(kind, xb, y8=y8)
        assert torch.isnan(y[at]).all() and not torch.isfinite(mean[at]) and torch.isnan(rstd[at])
        assert (y8[1][at] == 255).all() and (y8[0][at] == 0).all()
        for got, w in zip((y, mean, rstd, *y8), (*want, *want8)):
            assert torch.equal(got[keep], w[keep])
        # the backward pass of such a row: nothing of it is finite, and the sums are not either
        dx, dg, db = U.call_layer_norm_backward(kind, dy, xb, mean, rstd)
        assert torch.isnan(dx[at]).all() and torch.isnan(dg).all()
        assert torch.equal(dx[keep], back[0][keep]) and torch.equal(db, back[2])
        # of a checkpoint's block alone, with the statistics as they were
        xb8 = U.call_store(kind, xb)
        dx, dg, db = U.call_layer_norm_backward(kind, dy, xb8, *want[1:])
        block = cols // 32 == (width - 1) // 32
        assert torch.isnan(dx[at]).all() and torch.isnan(dg[block]).all()
        assert torch.equal(dx[keep], back8[0][keep]) and torch.equal(dg[~block], back8[1][~block]) and torch.equal(db, back8[2])
        # of a gradient's element
        dyb = dy.clone()
        dyb[at, 3] = bad
        dx, dg, db = U.call_layer_norm_backward(kind, dyb, x, *want[1:])
        assert not torch.isfinite(dx[at]).any() and torch.equal(dx[keep], back[0][keep])
        assert not torch.isfinite(dg[3]) and not torch.isfinite(db[3])
        assert torch.equal(dg[cols != 3], back[1][cols != 3]) and torch.equal(db[cols != 3], back[2][cols != 3])


# what lies past a row's end is no part of its sums: not where a row's mean times rstd leaves fp32's range either (equal values,
# whose rstd is epsilon's alone).  With x = mean the formula is dx = rstd (g - mean(g)) + add.
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n, width", [(1, 1), (5, 8), (3, 33), (300, 40), (4000, 100), (70, 777), (5, 4100), (3, 9001), (2500, 9001)])
def test_norm_backward_of_equal_large_values(n, width, kind):
    t = U.TYPES[kind][1]
    x, dy, add = torch.full((n, width), 2.0 ** 120, device="cuda").to(t), small(1, n, width, t=t), small(2, n, width, t=t)
    mean, rstd = torch.full((n,), 2.0 ** 120, device="cuda"), torch.full((n,), 1024.0, device="cuda")
    dx, dgamma, dbeta = U.call_layer_norm_backward(kind, dy, x, mean, rstd, add=add)
    want = 1024.0 * (dy.double() - dy.double().mean(-1, keepdim=True)) + add.double()
    tol = 1024.0 * 4 * 2.0 ** -23 * 3 + want.abs() * 2 * torch.finfo(t).eps  # sums of whole numbers, one quotient, a few roundings
    assert ((dx.double() - want).abs() <= tol).all()
    assert (dgamma == 0).all()
    equal(dbeta, dy.sum(0, dtype=torch.float64), "dbeta")
    assert torch.equal(U.call_layer_norm_backward(kind, dy, U.call_store(kind, x), mean, rstd, add=add)[0], dx)
