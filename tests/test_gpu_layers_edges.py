"""Activations of the linear layers over every value of their 16-bit types.

A result lies between the formula's value minus its bound and that plus its bound, both rounded to the output's type.  The
bounds are those of the evaluation in fp32, term by term:
 * exp: 2^x of x log2(e), off by 2^-23 (1 + |x|) relative; the logistic s = 1 / (1 + exp(-z)): 1 - s of that, and two roundings;
 * silu and both slopes: products of these; 1 - s next to 1 is off by 2^-21 of 1, 0 past z = 17.4 where z exp(-z) < 2^-20;
 * gelu: its tail |z| Phi(-|z|) by 1.2e-5 relative up to |z| = 8 and 5e-15 past it, its slope by 4e-7;
 * what the hardware's 2^x and 1/x flush: 2^-126, times |z| where z multiplies it.
"""
import math

import pytest
import torch

import layers_util as U

pytestmark = pytest.mark.gpu

E = 2.0 ** -23
FLUSH = 2.0 ** -126


def every_value(t):
    """All 65536 bit patterns of a 16-bit type, [1][65536]."""
    return torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(t).view(1, -1)


def phi(z):
    """The normal distribution function, relatively exact far below zero too (1 + erf loses its digits there)."""
    return torch.special.erfc(z * -math.sqrt(0.5)) / 2


def value(name, z):
    return z * phi(z) if name == "gelu" else U.act(name, z)


def slope(name, z):
    return phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi) if name == "gelu" else U.act_slope(name, z)


def logistic_error(z):
    s, r, a = torch.sigmoid(z), torch.sigmoid(-z), z.abs().clamp(max=1e6)
    return s * E * (2.5 + r * (1 + a))


def value_error(name, z):
    v, a = value(name, z), z.abs()
    if name in ("none", "relu"):
        return torch.zeros_like(z)
    if name == "exponential":
        return v * E * (1 + a.clamp(max=200)) * 1.01 + FLUSH
    if name == "logistic":
        return logistic_error(z) + FLUSH
    if name == "silu":
        return a * (logistic_error(z) + FLUSH) + v.abs() * E
    tail = a * phi(-a)
    return 1.2e-5 * tail + v.abs() * E + torch.where(a > 8, 5e-15, 0.0)


def slope_error(name, z):
    v, a, s = slope(name, z), z.abs(), torch.sigmoid(z)
    if name in ("none", "relu"):
        return torch.zeros_like(z)
    if name == "exponential":
        return v * E * (1 + a.clamp(max=200)) * 1.01 + FLUSH
    if name == "logistic":
        return logistic_error(z) * torch.sigmoid(-z) + logistic_error(-z) * s + v * E + FLUSH
    if name == "silu":
        b = a.clamp(max=1e6)
        return torch.where(z < 0, 2 * E * (3 + b) * (1 + b) * s + FLUSH * (1 + a), 2.0 ** -21 * (1 + a.clamp(max=18)))
    return torch.full_like(z, 4e-7)


def between(got, want, error, t, what):
    finite = torch.isfinite(want)
    error = torch.where(finite, error, torch.zeros_like(error)) + torch.where(finite, want.abs() * 2.0 ** -24, 0.0)
    low, high = (want - error).to(t).double(), (want + error).to(t).double()
    got = got.double()
    bad = ~((low <= got) & (got <= high))
    if bad.any():
        i = tuple(v[0] for v in torch.nonzero(bad, as_tuple=True))
        raise AssertionError((what, int(bad.sum()), float(got[i]), float(low[i]), float(high[i]), [int(k) for k in i]))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("name", U.ACTS)
def test_activations_of_every_value(name, kind):
    t = U.TYPES[kind][1]
    w = every_value(t)
    z, plain = w.double(), torch.isfinite(w)
    # forward: z = 1 w, by the kernel of a few rows and by the product
    for n in (1, 40):
        y = U.call_linear(kind, torch.ones(n, 1, dtype=t, device="cuda"), w.view(-1, 1), None, name)
        assert torch.equal(y[0].view(torch.int16)[plain[0]], y[-1].view(torch.int16)[plain[0]])
        between(y[:1][plain], value(name, z)[plain], value_error(name, z)[plain], t, (name, n))
        nan, pos, neg = y[0, torch.isnan(z[0])], float(y[0, z[0] == math.inf]), float(y[0, z[0] == -math.inf])
        assert torch.isnan(nan).all()
        assert pos == (1.0 if name == "logistic" else math.inf)
        if name == "none":
            assert neg == -math.inf
        elif name in ("relu", "logistic", "exponential"):
            assert neg == 0.0
        else:
            assert math.isnan(neg) or neg == 0.0  # -inf times 0, or the limit
    # the slope in fp32: db = act'(z) of a single row
    if name != "none":
        got = U.call_linear_backward(kind, torch.ones(1, 65536, dtype=t, device="cuda"), None, None, name, w, dx=None, dw=None, n_in=1)[2]
        between(got[plain[0]], slope(name, z)[plain], slope_error(name, z)[plain], torch.float32, (name, "slope"))
        assert name == "relu" or torch.isnan(got[torch.isnan(z[0])]).all()
        pos, neg = float(got[z[0] == math.inf]), float(got[z[0] == -math.inf])
        limit = {"relu": 1.0, "logistic": 0.0, "exponential": math.inf}.get(name, 1.0)
        assert pos == limit or (name in ("gelu", "silu") and math.isnan(pos))
        assert neg == 0.0 or (name in ("gelu", "silu") and math.isnan(neg))
        # as the activation below: dx = act'(p), dW = act(p) rounded to the type
        dx, dw, _ = U.call_linear_backward(kind, torch.ones(1, 1, dtype=t, device="cuda"), w, torch.ones(1, 65536, dtype=t, device="cuda"),
                                           x_activation=name, db=None)
        between(dx[plain], slope(name, z)[plain], slope_error(name, z)[plain], t, (name, "dx"))
        between(dw[plain], value(name, z)[plain], value_error(name, z)[plain], t, (name, "dw"))


@pytest.mark.parametrize("n", [3, 40, 300])
def test_checkpoints_of_sums_beyond_the_type(n):
    """z8 and y8 are kept from fp32: past float16's range they are infinite as float16, and what they are for a slope."""
    x, w = torch.full((n, 64), 1000.0, dtype=torch.float16, device="cuda"), torch.full((40, 64), 16.0, dtype=torch.float16, device="cuda")
    w[1::2] *= -1
    z8 = U.new8(n, 40)
    y = U.call_linear("f16", x, w, None, "none", z8=z8)
    z = 1000.0 * 16 * 64 * torch.tensor([1.0, -1.0], device="cuda").repeat(n, 20)
    assert torch.equal(y.float(), z * math.inf)
    q, e = U.store(z.double(), "f16")
    assert torch.equal(z8[0], q) and torch.equal(z8[1], e) and (e == 127 + 19).all()  # 2^19 < 1024000 < 2^20
    assert torch.equal(U.call_load("f32", z8, 40).double(), U.load(q, e))
    assert torch.equal(U.call_load("f16", z8, 40).float(), z * math.inf)
    dy = torch.ones(n, 40, dtype=torch.float16, device="cuda")
    for name in ("relu", "gelu", "silu", "logistic"):
        _, dw, db = U.call_linear_backward("f16", dy, torch.ones_like(x), w, name, z8, dx=None, dw_kind="f32")
        slope_ = torch.zeros(40, device="cuda") if name == "logistic" else (z[0] > 0).float()
        assert torch.equal(db, n * slope_) and torch.equal(dw, (n * slope_)[:, None].expand(40, 64))
    # a norm's y8, with a gain that leaves the type
    v = torch.tensor([1.0, -1.0], dtype=torch.float16, device="cuda").repeat(n, 32)
    y8 = U.new8(n, 64)
    y, mean, rstd = U.call_layer_norm("f16", v, torch.full((64,), 1e6, device="cuda"), eps=0.0, y8=y8)
    assert torch.equal(y.float(), v.float() * math.inf) and (mean == 0).all() and (rstd == 1).all()
    q, e = U.store(v.double() * 1e6, "f16")
    assert torch.equal(y8[0], q) and torch.equal(y8[1], e)
    dx, dgamma, dbeta = U.call_layer_norm_backward("f16", torch.ones_like(v), y8, mean, torch.full((n,), 2.0 ** -20, device="cuda"))
    assert torch.isfinite(dx).all() and torch.equal(dgamma.double(), n * 2.0 ** -20 * U.load(q, e)[0]) and (dbeta == n).all()
