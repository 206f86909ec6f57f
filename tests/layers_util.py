"""The layer operators of libngp_hip.so on torch tensors, and their formulas in 64 bits."""
import ctypes as C
import math

import torch

import ngp_abi as A

TYPES = {"f32": (A.TYPE_F32, torch.float32), "f16": (A.TYPE_F16, torch.float16), "bf16": (A.TYPE_BF16, torch.bfloat16)}
ACTS = ("none", "relu", "logistic", "exponential", "gelu", "silu")
# how far an activation (and a derivative) of the kernels may be off, relative to max(1, |value|): the fitted normal
# distribution is 1.1e-5 off, exp is 2^-23 (1 + |z|) off, |z| <= 40 in these tests: 4.9e-6, and a few roundings
ACT_TOL = 2e-5


def half_step(t):
    return torch.finfo(t).eps / 2


def rounding(ref, t):
    """The most that rounding `ref` to t moves it: half a step, of the smallest number's steps near zero."""
    return ref.abs() * half_step(t) + torch.finfo(t).smallest_normal * half_step(t)


# ---- formulas in 64 bits ---------------------------------------------------------------------------------------------
def act(name, z):
    if name == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), z)
    if name == "logistic":
        return torch.sigmoid(z)
    if name == "exponential":
        return torch.exp(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def act_slope(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "logistic":
        return torch.sigmoid(z) * torch.sigmoid(-z)
    if name == "exponential":
        return torch.exp(z)
    if name == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        return torch.sigmoid(z) * (1 + z * torch.sigmoid(-z))
    return torch.ones_like(z)


def linear_backward(dy, z, x, w, activation="none", x_activation="none", t=None):
    dz = dy * act_slope(activation, z) if activation != "none" else dy
    a = act(x_activation, x)
    if t is not None and x_activation != "none":
        a = a.to(t).double()
    dx = dz @ w
    return dx * act_slope(x_activation, x) if x_activation != "none" else dx, dz.t() @ a, dz.sum(0)


def layer_norm(x, gamma, beta, eps):
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    return (x - mean) * rstd * gamma + beta, mean[:, 0], rstd[:, 0]


def layer_norm_backward(dy, x, mean, rstd, gamma):
    xh = (x - mean[:, None]) * rstd[:, None]
    g = dy * gamma
    dx = rstd[:, None] * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def blocks(width):
    return (width + 31) // 32


def store(v, kind):
    """(q, scale) of the definition; v in 64 bits (float32 exponents: magnitudes from 2^-126)."""
    n, width = v.shape
    f = torch.zeros(n, blocks(width) * 32, dtype=torch.float64, device=v.device)
    f[:, :width] = v
    f = f.view(n, -1, 32)
    top = f.abs().amax(-1)
    scale = (torch.frexp(top)[1] + 126).clamp(min=109 if kind == "f16" else 0)
    scale = torch.where(top == 0, torch.full_like(scale, 109 if kind == "f16" else 0), scale)
    bad = ~torch.isfinite(top)
    q = torch.round(f * torch.exp2((133 - scale).double())[..., None]).clamp(-127, 127)
    q = torch.where(bad[..., None], torch.zeros_like(q), q)
    scale = torch.where(bad, torch.full_like(scale, 255), scale)
    return q.view(n, -1)[:, :width].to(torch.int8), scale.to(torch.uint8)


def load(q, scale):
    """The values in 64 bits."""
    width = q.shape[1]
    s = scale.double().repeat_interleave(32, 1)[:, :width]
    return torch.where(s == 255, torch.full_like(s, math.nan), q.double() * torch.exp2(s - 133))


# ---- calls -----------------------------------------------------------------------------------------------------------
def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def point(args, name, t):
    if t is None:
        return
    if isinstance(t, tuple):
        setattr(args, name, A.Checkpoint8(t[0].data_ptr(), t[1].data_ptr(), t[0].stride(0), t[1].stride(0)))
        return
    setattr(args, name, t.data_ptr())
    if hasattr(args, name + "_stride"):
        setattr(args, name + "_stride", t.stride(0))


def workspace(args, ask, fill=0xFF, device="cuda"):
    """The asked room between guards; a `fill` of 0xFF makes what nobody wrote a NaN."""
    size = C.c_size_t()
    A.check(ask(C.byref(args), C.byref(size)))
    room = torch.full((size.value + 512,), fill, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = room.data_ptr() + 256, size.value
    return room


def guards_hold(room, fill=0xFF):
    return bool((room[:256] == fill).all()) and bool((room[-256:] == fill).all())


class Framed:
    """A matrix inside a larger allocation, `pad` elements wider, with rows before and after: what a call must not touch."""

    def __init__(self, n, width, dtype, pad=0, offset=0, value=7.0, init=None):
        self.n, self.width, self.stride, self.offset = n, width, width + pad, offset
        self.flat = torch.full(((n + 2) * self.stride + offset + 8,), value, dtype=dtype, device="cuda")
        self.t = self.flat[offset:offset + (n + 2) * self.stride].view(n + 2, self.stride)[1:n + 1, :width]
        if init is not None:
            self.t.copy_(init)
        self.before = self.flat.clone()

    def untouched_outside(self):
        frame = self.flat.clone()
        view = frame[self.offset:self.offset + (self.n + 2) * self.stride].view(self.n + 2, self.stride)
        keep = self.before[self.offset:self.offset + (self.n + 2) * self.stride].view(self.n + 2, self.stride)
        view[1:self.n + 1, :self.width] = keep[1:self.n + 1, :self.width]
        return torch.equal(frame.view(torch.uint8), self.before.view(torch.uint8))


def call_linear(kind, x, w, b=None, activation="none", residual=None, y=None, z=None, z8=None):
    code, t = TYPES[kind]
    n, n_in = x.shape
    a = A.LinearArgs(n=n, n_in=n_in, n_out=w.shape[0], type=code, activation=ACTS.index(activation))
    y = torch.empty(n, w.shape[0], dtype=t, device="cuda") if y is None else y
    for name, v in (("x", x), ("weights", w), ("bias", b), ("residual", residual), ("y", y), ("z", z), ("z8", z8)):
        point(a, name, v)
    room = workspace(a, A.load().ngp_linear_workspace)
    A.check(A.load().ngp_linear_forward(C.byref(a), stream()))
    assert guards_hold(room)
    return y


def call_linear_backward(kind, dy, x, w, activation="none", z=None, x_activation="none", dw_kind=None, accumulate=False,
                         dx=True, dw=True, db=True, n_in=None):
    """dx, dw, db: True (made here), a tensor, or None; x and z: a tensor or a checkpoint (q, scale)."""
    code, t = TYPES[kind]
    n, n_out = dy.shape
    n_in = w.shape[1] if n_in is None else n_in
    dw_code, dw_t = TYPES[dw_kind or kind]
    a = A.LinearBackwardArgs(n=n, n_in=n_in, n_out=n_out, type=code, activation=ACTS.index(activation),
                             x_activation=ACTS.index(x_activation), dweights_type=dw_code, accumulate=int(accumulate))
    dx = torch.empty(n, n_in, dtype=t, device="cuda") if dx is True else dx
    dw = torch.empty(n_out, n_in, dtype=dw_t, device="cuda") if dw is True else dw
    db = torch.empty(n_out, dtype=torch.float32, device="cuda") if db is True else db
    point(a, "dy", dy), point(a, "weights", w)
    point(a, "x8" if isinstance(x, tuple) else "x", x)
    point(a, "z8" if isinstance(z, tuple) else "z", z)
    point(a, "dx", dx), point(a, "dweights", dw), point(a, "dbias", db)
    room = workspace(a, A.load().ngp_linear_backward_workspace)
    A.check(A.load().ngp_linear_backward(C.byref(a), stream()))
    assert guards_hold(room)
    return dx, dw, db


def call_layer_norm(kind, x, gamma=None, beta=None, eps=1e-5, y=None, y8=None):
    code, t = TYPES[kind]
    n, width = x.shape
    y = torch.empty(n, width, dtype=t, device="cuda") if y is None else y
    mean, rstd = (torch.empty(n, dtype=torch.float32, device="cuda") for _ in range(2))
    a = A.LayerNormArgs(n=n, width=width, type=code, epsilon=eps)
    for name, v in (("x", x), ("gamma", gamma), ("beta", beta), ("y", y), ("mean", mean), ("rstd", rstd), ("y8", y8)):
        point(a, name, v)
    A.check(A.load().ngp_layer_norm_forward(C.byref(a), stream()))
    return y, mean, rstd


def call_layer_norm_backward(kind, dy, x, mean, rstd, gamma=None, add=None, dx=True, dgamma=True, dbeta=True, accumulate=False):
    code, t = TYPES[kind]
    n, width = dy.shape
    dx = torch.empty(n, width, dtype=t, device="cuda") if dx is True else dx
    dgamma, dbeta = (torch.empty(width, dtype=torch.float32, device="cuda") if d is True else d for d in (dgamma, dbeta))
    a = A.LayerNormBackwardArgs(n=n, width=width, type=code, accumulate=int(accumulate))
    point(a, "x8" if isinstance(x, tuple) else "x", x)
    for name, v in (("dy", dy), ("mean", mean), ("rstd", rstd), ("gamma", gamma), ("dx_add", add), ("dx", dx),
                    ("dgamma", dgamma), ("dbeta", dbeta)):
        point(a, name, v)
    room = workspace(a, A.load().ngp_layer_norm_backward_workspace)
    A.check(A.load().ngp_layer_norm_backward(C.byref(a), stream()))
    assert guards_hold(room)
    return dx, dgamma, dbeta


def new8(n, width, pad=0):
    return (torch.full((n, width + pad), 85, dtype=torch.int8, device="cuda"),
            torch.full((n, blocks(width) + pad), 170, dtype=torch.uint8, device="cuda"))


def call_store(kind, v, c8=None):
    n, width = v.shape
    c8 = new8(n, width) if c8 is None else c8
    c = A.Checkpoint8(c8[0].data_ptr(), c8[1].data_ptr(), c8[0].stride(0), c8[1].stride(0))
    A.check(A.load().ngp_checkpoint_store(C.c_void_p(v.data_ptr()), v.stride(0), n, width, TYPES[kind][0], C.byref(c), stream()))
    return c8


def call_load(kind, c8, width, out=None):
    n = c8[0].shape[0]
    out = torch.empty(n, width, dtype=TYPES[kind][1], device="cuda") if out is None else out
    c = A.Checkpoint8(c8[0].data_ptr(), c8[1].data_ptr(), c8[0].stride(0), c8[1].stride(0))
    A.check(A.load().ngp_checkpoint_load(C.byref(c), n, width, TYPES[kind][0], C.c_void_p(out.data_ptr()), out.stride(0), stream()))
    return out
