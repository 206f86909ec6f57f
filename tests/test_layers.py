"""Layers of any width, on the CPU: what the calls refuse (before any GPU work), the argument blocks' layout against the
header, and the 64-bit formulas against differences."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import layers_util as U
import ngp_abi as A

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HERE = 1 << 40  # an address that no call reaches: every case is refused first


def refused(status, text):
    assert status == 1, status
    assert text in A.load().ngp_last_error().decode()


def linear(**kw):
    a = A.LinearArgs(n=4, n_in=8, n_out=16, type=A.TYPE_F16, x=HERE, x_stride=8, weights=HERE * 2, weights_stride=8,
                     y=HERE * 3, y_stride=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def backward(**kw):
    a = A.LinearBackwardArgs(n=4, n_in=8, n_out=16, type=A.TYPE_F16, dweights_type=A.TYPE_F16, dy=HERE, dy_stride=16,
                             x=HERE * 2, x_stride=8, weights=HERE * 3, weights_stride=8, dx=HERE * 4, dx_stride=8,
                             dweights=HERE * 5, dweights_stride=8)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def norm(**kw):
    a = A.LayerNormArgs(n=4, width=40, type=A.TYPE_F32, epsilon=1e-5, x=HERE, x_stride=40, y=HERE * 2, y_stride=40)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def norm_backward(**kw):
    a = A.LayerNormBackwardArgs(n=4, width=40, type=A.TYPE_F32, dy=HERE, dy_stride=40, x=HERE * 2, x_stride=40,
                                mean=HERE * 3, rstd=HERE * 4, dx=HERE * 5, dx_stride=40)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


EIGHT = A.Checkpoint8(HERE * 6, HERE * 7, 64, 2)


@pytest.mark.parametrize("kw, text", [
    (dict(type=A.TYPE_F32), "NGP_TYPE_F16"), (dict(type=9), "NGP_TYPE_F16"), (dict(activation=6), "NGP_ACT"),
    (dict(activation=-1), "NGP_ACT"), (dict(n=(1 << 29) + 1), "rows"), (dict(n_in=0), "widths"), (dict(n_out=0), "widths"),
    (dict(n_in=65537), "widths"), (dict(x=None), "null"), (dict(weights=None), "null"), (dict(y=None), "null"),
    (dict(x=HERE + 1), "aligned"), (dict(x_stride=7), "stride"), (dict(weights_stride=1 << 22), "stride"),
    (dict(y_stride=15), "stride"), (dict(residual=HERE * 9, residual_stride=3), "stride"),
    (dict(z=HERE * 9, z_stride=3), "stride"), (dict(bias=HERE + 2), "aligned"),
    (dict(z8=A.Checkpoint8(HERE, None, 16, 1)), "both q and scale"), (dict(z8=A.Checkpoint8(HERE, HERE, 15, 1)), "q_stride"),
    (dict(z8=A.Checkpoint8(HERE, HERE, 16, 0)), "scale_stride"), (dict(y=HERE), "must not be"),
    (dict(z=HERE * 3, z_stride=16), "must not be"), (dict(z=HERE, z_stride=16), "must not be"),
    (dict(residual=HERE * 3, residual_stride=24), "stride"),
])
def test_linear_refuses(kw, text):
    size = C.c_size_t()
    a = linear(**kw)
    refused(A.load().ngp_linear_forward(C.byref(a), None), text)
    refused(A.load().ngp_linear_workspace(C.byref(a), C.byref(size)), text)


@pytest.mark.parametrize("kw, text", [
    (dict(type=A.TYPE_F32), "NGP_TYPE_F16"), (dict(activation=6), "NGP_ACT"), (dict(x_activation=-1), "NGP_ACT"),
    (dict(n=(1 << 29) + 1), "rows"), (dict(n_in=0), "widths"), (dict(n_out=1 << 20), "widths"), (dict(accumulate=2), "accumulate"),
    (dict(dweights_type=A.TYPE_BF16), "dweights_type"), (dict(accumulate=1), "NGP_TYPE_F32 only"), (dict(dy=None), "null"),
    (dict(activation=A.ACT_GELU), "needs z or z8"), (dict(x=None), "needs x or x8"), (dict(weights=None), "needs the weights"),
    (dict(x=None, dweights=None, x_activation=A.ACT_RELU), "needs x or x8"), (dict(x8=EIGHT), "not in both"),
    (dict(z=HERE * 9, z_stride=16, z8=EIGHT), "not in both"), (dict(dy_stride=8), "stride"), (dict(dx_stride=7), "stride"),
    (dict(dweights=HERE + 1), "aligned"), (dict(dbias=HERE + 1), "aligned"), (dict(dx=HERE), "must not be"),
    (dict(dweights=HERE * 4), "must not be"), (dict(dweights=HERE * 2), "must not be"),
])
def test_linear_backward_refuses(kw, text):
    size = C.c_size_t()
    a = backward(**kw)
    refused(A.load().ngp_linear_backward(C.byref(a), None), text)
    refused(A.load().ngp_linear_backward_workspace(C.byref(a), C.byref(size)), text)


@pytest.mark.parametrize("kw, text", [
    (dict(type=3), "NGP_TYPE"), (dict(n=(1 << 29) + 1), "rows"), (dict(width=0), "widths"), (dict(width=65537), "widths"),
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(epsilon=-1.0), "epsilon"), (dict(epsilon=float("nan")), "epsilon"),
    (dict(x=HERE + 2), "aligned"), (dict(x_stride=39), "stride"), (dict(y_stride=1 << 22), "stride"),
    (dict(gamma=HERE + 1), "aligned"), (dict(mean=HERE + 2), "aligned"), (dict(y=HERE), "must not be"),
    (dict(y8=A.Checkpoint8(HERE, HERE, 40, 1)), "scale_stride"),
])
def test_layer_norm_refuses(kw, text):
    refused(A.load().ngp_layer_norm_forward(C.byref(norm(**kw)), None), text)


@pytest.mark.parametrize("kw, text", [
    (dict(type=-1), "NGP_TYPE"), (dict(width=0), "widths"), (dict(accumulate=-1), "accumulate"), (dict(dy=None), "null"),
    (dict(x=None), "null"), (dict(x8=EIGHT), "not in both"), (dict(mean=None), "null"), (dict(rstd=None), "null"),
    (dict(dx=HERE), "must not be"), (dict(dx=HERE * 2), "must not be"), (dict(dx_add=HERE * 5, dx_add_stride=48), "stride"),
    (dict(dgamma=HERE * 8, dbeta=HERE * 8), "must not be"), (dict(dx_stride=8), "stride"),
])
def test_layer_norm_backward_refuses(kw, text):
    size = C.c_size_t()
    a = norm_backward(**kw)
    refused(A.load().ngp_layer_norm_backward(C.byref(a), None), text)
    refused(A.load().ngp_layer_norm_backward_workspace(C.byref(a), C.byref(size)), text)


@pytest.mark.parametrize("values, stride, n, width, kind, c, text", [
    (HERE, 40, 4, 40, 3, A.Checkpoint8(HERE, HERE, 40, 2), "NGP_TYPE"),
    (HERE, 40, (1 << 29) + 1, 40, 0, A.Checkpoint8(HERE, HERE, 40, 2), "rows"),
    (HERE, 40, 4, 0, 0, A.Checkpoint8(HERE, HERE, 40, 2), "widths"),
    (None, 40, 4, 40, 0, A.Checkpoint8(HERE, HERE, 40, 2), "null"),
    (HERE, 40, 4, 40, 0, A.Checkpoint8(None, None, 40, 2), "null"),
    (HERE, 39, 4, 40, 0, A.Checkpoint8(HERE, HERE, 40, 2), "stride"),
    (HERE + 2, 40, 4, 40, 0, A.Checkpoint8(HERE, HERE, 40, 2), "aligned"),
    (HERE, 40, 4, 40, 0, A.Checkpoint8(HERE, HERE, 39, 2), "q_stride"),
    (HERE, 40, 4, 40, 0, A.Checkpoint8(HERE, HERE, 40, 1), "scale_stride"),
])
def test_checkpoints_refuse(values, stride, n, width, kind, c, text):
    refused(A.load().ngp_checkpoint_store(values, stride, n, width, kind, C.byref(c), None), text)
    refused(A.load().ngp_checkpoint_load(C.byref(c), n, width, kind, values, stride, None), text)


def test_null_arguments_and_small_workspaces_are_refused():
    lib, size = A.load(), C.c_size_t()
    refused(lib.ngp_linear_forward(None, None), "null")
    refused(lib.ngp_linear_backward(None, None), "null")
    refused(lib.ngp_layer_norm_forward(None, None), "null")
    refused(lib.ngp_layer_norm_backward(None, None), "null")
    refused(lib.ngp_linear_workspace(C.byref(linear()), None), "null")
    refused(lib.ngp_checkpoint_store(HERE, 40, 4, 40, 0, None, None), "null")
    for call, ask, a in [
        (lib.ngp_linear_backward, lib.ngp_linear_backward_workspace,
         backward(n=5000, dbias=HERE * 8, activation=A.ACT_SILU, z=HERE * 9, z_stride=16)),
        (lib.ngp_layer_norm_backward, lib.ngp_layer_norm_backward_workspace, norm_backward(n=5000, dgamma=HERE * 8)),
    ]:
        assert ask(C.byref(a), C.byref(size)) == 0 and size.value > 0
        refused(call(C.byref(a), None), "workspace")
        a.workspace, a.workspace_bytes = HERE * 16, size.value - 1
        refused(call(C.byref(a), None), "workspace")
        a.workspace, a.workspace_bytes = HERE * 16 + 8, size.value
        refused(call(C.byref(a), None), "16-byte")


@pytest.mark.parametrize("struct, cls", [("ngp_checkpoint8", A.Checkpoint8), ("ngp_linear_args", A.LinearArgs),
                                         ("ngp_linear_backward_args", A.LinearBackwardArgs),
                                         ("ngp_layer_norm_args", A.LayerNormArgs),
                                         ("ngp_layer_norm_backward_args", A.LayerNormBackwardArgs)])
def test_argument_blocks_match_the_header(struct, cls, tmp_path):
    src = tmp_path / "offsets.c"
    prints = "".join(f'printf("%zu ", offsetof({struct}, {f[0]}));' for f in cls._fields_)
    src.write_text(f'#include <stdio.h>\n#include "ngp_hip.h"\nint main(void) {{ {prints} printf("%zu", sizeof({struct})); }}')
    exe = str(tmp_path / "offsets")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe])
    want = [int(v) for v in subprocess.check_output([exe]).split()]
    assert want == [getattr(cls, f[0]).offset for f in cls._fields_] + [C.sizeof(cls)]


def differences(f, v, h=1e-5):
    """df/dv of a scalar function by central differences, in 64 bits."""
    g = torch.zeros_like(v)
    for k in range(v.numel()):
        w = v.clone().reshape(-1)
        w[k] += h
        up = f(w.view_as(v))
        w[k] -= 2 * h
        g.view(-1)[k] = (up - f(w.view_as(v))) / (2 * h)
    return g


@pytest.mark.parametrize("name", U.ACTS)
def test_the_linear_formulas_are_the_derivatives(name):
    torch.manual_seed(3)
    x, w, b, dy = (torch.randn(s, dtype=torch.float64) for s in ((5, 4), (3, 4), (3,), (5, 3)))
    x = x + 0.05 * x.sign()  # relu's corner stays further away than the differences reach

    def loss(x, w, b):
        return (dy * U.act(name, U.act(name, x) @ w.t() + b)).sum()

    z = U.act(name, x) @ w.t() + b
    assert z.abs().min() > 1e-3
    dx, dw, db = U.linear_backward(dy, z, x, w, name, name)
    # central differences: h^2 / 6 of a third derivative (below 1e3 here) and 2^-53 |loss| / h: 1e-8 and 1e-10
    for got, f, v in ((dx, lambda v: loss(v, w, b), x), (dw, lambda v: loss(x, v, b), w), (db, lambda v: loss(x, w, v), b)):
        assert torch.allclose(got, differences(f, v), rtol=1e-6, atol=1e-6)


def test_the_norm_formulas_are_the_derivatives():
    torch.manual_seed(4)
    x, gamma, beta, dy = (torch.randn(s, dtype=torch.float64) for s in ((4, 7), (7,), (7,), (4, 7)))

    def loss(x, gamma, beta):
        return (dy * U.layer_norm(x, gamma, beta, 1e-3)[0]).sum()

    _, mean, rstd = U.layer_norm(x, gamma, beta, 1e-3)
    dx, dg, db = U.layer_norm_backward(dy, x, mean, rstd, gamma)
    for got, f, v in ((dx, lambda v: loss(v, gamma, beta), x), (dg, lambda v: loss(x, v, beta), gamma),
                      (db, lambda v: loss(x, gamma, v), beta)):
        assert torch.allclose(got, differences(f, v), rtol=1e-6, atol=1e-6)


def test_the_checkpoint_definition():
    v = torch.tensor([[1.0, -1.99, 0.5, 2 ** -7, 3 * 2 ** -8] + [0.0] * 27, [127.4, -127.6, 64.5, 65.5, 0.49] + [0.0] * 27],
                     dtype=torch.float64)
    q, e = U.store(v, "f32")
    assert e.tolist() == [[127], [133]]
    assert q[0, :5].tolist() == [64, -127, 32, 0, 1] and q[1, :5].tolist() == [127, -127, 64, 66, 0]
    assert torch.equal(U.load(q, e)[0, :3], torch.tensor([1.0, -127 / 64, 0.5], dtype=torch.float64))
    bad = torch.zeros(1, 40, dtype=torch.float64)
    bad[0, 33] = float("inf")
    q, e = U.store(bad, "bf16")
    assert e.tolist() == [[0, 255]] and torch.isnan(U.load(q, e)[0, 32:]).all() and (U.load(q, e)[0, :32] == 0).all()
