"""What apply_rotary, linear_cross_entropy and expert_balance refuse, and what their C entries refuse before any launch."""
import ctypes

import pytest
import torch

from trimkv_b200 import _lib, apply_rotary, build, expert_balance, linear_cross_entropy


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def _rot(q=(1, 2, 3, 8), k=(1, 1, 3, 8), pos=(3,), freq=(4, 2), dt=torch.float32, pdt=torch.int64, fdt=torch.float32, **more):
    return apply_rotary(torch.zeros(q, dtype=dt), None if k is None else torch.zeros(k, dtype=dt), torch.zeros(pos, dtype=pdt),
                        torch.zeros(freq, dtype=fdt), **more)


@pytest.mark.parametrize("kw,error", [
    (dict(layout="interleaved"), ValueError), (dict(q=(2, 3, 8)), ValueError), (dict(k=(2, 1, 3, 8)), ValueError), (dict(k=(1, 1, 4, 8)), ValueError),
    (dict(k=(1, 1, 3, 6)), ValueError), (dict(dt=torch.float64), TypeError), (dict(pdt=torch.float32), TypeError), (dict(pdt=torch.int16), TypeError),
    (dict(pos=(4,)), ValueError), (dict(pos=(2, 3)), ValueError), (dict(pos=(1, 1, 3)), ValueError), (dict(freq=(5, 2)), ValueError),
    (dict(freq=(4,)), ValueError), (dict(freq=(4, 3)), ValueError), (dict(fdt=torch.float64), ValueError)])
def test_rotary_refuses(kw, error):
    with pytest.raises(error):
        _rot(**kw)


def test_rotary_refuses_mixed_types_and_cpu():
    with pytest.raises(TypeError):
        apply_rotary(torch.zeros(1, 1, 1, 8), torch.zeros(1, 1, 1, 8, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64), torch.zeros(4, 2))
    with pytest.raises(_lib.TrimKVNativeError):
        _rot()


@pytest.mark.parametrize("x,w,y,error", [
    (torch.zeros(3, 8), torch.zeros(5, 7), torch.zeros(3, dtype=torch.int64), ValueError),
    (torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64), ValueError),
    (torch.zeros(2, 3, 8), torch.zeros(5, 8), torch.zeros(6, dtype=torch.int64), ValueError),
    (torch.zeros(3, 8), torch.zeros(0, 8), torch.zeros(3, dtype=torch.int64), ValueError),
    (torch.zeros(3, 8), torch.zeros(8), torch.zeros(3, dtype=torch.int64), ValueError),
    (torch.zeros(3, 8), torch.zeros(5, 8).half(), torch.zeros(3, dtype=torch.int64), TypeError),
    (torch.zeros(3, 8).double(), torch.zeros(5, 8).double(), torch.zeros(3, dtype=torch.int64), TypeError),
    (torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3), TypeError),
    (torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64), _lib.TrimKVNativeError)])
def test_linear_cross_entropy_refuses(x, w, y, error):
    with pytest.raises(error):
        linear_cross_entropy(x, w, y)


def test_linear_cross_entropy_refuses_reductions():
    with pytest.raises(ValueError):
        linear_cross_entropy(torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64), reduction="avg")


@pytest.mark.parametrize("z,c,v,error", [
    (torch.zeros(3, 8), torch.zeros(4, 2, dtype=torch.int32), None, ValueError), (torch.zeros(3, 8), torch.zeros(3, dtype=torch.int32), None, ValueError),
    (torch.zeros(3, 0), torch.zeros(3, 2, dtype=torch.int32), None, ValueError), (torch.zeros(3, 8), torch.zeros(3, 2), None, TypeError),
    (torch.zeros(3, 8).double(), torch.zeros(3, 2, dtype=torch.int32), None, TypeError),
    (torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.bool), ValueError),
    (torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3), ValueError),
    (torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int32), None, _lib.TrimKVNativeError)])
def test_expert_balance_refuses(z, c, v, error):
    with pytest.raises(error):
        expert_balance(z, c, v)


def test_c_entries_refuse_before_any_launch(lib):
    buf = ctypes.create_string_buffer(1 << 16)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 255) // 256 * 256)
    rot = lambda q=p, heads=2, batch=1, tokens=3, dim=8, pairs=4, layout=0, dtype=0, pos=p, bits=64, freq=p: lib.tkv_rotary(  # noqa: E731
        q, 48, 8, 16, p, heads, None, 0, 0, 0, None, 0, pos, bits, 3, 1, freq, batch, tokens, dim, pairs, layout, 0, 1.0, dtype, None)
    assert rot(q=None) == rot(pos=None) == rot(freq=None) == -1 and b"NULL" in lib.tkv_last_error()
    assert rot(pairs=5) == rot(pairs=-1) == rot(batch=-1) == rot(tokens=-1) == rot(heads=-1) == -1
    assert rot(dtype=3) == rot(bits=16) == rot(layout=2) == -1
    assert rot(dim=65538) == rot(heads=16385) == -2
    assert rot(batch=0) == rot(tokens=0) == rot(heads=0) == rot(dim=0, pairs=0) == 0           # nothing to do

    need = lambda t=5, v=100, h=16, dt=0, back=0, dx=0: lib.tkv_vloss_workspace_bytes(t, v, h, dt, back, dx)  # noqa: E731
    assert need() > 0 and need(back=1, dx=1) > need(back=1) > 0
    assert need(t=-1) == need(v=0) == need(h=0) == need(dt=3) == need(t=(1 << 24) + 1) == need(v=(1 << 23) + 1) == need(h=65537) == -1
    assert lib.tkv_vloss_plan_words(5) == 29
    fwd = lambda x=p, stride=16, t=5, v=100, h=16, red=1, loss=p, out=p, plan=p, ws=p, n=1 << 15, dt=0: lib.tkv_vloss_forward(  # noqa: E731
        x, stride, p, p, -100, t, v, h, red, loss, out, plan, ws, n, dt, None, None)
    assert fwd(x=None) == fwd(loss=None) == fwd(out=None) == fwd(plan=None) == fwd(ws=None) == -1 and b"NULL" in lib.tkv_last_error()
    assert fwd(stride=15) == fwd(red=3) == fwd(t=-1) == fwd(v=0) == fwd(h=0) == fwd(dt=3) == -1
    assert fwd(n=need() - 1) == -1 and b"workspace" in lib.tkv_last_error()
    assert fwd(ws=ctypes.c_void_p(p.value + 4)) == -1
    assert fwd(t=1 << 25) == fwd(v=1 << 24) == fwd(t=1 << 22, v=1 << 22) == -2
    assert fwd(plan=ctypes.c_void_p(p.value + 4)) == -1 and b"aligned" in lib.tkv_last_error()
    bwd = lambda x=p, w=p, t=5, v=100, h=16, red=0, dx=p, dw=p, n=1 << 25, grad=p: lib.tkv_vloss_backward(  # noqa: E731
        x, 16, w, p, grad, 1, red, t, v, h, dx, dw, p, n, 0, None, None)
    assert bwd(x=None) == bwd(w=None) == bwd(grad=None) == bwd(dx=None, dw=None) == -1 and b"NULL" in lib.tkv_last_error()
    assert bwd(n=16) == bwd(red=-1) == bwd(t=-1) == bwd(dx=ctypes.c_void_p(p.value + 2)) == -1
    assert bwd(t=0, dw=None) == 0                                                              # nothing to do

    bal = lambda z=p, c=p, t=5, e=16, top=2, bits=32, loss=p, ws=p, n=1 << 15, dt=2: lib.tkv_moe_balance(  # noqa: E731
        z, 16, c, 2, bits, None, 0, t, e, top, loss, p, p, ws, n, dt, None)
    assert bal(z=None) == bal(c=None) == bal(loss=None) == bal(ws=None) == -1 and b"NULL" in lib.tkv_last_error()
    assert bal(t=-1) == bal(e=0) == bal(top=-1) == bal(bits=8) == bal(dt=3) == bal(n=8) == -1
    assert bal(e=1025) == bal(top=1025) == bal(t=1 << 30, top=8) == -2
    grad = lambda z=p, g=p, t=5, e=16, dt=2: lib.tkv_moe_balance_grad(z, 16, None, 0, p, g, t, e, p, 16, dt, None)  # noqa: E731
    assert grad(z=None) == grad(g=None) == grad(t=-1) == grad(e=0) == grad(dt=3) == -1 and grad(e=1025) == -2 and grad(t=0) == 0
