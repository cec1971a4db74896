"""gact.fused without a GPU: what the operators refuse before anything is launched, on the Python side and in the C ABI."""
import ctypes

import pytest
import torch


def buf():
    b = ctypes.create_string_buffer(1 << 16)
    return b, (ctypes.addressof(b) + 255) & ~255


def test_checkpoint_abi_refusals():
    from gact import _native as nv
    L = nv.lib
    b, p = buf()
    assert [L.gact_checkpoint8_pitch(n) for n in (0, 1, 32, 33, -1)] == [0, 32, 32, 64, -1]
    f = L.gact_checkpoint8
    assert f(p, 3, 2, 32, 32, 0, 0, p, p, None) == 2                  # dtype
    assert f(p, 0, -1, 32, 32, 0, 0, p, p, None) == 5                 # rows
    assert f(p, 0, 2, 32, 31, 0, 0, p, p, None) == 5                  # pitch shorter than a row
    assert f(p, 0, 2, 1 << 25, 1 << 25, 0, 0, p, p, None) == 5        # row too long
    assert f(p, 0, 1 << 35, 32, 32, 0, 0, p, p, None) == 5            # too many elements
    assert f(None, 0, 2, 32, 32, 0, 0, p, p, None) == 3
    assert f(p, 0, 2, 32, 32, 0, 0, p, None, None) == 3
    assert f(p + 2, 0, 2, 32, 32, 0, 0, p, p, None) == 4
    assert f(p, 0, 2, 32, 32, 0, 0, p + 16, p, None) == 4             # codes not on 32 bytes
    assert f(p, 0, 0, 32, 32, 0, 0, None, None, None) == 0
    g = L.gact_restore8
    assert g(p, p, 2, 32, 5, p, 32, None) == 2 and g(p, p, 2, 32, 0, p, 8, None) == 5 and g(p, None, 2, 32, 0, p, 32, None) == 3
    assert g(p, p, 2, 32, 1, p + 1, 32, None) == 4 and g(None, None, 0, 32, 1, None, 32, None) == 0
    h = L.gact_repitch16
    assert h(p, 4, 2, 8, p, 8, None) == 5 and h(p, 8, 2, 8, None, 8, None) == 3 and h(p + 1, 8, 2, 8, p, 8, None) == 4


def test_layer_norm_abi_refusals():
    from gact import _native as nv
    L = nv.lib
    b, p = buf()
    f = lambda x=p, dt=2, rows=2, cols=32, ld=32, w=p, bias=p, pdt=2, y=p, stats=p, codes=p, scales=p: L.gact_layer_norm(
        x, dt, rows, cols, ld, w, bias, pdt, 1e-5, y, stats, codes, scales, 0, 0, None)
    assert f(dt=4) == 2 and f(pdt=1) == 2 and f(dt=0, pdt=2) == 2
    assert f(rows=-1) == 5 and f(cols=0) == 5 and f(cols=16385, ld=16385) == 5 and f(ld=31) == 5
    assert f(x=None) == 3 and f(y=None) == 3 and f(scales=None) == 3
    assert f(x=p + 1) == 4 and f(y=p + 1) == 4 and f(codes=p + 16) == 4 and f(stats=p + 4) == 4 and f(w=p + 1) == 4 and f(bias=p + 2, pdt=0) == 4
    assert f(rows=0, x=None) == 0
    assert L.gact_layer_norm_backward_scratch_bytes(-1, 32) == -1 and L.gact_layer_norm_backward_scratch_bytes(1, 20000) == -1
    g = lambda dy=p, dt=2, rows=2, cols=32, ld=32, x=None, ldx=32, codes=p, scales=p, stats=p, w=p, pdt=2, dx=p, dw=p, db=p, scr=p: \
        L.gact_layer_norm_backward(dy, dt, rows, cols, ld, x, ldx, codes, scales, stats, w, pdt, dx, dw, db, scr, None)
    assert g(dt=7) == 2 and g(cols=0) == 5 and g(ld=8) == 5 and g(x=p, ldx=8) == 5
    assert g(dy=None) == 3 and g(codes=None) == 3 and g(scales=None) == 3 and g(stats=None) == 3 and g(scr=None) == 3
    assert g(dy=p + 1) == 4 and g(codes=p + 8) == 4 and g(scr=p + 4) == 4 and g(dx=p + 1) == 4
    assert g(dx=None, dw=None, db=None) == 0


def test_linear_abi_refusals():
    from gact import _native as nv
    L = nv.lib
    b, p = buf()
    f = lambda x=p, ldx=64, w=p, ldw=64, bias=p, res=p, ldr=32, dt=2, rows=4, cin=64, cout=32, act=2, y=p, xc=p, xs=p, z=None, zc=p, zs=p, scr=p: \
        L.gact_linear(x, ldx, w, ldw, bias, res, ldr, dt, rows, cin, cout, act, y, xc, xs, z, zc, zs, 0, 0, scr, None)
    assert f(dt=0) == 2 and f(dt=3) == 2 and f(act=5) == 6 and f(act=-1) == 6
    assert f(rows=-1) == 5 and f(cin=0) == 5 and f(cout=0) == 5 and f(ldx=63) == 5 and f(ldw=8) == 5 and f(ldr=31) == 5
    assert f(cin=1 << 25, ldx=1 << 25, ldw=1 << 25) == 5 and f(rows=1 << 31) == 5
    assert f(x=None) == 3 and f(w=None) == 3 and f(y=None) == 3 and f(zs=None) == 3 and f(xs=None) == 3
    assert f(x=p + 2) == 4 and f(ldx=65) == 4 and f(w=p + 8) == 4 and f(ldw=68) == 4 and f(y=p + 1) == 4 and f(zc=p + 16) == 4 and f(scr=p + 16) == 4
    assert f(bias=p + 1) == 4 and f(res=p + 1) == 4 and f(xc=p + 16) == 4
    assert f(rows=0, x=None) == 0
    d = lambda dz=p, ldz=32, w=p, ldw=64, dt=2, rows=4, cin=64, cout=32, dx=p, part=p, db=p, xc=p, xs=p, xr=p, scr=p: \
        L.gact_linear_dgrad(dz, ldz, w, ldw, dt, rows, cin, cout, dx, part, db, xc, xs, xr, scr, None)
    assert d(dt=0) == 2 and d(ldz=31) == 5 and d(dz=None) == 3 and d(dx=None) == 3 and d(dz=p + 4) == 4 and d(ldz=36) == 4 and d(rows=0, dz=None) == 0
    assert d(part=None) == 3 and d(db=None) == 3 and d(xc=None) == 3 and d(xs=None) == 3 and d(xr=p + 8) == 4 and d(db=p + 1) == 4 and d(part=p + 2) == 4
    e = lambda dz=p, ldz=32, x=p, ldx=64, dt=2, rows=4, cin=64, cout=32, dw=p, part=p, db=p, scr=p: \
        L.gact_linear_wgrad(dz, ldz, x, ldx, dt, rows, cin, cout, dw, part, db, scr, None)
    assert e(dt=0) == 2 and e(ldx=8) == 5 and e(x=None) == 3 and e(dw=None) == 3 and e(x=p + 4) == 4 and e(ldx=65) == 4
    assert e(part=None) == 3 and e(db=None) == 3 and e(db=p + 1) == 4
    g = lambda dy=p, dt=2, rows=4, cols=32, ld=32, act=2, z=None, ldz=32, zc=p, zs=p, dz=p, ldo=32, db=p, scr=p: L.gact_act_backward(
        dy, dt, rows, cols, ld, act, z, ldz, zc, zs, dz, ldo, db, scr, None)
    assert g(dt=0) == 2 and g(act=9) == 6 and g(cols=0) == 5 and g(ld=8) == 5 and g(ldo=8) == 5 and g(z=p, ldz=8) == 5
    assert g(dy=None) == 3 and g(dz=None) == 3 and g(zc=None) == 3 and g(scr=None) == 3 and g(zc=p + 8) == 4 and g(dy=p + 1) == 4
    assert g(act=0, db=None, scr=None, dz=None) == 0 and g(rows=0, db=None, dy=None) == 0
    assert L.gact_linear_scratch_bytes(4, 0, 32, 0) == -1 and L.gact_linear_scratch_bytes(4, 8, 8, 3) == -1 and L.gact_linear_scratch_bytes(0, 8, 8, 0) == 0


def test_python_refuses_host_tensors_and_wrong_arguments():
    from gact import fused
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    for call in (lambda: fused.op_checkpoint8(x), lambda: fused.op_layer_norm(x), lambda: fused.op_linear(x, w)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    with pytest.raises(TypeError):
        fused.op_restore8([x])
    c = fused.Checkpoint8(torch.zeros(4 * 33, dtype=torch.int8), (4, 8), torch.bfloat16)
    assert c.codes.shape == (4, 32) and c.scales.shape == (4, 1) and c.nbytes == 132
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fused.op_restore8(c)
    with pytest.raises(RuntimeError, match="type"):
        fused.op_restore8(c, torch.float64)


def test_convert_on_the_host():
    import torch.nn as nn
    from gact import layers

    class Own(nn.Linear):
        pass

    m = nn.Sequential(nn.Linear(4, 8), nn.ReLU(), nn.Sequential(nn.LayerNorm(8), nn.Linear(8, 8, bias=False)), nn.GELU(), Own(8, 2))
    hooked = nn.Linear(2, 2)
    hooked.register_forward_hook(lambda *a: None)
    m.append(hooked)
    params = list(m.parameters())
    keys = list(m.state_dict())
    layers.convert(m)
    assert all(a is b for a, b in zip(params, m.parameters())) and list(m.state_dict()) == keys
    assert m[0].activation == "relu" and isinstance(m[1], nn.Identity) and type(m[2][0]) is layers.LayerNorm
    assert m[2][1].bias is None and m[2][1].activation is None and isinstance(m[3], nn.GELU)      # not in one Sequential
    assert type(m[4]) is Own and m[5] is hooked
    assert type(layers.convert(nn.Linear(2, 2))) is layers.Linear
    with pytest.raises(RuntimeError, match="autocast"):
        m[0](torch.zeros(2, 4))


@pytest.mark.parametrize("shape, size", [((5,), (3, 7)), ((4, 6), (2, 6, 4)), ((4, 6), (24,)), ((2, 3), (6, 2, 4)), ((1,), ())])
def test_layer_norm_module_refuses_other_shapes(shape, size):
    """As nn.LayerNorm does, with and without parameters: an equal number of elements is not enough."""
    from gact import layers
    for affine in (True, False):
        with pytest.raises(RuntimeError, match="normalized_shape"):
            layers.LayerNorm(shape, elementwise_affine=affine)(torch.zeros(size))


def test_autocast_leaves_doubles_alone(monkeypatch):
    """As torch does: they are refused, not lowered to 16 bits."""
    from gact import layers
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda device: True)
    x = torch.zeros(2, 4, dtype=torch.float64)
    assert [t if t is None else t.dtype for t in layers._autocast(x, x.float(), None, x.int())] == \
        [torch.float64, torch.get_autocast_dtype("cuda"), None, torch.int32]
    with pytest.raises(RuntimeError, match="float64"):
        layers.Linear(4, 3)(x)


def test_config_has_the_rounding_switch():
    import gact
    assert gact.config.stochastic_checkpoints is False
    from gact import layers
    assert layers._next_seed() is None
    gact.config.stochastic_checkpoints = True
    a, b = layers._next_seed(), layers._next_seed()
    assert a != b and 0 <= a < 1 << 64
