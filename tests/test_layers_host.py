"""gact.layers without a GPU: what the autograd functions hand to autograd and to the operators, with plain stand-ins for the
operators of gact.fused."""
import pytest
import torch

from gact import fused, layers


@pytest.fixture
def plain(monkeypatch):
    """op_linear and its backward pass in plain torch on the host; collects the keyword arguments of each call."""
    calls = []

    def op_linear(input, weight, bias=None, activation=None, residual=None, compress=True, seed=None, save=True, checkpoint=None, **kw):
        assert weight.dtype == input.dtype and (bias is None or bias.dtype == input.dtype)
        assert residual is None or residual.dtype == input.dtype
        calls.append(dict(kw, save=save, checkpoint=checkpoint, compress=compress, seed=seed, residual=residual is not None))
        y = torch.nn.functional.linear(input.float(), weight.float(), None if bias is None else bias.float())
        y = (y if residual is None else y + residual.float()).to(input.dtype)
        if not save:
            return y, None
        kept = fused.Checkpoint8(torch.zeros(1, dtype=torch.int8), input.shape, input.dtype) if compress else input
        return y, fused.LinearSaved(kept if kw.get("keep_input", True) else None, None, weight, activation, y.shape, bias is not None)

    def op_linear_backward(dy, saved, needs=(True, True, True)):
        assert saved.weight is None or saved.weight.dtype == dy.dtype
        return tuple(None if not n else dy @ saved.weight if i == 0 else torch.ones(dy.shape[-1], saved.x.shape[-1], dtype=dy.dtype) if i == 1
                     else dy.sum(0) for i, n in enumerate(needs))

    monkeypatch.setattr(fused, "op_linear", op_linear)
    monkeypatch.setattr(fused, "op_linear_backward", op_linear_backward)
    return calls


@pytest.fixture
def autocast(monkeypatch):
    """Autocast of CUDA tensors to bfloat16, as the layers see it."""
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda device: True)
    monkeypatch.setattr(torch, "get_autocast_dtype", lambda device: torch.bfloat16)


def test_layer_norm_keeps_the_checkpoint_of_its_deviations(monkeypatch):
    """Codes of the input itself would lose rows whose mean is large against their deviation."""
    seen = []

    def op_layer_norm(input, weight=None, bias=None, eps=1e-5, compress=True, seed=None, save=True, center=False):
        seen.append((compress, center))
        kept = fused.Checkpoint8(torch.zeros(1, dtype=torch.int8), input.shape, input.dtype) if compress else input
        return input * 1, fused.LayerNormSaved(kept, torch.zeros(2, 2), weight, input.shape, input.dtype, input.dtype)

    monkeypatch.setattr(fused, "op_layer_norm", op_layer_norm)
    layers.LayerNorm(4)(torch.zeros(2, 4))
    layers.layer_norm(torch.zeros(2, 4, requires_grad=True))
    assert seen == [(True, True)] * 2


def saved_by(call):
    seen = []

    def pack(t):
        seen.append(t)
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        out = call()
    return out, seen


@pytest.mark.parametrize("compress", [True, False])
def test_under_autocast_the_parameters_themselves_are_saved(plain, autocast, compress):
    """Saved-tensor hooks know a parameter by its address; a cast copy that requires a gradient they would quantize."""
    m = layers.Linear(8, 4)
    x = torch.randn(5, 8, requires_grad=True)
    y, seen = saved_by(lambda: layers.linear(x, m.weight, m.bias, compress=compress))
    address = {p.data_ptr() for p in m.parameters()}
    strange = [t for t in seen if t.is_floating_point() and t.requires_grad and t.data_ptr() not in address]
    # (without compression the input in the computed type is an activation like any other)
    assert [tuple(t.shape) for t in strange] == ([] if compress else [(5, 8)])
    assert any(t.data_ptr() == m.weight.data_ptr() for t in seen)
    y.float().sum().backward()
    assert y.dtype == torch.bfloat16 and x.grad.dtype == m.weight.grad.dtype == m.bias.grad.dtype == torch.float32
    want = torch.ones(5, 4, dtype=torch.bfloat16) @ m.weight.detach().bfloat16()
    assert torch.equal(x.grad, want.float())


def test_layer_norm_refuses_unknown_ways_of_rounding():
    import ctypes
    from gact import _native as nv
    b = ctypes.create_string_buffer(1 << 12)
    p = (ctypes.addressof(b) + 255) & ~255
    for rounding, status in ((2, 6), (8, 6), (-1, 6)):
        assert nv.lib.gact_layer_norm(p, 2, 2, 32, 32, p, p, 2, 1e-5, p, p, p, p, rounding, 0, None) == status


def test_a_controller_without_compression_still_asks_for_lost_copies(monkeypatch):
    import gact
    import gact.controller
    asked = []
    monkeypatch.setattr(gact.controller, "_device_live", lambda: True)
    monkeypatch.setattr(gact.controller._nv, "check_pipeline", asked.append)
    gact.set_optimization_level("L0")
    c = gact.Controller(torch.nn.Linear(2, 2))
    c.install_hook()
    c.uninstall_hook()
    c.uninstall_hook()
    assert asked == ["Controller.uninstall_hook"]


def test_no_report_without_a_device():
    from gact import _native as nv
    assert nv.lib.gact_pipeline_reported() == 0


@pytest.mark.parametrize("compress", [True, False])
def test_only_what_a_gradient_needs_is_saved(plain, compress):
    """A frozen weight keeps no input, a frozen input no weight, a residual alone nothing; gradients come out where they are asked for."""
    for x_grad, w_grad, b_grad, r_grad in [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (1, 0, 1, 1), (0, 0, 0, 1), (1, 1, 1, 1)]:
        x, w, b, r = (torch.randn(*s).bfloat16().requires_grad_(bool(g)) for s, g in (((5, 8), x_grad), ((4, 8), w_grad), ((4,), b_grad), ((5, 4), r_grad)))
        w = torch.nn.Parameter(w.detach(), requires_grad=bool(w_grad))
        y, seen = saved_by(lambda: layers.linear(x, w, b, residual=r, compress=compress))
        assert plain[-1]["save"] == bool(x_grad or w_grad or b_grad) and plain[-1].get("keep_input", True) == bool(w_grad or not plain[-1]["save"])
        assert any(t.data_ptr() == w.data_ptr() for t in seen) == bool(x_grad)
        assert any(t.dtype == torch.int8 or t.data_ptr() == x.data_ptr() for t in seen) == bool(w_grad)
        if not x_grad:
            with torch.no_grad():
                w.mul_(2)                       # (nobody needs the old one)
        y.sum().backward()
        assert [t.grad is not None for t in (x, w, b, r)] == [bool(g) for g in (x_grad, w_grad, b_grad, r_grad)]


def test_a_plain_weight_without_gradient_says_whether_the_input_is_kept(plain):
    x, w = torch.randn(5, 8).bfloat16().requires_grad_(), torch.randn(4, 8).bfloat16()
    for asked, kept in ((None, True), (True, True), (False, False)):
        layers.linear(x, w, keep_input=asked)
        assert plain[-1]["keep_input"] == kept
    layers.linear(x, w.clone().requires_grad_(), keep_input=False)           # (its gradient needs it)
    assert plain[-1]["keep_input"]


def test_share_input_of_frozen_layers_makes_no_checkpoint(plain, monkeypatch):
    made = []
    monkeypatch.setattr(fused, "op_checkpoint8", lambda x, seed=None: made.append(x))

    class Two(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.b = layers.Linear(8, 8), layers.Linear(8, 8)

        def forward(self, x):
            return self.a(x) + self.b(x)

    m = Two().bfloat16().requires_grad_(False)
    layers.share_input(m, (m.a, m.b))
    m(torch.zeros(3, 8, dtype=torch.bfloat16, requires_grad=True))
    assert not made and not any(c["keep_input"] for c in plain)


def test_a_wider_residual_keeps_its_type_under_autocast(plain, autocast):
    """torch's linear + residual gives the wider type; a residual stream in fp32 must not be lowered to 16 bits."""
    x, w = torch.randn(5, 8), torch.nn.Parameter(torch.randn(4, 8))
    for dt in (torch.float32, torch.float64):
        r = torch.randn(5, 4, dtype=dt).requires_grad_()
        y = layers.linear(x, w, residual=r)
        assert y.dtype == dt and torch.equal(y, layers.linear(x, w) + r) and not plain[-1]["residual"]
        y.sum().backward()
        assert torch.equal(r.grad, torch.ones_like(r)) and w.grad.dtype == torch.float32
    assert layers.linear(x, w, residual=torch.randn(5, 4).bfloat16()).dtype == torch.bfloat16 and plain[-1]["residual"]
    with torch.no_grad():
        assert layers.linear(x, w, residual=torch.randn(5, 4)).dtype == torch.float32
    with pytest.raises(ValueError, match="residual must have shape"):
        layers.linear(x, w, residual=torch.randn(4))


def test_entry_points_refuse_unknown_ways_of_rounding():
    import ctypes
    from gact import _native as nv
    b = ctypes.create_string_buffer(1 << 14)
    p = (ctypes.addressof(b) + 255) & ~255
    L = nv.lib
    calls = [lambda r, seed: L.gact_checkpoint8(p, 0, 2, 32, 32, r, seed, p, p, None),
             lambda r, seed: L.gact_layer_norm(p, 2, 2, 32, 32, p, p, 2, 1e-5, p, p, p, p, r, seed, None),
             lambda r, seed: L.gact_linear(p, 64, p, 64, p, None, 0, 2, 4, 64, 32, 2, p, p, p, None, p, p, r, seed, p, None)]
    for i, f in enumerate(calls):
        for r in (2, 8, 6, -1) + (() if i == 1 else (4, 5)):
            assert f(r, p) == 6
        assert f(3, 0) == 3 and f(3, p + 4) == 4             # a seed on the device has an address of 8 bytes


class Attention(torch.nn.Module):
    """Two layers on one input, as query and key are."""

    def __init__(self, inside=None):
        super().__init__()
        self.a, self.b, self.inside = layers.Linear(8, 8), layers.Linear(8, 8), inside

    def forward(self, x):
        if self.inside is not None:
            self.inside()
        return self.a(x) + self.b(x)


@pytest.fixture
def checkpoints(monkeypatch):
    """op_checkpoint8 without a device; the checkpoints that were made."""
    made = []

    def op_checkpoint8(x, seed=None):
        made.append(fused.Checkpoint8(torch.zeros(x.numel() * 33 // 32, dtype=torch.int8), x.shape, x.dtype))
        return made[-1]

    monkeypatch.setattr(fused, "op_checkpoint8", op_checkpoint8)
    return made


def test_share_input_when_the_forward_pass_enters_another_autocast(plain, checkpoints, monkeypatch):
    """The shared checkpoint is of the type outside; layers that compute in another one keep their own instead of failing."""
    def enter():
        monkeypatch.setattr(torch, "is_autocast_enabled", lambda device: True)
        monkeypatch.setattr(torch, "get_autocast_dtype", lambda device: torch.float16)

    m = Attention(enter).bfloat16()
    layers.share_input(m, (m.a, m.b))
    x = torch.zeros(4, 8, dtype=torch.bfloat16, requires_grad=True)
    assert m(x).dtype == torch.float16 and len(checkpoints) == 1
    assert [c["checkpoint"] for c in plain] == [None, None]
    monkeypatch.undo()


@pytest.mark.parametrize("way", ["deepcopy", "pickle"])
def test_a_copy_shares_among_its_own_layers(plain, checkpoints, way):
    import copy
    import io
    m = Attention().bfloat16()
    layers.share_input(m, (m.a, m.b))
    if way == "deepcopy":
        twin = copy.deepcopy(m)
    else:
        file = io.BytesIO()
        torch.save(m, file)
        file.seek(0)
        twin = torch.load(file, weights_only=False)
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    twin(x)
    assert len(checkpoints) == 1 and [c["checkpoint"].buf.data_ptr() for c in plain] == [checkpoints[0].buf.data_ptr()] * 2
    assert all(c._shared is None for c in (m.a, m.b, twin.a, twin.b))
    m(x)
    assert len(checkpoints) == 2 and [c["checkpoint"].buf.data_ptr() for c in plain[2:]] == [checkpoints[1].buf.data_ptr()] * 2


def test_convert_leaves_norms_that_are_too_long():
    """What ran before conversion runs after it: the operator takes rows of at most 16384."""
    m = torch.nn.Sequential(torch.nn.LayerNorm(16385), torch.nn.LayerNorm((128, 129)), torch.nn.LayerNorm((128, 128)), torch.nn.LayerNorm(16384))
    layers.convert(m)
    assert [type(c) is layers.LayerNorm for c in m] == [False, False, True, True]
    x = torch.randn(2, 16385)
    assert torch.equal(m[0](x), torch.nn.functional.layer_norm(x, (16385,)))


def test_convert_leaves_float64_layers():
    """The operators have no float64: a head in double precision under a converted body goes on running."""
    m = torch.nn.Sequential(torch.nn.Linear(4, 4), torch.nn.Sequential(torch.nn.LayerNorm(4), torch.nn.Linear(4, 2), torch.nn.ReLU()).double())
    layers.convert(m)
    assert type(m[0]) is layers.Linear and type(m[1][0]) is torch.nn.LayerNorm and type(m[1][1]) is torch.nn.Linear and type(m[1][2]) is torch.nn.ReLU
    assert m[1](torch.randn(3, 4, dtype=torch.float64)).dtype == torch.float64


def test_convert_does_not_move_an_activation_into_a_layer_that_is_used_elsewhere():
    own = layers.Linear(4, 4)
    seen = []
    own.register_forward_hook(lambda m, a, y: seen.append(y))
    m = torch.nn.ModuleList([torch.nn.Sequential(own, torch.nn.ReLU()), own])
    layers.convert(m)
    assert m[0][0] is own is m[1] and own.activation is None and type(m[0][1]) is torch.nn.ReLU
    lin = torch.nn.Linear(4, 4)
    m = torch.nn.ModuleList([torch.nn.Sequential(lin, torch.nn.ReLU()), lin])
    layers.convert(m)
    assert m[0][0].activation == "relu" and m[1].activation is None and m[0][0].weight is m[1].weight is lin.weight


@pytest.mark.parametrize("compress", [True, False])
def test_a_computed_weight_is_no_activation(plain, compress):
    """A weight that is computed from parameters (a norm, an adapter's product) reaches the hooks without requiring a gradient, and a
    change in place is still noticed."""
    a, b = torch.randn(4, 2).bfloat16().requires_grad_(), torch.randn(2, 8).bfloat16().requires_grad_()
    x = torch.randn(5, 8).bfloat16().requires_grad_()
    w = a @ b
    y, seen = saved_by(lambda: layers.linear(x, w, compress=compress))
    assert not any(t.requires_grad for t in seen if t.is_floating_point() and t.data_ptr() != x.data_ptr())
    y.sum().backward(retain_graph=True)
    assert a.grad is not None and torch.equal(x.grad, torch.ones(5, 4).bfloat16() @ w.detach())
    y = layers.linear(x, w, compress=compress)          # (hooks do without the version check)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
