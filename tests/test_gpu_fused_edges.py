"""Edges of the fused operators: bounds of every output, side work beside the products, extreme values, refusals with tensors on
the GPU, first calls inside a capture, one saved state used twice."""
import ctypes
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

gpu = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def rand(*shape, seed=0, dtype=BF, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


class Guarded:
    """An output of `nbytes` bytes (at `shift` bytes from a 256-byte boundary) between two guard regions."""

    def __init__(self, nbytes, shift=0):
        self.n, self.lo = nbytes, 4096 + shift
        self.buf = torch.full((self.lo + nbytes + 4096,), 0xA5, dtype=torch.uint8, device="cuda")

    @property
    def ptr(self):
        return self.buf.data_ptr() + self.lo

    def check(self, what):
        assert bool((self.buf[:self.lo] == 0xA5).all()) and bool((self.buf[self.lo + self.n:] == 0xA5).all()), what

    def view(self, dtype, *shape):
        return self.buf[self.lo:self.lo + self.n].clone().view(dtype).view(*shape)


@gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 33), (17, 255), (40, 1000), (9, 4096), (1300, 2056), (1300, 1032)])
@pytest.mark.parametrize("shift", [0, 2])
def test_norm_and_checkpoint_write_only_their_outputs(rows, cols, shift):
    from gact import _native as nv, fused
    L, st = nv.lib, nv.stream_ptr()
    pitch = (cols + 31) // 32 * 32
    x, w = rand(rows, cols, seed=1), rand(cols, seed=2)
    out = {n: Guarded(b, s) for n, b, s in (("y", rows * cols * 2, shift), ("stats", rows * 8, 0), ("codes", rows * pitch, 0), ("scales", rows * pitch // 32, shift),
                                            ("dx", rows * cols * 2, shift), ("dw", cols * 2, shift), ("db", cols * 2, shift), ("back", rows * cols * 2, shift))}
    scr = Guarded(L.gact_layer_norm_backward_scratch_bytes(rows, cols))
    p = {n: g.ptr for n, g in out.items()}
    assert L.gact_layer_norm(x.data_ptr(), 2, rows, cols, cols, w.data_ptr(), w.data_ptr(), 2, 1e-5, p["y"], p["stats"], p["codes"], p["scales"], 0, 0, st) == 0
    assert L.gact_layer_norm_backward(x.data_ptr(), 2, rows, cols, cols, None, 0, p["codes"], p["scales"], p["stats"], w.data_ptr(), 2, p["dx"], p["dw"], p["db"],
                                      scr.ptr, st) == 0
    assert L.gact_restore8(p["codes"], p["scales"], rows, cols, 2, p["back"], cols, st) == 0
    torch.cuda.synchronize()
    for n, g in list(out.items()) + [("scratch", scr)]:
        g.check(n)
    y, s = fused.op_layer_norm(x, w, w)
    got = fused.op_layer_norm_backward(x, s)
    assert torch.equal(out["codes"].view(torch.int8, rows, pitch), s.x.codes)
    # Another alignment may take a kernel that sums in another order.  Each y is half a step (2^-9 of its value up to the next
    # power of two, so at most 2^-8 |y|) plus the fp32 error e from the exact one, so two of them differ by at most
    # 2^-7 |y| + 2 e, with e <= 64 * 2^-24 * (|x| + mean|x| + |x^|) r |w| + ... < 64 * 2^-24 * 100 for these inputs (|x^|, |w| < 6).
    a, b = out["y"].view(BF, rows, cols).double(), y.double()
    assert bool(((a - b).abs() <= 2.0 ** -7 * torch.maximum(a.abs(), b.abs()) + 2 * 64 * 2.0 ** -24 * 100).all())
    assert torch.equal(out["back"].view(BF, rows, cols), fused.op_restore8(s.x))
    for n, t in zip(("dx", "dw", "db"), got):
        # (another alignment may take another kernel: sums in another order)
        assert float((out[n].view(BF, *t.shape).double() - t.double()).abs().max()) <= 2.0 ** -7 * float(t.double().abs().max()) + 1e-6


@gpu
@pytest.mark.parametrize("rows,cin,cout", [(1, 8, 1), (5, 72, 3), (129, 64, 257), (130, 1024, 2), (300, 776, 331), (64, 4096, 40), (700, 520, 520)])
def test_linear_writes_only_its_outputs(rows, cin, cout):
    from gact import _native as nv, fused
    L, st = nv.lib, nv.stream_ptr()
    px, pz, po = (cin + 31) // 32 * 32, (cout + 31) // 32 * 32, (cout + 7) // 8 * 8
    x, w, b = rand(rows, cin, seed=1), rand(cout, cin, seed=2, std=0.1), rand(cout, seed=3)
    dy = rand(rows, cout, seed=4)
    sizes = {"y": rows * cout * 2, "xc": rows * px, "xs": rows * px // 32, "zc": rows * pz, "zs": rows * pz // 32, "dz": rows * po * 2, "dx": rows * cin * 2,
             "dw": cout * cin * 2, "db": cout * 2, "xr": rows * px * 2, "sums": L.gact_act_backward_scratch_bytes(rows, cout)}
    for d in range(3):
        sizes["scr%d" % d] = max(1, L.gact_linear_scratch_bytes(rows, cin, cout, d))
    out = {n: Guarded(v) for n, v in sizes.items()}
    p = {n: g.ptr for n, g in out.items()}
    assert L.gact_linear(x.data_ptr(), cin, w.data_ptr(), cin, b.data_ptr(), None, 0, 2, rows, cin, cout, 2, p["y"], p["xc"], p["xs"], None, p["zc"], p["zs"], 0, 0,
                         p["scr0"], st) == 0
    assert L.gact_act_backward(dy.data_ptr(), 2, rows, cout, cout, 2, None, 0, p["zc"], p["zs"], p["dz"], po, None, p["sums"], st) == 0
    assert L.gact_linear_dgrad(p["dz"], po, w.data_ptr(), cin, 2, rows, cin, cout, p["dx"], p["sums"], p["db"], p["xc"], p["xs"], p["xr"], p["scr1"], st) == 0
    assert L.gact_linear_wgrad(p["dz"], po, p["xr"], px, 2, rows, cin, cout, p["dw"], None, None, p["scr2"], st) == 0
    torch.cuda.synchronize()
    for n, g in out.items():
        g.check(n)
    y, s = fused.op_linear(x, w, b, "gelu")
    dx, dw, db = fused.op_linear_backward(dy, s)
    assert torch.equal(out["y"].view(BF, rows, cout), y) and torch.equal(out["dx"].view(BF, rows, cin), dx)
    assert torch.equal(out["dw"].view(BF, cout, cin), dw) and torch.equal(out["db"].view(BF, cout), db)
    assert torch.equal(out["xc"].view(torch.int8, rows, px), fused.op_checkpoint8(x).codes)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,cin,cout", [(64, 1024, 2), (1000, 771, 333), (4096, 4096, 512), (4096, 512, 4096), (40000, 136, 72), (2, 5000, 8)])
def test_work_beside_the_products_equals_work_on_its_own(rows, cin, cout, dtype):
    """The checkpoint of x is that of op_checkpoint8, the weight gradient that of the restored x, and the bias gradient that of a
    call that asks for nothing else, whatever was done beside which product."""
    from gact import fused
    x, w, b = rand(rows, cin, seed=1, dtype=dtype), rand(cout, cin, seed=2, std=0.05, dtype=dtype), rand(cout, seed=3, dtype=dtype)
    dy = rand(rows, cout, seed=4, dtype=dtype, std=0.1)
    for seed in (None, 5):
        y, s = fused.op_linear(x, w, b, "gelu", seed=seed)
        alone = fused.op_checkpoint8(x, seed)
        assert torch.equal(s.x.buf, alone.buf)
        dx, dw, db = fused.op_linear_backward(dy, s)
        restored = fused.LinearSaved(fused.op_restore8(alone), s.z, w, "gelu", s.out_shape, True)
        dx2, dw2, db2 = fused.op_linear_backward(dy, restored)
        assert torch.equal(dw, dw2) and torch.equal(dx, dx2) and torch.equal(db, db2)
        assert torch.equal(db, fused.op_linear_backward(dy, s, (False, False, True))[2])
        only = fused.op_linear_backward(dy, s, (False, True, True))
        assert only[0] is None and torch.equal(only[1], dw) and torch.equal(only[2], db)
        # the same saved state again (a graph kept for a second backward pass)
        again = fused.op_linear_backward(dy, s)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw) and torch.equal(again[2], db)


@gpu
def test_stochastic_pre_activation_is_within_a_step():
    from gact import fused
    x, w = rand(200, 64, seed=1), rand(96, 64, seed=2, std=0.1)
    z = (x.double() @ w.double().t()).cpu()
    for act in ("gelu", "relu"):
        a, b = fused.op_linear(x, w, None, act, seed=7)[1], fused.op_linear(x, w, None, act, seed=7)[1]
        assert torch.equal(a.z.buf, b.z.buf) and not torch.equal(a.z.buf, fused.op_linear(x, w, None, act, seed=8)[1].z.buf)
        kept = fused.op_restore8(a.z, F32).double().cpu()
        step = torch.exp2(a.z.scales.cpu().view(torch.uint8).double() - 127).repeat_interleave(32, 1)
        assert bool(((kept - z).abs() <= step * 1.01).all())
        if act == "relu":
            assert bool((kept > 0)[z > 1e-4].all())


@gpu
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_activations_at_extreme_values(act):
    """From far below zero to far above: finite values and slopes, right to the formula; z = 0 and huge z included."""
    from gact import fused
    z = torch.cat([torch.linspace(-30, 30, 4001), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e4, -1e4, 1e19, -1e19, 3e38, -3e38, 1e-3, -1e-3, 5e-4, 0.0039])])
    n = z.numel()
    x = z.to(BF).cuda().view(n, 1)
    one = torch.ones(1, 1, dtype=BF, device="cuda")
    z64 = x.double().cpu().view(-1)
    t = z64.clamp(-1e6, 1e6).requires_grad_()
    f = {"relu": torch.relu, "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh"), "silu": torch.nn.functional.silu}[act]
    ref = f(t)
    ref.sum().backward()
    for compress in (True, False):
        y, s = fused.op_linear(x, one, None, act, compress=compress)
        got = y.double().cpu().view(-1)
        small = z64.abs() <= 1e6
        assert bool(((got - ref.detach()).abs() <= 2.0 ** -8 * 1.01 * ref.detach().abs() + 2e-6 * z64.abs().clamp(max=50) + 1e-30)[small].all())
        assert bool((got == z64)[z64 > 1e6].all()) and bool((got.abs() < 1e-30)[z64 < -1e6].all())
        dz = torch.empty(0)
        dx = fused.op_linear_backward(torch.ones_like(y), s, (True, False, False))[0].double().cpu().view(-1)
        zk = z64 if not compress else fused.op_restore8(s.z, F32).double().cpu().view(-1)
        u = zk.clamp(-1e6, 1e6).requires_grad_()
        f(u).sum().backward()
        assert bool(((dx - u.grad).abs() <= 2.0 ** -8 * 1.01 * u.grad.abs() + 4e-6).all()), (act, compress)


@gpu
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_the_table_of_slopes_at_every_exponent(act):
    """Blocks of every scale from 2^-20 to 2^8 (below, inside and above the table), NaN blocks, all 255 codes, on a problem
    large enough for the table."""
    from gact import fused
    rows, cols = 20000, 320
    c = torch.arange(-127, 128, dtype=torch.float64)
    g = torch.Generator().manual_seed(1)
    codes = c[torch.randint(0, 255, (rows, cols), generator=g)]
    codes[:, ::32] = 127 * (torch.randint(0, 2, (rows, cols // 32), generator=g) * 2 - 1).double() * 0.99     # (the block's scale)
    e = torch.randint(-20, 9, (rows, cols // 32), generator=g).double()
    z = (codes * torch.exp2(e).repeat_interleave(32, 1)).to(F32).cuda()
    z[5, 40] = float("nan")
    ck = fused.op_checkpoint8(z)
    zk = fused.op_restore8(ck).double().cpu()
    dy = rand(rows, cols, seed=2)
    w = torch.ones(cols, 8, dtype=BF, device="cuda")
    saved = fused.LinearSaved(rand(rows, 8, seed=3), ck, w, act, torch.Size((rows, cols)), True)
    from gact import _native as nv
    L = nv.lib
    dz = torch.empty(rows, cols, dtype=BF, device="cuda")
    sums = torch.empty(L.gact_act_backward_scratch_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    db = torch.empty(cols, dtype=BF, device="cuda")
    assert L.gact_act_backward(dy.data_ptr(), 2, rows, cols, cols, nv.ACT_CODE[act], None, 0, ck.codes.data_ptr(), ck.scales.data_ptr(), dz.data_ptr(), cols,
                               db.data_ptr(), sums.data_ptr(), nv.stream_ptr()) == 0
    t = zk.requires_grad_()
    {"gelu": torch.nn.functional.gelu, "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh"), "silu": torch.nn.functional.silu}[act](t).sum().backward()
    want, got = t.grad * dy.double().cpu(), dz.double().cpu()
    assert bool((got.isnan() == want.isnan()).all()) and int(got.isnan().sum()) == 32
    ok = ~want.isnan()
    assert bool(((got - want).abs() <= 2.0 ** -8 * 1.01 * want.abs() + 4e-6 * dy.double().cpu().abs())[ok].all())
    cols_ok = torch.ones(cols, dtype=torch.bool)
    cols_ok[32:64] = False
    ref = want[:, cols_ok].sum(0)
    tol = 2.0 ** -8 * 1.01 * ref.abs() + (64 + rows / 64) * 2.0 ** -24 * want[:, cols_ok].abs().sum(0) + 4e-6 * dy.double().cpu().abs()[:, cols_ok].sum(0)
    assert bool(((db.double().cpu()[cols_ok] - ref).abs() <= tol).all()) and bool(db[32:64].isnan().all())


@gpu
def test_refusals_with_tensors_on_the_gpu():
    from gact import fused
    x, w = rand(4, 16), rand(8, 16)
    y, s = fused.op_linear(x, w, None, "gelu")
    n, t = fused.op_layer_norm(x)
    value = [lambda: fused.op_linear(x, rand(8, 15)), lambda: fused.op_linear(x, w, rand(7)), lambda: fused.op_linear(x, w, residual=rand(4, 9)),
             lambda: fused.op_linear(x, w, activation="tanh"), lambda: fused.op_linear(x, w[0]), lambda: fused.op_linear(x[:, :0], w[:, :0]),
             lambda: fused.op_linear(x, w, checkpoint=fused.op_checkpoint8(x[:2])), lambda: fused.op_linear_backward(y[:2], s),
             lambda: fused.op_layer_norm(x, rand(15)), lambda: fused.op_layer_norm(x, None, rand(16, 1)), lambda: fused.op_layer_norm(x[:, :0]),
             lambda: fused.op_layer_norm(rand(1, 16385)), lambda: fused.op_layer_norm_backward(n[:, :8], t), lambda: fused.op_checkpoint8(x[0, 0]),
             lambda: fused.op_restore8(fused.Checkpoint8(fused.op_checkpoint8(x).buf, (5, 16), BF)),
             lambda: fused.op_restore8(fused.Checkpoint8(fused.op_checkpoint8(x).buf[::2], (2, 16), BF))]
    kind = [lambda: fused.op_linear(x.float(), w.float()), lambda: fused.op_linear(x, w.half()), lambda: fused.op_linear(x, w, rand(8, dtype=F32)),
            lambda: fused.op_linear(x, w, residual=rand(4, 8, dtype=HF)), lambda: fused.op_linear(x, w.cpu()), lambda: fused.op_layer_norm(x, rand(16, dtype=HF)),
            lambda: fused.op_layer_norm(x, rand(16), rand(16, dtype=F32)), lambda: fused.op_layer_norm(x.double()), lambda: fused.op_layer_norm_backward(n.float(), t),
            lambda: fused.op_checkpoint8(x.int()), lambda: fused.op_checkpoint8(x.to_sparse()), lambda: fused.op_linear_backward(y.half(), s),
            lambda: fused.op_restore8(fused.op_checkpoint8(x), torch.float64)]
    types = [lambda: fused.op_linear(x, w, checkpoint=x), lambda: fused.op_restore8(x), lambda: fused.op_linear("x", w), lambda: fused.op_layer_norm(x, 3)]
    for calls, error in ((value, ValueError), (kind, RuntimeError), (types, TypeError)):
        for i, call in enumerate(calls):
            with pytest.raises(error):
                call()
                pytest.fail("%s %d was accepted" % (error.__name__, i), pytrace=False)
    torch.cuda.synchronize()
    assert torch.equal(fused.op_linear(x, w, None, "gelu")[0], y)


@gpu
@pytest.mark.parametrize("what", ["pair of blocks", "one block", "ring"])
def test_a_wait_that_runs_out_ends_the_launch_and_is_reported(what):
    """With one copy withheld (the diagnostics switch of the quantizer's pipeline) the products and layer norm's rings give up
    after the wait limit, record the error and end by themselves; after a reset the next call is right again."""
    from gact import _native as nv, fused
    if what == "ring":
        x = rand(2000, 2048)
        _, s = fused.op_layer_norm(x)
        call = lambda: fused.op_layer_norm_backward(x, s)
    else:
        x, w = (rand(2048, 1024), rand(2048, 1024, seed=1)) if what == "pair of blocks" else (rand(100, 256), rand(64, 256, seed=1))
        call = lambda: fused.op_linear(x, w, save=False)[:1]
    want = call()
    torch.cuda.synchronize()
    assert nv.lib.gact_pipeline_error() == 0
    nv.lib.gact_pipeline_test_hook(2000, 1)
    try:
        call()
        torch.cuda.synchronize()                                   # the launch finished on its own
        assert nv.lib.gact_pipeline_error() > 0
        with pytest.raises(nv.GactError):
            nv.check_pipeline("test")                              # (clears the word)
    finally:
        nv.lib.gact_pipeline_test_hook(0, 0)
        nv.lib.gact_pipeline_error_reset()
    assert nv.lib.gact_pipeline_error() == 0
    assert all(torch.equal(a, b) for a, b in zip(call(), want))


@gpu
def test_first_calls_inside_a_capture():
    """A process whose very first calls are captured: attributes, occupancy and the tensor-map encoder are looked up on the way."""
    code = """
import sys, torch
sys.path.insert(0, %r)
from gact import fused
x, w, b = (torch.randn(*s, device="cuda").bfloat16() for s in ((3000, 1032), (264, 1032), (264,)))
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y, s = fused.op_linear(x, w, b, "gelu")
    n, t = fused.op_layer_norm(x)
    out = [y, n, *fused.op_linear_backward(y, s), *fused.op_layer_norm_backward(n, t)[:1]]
x.normal_()
g.replay()
got = [o.clone() for o in out]
y, s = fused.op_linear(x, w, b, "gelu")
n, t = fused.op_layer_norm(x)
want = [y, n, *fused.op_linear_backward(y, s), *fused.op_layer_norm_backward(n, t)[:1]]
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("captured")
""" % str(ROOT / "gact-icml_b200")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@gpu
def test_two_graphs_replayed_side_by_side():
    """Two captured steps on two streams, replayed at the same time, give what they give alone (no shared workspace)."""
    from gact import fused
    work = []
    for i in range(2):
        x, w, b = rand(2000, 512, seed=i), rand(384, 512, seed=10 + i, std=0.1), rand(384, seed=20 + i)
        dy = rand(2000, 384, seed=30 + i)

        def step(x=x, w=w, b=b, dy=dy):
            y, s = fused.op_linear(x, w, b, "silu")
            n, t = fused.op_layer_norm(x, w[0], w[1])
            return [y, n, *fused.op_linear_backward(dy, s), *fused.op_layer_norm_backward(x, t)]

        want = step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        work.append((g, out, want, torch.cuda.Stream(), step))          # (step: the graph's inputs stay alive)
    for _ in range(20):
        for g, out, want, st, _keep in work:
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for g, out, want, st, _keep in work:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@gpu
def test_offsets_past_32_bits():
    """More than 2^32 bytes of input and of codes: the last rows come out as they do alone."""
    from gact import fused
    rows, cols = 1 << 20, 4224                      # 8.9 GB of bf16, 4.5 GB of codes
    x = torch.empty(rows, cols, dtype=BF, device="cuda")
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(3))
    y, s = fused.op_layer_norm(x)
    tail = x[-2000:].clone()
    yt, st = fused.op_layer_norm(tail)
    assert torch.equal(y[-2000:], yt) and torch.equal(s.x.codes[-2000:], st.x.codes) and torch.equal(s.stats[-2000:], st.stats)
    dx = fused.op_layer_norm_backward(y, s, (True, False, False))[0]
    assert torch.equal(dx[-2000:], fused.op_layer_norm_backward(yt, st, (True, False, False))[0])
    del y, dx, s
    c = fused.op_checkpoint8(x)
    assert torch.equal(c.codes[-2000:], st.x.codes)
    r = fused.op_restore8(c)
    assert torch.equal(r[-2000:], fused.op_restore8(st.x))
    del r, c
    w = rand(64, cols, std=0.02)
    y, s = fused.op_linear(x, w, None, "relu")
    yt, st = fused.op_linear(tail, w, None, "relu")
    assert torch.equal(s.x.codes[-2000:], st.x.codes)
    # another number of rows may split the reduction another way: fp32 sums of `cols` products, each within cols 2^-23 of the
    # magnitudes' sum, and a rounding to bf16 (at most 2^-8) each
    mag = tail.float().abs() @ w.float().abs().t()
    diff = (y[-2000:].float() - yt.float()).abs()
    assert bool((diff <= 2.0 ** -7 * 1.01 * torch.maximum(y[-2000:].float().abs(), yt.float().abs()) + 2 * (cols + 8) * 2.0 ** -23 * mag).all())
    dx, dw, _ = fused.op_linear_backward(y, s)

    def cut(c):
        return fused.Checkpoint8(torch.cat([c.codes[-2000:].flatten(), c.scales[-2000:].flatten()]), torch.Size((2000, c.shape[1])), c.dtype)

    # (64 outputs: the data gradient's reduction is one stage, whatever the number of rows)
    last = fused.LinearSaved(cut(s.x), cut(s.z), w, "relu", torch.Size((2000, 64)), False)
    assert torch.equal(dx[-2000:], fused.op_linear_backward(y[-2000:].clone(), last)[0])
    # the weight gradient over all rows against the sum of that over parts (fp32 sums of 2^20 terms, rounded to bf16 per part)
    parts = torch.zeros(64, cols, dtype=torch.float64, device="cuda")
    for lo in range(0, rows, 1 << 17):
        yp, sp = fused.op_linear(x[lo:lo + (1 << 17)], w, None, "relu")
        parts += fused.op_linear_backward(yp, sp)[1].double()
    assert float((dw.double() - parts).norm() / parts.norm()) < 4 * 2.0 ** -8
