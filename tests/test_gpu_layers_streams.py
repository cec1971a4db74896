"""Layers that share a checkpoint of their input, on several streams."""
import pytest
import torch

gpu = pytest.mark.gpu


def rand(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").bfloat16()


@gpu
def test_a_layer_on_another_stream_makes_its_own_checkpoint():
    """The second layer runs on a stream that waits only for the input: it must not read (nor keep) a checkpoint that the first stream
    may not have made yet and whose memory goes back to the first stream."""
    from gact import layers

    class Two(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.b = layers.Linear(64, 64), layers.Linear(64, 64)
            self.side = torch.cuda.Stream()

        def forward(self, x, ready=None):
            y = self.a(x)
            if ready is None:
                return y, self.b(x)
            self.side.wait_event(ready)
            with torch.cuda.stream(self.side):
                z = self.b(x)
            torch.cuda.current_stream().wait_stream(self.side)
            return y, z

    torch.manual_seed(0)
    m = Two().cuda().bfloat16()
    layers.share_input(m, (m.a, m.b))
    x = rand(256, 64, seed=1)
    y, z = m(x)
    shared = [t.grad_fn.saved_tensors[0] for t in (y, z)]
    assert shared[0].data_ptr() == shared[1].data_ptr()
    (y.float().square().sum() + z.float().square().sum()).backward()
    want = [p.grad.clone() for p in m.parameters()]
    m.zero_grad()
    ready = torch.cuda.Event()
    ready.record()
    y, z = m(x, ready)
    own = [t.grad_fn.saved_tensors[0] for t in (y, z)]
    assert own[0].data_ptr() != own[1].data_ptr() and torch.equal(own[1], shared[0])
    (y.float().square().sum() + z.float().square().sum()).backward()
    torch.cuda.synchronize()
    assert all(torch.equal(p.grad, w) for p, w in zip(m.parameters(), want))
    assert m.a._shared is None and m.b._shared is None
