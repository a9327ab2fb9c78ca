"""Two calls side by side, on two streams and as two captured graphs, with the calls that share no prefix worth a
kernel of its own (decode_shared under 128 tokens), plain decode and the dense prefill: each has its own workspace."""
import pytest
import torch

from lockstep_b200 import attention as A
from lockstep_b200 import decode as D

pytestmark = pytest.mark.gpu


def bits(x):
    return x.contiguous().view(torch.int16)


def side_by_side(call, inputs, grow):
    """call(x) for two inputs in flight at once, against the same calls alone; grow() is a larger call between them."""
    want = [call(x) for x in inputs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(x))
        graphs.append(g)
    grow()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(bits(o), bits(w)) for o, w in zip(outs, want))
        eager = []
        for x, s in zip(inputs, streams):
            with torch.cuda.stream(s):
                eager.append(call(x))
        torch.cuda.synchronize()
        assert all(torch.equal(bits(o), bits(w)) for o, w in zip(eager, want))
    A.check_device_errors(inputs[0].device)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("shared", [None, 0, 100])
def test_decode_calls_side_by_side(dh, shared):
    g = torch.Generator("cuda").manual_seed(dh)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)       # noqa: E731
    kv = D.contiguous_kv(draw(6, 2, 3001, dh), draw(6, 2, 3001, dh), sink=True)
    big = D.contiguous_kv(draw(12, 4, 6000, dh), draw(12, 4, 6000, dh))
    if shared is None:
        call = lambda x: D.decode(x, kv, check=False)                           # noqa: E731
    else:
        call = lambda x: D.decode_shared(x, kv, shared, check=False)            # noqa: E731
    side_by_side(call, (draw(6, 8, dh), draw(6, 8, dh)), lambda: D.decode(draw(12, 16, dh), big))


def test_prefill_calls_side_by_side():
    g = torch.Generator("cuda").manual_seed(1)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)       # noqa: E731
    k, v = draw(1, 2, 700, 64), draw(1, 2, 700, 64)
    side_by_side(lambda x: A.prefill(x, k, v, check=False), (draw(1, 4, 700, 64), draw(1, 4, 700, 64)),
                 lambda: A.prefill(draw(2, 4, 2000, 64), draw(2, 2, 2000, 64), draw(2, 2, 2000, 64)))
