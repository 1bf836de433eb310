"""Steps of a batch that mix prompts and single tokens behind a long prefix, run and captured, against
64-bit arithmetic under the tolerances of test_batch_gpu."""
import numpy as np
import pytest
import torch

from wick_amd.batch import DeviceBatch
from test_batch_gpu import DEV, U, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,start,t,prefix", [
    (32, 8, 128, [142, 52, 0], [1, 1, 32], 8764),
    (14, 2, 64, [9, 0], [18, 1], 35263),
    (32, 4, 64, [0, 100, 100], [15, 1, 1], 24000),
    (9, 3, 64, [0, 100, 100, 100, 100, 100], [38, 1, 1, 1, 1, 1], 24000),
    (16, 8, 128, [3, 100, 100, 100], [62, 1, 1, 1], 16384),
])
def test_a_prompt_beside_single_tokens(heads, kv_heads, d, start, t, prefix, dtype):
    Case(heads, kv_heads, d, start, t, prefix, dtype, seed=heads).fill().check()


@pytest.mark.parametrize("heads,kv_heads,d,start,t,prefix", [
    (32, 4, 64, [0, 100, 100], [15, 1, 1], 24000),
    (9, 3, 64, [0, 100, 100, 100, 100, 100], [38, 1, 1, 1, 1, 1], 24000),
])
def test_captured_beside_single_tokens(heads, kv_heads, d, start, t, prefix):
    """A handle with room for more tokens; the graph replays under its own plan and at other places."""
    c = Case(heads, kv_heads, d, start, t, prefix, seed=prefix + heads, capacity=1000)
    c.fill()
    want = c.check()
    elsewhere = [start[0] + 1] + [x - 50 for x in start[1:]]
    att = torch.zeros_like(want)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    c.b.set_stream(stream.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        c.b.attention_device(c.layer, c.q.data_ptr(), att.data_ptr())
    for i in range(3):
        for at, p in ((start, prefix), (elsewhere, prefix // 2), (start, prefix)):
            c.b.plan(at, t, p)
            with torch.cuda.stream(stream):
                att.zero_()
                graph.replay()
            torch.cuda.synchronize()
            assert float(torch.ones(10, device=DEV).sum()) == 10.0
            if at is start:
                assert torch.equal(c.check(att), want), i
            else:
                # the graph's join may sum in another order: each of two sums over at most n = 200
                # states is off by (n + 4) u of the largest value, below 6 here
                assert float((att - c.run()).abs().max()) < 2 * 204 * U * 6, i


def test_steps_beside_another_handles_capture():
    """Plans and steps of one handle while another's are captured: neither disturbs the other."""
    a, b = (Case(8, 2, 64, [50, 3], [1, 20], 400, seed=40 + i).fill() for i in range(2))
    wants = [a.check(), b.check()]
    att = torch.zeros_like(wants[1])
    out = torch.zeros_like(wants[0])
    q = a.q.cpu().numpy()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    b.b.set_stream(stream.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        b.b.attention_device(0, b.q.data_ptr(), att.data_ptr())
        for _ in range(3):
            a.b.plan(a.start, a.t, a.prefix)
            a.b.attention_device(0, a.q.data_ptr(), out.data_ptr())
        a.b.synchronize()
        host = a.b.attention(0, q)
        with DeviceBatch(1, 8, 2, 64, 1, 4) as other:
            other.plan([0], [2])
            other.append(0, np.ones((2, 128), np.float32), np.full((2, 128), 3, np.float32))
            k, v = other.read(0, 0, 0, 2)
            assert (k == 1).all() and (v == 3).all()
    torch.cuda.synchronize()
    assert torch.equal(out, wants[0]) and torch.equal(torch.from_numpy(host).to(DEV), wants[0])
    for _ in range(3):
        with torch.cuda.stream(stream):
            att.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(att, wants[1])


@pytest.mark.parametrize("heads,kv_heads,d,start,t,prefix", [
    (200, 1, 16, [0, 7], [3, 1], 200),       # a token's rows fill more than one item
    (257, 1, 32, [0, 30], [9, 2], 3000),
    (64, 64, 16, [0, 5, 0], [70, 1, 0], 150),
    (512, 2, 64, [40], [1], 9000),
])
def test_many_heads(heads, kv_heads, d, start, t, prefix):
    Case(heads, kv_heads, d, start, t, prefix, seed=heads).fill().check()


def test_many_sequences():
    """Most of them bring nothing, the others one token or a few."""
    rng = np.random.default_rng(5)
    t = [int(x) for x in rng.choice([0, 0, 0, 1, 1, 3], 1500)]
    Case(6, 2, 32, [int(x) for x in rng.integers(0, 9, 1500)], t, 700, seed=5).fill().check()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads,kv_heads,d,start,t,prefix", [
    (8, 2, 64, [0, 40], [9, 1], 0),
    (32, 8, 128, [0, 40, 3], [200, 1, 1], 2500),
])
def test_a_padding_row_of_queries(heads, kv_heads, d, start, t, prefix, bad):
    """Queries of one token that are no numbers: its result is none, the others' are as they were."""
    c = Case(heads, kv_heads, d, start, t, prefix, seed=60).fill()
    want, tol = c.want()
    q = c.q.clone()
    q[3] = bad
    got = c.run(q)
    assert not bool(torch.isfinite(got[3]).any())
    rest = torch.arange(len(got), device=DEV) != 3
    assert bool(((got.double() - want).abs() <= tol)[rest].all())
