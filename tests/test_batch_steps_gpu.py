"""Steps of a batch that mix prompts and single tokens behind a long prefix, run and captured, against
64-bit arithmetic under the tolerances of test_batch_gpu."""
import pytest
import torch

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
