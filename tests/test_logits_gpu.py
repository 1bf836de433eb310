"""The logit rules (include/wick_hip_logits.h) against the same f32 steps by numpy, to the bit."""
import numpy as np
import pytest
import torch

from wick_amd.logits import adjust_logits_device
from wick_amd.sampler import DeviceSampler, SamplerConfig

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(x, vocab, repetition=None, presence=None, frequency=None, tokens=None, n_tokens=None, n_prompt=None,
              bias=None, masks=None, mask_row=None):
    """The rules one after the other in float32; bias: per row a list of (id, value)."""
    y = x.copy()
    f = np.float32
    for r in range(len(x)):
        ids = [] if tokens is None else tokens[r][:min(max(n_tokens[r], 0), tokens.shape[1])]
        first = 0 if n_prompt is None else max(n_prompt[r], 0)
        count = {}
        for i in ids[first:]:
            count[int(i)] = count.get(int(i), 0) + 1
        for i in sorted(set(int(i) for i in ids)):
            if i >= vocab:
                continue
            v = y[r, i]
            p = f(1) if repetition is None else repetition[r]
            v = v / p if v > 0 else f(v * p)
            if count.get(i):
                v = f(v - f(f((f(0) if frequency is None else frequency[r]) * f(count[i])) + (f(0) if presence is None else presence[r])))
            y[r, i] = v
        for i, v in dict(bias[r] if bias else []).items():
            if i < vocab:
                y[r, i] = f(y[r, i] + v)
        m = r if mask_row is None else mask_row[r]
        if masks is not None and 0 <= m < len(masks):
            i = np.arange(vocab)
            y[r, :vocab][(masks[m][i // 32] >> (i % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    return y


def run(x, vocab, rows=None, in_place=False, offset=0, out_stride=None, stream=None, bias=None, masks=None, **rules):
    """x [rows][stride] through the kernel, its arrays `offset` floats into their allocations."""
    rows, stride = x.shape
    out_stride = out_stride or stride
    a = torch.zeros(rows * stride + 4, device=DEV)
    src = a[offset:offset + rows * stride]
    src.copy_(torch.from_numpy(x).reshape(-1))
    o = torch.full((rows * out_stride + 4,), 7.0, device=DEV)
    dst = src if in_place else o[offset:offset + rows * out_stride]
    keep = {}

    def ptr(name, v):
        v = np.ascontiguousarray(v)
        keep[name] = torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).to(DEV)
        return keep[name].data_ptr()

    args = {}
    for name in ("repetition", "presence", "frequency"):
        if rules.get(name) is not None:
            args[name] = ptr(name, np.asarray(rules[name], np.float32))
    if rules.get("tokens") is not None:
        args["tokens"], args["tokens_stride"] = ptr("tokens", np.asarray(rules["tokens"], np.uint32)), rules["tokens"].shape[1]
        args["n_tokens"] = ptr("n_tokens", np.asarray(rules["n_tokens"], np.int32))
        if rules.get("n_prompt") is not None:
            args["n_prompt"] = ptr("n_prompt", np.asarray(rules["n_prompt"], np.int32))
    if bias:
        args["bias_start"] = ptr("bias_start", np.cumsum([0] + [len(b) for b in bias]).astype(np.int32))
        args["bias_ids"] = ptr("bias_ids", np.array([i for b in bias for i, _ in b] or [0], np.uint32))
        args["bias"] = ptr("bias", np.array([v for b in bias for _, v in b] or [0], np.float32))
        args["n_bias"] = sum(len(b) for b in bias)
    if masks is not None:
        args["mask"], args["masks"] = ptr("mask", masks), len(masks)
        if rules.get("mask_row") is not None:
            args["mask_row"] = ptr("mask_row", np.asarray(rules["mask_row"], np.int32))
    torch.cuda.synchronize()
    adjust_logits_device(src.data_ptr(), rows, vocab, dst.data_ptr(), stride=stride, out_stride=out_stride, stream=stream, **args)
    torch.cuda.synchronize()
    if not in_place:
        assert torch.equal(src.cpu(), torch.from_numpy(x).reshape(-1)) or np.array_equal(
            src.cpu().numpy().view(np.uint32), x.reshape(-1).view(np.uint32))
        assert bool((o[:offset] == 7).all()) and bool((o[offset + rows * out_stride:] == 7).all())
    return dst.cpu().numpy().reshape(rows, out_stride if not in_place else stride)


def make(rows, vocab, stride, tokens, biases, masked, seed):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((rows, stride)) * 3).astype(np.float32)
    case = dict(repetition=(1 + rng.random(rows) * 0.5).astype(np.float32), presence=rng.random(rows).astype(np.float32),
                frequency=rng.random(rows).astype(np.float32),
                tokens=np.minimum((rng.random((rows, tokens)) ** 3 * (vocab + 3)).astype(np.uint32), 2 ** 32 - 1),
                n_tokens=rng.integers(0, tokens + 1, rows), n_prompt=None)
    case["n_prompt"] = [int(rng.integers(0, n + 1)) for n in case["n_tokens"]]
    if tokens > 2:
        case["tokens"][:, 1] = 0xFFFFFFFF  # no id
    if biases:
        case["bias"] = [[(int(i), np.float32(rng.standard_normal() * 4)) for i in rng.integers(0, vocab, rng.integers(0, biases + 1))]
                        for _ in range(rows)]
    if masked:
        case["masks"] = rng.integers(0, 2 ** 32, (rows, (vocab + 31) // 32), dtype=np.uint32)
    return x, case


def equal(got, want):
    return np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])


@pytest.mark.parametrize("rows,vocab,stride,tokens,biases,masked", [
    (1, 1, 1, 3, 1, True), (1, 31, 33, 5, 2, True), (2, 1024, 1024, 300, 40, True), (3, 1025, 1031, 50, 0, False),
    (5, 4095, 4097, 1000, 7, True), (1, 49152, 49152, 200, 8, False), (70, 16387, 16387, 700, 30, True),
    (4, 151936, 151936, 3000, 300, True), (64, 32001, 32010, 0, 5, True),
])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_rules_to_the_bit(rows, vocab, stride, tokens, biases, masked, offset):
    x, case = make(rows, vocab, stride, max(tokens, 1), biases, masked, rows + vocab)
    if not tokens:
        case["n_tokens"] = [0] * rows
    got = run(x, vocab, offset=offset, **case)
    want = reference(x[:, :vocab], vocab, **case)
    assert equal(got[:, :vocab], want)
    assert (got[:, vocab:] == 7).all()  # behind a row's vocabulary nothing is written


def test_in_place_and_other_strides():
    x, case = make(6, 5000, 5003, 100, 10, True, 1)
    want = reference(x[:, :5000], 5000, **case)
    got = run(x, 5000, in_place=True, **case)
    assert equal(got[:, :5000], want) and np.array_equal(got[:, 5000:], x[:, 5000:])
    assert equal(run(x, 5000, out_stride=5100, **case)[:, :5000], want)


def test_each_rule_alone():
    x, case = make(3, 3001, 3001, 200, 20, True, 2)
    tok = {k: case[k] for k in ("tokens", "n_tokens", "n_prompt")}
    for some in [{}, tok, tok | {"repetition": case["repetition"]}, tok | {"presence": case["presence"]},
                 tok | {"frequency": case["frequency"]}, {"bias": case["bias"]}, {"masks": case["masks"]},
                 {k: v for k, v in tok.items() if k != "n_prompt"} | {"frequency": case["frequency"]}]:
        assert equal(run(x, 3001, **some), reference(x, 3001, **some)), sorted(some)


def test_counts_out_of_range_and_repeated_biases():
    x, case = make(4, 2000, 2000, 50, 0, False, 3)
    case["n_tokens"], case["n_prompt"] = [-5, 50, 1000, 20], [3, -7, 2000, 20]
    case["bias"] = [[(7, np.float32(1)), (7, np.float32(2)), (3, np.float32(5)), (7, np.float32(4))], [],
                    [(2000, np.float32(1)), (2 ** 32 - 1, np.float32(1))], [(1999, np.float32(-1))]]
    assert equal(run(x, 2000, **case), reference(x, 2000, **case))


def test_grammars_shared_absent_and_empty():
    x, case = make(5, 1500, 1500, 30, 5, False, 4)
    masks = np.zeros((3, 47), np.uint32)
    masks[1] = 0xFFFFFFFF
    masks[2, 3] = 1 << 5
    x[:, 17] = np.nan  # hidden or not: minus infinity hides it too
    x[:, 18] = np.inf
    case |= dict(masks=masks, mask_row=[0, 1, 2, -1, 9])
    got = run(x, 1500, **case)
    assert equal(got, reference(x, 1500, **case))
    assert (got[0] == -np.inf).all()  # a grammar that allows nothing
    assert np.isfinite(got[2]).sum() == 1 and np.isnan(got[3, 17])


def test_the_samplers_repetition_penalty():
    """With a repetition penalty alone the rows are what the sampler's own penalty leaves."""
    x, case = make(1, 49152, 49152, 500, 0, False, 5)
    case = dict(repetition=np.array([1.3], np.float32), tokens=case["tokens"], n_tokens=[500])
    got = run(x, 49152, **case)
    logits = x[0].copy()
    with DeviceSampler(SamplerConfig(temperature=0.0, repetition_penalty=1.3), 49152) as s:
        best = s.sample(logits, case["tokens"][0])
    assert np.array_equal(got[0].view(np.uint32), logits.view(np.uint32)) and best == int(np.argmax(got[0]))


def test_on_a_stream_and_in_a_graph():
    x, case = make(3, 6000, 6000, 60, 6, True, 6)
    want = reference(x, 6000, **case)
    assert equal(run(x, 6000, stream=torch.cuda.Stream().cuda_stream, **case), want)
    t = torch.from_numpy(x).to(DEV)
    out = torch.zeros_like(t)
    rep, tok = torch.full((3,), 1.2, device=DEV), torch.from_numpy(case["tokens"].view(np.int32)).to(DEV)
    n = torch.tensor([60, 3, 0], dtype=torch.int32, device=DEV)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        adjust_logits_device(t.data_ptr(), 3, 6000, out.data_ptr(), repetition=rep.data_ptr(), tokens=tok.data_ptr(),
                             tokens_stride=60, n_tokens=n.data_ptr(), stream=stream.cuda_stream)
    for i in range(3):
        with torch.cuda.stream(stream):
            n.copy_(torch.tensor([60 - i, 3 + i, i], dtype=torch.int32))
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        want = reference(x, 6000, repetition=np.full(3, 1.2, np.float32), tokens=case["tokens"], n_tokens=[60 - i, 3 + i, i])
        assert equal(out.cpu().numpy(), want), i
        assert float(torch.ones(10, device=DEV).sum()) == 10.0
