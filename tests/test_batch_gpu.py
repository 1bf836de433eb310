"""The batch's attention (include/wick_hip_batch.h) against softmax(q k / sqrt(d)) v in
64 bits, at the lengths, head groups and plans where it can go wrong.

Tolerances, with u = 2^-24 (half an f32 step) and A = max_j sum_i |q_i k_ji| / sqrt(d) for
a row.  A score is summed by N = 6 d / 16 instructions (3 d / 16 on a bf16 cache), each rounding
the sum once or twice, from parts that are off by 2 u together with q's scaling: off by (2 N + 4)
u A.  A weight's relative error is that of its score and of the reference score, with the
exponential's two steps and the argument's rounding on a range of 2 A: (4 N + 8 + 3) u A + 4 u;
its share of the sum in the denominator doubles it.  The sum over n keys is rounded once or twice
an instruction, 6 of them for 16 keys, and four waves, the states and the division
add a few roundings: (2 * 6 n / 16 + 20) u.  All of it relative to sum_j w_j |v_j|.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from wick_amd import DeviceKvCache, _native
from wick_amd.batch import DeviceBatch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = "cuda"


def reference(q, k, v, last, heads, kv_heads, parts):
    """q [rows][heads][d], k and v [kv_heads][n][d] (64 bits), row i sees keys 0..=last[i]:
    (result, tolerance), [rows][heads][d]."""
    group, d, n = heads // kv_heads, q.shape[2], k.shape[1]
    hidden = torch.arange(n, device=q.device)[None, :] > last[:, None]
    out, tol = torch.empty_like(q), torch.empty_like(q)
    instr = (6 if parts == 3 else 3) * max(d // 16, 1)
    seen = (last + 1).double()[:, None]
    for h in range(heads):
        # hidden keys and values may be anything: left out before any product
        kk, vv = k[h // group], v[h // group]
        s = (q[:, h] @ torch.nan_to_num(kk, 0, 0, 0).t() / math.sqrt(d)).masked_fill(hidden, -math.inf)
        a = (q[:, h].abs() @ torch.nan_to_num(kk, 0, 0, 0).abs().t() / math.sqrt(d)).masked_fill(hidden, 0).amax(-1, keepdim=True)
        w = torch.softmax(s, -1)
        vz = torch.nan_to_num(vv, 0, 0, 0)
        out[:, h] = w @ vz
        tol[:, h] = (w @ vz.abs()) * U * (2 * ((4 * instr + 11) * a + 4) + 0.75 * seen + 20) + 1e-37
    return out, tol


class Case:
    """Random caches and queries of one plan, the handle filled the way a program does it."""

    def __init__(self, heads, kv_heads, d, start, t, prefix=0, dtype="f32", seed=0, layers=1, layer=0, capacity=None,
                 sharp=1.0, prefix_capacity=None):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.heads, self.kv_heads, self.d, self.start, self.t, self.prefix = heads, kv_heads, d, list(start), list(t), prefix
        self.n, self.layer, self.parts = len(t), layer, 3 if dtype == "f32" else 1
        self.lens = [a + b for a, b in zip(start, t)]
        self.capacity = capacity or max(self.lens)
        kvd = kv_heads * d
        self.dtype = torch.float32 if dtype == "f32" else torch.bfloat16

        def rows(n):
            return torch.randn(n, kvd, generator=g, device=DEV)

        self.pk, self.pv = rows(prefix), rows(prefix)
        self.k, self.v = [rows(n) for n in self.lens], [rows(n) for n in self.lens]
        self.q = torch.randn(sum(t), heads * d, generator=g, device=DEV) * sharp
        self.b = DeviceBatch(layers, heads, kv_heads, d, self.n, self.capacity,
                             prefix if prefix_capacity is None else prefix_capacity,
                             max(1, sum(self.lens)), dtype)

    def fill(self):
        """The prefix and all positions, the new ones among them."""
        torch.cuda.synchronize()
        if self.prefix:
            self.b.write_prefix_device(self.layer, 0, self.prefix, self.pk.data_ptr(), self.pv.data_ptr())
        k, v = torch.cat(self.k), torch.cat(self.v)
        torch.cuda.synchronize()
        self.b.plan([0] * self.n, self.lens, self.prefix)
        if len(k):
            self.b.append_device(self.layer, k.data_ptr(), v.data_ptr())
        self.b.plan(self.start, self.t, self.prefix)
        self.b.synchronize()
        return self

    def run(self, q=None):
        q = self.q if q is None else q
        att = torch.full((len(q) + 3, q.shape[1]), 7.0, device=DEV)
        torch.cuda.synchronize()
        self.b.attention_device(self.layer, q.data_ptr(), att.data_ptr())
        self.b.synchronize()
        assert bool((att[len(q):] == 7.0).all()), "rows behind the last token were written"
        return att[:len(q)]

    def want(self):
        out, tol, at = [], [], 0
        for s in range(self.n):
            if not self.t[s]:
                continue
            kv = [torch.cat([p, x]).to(self.dtype).double().view(-1, self.kv_heads, self.d).transpose(0, 1).contiguous()
                  for p, x in ((self.pk, self.k[s]), (self.pv, self.v[s]))]
            last = self.prefix + self.start[s] + torch.arange(self.t[s], device=DEV)
            q = self.q[at:at + self.t[s]].double().view(-1, self.heads, self.d)
            o, e = reference(q, *kv, last, self.heads, self.kv_heads, self.parts)
            out.append(o.reshape(self.t[s], -1))
            tol.append(e.reshape(self.t[s], -1))
            at += self.t[s]
        return torch.cat(out), torch.cat(tol)

    def check(self, got=None):
        got = self.run() if got is None else got
        want, tol = self.want()
        err = (got.double() - want).abs()
        worst = float((err / tol).max())
        print(f"worst error / tolerance {worst:.3f}, max abs {float(err.max()):.2e}", flush=True)
        assert bool(torch.isfinite(got).all())
        assert worst <= 1.0
        return got


SHAPES = [(1, 1, 16), (6, 2, 32), (9, 3, 64), (14, 2, 64), (32, 8, 128), (40, 1, 64)]
PLANS = [
    # (start, t, prefix)
    ([0], [1], 0),
    ([0, 0, 0], [1, 33, 7], 0),
    ([5, 0, 127, 300], [1, 1, 1, 1], 0),
    ([0, 63, 0, 0], [0, 2, 0, 70], 0),
    ([0, 0], [1, 1], 1),
    ([31, 0, 255, 16], [1, 1, 1, 1], 129),
    ([3, 0, 40], [5, 0, 90], 300),
    ([700, 1000], [37, 1], 2049),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", SHAPES)
@pytest.mark.parametrize("start,t,prefix", PLANS)
def test_parity(heads, kv_heads, d, start, t, prefix, dtype):
    Case(heads, kv_heads, d, start, t, prefix, dtype, seed=heads + prefix).fill().check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,start,t,prefix", [
    (32, 8, 128, [0, 0, 0], [401, 97, 300], 0),        # rows enough to fill the GPU: no joined states
    (32, 8, 128, [0, 10, 0, 33], [350, 1, 280, 1], 150),  # such sequences next to single tokens
    (14, 2, 64, [0, 500], [1031, 1200], 0),
    (9, 3, 64, [0] * 5, [1000, 1, 640, 3, 900], 77),
    (16, 8, 16, [0], [1500], 0),
])
def test_many_rows(heads, kv_heads, d, start, t, prefix, dtype):
    Case(heads, kv_heads, d, start, t, prefix, dtype, seed=d).fill().check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_prefix_many_sequences(dtype):
    start = [int(x) for x in np.random.default_rng(3).integers(0, 200, 33)]
    Case(32, 8, 128, start, [1] * 33, 9001, dtype, seed=3).fill().check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [4, 5, 8, 9, 13, 16, 17, 33])
def test_rows_against_a_long_prefix(n, dtype):
    """Single tokens of n sequences, 4 rows each: one to three narrow items or wide ones, some of their rows empty."""
    Case(32, 8, 128, [(17 * s) % 50 for s in range(n)], [1] * n, 8300, dtype, seed=n).fill().check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
def test_many_states_of_a_row(d, dtype):
    """One token over a long context: its keys are dealt to over a hundred workgroups."""
    Case(1, 1, d, [29000], [1], 0, dtype, seed=d).fill().check()
    Case(4, 2, d, [700], [1], 30001, dtype, seed=d + 1).fill().check()


def test_plans_of_all_kinds():
    """Steps drawn at random over the ranges where the plan changes its kind: sequences alone or
    together, narrow and wide items, whole and split."""
    rng = np.random.default_rng(60)
    for i in range(24):
        heads, kv_heads, d = [(9, 3, 64), (14, 2, 64), (16, 8, 128), (32, 8, 128), (32, 4, 64), (5, 1, 32)][i % 6]
        n = int(rng.integers(1, 20))
        prefix = int(rng.choice([0, 0, 90, 400, 3000]))
        one = rng.random() < 0.4
        start = [int(x) for x in rng.integers(0, rng.choice([5, 300, 900]), n)]
        t = [1 if one else int(x) for x in rng.integers(0, rng.choice([6, 60, 400]), n)]
        if sum(t) == 0:
            t[0] = 1
        print(i, heads, kv_heads, d, start, t, prefix, flush=True)
        Case(heads, kv_heads, d, start, t, prefix, "bf16" if i % 3 == 2 else "f32", seed=100 + i).fill().check()


def test_sharp_scores():
    """Score deviations of 40: weights that vanish, the reference maximum rising over the keys."""
    Case(8, 2, 64, [100, 900], [20, 1], 500, sharp=40.0, seed=4).fill().check()
    c = Case(4, 4, 64, [0], [700], 0, sharp=1.0, seed=5)
    c.k[0] *= torch.linspace(0.01, 12, 700, device=DEV)[:, None]  # the last keys weigh most
    c.fill().check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_position_is_its_value(dtype):
    """A context of one position has weight 1: the value itself, to the bit."""
    c = Case(8, 2, 128, [0, 0], [1, 1], 0, dtype, seed=6).fill()
    got = c.run().view(2, 2, 4, 128)
    for s in range(2):
        v = c.v[s].to(c.dtype).float().view(2, 1, 128)
        assert torch.equal(got[s], v.expand(2, 4, 128))


def test_bit_stable_and_in_place():
    c = Case(14, 2, 64, [100, 3, 0], [1, 20, 1], 1000, seed=7).fill()
    a = c.run()
    assert torch.equal(a, c.run())
    q = c.q.clone()
    torch.cuda.synchronize()
    c.b.attention_device(0, q.data_ptr(), q.data_ptr())
    c.b.synchronize()
    assert torch.equal(a, q)


def test_layers_and_capacities_apart():
    """Layer 1 of 3, capacities larger than what is used: nothing else is read or written."""
    c = Case(8, 2, 64, [4, 0, 9], [3, 2, 1], 50, seed=8, layers=3, layer=1, capacity=64, prefix_capacity=70).fill()
    c.check()
    for layer in (0, 2):
        for s in (-1, 0, 1, 2):
            k, v = c.b.read(layer, s, 0, 64)
            assert not k.any() and not v.any()
    k, v = c.b.read(1, 1, 0, 64)
    assert np.array_equal(k[:2], c.k[1].cpu().numpy()) and np.array_equal(v[:2], c.v[1].cpu().numpy())
    assert not k[2:].any() and not v[2:].any()
    k, v = c.b.read(1, -1, 0, 70)
    assert np.array_equal(k[:50], c.pk.cpu().numpy()) and not k[50:].any() and not v[50:].any()


def test_bf16_rounds_to_nearest():
    c = Case(2, 1, 32, [0], [9], 5, "bf16", seed=9).fill()
    k, v = c.b.read(0, 0, 0, 9)
    assert np.array_equal(k, c.k[0].bfloat16().float().cpu().numpy())
    assert np.array_equal(v, c.v[0].bfloat16().float().cpu().numpy())
    k, v = c.b.read(0, -1, 0, 5)
    assert np.array_equal(k, c.pk.bfloat16().float().cpu().numpy())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 2, 64), (32, 8, 128), (3, 3, 16)])
def test_hidden_positions_never_count(heads, kv_heads, d, bad, dtype):
    """Positions behind a sequence's last, behind the used prefix and behind a token's own
    hold infinities or NaN: tokens that do not see them are as if they were not there."""
    c = Case(heads, kv_heads, d, [0, 10, 0], [40, 1, 3], 60, dtype, seed=10, capacity=300, prefix_capacity=200).fill()
    clean = c.check()
    kvd = kv_heads * d
    junk = torch.full((300, kvd), bad, device=DEV)
    torch.cuda.synchronize()
    c.b.write_prefix_device(0, 60, 140, junk.data_ptr(), junk.data_ptr())
    for s in range(3):
        for at in range(c.lens[s], 300, 50):
            c.b.plan([at] * 3, [min(50, 300 - at) if i == s else 0 for i in range(3)], 60)
            c.b.append_device(0, junk.data_ptr(), junk.data_ptr())
    c.b.plan(c.start, c.t, 60)
    assert torch.equal(c.run(), clean)
    # position 25 of sequence 0: seen by its tokens 25.. alone
    c.b.plan([25, 0, 0], [1, 0, 0], 60)
    c.b.append_device(0, junk.data_ptr(), junk.data_ptr())
    c.b.plan(c.start, c.t, 60)
    got = c.run()
    want, tol = c.want()
    unseen = torch.ones(len(got), dtype=torch.bool, device=DEV)
    unseen[25:40] = False
    assert bool(((got - want).abs() <= tol)[unseen].all())
    assert not bool(torch.isfinite(got[~unseen]).any())


def test_values_without_parts():
    """Keys and values next to f32's largest, whose bf16 parts overflow: the row is computed in f32."""
    c = Case(4, 2, 64, [0, 5], [6, 1], 10, seed=11)
    big = 3.4e38
    c.k[0][2, 0] = big
    c.q[:, 0] *= 1e-38
    c.q[:, 64] *= 1e-38
    c.v[1][3, 70] = big
    c.fill()
    got, (want, tol) = c.run(), c.want()
    assert bool(torch.isfinite(got).all())
    assert bool(((got.double() - want).abs() <= tol).all())


SCALES = [(1e20, 1e-20, 1e-30), (1e-18, 1e18, 1e30), (1.0, 1.0, 1e-20)]


@pytest.mark.parametrize("q_by,k_by,v_by", SCALES)
@pytest.mark.parametrize("n", [1, 90])
def test_values_of_any_scale(q_by, k_by, v_by, n):
    """Queries, keys and values far from 1, narrow items and wide: as exact as near it."""
    c = Case(8, 2, 64, [40, 0], [n, n], 600, seed=13 + n)
    c.q *= q_by
    for x in [c.pk] + c.k:
        x *= k_by
    for x in [c.pv] + c.v:
        x *= v_by
    c.fill().check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_load_prefix_and_the_cache_it_came_from(dtype):
    """A prompt in a DeviceKvCache becomes the prefix; one more token attends as the cache's own call."""
    rng = np.random.default_rng(12)
    heads, kvh, d, n = 14, 2, 64, 333
    k, v = (rng.standard_normal((n + 1, kvh * d), dtype=np.float32) for _ in range(2))
    q = rng.standard_normal((1, heads * d), dtype=np.float32)
    with DeviceKvCache(2, n + 20, kvh, d) as kv, DeviceBatch(2, heads, kvh, d, 3, 8, prefix_capacity=n + 7, dtype=dtype) as b:
        for layer in (0, 1):
            kv.append(layer, 0, k, v)
        b.load_prefix(kv, n)
        for layer in (0, 1):
            pk, pv = b.read(layer, -1, 0, n + 7)
            held = [torch.from_numpy(x[:n]).to(torch.bfloat16 if dtype == "bf16" else torch.float32).float().numpy() for x in (k, v)]
            assert np.array_equal(pk[:n], held[0]) and np.array_equal(pv[:n], held[1]) and not pk[n:].any()
        b.plan([0, 0, 0], [1, 1, 1], n)
        want = kv.attention(1, heads, q, n)
        b.append(1, np.repeat(k[n:], 3, 0), np.repeat(v[n:], 3, 0))
        got = b.attention(1, np.repeat(q, 3, 0))
        # f32: two orders of the same sums (see the module's tolerances; A < 30 here).  bf16: a
        # key is off by up to 2^-8 of itself, a score by 2^-8 A / sqrt(d) at one deviation of its d
        # errors, a weight by e^that; the values by 2^-8 of their mean: 0.05 covers three deviations
        assert np.abs(got - want).max() < (2e-5 if dtype == "f32" else 0.05)
        assert np.array_equal(got[0], got[1]) and np.array_equal(got[1], got[2])


def test_refusals():
    with DeviceBatch(2, 4, 2, 64, 3, 16, prefix_capacity=8, max_tokens=20) as b:
        x = torch.zeros(20 * 256 + 4, device=DEV)
        p = x.data_ptr()
        for call in (lambda: b.append_device(0, p, p), lambda: b.attention_device(0, p, p)):
            with pytest.raises(_native.WickHipError, match="plan"):
                call()
        for start, t, prefix, says in [([0, 0, 0], [1, 1, -1], 0, "sequence 2"), ([-1, 0, 0], [1, 1, 1], 0, "sequence 0"),
                                       ([0, 16, 0], [1, 1, 1], 0, "sequence 1"), ([0, 0, 0], [16, 4, 1], 0, "max_tokens"),
                                       ([0, 0, 0], [1, 1, 1], 9, "prefix"), ([0, 0, 0], [1, 1, 1], -1, "prefix"),
                                       ([2 ** 31 - 1, 0, 0], [2 ** 31 - 1, 1, 1], 0, "sequence 0")]:
            with pytest.raises(_native.WickHipError, match=says):
                b.plan(start, t, prefix)
        with pytest.raises(ValueError):
            b.plan([0, 0], [1, 1])
        b.plan([0, 0, 0], [2, 0, 1], 8)
        for call, says in [(lambda: b.attention_device(2, p, p), "layer"), (lambda: b.attention_device(-1, p, p), "layer"),
                           (lambda: b.attention_device(0, p + 4, p), "aligned"), (lambda: b.attention_device(0, p, p + 8), "aligned"),
                           (lambda: b.attention_device(0, None, p), "null"), (lambda: b.append_device(0, p, None), "null"),
                           (lambda: b.append_device(0, p + 4, p), "aligned"),
                           (lambda: b.write_prefix_device(0, 8, 1, p, p), "prefix capacity"),
                           (lambda: b.write_prefix_device(0, 0, 0, p, p), "t must"),
                           (lambda: b.read(0, 3, 0, 1), "sequence"), (lambda: b.read(0, -1, 8, 1), "capacity"),
                           (lambda: b.read(0, 0, 0, 0), "positions")]:
            with pytest.raises(_native.WickHipError, match=says):
                call()
        with pytest.raises(ValueError):
            b.attention(0, np.zeros((2, 256), np.float32))
        with DeviceKvCache(2, 32, 2, 32) as kv, pytest.raises(_native.WickHipError, match="the cache has"):
            b.load_prefix(kv, 4)
        with DeviceKvCache(2, 32, 2, 64) as kv, pytest.raises(_native.WickHipError, match="exceed"):
            b.load_prefix(kv, 9)


def test_nothing_planned_is_nothing_to_do():
    with DeviceBatch(1, 4, 2, 64, 2, 16) as b:
        b.plan([0, 3], [0, 0])
        b.append_device(0, None, None)
        b.attention_device(0, None, None)
        assert b.attention(0, np.zeros((0, 256), np.float32)).shape == (0, 256)


def test_two_handles_on_two_streams():
    """Calls of two handles queued on two streams at once, and one handle moved between streams."""
    cs = [Case(8, 2, 64, [50, 0], [1, 90], 400, seed=20 + i).fill() for i in range(2)]
    want = [c.run() for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    atts = [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    for c, s in zip(cs, streams):
        c.b.set_stream(s.cuda_stream)
    for _ in range(5):
        for c, a in zip(cs, atts):
            c.b.attention_device(0, c.q.data_ptr(), a.data_ptr())
    torch.cuda.synchronize()
    assert all(torch.equal(a, w) for a, w in zip(atts, want))
    a = torch.zeros_like(want[0])
    torch.cuda.synchronize()
    for i in range(6):
        cs[0].b.set_stream([None, streams[0].cuda_stream, streams[1].cuda_stream][i % 3])
        cs[0].b.plan([50, 0], [1, 90], 400)
        cs[0].b.attention_device(0, cs[0].q.data_ptr(), a.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(a, want[0])


@pytest.mark.parametrize("dtype,prefix", [("f32", 260), ("bf16", 260), ("f32", 0)])
def test_graph_follows_the_plan(dtype, prefix):
    """A captured append + attention of single tokens replays for positions that move on, under each
    step's plan, and writes NaN under a plan of other tokens."""
    heads, kvh, d, n, steps = 8, 2, 64, 5, 6
    g = torch.Generator(device=DEV).manual_seed(30)
    start0 = [0, 3, 90, 127, 200]
    step = 25 if prefix else 90  # without a prefix the first plan joins nothing, the later ones do
    cap = 700
    pk, pv = (torch.randn(prefix, kvh * d, generator=g, device=DEV) for _ in range(2))
    old = [[torch.randn(x, kvh * d, generator=g, device=DEV) for _ in range(2)] for x in start0]
    new = torch.randn(steps, 2, n, kvh * d, generator=g, device=DEV)
    qs = torch.randn(steps, n, heads * d, generator=g, device=DEV)
    torch.cuda.synchronize()

    def make():
        b = DeviceBatch(1, heads, kvh, d, n, cap, prefix, 500, dtype)
        if prefix:
            b.write_prefix_device(0, 0, prefix, pk.data_ptr(), pv.data_ptr())
        b.plan([0] * n, start0, prefix)
        k, v = (torch.cat([o[i] for o in old]) for i in (0, 1))
        torch.cuda.synchronize()
        b.append_device(0, k.data_ptr(), v.data_ptr())
        b.synchronize()
        return b

    def at(i):  # far apart positions, so that later plans have more items than the captured one
        return [x + step * i for x in start0]

    eager, want = make(), []
    for i in range(steps):
        att = torch.empty(n, heads * d, device=DEV)
        torch.cuda.synchronize()
        eager.plan(at(i), [1] * n, prefix)
        eager.append_device(0, new[i, 0].data_ptr(), new[i, 1].data_ptr())
        eager.attention_device(0, qs[i].data_ptr(), att.data_ptr())
        eager.synchronize()
        want.append(att)

    b = make()
    q, kv, att = torch.empty(n, heads * d, device=DEV), torch.empty(2, n, kvh * d, device=DEV), torch.empty(n, heads * d, device=DEV)
    stream = torch.cuda.Stream()
    b.set_stream(stream.cuda_stream)
    b.plan(at(0), [1] * n, prefix)
    shape = b.shape()
    b.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        b.append_device(0, kv[0].data_ptr(), kv[1].data_ptr())
        b.attention_device(0, q.data_ptr(), att.data_ptr())
        with pytest.raises(_native.WickHipError, match="captured"):
            b.plan(at(0), [1] * n, prefix)
        with pytest.raises(_native.WickHipError, match="captured"):
            b.attention(0, np.zeros((n, heads * d), np.float32))
    for i in range(steps):
        with torch.cuda.stream(stream):
            q.copy_(qs[i])
            kv.copy_(new[i])
            att.zero_()
            b.plan(at(i), [1] * n, prefix)
            assert b.shape() == shape
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(att, want[i]), i
        assert float(torch.randn(100, device=DEV).sum()) != 0.0  # the program's own work in between
    before = b.read(0, 0, 0, cap)
    b.plan(at(0), [1, 1, 1, 1, 0], prefix)
    assert b.shape() != shape
    with torch.cuda.stream(stream):
        graph.replay()
    torch.cuda.synchronize()
    assert bool(torch.isnan(att).all())
    after = b.read(0, 0, 0, cap)
    assert np.array_equal(before[0], after[0]) and np.array_equal(before[1], after[1])


def test_shapes_are_known_again():
    """A step of other tokens in between leaves a shape's number and its graphs; past 32 others a new number."""
    c = Case(8, 2, 64, [40, 90, 7], [1, 1, 1], 150, seed=31).fill()
    want = c.check()
    n, stream = c.b.shape(), torch.cuda.Stream()
    q, att = c.q.clone(), torch.empty_like(want)
    torch.cuda.synchronize()
    c.b.set_stream(stream.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        c.b.attention_device(c.layer, q.data_ptr(), att.data_ptr())

    def replay():
        c.b.plan(c.start, c.t, c.prefix)
        with torch.cuda.stream(stream):
            att.zero_()
            graph.replay()
        torch.cuda.synchronize()

    for _ in range(3):
        c.b.plan([0, 0, 0], [30, 0, 5], c.prefix)
        assert c.b.shape() != n
        replay()
        assert c.b.shape() == n and torch.equal(att, want)
    for i in range(31):
        c.b.plan([0, 0, 0], [0, i + 2, 1], c.prefix)
    replay()
    assert c.b.shape() == n and torch.equal(att, want)
    for i in range(32):
        c.b.plan([0, 0, 0], [0, 2, i + 2 if i != 1 else 0], c.prefix)
    replay()
    assert c.b.shape() not in (0, n) and bool(torch.isnan(att).all())
    assert torch.equal(c.run(), want)


def test_offsets_past_32_bits():
    """The second sequence's and the second kv head's positions lie past 2^32 bytes and 2^31 values."""
    heads, kvh, d, cap = 4, 2, 128, 9_000_000
    with DeviceBatch(1, heads, kvh, d, 2, cap, prefix_capacity=cap, max_tokens=64, dtype="bf16") as b:
        g = torch.Generator(device=DEV).manual_seed(40)
        k, v = (torch.randn(40, kvh * d, generator=g, device=DEV) for _ in range(2))
        q = torch.randn(40, heads * d, generator=g, device=DEV)
        torch.cuda.synchronize()
        # zeros before: scores of 0 and values of 0 for most of a context of 9 million positions
        start = cap - 40
        b.plan([0, start], [0, 40], 0)
        b.append_device(0, k.data_ptr(), v.data_ptr())
        b.write_prefix_device(0, start, 40, k.data_ptr(), v.data_ptr())
        rk, rv = b.read(0, 1, start, 40)
        assert np.array_equal(rk, k.bfloat16().float().cpu().numpy()) and np.array_equal(rv, v.bfloat16().float().cpu().numpy())
        rk, _ = b.read(0, -1, start, 40)
        assert np.array_equal(rk, k.bfloat16().float().cpu().numpy())
        att = torch.empty(40, heads * d, device=DEV)
        torch.cuda.synchronize()
        for prefix in (0, cap):
            b.plan([0, start], [0, 40], prefix)
            b.attention_device(0, q.data_ptr(), att.data_ptr())
            b.synchronize()
            kk, vv = (x.bfloat16().double().view(40, kvh, d) for x in (k, v))
            scale = 1 / math.sqrt(d)
            for h in range(heads):
                s = q.view(40, heads, d)[:, h].double() @ kk[:, h // 2].t() * scale
                seen = torch.tril(torch.ones(40, 40, dtype=torch.bool, device=DEV))
                e = torch.exp(s)
                w = torch.where(seen, e, 0.0)
                if prefix:
                    w = w + e  # the same rows at the end of the prefix, all seen
                total = w.sum(-1, keepdim=True) + start * (2 if prefix else 1)
                want = w @ vv[:, h // 2] / total
                got = att.view(40, heads, d)[:, h].double()
                # n u of the long sum in the denominator is held down by its 32-bit states: 256
                # workgroups and 4 waves of at most 9e6 / 16 additions of 1 each lose 2^-24 * 3e3 of it
                assert float(((got - want).abs() / (w @ vv[:, h // 2].abs() / total)).max()) < 1e-3


def test_prompts_answers_and_rules_together():
    """A serving run: a prompt's cache becomes the prefix, questions of different lengths behind it,
    then single tokens chosen after penalties, biases and grammars -- every step against 64 bits."""
    from wick_amd.logits import adjust_logits_device
    heads, kvh, d, vocab, hidden, P = 8, 2, 64, 777, 96, 210
    g = torch.Generator(device="cpu").manual_seed(50)

    def mat(*s):
        return torch.randn(*s, generator=g).to(DEV) / math.sqrt(s[0])

    emb, wq, wk, wv, wo = mat(vocab, hidden) * 28, mat(hidden, heads * d), mat(hidden, kvh * d), mat(hidden, kvh * d), mat(heads * d, vocab)
    prompt = torch.randint(0, vocab, (P,), generator=g).to(DEV)
    questions = [torch.randint(0, vocab, (n,), generator=g).to(DEV) for n in (17, 1, 64)]
    n, steps, words = len(questions), 4, (vocab + 31) // 32
    rep, pres, freq = (torch.tensor(x, device=DEV) for x in ([1.3, 1.0, 1.1], [0.5, 0.0, 0.2], [0.2, 0.3, 0.0]))
    bias_start = torch.tensor([0, 1, 1, 3], dtype=torch.int32, device=DEV)
    bias_ids, bias = torch.tensor([5, 700, 9], dtype=torch.int32, device=DEV), torch.tensor([3.0, -8.0, 2.0], device=DEV)
    mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (1, words), generator=g).to(torch.int32).to(DEV)
    mask_row = torch.tensor([-1, 0, 0], dtype=torch.int32, device=DEV)
    bits = ((mask[0][torch.arange(vocab, device=DEV) // 32] >> (torch.arange(vocab, device=DEV) % 32)) & 1).bool()

    kv = DeviceKvCache(1, P, kvh, d)
    kv.append(0, 0, (emb[prompt] @ wk).cpu().numpy(), (emb[prompt] @ wv).cpu().numpy())
    b = DeviceBatch(1, heads, kvh, d, n, 80, prefix_capacity=P)
    b.load_prefix(kv, P)
    tokens = torch.zeros(n, 80, dtype=torch.int32, device=DEV)
    lens = [len(x) for x in questions]
    for s, x in enumerate(questions):
        tokens[s, :len(x)] = x
    n_prompt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    start, t = [0] * n, list(lens)
    ctx = [torch.cat([prompt, x]) for x in questions]
    for step in range(steps):
        ids = torch.cat([c[P + a:P + a + m] for c, a, m in zip(ctx, start, t)])
        x = emb[ids]
        q, k, v = x @ wq, x @ wk, x @ wv
        att = torch.empty_like(q)
        torch.cuda.synchronize()
        b.plan(start, t, P)
        b.append_device(0, k.data_ptr(), v.data_ptr())
        b.attention_device(0, q.data_ptr(), att.data_ptr())
        b.synchronize()
        ends = torch.tensor(t, device=DEV).cumsum(0) - 1
        logits = att[ends] @ wo
        out = torch.empty_like(logits)
        n_tokens = torch.tensor([a + m for a, m in zip(start, t)], dtype=torch.int32, device=DEV)
        torch.cuda.synchronize()
        adjust_logits_device(logits.data_ptr(), n, vocab, out.data_ptr(), repetition=rep.data_ptr(), presence=pres.data_ptr(),
                             frequency=freq.data_ptr(), tokens=tokens.data_ptr(), tokens_stride=80, n_tokens=n_tokens.data_ptr(),
                             n_prompt=n_prompt.data_ptr(), bias_start=bias_start.data_ptr(), bias_ids=bias_ids.data_ptr(),
                             bias=bias.data_ptr(), n_bias=3, mask=mask.data_ptr(), mask_row=mask_row.data_ptr(), masks=1)
        torch.cuda.synchronize()
        chosen = out.argmax(-1)
        for s in range(n):
            xs = emb[ctx[s]].double()
            kk, vv = ((xs @ w.double()).view(-1, kvh, d) for w in (wk, wv))
            qq = (xs[-1:] @ wq.double()).view(heads, d)
            y = torch.cat([torch.softmax(qq[h] @ kk[:, h // 4].t() / 8, -1) @ vv[:, h // 4] for h in range(heads)]) @ wo.double()
            own = ctx[s][P:]
            seen = own.unique()
            y[seen] = torch.where(y[seen] > 0, y[seen] / rep[s].double(), y[seen] * rep[s].double())
            new, count = own[lens[s]:].unique(return_counts=True)
            y[new] -= freq[s].double() * count + pres[s].double()
            for e in range(int(bias_start[s]), int(bias_start[s + 1])):
                y[bias_ids[e]] += bias[e].double()
            if s:
                y[~bits] = -math.inf
            fin = torch.isfinite(y)
            assert torch.equal(torch.isfinite(out[s]), fin)
            # f32 projections of width 96 and 512 on values of a few units: 1e-3 is 100 times their roundings
            assert float((out[s].double() - y)[fin].abs().max()) < 1e-3
            best = y.topk(2)[0]
            if float(best[0] - best[1]) > 2e-3:
                assert int(chosen[s]) == int(y.argmax())
            tokens[s, start[s] + t[s]] = int(chosen[s])
            ctx[s] = torch.cat([ctx[s], chosen[s:s + 1]])
        start, t = [a + m for a, m in zip(start, t)], [1] * n
    b.close()
    kv.close()
