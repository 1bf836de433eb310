"""The batch's attention at the ends of f32's range: scores next to its lowest value, values whose
unweighted sums pass its largest.

Tolerances as in test_batch_gpu; where all keys of a row are the same its weights are too, whatever
their score, and the result is off by the sums' roundings alone: (0.75 n + 20) u sum_j w_j |v_j|.
"""
import math

import pytest
import torch

from test_batch_gpu import DEV, U, Case

pytestmark = pytest.mark.gpu
LARGEST = 3.4028234663852886e38  # of f32

# heads, kv_heads, d, start, t, prefix: whole narrow items, whole wide ones, split ones of both kinds
STEPS = [
    (4, 2, 64, [0, 3], [5, 1], 0),
    (3, 3, 16, [0, 0], [1, 30], 20),
    (32, 8, 128, [0, 10], [400, 333], 0),
    (8, 2, 64, [40, 0, 9], [1, 1, 1], 9000),
    (32, 8, 128, [50, 0, 7], [40, 1, 1], 12000),
    (6, 2, 32, [700, 1000], [37, 1], 2049),
]


def means(c):
    """Each row's mean of the values that it sees, and of their magnitudes (64 bits)."""
    group, out, size, n = c.heads // c.kv_heads, [], [], []
    for s in range(c.n):
        v = torch.cat([c.pv, c.v[s]]).to(c.dtype).double()
        count = torch.arange(1, len(v) + 1, device=DEV).double()[:, None]
        for x, y in ((v, out), (v.abs(), size)):
            m = (x.cumsum(0) / count)[c.prefix + c.start[s]:c.prefix + c.lens[s]]
            y.append(m.view(-1, c.kv_heads, 1, c.d).expand(-1, -1, group, -1).reshape(len(m), -1))
        n.append(count[c.prefix + c.start[s]:c.prefix + c.lens[s]])
    return torch.cat(out), torch.cat(size), torch.cat(n)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("by", [1.25, 1.375])
@pytest.mark.parametrize("step", STEPS)
def test_scores_next_to_the_lowest(step, by, dtype):
    """Every score is -by 2^127 log2(e), -3.07e38 or -3.37e38, in the unit of the running maximum: finite."""
    c = Case(*step, dtype, seed=1)
    for x in [c.pk] + c.k:
        x.zero_()
        x.view(-1, c.kv_heads, c.d)[:, :, 0] = -by * 2.0 ** 63
    c.q.zero_()
    c.q.view(-1, c.heads, c.d)[:, :, 0] = 2.0 ** 64 * math.sqrt(c.d)
    got = c.fill().run().double()
    want, size, n = means(c)
    assert bool((((got - want).abs() <= (0.75 * n + 20) * U * size)).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_score_above_the_lowest(dtype):
    """Position 2 of each sequence at -3.07e38, all others at -3.37e38: its value, to the bit."""
    c = Case(8, 2, 64, [5, 3], [90, 1], 300, dtype, seed=2)
    for x in [c.pk] + c.k:
        x.zero_()
        x.view(-1, 2, 64)[:, :, 0] = -1.375 * 2.0 ** 63
    for x in c.k:
        x.view(-1, 2, 64)[2, :, 0] = -1.25 * 2.0 ** 63
    c.q.zero_()
    c.q.view(-1, 8, 64)[:, :, 0] = 2.0 ** 67
    got = c.fill().run().view(-1, 2, 4, 64)
    for rows, v in ((got[:90], c.v[0]), (got[90:], c.v[1])):
        v = v[2].to(c.dtype).float().view(1, 2, 1, 64)
        assert torch.equal(rows, v.expand_as(rows))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("step", STEPS)
def test_values_whose_sum_has_no_room(step, dtype):
    """Values up to f32's largest in every third dimension, ordinary ones in the others."""
    c = Case(*step, dtype, seed=3)
    g = torch.Generator(device=DEV).manual_seed(4)
    for x in [c.pv] + c.v:
        big = (torch.rand(x[:, ::3].shape, generator=g, device=DEV) * 0.5 + 0.5) * 3.38e38
        x[:, ::3] = torch.where(torch.rand(big.shape, generator=g, device=DEV) < 0.8, big, -big)
    got = c.fill().run()
    want, tol = c.want()
    assert bool(torch.isfinite(got).all())
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("step", STEPS)
def test_all_values_the_largest(step, dtype):
    """Their mean is the largest value itself, and never an infinity."""
    c = Case(*step, dtype, seed=5)
    top = LARGEST if dtype == "f32" else torch.finfo(torch.bfloat16).max
    for x in [c.pv] + c.v:
        x.fill_(top)
        x[:, 1::2] = -top
    got = c.fill().run()
    want, tol = c.want()
    assert bool(torch.isfinite(got).all())
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_an_infinite_value_stays_infinite(dtype):
    """Beside values whose sum has no room: a seen infinity is the result's, a hidden one is not."""
    c = Case(8, 2, 64, [0, 40], [60, 1], 3000, dtype, seed=6)
    for x in [c.pv] + c.v:
        x.fill_(3.0e38)
    c.v[0][30, 5], c.v[0][31, 6] = math.inf, -math.inf
    c.v[1][7, 9] = math.nan
    got = c.fill().run().view(-1, 2, 4, 64)
    odd = torch.zeros_like(got, dtype=torch.bool)
    odd[30:60, 0, :, 5] = odd[31:60, 0, :, 6] = odd[60, 0, :, 9] = True
    assert not bool(torch.isfinite(got[odd]).any())
    rest = got[~odd].double()
    # every value is the same: off by the sums' roundings over n <= 3060 keys
    v = float(torch.tensor(3.0e38).to(c.dtype))
    assert bool(((rest - v).abs() <= (0.75 * 3060 + 20) * U * v).all())
