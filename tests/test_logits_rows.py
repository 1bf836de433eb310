"""Rows of the logit rules (include/wick_hip_logits.h) that lie between the rows of their input: nothing
of either overlaps."""
import ctypes

import numpy as np
import pytest
import torch

from wick_amd import _native
from wick_amd.logits import LogitRules, adjust_logits_device

# rows, vocab, stride, first float of out behind the first of logits
APART = [(4, 8, 16, 8), (3, 5, 16, 7), (3, 5, 16, 11), (3, 5, 16, -9), (5, 8, 16, 8 + 2 * 16), (5, 8, 16, -8), (2, 1000, 2001, 1000)]
OVERLAP = [(4, 8, 16, 7), (4, 8, 16, 9), (4, 8, 16, 16), (2, 5, 16, -4), (4, 8, 15, 8), (3, 8, 16, 2 * 16)]


@pytest.mark.parametrize("rows,vocab,stride,at", OVERLAP)
def test_rows_that_overlap_are_refused(rows, vocab, stride, at):
    """The addresses are never followed."""
    r, x = LogitRules(), 1 << 20
    assert _native.load().wick_hip_logits_adjust_device(ctypes.byref(r), x, rows, vocab, stride, x + 4 * at, stride,
                                                        None) == _native.EINVAL
    assert "overlaps" in _native.load().wick_hip_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,stride,at", APART)
def test_rows_between_rows(rows, vocab, stride, at):
    x0 = max(0, -at)
    n = x0 + max(0, at) + rows * stride
    buf = torch.randn(n, generator=torch.Generator(device="cpu").manual_seed(at), dtype=torch.float32)
    want, rep = buf.clone(), 1.25
    for r in range(rows):
        x = buf[x0 + r * stride:][:vocab]
        y = want[x0 + at + r * stride:][:vocab]
        y.copy_(x)
        y[1] = x[1] / rep if x[1] > 0 else x[1] * rep
    dev = buf.to("cuda")
    tokens = torch.ones(rows, 1, dtype=torch.int32, device="cuda")
    held = torch.ones(rows, dtype=torch.int32, device="cuda")
    reps = torch.full((rows,), rep, device="cuda")
    torch.cuda.synchronize()
    adjust_logits_device(dev.data_ptr() + 4 * x0, rows, vocab, dev.data_ptr() + 4 * (x0 + at), stride=stride,
                         repetition=reps.data_ptr(), tokens=tokens.data_ptr(), n_tokens=held.data_ptr(), tokens_stride=1)
    torch.cuda.synchronize()
    assert np.array_equal(dev.cpu().numpy(), want.numpy())
