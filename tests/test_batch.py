"""Refusals of the batch (include/wick_hip_batch.h) and the logit rules (wick_hip_logits.h)
that need no GPU: every one comes before any device work."""
import ctypes

import numpy as np
import pytest

from wick_amd import _native
from wick_amd.batch import BatchConfig, DeviceBatch
from wick_amd.logits import LogitRules

GOOD = dict(layers=1, heads=4, kv_heads=2, head_dim=64, sequences=2, capacity=16, prefix_capacity=8, max_tokens=32, type=0)


@pytest.mark.parametrize("change,says", [
    (dict(layers=0), "layers"), (dict(kv_heads=0), "kv_heads"), (dict(sequences=0), "sequences"),
    (dict(capacity=0), "capacity"), (dict(max_tokens=0), "max_tokens"), (dict(heads=3), "heads"), (dict(heads=0), "heads"),
    (dict(head_dim=48), "head_dim"), (dict(head_dim=256), "head_dim"), (dict(prefix_capacity=-1), "prefix_capacity"),
    (dict(type=2), "type"), (dict(capacity=(1 << 30) + 1, max_tokens=1), "2^30"),
    (dict(prefix_capacity=(1 << 30) + 1), "2^30"), (dict(max_tokens=33), "max_tokens"),
    (dict(heads=1 << 20, capacity=1 << 20, max_tokens=1 << 20), "2^30"),
    (dict(heads=65536, kv_heads=65536), "65535"),
])
def test_create_refuses(change, says):
    lib = _native.load()
    cfg, h = BatchConfig(**{**GOOD, **change}), ctypes.c_void_p()
    assert lib.wick_hip_batch_create(ctypes.byref(cfg), ctypes.byref(h)) == _native.EINVAL
    assert says in lib.wick_hip_last_error().decode() and not h.value


def test_null_handles():
    lib = _native.load()
    cfg, h = BatchConfig(**GOOD), ctypes.c_void_p()
    assert lib.wick_hip_batch_create(None, ctypes.byref(h)) == _native.EINVAL
    assert lib.wick_hip_batch_create(ctypes.byref(cfg), None) == _native.EINVAL
    lib.wick_hip_batch_destroy(None)
    assert lib.wick_hip_batch_load_prefix(None, None, 0) == _native.EINVAL
    assert lib.wick_hip_batch_write_prefix_device(None, 0, 0, 1, None, None) == _native.EINVAL
    assert lib.wick_hip_batch_plan(None, None, None, 0) == _native.EINVAL
    assert lib.wick_hip_batch_append_device(None, 0, None, None) == _native.EINVAL
    assert lib.wick_hip_batch_attention_device(None, 0, None, None) == _native.EINVAL
    assert lib.wick_hip_batch_append(None, 0, None, None) == _native.EINVAL
    assert lib.wick_hip_batch_attention(None, 0, None, None) == _native.EINVAL
    assert lib.wick_hip_batch_read(None, 0, 0, 0, 1, None, None) == _native.EINVAL
    assert lib.wick_hip_batch_set_stream(None, None) == _native.EINVAL
    assert lib.wick_hip_batch_synchronize(None) == _native.EINVAL
    assert lib.wick_hip_batch_shape(None) == 0 and lib.wick_hip_batch_scratch_bytes(None) == 0


def test_no_device_is_an_error():
    try:
        import torch
        if torch.cuda.device_count() > 0:
            pytest.skip("a GPU is present")
    except ImportError:
        pass
    lib = _native.load()
    cfg, h = BatchConfig(**GOOD), ctypes.c_void_p()
    assert lib.wick_hip_batch_create(ctypes.byref(cfg), ctypes.byref(h)) == _native.EDEVICE
    x = np.zeros(8, np.float32)
    r = LogitRules()
    p = x.ctypes.data
    assert lib.wick_hip_logits_adjust_device(ctypes.byref(r), p, 1, 8, 8, p, 8, None) == _native.EDEVICE


def test_unknown_type_name():
    with pytest.raises(ValueError, match="dtype"):
        DeviceBatch(1, 4, 2, 64, 2, 16, dtype="fp8")


@pytest.mark.parametrize("rules,call,says", [
    (None, {}, "null"), ({}, dict(logits=None), "null"), ({}, dict(out=None), "null"), ({}, dict(rows=-1), "rows"),
    ({}, dict(vocab=0), "vocab"), ({}, dict(vocab=(1 << 30) + 1), "2^30"), ({}, dict(stride=7), "strides"), ({}, dict(out_stride=7), "strides"),
    (dict(tokens=4096), {}, "n_tokens"), (dict(tokens_stride=-1), {}, "tokens_stride"), (dict(n_bias=-1), {}, "n_bias"),
    (dict(bias=4096, bias_ids=4096), {}, "bias_start"), (dict(bias=4096, bias_start=4096), {}, "bias_ids"),
    (dict(mask=4096), {}, "masks"), (dict(mask=4096, masks=1), dict(rows=2), "masks"),
    (dict(mask=4096, mask_row=4096), {}, "masks"), (dict(repetition=4097), {}, "aligned"),
    ({}, dict(logits=4098), "aligned"), ({}, dict(out=8192 + 16), "overlaps"),
    ({}, dict(rows=2, out=8192, out_stride=9), "overlaps"),
    ({}, dict(rows=1 << 30, out=1 << 50), "too many"),
])
def test_logit_rules_refused(rules, call, says):
    """The addresses are never followed: each call is refused on the host."""
    lib = _native.load()
    c = dict(logits=8192, rows=1, vocab=8, stride=8, out=8192, out_stride=8) | call
    r = None if rules is None else ctypes.byref(LogitRules(**rules))
    assert lib.wick_hip_logits_adjust_device(r, c["logits"], c["rows"], c["vocab"], c["stride"], c["out"], c["out_stride"],
                                             None) == _native.EINVAL
    assert says in lib.wick_hip_last_error().decode()


def test_no_rows_is_nothing_to_do():
    lib = _native.load()
    r = LogitRules()
    assert lib.wick_hip_logits_adjust_device(ctypes.byref(r), 8192, 0, 8, 8, 8192, 8, None) == _native.OK
