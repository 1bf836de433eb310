"""ctypes wrapper of include/wick_hip_logits.h: penalties, biases and grammar masks on a
batch's logits, the step of wick's sampler at /root/reference/src/sampler.rs:75-83 and
what serving programs put next to it.
"""
import ctypes

from . import _native


class LogitRules(ctypes.Structure):
    """wick_hip_logit_rules: device pointers (None leaves a rule out) and sizes."""
    _fields_ = [("repetition", ctypes.c_void_p), ("presence", ctypes.c_void_p), ("frequency", ctypes.c_void_p),
                ("tokens", ctypes.c_void_p), ("n_tokens", ctypes.c_void_p), ("n_prompt", ctypes.c_void_p),
                ("tokens_stride", ctypes.c_int), ("bias_start", ctypes.c_void_p), ("bias_ids", ctypes.c_void_p),
                ("bias", ctypes.c_void_p), ("n_bias", ctypes.c_int), ("mask", ctypes.c_void_p),
                ("mask_row", ctypes.c_void_p), ("masks", ctypes.c_int)]


def adjust_logits_device(logits_ptr, rows, vocab, out_ptr, stride=None, out_stride=None, stream=None, **rules):
    """The rules (LogitRules' fields) applied to `rows` rows of `vocab` f32 logits, out_ptr may be
    logits_ptr; asynchronous on `stream` (None: the default stream) of the current device."""
    r = LogitRules(**rules)
    stride = vocab if stride is None else stride
    _native.check(_native.load().wick_hip_logits_adjust_device(ctypes.byref(r), logits_ptr, rows, vocab, stride, out_ptr,
                                                               stride if out_stride is None else out_stride, stream))
