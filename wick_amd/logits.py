"""ctypes wrapper of include/wick_hip_logits.h: penalties, biases and grammar masks on a
batch's logits, the step of wick's sampler at src/sampler.rs:75-83 and
what serving programs put next to it.
"""
import ctypes
import struct

from . import _native


class LogitRules(ctypes.Structure):
    """wick_hip_logit_rules: device pointers (None leaves a rule out) and sizes."""
    _fields_ = [("repetition", ctypes.c_void_p), ("presence", ctypes.c_void_p), ("frequency", ctypes.c_void_p),
                ("tokens", ctypes.c_void_p), ("n_tokens", ctypes.c_void_p), ("n_prompt", ctypes.c_void_p),
                ("tokens_stride", ctypes.c_int), ("bias_start", ctypes.c_void_p), ("bias_ids", ctypes.c_void_p),
                ("bias", ctypes.c_void_p), ("n_bias", ctypes.c_int), ("mask", ctypes.c_void_p),
                ("mask_row", ctypes.c_void_p), ("masks", ctypes.c_int)]


_RULES = struct.Struct("".join("P" if t is ctypes.c_void_p else "i" for _, t in LogitRules._fields_) + "0P")


def adjust_logits_device(logits_ptr, rows, vocab, out_ptr, stride=None, out_stride=None, stream=None, repetition=None,
                         presence=None, frequency=None, tokens=None, n_tokens=None, n_prompt=None, tokens_stride=0,
                         bias_start=None, bias_ids=None, bias=None, n_bias=0, mask=None, mask_row=None, masks=0):
    """The rules (LogitRules' fields) applied to `rows` rows of `vocab` f32 logits, out_ptr may be
    logits_ptr; asynchronous on `stream` (None: the default stream) of the current device."""
    # packed here: ctypes takes twice as long for the fields as for the call
    rules = _RULES.pack(repetition or 0, presence or 0, frequency or 0, tokens or 0, n_tokens or 0, n_prompt or 0,
                        tokens_stride, bias_start or 0, bias_ids or 0, bias or 0, n_bias, mask or 0, mask_row or 0, masks)
    stride = vocab if stride is None else stride
    rc = _native.load().wick_hip_logits_adjust_device(rules, logits_ptr, rows, vocab, stride, out_ptr,
                                                      stride if out_stride is None else out_stride, stream)
    if rc:
        _native.check(rc)
