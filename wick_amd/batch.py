"""ctypes wrapper of include/wick_hip_batch.h: several sequences over one shared prefix.

wick keeps one sequence's prompt prefix (src/engine.rs:127-132);
DeviceBatch holds one prefix for many sequences and attends for all of them at once, as
Model::attention (src/model.rs:518-553) does for each.
"""
import ctypes

import numpy as np

from . import _native

F32, BF16 = 0, 1
_TYPES = {"f32": F32, "bf16": BF16}


class BatchConfig(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("layers", "heads", "kv_heads", "head_dim", "sequences", "capacity",
                                            "prefix_capacity", "max_tokens", "type")]


def _f32(a, width):
    return np.ascontiguousarray(a, dtype=np.float32).reshape(-1, width)


class DeviceBatch:
    """The caches of `sequences` sequences of up to `capacity` own positions behind a
    prefix of up to `prefix_capacity` positions, f32 or bf16, on the current GPU.
    max_tokens: most tokens of one plan (default: every position)."""

    def __init__(self, layers, heads, kv_heads, head_dim, sequences, capacity, prefix_capacity=0, max_tokens=None,
                 dtype="f32"):
        if dtype not in _TYPES:
            raise ValueError(f"dtype must be one of {sorted(_TYPES)}, not {dtype!r}")
        lib = _native.load()
        self._lib = lib
        self.layers, self.heads, self.kv_heads, self.head_dim = layers, heads, kv_heads, head_dim
        self.sequences, self.capacity, self.prefix_capacity = sequences, capacity, prefix_capacity
        self.max_tokens = sequences * capacity if max_tokens is None else max_tokens
        self.tokens = 0  # of the current plan
        cfg = BatchConfig(layers, heads, kv_heads, head_dim, sequences, capacity, prefix_capacity, self.max_tokens,
                          _TYPES[dtype])
        h = ctypes.c_void_p()
        _native.check(lib.wick_hip_batch_create(ctypes.byref(cfg), ctypes.byref(h)))
        self.handle = h

    def close(self):
        if getattr(self, "handle", None):
            self._lib.wick_hip_batch_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def load_prefix(self, kv, length):
        """Positions 0..length of every layer of a DeviceKvCache become the prefix's."""
        _native.check(self._lib.wick_hip_batch_load_prefix(self.handle, kv.handle, length))

    def write_prefix_device(self, layer, start, t, k_ptr, v_ptr):
        """The prefix's positions start..start+t of `layer` from device arrays [t][kv_heads*head_dim]."""
        _native.check(self._lib.wick_hip_batch_write_prefix_device(self.handle, layer, start, t, k_ptr, v_ptr))

    def plan(self, start, t, prefix=0):
        """The step that follows: sequence s brings t[s] tokens at its positions start[s].., behind
        `prefix` positions of the prefix."""
        start = np.ascontiguousarray(start, dtype=np.int32).reshape(-1)
        t = np.ascontiguousarray(t, dtype=np.int32).reshape(-1)
        if start.size != self.sequences or t.size != self.sequences:
            raise ValueError(f"start and t must have {self.sequences} entries, not {start.size} and {t.size}")
        _native.check(self._lib.wick_hip_batch_plan(self.handle, start.ctypes.data, t.ctypes.data, prefix))
        self.tokens = int(t.sum())

    def shape(self):
        """The plan's launch shape: graphs captured under one replay under later plans of the same."""
        return self._lib.wick_hip_batch_shape(self.handle)

    # ---- host arrays (synchronous)
    def append(self, layer, k, v):
        """k and v of the planned tokens, [tokens][kv_heads*head_dim]."""
        k, v = (_f32(x, self.kv_heads * self.head_dim) for x in (k, v))
        if len(k) != self.tokens or len(v) != self.tokens:
            raise ValueError(f"k and v must have the plan's {self.tokens} rows, not {len(k)} and {len(v)}")
        _native.check(self._lib.wick_hip_batch_append(self.handle, layer, k.ctypes.data, v.ctypes.data))

    def attention(self, layer, q):
        """The planned tokens' attention, [tokens][heads*head_dim]."""
        q = _f32(q, self.heads * self.head_dim)
        if len(q) != self.tokens:
            raise ValueError(f"q must have the plan's {self.tokens} rows, not {len(q)}")
        att = np.empty_like(q)
        _native.check(self._lib.wick_hip_batch_attention(self.handle, layer, q.ctypes.data, att.ctypes.data))
        return att

    def read(self, layer, seq, pos0, n):
        """Positions pos0..pos0+n of sequence `seq` (-1: the prefix), [n][kv_heads*head_dim] each."""
        k = np.empty((max(n, 0), self.kv_heads * self.head_dim), np.float32)
        v = np.empty_like(k)
        _native.check(self._lib.wick_hip_batch_read(self.handle, layer, seq, pos0, n, k.ctypes.data, v.ctypes.data))
        return k, v

    # ---- device pointers (asynchronous on the handle's stream)
    def append_device(self, layer, k_ptr, v_ptr):
        _native.check(self._lib.wick_hip_batch_append_device(self.handle, layer, k_ptr, v_ptr))

    def attention_device(self, layer, q_ptr, att_ptr):
        _native.check(self._lib.wick_hip_batch_attention_device(self.handle, layer, q_ptr, att_ptr))

    def set_stream(self, stream_ptr):
        _native.check(self._lib.wick_hip_batch_set_stream(self.handle, stream_ptr))

    def synchronize(self):
        _native.check(self._lib.wick_hip_batch_synchronize(self.handle))

    def scratch_bytes(self):
        """Bytes the handle holds beyond its caches."""
        return int(self._lib.wick_hip_batch_scratch_bytes(self.handle))
