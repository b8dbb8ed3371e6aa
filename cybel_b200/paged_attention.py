"""Ragged batches over the paged cache: rotary tables, the append and the
attention of sequences of different lengths in one call.

``DecodeStack`` steps one sequence; a server steps many at once, each at a
position of its own, with whole prompts among them. ``RaggedBatch`` names the
rows of such a step, ``RopeTable`` holds the rotary frequencies, and
``PagedKVCache.append`` / ``PagedKVCache.attend`` (kv_cache.py) run the two
halves of the attention block over its pages::

    batch = RaggedBatch([1, 1, 700], [513, 90, 700])     # new tokens, lengths after them
    cache.ensure_batch(batch)
    q = cache.append(layer, k, v, batch, rope=table, q=q)
    out = cache.attend(layer, q, batch, softcap=50.0, window=4096)

The kernels read the lengths and the page table on the device, so a captured
graph replays with those that ``RaggedBatch.update`` and the cache put there.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from . import _native

_INT_MAX = 2 ** 31 - 1  # of the C entry points' ints, past which ctypes cuts numbers off


class RopeTable:
    """Rotary frequencies of the first ``rot_dim`` elements of a head.

    ``layout``: "interleaved" (pairs 2p, 2p + 1, the reference graph's,
    model_graph.cpp:1222-1323) or "half" (pairs p, p + rot_dim / 2).
    ``scaling``: "none", "linear" (frequencies divided by ``factor``),
    "llama3" (divided where a pair makes fewer than ``low`` turns over
    ``original_context`` positions, kept above ``high``, interpolated between;
    defaults 1 and 4) or "yarn" (interpolated over the pairs between the ones
    that make ``high`` and ``low`` turns; defaults 32 and 1; cos and sin times
    ``mag`` = 0.1 ln(factor) + 1).
    """

    def __init__(self, rot_dim: int, theta: float = 10000.0, layout: str = "interleaved", scaling: str = "none",
                 factor: float = 1.0, original_context: int = 0, low: float | None = None, high: float | None = None,
                 device: int | str = 0):
        if layout not in _native.ROPE_LAYOUTS:
            raise ValueError(f"unknown rotary layout {layout!r}")
        if scaling not in _native.ROPE_SCALINGS:
            raise ValueError(f"unknown rotary scaling {scaling!r}")
        if rot_dim <= 0 or rot_dim % 2 or rot_dim > 256:
            raise ValueError("rot_dim must be even and at most 256")
        if not 0 <= original_context <= _INT_MAX:
            raise ValueError("original_context out of range")
        low = 1.0 if low is None else float(low)
        high = (32.0 if scaling == "yarn" else 4.0) if high is None else float(high)
        turns = np.empty(rot_dim // 2, dtype=np.uint64)
        mag = ctypes.c_double()
        _native.check(_native.lib().b200q_rope_table(
            rot_dim, float(theta), _native.ROPE_SCALINGS[scaling], float(factor), low, high, int(original_context),
            turns.ctypes.data_as(ctypes.POINTER(ctypes.c_ulonglong)), ctypes.byref(mag)), "rotary table")
        self.rot_dim, self.layout, self.mag = rot_dim, layout, mag.value
        self.turns_host = turns
        self.dev = _native.torch_device(device)
        self.turns = torch.from_numpy(turns.view(np.int64)).to(self.dev)
        self._ptr, self._layout = self.turns.data_ptr(), _native.ROPE_LAYOUTS[layout]
        self._index = device_index(self.dev)

    def rotate(self, x, positions, out=None):
        """x [rows][heads][head_dim] (fp32 or fp16, heads packed) rotated to
        ``positions`` (int32 [rows], >= 0) into ``out`` (a new tensor when
        None; may be x). Current stream; b200q_rope_rows."""
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dt, shape, xs = _rows(x, "x", self._index)
        odt, oshape, os_ = _rows(out, "out", self._index)
        if oshape != shape or odt != dt:
            raise ValueError("out must have x's shape and type")
        n, heads, hd = shape
        if hd < self.rot_dim:
            raise ValueError("heads smaller than the table's rot_dim")
        _vector(positions, "positions", torch.int32, n, self._index)
        _call(self._index, _native.lib().b200q_rope_rows, "rotary rows", x.data_ptr(), out.data_ptr(), dt, n, heads,
              hd, xs, os_, positions.data_ptr(), self._ptr, self.rot_dim, self._layout, self.mag)
        return out


class RaggedBatch:
    """The rows of one step over a cache's sequences: ``q_lens[b]`` new
    tokens of sequence b (0: none), the last of them at position
    ``kv_lens[b] - 1``.

    ``cu_q`` and ``kv_len`` are the device arrays the kernels read.
    ``update`` gives the same rows other lengths in place (a captured graph
    replays with them): the new tokens must add up to at most the rows the
    batch was made with, and no length may pass ``max_q`` / ``max_kv``, which
    a batch that grows is made with."""

    def __init__(self, q_lens, kv_lens, device: int | str = 0, max_q: int | None = None, max_kv: int | None = None):
        self.dev = _native.torch_device(device)
        self._index = device_index(self.dev)
        q, kv = self._checked(q_lens, kv_lens)
        self.batch, self.n_tokens = len(q), sum(q)
        self.max_q = max(q) if max_q is None else min(int(max_q), self.n_tokens)  # (of all rows at most)
        self.max_kv = max(kv) if max_kv is None else int(max_kv)
        self.cu_q = torch.empty(self.batch + 1, dtype=torch.int32, device=self.dev)
        self.kv_len = torch.empty(self.batch, dtype=torch.int32, device=self.dev)
        self.update(q, kv)

    @staticmethod
    def _checked(q_lens, kv_lens):
        q, kv = [int(x) for x in q_lens], [int(x) for x in kv_lens]
        if not q or len(q) != len(kv):
            raise ValueError("q_lens and kv_lens must hold one length per sequence")
        if any(a < 0 or b < a for a, b in zip(q, kv)):
            raise ValueError("a sequence cannot be shorter than its new tokens")
        if max(kv) >= 2 ** 30 or sum(q) >= 2 ** 30:
            raise ValueError("lengths out of range")
        return q, kv

    def update(self, q_lens, kv_lens) -> None:
        q, kv = self._checked(q_lens, kv_lens)
        if len(q) != self.batch or sum(q) > self.n_tokens or max(q) > self.max_q or max(kv) > self.max_kv:
            raise ValueError("lengths past those the batch was made for")
        cu = [0]
        for x in q:
            cu.append(cu[-1] + x)
        self.q_lens, self.kv_lens = q, kv
        self.cu_q.copy_(torch.tensor(cu, dtype=torch.int32))
        self.kv_len.copy_(torch.tensor(kv, dtype=torch.int32))


# ---- argument checks and the call ---------------------------------------------
# These run before every launch of a decode step, whose kernels take 2-9 us:
# they ask torch for each property once and make no objects they can do without.
def device_index(dev) -> int:
    """Ordinal of a CUDA device, -1 for the host (as Tensor.get_device)."""
    return dev.index if dev.type == "cuda" else -1


def _row_stride(t, name: str) -> int:
    """Elements between the rows of t [rows][heads][head_dim], whose heads
    and elements must be packed."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [rows][heads][head_dim]")
    n, h, d = t.shape
    s0, s1, s2 = t.stride()
    if n <= 1:
        s0 = h * d
    if (s2 != 1 and d > 1) or (s1 != d and h > 1) or s0 < h * d:
        raise ValueError(f"{name}: the heads of a row must be packed and its rows apart")
    return s0


def _rows(t, name: str, index: int):
    """(element type, shape, row stride) of activation rows on device `index`."""
    dtype = t.dtype
    if dtype is torch.float32:
        dt = _native.F32
    elif dtype is torch.float16:
        dt = _native.F16
    else:
        raise ValueError(f"{name}: activation rows must be fp32 or fp16")
    stride = _row_stride(t, name)
    if t.get_device() != index:
        raise ValueError(f"{name} is on another device")
    return dt, t.shape, stride


def _vector(t, name: str, dtype, n: int, index: int) -> None:
    if t.dtype is not dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {dtype} [{n}]")
    if t.get_device() != index:
        raise ValueError(f"{name} is on another device")


def _call(index: int, fn, what: str, *args) -> None:
    """fn(*args, stream) on the current stream of device `index`, which is
    made current for the call where it is not."""
    if index < 0:
        raise RuntimeError("the ragged operators run on a CUDA device")
    # (the handle itself: torch.cuda.current_stream makes a Stream object, 2 us)
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch.cuda.current_device() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        raise _native.NativeError(rc, what)


def _check_batch(cache, batch, rows: int, index: int) -> None:
    if batch.batch != cache.batch:
        raise ValueError("the ragged batch has another number of sequences than the cache")
    if rows != batch.n_tokens:
        raise ValueError("rows and the batch's tokens differ")
    if batch.max_kv > cache.pages_per_seq * cache.page_size:
        raise ValueError("lengths past the cache")
    if batch._index != index:
        raise ValueError("the batch is on another device")


def append(cache, layer, k, v, batch, rope=None, q=None, q_out=None):
    """PagedKVCache.append."""
    index = device_index(cache.dev)
    dt, shape, ks = _rows(k, "k", index)
    vdt, vshape, vs = _rows(v, "v", index)
    n, kv_heads, hd = shape
    if (kv_heads != cache.kv_heads or hd != cache.head_dim or vshape != shape or vdt != dt or (ks != vs and n > 1)):
        raise ValueError("k and v must be [n_tokens][kv_heads][head_dim] of one type, rows equally far apart")
    _check_batch(cache, batch, n, index)
    heads = qs = qos = 0
    if q is not None:
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        qdt, qshape, qs = _rows(q, "q", index)
        odt, oshape, qos = _rows(q_out, "q_out", index)
        if qshape[0] != n or qshape[2] != hd or qdt != dt:
            raise ValueError("q must be [n_tokens][heads][head_dim] of k's type")
        if oshape != qshape or odt != dt:
            raise ValueError("q_out must have q's shape and type")
        heads = qshape[1]
    elif q_out is not None:
        raise ValueError("q_out without q")
    turns, rot, layout, mag = None, 0, 0, 1.0
    if rope is not None:
        if rope.rot_dim > hd:
            raise ValueError("heads smaller than the table's rot_dim")
        if rope._index != index:
            raise ValueError("the rotary table is on another device")
        turns, rot, layout, mag = rope._ptr, rope.rot_dim, rope._layout, rope.mag
    _call(index, _native.lib().b200q_rope_append_paged, "paged append", q.data_ptr() if heads else None, k.data_ptr(),
          v.data_ptr(), dt, n, batch.batch, batch.cu_q.data_ptr(), batch.kv_len.data_ptr(), heads, kv_heads, hd, qs,
          ks, q_out.data_ptr() if heads else None, qos, turns, rot, layout, mag, *cache._pools(layer))
    return q_out


def attend(cache, layer, q, batch, out=None, scale=None, softcap=0.0, slopes=None, window=0, prefix=None):
    """PagedKVCache.attend."""
    index = device_index(cache.dev)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dt, shape, qs = _rows(q, "q", index)
    odt, oshape, os_ = _rows(out, "out", index)
    n, heads, hd = shape
    if hd != cache.head_dim or heads % cache.kv_heads:
        raise ValueError("q must be [n_tokens][heads][head_dim], heads a multiple of the cache's")
    if oshape != shape or odt != dt:
        raise ValueError("out must have q's shape and type")
    _check_batch(cache, batch, n, index)
    if slopes is not None:
        _vector(slopes, "slopes", torch.float32, heads, index)
        slopes = slopes.data_ptr()
    if prefix is not None:
        _vector(prefix, "prefix", torch.int32, batch.batch, index)
        prefix = prefix.data_ptr()
    if window < 0:
        raise ValueError("window must not be negative")
    _call(index, _native.lib().b200q_attention_paged, "paged attention", q.data_ptr(), dt, n, batch.batch,
          batch.cu_q.data_ptr(), batch.kv_len.data_ptr(), batch.max_q, batch.max_kv, heads, cache.kv_heads, hd, qs,
          out.data_ptr(), os_, 1.0 / math.sqrt(hd) if scale is None else scale, softcap, slopes, min(window, _INT_MAX),
          prefix, *cache._pools(layer))
    return out
