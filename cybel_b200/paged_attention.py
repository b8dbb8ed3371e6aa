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

from . import _native


def _cuda_index(device):
    import torch

    dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    if dev.type == "cuda" and dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    return dev


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
        import numpy as np
        import torch

        if layout not in _native.ROPE_LAYOUTS:
            raise ValueError(f"unknown rotary layout {layout!r}")
        if scaling not in _native.ROPE_SCALINGS:
            raise ValueError(f"unknown rotary scaling {scaling!r}")
        if rot_dim <= 0 or rot_dim % 2 or rot_dim > 256:
            raise ValueError("rot_dim must be even and at most 256")
        low = 1.0 if low is None else float(low)
        high = (32.0 if scaling == "yarn" else 4.0) if high is None else float(high)
        turns = np.empty(rot_dim // 2, dtype=np.uint64)
        mag = ctypes.c_double()
        _native.check(_native.lib().b200q_rope_table(
            rot_dim, float(theta), _native.ROPE_SCALINGS[scaling], float(factor), low, high, int(original_context),
            turns.ctypes.data_as(ctypes.POINTER(ctypes.c_ulonglong)), ctypes.byref(mag)), "rotary table")
        self.rot_dim, self.layout, self.mag = rot_dim, layout, mag.value
        self.turns_host = turns
        self.dev = _cuda_index(device)
        self.turns = torch.from_numpy(turns.view(np.int64)).to(self.dev)
        self._ptr, self._layout = self.turns.data_ptr(), _native.ROPE_LAYOUTS[layout]

    def rotate(self, x, positions, out=None):
        """x [rows][heads][head_dim] (fp32 or fp16, heads packed) rotated to
        ``positions`` (int32 [rows], >= 0) into ``out`` (a new tensor when
        None; may be x). Current stream; b200q_rope_rows."""
        import torch

        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dt, xs, os_ = _dtype(x), _row_stride(x, "x"), _row_stride(out, "out")
        if out.shape != x.shape or out.dtype != x.dtype:
            raise ValueError("out must have x's shape and type")
        n, heads, hd = x.shape
        if hd < self.rot_dim:
            raise ValueError("heads smaller than the table's rot_dim")
        if positions.dtype != torch.int32 or positions.shape != (n,) or not positions.is_contiguous():
            raise ValueError("positions must be contiguous int32 [rows]")
        _same_device(self.dev, x, out, positions)
        with _on(self.dev):
            _native.check(_native.lib().b200q_rope_rows(
                x.data_ptr(), out.data_ptr(), dt, n, heads, hd, xs, os_, positions.data_ptr(), self._ptr, self.rot_dim,
                self._layout, self.mag, _stream(self.dev)), "rotary rows")
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
        import torch

        self.dev = _cuda_index(device)
        q, kv = self._checked(q_lens, kv_lens)
        self.batch, self.n_tokens = len(q), sum(q)
        self.max_q = max(q) if max_q is None else int(max_q)
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
        import torch

        q, kv = self._checked(q_lens, kv_lens)
        if len(q) != self.batch or sum(q) > self.n_tokens or max(q) > self.max_q or max(kv) > self.max_kv:
            raise ValueError("lengths past those the batch was made for")
        cu = [0]
        for x in q:
            cu.append(cu[-1] + x)
        self.q_lens, self.kv_lens = q, kv
        self.cu_q.copy_(torch.tensor(cu, dtype=torch.int32))
        self.kv_len.copy_(torch.tensor(kv, dtype=torch.int32))


# ---- argument checks ----------------------------------------------------------
def _dtype(t) -> int:
    import torch

    if t.dtype == torch.float32:
        return _native.F32
    if t.dtype == torch.float16:
        return _native.F16
    raise ValueError("activation rows must be fp32 or fp16")


def _row_stride(t, name: str) -> int:
    """Elements between the rows of t [rows][heads][head_dim], whose heads
    and elements must be packed."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [rows][heads][head_dim]")
    n, h, d = t.shape
    s0, s1, s2 = t.stride()
    if (s2 != 1 and d > 1) or (s1 != d and h > 1) or (n > 1 and s0 < h * d):
        raise ValueError(f"{name}: the heads of a row must be packed and its rows apart")
    return s0 if n > 1 else h * d


def _same_device(dev, *tensors) -> None:
    for t in tensors:
        if t.device != dev:
            raise ValueError(f"tensors on {t.device} and {dev}")


class _Here:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def _on(dev):
    """The tensors' device made current for the call (where it is not)."""
    import torch

    if dev.type != "cuda":
        raise RuntimeError("the ragged operators run on a CUDA device")
    return _HERE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _stream(dev) -> int:
    import torch

    return torch.cuda.current_stream(dev).cuda_stream


def _check_batch(cache, batch, rows: int) -> None:
    if batch.batch != cache.batch:
        raise ValueError("the ragged batch has another number of sequences than the cache")
    if rows != batch.n_tokens:
        raise ValueError("rows and the batch's tokens differ")
    if batch.max_kv > cache.pages_per_seq * cache.page_size:
        raise ValueError("lengths past the cache")
    _same_device(cache.dev, batch.kv_len)


def append(cache, layer, k, v, batch, rope=None, q=None, q_out=None):
    """PagedKVCache.append."""
    import torch

    dt = _dtype(k)
    ks, vs = _row_stride(k, "k"), _row_stride(v, "v")
    shape = (batch.n_tokens, cache.kv_heads, cache.head_dim)
    if k.shape != shape or v.shape != shape or v.dtype != k.dtype or (ks != vs and k.shape[0] > 1):
        raise ValueError("k and v must be [n_tokens][kv_heads][head_dim] of one type, rows equally far apart")
    _check_batch(cache, batch, k.shape[0])
    _same_device(cache.dev, k, v)
    heads = qs = qos = 0
    if q is not None:
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        qs, qos = _row_stride(q, "q"), _row_stride(q_out, "q_out")
        if q.shape[0] != shape[0] or q.shape[2] != shape[2] or q.dtype != k.dtype:
            raise ValueError("q must be [n_tokens][heads][head_dim] of k's type")
        if q_out.shape != q.shape or q_out.dtype != q.dtype:
            raise ValueError("q_out must have q's shape and type")
        _same_device(cache.dev, q, q_out)
        heads = q.shape[1]
    elif q_out is not None:
        raise ValueError("q_out without q")
    turns, rot, layout, mag = None, 0, 0, 1.0
    if rope is not None:
        if rope.rot_dim > cache.head_dim:
            raise ValueError("heads smaller than the table's rot_dim")
        _same_device(cache.dev, rope.turns)
        turns, rot, layout, mag = rope._ptr, rope.rot_dim, rope._layout, rope.mag
    with _on(cache.dev):
        _native.check(_native.lib().b200q_rope_append_paged(
            q.data_ptr() if heads else None, k.data_ptr(), v.data_ptr(), dt, shape[0], batch.batch,
            batch.cu_q.data_ptr(), batch.kv_len.data_ptr(), heads, cache.kv_heads, cache.head_dim, qs, ks,
            q_out.data_ptr() if heads else None, qos, turns, rot, layout, mag, *cache._pools(layer),
            _stream(cache.dev)), "paged append")
    return q_out


def attend(cache, layer, q, batch, out=None, scale=None, softcap=0.0, slopes=None, window=0, prefix=None):
    """PagedKVCache.attend."""
    import torch

    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dt, qs, os_ = _dtype(q), _row_stride(q, "q"), _row_stride(out, "out")
    n, heads, hd = q.shape
    if hd != cache.head_dim or heads % cache.kv_heads:
        raise ValueError("q must be [n_tokens][heads][head_dim], heads a multiple of the cache's")
    if out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must have q's shape and type")
    _check_batch(cache, batch, n)
    _same_device(cache.dev, q, out)
    if slopes is not None:
        if slopes.dtype != torch.float32 or slopes.shape != (heads,) or not slopes.is_contiguous():
            raise ValueError("slopes must be contiguous fp32 [heads]")
        _same_device(cache.dev, slopes)
    if prefix is not None:
        if prefix.dtype != torch.int32 or prefix.shape != (batch.batch,) or not prefix.is_contiguous():
            raise ValueError("prefix must be contiguous int32 [sequences]")
        _same_device(cache.dev, prefix)
    with _on(cache.dev):
        _native.check(_native.lib().b200q_attention_paged(
            q.data_ptr(), dt, n, batch.batch, batch.cu_q.data_ptr(), batch.kv_len.data_ptr(), batch.max_q,
            batch.max_kv, heads, cache.kv_heads, hd, qs, out.data_ptr(), os_,
            1.0 / math.sqrt(hd) if scale is None else float(scale), float(softcap),
            None if slopes is None else slopes.data_ptr(), int(window), None if prefix is None else prefix.data_ptr(),
            *cache._pools(layer), _stream(cache.dev)), "paged attention")
    return out
