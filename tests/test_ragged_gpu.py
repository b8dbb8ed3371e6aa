"""Ragged batches over the paged cache (b200q_rope_rows,
b200q_rope_append_paged, b200q_attention_paged) against oracle/ragged_ref.py
in 64 bits.

Tolerances, per element, fixed before the kernels ran:

* rotations: the angle's cos and sin carry at most 2^-23 relative to 1, the
  two products and their sum three roundings, so an output is within
  (|a| + |b|) mag 2^-21 of the exact one, plus the rounding to its type
  (2^-11 relative in fp16; cached fp16 rows the same);
* Q8 rows: the codes and scales are those of the exact rotation rounded to
  fp32 (the kernel rotates keys in fp64), compared for equality;
* attention: oracle's bound for the scores, plus, relative to the spread
  sum_j p_j |v_j|, the rounding of the weights and of the sums: fp16 rows
  2^-11 for weights rounded to fp16 and 2^-11 for the output (2^-10 in all),
  2^-14 for exponentials and 32-bit sums; fp32 rows (weights in two fp16
  parts, 2^-22) 2^-19 in all; and 2^-24 absolute for fp16 outputs below the
  smallest normal. Weights in fp16 have a smallest step, too, which matters
  where all but tiny weights meet exact zeros: the largest weight of a row is
  kept at 2^10 or more, so a weight is rounded to a multiple of 2^-24 / 2^10 of
  it, off by 2^-35; with Q8 scales the step is that of weight x scale / E,
  E at most twice the largest scale, so a value term is off by at most
  2^-35 x 2 max|v|. The softmax's sum is at least the largest weight, hence
  n 2^-34 max|v| over n visible positions.
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch

    return torch.float32 if name == "fp32" else torch.float16


def _half(t):
    return t.element_size() == 2


def _clean():
    import torch

    from cybel_b200 import _native

    torch.cuda.synchronize()
    _native.check_device(0)


# ---- rotary rows -----------------------------------------------------------------
SCALINGS = [("none", {}), ("linear", dict(factor=4.0)), ("llama3", dict(factor=8.0, original_context=8192)),
            ("yarn", dict(factor=16.0, original_context=4096))]


def _freq(rot, theta, scaling, kw):
    from oracle.ragged_ref import frequencies

    return frequencies(rot, theta, scaling, kw.get("factor", 1.0), kw.get("original_context", 0))


def _check_rot(got, x, want, freq, mag, half, f16):
    """got against want, both [rows][heads][hd]; x the input."""
    n = len(freq)
    x = np.abs(np.asarray(x, np.float64))
    pair = np.zeros_like(x)
    a, b = (x[..., :n], x[..., n:2 * n]) if half else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    if half:
        pair[..., :n] = pair[..., n:2 * n] = a + b
    else:
        pair[..., 0:2 * n:2] = pair[..., 1:2 * n:2] = a + b
    tol = pair * mag * 2.0 ** -21 + (np.abs(want) * 2.0 ** -11 * 1.001 + 2.0 ** -25 if f16 else 0.0)
    bad = np.abs(np.asarray(got, np.float64) - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:3], np.abs(np.asarray(got, np.float64) - want).max())


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("scaling,kw", SCALINGS)
@pytest.mark.parametrize("rows,heads,hd,rot", [(1, 1, 64, 64), (5, 3, 128, 128), (37, 8, 128, 56), (3, 5, 80, 20),
                                               (2, 2, 256, 256), (300, 2, 66, 34)])
def test_rope_rows(rows, heads, hd, rot, scaling, kw, half, dtype):
    import torch

    from cybel_b200.paged_attention import RopeTable
    from oracle.ragged_ref import rope

    theta = 500000.0
    g = np.random.default_rng(rows + hd + rot)
    x = torch.from_numpy(g.standard_normal((rows, heads, hd))).to(_dt(dtype)).cuda()
    pos = torch.from_numpy(g.integers(0, 1_000_000, rows).astype(np.int32)).cuda()
    pos[0] = 0
    pos[-1] = 2 ** 30 - 1 if rows > 4 else 131071
    t = RopeTable(rot, theta, "half" if half else "interleaved", scaling, **kw)
    freq, mag = _freq(rot, theta, scaling, kw)
    assert abs(t.mag - mag) <= mag * 2.0 ** -24
    want = rope(x.cpu().numpy(), pos.cpu().numpy(), freq, mag, half)
    if rows > 4:  # float64 angles at 2^30 are off by 2^-23: hold that row to its own exact turns
        from fractions import Fraction

        turns = [Fraction(int(u), 2 ** 64) * int(pos[-1]) for u in t.turns_host]
        ang = np.asarray([float(u - int(u)) for u in turns]) * 2 * np.pi
        want[-1:] = rope(x[-1:].cpu().numpy(), np.ones(1), ang, mag, half)
    got = t.rotate(x, pos)
    _check_rot(got.cpu().numpy(), x.cpu().numpy(), want, freq, mag, half, dtype == "fp16")
    assert torch.equal(got[..., rot:], x[..., rot:])
    # in place, and rows of a wider buffer, the same bits; what lies between the rows stays
    wide = torch.full((rows, heads * hd + 24), 7.0, dtype=x.dtype, device="cuda")
    view = wide[:, 8:8 + heads * hd].view(rows, heads, hd)
    view.copy_(x)
    assert t.rotate(view, pos, out=view) is view
    assert torch.equal(view, got)
    assert (wide[:, :8] == 7).all() and (wide[:, 8 + heads * hd:] == 7).all()
    odd = torch.zeros(rows * heads * hd + 1, dtype=x.dtype, device="cuda")[1:].view(rows, heads, hd)  # odd address
    odd.copy_(x)
    assert torch.equal(t.rotate(odd, pos, out=odd), got)
    _clean()


# ---- caches ----------------------------------------------------------------------
def _cache(q_lens, kv_lens, kv, hd, page, q8, seed, layers=1, extra=1, poison=False):
    """A cache whose pages hold values in scattered slots; with `poison`,
    everything that no sequence holds is NaN (fp16 rows, Q8 scales)."""
    import torch

    from cybel_b200.kv_cache import PagedKVCache
    from cybel_b200.paged_attention import RaggedBatch

    g = np.random.default_rng(seed)
    need = [(n + page - 1) // page for n in kv_lens]
    per = max(max(need), 1) + extra
    c = PagedKVCache(layers, kv, per * page, batch=len(kv_lens), page_size=page, q8=q8,
                     n_slots=layers * sum(need) + 2, head_dim=hd)
    order = g.permutation(c.n_slots).tolist()
    for li in range(layers):
        for b, n in enumerate(need):
            for p in range(n):
                c.assign(li, b, p, order.pop())
    c.sync_table()
    shape = tuple(c.k.shape)
    if q8:
        for t in (c.k, c.v):
            t.copy_(torch.from_numpy(g.integers(-127, 128, shape).astype(np.int8)))
        for t in (c.ks, c.vs):
            t.copy_(torch.from_numpy((g.random(shape[:3]) * 0.02 + 0.002).astype(np.float32)))
            if poison:
                _poison(c, t, kv_lens, page)
    else:
        for t in (c.k, c.v):
            t.copy_(torch.from_numpy(g.standard_normal(shape).astype(np.float16)))
            if poison:
                _poison(c, t, kv_lens, page)
    return c, RaggedBatch(q_lens, kv_lens)


def _poison(c, t, kv_lens, page):
    import torch

    keep = torch.zeros(t.shape[0], page, dtype=torch.bool)
    for li in range(c.layers):
        for b, n in enumerate(kv_lens):
            for j in range(n):
                s = c.table_host[li, b, j // page]
                if s >= 0:
                    keep[s, j % page] = True
    t.masked_fill_(~keep.cuda()[:, None, :].view(t.shape[0], 1, page, *([1] * (t.dim() - 3))), float("nan"))


def _rows64(c, layer, b, n):
    """Stored keys and values [n][kv][hd] of one sequence in float64 (0
    where the page is missing), and which positions are present."""
    import torch

    j = np.arange(n)
    slots = c.table_host[layer, b, j // c.page_size].astype(np.int64) if n else np.zeros(0, np.int64)
    here = (slots >= 0) & (slots < c.n_slots)
    si = torch.from_numpy(np.where(here, slots, 0)).cuda()
    oi = torch.from_numpy(j % c.page_size).cuda()
    out = []
    for t, sc in ((c.k, c.ks), (c.v, c.vs)):
        x = t[si, :, oi].double()
        if sc is not None:
            x = x * sc[si, :, oi].double()[..., None]
        out.append(x.cpu().numpy())
    return out[0], out[1], here


def _check_attend(c, layer, batch, q, got, scale=None, cap=0.0, slopes=None, window=0, prefix=None, nan_ok=False):
    from oracle.ragged_ref import attention

    f16 = _half(q)
    hd = q.shape[2]
    scale = 1.0 / np.sqrt(hd) if scale is None else scale
    got = got.double().cpu().numpy()
    qn = q.double().cpu().numpy()
    at = 0
    for b, (m, n) in enumerate(zip(batch.q_lens, batch.kv_lens)):
        if m:
            k, v, here = _rows64(c, layer, b, n)
            want, bound, spread = attention(
                qn[at:at + m], k, v, np.arange(n - m, n), n, scale, cap, None if slopes is None else slopes,
                window, 0 if prefix is None else prefix[b], here)
            tol = bound + spread * (2.0 ** -10 + 2.0 ** -14 if f16 else 2.0 ** -19) + (2.0 ** -24 if f16 else 1e-30)
            tol = tol + n * 2.0 ** -34 * np.abs(v[here], where=np.isfinite(v[here]), out=np.zeros_like(v[here])).max(initial=0)
            d = np.abs(got[at:at + m] - want)
            bad = ~(d <= tol)
            assert not bad.any(), (b, np.argwhere(bad)[:4], float(np.nanmax(d / tol)), int(bad.sum()), bad.size)
        at += m


LENS = {
    "step": ([1, 1, 1, 0, 1], [1, 64, 129, 40, 700]),
    "few": ([3, 1, 8, 2, 0, 5], [3, 200, 333, 65, 0, 128]),
    "prompts": ([257, 1, 130, 33], [257, 300, 131, 480]),
    "many": ([257, 1, 130, 0, 270], [257, 300, 700, 40, 900]),  # the many-row kernel's at most shapes below
}
SHAPES = [(128, 4, 1), (128, 8, 2), (64, 3, 1), (128, 16, 2), (64, 10, 2), (128, 2, 2)]  # hd, heads, kv_heads


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("hd,heads,kv", SHAPES)
@pytest.mark.parametrize("lens", list(LENS))
def test_attend_plain(lens, hd, heads, kv, dtype, q8):
    import torch

    ql, kl = LENS[lens]
    c, batch = _cache(ql, kl, kv, hd, 48, q8, seed=heads + hd, poison=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(heads)
    q = torch.randn(batch.n_tokens, heads, hd, generator=g, device="cuda").to(_dt(dtype)) * 2
    out = c.attend(0, q, batch)
    _clean()
    _check_attend(c, 0, batch, q, out)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("hd,heads,kv", [(128, 8, 2), (64, 3, 1)])
@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("form", ["cap", "alibi", "window", "prefix", "window1", "all"])
def test_attend_scores_and_masks(form, lens, hd, heads, kv, dtype, q8):
    import torch

    ql, kl = LENS[lens]
    c, batch = _cache(ql, kl, kv, hd, 33, q8, seed=heads + hd, poison=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(heads)
    q = torch.randn(batch.n_tokens, heads, hd, generator=g, device="cuda").to(_dt(dtype)) * 4
    kw, ref = {}, {}
    if form in ("cap", "all"):
        kw["softcap"] = ref["cap"] = 5.0
    if form in ("alibi", "all"):
        s = np.asarray([2.0 ** -(h + 1) for h in range(heads)], np.float32)
        kw["slopes"], ref["slopes"] = torch.from_numpy(s).cuda(), s.astype(np.float64)
    if form in ("window", "all"):
        kw["window"] = ref["window"] = 70
    if form == "window1":
        kw["window"] = ref["window"] = 1
    if form in ("prefix", "all"):
        p = [(37 * (b + 1)) % (n + 1) for b, n in enumerate(kl)]
        p[0] = kl[0] + 5  # past the sequence: all of it
        kw["prefix"], ref["prefix"] = torch.tensor(p, dtype=torch.int32, device="cuda"), p
    out = c.attend(0, q, batch, **kw)
    _clean()
    _check_attend(c, 0, batch, q, out, **ref)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("page", [1, 16, 100, 128, 4096])
def test_attend_pages_and_long_context(page, dtype, q8):
    """Pages that end inside a tile and contexts that are split."""
    import torch

    n = 2500 if page < 16 else 5000
    c, batch = _cache([1, 2, 40], [n, n - 7, n + 13], 2, 128, page, q8, seed=page, poison=True)
    q = torch.randn(batch.n_tokens, 8, 128, device="cuda").to(_dt(dtype))
    out = c.attend(0, q, batch)
    _clean()
    _check_attend(c, 0, batch, q, out)


@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("q8", [False, True])
def test_attend_missing_pages_and_empty_rows(lens, q8):
    """Pages dropped behind a window cost nothing and flag nothing; rows that
    lose every page are zeros; an entry outside the pool hides its positions
    and is recorded."""
    import torch

    from cybel_b200 import _native

    ql, kl = LENS[lens]
    c, batch = _cache(ql, kl, 2, 128, 16, q8, seed=3, poison=True)
    q = torch.randn(batch.n_tokens, 4, 128, device="cuda").half()
    c.table_host[0, 2, ::2] = -1
    c.table_host[0, 0, :] = -1
    c.sync_table()
    out = torch.full_like(q, 5.0)
    c.attend(0, q, batch, out=out)
    _clean()
    _check_attend(c, 0, batch, q, out)
    assert (out[:ql[0]] == 0).all()
    c.table_host[0, 2, 1] = c.n_slots
    c.table_host[0, 3, 0] = -7
    c.sync_table()
    out = c.attend(0, q, batch)
    torch.cuda.synchronize()
    with pytest.raises(_native.NativeError):
        _native.check_device(0)
    _check_attend(c, 0, batch, q, out)


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("lens", list(LENS))
def test_attend_non_finite_values_reach_only_rows_that_see_them(lens, dtype):
    import torch

    ql, kl = LENS[lens]
    c, batch = _cache(ql, kl, 2, 128, 16, False, seed=5)
    q = torch.randn(batch.n_tokens, 4, 128, device="cuda").to(_dt(dtype))
    clean = c.attend(0, q, batch)
    at, rows = 0, []
    for b, (m, n) in enumerate(zip(ql, kl)):
        if m > 1:
            j = n - 1 if m < 20 else n - m // 2  # seen by the last rows only
            s, o = c.table_host[0, b, j // 16], j % 16
            c.v[s, 0, o, 5] = float("inf")
            c.v[s, 1, o, 9] = float("nan")
            c.k[s, 1, o, 3] = float("nan")
            rows.append((at, at + m - (n - j), at + m))
        at += m
    out = c.attend(0, q, batch)
    _clean()
    seen = torch.zeros(batch.n_tokens, dtype=torch.bool, device="cuda")
    for a, first, end in rows:
        seen[first:end] = True
        assert torch.isinf(out[first:end, :2, 5]).all() and torch.isnan(out[first:end, 2:]).all()
        keep = [d for d in range(128) if d != 5]
        assert torch.equal(out[first:end, :2, keep], clean[first:end, :2, keep])
    assert torch.equal(out[~seen], clean[~seen])


def test_attend_extreme_scores():
    """Scores of thousands either way, equal scores, and fp32 queries past
    the range of fp16."""
    import torch

    c, batch = _cache([1, 40, 3], [300, 333, 70], 2, 128, 16, False, seed=9)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    base = torch.randn(batch.n_tokens, 8, 128, generator=g, device="cuda")
    for mult, scale in ((300.0, None), (0.0, None), (1e7, 1e-8), (1e-7, 1e5)):
        q = base * mult
        out = c.attend(0, q, batch, scale=scale)
        _clean()
        _check_attend(c, 0, batch, q, out, scale=scale)


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_attend_strides_streams_and_untouched_rows(dtype):
    """q as a part of wider rows, out rows apart, another stream, rows past
    the last sequence, layers of one cache."""
    import torch

    from cybel_b200.paged_attention import RaggedBatch

    ql, kl = [2, 1, 50], [90, 300, 333]
    c, _ = _cache(ql, kl, 2, 128, 48, False, seed=4, layers=2)
    batch = RaggedBatch([10, 10, 50], [90, 300, 333])
    batch.update(ql, kl)  # fewer rows than the batch holds
    n = batch.n_tokens
    wide = torch.randn(n, (8 + 4) * 128, device="cuda").to(_dt(dtype))
    q = wide[:, :8 * 128].view(n, 8, 128)
    obuf = torch.full((n, 8 * 128 + 64), 3.0, dtype=q.dtype, device="cuda")
    out = obuf[:, :8 * 128].view(n, 8, 128)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.attend(1, q, batch, out=out)
    torch.cuda.current_stream().wait_stream(s)
    _clean()
    used = sum(ql)
    assert (obuf[:, 8 * 128:] == 3).all() and (out[used:] == 3).all()
    _check_attend(c, 1, batch, q, out)


# ---- append -------------------------------------------------------------------------
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd,heads,kv,rot", [(128, 8, 2, 128), (64, 3, 3, 24), (128, 5, 1, 60), (64, 4, 4, 34)])
@pytest.mark.parametrize("lens", ["step", "few", "prompts"])  # its cache holds 768 positions
def test_append(lens, hd, heads, kv, rot, half, dtype, q8):
    import torch

    from cybel_b200.kv_cache import PagedKVCache
    from cybel_b200.paged_attention import RaggedBatch, RopeTable
    from oracle.paged_kv_ref import q8_rows
    from oracle.ragged_ref import rope

    ql, kl = LENS[lens]
    c = PagedKVCache(2, kv, 768, batch=len(ql), page_size=48, q8=q8, head_dim=hd)
    c.k.fill_(9), c.v.fill_(9)
    k0, v0 = c.k.clone(), c.v.clone()
    batch = RaggedBatch(ql, kl)
    c.ensure_batch(batch)
    g = np.random.default_rng(hd + heads)
    n = batch.n_tokens
    qkv = torch.from_numpy(g.standard_normal((n, (heads + 2 * kv) * hd))).to(_dt(dtype)).cuda()
    q = qkv[:, :heads * hd].view(n, heads, hd)
    k = qkv[:, heads * hd:(heads + kv) * hd].view(n, kv, hd)
    v = qkv[:, (heads + kv) * hd:].view(n, kv, hd)
    if n > 3:
        v[2] = 0
    table = RopeTable(rot, 10000.0, "half" if half else "interleaved", "yarn", factor=4.0, original_context=128)
    freq, mag = _freq(rot, 10000.0, "yarn", dict(factor=4.0, original_context=128))
    q_out = c.append(1, k, v, batch, rope=table, q=q)
    _clean()
    at = 0
    mask = torch.ones_like(c.k, dtype=torch.bool)
    for b, (m, end) in enumerate(zip(ql, kl)):
        if not m:
            continue
        pos = np.arange(end - m, end)
        sl = slice(at, at + m)
        _check_rot(q_out[sl].cpu().numpy(), q[sl].cpu().numpy(), rope(q[sl].cpu().numpy(), pos, freq, mag, half), freq,
                   mag, half, dtype == "fp16")
        kw = rope(k[sl].cpu().numpy(), pos, freq, mag, half)
        slots = torch.from_numpy(c.table_host[1, b, pos // 48].astype(np.int64)).cuda()
        off = torch.from_numpy(pos % 48).cuda()
        mask[slots, :, off] = False
        kc, vc = c.k[slots, :, off].cpu().numpy(), c.v[slots, :, off].cpu().numpy()
        if q8:
            for codes, scales, want in ((kc, c.ks, kw), (vc, c.vs, v[sl].cpu().numpy())):
                wc, ws = q8_rows(want.astype(np.float32))
                sc = scales[slots, :, off].cpu().numpy()
                assert np.array_equal(sc, ws) and np.array_equal(codes, wc)
        else:
            _check_rot(kc, k[sl].cpu().numpy(), kw, freq, mag, half, True)
            assert np.array_equal(vc, v[sl].half().cpu().numpy())
        at += m
    assert torch.equal(c.k[mask], k0[mask]) and torch.equal(c.v[mask], v0[mask])  # nothing else was written
    # queries in place; keys as they are without a table
    want = q_out.clone()
    assert c.append(1, k, v, batch, rope=table, q=q, q_out=q) is q
    assert torch.equal(q, want)
    assert c.append(0, k, v, batch) is None
    _clean()
    if not q8:
        b = next(i for i, m in enumerate(ql) if m)
        kc, _, _, _ = c.rows(0, b, 0, kl[b] - 1, kl[b])
        assert np.array_equal(kc[0], k[ql[b] - 1, 0].half().cpu().numpy())


def test_append_without_a_page_is_recorded_and_stores_nothing():
    import torch

    from cybel_b200 import _native

    c, batch = _cache([1, 4], [20, 40], 2, 128, 16, False, seed=1)
    k = torch.randn(5, 2, 128, device="cuda")
    c.table_host[0, 0, 1] = -1
    c.table_host[0, 1, 2] = c.n_slots + 3
    c.sync_table()
    k0, v0 = c.k.clone(), c.v.clone()
    c.append(0, k, k, batch)
    torch.cuda.synchronize()
    with pytest.raises(_native.NativeError):
        _native.check_device(0)
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)


# ---- together ------------------------------------------------------------------------
@pytest.mark.parametrize("q8", [False, True])
def test_prompt_then_steps_in_a_captured_graph(q8):
    """Two sequences prefilled with different prompts in one call, then
    stepped by a captured graph whose lengths move on: every step's output
    against the restatement over what the cache holds; a prompt fed in two
    chunks gives the rows of one pass."""
    import torch

    from cybel_b200.kv_cache import PagedKVCache
    from cybel_b200.paged_attention import RaggedBatch, RopeTable

    H, KV, D = 8, 2, 128
    c = PagedKVCache(1, KV, 512, batch=2, page_size=32, q8=q8)
    rope = RopeTable(D, 500000.0)
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    rand = (lambda n, h: torch.randn(n, h, D, generator=g, device="cuda"))
    batch = RaggedBatch([190, 67], [190, 67])
    c.ensure_batch(batch)
    q, k, v = rand(257, H), rand(257, KV), rand(257, KV)
    qr = c.append(0, k, v, batch, rope=rope, q=q)
    whole = c.attend(0, qr, batch)
    _clean()
    _check_attend(c, 0, batch, qr, whole)
    # the first sequence's last 90 rows again, as a chunk over the cache
    chunk = RaggedBatch([90, 0], [190, 67])
    part = c.attend(0, qr[100:190], chunk)
    _check_attend(c, 0, chunk, qr[100:190], part)
    step = RaggedBatch([1, 1], [191, 68], max_kv=512)
    qs, ks, vs = rand(2, H), rand(2, KV), rand(2, KV)
    qo, out = torch.empty_like(qs), torch.empty_like(qs)
    c.ensure_batch(step)

    def body():
        c.append(0, ks, vs, step, rope=rope, q=qs, q_out=qo)
        c.attend(0, qo, step, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body()
    for t in range(40):
        step.update([1, 1], [191 + t, 68 + t])
        c.ensure_batch(step)
        qs.copy_(rand(2, H)), ks.copy_(rand(2, KV)), vs.copy_(rand(2, KV))
        graph.replay()
        _clean()
        _check_attend(c, 0, step, qo, out)


def test_two_streams_at_once():
    """The operators keep nothing between calls: the same calls on two
    streams at once give the results of one alone."""
    import torch

    c, batch = _cache([1, 200, 3, 1], [3000, 700, 90, 5000], 2, 128, 48, False, seed=6)
    q = torch.randn(batch.n_tokens, 8, 128, device="cuda").half()
    want = c.attend(0, q, batch)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[] for _ in streams]
    for _ in range(10):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(c.attend(0, q, batch))
    _clean()
    assert all(torch.equal(x, want) for o in outs for x in o)


def test_refused_calls_launch_nothing():
    """Every refusal of the C entry points comes before a launch: the outputs
    keep what they held."""
    import torch

    from cybel_b200 import _native
    from cybel_b200.paged_attention import RopeTable

    L = _native.lib()
    st = torch.cuda.current_stream().cuda_stream
    c, b = _cache([2, 3], [40, 50], 2, 128, 16, True, seed=1)
    q = torch.randn(5, 4, 128, device="cuda")
    out = torch.full_like(q, 3.0)
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    t = RopeTable(128)
    k0 = c.k.clone()

    def attend(**kw):
        d = dict(q=q.data_ptr(), dtype=0, n=5, batch=2, cu=b.cu_q.data_ptr(), kl=b.kv_len.data_ptr(), mq=3, mk=50, h=4,
                 kv=2, hd=128, qs=0, out=out.data_ptr(), os=0, scale=0.1, cap=0.0, sl=None, w=0, pre=None, mode=1,
                 k=c.k.data_ptr(), v=c.v.data_ptr(), ks=c.ks.data_ptr(), vs=c.vs.data_ptr(), slots=c.n_slots, page=16,
                 tab=c.table_ptr(0), pps=c.pages_per_seq) | kw
        return L.b200q_attention_paged(*d.values(), st)

    def append(**kw):
        d = dict(q=q.data_ptr(), k=q.data_ptr(), v=q.data_ptr(), dtype=0, n=5, batch=2, cu=b.cu_q.data_ptr(),
                 kl=b.kv_len.data_ptr(), h=4, kv=2, hd=128, qs=0, kvs=512, out=out.data_ptr(), os=0,
                 turns=t.turns.data_ptr(), rot=128, layout=0, mag=1.0, mode=1, kp=c.k.data_ptr(), vp=c.v.data_ptr(),
                 ks=c.ks.data_ptr(), vs=c.vs.data_ptr(), slots=c.n_slots, page=16, tab=c.table_ptr(0),
                 pps=c.pages_per_seq) | kw
        return L.b200q_rope_append_paged(*d.values(), st)

    def rows(**kw):
        d = dict(x=q.data_ptr(), out=out.data_ptr(), dtype=0, n=5, h=4, hd=128, xs=0, os=0, pos=pos.data_ptr(),
                 turns=t.turns.data_ptr(), rot=128, layout=0, mag=1.0) | kw
        return L.b200q_rope_rows(*d.values(), st)

    inv, shape, align = -1, -3, -4
    for fn, cases in (
        (attend, [(dict(q=None), inv), (dict(out=None), inv), (dict(cu=None), inv), (dict(kl=None), inv),
                  (dict(dtype=2), inv), (dict(batch=0), inv), (dict(n=-1), inv), (dict(scale=0.0), inv),
                  (dict(scale=float("nan")), inv), (dict(cap=-1.0), inv), (dict(cap=float("inf")), inv),
                  (dict(w=-1), inv), (dict(mode=2), inv), (dict(ks=None), inv), (dict(tab=None), inv),
                  (dict(slots=0), inv), (dict(page=0), inv), (dict(h=5), shape), (dict(hd=96), shape),
                  (dict(qs=511), shape), (dict(os=100), shape), (dict(page=2 ** 30, pps=2), shape),
                  (dict(slots=2 ** 31 - 1), shape), (dict(q=q.data_ptr() + 4), align), (dict(qs=513), align),
                  (dict(k=c.k.data_ptr() + 8), align), (dict(tab=c.table_ptr(0) + 2), align)]),
        (append, [(dict(k=None), inv), (dict(v=None), inv), (dict(q=None), inv), (dict(dtype=7), inv),
                  (dict(layout=2), inv), (dict(mode=-1), inv), (dict(vs=None), inv), (dict(turns=None), shape),
                  (dict(rot=130), shape), (dict(rot=7), shape), (dict(kvs=255), shape), (dict(hd=256), shape),
                  (dict(k=q.data_ptr() + 2), align), (dict(turns=t.turns.data_ptr() + 4), align)]),
        (rows, [(dict(x=None), inv), (dict(pos=None), inv), (dict(turns=None), inv), (dict(dtype=3), inv),
                (dict(h=0), inv), (dict(layout=5), inv), (dict(rot=0), shape), (dict(rot=129), shape),
                (dict(hd=64), shape), (dict(xs=511), shape), (dict(x=q.data_ptr() + 2), align)]),
    ):
        for kw, want in cases:
            assert fn(**kw) == want, (fn.__name__, kw)
    torch.cuda.synchronize()
    assert (out == 3).all() and torch.equal(c.k, k0)
    assert attend(n=0) == 0 and append(n=0) == 0 and rows(n=0) == 0
    assert rows() == 0 and attend() == 0
    _clean()


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_attend_many_sequences_and_large_groups(dtype):
    """More sequences than a warp's lanes, some long and some empty, and more
    query heads per kv head than a tile of rows holds tokens for."""
    import torch

    ql = [(i * 7) % 5 if i % 11 else 70 for i in range(75)]
    kl = [n + (i * 37) % 200 for i, n in enumerate(ql)]
    for heads, kv in ((4, 2), (40, 1)):
        c, batch = _cache(ql, kl, kv, 64, 32, False, seed=kv, poison=True)
        q = torch.randn(batch.n_tokens, heads, 64, device="cuda").to(_dt(dtype))
        out = c.attend(0, q, batch)
        _clean()
        _check_attend(c, 0, batch, q, out)


def test_graph_with_a_split_and_changing_lengths():
    """A captured call over both kernels replays with other lengths: a long
    sequence's chunk shrinks to a single row and grows back."""
    import torch

    from cybel_b200.paged_attention import RaggedBatch

    c, _ = _cache([1, 1], [4000, 300], 2, 128, 64, False, seed=8)
    batch = RaggedBatch([100, 20], [4000, 300])
    q = torch.randn(batch.n_tokens, 8, 128, device="cuda").half()
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.attend(0, q, batch, out=out)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.attend(0, q, batch, out=out)
    for ql, kl in (([100, 20], [4000, 300]), ([1, 0], [2100, 7]), ([0, 0], [5, 0]), ([7, 90], [3999, 299])):
        batch.update(ql, kl)
        out.fill_(2.0)
        g.replay()
        _clean()
        _check_attend(c, 0, batch, q, out)
        assert (out[sum(ql):] == 2).all()


@pytest.mark.parametrize("lens", ["few", "prompts"])
def test_lengths_past_the_table_and_in_place(lens):
    """kv_len past what the page table reaches (the C entry point's caller may
    set it so): the positions past it are hidden and recorded, however far the
    length is off; the others give what they give. out may be q."""
    import torch

    from cybel_b200 import _native

    ql, kl = LENS[lens]
    c, batch = _cache(ql, kl, 2, 128, 48, False, seed=2, poison=True)
    q = torch.randn(batch.n_tokens, 4, 128, device="cuda").half()
    want = c.attend(0, q, batch)
    buf = q.clone()
    assert c.attend(0, buf, batch, out=buf) is buf and torch.equal(buf, want)
    _clean()
    reach = c.pages_per_seq * 48
    for far in (reach + 1, 2 ** 31 - 1):
        batch.kv_len.copy_(torch.tensor(kl, dtype=torch.int32))
        batch.kv_len[0] = far
        out = c.attend(0, q, batch)
        torch.cuda.synchronize()
        with pytest.raises(_native.NativeError):
            _native.check_device(0)
        # (the sequence's own rows see what the rest of its last page holds: NaN here)
        assert torch.equal(out[ql[0]:], want[ql[0]:])
    batch.kv_len[0] = -5
    out = c.attend(0, q, batch)
    _clean()
    assert (out[:ql[0]] == 0).all() and torch.equal(out[ql[0]:], want[ql[0]:])


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("hd,heads,kv", [(128, 8, 2), (64, 6, 2), (128, 2, 2)])
@pytest.mark.parametrize("ql,kl", [([300, 290, 280, 1], [300, 900, 1700, 20]), ([1, 400, 90], [1500, 4993, 1013]), ([64], [64]), ([9], [4100]), ([40, 1], [300, 2000]), ([30, 21, 64, 2], [30, 90, 70, 300]),
                                   ([64] * 24, [64 + 20 * i for i in range(24)]), ([2, 2, 1], [600, 2, 130])])
def test_attend_rows_between_one_kernel_and_the_other(ql, kl, hd, heads, kv, dtype, q8):
    """Batches that either kernel takes, by their size, single heads per kv
    head, and up to 8 rows, whose weights are split whatever the type."""
    import torch

    c, batch = _cache(ql, kl, kv, hd, 48, q8, seed=sum(kl), poison=True)
    q = torch.randn(batch.n_tokens, heads, hd, device="cuda").to(_dt(dtype)) * 2
    for window in (0, 50):
        out = c.attend(0, q, batch, window=window)
        _clean()
        _check_attend(c, 0, batch, q, out, window=window)


def test_a_sequence_longer_than_stated_costs_only_itself():
    """More new tokens than the max_q_len of the call (only a caller of the C
    entry point can): that sequence's rows may stay, the others are right."""
    import torch

    from cybel_b200.paged_attention import RaggedBatch

    for stated in (70, 3):
        ql, kl = [300, stated, 2, 600], [900, 200, 300, 600]
        c, batch = _cache(ql, kl, 2, 128, 64, False, seed=stated, poison=True)
        q = torch.randn(batch.n_tokens, 8, 128, device="cuda").half()
        batch.max_q = stated
        out = torch.full_like(q, 9.0)
        c.attend(0, q, batch, out=out)
        _clean()
        # (the others, checked alone: their rows and lengths in a batch of their own)
        rest = [1, 2]
        part = RaggedBatch([ql[b] for b in rest], [kl[b] for b in rest])
        part.q_lens, part.kv_lens = [0] + part.q_lens, [0] + part.kv_lens
        _check_attend(c, 0, part, q[300:], out[300:302 + stated])
