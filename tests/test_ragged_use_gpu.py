"""The ragged operators as a program mixes them with the rest of the
framework: the order of their launches, the calls at the ends of their ranges,
and both attention kernels on the inputs that can tell them apart.
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _clean():
    import torch

    from cybel_b200 import _native

    torch.cuda.synchronize()
    _native.check_device(0)


@pytest.mark.parametrize("between", [False, True])
@pytest.mark.parametrize("q8", [False, True])
def test_one_position_attention_right_behind_an_append(q8, between):
    """PagedKVCache.attention, which loads cached rows before it waits for
    the kernel ahead, sees every row of an append queued just before it, with
    and without an attend in between: a captured graph's outputs are those of
    the same calls with the host waiting after each. (A row read too early
    shows: the pages hold NaN until the append.)"""
    import torch

    from cybel_b200.kv_cache import PagedKVCache
    from cybel_b200.paged_attention import RaggedBatch, RopeTable

    heads, kv, hd, seqs, n = 8, 2, 128, 4, 2000
    c = PagedKVCache(1, kv, n + 1, batch=seqs, page_size=64, q8=q8)
    c.ensure(0, n)
    batch = RaggedBatch([n] * seqs, [n] * seqs)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    rand = (lambda *s: torch.randn(*s, hd, generator=g, device="cuda"))
    k, v, q = rand(seqs * n, kv), rand(seqs * n, kv), rand(seqs * n, heads)
    q1, k1, v1 = rand(seqs, heads), rand(seqs, kv), rand(seqs, kv)
    out, seen = torch.empty_like(q1), torch.empty_like(q)
    rope = RopeTable(hd)

    def wipe():
        for t in (c.ks, c.vs) if q8 else (c.k, c.v):
            t.fill_(float("nan"))
        out.zero_()

    def body(wait=(lambda: None)):
        c.append(0, k, v, batch, rope=rope)
        wait()
        if between:
            c.attend(0, q, batch, out=seen)
            wait()
        c.attention(0, q1.data_ptr(), k1.data_ptr(), v1.data_ptr(), n, heads, 10000.0, out.data_ptr(), None, 0,
                    torch.cuda.current_stream().cuda_stream)

    wipe()
    side = torch.cuda.Stream()  # (the attention's scratch belongs to its stream and has to exist before a capture)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body(torch.cuda.synchronize)
    _clean()
    want = out.clone()
    assert torch.isfinite(want).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        body()
    for _ in range(5):
        wipe()
        graph.replay()
        _clean()
        assert torch.equal(out, want)


# ---- attention against the formula in 64 bits, all rows at once --------------------
FEW = ([3, 1, 8, 0, 5], [300, 200, 333, 40, 128])
MANY = ([700, 1, 600, 0, 700], [700, 40, 1000, 30, 900])  # blocks of both kernels, at any shape below


def _plan(q, batch, kv, window=0, prefix=0, q8=False):
    import torch

    from tests.test_ragged_plan import plan

    return plan("fp32" if q.dtype == torch.float32 else "fp16", batch.q_lens, batch.kv_lens, q.shape[1], kv, window, prefix, q8,
                torch.cuda.get_device_properties(0).multi_processor_count)


def _both(q, batch, kv, **kw):
    """Whether a call launches both kernels."""
    few, _, blocks, _ = _plan(q, batch, kv, **kw)
    return blocks > 0 and max(batch.q_lens) * q.shape[1] // kv > few


def _cache(lens, kv, hd, page, q8, seed, layers=1):
    import torch

    from cybel_b200.kv_cache import PagedKVCache
    from cybel_b200.paged_attention import RaggedBatch

    q_lens, kv_lens = lens
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    per = (max(kv_lens) + page - 1) // page
    c = PagedKVCache(layers, kv, per * page, batch=len(kv_lens), page_size=page, q8=q8, head_dim=hd)
    slots = torch.randperm(c.n_slots, generator=g, device="cuda").cpu().numpy().reshape(c.table_host.shape)
    c.table_host[...] = slots
    c.sync_table()
    if q8:
        for t in (c.k, c.v):
            t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda", dtype=torch.int8))
        for t in (c.ks, c.vs):
            t.copy_(torch.rand(t.shape, generator=g, device="cuda") * 0.02 + 0.002)
    else:
        for t in (c.k, c.v):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    return c, RaggedBatch(q_lens, kv_lens), g


def _stored(c, layer, b, n):
    """Keys and values of one sequence [kv][n][hd] in 64 bits, the keys as
    they lie and their factors [kv][n] apart (a Q8 score is the product of the
    codes times the scale)."""
    import torch

    j = torch.arange(n, device="cuda")
    slot, off = c.table[layer, b, j // c.page_size].long(), j % c.page_size
    get = (lambda t: t[slot, :, off].double().transpose(0, 1))
    k, v = get(c.k), get(c.v)
    if c.ks is None:
        return k, torch.ones_like(k[..., 0]), v
    return k, get(c.ks), v * get(c.vs)[..., None]


def _check(c, layer, batch, q, got, scale=None, cap=0.0, slopes=None, window=0, prefix=None, terms=None):
    """got against the formula in 64 bits; returns the tolerances. They are
    those of test_ragged_gpu.py, with two terms taken by what they are: the
    products of a score number `terms` (nonzero elements of a query row), and a
    cap moves a score s by |s| 2^-20 in fp32 rows -- five factors and products
    of 2^-24 and tanh, 2^-24 below 1 and 2^-22 absolutely, hence 2^-21.6, above
    -- and by |s| 2^-19 in fp16 rows, whose tanh is 2^-20.8. A value that is not
    finite is added to the rows that give it a weight, as a product with that
    weight is; a row whose formula gives NaN or an infinity has to give it, and
    an fp32 row that sees an infinite element of a key may give NaN."""
    import torch

    f16 = q.dtype == torch.float16
    kv, hd = c.kv_heads, c.head_dim
    heads = q.shape[1]
    g = heads // kv
    terms = hd if terms is None else terms
    scale = hd ** -0.5 if scale is None else scale
    at, tols = 0, torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, (m, n) in enumerate(zip(batch.q_lens, batch.kv_lens)):
        if not m:
            continue
        k, ks, v = _stored(c, layer, b, n)
        odd = ~torch.isfinite(v)
        fine = v.masked_fill(odd, 0.0)
        x = q[at:at + m].double().view(m, kv, g, hd).permute(1, 2, 0, 3)
        s = scale * torch.einsum("agmd,and->agmn", x, k) * ks[:, None, None, :]
        mag = scale * torch.einsum("agmd,and->agmn", x.abs(), k.abs()) * ks.abs()[:, None, None, :]
        pos, j = torch.arange(n - m, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :]
        if cap:
            s = cap * torch.tanh(s / cap)
        d = mag * ((terms + 8) * 2.0 ** -24 + 2.0 ** -22) + s.abs() * 2.0 ** -22
        if cap:
            d = d + s.abs() * (2.0 ** -19 if f16 else 2.0 ** -20)
        if slopes is not None:
            bias = slopes.double().view(kv, g, 1, 1) * (pos - j).abs()
            s, d = s - bias, d + bias.abs() * 2.0 ** -22
        see = (j <= pos) & ((pos - j < window) if window else True)
        if prefix is not None:
            see = see | (j < prefix[b])
        s = s.masked_fill(~see, float("-inf"))
        p = torch.softmax(s, -1)
        p = torch.where(see.any(-1, keepdim=True), p, torch.zeros_like(p))
        d = torch.where(p > 0, d, torch.zeros_like(d))
        want = torch.einsum("agmn,and->agmd", p, fine)
        spread = torch.einsum("agmn,and->agmd", p, fine.abs())
        bound = 2 * (torch.einsum("agmn,and->agmd", p * d, fine.abs()) + (p * d).sum(-1, keepdim=True) * want.abs())
        for a, jj in odd.any(-1).nonzero().tolist():
            extra = torch.where(odd[a, jj], v[a, jj], torch.zeros_like(v[a, jj]))
            want[a] += torch.where((p[a, :, :, jj] > 0)[..., None], extra, torch.zeros_like(extra))
        tol = bound + spread * (2.0 ** -10 + 2.0 ** -14 if f16 else 2.0 ** -19) + (2.0 ** -24 if f16 else 1e-30)
        most = fine.abs().amax(-1)[:, None, None, :].masked_fill(~see, 0.0).amax(-1, keepdim=True)  # of what the row sees
        tol = tol + n * 2.0 ** -34 * most
        flat = (lambda t: t.permute(2, 0, 1, 3).reshape(m, heads, hd))
        want, tol = flat(want), flat(tol)
        mine = got[at:at + m].double()
        diff = (mine - want).abs()
        free = (torch.isinf(k).any(-1)[:, None, None, :] & see).any(-1) & (not f16)
        good = (mine.isnan() & flat(free[..., None].expand(kv, g, m, hd))) | torch.where(torch.isfinite(want), diff <= tol, (mine == want) | (mine.isnan() & want.isnan()))
        assert good.all(), (b, (~good).nonzero()[:4].tolist(), float((diff / tol).nan_to_num().max()), int((~good).sum()))
        tols[at:at + m] = tol
        at += m
    return tols


def _one_hot(n, heads, hd, value, g):
    """Query rows with one element each: a score is a single product."""
    import torch

    q = torch.zeros(n, heads, hd, device="cuda")
    q.scatter_(2, torch.randint(0, hd, (n, heads, 1), generator=g, device="cuda"), value)
    return q


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dtype,cap,far", [("fp32", 50.0, 30000.0), ("fp32", 1000.0, 30000.0), ("fp16", 50.0, 60000.0),
                                           ("fp16", 30000.0, 60000.0)])
@pytest.mark.parametrize("hd,heads,kv", [(128, 8, 2), (64, 6, 2)])
@pytest.mark.parametrize("lens", [FEW, MANY])
def test_a_capped_row_does_not_depend_on_its_neighbours(lens, hd, heads, kv, dtype, cap, far, q8):
    """Rows of small scores beside rows whose scores pass the cap: tanh of
    each score is as exact as if it stood alone. (One-hot queries, whose
    scores carry no error of a sum that would cover tanh's.)"""
    import torch

    c, batch, g = _cache(lens, kv, hd, 48, q8, seed=hd)
    q = _one_hot(batch.n_tokens, heads, hd, 2.0, g)
    q[::29] *= far / 2.0
    q = q.to(torch.float32 if dtype == "fp32" else torch.float16)
    assert lens is FEW or _both(q, batch, kv, q8=q8)
    out = c.attend(0, q, batch, softcap=cap, scale=1.0)
    _clean()
    _check(c, 0, batch, q, out, scale=1.0, cap=cap, terms=1)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("half", [False, True])
def test_rows_behind_the_last_sequence_take_no_part_in_an_append(half, dtype, q8):
    """A batch updated to fewer tokens than its rows: what the rows behind
    hold (here NaN) reaches nothing, and their queries stay as they were."""
    import torch

    from cybel_b200.paged_attention import RaggedBatch, RopeTable

    lens = ([30, 2, 40], [60, 20, 200])
    c, batch, g = _cache(lens, 2, 128, 16, q8, seed=4)
    batch.update([3, 0, 10], [60, 20, 200])
    n, used = batch.n_tokens, 13
    rows = torch.randn(n, 8 * 128, generator=g, device="cuda").to(torch.float32 if dtype == "fp32" else torch.float16)
    rows[used:] = float("nan")
    q, k, v = (rows[:, a * 128:b * 128].view(n, b - a, 128) for a, b in ((0, 4), (4, 6), (6, 8)))
    rope = RopeTable(128, layout="half" if half else "interleaved")
    q_out = torch.full((n, 4, 128), 7.0, dtype=q.dtype, device="cuda")
    pools = [t for t in (c.k, c.v, c.ks, c.vs) if t is not None]
    before = [t.clone() for t in pools]
    c.append(0, k, v, batch, rope=rope, q=q, q_out=q_out)
    _clean()
    assert (q_out[used:] == 7).all()
    got = [t.clone() for t in pools]
    short = RaggedBatch([3, 0, 10], [60, 20, 200])
    for t, b in zip(pools, before):
        t.copy_(b)
    want = c.append(0, k[:used], v[:used], short, rope=rope, q=q[:used])
    _clean()
    assert torch.equal(q_out[:used], want) and all(torch.equal(a, b) for a, b in zip(got, pools))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_a_step_without_new_tokens(dtype, q8):
    """No sequence has a token this time (rows of no memory at all): the calls
    do nothing, a new tensor has no rows, the cache keeps what it holds."""
    import torch

    from cybel_b200.paged_attention import RaggedBatch, RopeTable

    c, _, _ = _cache(([1, 1], [30, 20]), 2, 128, 16, q8, seed=1)
    batch = RaggedBatch([0, 0], [30, 20])
    rows = (lambda h: torch.empty(0, h, 128, dtype=torch.float32 if dtype == "fp32" else torch.float16, device="cuda"))
    rope = RopeTable(128)
    before = c.k.clone()
    c.ensure_batch(batch)
    assert c.append(0, rows(2), rows(2), batch, rope=rope, q=rows(4)).shape == (0, 4, 128)
    assert c.append(0, rows(2), rows(2), batch) is None
    assert c.attend(0, rows(4), batch, window=3).shape == (0, 4, 128)
    assert rope.rotate(rows(4), torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 4, 128)
    _clean()
    assert torch.equal(c.k, before)


def test_a_cache_on_the_current_device_by_name():
    """device="cuda" (a torch device string without an ordinal) is the
    current device, for the cache as for the tables and batches."""
    import torch

    from cybel_b200.kv_cache import PagedKVCache
    from cybel_b200.paged_attention import RaggedBatch, RopeTable

    c = PagedKVCache(1, 1, 32, batch=1, page_size=16, q8=False, device="cuda")
    batch = RaggedBatch([2], [2], device="cuda")
    c.ensure_batch(batch)
    x = torch.ones(2, 1, 128, device="cuda")
    q = c.append(0, x, x, batch, rope=RopeTable(128, device="cuda"), q=x)
    assert torch.equal(c.attend(0, q, batch), x)
    view = PagedKVCache.over_contiguous(*(torch.zeros(1, 1, 32, 128, dtype=torch.float16, device="cuda") for _ in range(2)))
    view.append(0, x, x, batch)
    assert torch.equal(view.attend(0, q, batch), x)
    _clean()


@pytest.mark.parametrize("lens", [FEW, MANY])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 32 + 5])
def test_a_window_past_every_length_is_none(lens, window):
    import torch

    c, batch, g = _cache(lens, 2, 128, 48, False, seed=2)
    q = torch.randn(batch.n_tokens, 8, 128, generator=g, device="cuda").half()
    assert lens is FEW or _both(q, batch, 2)
    assert torch.equal(c.attend(0, q, batch, window=window), c.attend(0, q, batch))
    _clean()


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_q8_rows_are_those_of_the_one_position_attention(dtype):
    """The codes and scales that append stores are those that
    PagedKVCache.attention stores for the same rows, whatever the rows hold:
    NaN, infinities, numbers too small for a scale, halves between two codes."""
    import torch

    from cybel_b200.kv_cache import PagedKVCache
    from cybel_b200.paged_attention import RaggedBatch, RopeTable

    seqs, kv = 9, 2
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    k, v = (torch.randn(seqs, kv, 128, generator=g, device="cuda") for _ in range(2))
    for t in (k, v):
        t[1, 0, 5] = float("nan")
        t[2, 1, 7] = float("inf")
        t[3, 0, 9] = float("-inf")
        t[3, 0, 11] = float("nan")
        t[4] = float("nan")
        t[5] = 0.0
        t[6] = 0.0
        t[6, :, ::3] = 2.0 ** -149 if dtype == "fp32" else 2.0 ** -24
        t[7] = (torch.randint(-254, 255, t[7].shape, generator=g, device="cuda") / 2).float()
        t[7, :, 0] = 127.0  # scale 1: halves
    if dtype == "fp16":
        k, v = k.half(), v.half()
    caches = [PagedKVCache(1, kv, 16, batch=seqs, page_size=16, q8=True) for _ in range(2)]
    for c in caches:
        c.ensure(0)
    caches[0].append(0, k, v, RaggedBatch([1] * seqs, [1] * seqs), rope=RopeTable(128))
    q, out = torch.ones(seqs, kv, 128, device="cuda"), torch.empty(seqs, kv, 128, device="cuda")
    kf, vf = k.float(), v.float()
    caches[1].attention(0, q.data_ptr(), kf.data_ptr(), vf.data_ptr(), 0, kv, 10000.0, out.data_ptr(), None, 0,
                        torch.cuda.current_stream().cuda_stream)
    _clean()
    for b in range(seqs):
        for h in range(kv):
            for got, want in zip(caches[0].rows(0, b, h, 0, 1), caches[1].rows(0, b, h, 0, 1)):
                assert np.array_equal(got, want), (b, h, got, want)


def test_heads_of_64_have_no_one_position_attention():
    """A cache of 64-wide heads serves append and attend; the one-position
    attention, built for 128, refuses it before a launch."""
    import torch

    from cybel_b200 import _native
    from cybel_b200.kv_cache import PagedKVCache

    c = PagedKVCache(1, 1, 32, batch=1, page_size=16, q8=False, head_dim=64)
    c.ensure(0)
    x, out = torch.ones(64, device="cuda"), torch.full((64,), 3.0, device="cuda")
    with pytest.raises(_native.NativeError):
        c.attention(0, x.data_ptr(), x.data_ptr(), x.data_ptr(), 0, 1, 10000.0, out.data_ptr(), None, 0,
                    torch.cuda.current_stream().cuda_stream)
    _clean()
    assert (out == 3).all() and not c.k.any()
