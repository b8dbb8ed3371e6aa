"""Both attention kernels of the ragged batches, each on the inputs that can
tell them apart: every test asserts which of them a call launches, on
batches far past the border between the two, so that a change of the rule that
chooses does not take the many-row kernel out of them."""

from __future__ import annotations

import numpy as np
import pytest

from tests.test_ragged_use_gpu import FEW, MANY, _both, _cache, _check, _clean, _one_hot, _plan

pytestmark = pytest.mark.gpu

TYPES = [("fp32", False), ("fp32", True), ("fp16", False), ("fp16", True)]


def _dt(name):
    import torch

    return torch.float32 if name == "fp32" else torch.float16


def _randn(batch, heads, hd, dtype, g, sigma=1.0):
    import torch

    return (torch.randn(batch.n_tokens, heads, hd, generator=g, device="cuda") * sigma).to(_dt(dtype))


def _reaches(lens, q, batch, kv, **kw):
    """FEW is the few-row kernel's alone, everything else both kernels'."""
    return (not _plan(q, batch, kv, **kw)[2]) if lens is FEW else _both(q, batch, kv, **kw)


@pytest.mark.parametrize("dtype,q8", TYPES)
@pytest.mark.parametrize("hd,heads,kv", [(128, 2, 2), (64, 3, 1), (128, 40, 1), (64, 10, 2)])
@pytest.mark.parametrize("window", [0, 1, 70])
def test_shapes_and_windows(window, hd, heads, kv, dtype, q8):
    c, batch, g = _cache(MANY, kv, hd, 33, q8, seed=heads)
    q = _randn(batch, heads, hd, dtype, g, 2.0)
    assert _reaches(MANY, q, batch, kv, window=window, q8=q8)
    out = c.attend(0, q, batch, window=window)
    _clean()
    _check(c, 0, batch, q, out, window=window)


@pytest.mark.parametrize("dtype,q8", TYPES)
@pytest.mark.parametrize("page", [1, 16, 100, 128, 4096])
@pytest.mark.parametrize("lens,heads,kv", [(([300, 2, 290], [5000, 700, 4000]), 8, 2), (([300], [9000]), 4, 2)])
def test_pages_and_splits(lens, heads, kv, page, dtype, q8):
    """Pages that end inside a tile, positions split over four and eight CTAs."""
    c, batch, g = _cache(lens, kv, 128, page, q8, seed=page)
    q = _randn(batch, heads, 128, dtype, g)
    few, _, blocks, split = _plan(q, batch, kv, q8=q8)
    assert blocks > 0 and split == (4 if len(lens[0]) > 1 else 8)
    out = c.attend(0, q, batch)
    _clean()
    _check(c, 0, batch, q, out)


@pytest.mark.parametrize("dtype,q8", TYPES)
@pytest.mark.parametrize("hd,heads,kv", [(128, 8, 2), (64, 6, 2)])
@pytest.mark.parametrize("cap", [30.0, 50.0, 1e6])
@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("lens", [FEW, MANY])
def test_caps_far_above_the_scores(lens, alibi, cap, hd, heads, kv, dtype, q8):
    """The usual case of a cap: scores that stay below half of it, in every row."""
    import torch

    c, batch, g = _cache(lens, kv, hd, 48, q8, seed=hd)
    q = _randn(batch, heads, hd, dtype, g)
    assert _reaches(lens, q, batch, kv, q8=q8)
    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(heads)], device="cuda") if alibi else None
    out = c.attend(0, q, batch, softcap=cap, slopes=slopes)
    _clean()
    _check(c, 0, batch, q, out, cap=cap, slopes=slopes)


@pytest.mark.parametrize("lens", [FEW, MANY])
@pytest.mark.parametrize("dtype,mult,scale", [("fp32", 300.0, None), ("fp32", 0.0, None), ("fp32", 1e7, 1e-8),
                                              ("fp32", 1e-7, 1e5), ("fp32", 1e-36, 1e35), ("fp32", 1e30, 1e-31),
                                              ("fp16", 300.0, None), ("fp16", 0.0, None), ("fp16", 1e4, 1e-5)])
def test_extreme_scores(lens, dtype, mult, scale):
    """Scores of thousands either way, equal scores, and fp32 queries past
    the range of fp16."""
    c, batch, g = _cache(lens, 2, 128, 16, False, seed=9)
    q = _randn(batch, 8, 128, dtype, g, mult)
    assert _reaches(lens, q, batch, 2)
    out = c.attend(0, q, batch, scale=scale)
    _clean()
    _check(c, 0, batch, q, out, scale=scale)


@pytest.mark.parametrize("dtype,q8", TYPES)
def test_strides_streams_and_untouched_rows(dtype, q8):
    """q as a part of wider rows, out rows apart, another stream, rows behind
    the last sequence, a layer in the middle of the cache."""
    import torch

    from cybel_b200.paged_attention import RaggedBatch

    c, _, g = _cache(MANY, 2, 128, 48, q8, seed=4, layers=3)
    ql, kl = MANY
    batch = RaggedBatch([m + 9 for m in ql[:2]] + [m for m in ql[2:]], [n + 9 for n in kl[:2]] + kl[2:], max_kv=max(kl))
    batch.update(ql, kl)  # fewer rows than the batch holds
    n, used = batch.n_tokens, sum(ql)
    wide = torch.randn(n, 12 * 128, generator=g, device="cuda").to(_dt(dtype))
    q = wide[:, :8 * 128].view(n, 8, 128)
    obuf = torch.full((n, 8 * 128 + 64), 3.0, dtype=q.dtype, device="cuda")
    out = obuf[:, :8 * 128].view(n, 8, 128)
    assert _both(q, batch, 2, q8=q8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.attend(1, q, batch, out=out)
    torch.cuda.current_stream().wait_stream(s)
    _clean()
    assert (obuf[:, 8 * 128:] == 3).all() and (out[used:] == 3).all()
    _check(c, 1, batch, q, out)
    # in place: out may be q
    want = out[:used].clone()
    assert c.attend(1, q, batch, out=q) is q
    _clean()
    assert torch.equal(q[:used], want)


@pytest.mark.parametrize("dtype,q8", TYPES)
def test_more_rows_than_stated(dtype, q8):
    """max_q_len below what a sequence has (a caller of the C entry point's
    mistake): its own rows may stay, those of the others are right."""
    import torch

    ql, kl = [900, 600, 1, 600], [900, 1000, 300, 700]
    c, batch, g = _cache((ql, kl), 2, 128, 64, q8, seed=2)
    q = _randn(batch, 8, 128, dtype, g)
    want = c.attend(0, q, batch)
    batch.max_q = 600
    from tests.test_ragged_plan import plan

    few, _, blocks, _ = plan(dtype, [600] * 4 + [1] * 0, kl, 8, 2, q8=q8)
    assert blocks > 0 and few < 600 * 4
    out = torch.full_like(q, 9.0)
    c.attend(0, q, batch, out=out)
    _clean()
    batch.max_q = 900
    part = out.clone()
    part[:900] = want[:900]  # (the long sequence's own)
    _check(c, 0, batch, q, part)


@pytest.mark.parametrize("dtype,q8", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", [FEW, MANY])
@pytest.mark.parametrize("what", ["values", "keys"])
def test_rows_that_are_not_finite_reach_only_those_that_see_them(what, lens, hd, dtype, q8):
    """Infinities and NaN in cached rows (fp16: one element, Q8: a scale, that
    is a whole row) at positions that a part of a sequence's rows sees: in
    those the formula's infinity or NaN, in the others nothing."""
    c, batch, g = _cache(lens, 2, hd, 16, q8, seed=hd)
    q = _randn(batch, 4, hd, dtype, g, 0.3)  # (small scores: no weight is too small to carry an infinity)
    assert _reaches(lens, q, batch, 2, q8=q8)
    kinds = [(0, float("inf")), (0, float("-inf")), (1, float("nan"))]
    for b, (m, n) in enumerate(zip(*lens)):
        for i, (head, x) in enumerate(kinds if m > 5 else kinds[:1]):
            j = n - 1 - i if m < 20 else n - m // 2 + 17 * i  # seen by the last rows only
            s, o = c.table_host[0, b, j // 16], j % 16
            if m:
                if q8:
                    (c.vs if what == "values" else c.ks)[s, head, o] = x
                else:
                    (c.v if what == "values" else c.k)[s, head, o, 5] = x
    out = c.attend(0, q, batch)
    _clean()
    _check(c, 0, batch, q, out)


@pytest.mark.parametrize("dtype,q8", TYPES)
def test_a_prompt_in_chunks_gives_its_rows_in_one_pass(dtype, q8):
    c, batch, g = _cache(([900], [900]), 2, 128, 32, q8, seed=3)
    from cybel_b200.paged_attention import RaggedBatch

    q = _randn(batch, 16, 128, dtype, g)
    assert _plan(q, batch, 2, q8=q8)[2]
    whole = c.attend(0, q, batch)
    tol = _check(c, 0, batch, q, whole)
    for a, b in ((0, 3), (3, 90), (90, 400), (400, 900)):
        chunk = RaggedBatch([b - a], [b])
        part = c.attend(0, q[a:b], chunk)
        _clean()
        # both are within tol of the same rows
        assert ((part.double() - whole[a:b].double()).abs() <= 2 * tol[a:b]).all()


@pytest.mark.parametrize("dtype,q8", TYPES)
def test_pools_past_32_bits(dtype, q8):
    """Cached rows whose element offsets pass 2^32 (fp16: byte offsets 2^33)."""
    import torch

    from cybel_b200.kv_cache import PagedKVCache
    from cybel_b200.paged_attention import RaggedBatch, RopeTable

    kv, page, slots = 8, 4096, 1100  # 36 million rows of 128
    c = PagedKVCache(1, kv, 2 * page, batch=2, page_size=page, q8=q8, n_slots=slots)
    for b in range(2):
        for p in range(2):
            c.assign(0, b, p, slots - 1 - 2 * b - p)
    c.sync_table()
    assert (slots - 4) * kv * page * 128 > 2 ** 32
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    ql, kl = [4500, 5], [4500, 5]
    batch = RaggedBatch(ql, kl)
    k, v = (torch.randn(batch.n_tokens, kv, 128, generator=g, device="cuda").to(_dt(dtype)) for _ in range(2))
    c.append(0, k, v, batch, rope=RopeTable(128))
    short = RaggedBatch([300, 5], kl)
    q = _randn(short, 16, 128, dtype, g)
    assert _both(q, short, kv, q8=q8)
    out = c.attend(0, q, short)
    _clean()
    _check(c, 0, short, q, out)
    kc, _, ks, _ = c.rows(0, 0, kv - 1, 0, 1)  # the first position, which the rotation leaves as it is
    first = k[0, kv - 1].float().cpu().numpy()
    got = kc[0].astype(np.float32) * (ks[0] if q8 else 1.0)
    assert np.abs(got - first).max() <= np.abs(first).max() * (0.51 / 127 if q8 else 2.0 ** -11)
    low = c.k[:slots - 4]
    assert not any(bool(low[a:a + 100].any()) for a in range(0, slots - 4, 100))  # nothing fell elsewhere


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", [FEW, MANY])
@pytest.mark.parametrize("form", ["causal", "window", "prefix"])
def test_large_value_scales_matter_to_rows_that_see_them_alone(form, lens, hd, dtype):
    """Q8 value scales 2^30 times the others' (fp16 rows: 2^18, to stay in
    their range) at positions that a part of the rows sees: the others lose
    nothing (the unit that a row's weights are kept in follows the scales that
    the row sees)."""
    import torch

    c, batch, g = _cache(lens, 2, hd, 16, True, seed=hd)
    q = _randn(batch, 8, hd, dtype, g)
    assert _reaches(lens, q, batch, 2, window=60 if form == "window" else 0, prefix=form == "prefix", q8=True)
    kw, ref = {}, {}
    if dtype == "fp16":
        c.vs *= 2.0 ** -10
    if form == "window":
        kw["window"] = ref["window"] = 60
    if form == "prefix":
        p = [n - m // 2 if m > 1 else n // 2 for m, n in zip(*lens)]
        kw["prefix"], ref["prefix"] = torch.tensor(p, dtype=torch.int32, device="cuda"), p
    for b, (m, n) in enumerate(zip(*lens)):
        for j in range(n - (m // 3 if m > 20 else 1), n) if form != "window" else range(n - m - 1, n - m + 1):
            if j >= 0:
                c.vs[c.table_host[0, b, j // 16], :, j % 16] *= 2.0 ** (30 if dtype == "fp32" else 18)
    out = c.attend(0, q, batch, **kw)
    _clean()
    _check(c, 0, batch, q, out, **ref)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("hd,heads,kv", [(128, 8, 2), (64, 33, 1)])
@pytest.mark.parametrize("lens", [FEW, MANY])
def test_steep_distance_biases_keep_the_near_positions_exact(lens, hd, heads, kv, q8):
    """Slopes near 1, with which the nearest positions have nearly all the
    weight: a bias is rounded by its own size, not by that of the farthest
    position of its step. (One-hot queries of small scores: no other error.)"""
    import torch

    c, batch, g = _cache(lens, kv, hd, 48, q8, seed=heads)
    q = _one_hot(batch.n_tokens, heads, hd, 0.015625, g)
    assert _reaches(lens, q, batch, kv, q8=q8)
    slopes = torch.tensor([0.97 - 0.015 * h for h in range(heads)], device="cuda")
    out = c.attend(0, q, batch, scale=1.0, slopes=slopes)
    _clean()
    _check(c, 0, batch, q, out, scale=1.0, slopes=slopes, terms=1)


@pytest.mark.parametrize("dtype,q8", TYPES)
@pytest.mark.parametrize("lens", [FEW, MANY])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_a_query_row_that_is_not_finite_stays_alone(cap, lens, dtype, q8):
    """NaN and infinities in a few query rows: every other row has the bits it
    has without them."""
    import torch

    c, batch, g = _cache(lens, 2, 128, 48, q8, seed=7)
    q = _randn(batch, 8, 128, dtype, g)
    assert _reaches(lens, q, batch, 2, q8=q8)
    want = c.attend(0, q, batch, softcap=cap)
    bad = torch.zeros(batch.n_tokens, 8, dtype=torch.bool, device="cuda")
    for i, x in ((0, float("nan")), (5, float("inf")), (8, float("-inf")), (batch.n_tokens - 3, float("nan"))):
        q[i, i % 8, 9] = x
        bad[i, i % 8] = True
    out = c.attend(0, q, batch, softcap=cap)
    _clean()
    assert torch.equal(out[~bad], want[~bad]) and torch.isnan(out[0, 0]).all()


@pytest.mark.parametrize("dtype,q8", TYPES)
@pytest.mark.parametrize("seqs,m,n", [(64, 1, 8000), (64, 1, 32000), (16, 8, 30000), (2, 600, 6000), (1, 1300, 30000)])
def test_long_sums_of_one_sign(seqs, m, n, dtype, q8):
    """Values that are all near 1, whose sums grow with every position: what a
    sum loses must not grow with its length. (The tensor cores cut their
    accumulators off, by 0.11 x 2^-24 a position. One-hot queries, whose scores
    carry no error of a sum that would cover it.)"""
    heads = 8 if m < 600 else 32
    kv = 8 if m < 600 else 1
    c, batch, g = _cache(([m] * seqs, [n] * seqs), kv, 128, 256, q8, seed=1)
    if q8:
        c.v.random_(90, 128)
        c.vs.fill_(0.01)
    else:
        c.v.normal_(1.0, 0.1)
    q = _one_hot(batch.n_tokens, heads, 128, 0.0625, g).to(_dt(dtype))
    assert bool(_plan(q, batch, kv, q8=q8)[2]) == (m >= 600)
    out = c.attend(0, q, batch, scale=1.0)
    _clean()
    rows = list(range(0, m, max(m // 3, 1)))  # some rows of the first sequence
    from cybel_b200.paged_attention import RaggedBatch

    for t in rows:
        one = RaggedBatch([1], [n - m + t + 1])
        _check(c, 0, one, q[t:t + 1], out[t:t + 1], scale=1.0, terms=1)


@pytest.mark.parametrize("q8", [False, True])
def test_a_step_over_two_million_positions(q8):
    """fp16 rows of many sequences at once (which share their pages), so that
    few CTAs would split each."""
    from cybel_b200.kv_cache import PagedKVCache
    from cybel_b200.paged_attention import RaggedBatch
    import torch

    seqs, n = 256, 2 ** 21
    c = PagedKVCache(1, 1, n, batch=seqs, page_size=4096, q8=q8, n_slots=n // 4096)
    c.table_host[...] = np.arange(n // 4096, dtype=np.int32)
    c.sync_table()
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    if q8:
        c.k.random_(-127, 128)
        c.v.random_(90, 128)
        c.vs.fill_(0.01)
    else:
        c.k.normal_()
        c.v.normal_(1.0, 0.1)
    batch = RaggedBatch([1] * seqs, [n] * seqs)
    q = _one_hot(seqs, 4, 128, 0.0625, g).half()
    assert not _plan(q, batch, 1, q8=q8)[2]
    out = c.attend(0, q, batch, scale=1.0)
    _clean()
    _check(c, 0, RaggedBatch([1], [n]), q[:1], out[:1], scale=1.0, terms=1)


@pytest.mark.parametrize("dtype,q8", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,m,heads", [(100_000, 1300, 32), (1_000_000, 1300, 32), (1_000_000, 300, 4)])
def test_sums_over_a_million_positions(n, m, heads, hd, dtype, q8):
    """A chunk of a long prompt whose blocks of rows fill the device, so that
    their positions need no split for that: values of one sign."""
    from cybel_b200.paged_attention import RaggedBatch

    c, batch, g = _cache(([m], [n]), 1, hd, 4096, q8, seed=1)
    if q8:
        c.v.random_(90, 128)
        c.vs.fill_(0.01)
    else:
        c.v.normal_(1.0, 0.1)
    q = _one_hot(batch.n_tokens, heads, hd, 0.0625, g).to(_dt(dtype))
    assert _plan(q, batch, 1, q8=q8)[2]
    out = c.attend(0, q, batch, scale=1.0)
    _clean()
    for t in (0, m // 2, m - 1):
        _check(c, 0, RaggedBatch([1], [n - m + t + 1]), q[t:t + 1], out[t:t + 1], scale=1.0, terms=1)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_masks_beside_a_context_past_the_plain_sums(hd, q8):
    """A context that eight CTAs cannot split into sums of 32768 positions: the
    many-row kernel's fp16 rows add their products in fp32, here with a
    window, a prefix, a cap and biases, for a long sequence and short ones."""
    import torch

    from cybel_b200.paged_attention import RaggedBatch

    ql, kl, kv, heads = [700, 1, 300], [300_000, 500, 300], 2, 8
    c, batch, g = _cache((ql, kl), kv, hd, 512, q8, seed=5)
    q = _randn(batch, heads, hd, "fp16", g, 2.0)
    prefix = torch.tensor([300, 40, 290], dtype=torch.int32, device="cuda")
    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(heads)], device="cuda")
    for kw in (dict(window=1500), dict(window=1500, softcap=30.0), dict(window=200, slopes=slopes)):
        assert _plan(q, batch, kv, prefix=1, q8=q8)[2:] != (0, 0)
        out = c.attend(0, q, batch, prefix=prefix, **kw)
        _clean()
        ref = dict(window=kw["window"], cap=kw.get("softcap", 0.0), slopes=kw.get("slopes"))
        at = 0
        for b, (m, n) in enumerate(zip(ql, kl)):
            for t in sorted({0, 1, m // 2, m - 1} & set(range(m))):
                one = RaggedBatch([0] * b + [1], [0] * b + [n - m + t + 1])
                pre = [0] * b + [int(prefix[b])]
                if n - m + t + 1 < pre[b]:  # (positions of the prefix behind the row are not in this shorter view)
                    continue
                _check(c, 0, one, q[at + t:at + t + 1], out[at + t:at + t + 1], prefix=pre, **ref)
            at += m
