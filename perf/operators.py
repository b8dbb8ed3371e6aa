"""Measured cases of the ragged paged-cache operators.

Three operators that serve a batch of sequences of different lengths over the
paged KV cache (``cybel_b200.kv_cache.PagedKVCache``):

* ``rope``: rotary positions of rows at positions of their own, interleaved or
  half layout, all or part of the head, frequencies scaled for long contexts
  (``RopeTable.rotate``);
* ``append``: the tokens of a ragged batch rotated and written into the
  cache's fp16 or Q8 pages, their queries rotated on the way
  (``PagedKVCache.append``);
* ``attend``: attention of a ragged batch of query tokens (one token, a few, a
  whole prompt) over those pages, with a tanh cap on the scores, a bias that
  falls with distance, a sliding window and a prefix that every query sees
  (``PagedKVCache.attend``).

``own`` false computes the plain form with elementary torch operations in 32
bits; ``own`` true makes the framework's calls.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
_GOLDEN = 0.6180339887498949


# ---- cases --------------------------------------------------------------------
def _rope(name, rows, heads, dim, rot, layout, scaling, far, dtype):
    return dict(name=name, op="rope", rows=rows, heads=heads, dim=dim, rot=rot, layout=layout, scaling=scaling,
                far=far, dtype=dtype)


def _append(name, batch, q_lo, q_hi, past_lo, past_hi, heads, kv_heads, dim, rot, layout, scaling, page, q8, dtype):
    return dict(name=name, op="append", batch=batch, q_lo=q_lo, q_hi=q_hi, past_lo=past_lo, past_hi=past_hi,
                heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, layout=layout, scaling=scaling, page=page, q8=q8,
                dtype=dtype)


def _attend(name, batch, q_lo, q_hi, past_lo, past_hi, heads, kv_heads, dim, page, q8, dtype, cap=0.0, alibi=False,
            window=0, prefix=0, single=0):
    return dict(name=name, op="attend", batch=batch, q_lo=q_lo, q_hi=q_hi, past_lo=past_lo, past_hi=past_hi,
                heads=heads, kv_heads=kv_heads, dim=dim, page=page, q8=q8, dtype=dtype, cap=cap, alibi=alibi,
                window=window, prefix=prefix, single=single)


def listed():
    return [
        # the query heads of one decode step: one token of the 8B stack, fp32 rows, where latency is all
        _rope("rope_one_token", 1, 32, 128, 128, "interleaved", "none", 2048, "fp32"),
        # a long-context prompt of the 70B stack's query heads, the first half of each head rotated, positions far out
        _rope("rope_far_prompt", 8191, 64, 128, 64, "half", "yarn", 1_000_000, "fp16"),
        # one decode step of 48 sequences of the 8B stack: one row each, pages of 64 positions
        _append("append_step_f16", 48, 1, 1, 0, 4000, 32, 8, 128, 128, "interleaved", "none", 64, False, "fp32"),
        # prompts of several sequences of the 70B stack at once into Q8 pages, the long-context frequencies
        _append("append_prompts_q8", 6, 257, 2000, 0, 100, 64, 8, 128, 128, "interleaved", "llama3", 256, True,
                "fp16"),
        # prompts into fp16 pages of an odd size, half layout, part of the head, heads of 64
        _append("append_prompts_odd", 7, 100, 2300, 0, 300, 24, 8, 64, 32, "half", "linear", 48, False, "fp16"),
        # the decode step of one sequence of the 8B stack at context 2048: the smallest attention, latency again
        _attend("attend_one_2048", 1, 1, 1, 2047, 2047, 32, 8, 128, 4096, False, "fp32"),
        # a decode step of a serving batch of ragged lengths, 70B heads, Q8 pages: bound by the cache's bytes
        _attend("attend_batch_q8", 64, 1, 1, 100, 8000, 64, 8, 128, 64, True, "fp16"),
        # a decode step of few sequences with long contexts, where one row's keys have to be split, with the capped
        # scores
        _attend("attend_long_f16", 2, 1, 1, 60_000, 120_000, 32, 8, 128, 256, False, "fp16", cap=30.0),
        # the drafted tokens of a speculative verify for a few sequences, fp32 rows
        _attend("attend_verify_8", 4, 8, 8, 1500, 2500, 32, 8, 128, 64, False, "fp32"),
        # whole prompts of the 8B stack from an empty cache: bound by the matrix products
        _attend("attend_prompts_f16", 4, 2049, 6000, 0, 0, 32, 8, 128, 128, False, "fp16"),
        # a chunk of a long prompt among decode steps of other sequences, sliding window and cap, Q8 pages of which
        # those behind the window are gone
        _attend("attend_mixed_window", 9, 2048, 2048, 9_000, 30_000, 64, 8, 128, 64, True, "fp16", cap=50.0,
                window=4096, single=8),
        # prompts with a prefix that every token sees and the distance bias, heads of 64, fp32 rows, odd pages
        _attend("attend_prefix_bias", 5, 33, 1500, 0, 700, 24, 8, 64, 48, False, "fp32", alibi=True, prefix=129),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend"])
    dim = rng.choice([64, 128, 128])
    layout = rng.choice(["interleaved", "half"])
    scaling = rng.choice(["none", "linear", "llama3", "yarn"])
    dtype = rng.choice(["fp32", "fp16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    rot = rng.choice([dim, dim // 2, dim // 4, dim - 8])
    page = rng.choice([16, 33, 48, 64, 128, 256, 1000, 4096])
    q8 = rng.random() < 0.5
    if op == "rope":
        rows = _log(rng, 1, 6000)
        return dict(_rope("", rows, heads, dim, rot, layout, scaling, _log(rng, rows + 1, 1_000_000), dtype), name=None)
    batch = _log(rng, 1, 40)
    if op == "append":
        q_hi = _log(rng, 1, max(1, 6000 // batch))
        return dict(_append("", batch, max(1, q_hi // rng.choice([1, 2, 9])), q_hi, 0, _log(rng, 1, 3000), heads,
                            kv_heads, dim, rot, layout, scaling, page, q8, dtype), name=None)
    kind = rng.choice(["step", "few", "prompt", "mixed"])
    single = 0
    if kind == "step":
        q_lo = q_hi = 1
        past = _log(rng, 1, max(2, min(60_000, 180_000 // batch)))
    elif kind == "few":
        q_lo, q_hi = 1, _log(rng, 2, 40)
        past = _log(rng, 1, max(2, min(20_000, 120_000 // batch)))
    else:
        batch = _log(rng, 1, 8)
        q_hi = _log(rng, 41, max(42, min(2800, 5000 // batch)))
        q_lo = max(1, q_hi // rng.choice([1, 2, 9]))
        past = _log(rng, 1, 2000)
        single = batch // 2 if kind == "mixed" else 0
    return dict(_attend("", batch, q_lo, q_hi, past // rng.choice([1, 3, 17]), past, heads, kv_heads, dim, page, q8,
                        dtype, cap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.3,
                        window=rng.choice([0, 0, _log(rng, 1, 5000)]), prefix=rng.choice([0, 0, _log(rng, 1, 700)]),
                        single=single), name=None)


# ---- lengths, from the case alone ----------------------------------------------
def _spread(lo, hi, n):
    """n lengths spread over lo .. hi."""
    return [lo + int((hi - lo + 1) * ((0.37 + i * _GOLDEN) % 1.0)) for i in range(n)]


def _lengths(case):
    """(query tokens, positions in the cache after them) of each sequence."""
    b = case["batch"]
    q = _spread(case["q_lo"], case["q_hi"], b)
    for i in range(case.get("single", 0)):  # the sequences of a mixed batch that take one decode step
        q[b - 1 - i] = 1
    past = _spread(case["past_lo"], case["past_hi"], b)[::-1]
    return q, [p + n for p, n in zip(past, q)]


def _dtype(case):
    return torch.float32 if case["dtype"] == "fp32" else torch.float16


def _size(case):
    return 4 if case["dtype"] == "fp32" else 2


def work(case):
    """Bytes that have to be read once and written once, and the operations of the products."""
    e, d = _size(case), case["dim"]
    if case["op"] == "rope":
        n = case["rows"] * case["heads"]
        return {"bytes": 2 * n * d * e + 4 * case["rows"], "flops": 3 * n * case["rot"]}
    q_len, kv_len = _lengths(case)
    tokens = sum(q_len)
    row = case["kv_heads"] * (d + 4 if case["q8"] else 2 * d)  # one position's keys (or values) of all kv heads
    if case["op"] == "append":
        q_bytes = 2 * tokens * case["heads"] * d * e
        kv_bytes = 2 * tokens * case["kv_heads"] * d * e + 2 * tokens * row
        return {"bytes": q_bytes + kv_bytes,
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rot"]}
    pairs, seen = 0, 0
    for q, n in zip(q_len, kv_len):
        w, pre = case["window"], min(case["prefix"], n)
        first = max(0, n - q - w + 1) if w else 0  # the first position that some query's window reaches
        seen += n - first + min(pre, first)
        for t in range(q):
            i = n - q + t
            lo = max(0, i - w + 1) if w else 0
            pairs += i - lo + 1 + min(pre, lo) + max(0, pre - i - 1)
    return {"bytes": 2 * tokens * case["heads"] * d * e + 2 * seen * row, "flops": 4 * pairs * case["heads"] * d}


# ---- inputs --------------------------------------------------------------------
def _frequencies(case):
    """Radians per position of each rotated pair (python floats) and the factor on cos and sin."""
    rot, theta, kind = case["rot"], 500000.0, case["scaling"]
    f = [theta ** (-2.0 * p / rot) for p in range(rot // 2)]
    factor, orig = 8.0, 8192
    if kind == "none":
        return f, 1.0
    if kind == "linear":
        return [x / factor for x in f], 1.0
    if kind == "llama3":
        lo, hi, out = 1.0, 4.0, []
        for x in f:
            turns = orig * x / (2 * math.pi)
            if turns > hi:
                out.append(x)
            elif turns < lo:
                out.append(x / factor)
            else:
                s = (turns - lo) / (hi - lo)
                out.append((1 - s) * x / factor + s * x)
        return out, 1.0

    def at(beta):
        return rot * math.log(orig / (beta * 2 * math.pi)) / (2 * math.log(theta))

    lo, hi = max(0, math.floor(at(32.0))), min(rot - 1, math.ceil(at(1.0)))
    hi = hi if hi > lo else lo + 0.001
    ramp = [min(1.0, max(0.0, (p - lo) / (hi - lo))) for p in range(rot // 2)]
    return [x / factor * r + x * (1 - r) for x, r in zip(f, ramp)], 0.1 * math.log(factor) + 1.0


def _rope_kwargs(case):
    kw = dict(rot_dim=case["rot"], theta=500000.0, layout=case["layout"], scaling=case["scaling"], device=0)
    if case["scaling"] != "none":
        kw.update(factor=8.0, original_context=8192)
    return kw


def _slopes(heads):
    """The geometric slopes of a distance bias over the heads."""
    return [2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = _dtype(case)
    randn = (lambda *s: torch.randn(*s, generator=g, device=DEV))
    st = {"case": case}
    if case["op"] == "rope":
        st["x"] = randn(case["rows"], case["heads"], case["dim"]).to(dt)
        first = case["far"] - case["rows"]
        st["positions"] = first + torch.arange(case["rows"], device=DEV, dtype=torch.int32)
        st["out"] = torch.empty_like(st["x"])
        if own:
            from cybel_b200.paged_attention import RopeTable
            st["rope"] = RopeTable(**_rope_kwargs(case))
        return st

    q_len, kv_len = _lengths(case)
    b, h, kv, d, page, q8 = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "page", "q8"))
    tokens = sum(q_len)
    pages_per_seq = (max(kv_len) + page - 1) // page
    used = [(n + page - 1) // page for n in kv_len]
    slots = sum(used) + 2
    # the slots of the sequences' pages in no order, two left over; pages behind a window (and its prefix) are gone
    order = torch.randperm(slots, generator=g, device=DEV).tolist()
    table = torch.full((1, b, pages_per_seq), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(used):
        table[0, i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
        if case.get("window"):
            gone = max(0, kv_len[i] - q_len[i] - case["window"] + 1) // page
            kept = (min(case["prefix"], kv_len[i]) + page - 1) // page
            table[0, i, kept:max(kept, gone)] = -1
    shape = (slots, kv, page, d)
    if q8:
        k = torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)
        v = torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)
        ks = torch.rand(shape[:3], generator=g, device=DEV) * 0.02 + 0.005
        vs = torch.rand(shape[:3], generator=g, device=DEV) * 0.02 + 0.005
    else:
        k, v = randn(*shape).half(), randn(*shape).half()
        ks = vs = None
    st.update(q_len=q_len, kv_len=kv_len, tokens=tokens, dev_table=table.to(DEV))
    if case["op"] == "append":
        # the rows of one q|k|v projection output
        qkv = randn(tokens, (h + 2 * kv) * d).to(dt)
        st["q"] = qkv[:, :h * d].view(tokens, h, d)
        st["k_new"] = qkv[:, h * d:(h + kv) * d].view(tokens, kv, d)
        st["v_new"] = qkv[:, (h + kv) * d:].view(tokens, kv, d)
        st["q_out"] = torch.empty(tokens, h, d, dtype=dt, device=DEV)
    else:
        st["q"] = randn(tokens, h, d).to(dt)
        st["out"] = torch.empty(tokens, h, d, dtype=dt, device=DEV)
        st["slopes"] = torch.tensor(_slopes(h), device=DEV) if case["alibi"] else None
        st["prefix_host"] = [min(case["prefix"], n) for n in kv_len]
        st["prefix"] = torch.tensor(st["prefix_host"], dtype=torch.int32, device=DEV) if case["prefix"] else None
    if own:
        from cybel_b200.kv_cache import PagedKVCache
        from cybel_b200.paged_attention import RaggedBatch, RopeTable
        cache = PagedKVCache(1, kv, pages_per_seq * page, batch=b, page_size=page, q8=q8, n_slots=slots, head_dim=d)
        cache.k.copy_(k)
        cache.v.copy_(v)
        if q8:
            cache.ks.copy_(ks)
            cache.vs.copy_(vs)
        cache.table_host[...] = table.numpy()
        cache.sync_table()
        k, v, ks, vs = cache.k, cache.v, cache.ks, cache.vs
        st["cache"] = cache
        st["batch"] = RaggedBatch(q_len, kv_len)
        if case["op"] == "append":
            st["rope"] = RopeTable(**_rope_kwargs(case))
    st.update(k=k, v=v, ks=ks, vs=vs)
    return st


# ---- the plain form --------------------------------------------------------------
def _rotate(case, x, pos):
    """x [rows][heads][dim], its first rot elements rotated to pos [rows], in x's type."""
    f, mag = _frequencies(case)
    rot = case["rot"]
    # the angles in 64 bits: far positions lose the phase in 32
    ang = pos.double()[:, None] * torch.tensor(f, dtype=torch.float64, device=x.device)[None, :]
    c, s = (torch.cos(ang) * mag).to(x.dtype)[:, None, :], (torch.sin(ang) * mag).to(x.dtype)[:, None, :]
    out = x.clone()
    if case["layout"] == "interleaved":
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2] = a * c - b * s
        out[..., 1:rot:2] = a * s + b * c
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out[..., :rot // 2] = a * c - b * s
        out[..., rot // 2:rot] = a * s + b * c
    return out


def _plain_append(st):
    case = st["case"]
    q_len, kv_len, page = st["q_len"], st["kv_len"], case["page"]
    pos = torch.cat([torch.arange(n - q, n, device=DEV) for q, n in zip(q_len, kv_len)])
    seq = torch.cat([torch.full((q,), i, device=DEV) for i, q in enumerate(q_len)])
    q = _rotate(case, st["q"].float(), pos)
    if case["q8"]:  # keys next to the border of two codes: rotated in 64 bits
        k = _rotate(case, st["k_new"].double(), pos).float()
    else:
        k = _rotate(case, st["k_new"].float(), pos)
    v = st["v_new"].float()
    slot = st["dev_table"][0, seq, pos // page].long()
    off = pos % page
    for pool, scales, rows in ((st["k"], st["ks"], k), (st["v"], st["vs"], v)):
        if case["q8"]:
            amax = rows.abs().amax(-1)
            scale = torch.where(amax > 0, amax, torch.ones_like(amax)) / torch.full_like(amax, 127.0)
            x = rows * (1.0 / scale)[..., None]
            codes = torch.clamp(torch.sign(x) * torch.floor(x.abs() + 0.5), -127, 127)  # halves away from zero
            pool[slot, :, off] = codes.to(torch.int8)
            scales[slot, :, off] = scale
        else:
            pool[slot, :, off] = rows.half()
    st["q_out"].copy_(q)
    return _append_outputs(st)


def _append_outputs(st):
    if st["case"]["q8"]:  # the pools as the values that their codes stand for
        return st["q_out"], st["k"] * st["ks"][..., None], st["v"] * st["vs"][..., None]
    return st["q_out"], st["k"], st["v"]


def _plain_attend(st):
    case = st["case"]
    h, kv, d, page, w = (case[k] for k in ("heads", "kv_heads", "dim", "page", "window"))
    at = 0
    for i, (q_len, n) in enumerate(zip(st["q_len"], st["kv_len"])):
        j = torch.arange(n, device=DEV)
        slot = st["dev_table"][0, i, j // page].long()
        here = slot >= 0
        slot = slot.clamp(min=0)
        k, v = st["k"][slot, :, j % page].float(), st["v"][slot, :, j % page].float()  # [n][kv][d]
        if case["q8"]:
            k = k * st["ks"][slot, :, j % page][..., None]
            v = v * st["vs"][slot, :, j % page][..., None]
        k, v = k.transpose(0, 1), v.transpose(0, 1)  # [kv][n][d]
        pre = st["prefix_host"][i]
        step = max(1, 2 ** 28 // (h * n))  # query tokens a block, so that the scores stay near a gigabyte
        for t0 in range(0, q_len, step):
            m = min(step, q_len - t0)
            pos = n - q_len + t0 + torch.arange(m, device=DEV)
            q = st["q"][at + t0:at + t0 + m].float().view(m, kv, h // kv, d).permute(1, 2, 0, 3)  # [kv][g][m][d]
            s = torch.matmul(q.reshape(kv, -1, d), k.transpose(1, 2)).view(kv, h // kv, m, n) * (1.0 / math.sqrt(d))
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            if case["alibi"]:
                s = s - st["slopes"].view(kv, h // kv, 1, 1) * (pos[:, None] - j[None, :]).abs()
            see = j[None, :] <= pos[:, None]
            if w:
                see = see & (pos[:, None] - j[None, :] < w)
            if pre:
                see = see | (j < pre)[None, :]
            see = see & here[None, :]
            s = s.masked_fill(~see, float("-inf"))
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
            o = torch.matmul(p.view(kv, -1, n), v).view(kv, h // kv, m, d) / p.sum(-1, keepdim=True).clamp(min=1e-30)
            st["out"][at + t0:at + t0 + m] = o.permute(2, 0, 1, 3).reshape(m, h, d)
        at += q_len
    return st["out"]


def run(st):
    case = st["case"]
    if case["op"] == "rope":
        if own:
            return st["rope"].rotate(st["x"], st["positions"], out=st["out"])
        st["out"].copy_(_rotate(case, st["x"].float(), st["positions"]))
        return st["out"]
    if case["op"] == "append":
        if own:
            st["cache"].append(0, st["k_new"], st["v_new"], st["batch"], rope=st["rope"], q=st["q"], q_out=st["q_out"])
            return _append_outputs(st)
        return _plain_append(st)
    if own:
        return st["cache"].attend(0, st["q"], st["batch"], out=st["out"], softcap=case["cap"], slopes=st["slopes"],
                                  window=case["window"], prefix=st["prefix"])
    return _plain_attend(st)


# ---- the definition in 64 bits -----------------------------------------------------
def _turned(case, x, pos):
    """Pairs of x (64 bits) as complex numbers times mag * exp(i pos f)."""
    f, mag = _frequencies(case)
    rot = case["rot"]
    head, rest = x[..., :rot], x[..., rot:]
    if case["layout"] == "interleaved":
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous())
    else:
        z = torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous())
    ang = torch.outer(pos.double(), torch.tensor(f, dtype=torch.float64, device=x.device))
    z = z * torch.polar(torch.full_like(ang, mag), ang)[:, None, :]
    if case["layout"] == "interleaved":
        head = torch.view_as_real(z).flatten(-2)
    else:
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, rest], -1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        return _turned(case, st["x"].double(), st["positions"])
    page = case["page"]
    if case["op"] == "append":
        starts, pos = 0, []
        k_pool, v_pool = st["k"].double(), st["v"].double()
        if case["q8"]:
            k_pool, v_pool = k_pool * st["ks"].double()[..., None], v_pool * st["vs"].double()[..., None]
        for i, (q, n) in enumerate(zip(st["q_len"], st["kv_len"])):
            p = torch.arange(n - q, n, device=DEV)
            pos.append(p)
            k = _turned(case, st["k_new"][starts:starts + q].double(), p)
            v = st["v_new"][starts:starts + q].double()
            slot = st["dev_table"][0, i][p // page].long()
            for pool, rows in ((k_pool, k), (v_pool, v)):
                if case["q8"]:
                    # the page format defines its codes by 32-bit steps: the row, scale = amax / 127, its inverse,
                    # the product, the nearest integer with halves away from zero
                    f32 = (lambda t: t.float().double())
                    rows = f32(rows)
                    unit = rows.abs().amax(-1, keepdim=True)
                    unit = f32(torch.where(unit > 0, unit, torch.ones_like(unit)) / 127.0)
                    steps = f32(rows * f32(1.0 / unit))
                    rows = torch.trunc(steps + 0.5 * torch.sign(steps)).clamp(-127, 127) * unit
                pool[slot, :, p % page] = rows
            starts += q
        return _turned(case, st["q"].double(), torch.cat(pos)), k_pool, v_pool
    if work(case)["flops"] > 2e13:
        return None
    h, kv, d, w, cap = (case[k] for k in ("heads", "kv_heads", "dim", "window", "cap"))
    g, start = h // kv, 0
    out = torch.zeros(st["tokens"], h, d, dtype=torch.float64, device=DEV)
    for i, (q_len, n) in enumerate(zip(st["q_len"], st["kv_len"])):
        j = torch.arange(n, device=DEV)
        slot = st["dev_table"][0, i][torch.div(j, page, rounding_mode="floor")].long()
        hidden = slot < 0
        slot = slot.masked_fill(hidden, 0)
        pos = torch.arange(n - q_len, n, device=DEV)
        dist = pos[:, None] - j[None, :]
        blocked = dist < 0
        if w:
            blocked |= dist >= w
        blocked &= (j >= st["prefix_host"][i])[None, :]
        blocked |= hidden[None, :]
        empty = blocked.all(-1)
        for c in range(kv):
            keys, vals = st["k"][slot, c, j % page].double(), st["v"][slot, c, j % page].double()
            if case["q8"]:
                keys = keys * st["ks"][slot, c, j % page].double()[:, None]
                vals = vals * st["vs"][slot, c, j % page].double()[:, None]
            for a in range(c * g, (c + 1) * g):
                s = st["q"][start:start + q_len, a].double() @ keys.T / math.sqrt(d)
                if cap:
                    s = torch.tanh(s / cap) * cap
                if case["alibi"]:
                    s = s - st["slopes"][a].double() * dist.abs()
                p = torch.softmax(s.masked_fill(blocked, -torch.inf), -1)
                out[start:start + q_len, a] = (p @ vals).masked_fill(empty[:, None], 0.0)
        start += q_len
    return out
