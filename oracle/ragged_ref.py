"""CPU restatement of the ragged paged operators in 64 bits -- TEST
INFRASTRUCTURE ONLY (imported by tests; never by the product).

* ``frequencies`` / ``rope``: rotary positions, pairs interleaved or in
  halves, part of a head, scaled frequencies; angles in float64.
* ``attention``: one sequence's query rows over its cached keys and values,
  with the first-order bound of what 32-bit arithmetic may add per output.

The Q8 row quantizer is oracle/paged_kv_ref.py's (model_graph.cpp:1545-1573).
"""

from __future__ import annotations

import math

import numpy as np


def frequencies(rot, theta, scaling="none", factor=1.0, original=0, low=None, high=None):
    """(radians per position of each pair, the factor on cos and sin)."""
    f = np.asarray([theta ** (-2.0 * p / rot) for p in range(rot // 2)])
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "llama3":
        low, high = 1.0 if low is None else low, 4.0 if high is None else high
        keep = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0.0, 1.0)
        return f * keep + f / factor * (1 - keep), 1.0
    assert scaling == "yarn"
    low, high = 1.0 if low is None else low, 32.0 if high is None else high

    def pair(turns):
        return rot * math.log(original / (2 * math.pi * turns)) / (2 * math.log(theta))

    a, b = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), rot - 1)
    b = b if b > a else a + 0.001
    slow = np.clip((np.arange(rot // 2) - a) / (b - a), 0.0, 1.0)
    return f / factor * slow + f * (1 - slow), 0.1 * math.log(factor) + 1.0


def rope(x, pos, freq, mag, half):
    """x [rows][heads][hd] rotated to pos [rows], float64."""
    y = np.array(x, dtype=np.float64)
    n = len(freq)
    ang = np.asarray(pos, np.float64)[:, None] * freq[None, :]
    c, s = (np.cos(ang) * mag)[:, None, :], (np.sin(ang) * mag)[:, None, :]
    a = y[..., :n].copy() if half else y[..., 0:2 * n:2].copy()
    b = y[..., n:2 * n].copy() if half else y[..., 1:2 * n:2].copy()
    if half:
        y[..., :n], y[..., n:2 * n] = a * c - b * s, a * s + b * c
    else:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = a * c - b * s, a * s + b * c
    return y


def attention(q, k, v, pos, n, scale, cap=0.0, slopes=None, window=0, prefix=0, present=None):
    """q [rows][heads][hd] at positions pos [rows] over k, v [n][kv][hd]
    (values as stored): (out, bound) [rows][heads][hd] in float64.

    bound is the first-order effect on the output of the 32-bit roundings of
    the scores: score j may be off by
      d_j = scale sum|q||k| ((hd + 8) 2^-24 + 2^-22)   products, sums, split q
            + (|s_j| + |bias_j|) 2^-22                 scale, exponent argument
            + cap 2^-20                                tanh from exponentials,
    and an output by sum_j p_j d_j (|v_j| + |out|), doubled for what is of
    second order. The roundings of the softmax weights and of the output are
    for the caller to add, relative to ``spread`` = sum_j p_j |v_j|, the third
    result."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    rows, heads, hd = q.shape
    g = heads // k.shape[1]
    j = np.arange(n)
    out = np.zeros((rows, heads, hd))
    bound, spread = np.zeros_like(out), np.zeros_like(out)
    for t in range(rows):
        i = int(pos[t])
        see = (j <= i) & ((i - j < window) if window else True) | (j < prefix)
        if present is not None:
            see &= present
        js = np.nonzero(see)[0]
        if i < 0 or not len(js):
            continue
        for h in range(heads):
            kk, vv = k[js, h // g], v[js, h // g]
            s = scale * (kk @ q[t, h])
            mag = scale * (np.abs(kk) @ np.abs(q[t, h]))
            if cap:
                s = cap * np.tanh(s / cap)
            bias = slopes[h] * np.abs(i - js) if slopes is not None else np.zeros(len(js))
            d = mag * ((hd + 8) * 2.0 ** -24 + 2.0 ** -22) + (np.abs(s) + np.abs(bias)) * 2.0 ** -22 + cap * 2.0 ** -20
            s = s - bias
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h] = p @ vv
            spread[t, h] = p @ np.abs(vv)
            bound[t, h] = 2 * ((p * d) @ np.abs(vv) + (p @ d) * np.abs(out[t, h]))
    return out, bound, spread
