"""Attention under a score rule and the weights it gives, in float64 with error bounds, for the tests of the scored kernels.

The bounds count roundings (half a step each, relative: bf16 2^-8, fp16 2^-11, fp32 2^-24) of what the kernels compute:

  scores    fp32 sums of D products of exact operands (quantized values: code times scale, one rounding), q as a hi + lo
            pair of 16-bit parts where its type is another (off by 2^-16 of q at most), the softmax scale and log2(e)
            folded in: |ds| <= (D + 8) 2^-24 A + 2^-16 A (pair), A = scale * sum |q_d k_d|.  The cap's slope is at most 1; it adds 2^-21 of the cap.
            The bias adds 2^-22 of itself (slope * log2 e rounded, one fused multiply-add).
  weights   p off by exp(2 max |ds|) - 1 (numerator and denominator) and 2^-20 (exponent argument up to 2^6 rounded at 2^-18 of
            its last bits, exponential, sums, reciprocal): (n / 2^12 + 16) 2^-20 for n keys.
  output    as the weights, times sum p |v|; P enters the products in fp16 or as a bf16 pair (2^-11 of it, and 2^-25 absolute
            where fp16 is subnormal, per key) and the output is rounded to its type.  The prefill's denominator sums the
            rounded P too: p_step = 2^-10; its bf16 V enters in fp16 (2^-25 absolute below 2^-14).
"""

from __future__ import annotations

import numpy as np
import torch

import cases
import oracle as O

HALF = {O.DTYPE_F32: 2.0 ** -24, O.DTYPE_F16: 2.0 ** -11, O.DTYPE_BF16: 2.0 ** -8}
NAN = {O.DTYPE_F32: np.float32(np.nan), O.DTYPE_BF16: 0x7FC0, O.DTYPE_F16: 0x7E00, O.DTYPE_FP8: 0x7F}
INF = {O.DTYPE_F32: np.float32(np.inf), O.DTYPE_BF16: 0x7F80, O.DTYPE_F16: 0x7C00}


def values(c, which):
    """The pool's values in float64."""
    pool, scale = (c.k_pool, c.k_scale) if which == "k" else (c.v_pool, c.v_scale)
    if c.kv == O.DTYPE_I8:
        return pool.astype(np.float64) * scale[..., None].astype(np.float64)
    if c.kv == O.DTYPE_FP8:
        return O.e4m3_to_f32(pool).astype(np.float64) * scale[:, None].astype(np.float64)
    return cases.decode(pool, c.kv).astype(np.float64)


def attention(q, k, v, pos, cap=0.0, slopes=None, window=0, begin=None, end=None, total=None, absent=None, act=None, kv=None,
              p_step=2.0 ** -11):
    """q [S, Hq, D] at positions pos .. pos + S - 1 over k, v [T, Hkv, D] (v None: the weights alone), float64 arrays.
    begin / end [S]: visible range of each query; total: the row's tokens; absent [T]: keys on no page.
    Returns out, its bound, weights [Hkv, T], their bound."""
    S, Hq, D = q.shape
    T, Hkv, _ = k.shape
    G = Hq // Hkv
    scale = 1.0 / np.sqrt(np.float64(D))
    i, j = pos + np.arange(S), np.arange(T)
    lo = np.zeros(S, np.int64) if begin is None else np.maximum(begin, 0)
    if window:
        lo = np.maximum(lo, i + 1 - window)
    hi = i + 1 if end is None else end
    seen = (j[None] >= lo[:, None]) & (j[None] < hi[:, None]) & (j[None] < (T if total is None else total))
    if absent is not None:
        seen &= ~absent[None]
    out, bound = np.zeros((S, Hq, D)), np.zeros((S, Hq, D))
    w, wb = np.zeros((Hkv, T)), np.zeros((Hkv, T))
    pair = 0.0 if act == kv or kv in (None, O.DTYPE_F32) else 2.0 ** -16
    for h in range(Hq):
        kh = k[:, h // G]
        k0 = np.where(seen.any(axis=0)[:, None], kh, 0.0)  # what no query sees plays no part, whatever it holds
        s = q[:, h] @ k0.T * scale
        ds = (np.abs(q[:, h]) @ np.abs(k0).T * scale) * ((D + 8) * 2.0 ** -24 + pair)
        if cap:
            s = cap * np.tanh(s / cap)
            ds = ds + cap * 2.0 ** -21
        if slopes is not None:
            b = np.float64(slopes[h]) * np.abs(i[:, None] - j[None])
            s, ds = s - b, ds + np.abs(b) * 2.0 ** -22 + 2.0 ** -22 * np.abs(s)
        s = np.where(seen, s, -np.inf)
        any_ = seen.any(axis=1)
        m = np.where(any_, s.max(axis=1, initial=-np.inf), 0.0)
        p = np.exp(s - m[:, None])
        l = p.sum(axis=1)
        p = p / np.where(l == 0, 1.0, l)[:, None]
        n = seen.sum(axis=1)
        # keys far below the maximum count in no sum: their scores' errors do not matter
        dm = np.where(seen & (p > 1e-9), ds, 0.0).max(axis=1, initial=0.0)
        rel = np.expm1(dm[:, None] + np.where(seen, ds, 0.0)) + ((n / 4096 + 16) * 2.0 ** -20)[:, None]
        w[h // G] += p.sum(axis=0)
        wb[h // G] += (p * rel).sum(axis=0) + 2.0 ** -120
        if v is None:
            continue
        vh = v[:, h // G]
        v0 = np.where(seen.any(axis=0)[:, None], vh, 0.0)
        out[:, h] = p @ v0
        exact = kv == O.DTYPE_F32
        step = np.abs(v0).max(initial=0.0) * (2.0 ** -25 * n if not exact else 0.0 * n)
        if kv == O.DTYPE_BF16:
            step = step + 2.0 ** -25
        if kv == O.DTYPE_I8:  # P carries the scales: an absolute 2^-25 of codes up to 127
            step = np.maximum(step, 127 * 2.0 ** -25 * n)
        bound[:, h] = (p * (rel + (0.0 if exact else p_step))) @ np.abs(v0) + step[:, None]
    if act is not None:
        bound += HALF[act] * np.abs(out) + 1e-30
    return out, bound, w, wb


def row(c, b, n, kf, vf):
    """Keys and values of the first n tokens of row b, and which of them lie on no page."""
    pages = c.block_table[b, :(n + 15) // 16]
    ok = (pages >= 0) & (pages < c.num_blocks)
    at = np.where(ok, pages, 0)
    absent = np.repeat(~ok, 16)[:n]
    return (kf[at].reshape(-1, c.Hkv, c.D)[:n], None if vf is None else vf[at].reshape(-1, c.Hkv, c.D)[:n], absent)


def poison(c, b, t):
    """Token t of row b holds what no query may meet: NaN in K, infinity or NaN in V (int8: its scales)."""
    page, slot = int(c.block_table[b, t // 16]), t % 16
    if page < 0:
        return
    if c.kv == O.DTYPE_I8:
        c.k_scale[page, slot] = np.nan
        c.v_scale[page, slot] = np.inf
        return
    c.k_pool[page, slot] = NAN[c.kv]
    c.v_pool[page, slot] = INF.get(c.kv, NAN[c.kv]) if t % 2 else NAN[c.kv]


def device(c, dev):
    """The case's tensors on the GPU: k_pool, v_pool, k_scale, v_scale, table, ctx, k_new, v_new, q."""
    import gpu_util as gu

    up = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    return (gu.to_dev(c.k_pool, c.kv, dev), gu.to_dev(c.v_pool, c.kv, dev), up(c.k_scale), up(c.v_scale),
            up(c.block_table), up(c.ctx), gu.to_dev(c.k_new, c.act, dev), gu.to_dev(c.v_new, c.act, dev),
            gu.to_dev(c.q, c.act, dev))


def host(t):
    return t.float().cpu().numpy().astype(np.float64)


def check(got, want, bound, what):
    err = np.abs(got - want)
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(np.nanmax(np.where(bad, err / bound, 0))), np.argwhere(bad)[:4].tolist())
