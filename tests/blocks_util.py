"""Rotary positions on several axes, key bounds, the choice of pages and attention over them, restated in float64 for the tests.

Rotation: cos and sin are off by at most 2^-22 + |position| 2^-48 (the fraction of the turns is exact to that in fp64; the
fp32 functions are good to two units of 2^-24, the low part of the fraction enters to first order), the rotation adds two
roundings of fp32, and the result is rounded to its type: |dy| <= (|lo| + |hi|) (2^-22 + |p| 2^-48 + 2^-23) + half a step.

Attention: the bounds of scored_util over the listed keys.
"""

from __future__ import annotations

import numpy as np

import cases
import oracle as O
import scored_util as su


def pair_axes(sections, D, interleaved):
    """The axis of each pair of dims."""
    half, A = D // 2, len(sections)
    if not interleaved:
        return np.repeat(np.arange(A), sections)
    axis = np.zeros(half, np.int64)
    for a in range(1, A):
        axis[a:a + A * sections[a]:A] = a
    return axis


def rotate(x, positions, sections, interleaved, theta, act):
    """x [B, S, H, D] float64, positions [A, B, S]: the rotated values and their bound."""
    D = x.shape[-1]
    half = D // 2
    i = np.arange(half, dtype=np.longdouble)
    rate = np.longdouble(np.float32(theta)) ** (-2 * i / D)
    pos = positions[pair_axes(sections, D, interleaved)].transpose(1, 2, 0).astype(np.longdouble)  # [B, S, half]
    angle = np.fmod(pos * rate, 2 * np.arccos(np.longdouble(-1)))[:, :, None]
    c, s = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
    lo, hi = x[..., :half], x[..., half:]
    y = np.concatenate((lo * c - hi * s, hi * c + lo * s), axis=-1)
    d = 2.0 ** -22 + 2.0 ** -23 + np.abs(pos[:, :, None]).astype(np.float64) * 2.0 ** -48
    e = (np.abs(lo) + np.abs(hi)) * d
    bound = np.concatenate((e, e), axis=-1) + su.HALF[act] * np.abs(y) + 1e-30
    if act == O.DTYPE_F16:
        bound += 2.0 ** -25
    return y, bound


def toward(x, down):
    """float32 as the bf16 (as float32) next to it toward -inf (down) or +inf."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    u = np.where(((u >> 31) != 0) == down, u + np.uint32(0xFFFF), u) & np.uint32(0xFFFF0000)
    return np.where(np.isnan(x), np.float32(np.nan), u.astype(np.uint32).view(np.float32))


def keys32(c):
    """The K pool's values as the kernel forms them, float32."""
    if c.kv == O.DTYPE_I8:
        return c.k_pool.astype(np.float32) * c.k_scale[..., None]
    if c.kv == O.DTYPE_FP8:
        return O.e4m3_to_f32(c.k_pool) * c.k_scale[:, None]
    return cases.decode(c.k_pool, c.kv)


def bounds(c, before, new, keys=None):
    """The bounds [N, Hkv, 2, D] float32 after `new` tokens from c.ctx on; `before` where nothing is written."""
    out = before.copy()
    x = keys32(c) if keys is None else keys
    eight = c.kv in (O.DTYPE_I8, O.DTYPE_FP8)
    for b in range(c.B):
        first, end = int(c.ctx[b]), min(int(c.ctx[b]) + new, c.max_blocks * 16)
        for page in range(max(first, 0) // 16, max(0, (end + 15) // 16)):
            phys = c.block_table[b, page]
            if not 0 <= phys < c.num_blocks:
                continue
            live = x[phys, :min(16, end - 16 * page)]
            lo, hi = live.min(axis=0), live.max(axis=0)
            out[phys, :, 0] = toward(lo, True) if eight else lo
            out[phys, :, 1] = toward(hi, False) if eight else hi
    return out


def select(q, box, table, ctx, count, sinks, recent, query_block, num_blocks, most=0):
    """Lists [B, blocks, Hkv, count]: q [B, S, Hq, D] and box [N, Hkv, 2, D] float64."""
    B, S, Hq, D = q.shape
    Hkv, T = box.shape[1], query_block
    blocks = -(-S // T)
    out = np.full((B, blocks, Hkv, count), -1, np.int32)
    cap = table.shape[1] if most <= 0 else min(table.shape[1], -(-most // 16))
    for b in range(B):
        phys = table[b, :cap]
        on = (phys >= 0) & (phys < num_blocks)
        for r in range(blocks):
            last = int(ctx[b]) + min((r + 1) * T, S) - 1
            n = min(0 if last < 0 else last // 16 + 1, cap)
            for h in range(Hkv):
                if n <= count:
                    out[b, r, h, :n] = np.arange(n)
                    continue
                x = q[b, r * T:(r + 1) * T, h * Hq // Hkv:(h + 1) * Hq // Hkv].reshape(-1, D)
                k = box[np.where(on, phys, 0)[:n], h]  # [n, 2, D]
                with np.errstate(invalid="ignore"):
                    score = np.zeros(n)
                    for row in x:
                        score += np.maximum(row * k[:, 0], row * k[:, 1]).sum(axis=1)
                score = np.where(on[:n], score, -np.inf).astype(np.float32)
                key = np.where(np.isnan(score), np.inf, score).astype(np.float64)
                key = np.where(np.isnan(score), 1e300, np.where(np.isinf(score) & (score > 0), 1e299, key))
                between = np.arange(sinks, n - recent)
                order = between[np.argsort(-key[between], kind="stable")][:count - sinks - recent]
                out[b, r, h] = np.sort(np.concatenate((np.arange(sinks), order, np.arange(n - recent, n))))
    return out


def attend(c, q, lists, query_block, act, S, p_step):
    """Outputs [B, S, Hq, D] and their bound: q [B, S, Hq, D] float64 over the pages of lists [B, blocks, Hkv, count]."""
    kf, vf = su.values(c, "k"), su.values(c, "v")
    G, T = c.Hq // c.Hkv, query_block
    out, bound = np.zeros((c.B, S, c.Hq, c.D)), np.zeros((c.B, S, c.Hq, c.D))
    for b in range(c.B):
        total = min(int(c.ctx[b]) + S, c.max_blocks * 16)
        for r in range(-(-S // T)):
            t = np.arange(r * T, min((r + 1) * T, S))
            pos = int(c.ctx[b]) + t
            for h in range(c.Hkv):
                lp = lists[b, r, h].astype(np.int64)
                lp = np.sort(lp[(lp >= 0) & (lp < c.max_blocks)])
                phys = c.block_table[b, lp] if len(lp) else np.zeros(0, np.int64)
                ok = (phys >= 0) & (phys < c.num_blocks)
                lp, phys = lp[ok], phys[ok]
                key = (lp[:, None] * 16 + np.arange(16)).reshape(-1)
                live = key < total
                k = kf[phys, :, h].reshape(-1, c.D)[live][:, None]
                v = vf[phys, :, h].reshape(-1, c.D)[live][:, None]
                end = (key[live][None] <= pos[:, None]).sum(axis=1)
                heads = slice(h * G, (h + 1) * G)
                with np.errstate(invalid="ignore", over="ignore"):
                    o, e, _, _ = su.attention(q[b, t][:, heads], k, v, 0, end=end, act=act, kv=c.kv, p_step=p_step)
                out[b, t, heads], bound[b, t, heads] = o, e
    return out, bound
