"""Attention over listed pages whose values are small or of very different sizes, against float64 with bounds that go with them.

The error of an output is counted in sum p |v|, never in absolute terms: scores, softmax and output as in scored_util; P in the
products 2^-11 (tiles of many tokens 2^-10, whose denominator sums the rounded P) of itself, and where it enters as fp16 and is
subnormal there, 2^-25 of the row's largest value per key; bf16 pages of tiles enter in fp16 while that is off by no more than
2^-11 of a query's largest output."""

import types

import numpy as np
import pytest

import blocks_util as bu
import cases
import oracle as O
import scored_util as su
from test_gpu_attention_blocks import lists, make, run

pytestmark = pytest.mark.gpu


def scaled(c, by):
    """Every value of V times `by` (its power of two in the scales of 8-bit caches)."""
    if c.kv in (O.DTYPE_I8, O.DTYPE_FP8):
        c.v_scale = (c.v_scale * np.float32(by)).astype(np.float32)
    else:
        c.v_pool = cases.encode((cases.decode(c.v_pool, c.kv) * np.float32(by)).astype(np.float32), c.kv)
    return c


def expect(c, li, T):
    S, q = c.q.shape[1], cases.decode(c.q, c.act).astype(np.float64)
    kf, vf = su.values(c, "k"), su.values(c, "v")
    wide = types.SimpleNamespace(B=c.B, Hq=c.Hq, Hkv=c.Hkv, D=c.D, ctx=c.ctx, max_blocks=c.max_blocks, num_blocks=c.num_blocks,
                                 block_table=c.block_table, kv=O.DTYPE_F32, k_pool=kf, v_pool=vf)
    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(su, "values", lambda o, which: o.k_pool if which == "k" else o.v_pool)
        want, bound = bu.attend(wide, q, li, T, c.act, S, 0.0)
        wide.v_pool = np.abs(vf)
        mass, _ = bu.attend(wide, q, li, T, c.act, S, 0.0)
    most = np.abs(vf).max() if c.kv != O.DTYPE_I8 else 0.0
    bound = bound + mass * (2.0 ** -10 if T > 1 else 2.0 ** -11) + most * 2.0 ** -25 * li.shape[-1] * 16
    if c.kv == O.DTYPE_I8:
        bound = bound + mass.max(axis=-1, keepdims=True) * 2.0 ** -25 * li.shape[-1] * 16
    if c.kv == O.DTYPE_BF16 and T > 1:
        bound = bound + 2.0 ** -11 * np.abs(want).max(axis=-1, keepdims=True)
    if c.act == O.DTYPE_F16:  # outputs below 2^-14 are fp16's multiples of 2^-24, half of which is 2^-25
        bound = bound + 2.0 ** -25
    return want, bound


STEPS = [  # whole and split lists, tokens one by one
    (8, 2, 128, [700, 33], 1, 20, 1), (8, 2, 128, [4000], 1, 200, 1), (14, 2, 80, [900], 1, 30, 1), (4, 1, 256, [500], 1, 20, 1),
    (20, 1, 112, [900, 5], 1, 33, 1), (8, 2, 128, [257], 5, 8, 2),
]
KV = [("bf16", "i8"), ("f16", "i8"), ("f32", "i8"), ("bf16", "bf16"), ("bf16", "fp8"), ("f16", "f16"), ("f32", "f32")]
SMALL = [(*k, by) for k in KV for by in (2.0 ** -10, 2.0 ** -17, 2.0 ** -40) if by > 2.0 ** -20 or "f16" not in k]  # (f16's zeros)


def small(ff, gpu, act, kv, by, Hq, Hkv, D, ctx, S, count, T):
    c = scaled(make(Hq + S, ctx, S, Hq, Hkv, D, act, kv), by)
    li = lists(c, S, count, T)
    want, bound = expect(c, li, T)
    su.check(su.host(run(ff, c, li, T, gpu)).reshape(want.shape), want, bound, "out")


@pytest.mark.parametrize("act,kv,by", SMALL)
@pytest.mark.parametrize("form", STEPS)
def test_steps(ff, gpu, act, kv, by, form):
    small(ff, gpu, act, kv, by, *form)


def int8_of_all_sizes(ff, gpu, big, Hq, Hkv, D, ctx, S, count, T):
    """Scales from 2^-30 to `big` within a row, the largest on keys that get little or no weight."""
    c = make(Hq * S, ctx, S, Hq, Hkv, D, "bf16", "i8", spread=6.0)
    c.v_scale = (c.v_scale * np.float32(2) ** c.rng.integers(-30, -9, c.v_scale.shape)).astype(np.float32)
    for b in range(c.B):  # keys of zero, which others outweigh
        some = c.block_table[b, c.rng.permutation(max(1, (int(c.ctx[b]) + S) // 16))[:3]]
        c.v_scale[some] = np.float32(big / 127)
        c.k_pool[some] = 0
    li = lists(c, S, count, T)
    want, bound = expect(c, li, T)
    su.check(su.host(run(ff, c, li, T, gpu)).reshape(want.shape), want, bound, "out")


@pytest.mark.parametrize("big", [1.0, 3000.0, 2.0 ** 30])
@pytest.mark.parametrize("form", STEPS)
def test_int8_steps_of_all_sizes(ff, gpu, big, form):
    int8_of_all_sizes(ff, gpu, big, *form)

TILES = [  # whole, in halves, split over their lists
    (8, 2, 128, [257], 270, 8, 2), (10, 2, 256, [700, 15], 140, 30, 40), (32, 1, 64, [500], 520, 21, 9),
    (36, 9, 128, [1100, 1300], 120, 61, 16), (24, 12, 64, [1700, 900], 130, 107, 16),
    (8, 2, 128, [2500, 40, 1200], 40, 150, 32), (5, 1, 64, [3000], 107, 170, 7), (20, 4, 256, [1531, 1908], 31, 100, 13),
]


@pytest.mark.parametrize("act,kv,by", SMALL)
@pytest.mark.parametrize("form", TILES)
def test_tiles(ff, gpu, act, kv, by, form):
    small(ff, gpu, act, kv, by, *form)


@pytest.mark.parametrize("big", [1.0, 3000.0, 2.0 ** 30])
@pytest.mark.parametrize("form", TILES)
def test_int8_tiles_of_all_sizes(ff, gpu, big, form):
    int8_of_all_sizes(ff, gpu, big, *form)


@pytest.mark.parametrize("Hq,Hkv,D,ctx,S,count,T", [(16, 4, 64, [2, 5, 9, 14], 1, 1, 1), (16, 2, 128, [3, 7, 20], 1, 2, 1),
                                                    (8, 2, 128, [3, 4], 6, 2, 2), (4, 2, 256, [1, 6], 1, 1, 1)])
def test_f16_pages_keep_p(ff, gpu, Hq, Hkv, D, ctx, S, count, T):
    """fp32 queries (fp16 values) over few tokens of fp16 pages, nearly equal weights: P takes part in 21 bits, not in fp16's 11.  The
    bound: scores, softmax and output in fp32, 2^-20 of sum p |v|, and 2^-25 of |v| a key where P's low part is subnormal."""
    c = make(D + S, ctx, S, Hq, Hkv, D, "f32", "f16", spread=0.1)
    c.q = cases.decode(cases.encode(c.q, O.DTYPE_F16), O.DTYPE_F16)
    li = lists(c, S, count, T)
    kf, vf = su.values(c, "k"), su.values(c, "v")
    wide = types.SimpleNamespace(B=c.B, Hq=Hq, Hkv=Hkv, D=D, ctx=c.ctx, max_blocks=c.max_blocks, num_blocks=c.num_blocks,
                                 block_table=c.block_table, kv=O.DTYPE_F32, k_pool=kf, v_pool=vf)
    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(su, "values", lambda o, which: o.k_pool if which == "k" else o.v_pool)
        want, bound = bu.attend(wide, c.q.astype(np.float64), li, T, c.act, S, 0.0)
        wide.v_pool = np.abs(vf)
        mass, _ = bu.attend(wide, c.q.astype(np.float64), li, T, c.act, S, 0.0)
    bound = bound + mass * 2.0 ** -20 + np.abs(vf).max() * 2.0 ** -25 * count * 16
    su.check(su.host(run(ff, c, li, T, gpu)).reshape(want.shape), want, bound, "out")
