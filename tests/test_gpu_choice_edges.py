"""The choice of pages where bounds are infinite, in every form that it takes, against the definition in float64."""

import numpy as np
import pytest
import torch

import blocks_util as bu
import cases
import gpu_util as gu

pytestmark = pytest.mark.gpu


def boxes(rng, N, Hkv, D):
    mean, half = rng.standard_normal((N, Hkv, D)) * 0.4, np.abs(rng.standard_normal((N, Hkv, D)) * 0.3 + 1.77)
    return np.stack((mean - half, mean + half), axis=2).astype(np.float32)


def up(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


@pytest.mark.parametrize("act,dtype", [("bf16", torch.bfloat16), ("f32", torch.float32), ("f16", torch.bfloat16)])
@pytest.mark.parametrize("Hq,Hkv,D,S,ctx,T", [
    (8, 2, 128, 1, [1500, 900], 1), (2, 2, 64, 1, [2000], 1), (3, 1, 256, 1, [1200], 1), (6, 2, 80, 2, [700, 1033], 2),
    (8, 2, 128, 33, [800, 1100], 16), (4, 1, 64, 20, [900], 20), (2, 1, 256, 9, [1000], 2), (6, 1, 112, 5, [1300], 1),
])
@pytest.mark.parametrize("wide", [False, True])  # behind a wide table the choice takes other kernels
def test_infinite_bounds(ff, gpu, act, dtype, Hq, Hkv, D, S, ctx, T, wide):
    """Queries of one sign in some dims, of both in others and of none in two: an infinite bound that no query takes adds nothing."""
    c = cases.make_case(Hq + S, len(ctx), Hq, Hkv, 8, ctx, act=act, S=S, max_blocks=4000 if wide else None)
    rng = np.random.default_rng(D + S)
    q = rng.standard_normal((c.B, S, Hq, D), dtype=np.float32) * np.float32(2)
    third = D // 3
    q[..., :third], q[..., third:2 * third] = np.abs(q[..., :third]) + 0.1, -np.abs(q[..., third:2 * third]) - 0.1
    q[..., 5], q[..., D - 2] = 0.0, -0.0
    q = cases.encode(q, c.act)
    box = boxes(rng, c.num_blocks, Hkv, D)
    for n, p in enumerate(rng.permutation(c.num_blocks)[:c.num_blocks // 2]):  # most infinities are of one kind a page
        h, dims = rng.integers(Hkv), rng.integers(0, D, 3)
        if n % 5 == 0:
            dims = np.array([5, D - 2])
        if n % 3 != 1:
            box[p, h, 0, dims] = -np.inf
        if n % 3 != 0:
            box[p, h, 1, dims] = np.inf
        if n % 17 == 0:
            box[p, h, :, dims[0]] = np.inf if n % 2 else -np.inf
    box[c.block_table[0, 20], 0, :, 7] = np.nan
    held = up(box, gpu).to(dtype)
    box = held.double().cpu().numpy()
    got = ff.select_blocks(gu.to_dev(q, c.act, gpu), held, up(c.block_table, gpu), up(c.ctx, gpu), 23, sinks=1, recent=3,
                           query_block=T).cpu().numpy()
    flat = box.copy()  # 0 times infinity is 0 here
    flat[..., [5, D - 2]] = np.where(np.isinf(flat[..., [5, D - 2]]), 0.0, flat[..., [5, D - 2]])
    with np.errstate(invalid="ignore"):
        want = bu.select(cases.decode(q, c.act).astype(np.float64), flat, c.block_table, c.ctx, 23, 1, 3, T, c.num_blocks)
    assert np.array_equal(got, want)


def beside(rng, D, dev, rows, T, pages=60):
    """Row 0's case for any batch: `rows` of the block's query rows in fp32, and two kinds of page whose scores differ by a rounding."""
    S = T
    q = np.zeros((1, S, 1, D), np.float32)
    for at, v in rows:
        q[0, at, 0, 0] = v
    q[0, 0, 0, 1] = 1.0  # what the other kind's score is
    box = np.zeros((pages, 1, 2, D), np.float32)
    box[::2, 0, 1, 1] = 1.0
    box[1::2, 0, 1, 0] = 1.0
    return q, box, np.arange(pages, dtype=np.int32)[None]


# One, half a step of fp32 beside it, and values that fp64 keeps beside that if they are added up first: which of the two kinds of
# page comes first hangs on the order of the sum.
TINY = [(0, 1.0), (1, 2.0 ** -24)]


@pytest.mark.parametrize("rows,T", [
    (TINY + [(2, 1.5 * 2.0 ** -54), (3, 1.5 * 2.0 ** -54)], 4),       # few query rows: one after the other
    (TINY + [(i, 2.0 ** -54) for i in (32, 96, 160, 224)], 256), (TINY + [(i, 2.0 ** -54) for i in (16, 48, 80, 112)], 128),
    (TINY + [(i, 2.0 ** -54) for i in (32, 64, 96, 128)], 129),
    (TINY + [(i, 2.0 ** -54) for i in (64, 192, 320, 448)], 512), (TINY + [(i, 2.0 ** -54) for i in (2, 3, 6, 7)], 9),
    (TINY + [(i, 2.0 ** -54) for i in (32, 96, 160, 224)], 700), (TINY + [(i, 2.0 ** -54) for i in (64, 192, 320, 448)], 700),
])
@pytest.mark.parametrize("D", [64, 128, 256, 80])
@pytest.mark.parametrize("blocks", [1, 2])
def test_choice_does_not_hang_on_the_batch(ff, gpu, rows, T, D, blocks):
    """fp32 queries: a row's lists alone, with its block of queries once and twice, and beside 300 others."""
    rng = np.random.default_rng(1)
    q, box, table = beside(rng, D, gpu, rows, T)
    got = []
    for B in (1, 300):
        for wide in (0, 3000):
            for n in (1, blocks):
                tab = np.full((B, max(60, wide)), -1, np.int32)
                tab[:, :60] = table
                li = ff.select_blocks(up(np.tile(q, (B, n, 1, 1)), gpu), up(box, gpu), up(tab, gpu),
                                      up(np.full(B, 60 * 16 - T * n, np.int32), gpu), 20, sinks=0, recent=0, query_block=T)
                got.append(li[0, -1, 0].cpu().numpy())  # (the last block sees all pages)
                assert (li == li[:1]).all()
    assert all(np.array_equal(g, got[0]) for g in got[1:]), got
