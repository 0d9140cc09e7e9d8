"""The pages' key bounds, to the bit, and the choice of pages by them, against float64."""

import numpy as np
import pytest
import torch

import blocks_util as bu
import cases
import gpu_util as gu
import oracle as O

pytestmark = pytest.mark.gpu


def tensors(c, dev):
    up = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    return gu.to_dev(c.k_pool, c.kv, dev), up(c.k_scale), up(c.block_table), up(c.ctx)


@pytest.mark.parametrize("kv", ["bf16", "f16", "f32", "i8", "fp8"])
@pytest.mark.parametrize("Hkv,D,S,ctx", [
    (8, 128, 1, [0, 15, 16, 17, 300]), (1, 8, 1, [3]), (2, 64, 16, [0, 1, 15, 31]), (3, 80, 17, [0, 15, 100]),
    (4, 256, 50, [7, 64]), (5, 112, 1000, [13]), (2, 96, 3, [14, 29, 5]),
])
def test_bounds(ff, gpu, kv, Hkv, D, S, ctx):
    c = cases.make_case(Hkv * D + S, len(ctx), Hkv, Hkv, D, ctx, act="f32" if kv == "f32" else "bf16", kv=kv, S=S, max_blocks=70,
                        outlier_frac=0.01)
    c.block_table[0, int(c.ctx[0]) // 16] = -1  # on no page
    if len(ctx) > 1:
        c.block_table[1, int(c.ctx[1]) // 16] = c.num_blocks
    kp, ks, bt, cx = tensors(c, gpu)
    box = ff.key_bounds(kp)
    box.fill_(7.0)
    want = bu.bounds(c, box.float().cpu().numpy(), S)
    ff.update_key_bounds(kp, box, bt, cx, S, k_scale=ks)
    assert np.array_equal(box.float().cpu().numpy(), want)
    x = bu.keys32(c)
    for b in range(c.B):  # what they are for: no key of a page lies outside
        for p in range(int(c.ctx[b]) // 16, (int(c.ctx[b]) + S + 15) // 16):
            phys = c.block_table[b, p]
            if 0 <= phys < c.num_blocks:
                live = x[phys, :min(16, int(c.ctx[b]) + S - 16 * p)]
                assert (want[phys, :, 0] <= live).all() and (live <= want[phys, :, 1]).all()


def test_bounds_of_strange_keys(ff, gpu):
    """NaN and infinite keys; tokens past the row's end; rows before the cache, past the table, and of no tokens."""
    c = cases.make_case(5, 4, 2, 2, 64, [10, 0, 30, 16], S=4)
    c.ctx[1], c.ctx[2], c.ctx[3] = -2, 10 ** 9, -70
    p = c.block_table[0, 0]
    kf = cases.decode(c.k_pool, c.kv)
    kf[p, 3, 0, 5], kf[p, 11, 1, 7], kf[p, 12, 1, 8], kf[p, 14] = np.nan, np.inf, -np.inf, np.nan  # 14: past the row's end
    kf[p, 0, 1, 9] = -0.0
    c.k_pool = cases.encode(kf, c.kv)
    kp, _, bt, cx = tensors(c, gpu)
    box = ff.key_bounds(kp)
    box.fill_(7.0)
    want = bu.bounds(c, box.float().cpu().numpy(), 4)
    ff.update_key_bounds(kp, box, bt, cx, 4)
    got = box.float().cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True) and np.isnan(got[p, 0, :, 5]).all() and np.isnan(got).sum() == 2
    ff.update_key_bounds(kp, box, bt, cx, 0)
    assert np.array_equal(box.float().cpu().numpy(), want, equal_nan=True)


def choose(ff, c, q, box, dev, count, sinks, recent, T, **kw):
    _, _, bt, cx = tensors(c, dev)
    return ff.select_blocks(gu.to_dev(q, c.act, dev), box, bt, cx, count, sinks=sinks, recent=recent, query_block=T, **kw)


def boxes(rng, N, Hkv, D, dtype, dev):
    mean, half = rng.standard_normal((N, Hkv, D)) * 0.4, np.abs(rng.standard_normal((N, Hkv, D)) * 0.3 + 1.77)
    return torch.from_numpy(np.stack((mean - half, mean + half), axis=2).astype(np.float32)).to(dev).to(dtype)


@pytest.mark.parametrize("act,dtype", [("bf16", torch.bfloat16), ("f16", torch.float16), ("f32", torch.float32),
                                       ("bf16", torch.float32), ("f32", torch.bfloat16)])
@pytest.mark.parametrize("Hq,Hkv,D,S,ctx,count,sinks,recent,T", [
    (8, 2, 128, 1, [0, 15, 16, 900, 2000], 9, 1, 2, 1),       # rows of one page, of fewer than are taken, of more
    (4, 4, 64, 1, [5000], 40, 0, 0, 1),                       # no page for sure
    (7, 1, 256, 1, [3000, 160], 12, 5, 7, 1),                 # all for sure
    (6, 2, 80, 5, [700, 33], 3, 1, 1, 1),                     # every query by itself
    (8, 2, 96, 37, [800, 0, 100], 8, 2, 3, 16),               # blocks of queries, the last one short
    (2, 1, 8, 3, [40000], 100, 1, 1, 4),                      # 2500 pages, a block longer than the call
    (40, 2, 112, 2, [16000, 20000], 1, 0, 0, 1),              # one page
    (8, 8, 128, 64, [600], 20, 1, 5, 64), (24, 2, 128, 1, [2000, 1999], 30, 1, 2, 1), (18, 1, 64, 3, [9000, 40], 25, 3, 5, 2),
])
@pytest.mark.parametrize("wide", [False, True])  # behind a wide table the choice takes other kernels
def test_choice(ff, gpu, act, dtype, Hq, Hkv, D, S, ctx, count, sinks, recent, T, wide):
    c = cases.make_case(Hq + S, len(ctx), Hq, Hkv, 8, ctx, act=act, S=S, max_blocks=3001 if wide else None)
    rng = np.random.default_rng(D + S)
    q = cases.encode(rng.standard_normal((c.B, S, Hq, D), dtype=np.float32) * np.float32(2), c.act)
    box = boxes(rng, c.num_blocks, Hkv, D, dtype, gpu)
    got = choose(ff, c, q, box, gpu, count, sinks, recent, T).cpu().numpy()
    want = bu.select(cases.decode(q, c.act).astype(np.float64), box.double().cpu().numpy(), c.block_table, c.ctx, count, sinks,
                     recent, T, c.num_blocks)
    assert np.array_equal(got, want)


def test_long_rows(ff, gpu):
    """More pages than a workgroup holds (8192), beside a short row, and a bound that cuts."""
    c = cases.make_case(1, 2, 2, 1, 8, [150000, 100])
    rng = np.random.default_rng(4)
    q = cases.encode(rng.standard_normal((2, 1, 2, 64), dtype=np.float32), c.act)
    box = boxes(rng, c.num_blocks, 1, 64, torch.bfloat16, gpu)
    qv, bv = cases.decode(q, c.act).astype(np.float64), box.double().cpu().numpy()
    for most in (0, 140000, 16 * 8192):
        got = choose(ff, c, q, box, gpu, 300, 4, 9, 1, max_context_len=most).cpu().numpy()
        assert np.array_equal(got, bu.select(qv, bv, c.block_table, c.ctx, 300, 4, 9, 1, c.num_blocks, most))


@pytest.mark.parametrize("wide", [None, 2000])
def test_ties_and_strange_scores(ff, gpu, wide):
    """Equal scores go to the lower page, NaN before all, pages on no table entry last; zero queries tie everywhere."""
    c = cases.make_case(9, 3, 4, 2, 8, [1600, 1600, 1600], max_blocks=wide)
    rng = np.random.default_rng(6)
    q = cases.encode(np.abs(rng.standard_normal((3, 1, 4, 64), dtype=np.float32)) + np.float32(0.1), c.act)
    q[1] = 0
    few = boxes(rng, 4, 2, 64, torch.bfloat16, gpu)
    box = few[torch.arange(c.num_blocks, device=gpu) % 4].contiguous()  # four kinds of page
    box[c.block_table[0, 50], 0, 1, 3] = float("nan")
    box[c.block_table[0, 60], 1, 1, 3] = float("inf")
    box[c.block_table[0, 61], 1, 0, 3] = -float("inf")
    c.block_table[2, 10:90] = -1
    c.block_table[2, 20:60] = c.num_blocks
    got = choose(ff, c, q, box, gpu, 30, 1, 2, 1).cpu().numpy()
    want = bu.select(cases.decode(q, c.act).astype(np.float64), box.double().cpu().numpy(), c.block_table, c.ctx, 30, 1, 2, 1,
                     c.num_blocks)
    assert np.array_equal(got[1:], want[1:])
    assert 50 in got[0, 0, 0] and 60 in got[0, 0, 1] and np.array_equal(got[1, 0, 0], np.r_[0:28, 99, 100])
    # row 2 has 21 pages for its 30: the others are of those on no entry, the lowest first
    assert set(range(10)) | set(range(90, 101)) <= set(got[2, 0, 0])


def test_split_and_batch_do_not_matter(ff, gpu):
    """A row's choice is the same alone, in a batch, and behind a wide table."""
    ctx = [30000, 12000, 500, 31000]
    c = cases.make_case(2, 4, 8, 2, 8, ctx, max_blocks=4000)
    rng = np.random.default_rng(8)
    q = cases.encode(rng.standard_normal((4, 1, 8, 128), dtype=np.float32), c.act)
    box = boxes(rng, c.num_blocks, 2, 128, torch.bfloat16, gpu)
    every = choose(ff, c, q, box, gpu, 64, 1, 4, 1)
    qd, (_, _, bt, cx) = gu.to_dev(q, c.act, gpu), tensors(c, gpu)
    for b in range(4):
        one = ff.select_blocks(qd[b:b + 1], box, bt[b:b + 1, :2000].contiguous(), cx[b:b + 1], 64, sinks=1, recent=4)
        assert torch.equal(one, every[b:b + 1])


def test_capture(ff, gpu):
    c = cases.make_case(2, 4, 8, 2, 8, [30000, 12000, 500, 31000])
    rng = np.random.default_rng(8)
    box = boxes(rng, c.num_blocks, 2, 128, torch.bfloat16, gpu)
    q = torch.randn(4, 1, 8, 128, device=gpu).bfloat16()
    _, _, bt, cx = tensors(c, gpu)
    ws = ff.select_blocks_workspace(4, 1, 8, 2, 128, 64, 1, c.max_blocks)
    out = torch.empty(4, 1, 2, 64, dtype=torch.int32, device=gpu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ff.select_blocks(q, box, bt, cx, 64, blocks=out, workspace=ws)
        with pytest.raises(ff.FFKVError):
            ff.select_blocks(q, box, bt, cx, 64, blocks=out)
    for i in range(3):
        q.mul_(-1.5)
        cx.sub_(100)
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, ff.select_blocks(q, box, bt, cx, 64))
