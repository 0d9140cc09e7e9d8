"""Attention over listed pages, against float64."""

import numpy as np
import pytest
import torch

import blocks_util as bu
import cases
import oracle as O
import scored_util as su

pytestmark = pytest.mark.gpu


def make(seed, ctx, S, Hq, Hkv, D, act="bf16", kv=None, spread=2.0, **kw):
    c = cases.make_case(seed, len(ctx), Hq, Hkv, D, ctx, act=act, kv=kv, S=S, **kw)
    c.rng = np.random.default_rng(seed + 1)
    c.q = cases.encode(c.rng.standard_normal((c.B, S, Hq, D), dtype=np.float32) * np.float32(spread), c.act)
    return c


def lists(c, S, count, T, shuffle=False):
    """Lists of a row's pages: some of them, in order, -1 behind; shuffled: in any order, with pages that are none."""
    blocks = -(-S // T)
    out = np.full((c.B, blocks, c.Hkv, count), -1, np.int32)
    for b in range(c.B):
        for r in range(blocks):
            n = (int(c.ctx[b]) + min((r + 1) * T, S) - 1) // 16 + 1
            for h in range(c.Hkv):
                got = np.sort(c.rng.permutation(n)[:count])
                out[b, r, h, :len(got)] = got
                if shuffle:
                    bad = c.rng.random(count) < 0.2
                    out[b, r, h, bad] = c.rng.choice([-1, -7, c.max_blocks, c.max_blocks + 3, 2 ** 31 - 1, -2 ** 31], bad.sum())
                    out[b, r, h] = c.rng.permutation(out[b, r, h])
    return out


def run(ff, c, li, T, dev, workspace=None, **kw):
    kp, vp, ks, vs, bt, cx, _, _, q = su.device(c, dev)
    return ff.paged_attention_blocks(q, kp, vp, bt, cx, torch.from_numpy(li).to(dev), query_block=T, k_scale=ks, v_scale=vs,
                                     workspace=workspace, **kw)


def check(ff, c, li, T, dev, what="out"):
    S = c.q.shape[1]
    got = su.host(run(ff, c, li, T, dev)).reshape(c.B, S, c.Hq, c.D)
    q = cases.decode(c.q, c.act).astype(np.float64)
    want, bound = bu.attend(c, q, li, T, c.act, S, 2.0 ** -10 if T > 1 else 2.0 ** -11)
    su.check(got, want, bound, what)
    return got


KV = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "i8"), ("bf16", "fp8"), ("f32", "f32"), ("f16", "i8"), ("f32", "bf16"),
      ("f16", "fp8"), ("bf16", "f16")]


@pytest.mark.parametrize("act,kv", KV)
@pytest.mark.parametrize("Hq,Hkv,D,ctx,count", [
    (16, 8, 128, [17, 64, 100, 255], 4), (28, 4, 128, [3000], 150), (5, 1, 64, [0, 15, 16, 900], 7), (8, 8, 256, [500, 31], 20),
    (6, 2, 96, [1000, 3], 33), (3, 3, 80, [200, 400], 5), (4, 2, 112, [640], 41), (20, 1, 128, [800, 900], 30),
    (2, 2, 8, [100], 3), (36, 2, 64, [333], 9), (32, 2, 256, [700], 40), (14, 2, 80, [1900, 1400], 90), (3, 1, 112, [33, 0], 2),
    (21, 1, 112, [777], 25), (4, 4, 72, [100, 333], 11),
])
def test_step(ff, gpu, act, kv, Hq, Hkv, D, ctx, count):
    c = make(Hq + D, ctx, 1, Hq, Hkv, D, act, kv)
    check(ff, c, lists(c, 1, count, 1), 1, gpu)


@pytest.mark.parametrize("act,kv", KV)
@pytest.mark.parametrize("Hq,Hkv,D,ctx,S,count,T", [
    (8, 2, 128, [700, 0], 70, 12, 64), (4, 4, 64, [100], 33, 6, 16), (10, 2, 256, [300, 15], 40, 9, 40),
    (14, 2, 128, [64], 17, 3, 100), (8, 2, 128, [257], 5, 8, 2), (6, 2, 96, [90], 20, 5, 8), (32, 1, 64, [500], 9, 21, 9),
    (4, 1, 128, [40, 300], 6, 7, 1), (10, 2, 80, [300, 15], 40, 9, 16), (7, 1, 112, [64], 17, 3, 100), (6, 3, 104, [50], 9, 4, 3),
    # of more tokens
    (8, 2, 128, [1100, 0], 70, 60, 64), (4, 4, 64, [900], 133, 31, 16), (10, 2, 256, [700, 15], 140, 30, 40),
    (14, 2, 128, [64], 300, 3, 100), (8, 2, 128, [257], 270, 8, 2), (32, 1, 64, [500], 520, 21, 9),
])
def test_chunk(ff, gpu, act, kv, Hq, Hkv, D, ctx, S, count, T):
    c = make(Hq + S, ctx, S, Hq, Hkv, D, act, kv)
    check(ff, c, lists(c, S, count, T), T, gpu)


@pytest.mark.parametrize("act,kv", [("bf16", "bf16"), ("bf16", "i8"), ("bf16", "fp8"), ("f32", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("S,T", [(1, 1), (9, 1), (50, 16), (200, 16)])
def test_any_order(ff, gpu, act, kv, S, T):
    """Lists out of order, with entries that are no page, pages past the query, and pages on no table entry."""
    c = make(S + T, [700, 40, 0], S, 8, 2, 128, act, kv)
    c.block_table[0, 5], c.block_table[0, 9], c.block_table[1, 1] = -1, c.num_blocks, -3
    li = lists(c, S, 30, T, shuffle=True)
    li[:, :, :, 3] = np.maximum(li[:, :, :, 3], 40)  # past the shorter rows
    check(ff, c, li, T, gpu)


@pytest.mark.parametrize("S,T", [(1, 1), (20, 10), (100, 10)])
def test_nothing_and_twice(ff, gpu, S, T):
    """Lists without any page give zeros; a page listed twice counts twice."""
    c = make(4, [300, 200, 100], S, 4, 2, 128)
    li = lists(c, S, 6, T)
    li[0, :, 0], li[1] = -1, 99
    li[2, :, :, 4] = li[2, :, :, 1]
    got = check(ff, c, li, T, gpu)
    assert not got[0, :, :2].any() and not got[1].any() and got[2].any()


@pytest.mark.parametrize("act,kv", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "fp8"), ("bf16", "i8"), ("f32", "f32")])
@pytest.mark.parametrize("S,T", [(1, 1), (6, 1), (40, 16), (150, 16)])
def test_hidden_values_do_not_reach(ff, gpu, act, kv, S, T):
    """NaN and infinite values in the slots behind the row and, of a chunk, behind each query; in pages that are not listed."""
    c = make(31, [90, 205], S, 8, 2, 128, act, kv)
    li = lists(c, S, 8, T)
    for b in range(2):
        last = int(c.ctx[b]) + S - 1
        li[b, :, :, -1] = last // 16 if S == 1 else -1
        for r in range(li.shape[1]):  # the page of the block's first query, whose later slots it must not see
            li[b, r, :, -1] = (int(c.ctx[b]) + r * T) // 16
            for h in range(c.Hkv):
                li[b, r, h, :-1][li[b, r, h, :-1] == li[b, r, h, -1]] = -1
        for t in range(last + 1, 16 * ((last + 16) // 16)):
            su.poison(c, b, t)
    dense = bu.attend(c, cases.decode(c.q, c.act).astype(np.float64), li, T, c.act, S, 2.0 ** -10)
    if S > 1 and kv != "i8":  # a value that only the last queries see: the others are what they were
        seen = int(c.ctx[0]) + S - 2
        su.poison(c, 0, seen)
    got = su.host(run(ff, c, li, T, gpu)).reshape(c.B, S, c.Hq, c.D)
    upto = S - 2 if S > 1 and kv != "i8" else S
    su.check(got[:1, :upto], dense[0][:1, :upto], dense[1][:1, :upto], "row 0")
    su.check(got[1:], dense[0][1:], dense[1][1:], "row 1")
    assert np.isfinite(got[:1, :upto]).all() and np.isfinite(got[1:]).all()


@pytest.mark.parametrize("act,kv", [("bf16", "bf16"), ("bf16", "i8"), ("f32", "f32")])
def test_all_pages_are_the_dense_attention(ff, gpu, act, kv):
    c = make(12, [500, 33], 1, 8, 2, 128, act, kv)
    li = np.broadcast_to(np.arange(c.max_blocks, dtype=np.int32), (2, 1, 2, c.max_blocks)).copy()
    got = check(ff, c, li, 1, gpu)
    kp, vp, ks, vs, bt, cx, _, _, q = su.device(c, gpu)
    dense = su.host(ff.paged_attention(q, kp, vp, bt, cx, k_scale=ks, v_scale=vs)).reshape(got.shape)
    _, bound = bu.attend(c, cases.decode(c.q, c.act).astype(np.float64), li, 1, c.act, 1, 2.0 ** -11)
    su.check(got, dense, 2 * bound, "dense")  # each is off by the bound


@pytest.mark.parametrize("scale", [0.0, 0.5])
def test_scale_workspace_stream(ff, gpu, scale):
    """A split call with its workspace, without one, and on another stream gives the same bits."""
    c = make(21, [4000], 1, 8, 2, 128)
    li = lists(c, 1, 200, 1)
    n = ff.lib.ffkv_paged_attention_blocks_workspace_bytes(c.act, c.kv, 1, 1, 8, 2, 128, 200, 1)
    assert n > 0
    ws = ff.attention_blocks_workspace(c.act, c.kv, 1, 1, 8, 2, 128, 200)
    a = run(ff, c, li, 1, gpu, workspace=ws, scale=scale)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    b = run(ff, c, li, 1, gpu, scale=scale, stream=side)
    side.synchronize()
    assert torch.equal(a, b)
    c.q = cases.encode(cases.decode(c.q, c.act) * np.float32(scale * 128 ** 0.5 if scale else 1), c.act)
    if scale == 0.0:
        check(ff, c, li, 1, gpu)


@pytest.mark.parametrize("S,T", [(1, 1), (24, 8)])
def test_capture(ff, gpu, S, T):
    """Captured with and without a workspace, replayed over new queries, lists and lengths."""
    c = make(6, [4000, 900], S, 8, 2, 128)
    kp, vp, ks, vs, bt, cx, _, _, q = su.device(c, gpu)
    li = torch.from_numpy(lists(c, S, 200, T)).to(gpu)
    ws = ff.attention_blocks_workspace(c.act, c.kv, 2, S, 8, 2, 128, 200, T)
    out, whole = torch.empty(2, S, 8 * 128, dtype=q.dtype, device=gpu), torch.empty(2, S, 8 * 128, dtype=q.dtype, device=gpu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ff.paged_attention_blocks(q, kp, vp, bt, cx, li, query_block=T, out=out, workspace=ws)
        ff.paged_attention_blocks(q, kp, vp, bt, cx, li, query_block=T, out=whole)
    for i in range(3):
        q.mul_(-0.7)
        li.copy_(li.roll(1, dims=-1))
        cx.sub_(30)
        graph.replay()
        got, got_whole = out.clone(), whole.clone()
        torch.cuda.synchronize()
        eager = ff.paged_attention_blocks(q, kp, vp, bt, cx, li, query_block=T, workspace=ws)
        assert torch.equal(got, eager)
        # an unsplit softmax is the same up to its sums' roundings and the output's
        assert (got.float() - got_whole.float()).abs().max().item() <= 2.0 ** -7 * got.float().abs().max().item()


@pytest.mark.parametrize("act,kv", KV)
@pytest.mark.parametrize("Hq,Hkv,D,ctx,S,count,T", [
    (8, 2, 128, [2500, 40, 1200], 13, 130, 32), (5, 1, 64, [3000], 40, 170, 7), (20, 4, 256, [1531, 1908], 13, 100, 13),
    (8, 2, 128, [2500, 40, 1200], 40, 150, 32), (5, 1, 64, [3000], 107, 170, 7), (20, 4, 256, [1531, 1908], 31, 100, 13),
])
def test_split_chunk(ff, gpu, act, kv, Hq, Hkv, D, ctx, S, count, T):
    """Few blocks of queries over long lists, split over the lists; the same whole, in a capture without a workspace."""
    c = make(Hq + D, ctx, S, Hq, Hkv, D, act, kv)
    n = ff.lib.ffkv_paged_attention_blocks_workspace_bytes(c.act, c.kv, c.B, S, Hq, Hkv, D, count, T)
    assert n > 0 or kv == "f32"
    li = lists(c, S, count, T, shuffle=True)
    check(ff, c, li, T, gpu)
    kp, vp, ks, vs, bt, cx, _, _, q = su.device(c, gpu)
    ld, out = torch.from_numpy(li).to(gpu), torch.empty(c.B, S, Hq * D, dtype=q.dtype, device=gpu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ff.paged_attention_blocks(q, kp, vp, bt, cx, ld, query_block=T, out=out, k_scale=ks, v_scale=vs)
    graph.replay()
    want, bound = bu.attend(c, cases.decode(c.q, c.act).astype(np.float64), li, T, c.act, S, 2.0 ** -10)
    su.check(su.host(out).reshape(want.shape), want, bound, "whole")


@pytest.mark.parametrize("act,kv", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "fp8"), ("bf16", "i8")])
@pytest.mark.parametrize("S", [12, 160])
def test_split_hidden_values(ff, gpu, act, kv, S):
    """As test_hidden_values_do_not_reach, with the strange values in one piece of a split list."""
    c = make(77, [2000], S, 8, 2, 128, act, kv)
    li = lists(c, S, 120, S)
    li[0, 0, :, 60] = 2000 // 16
    for h in range(2):
        li[0, 0, h, 61:][li[0, 0, h, 61:] == 2000 // 16] = -1
        li[0, 0, h, :60][li[0, 0, h, :60] == 2000 // 16] = -1
    q = cases.decode(c.q, c.act).astype(np.float64)
    want, bound = bu.attend(c, q, li, S, c.act, S, 2.0 ** -10)
    for t in range(2008, 2016):  # seen by the queries from the eighth on, or by none
        su.poison(c, 0, t)
    got = su.host(run(ff, c, li, S, gpu)).reshape(want.shape)
    su.check(got[:, :8], want[:, :8], bound[:, :8], "before")
    assert not np.isfinite(got[:, 8:]).any()


@pytest.mark.parametrize("act,kv", KV)
@pytest.mark.parametrize("Hq,Hkv,D,ctx,S,count,T", [
    (36, 9, 128, [1100, 1300], 120, 61, 16), (24, 12, 64, [1700, 900], 130, 107, 16), (50, 10, 128, [1600, 1], 70, 97, 7),
    (8, 2, 128, [300, 0, 90], 60, 16, 30), (4, 4, 64, [700], 17, 31, 4), (8, 2, 128, [300, 0, 90], 100, 16, 30),
    (4, 4, 64, [700], 140, 31, 4),
])
def test_lists_in_halves(ff, gpu, act, kv, Hq, Hkv, D, ctx, S, count, T):
    """At most as many blocks of queries as half fills the chip, or short lists: a list's halves by those of a workgroup."""
    c = make(Hq + D, ctx, S, Hq, Hkv, D, act, kv)
    check(ff, c, lists(c, S, count, T, shuffle=True), T, gpu)


@pytest.mark.parametrize("act,kv", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "fp8"), ("bf16", "i8")])
@pytest.mark.parametrize("place", [3, 90])
def test_halves_hidden_values(ff, gpu, act, kv, place):
    """As test_split_hidden_values, the strange values in one half of the first list."""
    c = make(79, [2000, 1700], 100, 40, 10, 128, act, kv)
    li = lists(c, 100, 100, 10)
    li[0, 0][li[0, 0] == 125] = -1
    li[0, 0, :, place] = 125
    li[0, 1:][li[0, 1:] == 125] = -1
    q = cases.decode(c.q, c.act).astype(np.float64)
    want, bound = bu.attend(c, q, li, 10, c.act, 100, 2.0 ** -10)
    for t in range(2008, 2016):  # seen by the first list's queries from the eighth on
        su.poison(c, 0, t)
    got = su.host(run(ff, c, li, 10, gpu)).reshape(want.shape)
    seen = np.zeros((2, 100), bool)
    seen[0, 8:10] = True
    su.check(got[~seen], want[~seen], bound[~seen], "others")
    assert not np.isfinite(got[seen]).any()


@pytest.mark.parametrize("S,T,ctx,count", [(100, 10, [2000, 1700], 100), (12, 12, [2000], 120), (24, 24, [2000], 120),
                                              (20, 20, [200], 12), (60, 60, [200], 12)])
def test_int8_large_values(ff, gpu, S, T, ctx, count):
    """int8 V scales past 256 take the products again in a smaller scale, whichever part of the list they lie in."""
    c = make(80, ctx, S, 40, 10, 128, "bf16", "i8")
    c.v_scale[int(c.block_table[0, 2])] *= np.float32(20000)
    li = lists(c, S, count, T)
    li[0, :, :, 0] = 2
    li[0, :, :, 1:][li[0, :, :, 1:] == 2] = -1
    got = check(ff, c, li, T, gpu)
    assert np.isfinite(got).all() and np.abs(got[0]).max() > 1e3
