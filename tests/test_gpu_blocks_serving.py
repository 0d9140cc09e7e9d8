"""Rotary positions on several axes, key bounds, the choice of pages and the attention over them as a server uses them: prompts
with images in chunks, then steps, in one cache; and the four calls of a step in one graph."""

import numpy as np
import pytest
import torch

import blocks_util as bu
import cases
import gpu_util as gu
import oracle as O
import scored_util as su
from test_gpu_attention_blocks import make

pytestmark = pytest.mark.gpu

SECTIONS, THETA = (16, 8, 8), 1e6


def prompt_positions(rng, n):
    """Positions [3, n] of text with images in it: an image's tokens share their time and lie on a grid."""
    out, at = [], 0
    while len(out) < n:
        run = int(rng.integers(3, 30))
        out += [(at + i,) * 3 for i in range(run)]
        at += run
        h, w = int(rng.integers(2, 9)), int(rng.integers(2, 9))
        out += [(at, at + y, at + x) for y in range(h) for x in range(w)]
        at += max(h, w)
    return np.array(out[:n], np.int32).T, at


class Server:
    """Rows of one cache with their bounds, and beside them what the rows hold, in float64."""

    def __init__(self, ff, gpu, kv, room):
        self.ff, self.gpu, self.kv = ff, gpu, kv
        B = len(room)
        self.c = cases.make_case(3, B, 8, 2, 64, [16 * n - 1 for n in room], act="bf16", kv=kv, pool_extra=0.3)
        c = self.c
        self.k, self.v, self.ks, self.vs, self.table, _, _, _, _ = su.device(c, gpu)
        self.k.zero_(), self.v.zero_()
        self.box = ff.key_bounds(self.k).zero_()
        self.lens = [0] * B

    def call(self, q, k, v, pos, S, count, sinks, recent, T, rows):
        """One layer of the given rows' next S tokens, the lists checked and the outputs against float64."""
        ff, c = self.ff, self.c
        c.ctx = np.array([self.lens[b] for b in rows], np.int32)
        ctx = torch.from_numpy(c.ctx).to(self.gpu)
        table = self.table[rows].contiguous()
        at = torch.from_numpy(np.ascontiguousarray(pos)).to(self.gpu)
        qr = ff.rope_append_axes(q, k, v, at, SECTIONS, self.k, self.v, table, ctx, theta=THETA, k_scale=self.ks, v_scale=self.vs,
                                 q_out=torch.empty_like(q))
        ff.update_key_bounds(self.k, self.box, table, ctx, S, k_scale=self.ks)
        li = ff.select_blocks(qr, self.box, table, ctx, count, sinks=sinks, recent=recent, query_block=T)
        out = ff.paged_attention_blocks(qr, self.k, self.v, table, ctx, li, query_block=T, k_scale=self.ks, v_scale=self.vs)

        full, fulltable = c.block_table, self.table.cpu().numpy()
        c.block_table, c.B = fulltable[rows], len(rows)
        c.k_pool = gu.to_host(self.k, c.k_pool.dtype).reshape(c.k_pool.shape)
        c.v_pool = gu.to_host(self.v, c.v_pool.dtype).reshape(c.v_pool.shape)
        if self.ks is not None:
            c.k_scale, c.v_scale = self.ks.cpu().numpy(), self.vs.cpu().numpy()
        x, e = bu.rotate(q.double().cpu().numpy(), pos, SECTIONS, False, THETA, O.DTYPE_BF16)
        su.check(qr.double().cpu().numpy(), x, e, "rotated q")
        qv = qr.double().cpu().numpy()
        want = bu.select(qv, self.box.double().cpu().numpy(), c.block_table, c.ctx, count, sinks, recent, T, c.num_blocks)
        assert np.array_equal(li.cpu().numpy(), want)
        o, e = bu.attend(c, qv, want, T, O.DTYPE_BF16, S, 2.0 ** -10)
        su.check(su.host(out).reshape(o.shape), o, e, "attention")
        # the bounds are those of the rows' tokens, whichever calls brought them
        lo = self.box.float().cpu().numpy()
        before = c.ctx.copy()
        c.ctx = np.zeros_like(before)
        for i, b in enumerate(rows):
            n = int(before[i]) + S
            one = cases.Case(**{**c.__dict__, "B": 1, "ctx": np.zeros(1, np.int32), "block_table": fulltable[[b]]})
            assert np.array_equal(bu.bounds(one, lo, n), lo)
        c.block_table = full
        for b in rows:
            self.lens[b] += S
        return out


@pytest.mark.parametrize("kv", ["bf16", "i8", "fp8"])
def test_prompts_and_steps(ff, gpu, kv):
    rng = np.random.default_rng(17)
    prompts = [330, 70, 501]
    s = Server(ff, gpu, kv, [(n + 40 + 15) // 16 for n in prompts])
    rnd = lambda *d: torch.from_numpy(rng.standard_normal(d, dtype=np.float32)).to(gpu).bfloat16()  # noqa: E731
    nexts = []
    for b, n in enumerate(prompts):  # each prompt by itself, in chunks
        pos, after = prompt_positions(rng, n)
        nexts.append(after)
        for at in range(0, n, 300):
            S = min(300, n - at)
            packed = rnd(1, S, 12, 64)
            s.call(packed[:, :, :8], packed[:, :, 8:10], packed[:, :, 10:], pos[:, None, at:at + S], S, 10, 1, 5, 32, [b])
    for step in range(20):  # all rows together
        packed = rnd(3, 1, 12, 64)
        pos = np.array([[x + step] for x in nexts], np.int32)[None].repeat(3, axis=0)
        s.call(packed[:, :, :8], packed[:, :, 8:10], packed[:, :, 10:], pos, 1, 9, 1, 2, 1, [0, 1, 2])
    assert s.lens == [n + 20 for n in prompts]


def test_captured_step(ff, gpu):
    """The four calls of a step in one graph, one workspace for all, replayed as the rows grow, with eager calls on the same
    workspace in between."""
    B, Hq, Hkv, D, count = 4, 8, 2, 128, 24
    c = cases.make_case(11, B, Hq, Hkv, D, [9000, 700, 40, 15000], act="bf16")
    kp, vp, _, _, bt, cx, kn, vn, q = su.device(c, gpu)
    box = ff.key_bounds(kp).zero_()
    ff.update_key_bounds(kp, box, bt, torch.zeros_like(cx), 15000)
    pos = torch.randint(0, 20000, (3, B, 1), dtype=torch.int32, device=gpu)
    ws = max((ff.select_blocks_workspace(B, 1, Hq, Hkv, D, count, 1, c.max_blocks, device=gpu),
              ff.attention_blocks_workspace(c.act, c.kv, B, 1, Hq, Hkv, D, count, device=gpu)), key=lambda t: t.numel())
    cx.sub_(8)

    def calls(qo, kp, vp, box, li, out):
        ff.rope_append_axes(q, kn, vn, pos, (24, 20, 20), kp, vp, bt, cx, interleaved=True, q_out=qo)
        ff.update_key_bounds(kp, box, bt, cx, 1)
        ff.select_blocks(qo, box, bt, cx, count, sinks=1, recent=2, blocks=li, workspace=ws)
        ff.paged_attention_blocks(qo, kp, vp, bt, cx, li, out=out, workspace=ws)

    def buffers():
        return (torch.zeros_like(q), kp.clone(), vp.clone(), box.clone(),
                torch.zeros(B, 1, Hkv, count, dtype=torch.int32, device=gpu), torch.zeros(B, 1, Hq * D, dtype=q.dtype, device=gpu))

    eager, got = buffers(), buffers()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(*got)
    for i in range(5):
        q.mul_(-1.1)
        kn.mul_(1.2)
        pos.add_(1)
        graph.replay()
        calls(*eager)
        torch.cuda.synchronize()
        for a, b in zip(eager, got):
            assert torch.equal(a, b)
        cx.add_(1)


@pytest.mark.parametrize("kv", ["bf16", "i8", "f32"])
@pytest.mark.parametrize("S,T,count", [(1, 1, 8), (9, 4, 8), (200, 16, 8), (200, 40, 30), (40, 40, 150)])
@pytest.mark.parametrize("width", [None, 2600])
def test_rows_that_are_not_there(ff, gpu, kv, S, T, count, width):
    """Rows padded with negative lengths, wholly or for their first tokens, beside one that is there."""
    ctx = [500, -S, -1000, -(S // 2)]
    c = make(S + count, [500, S, S, S], S, 8, 2, 64, "f32" if kv == "f32" else "bf16", kv, max_blocks=width)
    k, v, ks, vs, table, _, kn, vn, q = su.device(c, gpu)
    cx = torch.tensor(ctx, dtype=torch.int32, device=gpu)
    pos = torch.zeros(2, 4, S, dtype=torch.int32, device=gpu)
    before = k.clone()
    ff.rope_append_axes(q, kn, vn, pos, (16, 16), k, v, table, cx, k_scale=ks, v_scale=vs)
    box = ff.key_bounds(k).fill_(7)
    ff.update_key_bounds(k, box, table, cx, S, k_scale=ks)
    li = ff.select_blocks(q, box, table, cx, count, sinks=1, recent=(T + 14) // 16 + 1, query_block=T)
    out = ff.paged_attention_blocks(q, k, v, table, cx, li, query_block=T, k_scale=ks, v_scale=vs)
    for b in (1, 2):  # not there: no page written, none listed, nothing attended
        own = torch.from_numpy(c.block_table[b][c.block_table[b] >= 0]).long().to(gpu)
        assert torch.equal(k[own], before[own]) and (box[own] == 7).all()
        assert (li[b] == -1).all() and not out[b].any()
    there = S - S // 2  # tokens of row 3 from its position 0 on
    first = S // 2
    assert not out[3, :first].any() and (there == 0 or out[3, first:].any(dim=-1).all())
    # both rows that are there, as without the others
    c.ctx = np.array(ctx, np.int32)
    c.k_pool, c.v_pool = gu.to_host(k, c.k_pool.dtype).reshape(c.k_pool.shape), gu.to_host(v, c.v_pool.dtype).reshape(c.v_pool.shape)
    if ks is not None:
        c.k_scale, c.v_scale = ks.cpu().numpy(), vs.cpu().numpy()
    qv, lists = q.double().cpu().numpy(), li.cpu().numpy()
    want = bu.select(qv, box.double().cpu().numpy(), c.block_table, c.ctx, count, 1, (T + 14) // 16 + 1, T, c.num_blocks)
    assert np.array_equal(lists, want)
    o, e = bu.attend(c, qv, lists, T, c.act, S, 2.0 ** -10)
    su.check(su.host(out).reshape(o.shape), o, e, "attention")


def test_pages_past_32_bits(ff, gpu):
    """Pages whose bytes and elements lie past 2^32 and 2^31 of their pool: the bits of the same rows in a small pool."""
    N, Hkv, D, B, S = 140_000, 8, 128, 2, 70
    rng = np.random.default_rng(5)
    small = 160
    kp = torch.randn(small, 16, Hkv, D, device=gpu).bfloat16()
    vp = torch.randn(small, 16, Hkv, D, device=gpu).bfloat16()
    table = torch.from_numpy(rng.permutation(small).astype(np.int32).reshape(B, 80)).to(gpu)
    far = table + (N - small)
    K, V = torch.empty(N, 16, Hkv, D, dtype=kp.dtype, device=gpu), torch.empty(N, 16, Hkv, D, dtype=kp.dtype, device=gpu)
    K[N - small:], V[N - small:] = kp, vp
    box, Box = ff.key_bounds(kp), ff.key_bounds(K)
    packed = torch.randn(B, S, 32 + 2 * Hkv, D, device=gpu).bfloat16()
    q, k, v = packed[:, :, :32], packed[:, :, 32:32 + Hkv], packed[:, :, 32 + Hkv:]
    pos = torch.randint(0, 1000, (3, B, S), dtype=torch.int32, device=gpu)
    cx = torch.tensor([1200, 777], dtype=torch.int32, device=gpu)
    got = []
    for pk, pv, pb, bt in ((kp, vp, box, table), (K, V, Box, far)):
        qr = ff.rope_append_axes(q, k, v, pos, (16, 24, 24), pk, pv, bt, cx, q_out=torch.empty(B, S, 32, D, dtype=q.dtype, device=gpu))
        ff.update_key_bounds(pk, pb, bt, torch.zeros_like(cx), 1270)
        res = [qr]
        for T, count in ((1, 20), (16, 20), (70, 60)):
            li = ff.select_blocks(qr, pb, bt, cx, count, sinks=1, recent=7, query_block=T)
            res += [li, ff.paged_attention_blocks(qr, pk, pv, bt, cx, li, query_block=T)]
        one = qr[:, :1].contiguous()
        li = ff.select_blocks(one, pb, bt, cx, 20)
        got.append(res + [li, ff.paged_attention_blocks(one, pk, pv, bt, cx, li)])
    assert torch.equal(K[N - small:], kp) and torch.equal(V[N - small:], vp)
    assert torch.equal(Box[far.long().flatten()], box[table.long().flatten()])
    for a, b in zip(*got):
        assert torch.equal(a, b)
