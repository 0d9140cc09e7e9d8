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
