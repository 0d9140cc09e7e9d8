"""Eviction from the cache by attention weight: which tokens stay, and where they, their scales and weights go."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "i8": torch.int8, "fp8": torch.uint8}


def choose(w, n, keep, sinks, recent):
    """The kept positions of one head's n weights, in plain Python order."""
    if n <= keep:
        return list(range(n))
    mid = range(sinks, n - recent)
    key = lambda i: (-math.inf if math.isnan(w[i]) else 0.0, w[i]) if not math.isnan(w[i]) else (-math.inf, 0.0)  # noqa: E731
    best = sorted(mid, key=lambda i: (key(i)[0] == -math.inf, -key(i)[1], i))[:keep - sinks - recent]
    return list(range(sinks)) + sorted(best) + list(range(n - recent, n))


class Cache:
    def __init__(self, seed, lens, keep, hkv, d, kv, dev, width=None, stride=None, kind="random"):
        g = np.random.default_rng(seed)
        self.lens, self.hkv, self.kv, B = lens, hkv, kv, len(lens)
        need = [(max(n, 0) + 15) // 16 for n in lens]
        room = (keep + 15) // 16
        self.pages = sum(need) + B * room + 3
        perm = g.permutation(self.pages).astype(np.int32)
        width = width or max(need + [1])
        table, at = np.full((B, width), -1, np.int32), 0
        for b, m in enumerate(need):
            m = min(m, width)
            table[b, :m] = perm[at:at + m]
            at += m
        self.dst_h = perm[at:at + B * room].reshape(B, room).copy()
        self.table_h = table
        T = stride or max(max(lens), 1)
        w = g.standard_normal((B, hkv, T)).astype(np.float32)
        if kind == "ties":
            w = np.round(w * 2) / 2
        elif kind == "zeros":
            w = np.where(g.random(w.shape) < 0.9, np.where(g.random(w.shape) < 0.5, -0.0, 0.0), np.exp(w)).astype(np.float32)
        elif kind == "equal":
            w[:] = 0.25
        elif kind == "special":
            w = np.where(g.random(w.shape) < 0.3, np.nan, w)
            w = np.where(g.random(w.shape) < 0.2, np.inf, w)
            w = np.where(g.random(w.shape) < 0.2, -np.inf, w)
            w = np.where(g.random(w.shape) < 0.2, np.float32(1e-42), w).astype(np.float32)
        elif kind == "positive":
            w = np.exp(4 * w)
        self.w_h = w
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
        self.w, self.table, self.dst = up(w), up(table), up(self.dst_h)
        self.ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
        es = {"f32": 4, "bf16": 2, "f16": 2}.get(kv, 1)
        raw = lambda: up(g.integers(0, 256, (self.pages, 16, hkv, d * es), dtype=np.uint8)).view(TYPES[kv])  # noqa: E731
        self.k, self.v = raw(), raw()
        sc = lambda: up(g.random((self.pages, 16, hkv), dtype=np.float32)) if kv == "i8" else None  # noqa: E731
        self.ks, self.vs = sc(), sc()

    def pools(self):
        return [p for p in (self.k, self.v, self.ks, self.vs) if p is not None]

    def bytes(self):
        return [p.view(torch.uint8).cpu().numpy().reshape(self.pages * 16, self.hkv, -1) for p in self.pools()]


def run(ff, c, keep, sinks, recent, in_place, weights_out="apart", **kw):
    """One call, checked against the plain choice, token by token."""
    before = c.bytes()
    B, hkv, T = c.w.shape
    kept = torch.full((B, hkv, keep), -7, dtype=torch.int32, device=c.w.device)
    out = {"apart": torch.full((B, hkv, T + 3), 9.0, device=c.w.device), "in place": c.w, "none": None}[weights_out]
    got, lens = ff.evict_tokens(c.w, c.k, c.v, c.table, c.ctx, keep, sinks, recent, None if in_place else c.dst, out, kept,
                                k_scale=c.ks, v_scale=c.vs, **kw)
    assert got is kept
    kept, lens, after = kept.cpu().numpy(), lens.cpu().numpy(), c.bytes()
    want = [p.copy() for p in before]
    w_want = (c.w_h if weights_out == "in place" else np.full((B, hkv, T + 3), 9.0, np.float32)).copy()
    nb = kw.get("num_blocks", c.pages)
    for b in range(B):
        n = min(max(c.lens[b], 0), T, c.table_h.shape[1] * 16)
        assert lens[b] == min(n, keep)
        to = c.table_h if in_place else c.dst_h
        slot = lambda t, j: -1 if j // 16 >= t.shape[1] or not 0 <= t[b, j // 16] < nb else t[b, j // 16] * 16 + j % 16  # noqa: E731
        for h in range(hkv):
            idx = choose(c.w_h[b, h], n, keep, sinks, recent)
            assert kept[b, h, :len(idx)].tolist() == idx, (b, h)
            assert (kept[b, h, len(idx):] == -7).all()
            w_want[b, h, :len(idx)] = c.w_h[b, h, idx]
            for j, i in enumerate(idx):
                s, d = slot(c.table_h, i), slot(to, j)
                if s >= 0 and d >= 0:
                    for p, o in zip(want, before):
                        p[d, h] = o[s, h]
    for p, o in zip(after, want):
        assert np.array_equal(p, o)
    if out is not None:
        assert np.array_equal(out.cpu().numpy(), w_want, equal_nan=True)
    return kept, lens


@pytest.mark.parametrize("kind", ["random", "ties", "zeros", "equal", "special", "positive"])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (16, 4, 5), (100, 0, 0), (100, 100, 0), (100, 0, 100), (33, 1, 31),
                                               (500, 7, 100)])
@pytest.mark.parametrize("in_place", [False, True])
def test_choice(ff, gpu, kind, keep, sinks, recent, in_place):
    c = Cache(1, [0, 1, 15, 16, 99, 100, 101, 257, 1023, 1030, -3], keep, 2, 8, "bf16", gpu, kind=kind)
    run(ff, c, keep, sinks, recent, in_place, "in place" if in_place else "apart")


@pytest.mark.parametrize("kv", list(TYPES))
@pytest.mark.parametrize("d", [8, 40, 64, 80, 128, 256])
@pytest.mark.parametrize("in_place", [False, True])
def test_types(ff, gpu, kv, d, in_place):
    c = Cache(2, [300, 20, 77, 1200], 75, 3, d, kv, gpu)
    run(ff, c, 75, 2, 30, in_place, "none" if d == 64 else "apart")


@pytest.mark.parametrize("n", [32767, 32768, 32769, 70001, 131000])
@pytest.mark.parametrize("kind", ["positive", "zeros"])
@pytest.mark.parametrize("in_place", [False, True])
def test_long_rows(ff, gpu, n, kind, in_place):
    """One and several tiles of weights, many rounds of moves."""
    c = Cache(3, [n, 5000], 4099, 1, 16, "fp8", gpu, kind=kind)
    run(ff, c, 4099, 17, 1000, in_place, "in place" if kind == "zeros" else "apart")


@pytest.mark.parametrize("n,hkv", [(4000, 3), (8100, 2), (9000, 256)])
def test_wide_ends_in_place(ff, gpu, n, hkv):
    """Rows mostly of their first and last tokens, the weights in place, in every number of weights a thread holds."""
    c = Cache(10, [n], n - 100, hkv, 8, "fp8", gpu, kind="positive")
    run(ff, c, n - 100, n // 4, n // 2, True, "in place")


def test_bounds(ff, gpu):
    """Lengths beyond the table or the weights, a destination with too few pages, absent pages, fewer blocks than the
    pool has: nothing else is touched."""
    c = Cache(4, [500, 500, 90], 120, 2, 32, "bf16", gpu, width=20, stride=310)
    c.table_h[1, 3], c.table_h[1, 4] = -1, c.pages
    c.dst_h = c.dst_h[:, :5].copy()
    c.dst_h[2, 1] = -1
    c.table, c.dst = torch.from_numpy(c.table_h).to(gpu), torch.from_numpy(c.dst_h).to(gpu)
    run(ff, c, 120, 0, 10, False)
    c = Cache(5, [500, 300], 120, 2, 32, "i8", gpu)
    run(ff, c, 120, 3, 10, True, num_blocks=c.pages - 20)


def test_shared_pages_stay_whole(ff, gpu):
    """Rows over the same first pages, cut into pages of their own: each gets its tokens, the shared ones are not written."""
    c = Cache(6, [200, 220], 64, 2, 64, "bf16", gpu)
    c.table_h[1, :8] = c.table_h[0, :8]
    c.table = torch.from_numpy(c.table_h).to(gpu)
    shared = c.table_h[0, :8].astype(np.int64)
    before = c.k.view(torch.uint8).cpu().numpy()[shared]
    run(ff, c, 64, 4, 16, False)
    assert np.array_equal(before, c.k.view(torch.uint8).cpu().numpy()[shared])


def test_no_rows_and_streams(ff, gpu):
    e = torch.zeros(0, 2, 5, device=gpu)
    pool = torch.zeros(3, 16, 2, 64, device=gpu)
    i = torch.zeros(0, dtype=torch.int32, device=gpu)
    kept, lens = ff.evict_tokens(e, pool, pool.clone(), torch.zeros(0, 1, dtype=torch.int32, device=gpu), i, 4)
    assert kept.shape == (0, 2, 4) and lens.shape == (0,)
    c = Cache(7, [300, 600], 80, 2, 64, "bf16", gpu, kind="ties")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    a, al = ff.evict_tokens(c.w, c.k, c.v, c.table, c.ctx, 80, dst_table=c.dst, stream=s)
    s.synchronize()
    kept, lens = torch.zeros_like(a), torch.zeros_like(al)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ff.evict_tokens(c.w, c.k, c.v, c.table, c.ctx, 80, dst_table=c.dst, kept=kept, kept_lens=lens)
    for _ in range(3):
        kept.zero_()
        g.replay()
        b, bl = ff.evict_tokens(c.w, c.k, c.v, c.table, c.ctx, 80, dst_table=c.dst)
        torch.cuda.synchronize()
        assert torch.equal(a, kept) and torch.equal(al, lens) and torch.equal(a, b) and torch.equal(al, bl)


def test_long_rows_workspace_and_graph(ff, gpu):
    """Rows long enough for their choice to be split over workgroups: a workspace of the caller's, weights in place where
    more than the row is kept, and a captured call replayed between eager ones."""
    c = Cache(8, [20000, 300, 9000], 4000, 2, 64, "bf16", gpu, kind="ties")
    ws = ff.evict_workspace(3, 2, 4000, c.w.shape[2], c.table.shape[1], device=gpu)
    assert ff.lib.ffkv_evict_workspace_bytes(3, 2, 4000, c.w.shape[2], c.table.shape[1]) > 0
    a, al = run(ff, c, 4000, 5, 70, False, workspace=ws)
    kept, lens, out = (torch.zeros(3, 2, 4000, dtype=torch.int32, device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu),
                       torch.zeros(3, 2, 4000, device=gpu))
    args = (c.w, c.k, c.v, c.table, c.ctx, 4000, 5, 70, c.dst)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ff.evict_tokens(*args, weights_out=out, kept=kept, kept_lens=lens, workspace=ws)
    for _ in range(3):
        kept.fill_(-7)
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(kept.cpu().numpy(), a) and np.array_equal(lens.cpu().numpy(), al)
        b, _ = ff.evict_tokens(*args, kept=torch.full_like(kept, -7), workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(b, kept)
    c = Cache(9, [20000, 300, 9000], 30000, 2, 64, "bf16", gpu, kind="positive")
    run(ff, c, 30000, 5, 70, True, "in place")
