"""The scored operators together, as a server that evicts uses them: prompts appended and prefilled under the model's score
rule, the weights of their last tokens, the cut into new pages, decode steps that accumulate weights on what was kept, a cut in
place, and decode steps again.  Every output and weight is held to float64 on the tokens that each head then holds."""

import numpy as np
import pytest
import torch

import cases
import oracle as O
import scored_util as su
from test_gpu_evict import choose

pytestmark = pytest.mark.gpu
ACT = torch.bfloat16


class Server:
    """A batch's cache on the GPU and, in float64, the keys and values that every head of every row holds."""

    def __init__(self, kv, lens, Hq, Hkv, D, rule, dev, seed=0):
        self.g = np.random.default_rng(seed)
        self.kv, self.B, self.Hq, self.Hkv, self.D, self.rule, self.dev = kv, len(lens), Hq, Hkv, D, rule, dev
        self.width = 24
        self.N = 3 * self.B * self.width
        self.free = list(self.g.permutation(self.N))
        t = {"bf16": torch.bfloat16, "i8": torch.int8, "f32": torch.float32}[kv]
        self.k = torch.zeros(self.N, 16, Hkv, D, dtype=t, device=dev)
        self.v = torch.zeros_like(self.k)
        sc = lambda: torch.zeros(self.N, 16, Hkv, device=dev) if kv == "i8" else None  # noqa: E731
        self.ks, self.vs = sc(), sc()
        self.act = torch.float32 if kv == "f32" else ACT
        self.code = O.DTYPE_F32 if kv == "f32" else O.DTYPE_BF16
        self.table = self.pages([(n + 40 + 15) // 16 for n in lens])
        self.lens = [0] * self.B
        self.slopes = (2.0 ** (-np.arange(1, Hq + 1) / 2)).astype(np.float32)

    def pages(self, need):
        t = np.full((self.B, self.width), -1, np.int32)
        for b, n in enumerate(need):
            t[b, :n] = [self.free.pop() for _ in range(n)]
        return t

    def up(self, a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(self.dev)

    def ctx(self):
        return self.up(np.array(self.lens, np.int32))

    def randn(self, *shape, times=1.0):
        return (torch.from_numpy(self.g.standard_normal(shape, dtype=np.float32)) * times).to(self.dev).to(self.act)

    def held(self, b, n):
        """The first n cached keys and values of row b, [n, Hkv, D], from the pages as they are."""
        pages = self.up(self.table[b, :(n + 15) // 16].astype(np.int64))
        got = []
        for pool, scale in ((self.k, self.ks), (self.v, self.vs)):
            x = pool[pages].cpu().double()
            if scale is not None:
                x = x * scale[pages].cpu().double()[..., None]
            got.append(x.reshape(-1, self.Hkv, self.D)[:n].numpy())
        return got

    def rules(self):
        return {"score_cap": self.rule["cap"], "slopes": self.up(self.slopes), "window": self.rule["window"]}

    def expect(self, q, b, pos, n, v=True, **kw):
        k, val = self.held(b, n)
        return su.attention(su.host(q)[b], k, val if v else None, pos, self.rule["cap"], self.slopes, self.rule["window"],
                            act=self.code if v else None,
                            kv={"bf16": O.DTYPE_BF16, "i8": O.DTYPE_I8, "f32": O.DTYPE_F32}[self.kv], p_step=2.0 ** -10, **kw)


@pytest.mark.parametrize("kv", ["bf16", "i8", "f32"])
@pytest.mark.parametrize("rule", [{"cap": 6.0, "window": 0}, {"cap": 0.0, "window": 90}])
def test_prompt_cut_decode_cut_decode(ff, gpu, kv, rule):
    prompt, keep, sinks, recent = [150, 61, 200], 64, 4, 20
    s = Server(kv, prompt, 8, 2, 64, rule, gpu)
    S, T = max(prompt), 16 * s.width
    scales = {"k_scale": s.ks, "v_scale": s.vs}

    # a padded batch of prompts: rows end before the chunk does, their padding sees nothing and is forgotten
    q, kn, vn = s.randn(s.B, S, 8, 64, times=2.0), s.randn(s.B, S, 2, 64), s.randn(s.B, S, 2, 64)
    end = np.array([[t + 1 if t < n else 0 for t in range(S)] for n in prompt], np.int32)
    ff.append_kv_cache(kn, vn, s.k, s.v, s.up(s.table), s.ctx(), s.ks, s.vs)
    if kv != "f32":  # prefill takes 16- and 8-bit caches
        out = su.host(ff.paged_prefill_scored(q, s.k, s.v, s.up(s.table), s.ctx(), key_end=s.up(end), **s.rules(), **scales))
        for b, n in enumerate(prompt):
            o, e, _, _ = s.expect(q, b, 0, n, end=end[b].astype(np.int64))
            su.check(out.reshape(s.B, S, 8, 64)[b], o, e, f"prefill, row {b}")

    # what the prompts' last 16 tokens look at
    last = 16
    ql = torch.stack([q[b, n - last:n] for b, n in enumerate(prompt)])
    s.lens = [n - last for n in prompt]
    w = ff.attention_weights(ql, s.k, s.up(s.table), s.ctx(), k_scale=s.ks, max_context_len=T, **s.rules())
    for b, n in enumerate(prompt):
        _, _, x, e = s.expect(ql, b, n - last, n, v=False)
        su.check(su.host(w)[b, :, :n], x, e, f"weights, row {b}")
    s.lens = list(prompt)

    def cut(w, dst):
        before = [s.held(b, s.lens[b]) for b in range(s.B)]
        wh = su.host(w)
        kept, lens = ff.evict_tokens(w, s.k, s.v, s.up(s.table), s.ctx(), keep, sinks, recent,
                                     None if dst is None else s.up(dst), w, **scales)
        s.table = s.table if dst is None else dst
        for b in range(s.B):
            n = s.lens[b]
            s.lens[b] = int(lens[b])
            assert s.lens[b] == min(n, keep)
            k, v = s.held(b, s.lens[b])
            for h in range(2):
                idx = choose(wh[b, h], n, keep, sinks, recent)
                assert kept[b, h, :len(idx)].tolist() == idx
                assert np.array_equal(k[:, h], before[b][0][idx, h]) and np.array_equal(v[:, h], before[b][1][idx, h])
                assert np.array_equal(su.host(w)[b, h, :len(idx)], wh[b, h, idx])

    def steps(n, w):
        for _ in range(n):
            q, kn, vn = s.randn(s.B, 1, 8, 64, times=2.0), s.randn(s.B, 1, 2, 64), s.randn(s.B, 1, 2, 64)
            earlier = su.host(w)
            out = ff.paged_attention_scored(q, s.k, s.v, s.up(s.table), s.ctx(), k_new=kn, v_new=vn, weights=w, prior=w,
                                            decay=0.9, max_context_len=T, **s.rules(), **scales)
            for b in range(s.B):
                pos = s.lens[b]
                o, e, x, we = s.expect(q, b, pos, pos + 1)
                su.check(su.host(out).reshape(s.B, 8, 64)[b], o[0], e[0], f"decode, row {b}")
                x = x + np.pad(0.9 * earlier[b, :, :pos], ((0, 0), (0, 1)))
                su.check(su.host(w)[b, :, :pos + 1], x, we + 2.0 ** -22 * x, f"accumulated, row {b}")
                s.lens[b] += 1

    cut(w, s.pages([(keep + 30 + 15) // 16] * s.B))
    steps(20, w)
    cut(w, None)
    steps(3, w)


@pytest.mark.skip(reason="the replay faulted when the library still allocated inside a capture; such calls are refused now "
                         "(test_capture_needs_workspaces), and graphs are given workspaces (test_captured_together)")
def test_captured_without_workspaces(ff, gpu):
    """Weights of a prompt's end, a decode step with weights and an eviction of long rows, captured in one graph with memory of
    their own: every replay gives what the eager calls give, with eager calls in between."""
    B, n, keep, Hq, Hkv, D = 2, 9000, 4000, 4, 2, 64
    g = torch.Generator(device=gpu).manual_seed(3)
    room = (n + 16) // 16
    rnd = lambda *s: torch.randn(s, generator=g, device=gpu, dtype=torch.float32).to(torch.bfloat16)  # noqa: E731
    k, v = rnd(B * room * 2, 16, Hkv, D), rnd(B * room * 2, 16, Hkv, D)
    order = torch.randperm(B * room * 2, generator=g, device=gpu).to(torch.int32)
    table, dst = order[:B * room].view(B, room).contiguous(), order[B * room:].view(B, room).contiguous()
    lens = torch.tensor([n, n - 500], dtype=torch.int32, device=gpu)
    before = lens - 16
    ql, q = rnd(B, 16, Hq, D), rnd(B, 1, Hq, D)
    T = n + 1

    def calls(w, kept, left, out, cut):
        ff.attention_weights(ql, k, table, before, weights=w, max_context_len=T, score_cap=20.0)
        ff.paged_attention_scored(q, k, v, table, lens, weights=w, prior=w, decay=0.5, out=out, max_context_len=T, window=3000)
        ff.evict_tokens(w, k, v, table, lens, keep, 4, 300, dst, cut, kept, left)

    def buffers():
        return (torch.zeros(B, Hkv, T, device=gpu), torch.zeros(B, Hkv, keep, dtype=torch.int32, device=gpu),
                torch.zeros(B, dtype=torch.int32, device=gpu), torch.zeros(B, 1, Hq * D, dtype=torch.bfloat16, device=gpu),
                torch.zeros(B, Hkv, keep, device=gpu))

    eager, got = buffers(), buffers()
    calls(*eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(*got)
    for _ in range(4):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, got):
            assert torch.equal(a, b)
        again = buffers()
        calls(*again)
        torch.cuda.synchronize()
        for a, b in zip(eager, again):
            assert torch.equal(a, b)


def test_capture_needs_workspaces(ff, gpu):
    """A captured call that would have to allocate is refused before anything is launched; one that needs nothing is not."""
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16, device=gpu)
    k, v = (torch.zeros(600, 16, 2, 64, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    table = torch.arange(600, dtype=torch.int32, device=gpu)[None]
    lens = torch.tensor([9500], dtype=torch.int32, device=gpu)
    w, out = torch.zeros(1, 2, 9600, device=gpu), torch.zeros(1, 1, 256, dtype=torch.bfloat16, device=gpu)
    kept, left = torch.zeros(1, 2, 100, dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out.fill_(1.0)
        for call in (lambda: ff.attention_weights(q, k, table, lens, weights=w),
                     lambda: ff.paged_attention_scored(q, k, v, table, lens, weights=w, out=out),
                     lambda: ff.evict_tokens(w, k, v, table, lens, 100, kept=kept, kept_lens=left)):
            with pytest.raises(ff.FFKVError, match="workspace"):
                call()
    graph.replay()
    torch.cuda.synchronize()
    assert (out == 1.0).all() and (w == 0).all() and (kept == 0).all()


def test_captured_together(ff, gpu):
    """Weights of a prompt's end, a decode step with weights and an eviction of long rows in one graph, one workspace for all:
    every replay gives what the eager calls give, with eager calls on the same workspace in between."""
    B, n, keep, Hq, Hkv, D = 2, 9000, 4000, 4, 2, 64
    g = torch.Generator(device=gpu).manual_seed(3)
    room = (n + 16) // 16
    rnd = lambda *s: torch.randn(s, generator=g, device=gpu, dtype=torch.float32).to(torch.bfloat16)  # noqa: E731
    k, v = rnd(B * room * 2, 16, Hkv, D), rnd(B * room * 2, 16, Hkv, D)
    order = torch.randperm(B * room * 2, generator=g, device=gpu).to(torch.int32)
    table, dst = order[:B * room].view(B, room).contiguous(), order[B * room:].view(B, room).contiguous()
    lens = torch.tensor([n, n - 500], dtype=torch.int32, device=gpu)
    before = lens - 16
    ql, q = rnd(B, 16, Hq, D), rnd(B, 1, Hq, D)
    T = n + 1
    ws = max((ff.decode_scored_workspace(B, Hq, D, room, T, weights=True, device=gpu),
              ff.attention_weights_workspace(B, 16, Hq, Hkv, D, room, T, device=gpu),
              ff.evict_workspace(B, Hkv, keep, T, room, device=gpu)), key=lambda t: t.numel())

    def calls(w, kept, left, out, cut):
        ff.attention_weights(ql, k, table, before, weights=w, max_context_len=T, score_cap=20.0, workspace=ws)
        ff.paged_attention_scored(q, k, v, table, lens, weights=w, prior=w, decay=0.5, out=out, max_context_len=T, window=3000,
                                  workspace=ws)
        ff.evict_tokens(w, k, v, table, lens, keep, 4, 300, dst, cut, kept, left, workspace=ws)

    def buffers():
        return (torch.zeros(B, Hkv, T, device=gpu), torch.zeros(B, Hkv, keep, dtype=torch.int32, device=gpu),
                torch.zeros(B, dtype=torch.int32, device=gpu), torch.zeros(B, 1, Hq * D, dtype=torch.bfloat16, device=gpu),
                torch.zeros(B, Hkv, keep, device=gpu))

    eager, got = buffers(), buffers()
    calls(*eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(*got)
    for _ in range(4):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, got):
            assert torch.equal(a, b)
        again = buffers()
        calls(*again)
        torch.cuda.synchronize()
        for a, b in zip(eager, again):
            assert torch.equal(a, b)
