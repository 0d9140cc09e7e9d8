"""Steps captured without a workspace of the caller's: nothing is allocated inside the graph.  The C ABI's plain decodes leave
their rows whole there, the C++ API allocates its thread's workspace beside the graph."""

import ctypes
import os
from pathlib import Path

import numpy as np
import pytest
import torch

import cases
import gpu_util as gu
import oracle as O
import scored_util as su
from test_gpu_decode_row import NAME
from test_gpu_parity import TOL, half_ulp

pytestmark = pytest.mark.gpu
CPP = Path(__file__).resolve().parent / "cpp"


def _replays(graph, outs, between):
    """The captured outputs, the same bits after each of several replays with eager work between them."""
    first = None
    for _ in range(4):
        for t in outs:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, got))
        first = got
        between()
        torch.cuda.synchronize()
    return first


@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [("bf16", "bf16", 32, 8, 128), ("f16", "f16", 7, 1, 64), ("bf16", "i8", 40, 2, 112),
                                             ("bf16", "fp8", 4, 1, 256), ("f32", "f32", 16, 2, 128), ("bf16", "bf16", 8, 2, 72)])
def test_plain_decode(ff, gpu, act, kv, Hq, Hkv, D):
    """Three layers' decodes in one graph, of rows long enough to be split eagerly, each against the checker."""
    c = cases.make_case(71, 3, Hq, Hkv, D, [3000, 0, 1777], act=act, kv=kv, input_scale=1 / np.sqrt(D))
    kp, vp = c.k_pool.copy(), c.v_pool.copy()
    ks, vs = (None if x is None else x.copy() for x in (c.k_scale, c.v_scale))
    O.append(c.k_new, c.v_new, c.act, kp, vp, c.kv, c.block_table, c.ctx, ks, vs)
    _, ref = O.paged_decode(c.q, c.act, kp, vp, c.kv, c.block_table, c.ctx, ks, vs)
    dk, dv, dks, dvs, bt, cx, kn, vn, q = su.device(c, gpu)
    kw = {"k_scale": dks, "v_scale": dvs}
    outs = [torch.empty(3, 1, Hq * D, dtype=q.dtype, device=gpu) for _ in range(3)]

    def step(outs):
        ff.append_paged_attention(kn, vn, q, dk, dv, bt, cx, out=outs[0], **kw)
        ff.paged_attention(q, dk, dv, bt, cx, out=outs[1], **kw)
        ff.paged_attention_shared_prefix(q, dk, dv, bt, cx, 0, out=outs[2], **kw)

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(outs)
    eager = [torch.empty_like(t) for t in outs]
    for got in _replays(graph, outs, lambda: step(eager)):
        g = got.float().cpu().numpy().reshape(ref.shape).astype(np.float64)
        excess = np.abs(g - ref) - half_ulp(np.maximum(np.abs(g), np.abs(ref)), c.act)
        assert float(excess.max()) <= TOL.get((NAME[c.act], NAME[c.kv]), 2e-3)


def test_shared_prefix(ff, gpu):
    """A shared prefix is attended with the rows' own pages."""
    B, shared = 12, 20
    c = cases.make_case(73, B, 8, 2, 128, [shared * 16 + 10 * b for b in range(B)], act="bf16", shared_prefix_blocks=shared)
    _, ref = O.paged_decode(c.q, c.act, c.k_pool, c.v_pool, c.kv, c.block_table, c.ctx)
    dk, dv, q = gu.to_dev(c.k_pool, c.kv, gpu), gu.to_dev(c.v_pool, c.kv, gpu), gu.to_dev(c.q, c.act, gpu)
    bt, cx = torch.from_numpy(c.block_table).to(gpu), torch.from_numpy(c.ctx).to(gpu)
    out, eager = (torch.empty(B, 1, 8 * 128, dtype=q.dtype, device=gpu) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ff.paged_attention_shared_prefix(q, dk, dv, bt, cx, shared, out=out)
    got, = _replays(graph, [out], lambda: ff.paged_attention_shared_prefix(q, dk, dv, bt, cx, shared, out=eager))
    for t in (got, eager):
        g = t.float().cpu().numpy().reshape(ref.shape).astype(np.float64)
        assert float((np.abs(g - ref) - half_ulp(np.maximum(np.abs(g), np.abs(ref)), c.act)).max()) <= 2e-3


def test_cxx_scored(ff, gpu):
    """Weights of a prompt's end, a decode step with weights and an eviction of long rows through the C++ API, captured on a
    stream that has run nothing yet: each replay gives the eager calls' bits."""
    shim = ctypes.CDLL(str(CPP / "libscored_api_shim.so"), mode=os.RTLD_NOW)
    vp, i, f = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
    shim.sas_attention.argtypes = [vp] * 8 + [i] * 9 + [f, vp, i, vp, vp, vp, vp, f, i, vp]
    shim.sas_weights.argtypes = [vp] * 5 + [i] * 9 + [f, vp, i, vp, vp, vp, vp, f, i, vp]
    shim.sas_evict.argtypes = [vp, i] + [vp] * 6 + [i] * 9 + [vp] * 3 + [i, vp, vp]
    shim.sas_last_error.restype = ctypes.c_char_p
    B, n, keep, Hq, Hkv, D = 2, 9000, 4000, 4, 2, 64
    g = torch.Generator(device=gpu).manual_seed(5)
    room = (n + 16) // 16
    N, T = 2 * B * room, n + 1
    rnd = lambda *s: torch.randn(s, generator=g, device=gpu, dtype=torch.float32).to(torch.bfloat16)  # noqa: E731
    k, v = rnd(N, 16, Hkv, D), rnd(N, 16, Hkv, D)
    order = torch.randperm(N, generator=g, device=gpu).to(torch.int32)
    table, dst = order[:B * room].view(B, room).contiguous(), order[B * room:].view(B, room).contiguous()
    lens = torch.tensor([n, n - 500], dtype=torch.int32, device=gpu)
    before = lens - 16
    ql, q = rnd(B, 16, Hq, D), rnd(B, 1, Hq, D)
    p = lambda t: t.data_ptr()  # noqa: E731

    def calls(bufs, stream):
        w, kept, left, out, cut = map(p, bufs)
        st = stream.cuda_stream
        assert shim.sas_weights(p(ql), p(k), None, p(table), p(before), B, 16, Hq, Hkv, D, N, room, 2, 2, 20.0, None, 0, None, None,
                                w, None, 1.0, T, st) == 0, shim.sas_last_error()
        assert shim.sas_attention(p(q), p(k), p(v), None, None, out, p(table), p(lens), B, 1, Hq, Hkv, D, N, room, 2, 2, 0.0, None,
                                  3000, None, None, w, w, 0.5, T, st) == 0, shim.sas_last_error()
        assert shim.sas_evict(w, T, p(k), p(v), None, None, p(table), p(lens), B, Hkv, D, N, room, 2, keep, 4, 300, kept, left,
                              p(dst), room, cut, st) == 0, shim.sas_last_error()

    def buffers():
        return (torch.zeros(B, Hkv, T, device=gpu), torch.zeros(B, Hkv, keep, dtype=torch.int32, device=gpu),
                torch.zeros(B, dtype=torch.int32, device=gpu), torch.zeros(B, 1, Hq * D, dtype=torch.bfloat16, device=gpu),
                torch.zeros(B, Hkv, T, device=gpu))

    want, got = buffers(), buffers()
    side, cur = torch.cuda.Stream(), torch.cuda.current_stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        calls(got, side)
    calls(want, cur)
    for _ in range(4):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        again = buffers()
        calls(again, cur)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, x) for a, b, x in zip(want, got, again))


def test_cxx_step(gpu):
    """kernels::append_kv_cache and kernels::attention of three layers, captured on a stream that has run nothing yet."""
    shim = ctypes.CDLL(str(CPP / "libdecode_step_shim.so"), mode=os.RTLD_NOW)
    vp, i = ctypes.c_void_p, ctypes.c_int
    ip, pp = ctypes.POINTER(i), ctypes.POINTER(vp)
    shim.dss_create.restype, shim.dss_create.argtypes = vp, [i, i]
    shim.dss_destroy.argtypes = [vp]
    shim.dss_error.restype, shim.dss_error.argtypes = ctypes.c_char_p, [vp]
    shim.dss_pack.argtypes = [vp, i, ip, ip, ip]
    shim.dss_upload.argtypes = [vp, vp]
    shim.dss_host_table.restype, shim.dss_host_table.argtypes = ip, [vp]
    shim.dss_step.argtypes = [vp, i, i] + [pp] * 6 + [i] * 5 + [vp]
    shim.dss_launch.argtypes = [vp, vp]
    L, B, Hq, Hkv, D, N, stride = 3, 2, 32, 8, 128, 200, 64
    rng = np.random.default_rng(79)
    ctx = [900, 333]
    pages = rng.permutation(N)
    nblk = [(n + 16) // 16 for n in ctx]
    arr = lambda x: (i * len(x))(*map(int, x))  # noqa: E731
    enc = lambda *s: cases.encode(rng.standard_normal(s, dtype=np.float32), O.DTYPE_BF16)  # noqa: E731
    stream = torch.cuda.Stream().cuda_stream
    h = shim.dss_create(B, stride)
    try:
        shim.dss_pack(h, B, arr(ctx), arr(nblk), arr(pages[:sum(nblk)]))
        assert shim.dss_upload(h, stream) == 0
        table = np.ctypeslib.as_array(shim.dss_host_table(h), shape=(B * stride,)).reshape(B, stride).copy()
        host = [{n: enc(*s) for n, s in (("q", (B, 1, Hq, D)), ("k", (B, 1, Hkv, D)), ("v", (B, 1, Hkv, D)),
                                         ("kp", (N, 16, Hkv, D)), ("vp", (N, 16, Hkv, D)))} for _ in range(L)]
        dev = [{n: gu.to_dev(x, O.DTYPE_BF16, gpu) for n, x in l.items()} for l in host]
        outs = [torch.zeros(B, 1, Hq * D, dtype=torch.bfloat16, device=gpu) for _ in range(L)]
        ptrs = lambda ts: (vp * L)(*[t.data_ptr() for t in ts])  # noqa: E731
        torch.cuda.synchronize()
        args = [ptrs([l[n] for l in dev]) for n in ("q", "k", "v", "kp", "vp")] + [ptrs(outs), Hq, Hkv, D, N, O.DTYPE_BF16, stream]
        assert shim.dss_step(h, 0, L, *args) == 0, shim.dss_error(h)
        for _ in range(4):
            for t in outs:
                t.fill_(float("nan"))
            torch.cuda.synchronize()
            assert shim.dss_launch(h, stream) == 0, shim.dss_error(h)
            torch.cuda.synchronize()
            for l, t in zip(host, outs):
                kp, vp_ = l["kp"].copy(), l["vp"].copy()
                O.append(l["k"], l["v"], O.DTYPE_BF16, kp, vp_, O.DTYPE_BF16, table, np.array(ctx, np.int32))
                _, ref = O.paged_decode(l["q"], O.DTYPE_BF16, kp, vp_, O.DTYPE_BF16, table, np.array(ctx, np.int32))
                g = t.float().cpu().numpy().reshape(ref.shape).astype(np.float64)
                assert float((np.abs(g - ref) - half_ulp(np.maximum(np.abs(g), np.abs(ref)), O.DTYPE_BF16)).max()) <= 2e-3
            assert shim.dss_step(h, 1, L, *args) == 0, shim.dss_error(h)  # eager between the replays
            torch.cuda.synchronize()
    finally:
        shim.dss_destroy(h)
