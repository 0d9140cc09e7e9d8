"""Rotary embedding by positions on several axes, alone and fused with the append, against the formula in long double."""

import numpy as np
import pytest
import torch

import blocks_util as bu
import cases
import gpu_util as gu
import oracle as O
import scored_util as su

pytestmark = pytest.mark.gpu

BF, F16, F32 = O.DTYPE_BF16, O.DTYPE_F16, O.DTYPE_F32
TORCH = {BF: torch.bfloat16, F16: torch.float16, F32: torch.float32}


def inputs(rng, act, B, S, Hq, Hkv, D, axes, far, dev):
    """q, k, v as views of one projection, and positions."""
    x = cases.encode(rng.standard_normal((B, S, Hq + 2 * Hkv, D), dtype=np.float32), act)
    packed = gu.to_dev(x, act, dev)
    pos = rng.integers(-far // 8, far + 1, (axes, B, S)).astype(np.int32)
    return x, packed, packed[:, :, :Hq], packed[:, :, Hq:Hq + Hkv], packed[:, :, Hq + Hkv:], pos


def f64(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("act", [BF, F16, F32])
@pytest.mark.parametrize("B,S,Hq,Hkv,D,sections,interleaved,far", [
    (1, 1, 1, 1, 128, (64,), False, 100), (3, 1, 16, 8, 128, (16, 24, 24), False, 40000),
    (2, 7, 5, 1, 64, (8, 0, 12, 12), False, 1 << 24), (2, 33, 28, 4, 128, (24, 20, 20), True, 200000),
    (1, 130, 3, 3, 256, (43, 43, 42), True, 1000000), (4, 2, 8, 2, 64, (30, 2), True, 70), (1, 700, 9, 3, 256, (1, 127), False, 5000),
    (5, 1, 64, 8, 128, (22, 21, 21), True, 1 << 24),
])
def test_rotation(ff, gpu, act, B, S, Hq, Hkv, D, sections, interleaved, far):
    rng = np.random.default_rng(B * 1000 + S)
    x, _, q, k, _, pos = inputs(rng, act, B, S, Hq, Hkv, D, len(sections), far, gpu)
    at = torch.from_numpy(pos).to(gpu)
    q_out, k_out = torch.empty((B, S, Hq, D), dtype=q.dtype, device=gpu), torch.empty((B, S, Hkv, D), dtype=q.dtype, device=gpu)
    got = ff.apply_rope_axes(q, k, at, sections, interleaved=interleaved, theta=5e5, q_out=q_out, k_out=k_out)
    assert got[0] is q_out and got[1] is k_out
    xv = cases.decode(x, act).astype(np.float64)
    want, bound = bu.rotate(xv, pos, sections, interleaved, 5e5, act)
    su.check(f64(q_out), want[:, :, :Hq], bound[:, :, :Hq], "q")
    su.check(f64(k_out), want[:, :, Hq:Hq + Hkv], bound[:, :, Hq:Hq + Hkv], "k")
    assert np.array_equal(f64(q), xv[:, :, :Hq])  # the projection is only read
    ff.apply_rope_axes(q, k, at, sections, interleaved=interleaved, theta=5e5)  # in place, where it lies
    assert torch.equal(q, q_out) and torch.equal(k, k_out)


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kv", ["bf16", "f16", "f32", "i8", "fp8"])
@pytest.mark.parametrize("D,S,ctx", [(64, 3, [5, 31, 1000]), (128, 1, [0, 17, 300, 4000]), (256, 20, [0, 9])])
def test_append(ff, gpu, act, kv, D, S, ctx):
    """The pages are those of the rotation followed by the append, to the bit, and nothing else of the pools is written."""
    Hq, Hkv, B = 6, 2, len(ctx)
    c = cases.make_case(D + S, B, Hq, Hkv, D, ctx, act=act, kv=kv, S=S)
    c.block_table[-1, -1] = c.num_blocks  # a page that is none
    rng = np.random.default_rng(S)
    _, packed, q, k, v, pos = inputs(rng, c.act, B, S, Hq, Hkv, D, 3, 5000, gpu)
    sections = (D // 2 - 2 * (D // 6), D // 6, D // 6)
    at, bt, cx = (torch.from_numpy(a).to(gpu) for a in (pos, c.block_table, c.ctx))
    kp, vp = gu.to_dev(c.k_pool, c.kv, gpu), gu.to_dev(c.v_pool, c.kv, gpu)
    ks = None if c.k_scale is None else torch.from_numpy(c.k_scale.copy()).to(gpu)
    vs = None if c.v_scale is None else torch.from_numpy(c.v_scale.copy()).to(gpu)
    q_out = ff.rope_append_axes(q, k, v, at, sections, kp, vp, bt, cx, interleaved=S == 1, k_scale=ks, v_scale=vs,
                                q_out=torch.empty((B, S, Hq, D), dtype=q.dtype, device=gpu))
    rk, rq = torch.empty((B, S, Hkv, D), dtype=q.dtype, device=gpu), torch.empty_like(q_out)
    ff.apply_rope_axes(q, k, at, sections, interleaved=S == 1, q_out=rq, k_out=rk)
    assert torch.equal(q_out, rq)
    pack = np.uint16 if c.act != F32 else np.float32
    O.append(gu.to_host(rk, pack), gu.to_host(v.contiguous(), pack), c.act, c.k_pool, c.v_pool, c.kv, c.block_table, c.ctx,
             c.k_scale, c.v_scale)
    def same(t, want):
        return np.array_equal(gu.to_host(t, want.dtype).view(np.uint8), want.view(np.uint8))
    assert same(kp, c.k_pool) and same(vp, c.v_pool)
    if kv == "i8":
        assert same(ks, c.k_scale) and same(vs, c.v_scale)


def test_as_the_plain_rotation(ff, gpu):
    """Equal positions on all axes are the plain rotary embedding, up to the rounding of its angle (2^-24 of it)."""
    B, S, Hq, Hkv, D = 2, 40, 4, 2, 128
    q, k = torch.randn(B, S, Hq, D, device=gpu), torch.randn(B, S, Hkv, D, device=gpu)
    ctx = torch.tensor([3, 900], dtype=torch.int32, device=gpu)
    pos = (ctx[:, None] + torch.arange(S, device=gpu, dtype=torch.int32)).expand(3, B, S).contiguous()
    a, b = ff.apply_rope_axes(q, k, pos, (16, 24, 24), q_out=torch.empty_like(q), k_out=torch.empty_like(k))
    norm = q.abs().max().item(), k.abs().max().item()
    ff.apply_rope(q, k, ctx, 1e6)
    # an angle up to 940 is off by 940 (2^-24 of the product, 2^-24 of the frequency), cos, sin and rotation by 2^-21
    tol = 2 * (940 * 2.0 ** -23 + 2.0 ** -21)
    assert (a - q).abs().max().item() <= tol * norm[0] and (b - k).abs().max().item() <= tol * norm[1]


def test_odd_calls(ff, gpu):
    """Without q; rows before the cache's beginning; a context that is none; nothing to do."""
    c = cases.make_case(3, 3, 4, 2, 64, [0, 40, 3], S=2)
    bt = torch.from_numpy(c.block_table).to(gpu)
    ctx = torch.tensor([-1, 40, -9], dtype=torch.int32, device=gpu)  # row 0's second token goes to 0, row 2's to nowhere
    k, v = gu.to_dev(c.k_new, c.act, gpu), gu.to_dev(c.v_new, c.act, gpu)
    kp, vp = gu.to_dev(c.k_pool, c.kv, gpu), gu.to_dev(c.v_pool, c.kv, gpu)
    before = kp.clone()
    pos = torch.randint(0, 99, (2, 3, 2), dtype=torch.int32, device=gpu)
    assert ff.rope_append_axes(None, k, v, pos, (16, 16), kp, vp, bt, ctx) is None
    rk = ff.apply_rope_axes(None, k, pos, (16, 16), k_out=torch.empty_like(k))[1]
    want = before.clone()
    want[c.block_table[0, 0], 0] = rk[0, 1]
    for t in range(2):
        want[c.block_table[1, 2], 8 + t] = rk[1, t]
    assert torch.equal(kp, want)
    fresh = kp.clone()
    ff.rope_append_axes(None, k, v, pos, (16, 16), fresh, vp, bt, None)  # from position 0 on
    for b in range(3):
        assert torch.equal(fresh[c.block_table[b, 0], :2], rk[b])
    ff.apply_rope_axes(k[:, :0], k[:, :0], pos[:, :, :0].contiguous(), (16, 16))


def test_streams_and_graphs(ff, gpu):
    c = cases.make_case(8, 4, 8, 2, 128, [5, 60, 16, 100])
    bt, ctx = torch.from_numpy(c.block_table).to(gpu), torch.from_numpy(c.ctx).to(gpu)
    q, k, v = (gu.to_dev(a, c.act, gpu) for a in (c.q, c.k_new, c.v_new))
    pos = torch.randint(0, 9999, (3, 4, 1), dtype=torch.int32, device=gpu)
    kp, vp = gu.to_dev(c.k_pool, c.kv, gpu), gu.to_dev(c.v_pool, c.kv, gpu)
    out = torch.empty_like(q)
    run = lambda s=None: ff.rope_append_axes(q, k, v, pos, (16, 24, 24), kp, vp, bt, ctx, q_out=out, stream=s)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    run(side)
    side.synchronize()
    first, pages = out.clone(), kp.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(3):
        pos.add_(i)
        out.zero_()
        kp.zero_()
        graph.replay()
        got, gp = out.clone(), kp.clone()
        torch.cuda.synchronize()
        kp.zero_()
        run()
        assert torch.equal(got, out) and torch.equal(gp, kp)
        if i == 0:
            assert torch.equal(got, first) and not torch.equal(gp, pages)


def test_many_tokens(ff, gpu):
    """More tokens than the launch has waves: each as in a call of its own."""
    S, sections = 300_007, (16, 8, 8)
    k = torch.randn(1, S, 2, 64, device=gpu).half()
    pos = torch.randint(-5, 1 << 20, (3, 1, S), dtype=torch.int32, device=gpu)
    _, got = ff.apply_rope_axes(None, k, pos, sections, k_out=torch.empty_like(k))
    at = S // 3
    for part in (slice(0, at), slice(at, 2 * at), slice(2 * at, S)):
        x = k[:, part].clone()
        ff.apply_rope_axes(None, x, pos[:, :, part].contiguous(), sections)
        assert torch.equal(got[:, part], x)
    tail = slice(S - 2000, S)
    want, bound = bu.rotate(f64(k[:, tail]), pos[:, :, tail].cpu().numpy(), sections, False, 1e6, F16)
    su.check(f64(got[:, tail]), want, bound, "tail")
