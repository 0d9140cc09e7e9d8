"""The softmax scale of the attention over listed pages, in each of its kernels: queries times scale * sqrt(D) at the default."""

import numpy as np
import pytest
import torch

import blocks_util as bu
import cases
import scored_util as su
from test_gpu_attention_blocks import lists, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,kv", [("bf16", "bf16"), ("bf16", "i8"), ("bf16", "fp8"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("Hq,Hkv,D,ctx,S,count,T", [
    (8, 2, 128, [700, 33], 1, 20, 1), (8, 2, 128, [4000], 1, 200, 1), (14, 2, 80, [900], 1, 30, 1),  # a step, whole and split
    (8, 2, 128, [257], 5, 8, 2), (8, 2, 128, [257], 270, 8, 2), (10, 2, 256, [700, 15], 140, 30, 40),  # few and many tokens
    (36, 9, 128, [1100, 1300], 120, 61, 16), (24, 12, 64, [1700, 900], 130, 107, 16),  # in halves
    (8, 2, 128, [2500, 40, 1200], 40, 150, 32), (5, 1, 64, [3000], 107, 170, 7),  # split
    (4, 4, 72, [100, 333], 3, 11, 1),
])
@pytest.mark.parametrize("scale", [0.31, 0.02])
def test_scale(ff, gpu, act, kv, Hq, Hkv, D, ctx, S, count, T, scale):
    c = make(Hq + S, ctx, S, Hq, Hkv, D, act, kv)
    li = lists(c, S, count, T)
    q = cases.decode(c.q, c.act).astype(np.float64) * (np.float64(np.float32(scale)) * np.sqrt(D))
    want, bound = bu.attend(c, q, li, T, c.act, S, 2.0 ** -10 if T > 1 else 2.0 ** -11)
    su.check(su.host(run(ff, c, li, T, gpu, scale=scale)).reshape(want.shape), want, bound, "out")


@pytest.mark.parametrize("S,T,ctx,count", [(1, 1, [4000], 200), (40, 32, [2500, 40], 150)])
def test_scale_in_a_capture(ff, gpu, S, T, ctx, count):
    """Captured without a workspace, lists stay whole: the scale goes there too."""
    c = make(3, ctx, S, 8, 2, 128)
    kp, vp, _, _, bt, cx, _, _, q = su.device(c, gpu)
    li = lists(c, S, count, T)
    ld, out = torch.from_numpy(li).to(gpu), torch.empty(c.B, S, 8 * 128, dtype=q.dtype, device=gpu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ff.paged_attention_blocks(q, kp, vp, bt, cx, ld, query_block=T, out=out, scale=0.25)
    for _ in range(2):
        out.zero_()
        graph.replay()
        wide = cases.decode(c.q, c.act).astype(np.float64) * (0.25 * np.sqrt(128.0))
        want, bound = bu.attend(c, wide, li, T, c.act, S, 2.0 ** -10 if T > 1 else 2.0 ** -11)
        su.check(su.host(out).reshape(want.shape), want, bound, "out")
