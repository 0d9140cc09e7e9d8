"""A layer's calls through the C++ API of rotary positions on several axes, key bounds, the choice of pages and the attention
over them (include/firefly/kernels.h), against the Python calls: the same bits."""

import ctypes
import os
from pathlib import Path

import pytest
import torch

import oracle as O
import scored_util as su
from test_gpu_attention_blocks import make

SHIM = Path(__file__).resolve().parent / "cpp" / "libblocks_api_shim.so"


@pytest.fixture(scope="module")
def shim(ff):
    lib = ctypes.CDLL(str(SHIM), mode=os.RTLD_NOW)
    vp, i = ctypes.c_void_p, ctypes.c_int
    lib.bas_layer.argtypes = [vp] * 4 + [ctypes.POINTER(i), i, i] + [vp] * 9 + [i] * 14 + [vp]
    lib.bas_rope.argtypes = [vp] * 3 + [ctypes.POINTER(i)] + [i] * 7 + [vp]
    lib.bas_last_error.restype = ctypes.c_char_p
    return lib


def _p(t):
    return None if t is None else t.data_ptr()


@pytest.mark.parametrize("op", range(18))
def test_refusals(shim, op):
    assert shim.bas_refusal(op) == -1 and shim.bas_last_error() != b""
    assert shim.bas_refusal(-1) == 0 and shim.bas_last_error() == b""  # the next call's own result


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "i8"])
@pytest.mark.parametrize("S,T", [(1, 1), (30, 16)])
def test_layer(ff, gpu, shim, kv, S, T):
    c = make(5, [700, 40, 1600], S, 8, 2, 128, "bf16", kv)
    sections, count = (16, 24, 24), 12
    pos = torch.randint(0, 3000, (3, 3, S), dtype=torch.int32, device=gpu)
    li = torch.full((3, -(-S // T), 2, count), -1, dtype=torch.int32, device=gpu)
    stream = torch.cuda.current_stream().cuda_stream

    def state():
        kp, vp, ks, vs, bt, cx, kn, vn, q = su.device(c, gpu)
        box = ff.key_bounds(kp).zero_()
        ff.update_key_bounds(kp, box, bt, torch.zeros_like(cx), int(c.ctx.max()), k_scale=ks)
        return kp, vp, ks, vs, bt, cx, kn, vn, q, box

    kp, vp, ks, vs, bt, cx, kn, vn, q, box = state()
    ff.rope_append_axes(q, kn, vn, pos, sections, kp, vp, bt, cx, k_scale=ks, v_scale=vs)
    ff.update_key_bounds(kp, box, bt, cx, S, k_scale=ks)
    want_li = ff.select_blocks(q, box, bt, cx, count, sinks=1, recent=3, query_block=T)
    want = ff.paged_attention_blocks(q, kp, vp, bt, cx, want_li, query_block=T, k_scale=ks, v_scale=vs)
    kp2, vp2, ks2, vs2, bt, cx, kn, vn, q2, box2 = state()
    out = torch.full_like(want, float("nan"))
    rc = shim.bas_layer(_p(q2), _p(kn), _p(vn), _p(pos), (ctypes.c_int * 3)(*sections), 3, 0, _p(kp2), _p(vp2), _p(ks2), _p(vs2),
                        _p(box2), _p(li), _p(out), _p(bt), _p(cx), 3, S, 8, 2, 128, c.num_blocks, c.max_blocks, c.act, c.kv,
                        O.DTYPE_BF16, count, 1, 3, T, stream)
    assert rc == 0, shim.bas_last_error()
    for a, b in ((q, q2), (kp, kp2), (vp, vp2), (ks, ks2), (vs, vs2), (box, box2), (want_li, li), (want, out)):
        assert (a is None and b is None) or torch.equal(a, b)
    x, y = kn.clone(), q.clone()
    ff.apply_rope_axes(y, x, pos, sections)
    rc = shim.bas_rope(_p(q2), _p(kn), _p(pos), (ctypes.c_int * 3)(*sections), 3, 3, S, 8, 2, 128, c.act, stream)
    assert rc == 0 and torch.equal(q2, y) and torch.equal(kn, x)
