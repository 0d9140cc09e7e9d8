"""The C++ API of scored attention, attention weights and eviction (include/firefly/kernels.h) against the Python calls: the
same bits, and the errors that it reports."""

import ctypes
import os
from pathlib import Path

import numpy as np
import pytest
import torch

import scored_util as su
from test_gpu_scored_prefill import make, masked, rule_of

SHIM = Path(__file__).resolve().parent / "cpp" / "libscored_api_shim.so"


@pytest.fixture(scope="module")
def shim(ff):
    lib = ctypes.CDLL(str(SHIM), mode=os.RTLD_NOW)
    vp, i, f = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
    lib.sas_attention.argtypes = [vp] * 8 + [i] * 9 + [f, vp, i, vp, vp, vp, vp, f, i, vp]
    lib.sas_weights.argtypes = [vp] * 5 + [i] * 9 + [f, vp, i, vp, vp, vp, vp, f, i, vp]
    lib.sas_evict.argtypes = [vp, i] + [vp] * 6 + [i] * 9 + [vp] * 3 + [i, vp, vp]
    lib.sas_last_error.restype = ctypes.c_char_p
    return lib


def test_symbols(shim):
    assert shim.sas_last_error() == b""


def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "i8"])
def test_decode_weights_and_evict(ff, gpu, shim, kv):
    c = make(3, [700, 40, 130], 1, 8, 2, 128, "bf16", kv)
    kp, vp, ks, vs, bt, cx, _, _, q = su.device(c, gpu)
    T = 16 * c.max_blocks
    sl = torch.rand(8, device=gpu)
    begin = torch.tensor([5, 0, 3], dtype=torch.int32, device=gpu)
    prior = torch.rand(3, 2, T, device=gpu)
    w, w2, out = torch.zeros_like(prior), torch.zeros_like(prior), torch.empty(3, 1, 8 * 128, dtype=q.dtype, device=gpu)
    want = ff.paged_attention_scored(q, kp, vp, bt, cx, 9.0, sl, 600, begin, weights=w, prior=prior, decay=0.5, k_scale=ks,
                                     v_scale=vs, max_context_len=T)
    rc = shim.sas_attention(_p(q), _p(kp), _p(vp), _p(ks), _p(vs), _p(out), _p(bt), _p(cx), 3, 1, 8, 2, 128, c.num_blocks,
                            c.max_blocks, c.act, c.kv, 9.0, _p(sl), 600, _p(begin), None, _p(w2), _p(prior), 0.5, T, _stream())
    assert rc == 0, shim.sas_last_error()
    assert torch.equal(want, out) and torch.equal(w, w2)
    rc = shim.sas_weights(_p(q), _p(kp), _p(ks), _p(bt), _p(cx), 3, 1, 8, 2, 128, c.num_blocks, c.max_blocks, c.act, c.kv, 9.0,
                          _p(sl), 600, _p(begin), None, _p(w2), _p(prior), 0.5, T, _stream())
    assert rc == 0, shim.sas_last_error()
    assert torch.equal(w2, ff.attention_weights(q, kp, bt, cx, torch.zeros_like(w), prior, 0.5, 9.0, sl, 600, begin.view(3, 1),
                                                k_scale=ks))
    lens = cx + 1
    kept, n = torch.full((3, 2, 50), -1, dtype=torch.int32, device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu)
    kc, vc, kw = kp.clone(), vp.clone(), w.clone()
    a, an = ff.evict_tokens(kw, kc, vc, bt, lens, 50, 2, 10, None, kw, torch.full_like(kept, -1), k_scale=None if ks is None else ks.clone(),
                            v_scale=None if vs is None else vs.clone())
    rc = shim.sas_evict(_p(w), T, _p(kp), _p(vp), _p(ks), _p(vs), _p(bt), _p(lens), 3, 2, 128, c.num_blocks, c.max_blocks, c.kv,
                        50, 2, 10, _p(kept), _p(n), None, 0, _p(w), _stream())
    assert rc == 0, shim.sas_last_error()
    torch.cuda.synchronize()
    assert torch.equal(a, kept) and torch.equal(an, n) and torch.equal(kw, w)
    assert torch.equal(kc, kp) and torch.equal(vc, vp)


@pytest.mark.gpu
@pytest.mark.parametrize("paged", [True, False])
def test_prefill(ff, gpu, shim, paged):
    c = make(5, [0, 0] if not paged else [2100, 30], 70, 6, 2, 128, "f16", "f16")
    r = masked(c, rule_of(c), "documents")
    kp, vp, _, _, bt, cx, kn, vn, q = su.device(c, gpu)
    begin = torch.from_numpy(r["begin"]).to(gpu)
    out = torch.empty(2, 70, 6 * 128, dtype=q.dtype, device=gpu)
    k, v, t, x = (kp, vp, bt, cx) if paged else (kn, vn, None, None)
    want = ff.paged_prefill_scored(q, k, v, t, x, score_cap=4.0, window=50, key_begin=begin)
    rc = shim.sas_attention(_p(q), _p(k), _p(v), None, None, _p(out), _p(t), _p(x), 2, 70, 6, 2, 128, c.num_blocks, c.max_blocks,
                            c.act, c.kv, 4.0, None, 50, _p(begin), None, None, None, 1.0, 0, _stream())
    assert rc == 0, shim.sas_last_error()
    assert torch.equal(want, out)


@pytest.mark.gpu
def test_errors(ff, gpu, shim):
    x = torch.zeros(1, device=gpu)
    p = _p(x)
    a = dict(q=p, k=p, v=p, ks=None, vs=None, out=p, table=p, ctx=p, B=1, S=1, Hq=4, Hkv=2, D=64, N=4, mb=2, qd=2, cd=2, cap=0.0,
             slopes=None, window=0, begin=None, end=None, weights=None, prior=None, decay=1.0, T=0, stream=None)
    for kw, what in ((dict(cap=-1.0), b"score_cap"), (dict(window=-1), b"window"), (dict(end=p), b"key_end"),
                     (dict(prior=p), b"prior"), (dict(S=3, weights=p, T=8), b"weights"), (dict(cd=3), b"k_scale")):
        assert shim.sas_attention(*{**a, **kw}.values()) == -1
        assert what in shim.sas_last_error()
