"""A prompt's chunks through the C++ API of scored attention (include/firefly/kernels.h), down to one token under a mask, and
decode steps with their append, against the Python calls: the same bits."""

import ctypes
import os
from pathlib import Path

import numpy as np
import pytest
import torch

import scored_util as su
from test_gpu_scored_prefill import make

SHIM = Path(__file__).resolve().parent / "cpp" / "libscored_prompt_shim.so"


@pytest.fixture(scope="module")
def shim(ff):
    lib = ctypes.CDLL(str(SHIM), mode=os.RTLD_NOW)
    vp, i, f = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
    lib.sps_attention.argtypes = [vp] * 6 + [i] * 8 + [f, i, vp, vp, i, vp]
    lib.sps_step.argtypes = [vp] * 8 + [i] * 10 + [vp] * 4 + [i, i, vp]
    lib.sps_last_error.restype = ctypes.c_char_p
    return lib


def _p(t):
    return None if t is None else t.data_ptr()


def test_decode_has_no_key_end(shim):
    a = [16] * 6 + [1, 1, 4, 2, 64, 4, 2, 2, 0.0, 0, None, 16, 0, None]
    assert shim.sps_attention(*a) == -1
    assert b"key_end" in shim.sps_last_error() and b"prefill" in shim.sps_last_error()
    a[6], a[18] = 0, 1
    assert shim.sps_attention(*a) == 0 and shim.sps_last_error() == b""  # no rows


@pytest.mark.parametrize("op", range(7))
@pytest.mark.parametrize("block", [8, 32])
def test_block_size(shim, op, block):
    """Caches whose pages are not of 16 tokens would be read past their end."""
    assert shim.sps_block_size(op, block, 1) == -1
    assert b"num_blocks, 16, " in shim.sps_last_error()
    assert shim.sps_block_size(op, 16, 0) == 0 and shim.sps_last_error() == b""


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 2, 33])
@pytest.mark.parametrize("ends", [False, True])
def test_chunks(ff, gpu, shim, S, ends):
    """Chunks of a document's tokens that see a range of keys, or nothing (padding)."""
    c = make(7, [700, 40, 0, 130], S, 8, 2, 128, "bf16", "bf16")
    kp, vp, _, _, bt, cx, _, _, q = su.device(c, gpu)
    pos = np.array([700, 40, 0, 130], np.int32)[:, None] + np.arange(S, dtype=np.int32)
    begin = torch.from_numpy(np.maximum(pos - 50, 0).astype(np.int32)).to(gpu)
    last = (pos + 1).astype(np.int32)
    last[0], last[1] = 690, 0
    end = torch.from_numpy(last).to(gpu) if ends else None
    want = ff.paged_prefill_scored(q, kp, vp, bt, cx, 7.0, None, 600, begin, end)
    out = torch.full_like(want, float("nan"))
    rc = shim.sps_attention(_p(q), _p(kp), _p(vp), _p(out), _p(bt), _p(cx), 4, S, 8, 2, 128, c.num_blocks, c.max_blocks, c.act, 7.0,
                            600, _p(begin), _p(end), 1, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, shim.sps_last_error()
    assert torch.equal(want, out)
    assert not ends or not out[1].float().any()


def test_new_tokens_refused(shim):
    a = [256] * 3 + [None, None] + [256] * 3 + [0, 1, 4, 2, 64, 4, 2, 2, 2, 0, 256, 256, None, None, 0, 0, None]
    assert shim.sps_step(*a) == 0 and shim.sps_last_error() == b""  # no rows
    for at, value in ((19, None), (18, None), (9, 2), (23, 1)):  # half a pair, two tokens a row, a prompt's chunk
        b = list(a)
        b[at] = value
        assert shim.sps_step(*b) == -1
        assert b"k_new" in shim.sps_last_error()
    assert shim.sps_step(*a) == 0 and shim.sps_last_error() == b""


@pytest.mark.gpu
@pytest.mark.parametrize("act,kv,D", [("bf16", "bf16", 128), ("bf16", "i8", 128), ("f16", "f16", 72), ("f32", "f32", 64)])
@pytest.mark.parametrize("ctx", [[0, 31, 200], [5000, 9, 777]])
def test_step_with_append(ff, gpu, shim, act, kv, D, ctx):
    c = make(9, ctx, 1, 8, 2, D, act, kv)
    a, b = su.device(c, gpu), su.device(c, gpu)
    T = 16 * c.max_blocks
    prior = torch.rand(3, 2, T, device=gpu)
    w, w2 = torch.zeros_like(prior), torch.zeros_like(prior)
    want = ff.paged_attention_scored(a[8], *a[:2], a[4], a[5], window=600, k_new=a[6], v_new=a[7], weights=w, prior=prior, decay=0.5,
                                     k_scale=a[2], v_scale=a[3], max_context_len=T)
    out = torch.full_like(want, float("nan"))
    rc = shim.sps_step(_p(b[8]), *map(_p, b[:4]), _p(out), _p(b[4]), _p(b[5]), 3, 1, 8, 2, D, c.num_blocks, c.max_blocks, c.act, c.kv,
                       600, _p(b[6]), _p(b[7]), _p(w2), _p(prior), T, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, shim.sps_last_error()
    assert torch.equal(want, out) and torch.equal(w, w2)
    for x, y in zip(a[:4], b[:4]):
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
