"""A prompt's chunks through the C++ API of scored attention (include/firefly/kernels.h), down to one token under a mask,
against the Python calls: the same bits."""

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
