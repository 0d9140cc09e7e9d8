"""What rotary positions on several axes, key bounds, the choice of pages and the attention over them refuse, without a GPU: the
C ABI's status codes before a device is touched, and the Python front end's checks of its tensors."""

import ctypes

import pytest
import torch

NAN, INF = float("nan"), float("inf")
HKV, D = 2, 64


def _ints(*v):
    return (ctypes.c_int * len(v))(*v)


def _call(fn, a, kw):
    assert set(kw) <= set(a), set(kw) - set(a)
    a.update(kw)
    return fn(*a.values())


def _rope(ff, **kw):
    return _call(ff.lib.ffkv_rope_axes, dict(
        q=16, q_stride=0, q_out=16, q_out_stride=0, k=16, k_stride=0, k_out=16, k_out_stride=0, dtype=ff.DTYPE_BF16,
        positions=16, sections=_ints(16, 24, 24), axes=3, interleaved=0, batch=1, seq_len=1, num_heads=8, num_kv_heads=2,
        head_dim=128, rope_theta=1e6, stream=None), kw)


def _append(ff, **kw):
    return _call(ff.lib.ffkv_rope_append_axes, dict(
        q=16, q_stride=0, q_out=16, q_out_stride=0, k=16, k_stride=0, v=16, v_stride=0, src_dtype=ff.DTYPE_BF16, k_cache=16,
        v_cache=16, cache_dtype=ff.DTYPE_BF16, k_scale=None, v_scale=None, block_table=16, context_lens=16, positions=16,
        sections=_ints(16, 24, 24), axes=3, interleaved=0, batch=1, seq_len=1, num_heads=8, num_kv_heads=2, head_dim=128,
        block_size=16, max_blocks=4, num_blocks=4, rope_theta=1e6, stream=None), kw)


def _bounds(ff, **kw):
    return _call(ff.lib.ffkv_key_bounds, dict(
        k_cache=16, cache_dtype=ff.DTYPE_BF16, k_scale=None, bounds=16, block_table=16, context_lens=16, batch=1, new_tokens=1,
        num_kv_heads=2, head_dim=128, block_size=16, max_blocks=4, num_blocks=4, stream=None), kw)


def _select(ff, **kw):
    return _call(ff.lib.ffkv_select_blocks, dict(
        q=16, q_dtype=ff.DTYPE_BF16, bounds=16, bounds_dtype=ff.DTYPE_BF16, block_table=16, context_lens=16, blocks=16, count=4,
        sinks=1, recent=1, query_block=1, batch=1, seq_len=1, num_heads=8, num_kv_heads=2, head_dim=128, block_size=16,
        max_blocks=64, num_blocks=4, max_context_len=0, workspace=None, workspace_bytes=0, stream=None), kw)


def _attend(ff, **kw):
    return _call(ff.lib.ffkv_paged_attention_blocks, dict(
        q=16, out=16, qo_dtype=ff.DTYPE_BF16, k_cache=16, v_cache=16, cache_dtype=ff.DTYPE_BF16, k_scale=None, v_scale=None,
        block_table=16, context_lens=16, blocks=16, count=64, query_block=1, batch=1, seq_len=1, num_heads=8, num_kv_heads=2,
        head_dim=128, block_size=16, max_blocks=64, num_blocks=4, scale=0.0, workspace=None, workspace_bytes=0, stream=None), kw)


AXES = [
    (dict(head_dim=96, sections=_ints(16, 16, 16)), -2), (dict(num_kv_heads=0), -1), (dict(batch=-1), -1),
    (dict(seq_len=-1), -1), (dict(rope_theta=0.0), -1), (dict(rope_theta=NAN), -1), (dict(rope_theta=INF), -1),
    (dict(axes=0), -1), (dict(axes=5, sections=_ints(16, 16, 16, 8, 8)), -1), (dict(sections=None), -1),
    (dict(sections=_ints(16, 24, 23)), -1), (dict(sections=_ints(-8, 48, 24)), -1),
    (dict(sections=_ints(1 << 30, 1 << 30, 64)), -1), (dict(sections=_ints(16, 24, 24), interleaved=1), -1),
    (dict(sections=_ints(0, 0, 64), interleaved=1), -1), (dict(q_stride=8 * 128 - 8), -1), (dict(q_stride=8 * 128 + 4), -1),
    (dict(k_stride=128), -1), (dict(k_stride=-256), -1), (dict(q_out_stride=8 * 128 + 2), -1), (dict(positions=None), -1),
    (dict(k=None), -1), (dict(q_out=None), -1), (dict(q=24), -1), (dict(k=20), -1), (dict(q_out=8), -1),
    (dict(positions=18), -1), (dict(q_stride=2048), -1), (dict(num_heads=70000), -2), (dict(batch=2 ** 15, seq_len=2 ** 14), -2),
]


@pytest.mark.parametrize("kw,code", AXES + [(dict(dtype=3), -2), (dict(k_out=None), -1), (dict(k_out_stride=8), -1),
                                            (dict(k_stride=512), -1)])
def test_rope_rejects(ff, kw, code):
    assert _rope(ff, **kw) == code and ff.lib.ffkv_last_error() != b""


@pytest.mark.parametrize("kw,code", AXES + [
    (dict(src_dtype=3), -2), (dict(cache_dtype=7), -2), (dict(block_size=8), -2), (dict(v=None), -1), (dict(v=24), -1),
    (dict(k_cache=None), -1), (dict(v_cache=None), -1), (dict(k_cache=None, v_cache=None), -1), (dict(block_table=None), -1),
    (dict(cache_dtype=3), -1), (dict(cache_dtype=8, k_scale=16), -1), (dict(v_stride=8), -1), (dict(v_stride=260), -1),
    (dict(max_blocks=-1), -1), (dict(num_blocks=-1), -1)])
def test_rope_append_rejects(ff, kw, code):
    assert _append(ff, **kw) == code and ff.lib.ffkv_last_error() != b""


@pytest.mark.parametrize("kw,code", [
    (dict(block_size=32), -2), (dict(cache_dtype=7), -2), (dict(head_dim=136), -2), (dict(head_dim=12), -2),
    (dict(batch=-1), -1), (dict(new_tokens=-1), -1), (dict(num_kv_heads=0), -1), (dict(batch=65536), -2),
    (dict(k_cache=None), -1), (dict(bounds=None), -1), (dict(block_table=None), -1), (dict(context_lens=None), -1),
    (dict(cache_dtype=3), -1), (dict(cache_dtype=8), -1), (dict(bounds=8), -1), (dict(k_cache=4), -1)])
def test_bounds_rejects(ff, kw, code):
    assert _bounds(ff, **kw) == code and ff.lib.ffkv_last_error() != b""


@pytest.mark.parametrize("kw,code", [
    (dict(block_size=8), -2), (dict(q_dtype=3), -2), (dict(bounds_dtype=3), -2), (dict(head_dim=20), -2),
    (dict(num_heads=7), -1), (dict(num_heads=0), -1), (dict(batch=-1), -1), (dict(batch=65536), -2), (dict(query_block=0), -1),
    (dict(count=0), -1), (dict(sinks=-1), -1), (dict(recent=-1), -1), (dict(sinks=3, recent=2), -1),
    (dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), -1), (dict(q=None), -1), (dict(bounds=None), -1), (dict(blocks=None), -1),
    (dict(context_lens=None), -1), (dict(q=8), -1), (dict(bounds=8), -1), (dict(blocks=18), -1), (dict(workspace=8), -1),
    (dict(workspace=16, workspace_bytes=2 * 6000 * 4 - 1, max_blocks=6000), -3),
    (dict(seq_len=2 ** 31 - 1, batch=60000, num_heads=60000, num_kv_heads=60000), -2),
    (dict(seq_len=2 ** 31 - 1, query_block=2 ** 31 - 1, num_heads=64, num_kv_heads=1), -2),
    (dict(seq_len=2 ** 20, max_blocks=2 ** 26), -2), (dict(count=2 ** 26 + 1), -2), (dict(count=2 ** 31 - 1), -2),
    (dict(num_blocks=0), -1)])
def test_select_rejects(ff, kw, code):
    assert _select(ff, **kw) == code and ff.lib.ffkv_last_error() != b""


@pytest.mark.parametrize("kw,code", [
    (dict(block_size=8), -2), (dict(qo_dtype=3), -2), (dict(cache_dtype=7), -2), (dict(head_dim=130), -2),
    (dict(num_heads=7), -1), (dict(num_kv_heads=0), -1), (dict(batch=-1), -1), (dict(seq_len=-1), -1), (dict(batch=65536), -2),
    (dict(count=0), -1), (dict(query_block=0), -1), (dict(query_block=-4), -1), (dict(q=None), -1), (dict(out=None), -1),
    (dict(v_cache=None), -1), (dict(blocks=None), -1), (dict(context_lens=None), -1), (dict(cache_dtype=3), -1),
    (dict(cache_dtype=8, v_scale=16), -1), (dict(q=8), -1), (dict(out=4), -1), (dict(blocks=18), -1), (dict(workspace=8), -1),
    (dict(workspace=16, workspace_bytes=16, count=256), -3), (dict(seq_len=2 ** 31 - 1), -2),
    (dict(count=2 ** 26 + 1), -2), (dict(count=2 ** 31 - 1, query_block=2, seq_len=2), -2)])
def test_attention_rejects(ff, kw, code):
    assert _attend(ff, **kw) == code and ff.lib.ffkv_last_error() != b""


def test_empty_is_ok(ff):
    none = dict(batch=0)
    assert _rope(ff, q=None, k=None, positions=None, **none) == 0 and _append(ff, k=None, seq_len=0) == 0
    assert _bounds(ff, k_cache=None, **none) == 0 and _bounds(ff, k_cache=None, new_tokens=0) == 0
    assert _select(ff, q=None, **none) == 0 and _select(ff, q=None, seq_len=0) == 0
    assert _attend(ff, q=None, **none) == 0 and _attend(ff, q=None, seq_len=0) == 0
    assert ff.lib.ffkv_last_error() == b""


def test_workspace_bytes(ff):
    f = ff.lib.ffkv_select_blocks_workspace_bytes
    lists = 2 * 4 * 4
    assert f(2, 100, 8, 4, 64, 8, 32, 5000, 0) == lists * (5000 * 4 + 64 * 16)
    assert f(2, 100, 8, 4, 64, 8, 32, 5000, 4000 * 16) == lists * (4000 * 4 + 64 * 16)
    assert f(2, 1, 8, 4, 64, 8, 1, 2000, 0) == 8 * 2000 * 4  # a step's queries are summed where they are used
    assert f(2, 100, 8, 4, 64, 8, 32, 50, 0) == 0 and f(2, 1, 8, 4, 64, 8, 1, 64, 0) == 0  # few pages: no scores are written
    assert f(2, 100, 8, 4, 64, 50, 32, 50, 0) == 0 and f(2, 100, 8, 4, 64, 19, 32, 50, 300) == 0
    assert f(0, 1, 1, 1, 64, 1, 1, 9, 0) == 0 and f(1, 1, 1, 1, 64, 0, 1, 9, 0) == 0 and f(1, 1, 1, 1, 64, 1, 0, 9, 0) == 0
    g = ff.lib.ffkv_paged_attention_blocks_workspace_bytes
    assert g(ff.DTYPE_BF16, ff.DTYPE_BF16, 64, 1, 32, 8, 128, 64, 1) == 0  # enough lists for the chip
    assert g(ff.DTYPE_BF16, ff.DTYPE_BF16, 1, 1, 32, 8, 128, 256, 1) > 0
    assert g(ff.DTYPE_BF16, ff.DTYPE_BF16, 1, 1, 32, 8, 128, 256, 64) == g(ff.DTYPE_BF16, ff.DTYPE_BF16, 1, 1, 32, 8, 128, 256, 1)  # one token, one list
    assert g(ff.DTYPE_BF16, ff.DTYPE_FP8_E4M3, 1, 64, 32, 8, 128, 256, 64) > 0  # a chunk of few lists is split too
    assert g(ff.DTYPE_BF16, ff.DTYPE_BF16, 8, 1024, 32, 8, 128, 256, 64) == 0 and g(3, 2, 1, 1, 32, 8, 128, 256, 1) == 0
    assert g(ff.DTYPE_BF16, 7, 1, 1, 32, 8, 128, 256, 1) == 0 and g(ff.DTYPE_BF16, ff.DTYPE_BF16, 1, 1, 30, 8, 128, 256, 1) == 0


# ---- the Python front end's checks (calls without rows touch no GPU) -------------------------------------------------


def _raises(fn, bad):
    for error, kw in bad:
        with pytest.raises(error):
            fn(**kw)


def test_rope_front(ff):
    bf = torch.bfloat16
    packed = torch.zeros(0, 3, 8, D, dtype=bf)
    t = dict(q=packed[:, :, :4], k=packed[:, :, 4:6], positions=torch.zeros(2, 0, 3, dtype=torch.int32), sections=(20, 12),
             stream=0)
    ff.apply_rope_axes(**t)
    ff.apply_rope_axes(**dict(t, q=None))
    ff.apply_rope_axes(**dict(t, sections=[20, 12], interleaved=True, theta=1e4))
    bad = [
        (ValueError, dict(t, sections=())), (ValueError, dict(t, sections=(8, 8, 8, 4, 4))), (TypeError, dict(t, sections=5)),
        (TypeError, dict(t, sections=(20.0, 12))), (ValueError, dict(t, sections=(16, 8, 8))),
        (TypeError, dict(t, positions=t["positions"].long())), (ValueError, dict(t, positions=t["positions"][:1])),
        (TypeError, dict(t, positions=None)), (TypeError, dict(t, q=t["q"].half())), (ValueError, dict(t, q=t["q"][:, :2])),
        (ValueError, dict(t, q=t["q"][..., :32])), (TypeError, dict(t, k_out=t["k"].float())),
        (ValueError, dict(t, q_out=t["q"][:, :, :2])), (ff.FFKVError, dict(t, sections=(20, 11))),
        (ValueError, dict(t, k=torch.zeros(0, 3, D, dtype=bf))),
    ]
    _raises(ff.apply_rope_axes, bad)
    pool = torch.zeros(4, 16, 2, D, dtype=bf)
    a = dict(t, v=packed[:, :, 6:], k_cache=pool, v_cache=pool.clone(), block_table=torch.zeros(0, 3, dtype=torch.int32),
             context_lens=torch.zeros(0, dtype=torch.int32))
    ff.rope_append_axes(**a)
    ff.rope_append_axes(**dict(a, context_lens=None, q=None))
    _raises(ff.rope_append_axes, [
        (TypeError, dict(a, v=a["v"].half())), (ValueError, dict(a, v=a["v"][:, :, :1])),
        (ValueError, dict(a, k_cache=pool[:, :8])), (TypeError, dict(a, v_cache=pool.half())),
        (ValueError, dict(a, v_cache=pool[:2])), (ValueError, dict(a, num_blocks=5)),
        (TypeError, dict(a, block_table=a["block_table"].long())), (ValueError, dict(a, context_lens=torch.zeros(1, dtype=torch.int32))),
    ])
    # rows that are there, on the CPU: their layout is looked at first
    x = torch.zeros(2, 3, 8, D, dtype=bf)
    g = dict(q=x[:, :, :4], k=x[:, :, 4:6], positions=torch.zeros(2, 2, 3, dtype=torch.int32), sections=(20, 12), stream=0)
    _raises(ff.apply_rope_axes, [
        (ValueError, g), (ValueError, dict(g, q=x.transpose(1, 2).contiguous().transpose(1, 2)[:, :, :4])),
        (ValueError, dict(g, q=torch.zeros(2, 3, 4, 2 * D, dtype=bf)[..., ::2])),
        (ValueError, dict(g, k=torch.zeros(2, 6, 2, D, dtype=bf)[:, :3])), (ValueError, dict(g, k=x[:, :, 0:4:2])),
        (ValueError, dict(g, q=torch.zeros(1, 1, 4, D, dtype=bf).expand(2, 3, 4, D))),
    ])


def test_bounds_front(ff):
    pool = torch.zeros(4, 16, HKV, D, dtype=torch.bfloat16)
    t = dict(k_cache=pool, bounds=ff.key_bounds(pool), block_table=torch.zeros(0, 3, dtype=torch.int32),
             context_lens=torch.zeros(0, dtype=torch.int32), new_tokens=2, stream=0)
    ff.update_key_bounds(**t)
    i8 = pool.to(torch.int8)
    assert ff.key_bounds(i8).dtype == torch.bfloat16 and ff.key_bounds(pool.float()).dtype == torch.float32
    ff.update_key_bounds(**dict(t, k_cache=i8, k_scale=torch.zeros(4, 16, HKV)))
    _raises(ff.update_key_bounds, [
        (TypeError, dict(t, bounds=t["bounds"].half())), (ValueError, dict(t, bounds=t["bounds"][:3])),
        (ValueError, dict(t, bounds=t["bounds"].transpose(1, 2))), (TypeError, dict(t, new_tokens=2.0)),
        (ff.FFKVError, dict(t, new_tokens=-1)), (ValueError, dict(t, k_cache=pool[:, :8])),
        (TypeError, dict(t, block_table=t["block_table"].float())), (ValueError, dict(t, block_table=torch.zeros(2, 3, dtype=torch.int32))),
        (ValueError, dict(t, num_blocks=5)), (TypeError, dict(t, k_cache=i8, bounds=i8)),
        (ValueError, dict(t, k_cache=i8, k_scale=torch.zeros(4, 16))),
        (ValueError, dict(t, context_lens=torch.zeros(1, dtype=torch.int32), block_table=torch.zeros(1, 3, dtype=torch.int32))),
    ])


def test_select_front(ff):
    box = torch.zeros(4, HKV, 2, D, dtype=torch.bfloat16)
    t = dict(q=torch.zeros(0, 5, 4, D, dtype=torch.bfloat16), bounds=box, block_table=torch.zeros(0, 9, dtype=torch.int32),
             context_lens=torch.zeros(0, dtype=torch.int32), count=3, query_block=2, stream=0)
    assert ff.select_blocks(**t).shape == (0, 3, HKV, 3)
    _raises(ff.select_blocks, [
        (ff.FFKVError, dict(t, count=0)), (ff.FFKVError, dict(t, query_block=0)), (ff.FFKVError, dict(t, sinks=2, recent=2)),
        (TypeError, dict(t, sinks=1.0)), (ValueError, dict(t, blocks=torch.zeros(0, 5, HKV, 3, dtype=torch.int32))),
        (TypeError, dict(t, blocks=torch.zeros(0, 3, HKV, 3))), (ValueError, dict(t, bounds=box[..., :32])),
        (ValueError, dict(t, bounds=box[:, :, :1])), (TypeError, dict(t, bounds=box.to(torch.int32))),
        (ValueError, dict(t, q=t["q"][:, 0])), (ValueError, dict(t, num_blocks=5)), (OverflowError, dict(t, count=2 ** 31)),
        (TypeError, dict(t, context_lens=t["context_lens"].long())),
    ])


def test_attention_front(ff):
    pool = torch.zeros(4, 16, HKV, D, dtype=torch.bfloat16)
    t = dict(q=torch.zeros(0, 5, 4, D, dtype=torch.bfloat16), k_cache=pool, v_cache=pool.clone(),
             block_table=torch.zeros(0, 9, dtype=torch.int32), context_lens=torch.zeros(0, dtype=torch.int32),
             blocks=torch.zeros(0, 3, HKV, 7, dtype=torch.int32), query_block=2, stream=0)
    assert ff.paged_attention_blocks(**t).shape == (0, 5, 4 * D)
    step = dict(t, q=t["q"][:, 0], query_block=1, blocks=torch.zeros(0, 1, HKV, 7, dtype=torch.int32))
    assert ff.paged_attention_blocks(**step).shape == (0, 1, 4 * D)
    _raises(ff.paged_attention_blocks, [
        (ValueError, dict(t, query_block=1)), (ff.FFKVError, dict(t, query_block=0)), (ff.FFKVError, dict(t, blocks=t["blocks"][..., :0].contiguous())),
        (TypeError, dict(t, blocks=t["blocks"].long())), (ValueError, dict(t, blocks=t["blocks"][:, :2])),
        (ValueError, dict(t, v_cache=pool[:2])), (TypeError, dict(t, v_cache=pool.half())),
        (ValueError, dict(t, q=torch.zeros(0, 1, 5, 4, D, dtype=torch.bfloat16))), (TypeError, dict(t, out=torch.zeros(0, 5, 4 * D))),
        (ValueError, dict(t, out=torch.zeros(1, 5, 4 * D, dtype=torch.bfloat16))), (ValueError, dict(t, num_blocks=5)),
        (ValueError, dict(t, q=torch.zeros(1, 5, 4, 2 * D, dtype=torch.bfloat16)[..., ::2])),  # (without rows all is contiguous)
        (ValueError, dict(step, q=torch.zeros(1, 4, D, dtype=torch.bfloat16))),
    ])
