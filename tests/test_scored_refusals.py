"""What the scored operators refuse, without a GPU: the C ABI's status codes before a device is touched, and the Python
front end's checks of its tensors."""

import ctypes

import pytest
import torch

HKV, D = 2, 64
NAN, INF = float("nan"), float("inf")


def _decode(ff, **kw):
    a = dict(q=16, out=16, qo_dtype=ff.DTYPE_BF16, k_cache=16, v_cache=16, cache_dtype=ff.DTYPE_BF16, k_scale=None,
             v_scale=None, block_table=16, context_lens=16, batch=1, num_heads=32, num_kv_heads=8, head_dim=128,
             block_size=16, max_blocks=4, num_blocks=4, max_context_len=0, scale=0.0, score_cap=0.0, slopes=None, window=0,
             key_begin=None, k_new=None, v_new=None, src_dtype=ff.DTYPE_BF16, weights=None, prior=None, decay=1.0,
             weight_stride=0, workspace=None, workspace_bytes=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return ff.lib.ffkv_paged_decode_scored(*a.values())


DECODE = [
    (dict(block_size=8), -2), (dict(head_dim=84), -2), (dict(head_dim=144), -2), (dict(qo_dtype=3), -2),
    (dict(cache_dtype=7), -2), (dict(num_heads=30), -1), (dict(num_heads=0), -1), (dict(max_blocks=-1), -1),
    (dict(num_heads=8 * 17, cache_dtype=0), -2), (dict(num_heads=8 * 17, head_dim=72), -2), (dict(batch=70000), -2),
    (dict(context_lens=None), -1), (dict(q=None), -1), (dict(cache_dtype=3), -1), (dict(q=20), -1), (dict(k_new=16), -1),
    (dict(v_new=16), -1), (dict(k_new=24, v_new=16), -1), (dict(k_new=16, v_new=16, src_dtype=3), -2),
    (dict(score_cap=-1.0), -1), (dict(score_cap=NAN), -1), (dict(score_cap=INF), -1), (dict(window=-1), -1),
    (dict(slopes=18), -1), (dict(key_begin=17), -1),
    (dict(prior=16), -1), (dict(weights=16, weight_stride=63), -1), (dict(weights=16, weight_stride=64, decay=-0.5), -1),
    (dict(weights=16, weight_stride=64, decay=NAN), -1), (dict(weights=18, weight_stride=64), -1),
    (dict(weights=16, weight_stride=64, prior=18), -1),
    (dict(workspace=24, workspace_bytes=1 << 30), -1), (dict(workspace=256, workspace_bytes=64, max_blocks=6000), -3),
    (dict(weights=16, weight_stride=1 << 30, max_blocks=1 << 26, batch=31, num_heads=65528), -2),
]


@pytest.mark.parametrize("kw,code", DECODE)
def test_decode_rejects(ff, kw, code):
    assert _decode(ff, **kw) == code
    assert ff.lib.ffkv_last_error().decode() != ""


def test_empty_is_ok(ff):
    assert _decode(ff, batch=0, q=None) == 0 and ff.lib.ffkv_last_error() == b""


def test_decode_workspace_bytes(ff):
    f = ff.lib.ffkv_decode_scored_workspace_bytes
    plain = ff.decode_workspace_bytes(4, 32, 128, 600)
    assert f(4, 32, 128, 600, 0, 0) == plain
    assert f(4, 32, 128, 600, 0, 1) >= plain + 4 * 32 * 9600 * 4
    assert f(4, 32, 128, 600, 100, 1) < f(4, 32, 128, 600, 0, 1)
    g = ff.lib.ffkv_decode_scored_scratch_bytes
    for types in ((ff.DTYPE_BF16, ff.DTYPE_BF16), (ff.DTYPE_F32, ff.DTYPE_F32), (ff.DTYPE_BF16, ff.DTYPE_I8)):
        for B, Hq, Hkv, D, mb, window in ((4, 32, 8, 128, 600, 0), (4, 32, 8, 128, 600, 100), (70, 8, 8, 64, 33, 0),
                                          (1, 16, 1, 256, 9000, 0), (3, 4, 2, 72, 700, 50)):
            for w in (0, 1):
                assert g(*types, B, Hq, Hkv, D, mb, 0, window, w) <= f(B, Hq, D, mb, 0, w)
    assert g(ff.DTYPE_BF16, ff.DTYPE_BF16, 2, 8, 8, 128, 8, 0, 0, 0) == 0  # one launch, no partials
    assert g(ff.DTYPE_BF16, ff.DTYPE_BF16, 2, 8, 3, 128, 8, 0, 0, 1) == 0 and g(3, 2, 2, 8, 8, 128, 8, 0, 0, 1) == 0
    assert f(0, 32, 128, 600, 0, 1) == 0 and f(65535, 65535, 128, 1 << 26, 0, 1) == 0


def _tensors(B=0, dtype=torch.bfloat16, Hq=4, cache=None):
    pool = torch.zeros(4, 16, HKV, D, dtype=cache or dtype)
    return dict(q=torch.zeros(B, 1, Hq, D, dtype=dtype), k_cache=pool, v_cache=pool.clone(),
                block_table=torch.zeros(B, 3, dtype=torch.int32), context_lens=torch.zeros(B, dtype=torch.int32))


def test_decode_front(ff):
    t = _tensors()
    w = torch.zeros(0, HKV, 48)
    k = torch.zeros(0, 1, HKV, D, dtype=torch.bfloat16)
    out = ff.paged_attention_scored(**t, score_cap=5, slopes=torch.zeros(4), window=3, weights=w, prior=w,
                                    key_begin=torch.zeros(0, dtype=torch.int32), k_new=k, v_new=k, stream=0)
    assert out.shape == (0, 1, 4 * D)
    i8 = _tensors(cache=torch.int8)
    s = torch.zeros(4, 16, HKV)
    ff.paged_attention_scored(**i8, k_scale=s, v_scale=s, stream=0)
    bad = [
        (ValueError, dict(t, q=torch.zeros(0, 2, 4, D, dtype=torch.bfloat16))),
        (TypeError, dict(t, block_table=t["block_table"].long())),
        (ValueError, dict(t, block_table=torch.zeros(1, 3, dtype=torch.int32))),
        (ValueError, dict(t, context_lens=torch.zeros(2, dtype=torch.int32))),
        (TypeError, dict(t, context_lens=t["context_lens"].float())),
        (ValueError, dict(t, v_cache=t["v_cache"][:2])),
        (ValueError, dict(t, k_cache=t["k_cache"][:, :8])),
        (ValueError, dict(t, k_cache=torch.zeros(4, 16, HKV, 2 * D, dtype=torch.bfloat16)[..., ::2])),
        (TypeError, dict(t, v_cache=t["v_cache"].half())),
        (ValueError, dict(t, slopes=torch.zeros(3))),
        (TypeError, dict(t, slopes=torch.zeros(4).double())),
        (ValueError, dict(t, key_begin=torch.zeros(1, dtype=torch.int32))),
        (ValueError, dict(t, weights=torch.zeros(0, HKV + 1, 48))),
        (ValueError, dict(t, weights=w, prior=torch.zeros(0, HKV, 47))),
        (TypeError, dict(t, weights=w.half())),
        (TypeError, dict(t, k_new=k, v_new=k.half())),
        (ValueError, dict(t, k_new=k[..., :32], v_new=k[..., :32])),
        (ValueError, dict(t, k_new=k)),
        (ValueError, dict(t, v_new=k)),
        (ValueError, dict(t, prior=w)),
        (TypeError, dict(t, window=2.0)),
        (TypeError, dict(t, out=torch.zeros(0, 1, 4 * D))),
        (ValueError, dict(t, out=torch.zeros(1, 1, 4 * D, dtype=torch.bfloat16))),
        (ValueError, dict(t, num_blocks=5)),
        (ValueError, dict(i8, k_scale=s[:2], v_scale=s)),
        (TypeError, dict(i8, k_scale=s.half(), v_scale=s)),
        (TypeError, dict(t, k_cache=torch.zeros(4, 16, HKV, D, dtype=torch.int32))),
        (ValueError, dict(t, slopes=torch.zeros(4, device="meta"))),
    ]
    for error, kw in bad:
        with pytest.raises(error):
            ff.paged_attention_scored(**kw, stream=0)
    with pytest.raises(ValueError, match="GPU"):
        ff.paged_attention_scored(**_tensors(B=1), stream=0)


def _prefill(ff, **kw):
    a = dict(q=16, out=16, qo_dtype=ff.DTYPE_BF16, k_cache=16, v_cache=16, cache_dtype=ff.DTYPE_BF16, k_scale=None,
             v_scale=None, block_table=16, context_lens=16, batch=1, seq_len=4, num_heads=32, num_kv_heads=8, head_dim=128,
             block_size=16, max_blocks=4, num_blocks=4, max_context_len=0, scale=0.0, score_cap=0.0, slopes=None, window=0,
             key_begin=None, key_end=None, workspace=None, workspace_bytes=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return ff.lib.ffkv_paged_prefill_scored(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(block_size=8), -2), (dict(head_dim=96), -2), (dict(qo_dtype=8), -2), (dict(cache_dtype=0), -2),
    (dict(cache_dtype=4), -2), (dict(num_heads=30), -1), (dict(batch=-1), -1), (dict(seq_len=-1), -1), (dict(batch=70000), -2),
    (dict(seq_len=1 << 30), -2), (dict(context_lens=None), -1), (dict(out=None), -1), (dict(cache_dtype=3), -1),
    (dict(cache_dtype=3, block_table=None, k_scale=16, v_scale=16), -2), (dict(k_cache=24), -1), (dict(workspace=8), -1),
    (dict(score_cap=-2.0), -1), (dict(score_cap=NAN), -1), (dict(window=-5), -1), (dict(slopes=2), -1),
    (dict(key_begin=6), -1), (dict(key_end=7), -1),
])
def test_prefill_rejects(ff, kw, code):
    assert _prefill(ff, **kw) == code
    assert ff.lib.ffkv_last_error().decode() != ""
    assert _prefill(ff, seq_len=0, q=None) == 0


def test_prefill_front(ff):
    t = _tensors()
    q = torch.zeros(0, 5, 4, D, dtype=torch.bfloat16)
    r = torch.zeros(0, 5, dtype=torch.int32)
    t["q"] = q
    assert ff.paged_prefill_scored(**t, key_begin=r, key_end=r, slopes=torch.zeros(4), stream=0).shape == (0, 5, 4 * D)
    k = torch.zeros(0, 5, HKV, D, dtype=torch.bfloat16)
    assert ff.paged_prefill_scored(q, k, k, None, None, window=2, stream=0).shape == (0, 5, 4 * D)
    bad = [
        (ValueError, dict(t, q=q[:, 0])), (ValueError, dict(t, key_begin=r[:, :4])), (TypeError, dict(t, key_end=r.long())),
        (TypeError, dict(t, block_table=t["block_table"].long())), (ValueError, dict(t, context_lens=torch.zeros(1, dtype=torch.int32))),
        (ValueError, dict(t, v_cache=t["v_cache"][:1])), (ValueError, dict(t, slopes=torch.zeros(5))),
        (ValueError, dict(t, block_table=None)), (ValueError, dict(t, num_blocks=9)),
        (ValueError, dict(q=q, k_cache=k[:, :4], v_cache=k[:, :4], block_table=None, context_lens=None)),
        (TypeError, dict(t, out=torch.zeros(0, 5, 4 * D))), (ff.FFKVError, dict(t, window=-1)),
        (ff.FFKVError, dict(t, score_cap=-1.0)), (TypeError, dict(t, window="3")),
    ]
    for error, kw in bad:
        with pytest.raises(error):
            ff.paged_prefill_scored(**kw, stream=0)
    with pytest.raises(ValueError, match="GPU"):
        ff.paged_prefill_scored(**dict(_tensors(B=1), q=torch.zeros(1, 2, 4, D, dtype=torch.bfloat16)), stream=0)


def _evict(ff, **kw):
    a = dict(weights=16, weight_stride=64, context_lens=16, keep=8, sinks=2, recent=3, k_cache=16, v_cache=16,
             cache_dtype=ff.DTYPE_BF16, k_scale=None, v_scale=None, block_table=16, max_blocks=4, dst_table=None, dst_blocks=0,
             kept=16, kept_lens=32, weights_out=None, out_stride=0, batch=1, num_kv_heads=2, head_dim=64, block_size=16,
             num_blocks=4, workspace=None, workspace_bytes=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return ff.lib.ffkv_evict(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(block_size=8), -2), (dict(cache_dtype=6), -2), (dict(head_dim=100), -2), (dict(batch=-1), -1), (dict(batch=65536), -2),
    (dict(num_kv_heads=0), -1), (dict(keep=0), -1), (dict(keep=-4), -1), (dict(sinks=-1), -1), (dict(recent=-1), -1),
    (dict(sinks=6), -1), (dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), -1), (dict(weights_out=64, out_stride=7), -1),
    (dict(weights_out=16, out_stride=65), -1), (dict(weights=None), -1), (dict(kept=None), -1), (dict(kept_lens=None), -1),
    (dict(kept_lens=16), -1), (dict(cache_dtype=3), -1), (dict(k_cache=24), -1), (dict(weights=18), -1), (dict(kept=18), -1),
    (dict(weight_stride=-1), -1), (dict(weight_stride=1 << 40, max_blocks=2 ** 31 - 1), -2), (dict(dst_blocks=-1), -1),
    (dict(dst_table=16, dst_blocks=4), -1),
    (dict(workspace=8), -1), (dict(workspace=256, workspace_bytes=100, weight_stride=1 << 20, max_blocks=9000), -3),
])
def test_evict_rejects(ff, kw, code):
    assert _evict(ff, **kw) == code
    assert ff.lib.ffkv_last_error().decode() != ""
    assert _evict(ff, batch=0, weights=None) == 0


def test_evict_front(ff):
    pool = torch.zeros(4, 16, HKV, D)
    t = dict(weights=torch.zeros(0, HKV, 9), k_cache=pool, v_cache=pool.clone(), block_table=torch.zeros(0, 3, dtype=torch.int32),
             context_lens=torch.zeros(0, dtype=torch.int32), keep=4)
    kept, lens = ff.evict_tokens(**t, sinks=1, recent=3, dst_table=torch.zeros(0, 1, dtype=torch.int32), stream=0)
    assert kept.shape == (0, HKV, 4) and lens.shape == (0,)
    i = torch.zeros(0, HKV, 4, dtype=torch.int32)
    bad = [
        (ff.FFKVError, dict(t, keep=0)), (ff.FFKVError, dict(t, sinks=5)), (ValueError, dict(t, kept=i[..., :3])),
        (TypeError, dict(t, kept=i.long())), (ValueError, dict(t, weights=torch.zeros(0, HKV + 1, 9))),
        (ValueError, dict(t, weights=torch.zeros(1, HKV, 9))), (TypeError, dict(t, weights=torch.zeros(0, HKV, 9).half())),
        (TypeError, dict(t, dst_table=torch.zeros(0, 1))), (ValueError, dict(t, dst_table=torch.zeros(1, 1, dtype=torch.int32))),
        (ValueError, dict(t, kept_lens=torch.zeros(2, dtype=torch.int32))), (ValueError, dict(t, v_cache=pool[:3])),
        (TypeError, dict(t, block_table=torch.zeros(0, 3))), (TypeError, dict(t, keep=4.0)),
        (ValueError, dict(t, weights_out=torch.zeros(0, 1, 9))), (ValueError, dict(t, num_blocks=5)),
        (ValueError, dict(t, k_cache=torch.zeros(4, 16, HKV, 2 * D)[..., ::2])),
    ]
    for error, kw in bad:
        with pytest.raises(error):
            ff.evict_tokens(**kw, stream=0)
    with pytest.raises(ValueError, match="GPU"):
        ff.evict_tokens(torch.zeros(1, HKV, 9), pool, pool, torch.zeros(1, 3, dtype=torch.int32),
                        torch.zeros(1, dtype=torch.int32), 4, stream=0)


def _weights(ff, **kw):
    a = dict(q=16, qo_dtype=ff.DTYPE_BF16, k_cache=16, cache_dtype=ff.DTYPE_BF16, k_scale=None, block_table=16,
             context_lens=16, batch=1, seq_len=4, num_heads=32, num_kv_heads=8, head_dim=128, block_size=16, max_blocks=4,
             num_blocks=4, max_context_len=0, scale=0.0, score_cap=0.0, slopes=None, window=0, key_begin=None, key_end=None,
             weights=16, prior=None, decay=1.0, weight_stride=64, workspace=None, workspace_bytes=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return ff.lib.ffkv_attention_weights(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(block_size=8), -2), (dict(head_dim=84), -2), (dict(qo_dtype=3), -2), (dict(cache_dtype=7), -2),
    (dict(num_heads=30), -1), (dict(batch=-1), -1), (dict(batch=70000), -2), (dict(seq_len=1 << 19), -2), (dict(q=None), -1),
    (dict(weights=None), -1), (dict(cache_dtype=3), -1), (dict(cache_dtype=8), -1), (dict(q=20), -1), (dict(weights=18), -1),
    (dict(weight_stride=63), -1), (dict(decay=-1.0), -1), (dict(decay=INF), -1), (dict(score_cap=-1.0), -1),
    (dict(window=-1), -1), (dict(key_end=5), -1), (dict(workspace=8), -1), (dict(workspace=256, workspace_bytes=16), -3),
    (dict(batch=65535, seq_len=40000, num_heads=65528, num_kv_heads=65528), -2),
])
def test_weights_rejects(ff, kw, code):
    assert _weights(ff, **kw) == code
    assert ff.lib.ffkv_last_error().decode() != ""
    assert _weights(ff, batch=0, q=None) == 0


def test_weights_front(ff):
    t = _tensors()
    t.pop("v_cache")
    r = torch.zeros(0, 1, dtype=torch.int32)
    assert ff.attention_weights(**t, key_begin=r, key_end=r, stream=0).shape == (0, HKV, 48)
    assert ff.attention_weights(**t, max_context_len=20, stream=0).shape == (0, HKV, 20)
    w = torch.zeros(0, HKV, 48)
    bad = [
        (ValueError, dict(t, q=t["q"][:, 0])), (ValueError, dict(t, key_begin=torch.zeros(0, 2, dtype=torch.int32))),
        (TypeError, dict(t, key_end=r.float())), (ValueError, dict(t, weights=w[..., 0])), (TypeError, dict(t, weights=w.half())),
        (ValueError, dict(t, weights=w, prior=torch.zeros(0, HKV, 40))), (ValueError, dict(t, slopes=torch.zeros(1))),
        (TypeError, dict(t, block_table=t["block_table"].long())), (ValueError, dict(t, num_blocks=5)),
        (ValueError, dict(t, context_lens=torch.zeros(1, dtype=torch.int32))), (ff.FFKVError, dict(t, window=-1)),
        (ValueError, dict(t, k_cache=torch.zeros(4, 16, HKV, 2 * D, dtype=torch.bfloat16)[..., ::2])),
    ]
    for error, kw in bad:
        with pytest.raises(error):
            ff.attention_weights(**kw, stream=0)


@pytest.mark.parametrize("S", [1, 0])
def test_weights_front_device(ff, S):
    """Rows in CPU tensors are refused, also where there are no queries: their earlier weights would still be decayed."""
    t = _tensors(B=1)
    t.pop("v_cache")
    t["q"] = torch.zeros(1, S, 4, D, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        ff.attention_weights(**t, stream=0)
    w = torch.zeros(1, HKV, 48)
    with pytest.raises(ValueError, match="GPU"):
        ff.attention_weights(**t, weights=w, prior=w, stream=0)


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 4, -2 ** 31 - 1, 2 ** 63 - 1, -2 ** 80])
def test_front_integers(ff, n):
    """An int that does not fit the library's 32 bits is refused, not cut to its lower ones (a window of 2^32 + 4 keys was
    one of 4)."""
    t = _tensors()
    with pytest.raises(OverflowError):
        ff.paged_attention_scored(**t, window=n, stream=0)
    with pytest.raises(OverflowError):
        ff.paged_prefill_scored(**t, max_context_len=n, stream=0)
    with pytest.raises(OverflowError):
        ff.paged_attention(**t, max_context_len=n, stream=0)
    t.pop("v_cache")
    with pytest.raises(OverflowError):
        ff.attention_weights(**t, weights=torch.zeros(0, HKV, 48), window=n, stream=0)
    pool = torch.zeros(4, 16, HKV, D)
    with pytest.raises(OverflowError):
        ff.evict_tokens(torch.zeros(0, HKV, 9), pool, pool, t["block_table"], t["context_lens"], 4, sinks=n,
                        kept=torch.zeros(0, HKV, 4, dtype=torch.int32), stream=0)
