"""Calls whose launches would pass the 2^32 - 1 threads of a grid are refused by name, before anything is allocated."""

import pytest

from test_blocks_refusals import _attend, _bounds, _select

UNSUPPORTED = -2


@pytest.mark.parametrize("kw", [
    dict(seq_len=8_400_000),                                                          # a workgroup a list
    dict(batch=2, seq_len=64 * 1_050_000, query_block=64, num_heads=16, max_blocks=128),  # the sums of long blocks
    dict(batch=65535, seq_len=2, num_kv_heads=8, max_blocks=4096),                    # the scores
    dict(seq_len=4_200_000, max_blocks=4097, max_context_len=0),                      # choices of long rows
])
def test_select(ff, kw):
    assert _select(ff, **{"count": 64, **kw}) == UNSUPPORTED
    assert b"too many" in ff.lib.ffkv_last_error()


@pytest.mark.parametrize("kw", [
    dict(seq_len=16_800_000, num_heads=1, num_kv_heads=1, head_dim=72),
    dict(seq_len=16_800_000, num_heads=2, num_kv_heads=2, query_block=1),
    dict(seq_len=33_600_000, num_heads=1, num_kv_heads=1, query_block=2),
    dict(seq_len=16_800_000, num_heads=1, num_kv_heads=1, query_block=2, head_dim=256),
])
def test_attention(ff, kw):
    assert _attend(ff, **kw) == UNSUPPORTED
    assert b"too many" in ff.lib.ffkv_last_error()


def test_key_bounds(ff):
    assert _bounds(ff, new_tokens=700_000_000, num_kv_heads=8, max_blocks=40_000_000) == UNSUPPORTED
    assert b"too many" in ff.lib.ffkv_last_error()


def test_workspace_of_refused_calls(ff):
    """Sizes that the choice refuses need nothing: batch, seq_len, heads, KV heads, head_dim, count, query_block, max_blocks, bound."""
    size = ff.lib.ffkv_select_blocks_workspace_bytes
    assert size(2, 64 * 1_050_000, 16, 2, 128, 64, 64, 128, 0) == 0 and size(65535, 2, 8, 8, 128, 64, 1, 4096, 0) == 0
    assert size(2, 64 * 1_000, 16, 2, 128, 64, 64, 128, 0) > 0
