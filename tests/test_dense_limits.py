"""Sizes that the dense operators' kernels could not count are refused before any HIP call."""

import ctypes

import pytest

from tests.test_dense_abi import INVALID, OVERFLOW, P, _args, lib  # noqa: F401


def test_attention_of_more_tiles_than_a_launch_has(lib):  # noqa: F811
    a = _args(batch=1 << 25, queries=1, q_heads=1, kv_heads=1, keys=32)
    assert lib.nacho_block_attention(ctypes.byref(a), None, None) == OVERFLOW
    assert lib.nacho_block_attention_backward(ctypes.byref(a), None, None) == OVERFLOW


@pytest.mark.parametrize("changes", [
    dict(batch=1 << 16, queries=1, q_heads=1, kv_heads=1, keys=1 << 14, block=64),
    dict(batch=1 << 16, queries=0, q_heads=1, kv_heads=1, keys=1 << 14, block=128, dtype=0),
], ids=str)
def test_gradients_of_more_keys_than_a_launch_has(lib, changes):  # noqa: F811
    a = _args(**changes)
    assert lib.nacho_block_attention_backward(ctypes.byref(a), None, None) == OVERFLOW


def test_scores_of_more_queries_than_a_launch_has(lib):  # noqa: F811
    from nacho_amd import _lib

    h = ctypes.byref(_lib.Heads(0x10000, 1 << 20, 256, 64))
    assert lib.nacho_block_scores(2, 1 << 25, 1, 32, 1, 1, 64, 32, 1, 0.125, h, P(0x1000), None,
                                  P(0x1000), None) == OVERFLOW


MOST_IDS = (2 ** 31 - 1 - 256) // 128  # ids of a query: 128 queries of a tile times these are counted


def test_attention_of_more_ids_than_a_tile_counts(lib):  # noqa: F811
    for count in (MOST_IDS + 1, 1 << 24, (2 ** 31 - 1) // 64):
        a = _args(count=count)
        assert lib.nacho_block_attention(ctypes.byref(a), None, None) == OVERFLOW
        assert lib.nacho_block_attention_backward(ctypes.byref(a), None, None) == OVERFLOW


def test_selection_of_more_ids_than_a_row_counts(lib):  # noqa: F811
    for count in (2 ** 31 - 64, 2 ** 31 - 1):
        assert lib.nacho_block_select(1, 1, 1, 100, 32, count, 1, 1, 1, P(0x1000), None, P(0x1000),
                                      None) == OVERFLOW


def test_rows_of_more_entries_than_are_counted(lib):  # noqa: F811
    x = P(0x1000)
    for tokens, per_token in ((1, 2 ** 31 - 1), (1, 2 ** 31 - 1000), (1 << 20, 2048)):
        assert lib.nacho_dispatch(2, tokens, per_token, 4, 8, x, 8, x, x, x, None) == OVERFLOW
        assert lib.nacho_combine(2, tokens, per_token, 8, x, 8, None, x, x, None) == OVERFLOW
        assert lib.nacho_combine_backward(2, tokens, per_token, 4, 8, x, 8, x, x, x, x, 8, x, x,
                                          None) == OVERFLOW


@pytest.mark.parametrize("scale", (2.4e38, -2.4e38, 3.4e38))
def test_attention_of_a_scale_whose_base_2_factor_is_infinite(lib, scale):  # noqa: F811
    a = _args(scale=scale)
    assert lib.nacho_block_attention(ctypes.byref(a), None, None) == INVALID
    assert lib.nacho_block_attention_backward(ctypes.byref(a), None, None) == INVALID


@pytest.mark.parametrize("scale", (1e39, -1e300, 3.5e38, float("inf"), float("nan")))
def test_a_scale_past_float32_is_named(scale):
    from nacho_amd import blocks

    with pytest.raises(ValueError, match="scale must be finite"):
        blocks._scale(scale, (1, 1, 1, 64))


def test_scales_in_range_are_kept():
    from nacho_amd import blocks

    for scale in (0.0, -2.5, 2.3e38, 1e-45):
        assert blocks._scale(scale, (1, 1, 1, 64)) == scale
    assert blocks._scale(None, (1, 1, 1, 64)) == 0.125
