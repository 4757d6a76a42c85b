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
