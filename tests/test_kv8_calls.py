"""Calls around the 8-bit KV cache that need no device: what a call makes by itself,
and objects with methods of their own beside it."""
import pytest
import torch


@pytest.mark.parametrize("bits", [8, 16])
def test_a_tree_buffer_is_made_with_its_cache(monkeypatch, bits):
    """Made by the first tree call, its fill went to the current stream while the tree's
    kernels ran on the call's: nothing ordered the two."""
    from vates_amd.attention import KVCache, KVCache8
    cache = (KVCache8 if bits == 8 else KVCache)(2, 64, "cpu")

    def refuse(*args, **kw):
        raise AssertionError("a tree call makes its buffer")

    for name in ("zeros", "empty", "zeros_like", "empty_like"):
        monkeypatch.setattr(torch, name, refuse)
    a, b = cache.tree_buffer(2, 3), cache.tree_buffer(4, 4)
    assert a.data_ptr() == b.data_ptr() and b.shape[:2] == (4, 2) and not bool(b.any())
