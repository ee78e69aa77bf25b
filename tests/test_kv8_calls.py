"""Calls around the 8-bit KV cache that need no device: what a call makes by itself,
and objects with methods of their own beside it."""
import types

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


class OwnAttention:
    """An attention object of a program's own, as bf16 caches use it."""
    n_heads, n_kv = 4, 2

    def __init__(self):
        self.made = []

    def prompt_workspace_bytes(self, T):
        return 100 * T


def test_a_layer_whose_prompt_workspace_takes_tokens_alone(monkeypatch):
    """The MTP layer's query for its cache's fill, and the layer's own prompt call, ask it as before."""
    from vates_amd import attention, mtp
    from vates_amd.attention import AttentionLayer, KVCache

    layer = mtp.MTPLayer.__new__(mtp.MTPLayer)
    layer.hidden, layer.w = 512, types.SimpleNamespace(fc=None, attn=OwnAttention())
    monkeypatch.setattr(mtp, "qgemm_workspace_bytes", lambda w, T, K: 7)
    cache = KVCache(2, 64, "cpu")
    assert layer.fill_workspace_bytes(5) == 500 and layer.fill_workspace_bytes(5, cache) == 500

    class Sized(AttentionLayer):
        def prompt_workspace_bytes(self, T):
            return 100 * T

    asked = []

    def scratch(nbytes, device, stream=None):
        asked.append(nbytes)
        raise MemoryError

    sized = Sized.__new__(Sized)
    sized.__dict__.update(hidden=512, n_kv=2, n_heads=4, device=torch.device("cpu"))
    monkeypatch.setattr(attention, "scratch", scratch)
    monkeypatch.setattr(attention, "_stream_handle", lambda stream: 0)
    with pytest.raises(MemoryError):
        sized.prompt(torch.zeros((5, 512), dtype=torch.bfloat16), cache, pos0=0)
    assert asked == [500]


def test_a_layer_whose_new_cache_takes_the_length_alone():
    """Models and drafters ask for bf16 caches as before, for 8-bit ones by name."""
    from vates_amd.decode import DecoderLayer, SpecModel
    from vates_amd.mtp import MTPDrafter

    class Own:
        def new_cache(self, max_len):
            return ("own", max_len)

    class Both:
        def new_cache(self, max_len, bits=16):
            return ("both", max_len, bits)

    model = SpecModel.__new__(SpecModel)
    model.layers = [DecoderLayer(None, attn=Own()), DecoderLayer(None, attn=Both()), DecoderLayer(None)]
    assert model.new_caches(64) == [("own", 64), ("both", 64, 16), None]
    model.layers = model.layers[1:]
    assert model.new_caches(64, kv_bits=8) == [("both", 64, 8), None]
    for attn, kw, want in ((Own(), {}, ("own", 9)), (Both(), dict(kv_bits=8), ("both", 9, 8))):
        assert MTPDrafter(types.SimpleNamespace(w=types.SimpleNamespace(attn=attn)), 9, **kw).cache == want
