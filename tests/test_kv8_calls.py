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


def test_rotations_past_the_counted_turns_are_refused():
    """The heads' kernel counts quarter turns in 32 bits: with a theta below 1 the last
    pair turns by theta^(2/rope_dim - 1) a position, which passes them."""
    import ctypes

    from vates_amd._lib import QMat, load
    from vates_amd.attention import AttnDesc
    lib, P, big = load(), 1 << 20, 1 << 40

    def append(theta, rd, max_len, q_norm=P):
        return lib.vmi_kv8_append(P, 1, 4, 2, q_norm, P, 1e-6, rd, theta, 0, None, P, max_len, P, None, None)

    def layers(theta, rd, max_len, x=P):
        d = AttnDesc()
        d.hidden, d.n_heads, d.n_kv_heads, d.head_dim, d.rope_dim, d.bits, d.group = 2048, 16, 2, 256, rd, 4, 64
        d.q_proj = d.k_proj = d.v_proj = d.o_proj = QMat(P, P, P)
        d.input_norm = d.q_norm = d.k_norm = P
        d.rope_theta, d.norm_eps = theta, 1e-6
        r = ctypes.byref(d)
        # (the workspace a byte short, so that what is not refused for its angles is for that)
        return (lib.vmi_attention_layer_kv8(r, x, 1, 0, None, P, max_len, P, None, P, 16, None),
                lib.vmi_attention_tree_kv8(r, x, 2, 2, 0, None, P, max_len, P, P, None, P, 16, None),
                lib.vmi_attention_prompt_kv8(r, x, 20, 0, P, max_len, P, P, 16, None))

    invalid, short = -1, -4
    for theta, rd, max_len in ((1e-6, 64, 262144), (1e-30, 256, 64), (1e-7, 4, 1 << 30), (float("nan"), 0, 64), (-1.0, 0, 64)):
        assert append(theta, rd, max_len) == invalid and b"rope_theta" in lib.vmi_last_error()
        for rc in layers(theta, rd, max_len):
            assert rc in (invalid, -2)
    # what can be formed still goes on to the next check
    for theta, rd, max_len in ((1e7, 64, 1 << 30), (1.0, 256, 1 << 30), (0.5, 64, 262144), (1e-30, 2, 262144), (1e-30, 0, 64)):
        assert append(theta, rd, max_len, q_norm=None) == invalid and b"null" in lib.vmi_last_error()
        assert layers(theta, rd, max_len) == (short, short, short)
