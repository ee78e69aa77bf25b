"""The 8-bit KV cache without a device: sizes, workspaces, and what its entry
points refuse (no call here reaches a kernel; the pointers are never read)."""
import ctypes

import pytest
import torch

P = 1 << 20   # a 16-byte aligned address
ERR_INVALID, ERR_UNSUPPORTED, ERR_WORKSPACE = -1, -2, -4   # include/vmi.h


@pytest.fixture(scope="module")
def lib():
    from vates_amd._lib import load
    return load()


def refused(lib, code):
    """Refused for its arguments, with a message: not by a launch that failed."""
    return code in (ERR_INVALID, ERR_UNSUPPORTED, ERR_WORKSPACE) and bool(lib.vmi_last_error())


def test_bytes(lib):
    for n_kv, max_len in ((1, 32), (2, 4096), (8, 262144), (1024, 64)):
        assert lib.vmi_kv8_bytes(n_kv, max_len) == n_kv * max_len // 32 * 16640
    for n_kv, max_len in ((0, 32), (1025, 32), (1, 0), (1, 33), (1, -32)):
        assert lib.vmi_kv8_bytes(n_kv, max_len) == 0


@pytest.mark.parametrize("n_heads,n_kv", [(16, 2), (1, 1), (8, 8), (32, 4), (5, 1), (1024, 1)])
def test_workspace_covers_every_shorter_batch(lib, n_heads, n_kv):
    """decode.prefill asks once, for its block, and runs a shorter last one in it."""
    size = [lib.vmi_kv8_attention_workspace_bytes(T, n_heads, n_kv) for T in range(1, 8193)]
    assert size[0] > 0 and all(b >= a for a, b in zip(size, size[1:]))
    assert lib.vmi_kv8_attention_workspace_bytes(8193, n_heads, n_kv) == 0
    assert lib.vmi_kv8_attention_workspace_bytes(0, n_heads, n_kv) == 0


def test_workspace_of_unbuilt_forms_is_zero(lib):
    for n_heads, n_kv in ((0, 1), (3, 2), (2, 0), (1025, 1), (-2, -1)):
        assert lib.vmi_kv8_attention_workspace_bytes(4, n_heads, n_kv) == 0
    ok = lib.vmi_attention_kv8_workspace_bytes
    assert ok(1, 8, 2048, 16, 2) > 0 and ok(4, 4, 2048, 16, 2) > 0 and ok(16, 1, 1024, 4, 4) > 0
    for bad in ((0, 1, 2048, 16, 2), (1, 9, 2048, 16, 2), (4, 5, 2048, 16, 2), (17, 1, 2048, 16, 2), (1, 8, 2048, 32, 2),
                (1, 1, 2000, 16, 2), (1, 1, 2048, 15, 2)):
        assert ok(*bad) == 0, bad


def test_write_and_read_refuse(lib):
    def write(k=P, kh=256, kr=256, v=P, vh=256, vr=256, n_kv=2, pos=0, n=1, cache=P, max_len=64):
        return lib.vmi_kv8_write(k, kh, kr, v, vh, vr, n_kv, pos, n, cache, max_len, None)

    for bad in (dict(k=None), dict(v=None), dict(cache=None), dict(k=P + 8), dict(v=P + 2), dict(cache=P + 8), dict(kh=4),
                dict(kr=257), dict(vh=-1), dict(vr=12), dict(n_kv=0), dict(n_kv=1025), dict(pos=-1), dict(pos=64),
                dict(pos=60, n=5), dict(n=0), dict(n=-1), dict(n=65), dict(max_len=0), dict(max_len=63),
                dict(pos=2 ** 31 - 1)):
        assert refused(lib, write(**bad)), bad

    def read(cache=P, n_kv=2, max_len=64, pos=0, n=1, k=P, v=P, dtype=1):
        return lib.vmi_kv8_read(cache, n_kv, max_len, pos, n, k, v, dtype, None)

    for bad in (dict(cache=None), dict(n_kv=0), dict(max_len=40), dict(pos=-3), dict(pos=63, n=2), dict(n=0),
                dict(k=None, v=None), dict(k=P + 4), dict(v=P + 8), dict(dtype=9), dict(dtype=-1)):
        assert refused(lib, read(**bad)), bad


def test_append_refuses(lib):
    def append(qkv=P, T=1, n_heads=4, n_kv=2, qn=P, kn=P, eps=1e-6, rd=64, theta=1e7, pos=0, dev=None, cache=P, max_len=64,
               q=P):
        return lib.vmi_kv8_append(qkv, T, n_heads, n_kv, qn, kn, eps, rd, theta, pos, dev, cache, max_len, q, None, None)

    for bad in (dict(qkv=None), dict(qkv=P + 4), dict(T=0), dict(T=65), dict(n_heads=3), dict(n_heads=0), dict(n_kv=0),
                dict(n_heads=1026), dict(qn=None), dict(kn=None), dict(rd=-2), dict(rd=7), dict(rd=258), dict(theta=0.0),
                dict(theta=float("nan")), dict(pos=64), dict(pos=-1), dict(cache=None), dict(max_len=50), dict(q=P + 8),
                dict(T=65, dev=P)):
        assert refused(lib, append(**bad)), bad


def test_attention_refuses(lib):
    need = lib.vmi_kv8_attention_workspace_bytes(8, 16, 2)

    def attend(q=P, T=8, n_heads=16, n_kv=2, pos=0, dev=None, cache=P, max_len=16384, gate=None, gt=0, gh=0, out=P, ws=P,
               nbytes=need):
        return lib.vmi_kv8_attention(q, T, n_heads, n_kv, pos, dev, cache, max_len, gate, gt, gh, out, None, ws, nbytes, None)

    for bad in (dict(q=None), dict(q=P + 8), dict(out=None), dict(out=P + 2), dict(T=0), dict(T=8193, nbytes=1 << 40),
                dict(n_heads=15), dict(n_heads=0), dict(n_kv=0), dict(pos=-1), dict(pos=16384), dict(pos=16380),
                dict(cache=None), dict(cache=P + 4), dict(max_len=31), dict(gate=P + 4, gt=256, gh=256),
                dict(gate=P, gt=255, gh=256), dict(gate=P, gt=256, gh=2), dict(ws=None), dict(ws=P + 8), dict(nbytes=need - 1)):
        assert refused(lib, attend(**bad)), bad


def test_layer_entries_refuse(lib):
    from vates_amd._lib import QMat
    from vates_amd.attention import AttnDesc

    def desc(**kw):
        d = AttnDesc()
        d.hidden, d.n_heads, d.n_kv_heads, d.head_dim, d.rope_dim, d.bits, d.group = 2048, 16, 2, 256, 64, 4, 64
        d.q_proj = d.k_proj = d.v_proj = d.o_proj = QMat(P, P, P)
        d.input_norm = d.q_norm = d.k_norm = P
        d.rope_theta, d.norm_eps = 1e7, 1e-6
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    big = 1 << 40

    def layer(d, T=1, pos=0, cache=P, max_len=64, x=P, out=P, ws=P, nbytes=big):
        return lib.vmi_attention_layer_kv8(d, x, T, pos, None, cache, max_len, out, None, ws, nbytes, None)

    def tree(d, paths=2, span=2, pos=0, cache=P, max_len=64, rows=P, x=P, out=P, ws=P, nbytes=big):
        return lib.vmi_attention_tree_kv8(d, x, paths, span, pos, None, cache, max_len, rows, out, None, ws, nbytes, None)

    def prompt(d, T=40, pos=0, cache=P, max_len=64, x=P, out=P, ws=P, nbytes=big):
        return lib.vmi_attention_prompt_kv8(d, x, T, pos, cache, max_len, out, ws, nbytes, None)

    for call in (layer, tree, prompt):
        assert refused(lib, call(None))
        for bad in (dict(head_dim=128), dict(bits=3), dict(group=32), dict(rope_dim=65), dict(rope_dim=-2), dict(n_heads=15),
                    dict(hidden=2000), dict(q_proj=QMat(None, P, P)), dict(o_proj=QMat(P + 4, P, P)), dict(input_norm=None),
                    dict(k_norm=None)):
            assert refused(lib, call(desc(**bad))), (call.__name__, bad)
        for bad in (dict(pos=-1), dict(pos=63), dict(cache=None), dict(cache=P + 8), dict(max_len=33), dict(x=None),
                    dict(out=None), dict(ws=None), dict(ws=P + 8), dict(nbytes=64)):
            if call is layer and bad == dict(pos=63):
                bad = dict(pos=64)
            if call is prompt and bad == dict(out=None):
                continue   # a prompt without an output forms the keys and values alone
            assert refused(lib, call(desc(), **bad)), (call.__name__, bad)
    for bad in (dict(T=0), dict(T=9)):
        assert refused(lib, layer(desc(), **bad)), bad
    for bad in (dict(paths=0), dict(span=9), dict(paths=9), dict(rows=None), dict(rows=P + 8)):
        assert refused(lib, tree(desc(), **bad)), bad
    for bad in (dict(T=0), dict(T=65)):
        assert refused(lib, prompt(desc(), **bad)), bad


def test_python_refuses():
    from vates_amd._lib import VmiError
    from vates_amd.attention import KVCache8, attend, norm_rope_append
    for bad in (dict(head_dim=128), dict(n_kv_heads=0), dict(max_len=0), dict(n_kv_heads=2000)):
        with pytest.raises(VmiError):
            KVCache8(**{**dict(n_kv_heads=2, max_len=64, device="cpu"), **bad})
    c = KVCache8(2, 40, "cpu")
    assert c.max_len == 64 and c.data.numel() == 2 * 2 * 16640 and c.length == 0
    k = torch.zeros((2, 1, 256), dtype=torch.bfloat16)
    for call in (lambda: c.write(0, k, k), lambda: c.read(0, 1), lambda: attend(k, c, pos0=0),
                 lambda: norm_rope_append(torch.zeros(1, 10 * 256), c, k[0, 0], k[0, 0], n_heads=4)):
        with pytest.raises(VmiError, match="device"):
            call()
    with pytest.raises(VmiError):
        c.read(0, 65)
    with pytest.raises(VmiError):
        c.read(0, 1, dtype=torch.float16)
    with pytest.raises(VmiError):
        c.tree_buffer(4, 5)
