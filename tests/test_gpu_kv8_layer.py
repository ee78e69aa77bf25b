"""Attention layers and decoding over the 8-bit KV cache: the layer equals its
public operators run one after the other bit for bit, a batch equals single
steps and a tree its paths bit for bit, a prompt equals verify batches up to
rounding, and speculative decoding (eager, graph, tree) emits the greedy stream."""
import pytest

pytestmark = pytest.mark.gpu


def log(msg):
    print(msg, flush=True)


def make_layer(gpu, seed, H=2048, n_heads=16, n_kv=2, rope_dim=64):
    from vates_amd.attention import AttentionLayer
    from vates_amd.synth import synth_bf16, synth_proj
    import torch
    w = [synth_proj(seed, i + 1, 1, n, k, device=gpu) for i, (n, k) in enumerate(
        ((n_heads * 512, H), (n_kv * 256, H), (n_kv * 256, H), (H, n_heads * 256)))]
    norms = [(synth_bf16(seed, 5 + i, (n,), std=0.1, device=gpu).float() + 1.0).to(torch.bfloat16)
             for i, n in enumerate((H, 256, 256))]
    return AttentionLayer(*w, *norms, n_heads=n_heads, n_kv_heads=n_kv, rope_dim=rope_dim)


def filled(layer, seed, n, max_len, gpu):
    from vates_amd.synth import synth_bf16
    c = layer.new_cache(max_len, bits=8)
    if n:
        c.write(0, synth_bf16(seed, 20, (layer.n_kv, n, 256), device=gpu), synth_bf16(seed, 21, (layer.n_kv, n, 256), device=gpu))
    c.length = n
    return c


def composed(layer, x, cache, pos0):
    """The layer by its public parts."""
    import torch
    from vates_amd.attention import attend, norm_rope_append, qgemv
    from vates_amd.mtp import rmsnorm
    q, k, v, o, inn, qn, kn = layer._keep
    T = x.shape[0]
    xn = rmsnorm(x, inn, eps=layer.desc.norm_eps)
    qkv = torch.cat([qgemv(xn, w) for w in (q, k, v)], dim=1).contiguous()
    rows = norm_rope_append(qkv, cache, qn, kn, n_heads=layer.n_heads, rope_dim=layer.desc.rope_dim,
                            rope_theta=layer.desc.rope_theta, eps=layer.desc.norm_eps, pos0=pos0)
    gate = qkv[:, :layer.n_heads * 512].view(T, layer.n_heads, 2, 256)[:, :, 1]
    y = attend(rows, cache, pos0=pos0, gate=gate)
    out = torch.empty_like(x)
    return qgemv(y.view(T, -1), o, out_bf16=out, residual=x)


@pytest.mark.parametrize("T,pos0,max_len,heads", [(1, 0, 64, (16, 2)), (4, 0, 256, (16, 2)), (8, 1000, 1024, (16, 2)),
                                                  (4, 30, 64, (4, 4)), (4, 32764, 32768, (16, 2)), (3, 5000, 6000, (6, 2))])
def test_layer_is_its_parts(gpu, T, pos0, max_len, heads):
    import torch
    from vates_amd.synth import synth_bf16
    log(f"case: kv8 layer T={T} pos0={pos0} max_len={max_len} heads={heads}")
    layer = make_layer(gpu, 31, H=2048 if heads[0] == 16 else 512, n_heads=heads[0], n_kv=heads[1])
    a, b, c = (filled(layer, 31, pos0, max_len, gpu) for _ in range(3))
    x = synth_bf16(31, 30 + T, (T, layer.hidden), device=gpu)
    got = layer(x, a, pos0=pos0)
    want = composed(layer, x, b, pos0)
    assert a.length == b.length == pos0 + T
    assert torch.equal(a.data, b.data) and torch.equal(got, want)
    # single steps, in a larger cache, with the position on the device
    d = filled(layer, 31, pos0, max_len + 8000, gpu)
    steps = torch.cat([layer(x[t:t + 1].contiguous(), c) for t in range(T)])
    dev = torch.cat([layer(x[t:t + 1].contiguous(), d, pos_device=torch.tensor([pos0 + t], dtype=torch.int32, device=gpu))
                     for t in range(T)])
    assert torch.equal(steps, got) and torch.equal(dev, got) and torch.equal(c.data, a.data)
    assert d.length == pos0 and int(d.status) == 0


def test_layer_is_close_to_the_bf16_one(gpu):
    """A row's elements are off by up to half a code step, a / 254 with a about 3.3
    times the row's RMS: 0.0075 of it in the mean square.  Averaging over positions
    scales values and their errors alike, and a score moves by 0.0075 times the
    scores' spread (about 1), its weight by as much: 0.011 together, below 2 % of
    the attention half.  The block's output x + y is rounded to bf16 on both sides,
    half a step or 2^-8 |x + y| each, whatever the cache."""
    import torch
    from vates_amd.synth import synth_bf16
    layer = make_layer(gpu, 32)
    k, v = (synth_bf16(32, i, (2, 3000, 256), device=gpu) for i in (20, 21))
    x = synth_bf16(32, 9, (4, 2048), device=gpu)
    outs = []
    for bits in (16, 8):
        c = layer.new_cache(4096, bits)
        c.write(0, k, v)
        outs.append(layer(x, c, pos0=3000).float())
    assert float((outs[1] - outs[0]).norm()) <= 0.02 * float((outs[0] - x.float()).norm()) + 2 * 2 ** -8 * float(outs[0].norm())


@pytest.mark.parametrize("pos0", [0, 29, 1000, 33100])
def test_tree_equals_paths_and_commits(gpu, pos0):
    import torch
    from vates_amd.decode import TreeCommit
    from vates_amd.synth import synth_bf16
    log(f"case: kv8 tree 3 x 4 at {pos0}")
    P, S = 3, 4
    layer = make_layer(gpu, 33)
    base = filled(layer, 33, pos0, pos0 + 64, gpu)
    x = synth_bf16(33, 30, (P * S, 2048), device=gpu)
    before = base.data.clone()
    out = layer.tree(x, base, P)
    commit = TreeCommit([base], P, S)
    assert torch.equal(base.data, before) and base.length == pos0
    for p, acc in ((0, 1), (2, 4), (1, 3)):
        alone = filled(layer, 33, pos0, pos0 + 64, gpu)
        got = layer(x[p * S:(p + 1) * S].contiguous(), alone)
        assert torch.equal(got, out[p * S:(p + 1) * S]), p
        base.data.copy_(before)
        rec = torch.tensor([acc, acc, acc, p] + [0] * (S + 1), dtype=torch.int32, device=gpu)
        commit(rec, pos0=pos0)
        want = filled(layer, 33, pos0, pos0 + 64, gpu)
        layer(x[p * S:p * S + acc].contiguous(), want)
        assert torch.equal(base.data, want.data), (p, acc)


@pytest.mark.parametrize("T,pos0", [(17, 0), (100, 13), (333, 700)])
def test_prompt_equals_batches(gpu, T, pos0):
    """The prompt form against verify batches on the same cache: rows differ by the
    order of fp32 sums in the projections (a code here and there one step off), the
    attention's rows and the block's outputs x + y by bf16 rounding.  Each side rounds
    the attention's rows within half a step, 2^-8 of them, which the output projection
    carries to y, and then x + y within 2^-8 |x + y|: 2^-7 of both norms together."""
    import torch
    from vates_amd.synth import synth_bf16
    log(f"case: kv8 prompt T={T} pos0={pos0}")
    layer = make_layer(gpu, 34)
    a, b, c = (filled(layer, 34, pos0, pos0 + T, gpu) for _ in range(3))
    x = synth_bf16(34, 30, (T, 2048), device=gpu)
    got = layer.prompt(x, a, pos0=pos0)
    want = torch.cat([layer(x[i:i + 8].contiguous(), b) for i in range(0, T, 8)])
    assert a.length == b.length == pos0 + T
    y = (want.float() - x.float()).norm()
    assert float((got.float() - want.float()).norm()) <= 2 ** -7 * float(y + want.float().norm())
    for u, w in zip(a.read(0, dtype=torch.float32), b.read(0, dtype=torch.float32)):
        assert bool(((u - w).abs() <= 1.01 * w.abs().amax(-1, keepdim=True) / 127).all())
        assert float((u - w).norm() / w.norm()) <= 1e-3
    assert layer.prompt(x, c, pos0=pos0, keys_only=True) is None
    assert torch.equal(c.data, a.data)
    # rows so small that x + y is y (the block normalises its input): the attention half alone
    small = (x.float() * 2.0 ** -12).to(torch.bfloat16)
    got = layer.prompt(small, a, pos0=pos0).float()
    want = torch.cat([layer(small[i:i + 8].contiguous(), b, pos0=pos0 + i) for i in range(0, T, 8)]).float()
    assert float((got - want).norm()) <= 2 ** -7 * 2 * float(want.norm())


SMALL = dict(n_layers=4, attn_every=2, hidden=512, inter=128, num_experts=64, top_k=4, vocab=4096, n_heads=4,
             n_kv_heads=2, n_k_heads=2, n_v_heads=4)


@pytest.fixture(scope="module")
def model(gpu):
    from vates_amd.workload import synth_spec_model
    return synth_spec_model(91, **SMALL, device=gpu)


def started(model, prompt, max_len=256):
    from vates_amd.attention import KVCache8
    from vates_amd.decode import prefill
    from vates_amd.mtp import MTPDrafter
    caches, drafter = model.new_caches(max_len, kv_bits=8), MTPDrafter(model.mtp, max_len, kv_bits=8)
    assert any(isinstance(c, KVCache8) for c in caches) and isinstance(drafter.cache, KVCache8)
    x, h = prefill(model, prompt, caches, drafter)
    return caches, drafter, x, h


@pytest.mark.parametrize("P", [8, 50])
def test_decoding_emits_the_greedy_stream(gpu, model, P):
    import torch
    from vates_amd.decode import (GraphGreedyDecoder, GraphSpecDecoder, greedy_decode, speculative_decode,
                                  tree_speculative_decode)
    prompt = torch.randint(0, SMALL["vocab"], (P,), dtype=torch.int32, device=gpu, generator=torch.Generator(gpu).manual_seed(P))
    n = 60
    caches, drafter, x, h = started(model, prompt)
    truth = greedy_decode(model, caches, x, P, n + 8).tokens
    log(f"case: kv8 decoding P={P} {truth[:8]}...")
    caches, drafter, x, h = started(model, prompt)
    assert speculative_decode(model, drafter, caches, x, h, P, n).tokens == truth[:n]
    caches, drafter, x, h = started(model, prompt)
    assert tree_speculative_decode(model, drafter, caches, x, h, P, n).tokens == truth[:n]
    caches, drafter, x, h = started(model, prompt)
    dec = GraphSpecDecoder(model, drafter, caches, planted=True)
    dec.start(x, h, P)

    def plant(step, pos):   # every acceptance length in turn
        return [truth[pos - P + i] if i < step % 4 else (truth[pos - P + i] + 1) % SMALL["vocab"] for i in range(3)]

    st = dec.run(n, plant=plant)
    assert st.tokens == truth[:n] and set(st.accept_hist) == {0, 1, 2, 3}
    caches, drafter, x, h = started(model, prompt)
    g = GraphGreedyDecoder(model, caches, n)
    g.start(x, P)
    assert g.run(n).tokens == truth[:n]


def test_prompt_blocks_and_batches_agree(gpu, model, monkeypatch):
    """decode.prefill into 8-bit caches through the prompt kernels, in one block
    and in ragged ones, against verify batches."""
    import torch
    from vates_amd import decode
    P = 203
    prompt = torch.randint(0, SMALL["vocab"], (P,), dtype=torch.int32, device=gpu, generator=torch.Generator(gpu).manual_seed(3))
    ends = []
    for block, least in ((4096, 10 ** 9), (4096, 16), (64, 16), (101, 16)):
        monkeypatch.setattr(decode, "PROMPT_BLOCK", block)
        monkeypatch.setattr(decode, "PROMPT_MIN", least)
        caches, drafter, x, h = started(model, prompt)
        assert drafter.cache.length == P - 1
        ends.append((h.float(), drafter.cache.values().float()))
    for h, v in ends[1:]:
        assert float((h - ends[0][0]).norm() / ends[0][0].norm()) <= 0.03
        assert float((v - ends[0][1]).norm() / ends[0][1].norm()) <= 0.03


def test_a_cache_of_another_layer_is_refused(gpu):
    import torch
    from vates_amd._lib import VmiError
    layer = make_layer(gpu, 41)
    other = make_layer(gpu, 42, H=512, n_heads=4, n_kv=1).new_cache(128, 8)
    x = torch.zeros((40, layer.hidden), dtype=torch.bfloat16, device=gpu)
    for call in (lambda: layer(x[:1], other), lambda: layer.prompt(x, other, pos0=0), lambda: layer.tree(x[:4], other, 2),
                 lambda: layer(x[:9], layer.new_cache(128, 8)), lambda: layer.prompt(x, layer.new_cache(32, 8), pos0=0),
                 lambda: layer(x[:4], layer.new_cache(32, 8), pos0=29), lambda: layer.new_cache(64, 4)):
        with pytest.raises(VmiError):
            call()
