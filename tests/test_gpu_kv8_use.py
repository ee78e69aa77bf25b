"""The 8-bit KV cache as it is used: appends and attention in turn, captured
graphs, other streams, positions on the device, rows that are not finite, value
scales and queries of extreme sizes, a cache past 4 GiB.

Reference and bars: attend64 and held of tests/test_gpu_kv8.py, where the bars are
derived."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import DIM, attend64, held, log, new_cache, projections, queries, rows, same

pytestmark = pytest.mark.gpu


def check_attend(got, q, cache, pos0, gate):
    k, v = cache.read(0, pos0 + q.shape[0], dtype=torch.float32)
    want, tol = attend64(q, k, v, pos0, gate)
    # a gate below -87 has a sigmoid under fp32's normal range, 2^-126: zero or not, the
    # output, of at most max |v|, is off by no more than that of it
    tol = tol + 2.0 ** -126 * v.abs().max().double()
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("T,pos0,n_heads,n_kv", [(8, 60000, 16, 2), (3, 99990, 16, 2), (4, 61437, 32, 4), (2, 50000, 24, 1)])
def test_batch_and_capacity_do_not_change_a_token(gpu, T, pos0, n_heads, n_kv):
    """Long enough that a batch's workgroups hold two row groups where a token's hold one."""
    log(f"case: kv8 batch T={T} pos0={pos0} {n_heads}/{n_kv}")
    from vates_amd.attention import attend
    k, v = rows(31, n_kv, pos0 + T, gpu)
    q, gate = queries(32, T, n_heads, gpu)
    cache, wide = new_cache(n_kv, pos0 + T, gpu), new_cache(n_kv, 2 * pos0, gpu)
    for c in (cache, wide):
        c.write(0, k, v)
    got = attend(q, cache, pos0=pos0, gate=gate)
    check_attend(got, q, cache, pos0, gate)
    assert torch.equal(attend(q, wide, pos0=pos0, gate=gate), got)
    dev = torch.tensor([pos0], dtype=torch.int32, device=gpu)
    assert torch.equal(attend(q, wide, pos_device=dev, gate=gate), got)
    steps = torch.cat([attend(q[t:t + 1], cache, pos0=pos0 + t, gate=gate[t:t + 1]) for t in range(T)])
    assert torch.equal(steps, got)


@pytest.mark.parametrize("T,pos0,n_heads,n_kv", [(600, 3000, 16, 2), (1111, 0, 12, 4), (130, 40000, 8, 1), (2500, 77, 8, 2)])
def test_prompts_with_much_work(gpu, T, pos0, n_heads, n_kv):
    """Sizes of the paired form; an odd number of tiles, one tile alone, tiles that see one record."""
    log(f"case: kv8 prompt T={T} pos0={pos0} {n_heads}/{n_kv}")
    from vates_amd.attention import attend
    cache = new_cache(n_kv, pos0 + T + 40, gpu)
    cache.data.fill_(255)                      # what lies behind the last position: NaN scales
    cache.write(0, *rows(33, n_kv, pos0 + T, gpu))
    q, gate = queries(34, T, n_heads, gpu)
    check_attend(attend(q, cache, pos0=pos0, gate=gate), q, cache, pos0, gate)
    check_attend(attend(q, cache, pos0=pos0), q, cache, pos0, None)


def test_operators_in_turn(gpu):
    """A conversation: prompt, tokens, a batch, rejected positions given back and
    written again, a second prompt; every answer against the rows as they are read."""
    from vates_amd.attention import attend, norm_rope_append
    n_heads, n_kv = 16, 2
    cache, again = new_cache(n_kv, 700, gpu), new_cache(n_kv, 700, gpu)
    at, seed = 0, 40
    for T, keep in ((37, 37), (1, 1), (4, 2), (1, 1), (8, 3), (300, 300), (1, 1), (5, 5), (65, 1), (1, 1)):
        log(f"case: kv8 turn T={T} at {at}")
        qkv, qn, kn = projections(seed, T, n_heads, n_kv, gpu)
        seed += 1
        cache.length = at
        q = norm_rope_append(qkv, cache, qn, kn, n_heads=n_heads)
        assert cache.length == at + T
        gate = qkv.view(T, -1, DIM)[:, 1:2 * n_heads:2]      # as the projections lie
        got = attend(q, cache, gate=gate)
        check_attend(got, q, cache, at, gate)
        again.length = at
        norm_rope_append(qkv[:keep].contiguous(), again, qn, kn, n_heads=n_heads)
        at += keep
        a, b = cache.read(0, at, dtype=torch.float32), again.read(0, at, dtype=torch.float32)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_captured_step(gpu):
    """One decoded token captured, its position advanced on the device, replayed with
    eager work between: each replay equals the eager step, bit for bit."""
    from vates_amd.attention import attend, norm_rope_append
    n_heads, n_kv, start, steps = 16, 2, 90, 8
    qkv, qn, kn = projections(50, steps, n_heads, n_kv, gpu)
    k, v = rows(51, n_kv, start, gpu)
    eager, cap = new_cache(n_kv, 160, gpu), new_cache(n_kv, 160, gpu)
    for c in (eager, cap):
        c.write(0, k, v)
        c.length = start
    row = qkv[:1].clone()
    pos = torch.tensor([start], dtype=torch.int32, device=gpu)

    def step():
        q = norm_rope_append(row, cap, qn, kn, n_heads=n_heads, pos_device=pos)
        out = attend(q, cap, pos_device=pos, gate=row.view(1, -1, DIM)[:, 1:2 * n_heads:2])
        pos.add_(1)
        return out

    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        step()
    torch.cuda.synchronize()
    pos.fill_(start)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        out = step()
    for t in range(steps):
        log(f"case: kv8 replay {t}")
        row.copy_(qkv[t:t + 1])
        q = norm_rope_append(qkv[t:t + 1].contiguous(), eager, qn, kn, n_heads=n_heads)
        want = attend(q, eager, gate=qkv[t:t + 1].view(1, -1, DIM)[:, 1:2 * n_heads:2])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and int(pos) == start + t + 1
    assert torch.equal(cap.data, eager.data) and int(cap.status) == 0


def test_captured_prompt(gpu):
    """A prompt's attention in a graph, both forms, replayed on other queries."""
    from vates_amd.attention import attend
    for T, pos0 in ((200, 50), (700, 3000)):
        log(f"case: kv8 captured prompt T={T} pos0={pos0}")
        cache = new_cache(2, pos0 + T, gpu)
        cache.write(0, *rows(55, 2, pos0 + T, gpu))
        q, gate = queries(56, T, 16, gpu)
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            attend(q, cache, pos0=pos0, gate=gate)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = attend(q, cache, pos0=pos0, gate=gate)
        for i in range(3):
            q.copy_(queries(57 + i, T, 16, gpu)[0])
            want = attend(q, cache, pos0=pos0, gate=gate)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_two_streams(gpu):
    """Calls on two streams at once, each with its own cache."""
    from vates_amd.attention import attend, norm_rope_append
    n_heads, n_kv, T = 16, 2, 4
    sets = []
    for i in range(2):
        qkv, qn, kn = projections(60 + i, 20 * T, n_heads, n_kv, gpu)
        sets.append((qkv, qn, kn, new_cache(n_kv, 5000, gpu), new_cache(n_kv, 5000, gpu), torch.cuda.Stream()))
        k, v = rows(62 + i, n_kv, 4800, gpu)
        for c in sets[-1][3:5]:
            c.write(0, k, v)
            c.length = 4800
    torch.cuda.synchronize()
    outs, wants = ([], []), ([], [])
    for t in range(0, 20 * T, T):
        for i, (qkv, qn, kn, c, _, st) in enumerate(sets):
            q = norm_rope_append(qkv[t:t + T], c, qn, kn, n_heads=n_heads, stream=st)
            outs[i].append(attend(q, c, stream=st))
    read = [s[3].read(4800, 4880, stream=s[5]) for s in sets]
    torch.cuda.synchronize()
    for i, (qkv, qn, kn, _, c, _) in enumerate(sets):
        for t in range(0, 20 * T, T):
            q = norm_rope_append(qkv[t:t + T], c, qn, kn, n_heads=n_heads)
            wants[i].append(attend(q, c))
        assert torch.equal(torch.cat(outs[i]), torch.cat(wants[i]))
        for a, b in zip(read[i], c.read(4800, 4880)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 4, 100])
def test_position_outside_the_capacity(gpu, T):
    """Clamped into it, and reported: the call equals that of the nearest position."""
    from vates_amd._lib import VMI_STATUS_BAD_POS
    from vates_amd.attention import attend, norm_rope_append
    n_heads, n_kv = 8, 2
    qkv, qn, kn = projections(70, T, n_heads, n_kv, gpu)
    k, v = rows(71, n_kv, 256, gpu)
    for at, use in ((256 - T + 1, 256 - T), (-1, 0), (2 ** 31 - 1, 256 - T), (-2 ** 31, 0), (256 - T, 256 - T)):
        log(f"case: kv8 position {at} T={T}")
        a, b = new_cache(n_kv, 256, gpu), new_cache(n_kv, 256, gpu)
        for c in (a, b):
            c.write(0, k, v)
        dev = torch.tensor([at], dtype=torch.int32, device=gpu)
        q = norm_rope_append(qkv, a, qn, kn, n_heads=n_heads, pos_device=dev)
        want = norm_rope_append(qkv, b, qn, kn, n_heads=n_heads, pos0=use)
        assert torch.equal(q, want) and torch.equal(a.data, b.data)
        assert int(a.status) == (VMI_STATUS_BAD_POS if at != use else 0)
        a.status.zero_()
        got = attend(q, a, pos_device=dev)
        assert int(a.status) == (VMI_STATUS_BAD_POS if at != use else 0)
        check_attend(got, q, b, use, None)


@pytest.mark.parametrize("T,pos0", [(1, 100), (4, 2000), (8, 20000), (90, 64), (700, 3000)])
@pytest.mark.parametrize("which", ["key", "value"])
def test_rows_that_are_not_finite(gpu, T, pos0, which):
    """A row with an infinity or NaN at position p: the tokens before it keep their
    results, those that see it are NaN in its kv head's query heads alone."""
    log(f"case: kv8 not finite T={T} pos0={pos0} {which}")
    from vates_amd.attention import attend
    n_heads, n_kv = 8, 2
    cache = new_cache(n_kv, pos0 + T, gpu)
    k, v = rows(80, n_kv, pos0 + T, gpu)
    q, gate = queries(81, T, n_heads, gpu)
    cache.write(0, k, v)
    clean = attend(q, cache, pos0=pos0, gate=gate)
    p = pos0 + T // 2
    for bad in (float("nan"), float("inf"), -float("inf")):
        t = (k if which == "key" else v).clone()
        t[1, p, 77] = bad
        cache.write(0, t if which == "key" else k, t if which == "value" else v)
        got = attend(q, cache, pos0=pos0, gate=gate)
        assert torch.equal(got[:, :4], clean[:, :4]) and torch.equal(got[:T // 2, 4:], clean[:T // 2, 4:])
        assert bool(torch.isnan(got[T // 2:, 4:]).all())
    # a query that is not finite is NaN, and no other row's business
    cache.write(0, k, v)
    q2 = q.clone()
    q2[T // 2, 3, 10] = float("inf")
    got = attend(q2, cache, pos0=pos0, gate=gate)
    assert bool(torch.isnan(got[T // 2, 3]).all())
    got[T // 2, 3] = clean[T // 2, 3]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("T,pos0", [(1, 300), (8, 5000), (100, 200), (700, 3000)])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 300.0])
def test_queries_of_any_size(gpu, T, pos0, size):
    """From scores that are all alike to one key that takes everything; heads of zeros."""
    log(f"case: kv8 queries of {size} T={T} pos0={pos0}")
    from vates_amd.attention import attend
    cache = new_cache(2, pos0 + T, gpu)
    cache.write(0, *rows(85, 2, pos0 + T, gpu))
    q, gate = queries(86, T, 8, gpu, size)
    q[:, 2] = 0.0
    check_attend(attend(q, cache, pos0=pos0, gate=gate), q, cache, pos0, gate)


@pytest.mark.parametrize("T,pos0", [(1, 300), (8, 5000), (100, 200), (700, 3000)])
def test_value_scales_far_apart(gpu, T, pos0):
    """Values of 2^-60 to 2^60, in rising and falling order, and rows of zeros."""
    log(f"case: kv8 value scales T={T} pos0={pos0}")
    from vates_amd.attention import attend
    n = pos0 + T
    k, v = rows(90, 2, n, gpu)
    v = torch.nn.functional.normalize(v.float(), dim=-1)
    e = torch.linspace(-60.0, 60.0, n, device=gpu)
    v = v * torch.exp2(torch.stack([e, -e]))[..., None]
    v[:, ::7] = 0.0
    v = v.bfloat16()
    cache = new_cache(2, n, gpu)
    cache.write(0, k, v)
    q, gate = queries(91, T, 8, gpu)
    check_attend(attend(q, cache, pos0=pos0, gate=gate), q, cache, pos0, gate)


@pytest.mark.parametrize("T", [1, 4, 100])
def test_one_position(gpu, T):
    """From an empty cache: the first token sees itself alone and gives its value back."""
    from vates_amd.attention import attend
    cache = new_cache(2, 128, gpu)
    k, v = rows(95, 2, T, gpu)
    cache.write(0, k, v)
    q, _ = queries(96, T, 8, gpu)
    got = attend(q, cache, pos0=0)
    want = held(v)[:, :1].transpose(0, 1).repeat_interleave(4, 1).to(gpu)
    # the probability is 1, its sum 1: fp16's roundings of the scale and the product, then bf16's
    assert bool(((got[0].float() - want[0]).abs() <= (2.0 ** -8 + 3 * 2.0 ** -11) * want[0].abs()).all())


def test_no_tokens(gpu):
    from vates_amd.attention import attend, norm_rope_append
    cache = new_cache(2, 64, gpu)
    before = cache.data.clone()
    k = torch.zeros((2, 0, DIM), dtype=torch.bfloat16, device=gpu)
    w = torch.ones(DIM, dtype=torch.bfloat16, device=gpu)
    cache.write(64, k, k)
    assert cache.read(5, 5)[0].shape == (2, 0, DIM)
    q = norm_rope_append(torch.zeros((0, 20 * DIM), device=gpu), cache, w, w, n_heads=8)
    assert q.shape == (0, 8, DIM) and cache.length == 0
    assert attend(q, cache).shape == (0, 8, DIM)
    assert torch.equal(cache.data, before)


def test_python_refuses_on_the_device(gpu):
    from vates_amd._lib import VmiError
    from vates_amd.attention import attend, norm_rope_append
    cache = new_cache(2, 64, gpu)
    k, v = rows(97, 2, 4, gpu)
    q, gate = queries(98, 4, 8, gpu)
    qkv, qn, kn = projections(99, 4, 8, 2, gpu)
    pos = torch.zeros(1, dtype=torch.int32, device=gpu)
    for call in (lambda: cache.write(61, k, v), lambda: cache.write(-1, k, v), lambda: cache.write(0, k.float(), v),
                 lambda: cache.write(0, k, v[:, :3]), lambda: cache.write(0, k[:1], v[:1]), lambda: cache.write(0, k.cpu(), v),
                 lambda: cache.write(0, k.transpose(1, 2), v), lambda: cache.read(0, 65), lambda: cache.read(3, 2),
                 lambda: cache.read(0, 4, dtype=torch.float16),
                 lambda: attend(q, cache, pos0=61), lambda: attend(q, cache, pos0=-1), lambda: attend(q, cache),
                 lambda: attend(q.float(), cache, pos0=0), lambda: attend(q[:, :7], cache, pos0=0),
                 lambda: attend(q, cache, pos0=0, gate=gate[:3]), lambda: attend(q, cache, pos0=0, gate=gate.bfloat16()),
                 lambda: attend(q, cache, pos0=0, out=q[:2]), lambda: attend(q, cache, pos_device=pos.long()),
                 lambda: attend(q, cache, pos_device=pos.cpu()), lambda: attend(q[:, :, :128], cache, pos0=0),
                 lambda: norm_rope_append(qkv, cache, qn, kn, n_heads=7), lambda: norm_rope_append(qkv, cache, qn, kn, n_heads=8, pos0=61),
                 lambda: norm_rope_append(qkv.bfloat16(), cache, qn, kn, n_heads=8),
                 lambda: norm_rope_append(qkv, cache, qn[:128], kn, n_heads=8),
                 lambda: norm_rope_append(qkv, cache, qn, kn, n_heads=8, rope_dim=63),
                 lambda: norm_rope_append(qkv, cache, qn, kn.float(), n_heads=8)):
        with pytest.raises(VmiError):
            call()
    torch.cuda.synchronize()
    assert cache.length == 0 and not bool(cache.data.any())


def test_a_cache_past_four_gib(gpu):
    """The last positions of the last head lie behind 2^32 bytes; every other row is
    zero, so that the sum over a million positions is known: with w(p) = exp(q k(p) / 16),
    out = sum w(p) v(p) / (zeros + sum w(p))."""
    n_kv, max_len, n = 8, 1 << 20, 40
    log(f"case: kv8 cache of {n_kv * max_len // 32 * 16640 / 2 ** 30:.2f} GiB")
    from vates_amd.attention import attend
    cache = new_cache(n_kv, max_len, gpu)
    assert cache.data.numel() > 1 << 32
    k, v = rows(100, n_kv, n, gpu)
    start = max_len - n
    cache.write(start, k, v)
    gk, gv = cache.read(start, max_len, dtype=torch.float32)
    assert same(gk, held(k)) and same(gv, held(v))
    assert not bool(cache.read(0, 64)[0].any()) and not bool(cache.read(start - 64, start)[1].any())
    q, _ = queries(101, 2, n_kv, gpu, 4.0)
    got = attend(q, cache, pos0=max_len - 2)
    hk, hv = held(k).double().cpu(), held(v).double().cpu()
    for h in range(n_kv):
        for t in range(2):
            see = n - 1 + t
            qq = q[t, h].double().cpu()
            w = torch.exp(hk[h, :see] @ qq / 16.0)
            den = start + w.sum()
            want, A = (w @ hv[h, :see]) / den, (w @ hv[h, :see].abs()) / den
            d = float(qq.abs().max() * hk[h].abs().sum(-1).max() / (16 * 65024) + 5 * 2.0 ** -24 * qq.abs().sum() * hk[h].abs().max() / 16)
            tol = 2.0 ** -8 * want.abs() + (3 * 2.0 ** -11 + 2 * d + 2.0 ** -16) * A + (n * 2.0 ** -39 + 2.0 ** -33) * hv[h].abs().max()
            assert bool(((got[t, h].double().cpu() - want).abs() <= tol).all()), (h, t)
    del cache
    torch.cuda.empty_cache()


def test_strides_that_no_step_takes(gpu):
    """One kv head, one position, one token: the stride between them may be anything."""
    from vates_amd.attention import attend
    k, v = rows(110, 1, 4, gpu)
    a, b = new_cache(1, 64, gpu), new_cache(1, 64, gpu)
    a.write(0, k, v)
    b.write(0, k.as_strided((1, 4, DIM), (3, DIM, 1)), v)
    for t in range(4):
        b.write(t, k[:, t:t + 1].as_strided((1, 1, DIM), (5, 7, 1), t * DIM), v[:, t:t + 1])
    assert torch.equal(a.data, b.data)
    q, gate = queries(111, 1, 8, gpu)
    want = attend(q, a, pos0=3, gate=gate)
    assert torch.equal(attend(q, a, pos0=3, gate=gate.as_strided((1, 8, DIM), (1, DIM, 1))), want)


@pytest.mark.parametrize("T,pos0", [(9, 40), (100, 0), (100, 5000), (700, 31)])
def test_device_position_far_below_the_capacity(gpu, T, pos0):
    """The form and its parts are chosen by the capacity, the work by the position."""
    log(f"case: kv8 T={T} at {pos0} of 200,000")
    from vates_amd.attention import attend
    cache = new_cache(2, 200000, gpu)
    cache.data.fill_(255)
    cache.write(0, *rows(120, 2, pos0 + T, gpu))
    q, gate = queries(121, T, 16, gpu)
    pos = torch.tensor([pos0], dtype=torch.int32, device=gpu)
    check_attend(attend(q, cache, pos_device=pos, gate=gate), q, cache, pos0, gate)
    assert int(cache.status) == 0
