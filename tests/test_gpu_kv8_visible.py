"""Attention over the 8-bit KV cache: what a token may not see does not reach its
result, whatever its size.

Bars, for the output o = sum p v of one row with A = sum p |v| and V the largest |v|
among the positions that this row sees (fp16 and bf16 roundings counted as half steps):
* half a bf16 step of o: 2^-8 |o|.
* three roundings to fp16, 2^-11 A each: a probability, a value's scale, the scale
  times the code (a record that is not seen to its end takes one, of the
  probability times the scale).
* what lies below fp16's normal range: a weight of at most 2^8 to 2^14, off by 2^-25, times
  operands of at most 127 * 2^8: n 2^-39 V over n positions; scales held to
  2^-25 where the largest is 2^8: 2^-33 V.
* a score's error d shifts p by d, on numerator and denominator alike: 2 d A.  Query
  elements are off by at most max|q| / 65024, and five fp32 roundings of scores of at
  most sum|q| max|k| / 16 follow: d <= max|q| sum|k| / (16 * 65024) + 5 * 2^-24 sum|q|
  max|k| / 16, with the keys that the row sees.
* exp2, sums and merge in fp32: 2^-16 A."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import DIM, log, new_cache, queries, rows

pytestmark = pytest.mark.gpu


def attend64(q, k, v, pos0, roundings=3, scales=2.0 ** -33):
    """(outputs, bars) for fp32 rows k, v [n_kv, L, 256]; every maximum over the row's own positions.
    roundings: to fp16; scales: of V, where scales are held by themselves."""
    T, nh, _ = q.shape
    G = nh // k.shape[0]
    dev = k.device
    out = torch.empty((T, nh, DIM), dtype=torch.float64, device=dev)
    tol = torch.empty_like(out)
    L = k.shape[1]
    see = torch.arange(L, device=dev)[None] <= (pos0 + torch.arange(T, device=dev))[:, None]
    last = pos0 + torch.arange(T, device=dev)
    n = last[:, None] + 1
    for h in range(nh):
        qq, kk, vv = q[:, h].double(), k[h // G].double(), v[h // G].double()
        ksum = kk.abs().sum(-1).cummax(0).values[last][:, None]
        kmax = kk.abs().amax(-1).cummax(0).values[last][:, None]
        vmax = vv.abs().amax(-1).cummax(0).values[last][:, None]
        p = torch.softmax((torch.matmul(qq, kk.t().contiguous()) / 16.0).masked_fill(~see, -np.inf), -1)
        o, A = torch.matmul(p, vv), torch.matmul(p, vv.abs())
        d = qq.abs().amax(-1, keepdim=True) * ksum / (16 * 65024) + 5 * 2.0 ** -24 * qq.abs().sum(-1, keepdim=True) * kmax / 16
        out[:, h] = o
        tol[:, h] = 2.0 ** -8 * o.abs() + (roundings * 2.0 ** -11 + 2 * d + 2.0 ** -16) * A + (n * 2.0 ** -39 + scales) * vmax
    return out, tol


def check(got, q, cache, pos0):
    k, v = cache.read(0, pos0 + q.shape[0], dtype=torch.float32)
    want, tol = attend64(q, k, v, pos0)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


# both forms of prompts: few and many heads a kv head, one tile, tiles in pairs, a tile without a partner
PROMPTS = [(9, 3, 16, 2), (100, 0, 16, 2), (100, 205, 8, 2), (130, 0, 1, 1), (333, 1000, 6, 2), (700, 3000, 16, 2),
           (1111, 2000, 12, 4), (1024, 4096, 4, 4), (130, 40000, 8, 1)]


@pytest.mark.parametrize("T,pos0,n_heads,n_kv", PROMPTS)
@pytest.mark.parametrize("size", [2.0 ** 24, 2.0 ** 40, 2.0 ** 100])
def test_a_later_token_of_any_size(gpu, T, pos0, n_heads, n_kv, size):
    """A position's value (or key) that much larger: the tokens before it keep their
    results bit for bit, every token stays within its own bar."""
    log(f"case: kv8 visible T={T} pos0={pos0} {n_heads}/{n_kv} size={size:g}")
    from vates_amd.attention import attend
    cache = new_cache(n_kv, pos0 + T, gpu)
    k, v = rows(201, n_kv, pos0 + T, gpu)
    q, _ = queries(202, T, n_heads, gpu)
    cache.write(0, k, v)
    clean = attend(q, cache, pos0=pos0)
    check(clean, q, cache, pos0)
    for t in (T - 1, T // 2, 1):
        big = v.clone()
        big[:, pos0 + t] = (big[:, pos0 + t].float() * size).bfloat16()
        cache.write(0, k, big)
        got = attend(q, cache, pos0=pos0)
        check(got, q, cache, pos0)
        assert torch.equal(got[:t], clean[:t])
    key = k.clone()
    key[:, pos0 + T // 2] = (key[:, pos0 + T // 2].float() * size).bfloat16()
    cache.write(0, key, v)
    assert torch.equal(attend(q, cache, pos0=pos0)[:T // 2], clean[:T // 2])


@pytest.mark.parametrize("T,pos0,n_heads,n_kv", PROMPTS + [(1, 40, 16, 2), (8, 1000, 16, 2), (5, 70000, 16, 2)])
def test_what_lies_behind_the_last_token(gpu, T, pos0, n_heads, n_kv):
    """Rejected drafts, another sequence's rows, memory that was never written: finite
    rows of any size and infinite scales behind the last token change nothing."""
    log(f"case: kv8 behind T={T} pos0={pos0} {n_heads}/{n_kv}")
    from vates_amd.attention import attend
    n = pos0 + T
    cache = new_cache(n_kv, n + 70, gpu)
    cache.write(0, *rows(211, n_kv, n, gpu))
    q, gate = queries(212, T, n_heads, gpu)
    clean = attend(q, cache, pos0=pos0, gate=gate)
    rest = cache.max_len - n
    k, v = rows(213, n_kv, rest, gpu)
    for size in (2.0 ** 30, 1e30):
        cache.write(n, (k.float() * size).bfloat16(), (v.float() * size).bfloat16())
        assert torch.equal(attend(q, cache, pos0=pos0, gate=gate), clean)
    scales = cache.data.view(n_kv, -1, 16640)[:, :, 16384:].view(torch.float32)   # 32 key, 32 value scales a record
    for at in range(n, cache.max_len):
        scales[:, at // 32, at % 32] = float("inf")
        scales[:, at // 32, 32 + at % 32] = float("inf")
    assert torch.equal(attend(q, cache, pos0=pos0, gate=gate), clean)
    pos = torch.tensor([pos0], dtype=torch.int32, device=gpu)
    dev = attend(q, cache, pos_device=pos, gate=gate)
    cache.write(n, torch.zeros_like(k), torch.zeros_like(v))
    assert torch.equal(attend(q, cache, pos_device=pos, gate=gate), dev)
