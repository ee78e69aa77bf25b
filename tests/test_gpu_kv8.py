"""The 8-bit KV cache against plain forms in 64 bits: rows stored and read back,
a batch's heads formed and appended, attention over the cache.

Bars, from the arithmetic (written here before the first run):
* stored rows: bit for bit.  s = fp32(a / 127) and the codes of exact arithmetic
  (vmi_kv8.hip says why one fp32 division finds them), so fp32(s c) is fixed.
* queries: half a bf16 step, 2^-8 |x|, and the fp32 work in front of it: RMS,
  weight, rotation, about ten roundings of 2^-24 on terms of at most the row's
  largest magnitude times sqrt(2): 2^-20 of that magnitude.
* appended keys and values: half a code step of the 64-bit row, a / 254, and
  2^-20 a for the same fp32 work (keys) or the division (values).
* attention, per output o = sum p v with A = sum p |v|: half a bf16 step of o,
  2^-8 |o|; up to three roundings to fp16, 2^-11 A each: a probability times its
  value's scale, or (prompts) the probability, the scale, and the scale times the
  code; what lies below fp16's normal range, 2^-25 of 2^14 times the largest value
  scale times 127 summed over the keys, n 2^-39 max |v|, and (prompts) scales below
  2^-22 of the largest, held to 2^-25 where that is 2^8: 127 * 2^-25 / (127 * 2^8) =
  2^-33 max |v|; each score's error d shifts p by d, on numerator and denominator
  alike, 2 d A.  A query is rounded to integers of its largest element / 32512, so
  each element is off by at most that / 65024 and a score by max|q| sum|k| / (16 *
  65024); the integer sums are exact, and their conversion, the key's scale, the row's
  factor and the subtraction round five times by 2^-24 of scores of at most sum|q|
  max|k| / 16: d <= max|q| sum|k| / (16 * 65024) + 5 * 2^-24 sum|q| max|k| / 16.
  Hardware exp2, sums and merge: 2^-16 A.  Batches multiply codes + 128 and take 128
  times the probabilities off: sums of up to 255 / 127 max |v|, two roundings of 2^-24 a
  record of a wave's, of which n positions give n / 4096 + 1 at most (eight kv heads on
  256 CUs: 128 waves each): (n / 4096 + 1) 2^-22 max |v|.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DIM = 256


def log(msg):
    print(msg, flush=True)


def rows(seed, n_kv, n, gpu):
    """Keys and values bf16 [n_kv, n, 256]: strong channels, sizes that vary by token."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    k = torch.randn((n_kv, n, DIM), generator=g, device=gpu)
    k[..., 7] *= 8.0
    v = torch.randn((n_kv, n, DIM), generator=g, device=gpu) * torch.exp(torch.randn((n_kv, n, 1), generator=g, device=gpu))
    return k.bfloat16(), v.bfloat16()


def held(x):
    """What bf16 rows are held as: fp32(s c)."""
    d = x.double().cpu()
    a = d.abs().amax(-1, keepdim=True)
    c = torch.round(127.0 * d / torch.where(a > 0, a, torch.ones_like(a)))
    s = a.float() / 127.0
    s = torch.where(torch.isfinite(a), s, torch.full_like(s, float("nan")))
    c = torch.where(torch.isfinite(a), c, torch.zeros_like(c))
    return s * c.float()


def same(a, b):
    a, b = a.cpu(), b.cpu()
    return bool(torch.equal(torch.nan_to_num(a, nan=1e9), torch.nan_to_num(b, nan=1e9)))


def new_cache(n_kv, max_len, gpu):
    from vates_amd.attention import KVCache8
    return KVCache8(n_kv, max_len, gpu)


# ------------------------------------------------------------- store and load
@pytest.mark.parametrize("n_kv,start,n,order", [(2, 0, 1, "heads"), (1, 31, 1, "heads"), (2, 5, 3, "tokens"), (3, 0, 32, "heads"),
                                                (2, 32, 64, "tokens"), (2, 7, 130, "heads"), (4, 1000, 777, "tokens"),
                                                (1, 29, 8, "heads"), (5, 16, 9, "tokens")])
def test_write_then_read(gpu, n_kv, start, n, order):
    log(f"case: kv8 write n_kv={n_kv} start={start} n={n} {order}")
    cache = new_cache(n_kv, start + n + 40, gpu)
    bk, bv = rows(1, n_kv, cache.max_len, gpu)
    cache.write(0, bk, bv)
    before = cache.data.clone()
    k, v = rows(2, n_kv, n, gpu)
    if order == "tokens":
        k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
    cache.write(start, k, v)
    for dt in (torch.float32, torch.bfloat16):
        gk, gv = cache.read(0, cache.max_len, dtype=dt)
        for got, base, new in ((gk, bk, k), (gv, bv, v)):
            want = held(base)
            want[:, start:start + n] = held(new)
            assert same(got, want.to(dt))
    assert same(cache.keys(start, start + n, dtype=torch.float32), held(k))
    assert same(cache.values(start, start + n), held(v).bfloat16())
    # written again in other pieces: the same bytes
    after = cache.data.clone()
    cache.data.copy_(before)
    for i in range(0, n, 5):
        cache.write(start + i, k[:, i:i + 5], v[:, i:i + 5])
    torch.cuda.synchronize()
    assert torch.equal(cache.data, after)
    assert cache.read(3, 3)[0].shape == (n_kv, 0, DIM)


def test_rows_at_the_ends_of_the_range(gpu):
    """Zeros, subnormals, the largest finite values, exact ties, infinities and NaN."""
    log("case: kv8 special rows")
    k = torch.zeros((1, 9, DIM), dtype=torch.bfloat16, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(3)
    k[0, 1] = (torch.randn(DIM, generator=g, device=gpu) * 1e-39).bfloat16()          # subnormal in bf16
    k[0, 2] = (torch.randn(DIM, generator=g, device=gpu) * 8e37).bfloat16()
    k[0, 2, 5] = 3.3895313892515355e38
    k[0, 3, :128] = torch.arange(-64, 64, device=gpu).bfloat16() + 0.5                # ties against a = 127
    k[0, 3, 200] = 127.0
    k[0, 4] = 1.0
    k[0, 4, 9] = float("inf")
    k[0, 5] = -2.0
    k[0, 5, 255] = float("nan")
    k[0, 6, 0] = -7e-39
    k[0, 7] = torch.randn(DIM, generator=g, device=gpu).bfloat16()
    k[0, 8] = -1.0
    cache = new_cache(1, 32, gpu)
    cache.write(0, k, k.flip(1))
    gk, gv = cache.read(0, 9, dtype=torch.float32)
    want = held(k)
    assert torch.isnan(want[0, 4]).all() and torch.isnan(want[0, 5]).all() and torch.isfinite(want[0, [0, 1, 2, 3, 6, 7, 8]]).all()
    assert same(gk, want) and same(gv, want.flip(1))


# ------------------------------------------------------------------- heads
def heads64(qkv, q_norm, k_norm, n_heads, n_kv, rd, theta, eps, pos0):
    x = qkv.double().cpu().view(qkv.shape[0], -1, DIM)
    T = x.shape[0]
    pos = torch.arange(pos0, pos0 + T, dtype=torch.float64)

    def form(y, w):
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double().cpu()
        out = y.clone()
        for i in range(rd // 2):
            ang = pos * theta ** (-2.0 * i / rd)
            c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
            a, b = y[..., i], y[..., i + rd // 2]
            out[..., i], out[..., i + rd // 2] = a * c - b * s, b * c + a * s
        return out

    return form(x[:, 0:2 * n_heads:2], q_norm), form(x[:, 2 * n_heads:2 * n_heads + n_kv], k_norm), x[:, 2 * n_heads + n_kv:]


def projections(seed, T, n_heads, n_kv, gpu):
    g = torch.Generator(device=gpu).manual_seed(seed)
    qkv = torch.randn((T, (2 * n_heads + 2 * n_kv) * DIM), generator=g, device=gpu) * torch.exp(
        torch.randn((T, 1), generator=g, device=gpu))
    w = [(1.0 + 0.2 * torch.randn(DIM, generator=g, device=gpu)).bfloat16() for _ in range(2)]
    return qkv, w[0], w[1]


@pytest.mark.parametrize("T,pos0,n_heads,n_kv,rd", [(1, 0, 16, 2, 64), (4, 8190, 16, 2, 64), (8, 27, 4, 4, 128), (1, 262143, 5, 1, 256),
                                                    (33, 250000, 6, 2, 32), (100, 3, 16, 2, 64), (3, 30, 2, 1, 0), (2, 9, 2, 2, 10),
                                                    (9, 1234, 3, 3, 2)])
def test_heads(gpu, T, pos0, n_heads, n_kv, rd):
    log(f"case: kv8 heads T={T} pos0={pos0} {n_heads}/{n_kv} rope={rd}")
    from vates_amd.attention import norm_rope_append
    qkv, qn, kn = projections(11, T, n_heads, n_kv, gpu)
    cache = new_cache(n_kv, pos0 + T, gpu)
    q = norm_rope_append(qkv, cache, qn, kn, n_heads=n_heads, rope_dim=rd, pos0=pos0)
    assert cache.length == pos0 + T
    fq, fk, fv = heads64(qkv, qn, kn, n_heads, n_kv, rd, 1e7, 1e-6, pos0)
    big = fq.abs().amax(-1, keepdim=True)
    assert ((q.double().cpu() - fq).abs() <= 2 ** -8 * fq.abs() + 2 ** -20 * big).all()
    k, v = cache.read(pos0, pos0 + T, dtype=torch.float32)
    for got, want in ((k, fk), (v, fv)):
        want = want.transpose(0, 1)
        a = want.abs().amax(-1, keepdim=True)
        assert ((got.double().cpu() - want).abs() <= a / 254 + 2 ** -20 * a).all()
    if pos0:
        assert not cache.read(0, pos0, dtype=torch.float32)[0].any()
    # in other pieces: the same queries and bytes
    c2 = new_cache(n_kv, pos0 + T, gpu)
    c2.length = pos0
    parts = [norm_rope_append(qkv[i:i + 3].contiguous(), c2, qn, kn, n_heads=n_heads, rope_dim=rd) for i in range(0, T, 3)]
    assert torch.equal(torch.cat(parts), q) and torch.equal(c2.data, cache.data)
    # and with the position on the device
    c3 = new_cache(n_kv, pos0 + T, gpu)
    q3 = norm_rope_append(qkv, c3, qn, kn, n_heads=n_heads, rope_dim=rd,
                          pos_device=torch.tensor([pos0], dtype=torch.int32, device=gpu))
    assert torch.equal(q3, q) and torch.equal(c3.data, cache.data) and int(c3.status) == 0


# --------------------------------------------------------------- attention
def attend64(q, k, v, pos0, gate):
    """(outputs, bound of the error) for fp32 rows k, v [n_kv, L, 256], on k's device."""
    T, nh, _ = q.shape
    G = nh // k.shape[0]
    q, dev = q.double(), k.device
    out, tol = torch.empty((T, nh, DIM), dtype=torch.float64, device=dev), torch.empty((T, nh, DIM), dtype=torch.float64, device=dev)
    at = torch.arange(k.shape[1], device=dev)
    see = at[None] <= (pos0 + torch.arange(T, device=dev))[:, None]
    for h in range(nh):
        kk, vv = k[h // G].double(), v[h // G].double()
        x = torch.matmul(q[:, h], kk.t().contiguous()) / 16.0
        p = torch.softmax(x.masked_fill(~see, -np.inf), -1)
        o, A = torch.matmul(p, vv), torch.matmul(p, vv.abs())
        qa = q[:, h].abs()
        d = qa.amax(-1, keepdim=True) * kk.abs().sum(-1).max() / (16 * 65024) + \
            5 * 2.0 ** -24 * qa.sum(-1, keepdim=True) * kk.abs().max() / 16
        n = see.sum(-1, keepdim=True)
        tol[:, h] = 2.0 ** -8 * o.abs() + (3 * 2.0 ** -11 + 2 * d + 2.0 ** -16) * A + (n * 2.0 ** -39 + 2.0 ** -33 + (n / 4096 + 1) * 2.0 ** -22) * vv.abs().max()
        out[:, h] = o
    if gate is not None:
        s = torch.sigmoid(gate.double().to(dev))
        out, tol = out * s, tol * s + 2.0 ** -20 * out.abs() * s
    return out, tol


def queries(seed, T, n_heads, gpu, size=1.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return (torch.randn((T, n_heads, DIM), generator=g, device=gpu) * size).bfloat16(), \
        2.0 * torch.randn((T, n_heads, DIM), generator=g, device=gpu)


CASES = [(1, 0, 16, 2, True), (1, 1, 16, 2, False), (4, 29, 16, 2, True), (8, 1000, 16, 2, True), (1, 31, 4, 4, False),
         (2, 5000, 5, 1, True), (3, 700, 6, 2, False), (1, 9999, 16, 2, True), (8, 20000, 8, 8, False), (7, 4090, 32, 4, True),
         (9, 0, 16, 2, True), (16, 3000, 16, 2, False), (40, 33, 16, 2, True), (65, 0, 1, 1, False), (200, 1234, 16, 2, True),
         (777, 0, 16, 2, True), (1500, 2000, 6, 2, False)]


@pytest.mark.parametrize("T,pos0,n_heads,n_kv,gated", CASES)
def test_attend(gpu, T, pos0, n_heads, n_kv, gated):
    log(f"case: kv8 attend T={T} pos0={pos0} {n_heads}/{n_kv} gate={gated}")
    from vates_amd.attention import attend
    cache = new_cache(n_kv, pos0 + T + 70, gpu)
    cache.data.fill_(255)                      # what lies behind the last position: NaN scales
    cache.write(0, *rows(21, n_kv, pos0 + T, gpu))
    q, gate = queries(22, T, n_heads, gpu)
    gate = gate if gated else None
    got = attend(q, cache, pos0=pos0, gate=gate)
    k, v = cache.read(0, pos0 + T, dtype=torch.float32)
    want, tol = attend64(q, k, v, pos0, gate)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
