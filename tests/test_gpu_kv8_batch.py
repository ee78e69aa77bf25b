"""Attention of batches (T * n_heads / n_kv <= 64) over the 8-bit KV cache, by bars of
their own: such a call rounds once to fp16, the probability times its value's
scale over the largest that the row has seen, times 2^14.  So, beside what
test_gpu_kv8_visible counts for every form (half a bf16 step of the output, the
scores' errors, exp2 and fp32 sums), one rounding of 2^-11 A where prompts have three, below
fp16's normal range 2^-25 of 2^14 times V over n positions, n 2^-39 V, and no other term
in V: the sums are of the codes themselves."""
import pytest
import torch

from test_gpu_kv8 import DIM, log, new_cache, queries, rows
from test_gpu_kv8_visible import attend64

pytestmark = pytest.mark.gpu


def check(got, q, cache, pos0):
    k, v = cache.read(0, pos0 + q.shape[0], dtype=torch.float32)
    want, tol = attend64(q, k, v, pos0, roundings=1, scales=0.0)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("T,pos0,n_heads,n_kv", [(1, 0, 16, 2), (1, 1, 16, 2), (4, 29, 16, 2), (8, 1000, 16, 2), (1, 31, 4, 4),
                                                 (2, 5000, 5, 1), (3, 700, 6, 2), (1, 9999, 16, 2), (8, 20000, 8, 8),
                                                 (7, 4090, 32, 4), (16, 3000, 8, 2), (64, 100, 1, 1), (2, 262000, 16, 2)])
def test_ordinary_rows(gpu, T, pos0, n_heads, n_kv):
    log(f"case: kv8 batch bars T={T} pos0={pos0} {n_heads}/{n_kv}")
    from vates_amd.attention import attend
    cache = new_cache(n_kv, pos0 + T, gpu)
    cache.write(0, *rows(301, n_kv, pos0 + T, gpu))
    q, _ = queries(302, T, n_heads, gpu)
    check(attend(q, cache, pos0=pos0), q, cache, pos0)


@pytest.mark.parametrize("T,pos0,n_heads,n_kv", [(1, 7, 16, 2), (1, 40, 16, 2), (8, 33, 16, 2), (4, 100, 4, 4), (5, 300, 8, 1)])
@pytest.mark.parametrize("size", [2.0 ** -10, 2.0 ** -16, 2.0 ** -20])
def test_small_rows_beside_a_large_one(gpu, T, pos0, n_heads, n_kv, size):
    """A row that is large in one dim and zero in the others takes nothing from what
    the small rows give to those.  (Held as codes + 128, with the 128 taken off at the
    end, it added 128 times its scale to every dim's sum, 2^-24 of which is more than they are.)"""
    log(f"case: kv8 batch small rows T={T} pos0={pos0} {n_heads}/{n_kv} size={size:g}")
    from vates_amd.attention import attend
    n = pos0 + T
    k, _ = rows(303, n_kv, n, gpu)
    g = torch.Generator(device=gpu).manual_seed(304)
    v = (torch.randn((n_kv, n, DIM), generator=g, device=gpu) * size).bfloat16()
    v[:, 3] = 0.0
    v[:, 3, 0] = 127.0
    cache = new_cache(n_kv, n, gpu)
    cache.write(0, k, v)
    q, _ = queries(305, T, n_heads, gpu, 0.1)
    check(attend(q, cache, pos0=pos0), q, cache, pos0)
