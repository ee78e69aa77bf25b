"""The pass that forms a batch's heads, at other thetas than the models': bars of
tests/test_gpu_kv8.py (half a bf16 step and 2^-20 of the row's largest magnitude; half a
code step and 2^-20 of it)."""
import pytest
import torch

from test_gpu_kv8 import heads64, log, new_cache, projections

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("theta,rd,pos0", [(1.0, 64, 200000), (0.5, 64, 262000), (0.01, 32, 5000), (1e-3, 256, 1000), (1e4, 128, 100)])
def test_heads_at_any_theta(gpu, theta, rd, pos0):
    log(f"case: kv8 heads theta={theta} rope={rd} pos0={pos0}")
    from vates_amd.attention import norm_rope_append
    T, n_heads, n_kv = 5, 4, 2
    qkv, qn, kn = projections(401, T, n_heads, n_kv, gpu)
    cache = new_cache(n_kv, pos0 + T, gpu)
    q = norm_rope_append(qkv, cache, qn, kn, n_heads=n_heads, rope_dim=rd, rope_theta=theta, pos0=pos0)
    theta = float(torch.tensor(theta, dtype=torch.float32))   # as the call takes it
    fq, fk, _ = heads64(qkv, qn, kn, n_heads, n_kv, rd, theta, 1e-6, pos0)
    big = fq.abs().amax(-1, keepdim=True)
    assert ((q.double().cpu() - fq).abs() <= 2 ** -8 * fq.abs() + 2 ** -20 * big).all()
    k, want = cache.keys(pos0, pos0 + T, dtype=torch.float32).double().cpu(), fk.transpose(0, 1)
    a = want.abs().amax(-1, keepdim=True)
    assert ((k - want).abs() <= a / 254 + 2 ** -20 * a).all()
