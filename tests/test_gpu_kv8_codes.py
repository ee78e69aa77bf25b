"""Rows of every pair of bf16 mantissas through the store's kernel, bit for bit (the
restated steps: tests/test_kv8_codes.py)."""
import pytest
import torch

from test_gpu_kv8 import held, log, new_cache, same

pytestmark = pytest.mark.gpu


def test_every_pair_of_mantissas(gpu):
    """Row (ma, gap): its largest element ma 2^e, beside it mx 2^(e - gap) of both signs
    for every mx that is no larger; a kv head for each e."""
    log("case: kv8 every pair of mantissas")
    m = torch.arange(128, 256, dtype=torch.float64)
    heads = []
    for e in (-110, -60, 0, 60, 119):
        top = (m * 2.0 ** e).view(128, 1, 1)
        x = (m * 2.0 ** e).view(1, 1, 128) * 2.0 ** -torch.arange(10, dtype=torch.float64).view(1, 10, 1)
        x = torch.where(x <= top, x, torch.zeros_like(x))
        row = torch.cat([-x, x], -1)
        row[..., 0] = top[..., 0]
        heads.append(row.view(-1, 256))
    k = torch.stack(heads)
    assert torch.equal(k.bfloat16().double(), k)
    k = k.bfloat16().to(gpu)
    cache = new_cache(k.shape[0], k.shape[1], gpu)
    cache.write(0, k, k.flip(2))
    gk, gv = cache.read(0, k.shape[1], dtype=torch.float32)
    assert same(gk, held(k)) and same(gv, held(k.flip(2)))
