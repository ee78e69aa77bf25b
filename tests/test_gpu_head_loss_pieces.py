"""Gradients of the loss under a head where they are put together: g's second part, several
pieces of the vocabulary by several blocks of tokens, the benchmark's whole head.

Bars as in test_gpu_head_loss.py (u = 2^-24), g's rounding apart: up to 64 tokens g is two
bf16 parts, off by half a step of the second, 2^-8 of the first's 2^-8 (2^-16 |g|); above, one, 2^-8 |g|.
"""
import pytest

from test_gpu_head_loss import U, _inputs, _reference, _within

pytestmark = pytest.mark.gpu


def log(msg):
    print(msg, flush=True)


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65])
def test_both_parts_of_g(gpu, T):
    """Up to 64 tokens both of g's parts reach the head's gradient and dx.  One hidden value is the same in the
    whole head and 0 in x: its dx is the sum of g alone, d_lse, where a part left out stands bare."""
    import torch
    from vates_amd.head import head_loss, head_loss_grad
    H, V, j = 64, 1003, 5
    log(f"case: parts of g T={T}")
    x, w, y, a, _ = _inputs(gpu, T, H, V, seed=7)
    x[:, j], w[:, j] = 0.0, 1.0
    b = torch.zeros_like(a)
    loss, lse = head_loss(x, w, y)
    dx, dw = head_loss_grad(x, w, y, lse, a, b, dweight_dtype=torch.float32)
    xd, wd, ad = x.double(), w.double(), a.double()[:, None]
    z = xd @ wd.t().contiguous()
    ez = H * U * (xd.abs() @ wd.abs().t().contiguous())
    p = torch.exp(z - torch.logsumexp(z, -1)[:, None])
    one = torch.zeros_like(z).scatter_(1, y[:, None], 1.0)
    g = ad * (p - one)
    eg = (2.0 ** -16 if T <= 64 else 2.0 ** -8) * g.abs() + ad * p * (2 * ez + 2.0 ** -15) + U * ad * one
    want = g.t().contiguous() @ xd
    _within(dw, (want, eg.t().contiguous() @ xd.abs() + 2 * T * U * (g.abs().t().contiguous() @ xd.abs()) + U * want.abs()), "dweight")
    want = g @ wd
    bound = eg @ wd.abs() + 2 * V * U * (g.abs() @ wd.abs())
    _within(dx, (want, bound + 2.0 ** -8 * (want.abs() + bound)), "dx")


# tokens, vocabulary rows, left out, a block's tokens where g's rows end inside a step of 64
PIECES = [(4100, 69800, 9, None), (4100, 150700, 9, None), (3363, 150700, 11, 224), (2390, 151936, 1, 160)]


@pytest.mark.parametrize("T,V,ignored,bn", PIECES)
def test_pieces_by_blocks(gpu, monkeypatch, T, V, ignored, bn):
    """Two and three pieces, the last one shorter and ragged, by eight blocks of tokens and more: dx's sums
    over the pieces, the last piece's own strips, g's rows of zeros behind a last block of 160 or 224 tokens, which every piece reads.
    The workspace held NaN; that there are several pieces shows in its size, below g's of the whole vocabulary."""
    import torch
    import vates_amd.head as head
    H = 64
    log(f"case: pieces by blocks T={T} V={V}")
    held = []

    def scratch(n, dev):
        held.append(torch.full((n,), 255, dtype=torch.uint8, device=dev))
        return held[-1]

    monkeypatch.setattr(head, "scratch", scratch)
    x, w, y, a, b = _inputs(gpu, T, H, V, ignored=ignored)
    loss, lse = head.head_loss(x, w, y)
    dx, dw = head.head_loss_grad(x, w, y, lse, a, b)
    assert held[-1].numel() < 2 * T * V
    nv, wide = held[-1][:8].view(torch.int32).tolist()
    assert nv == T - ignored
    if bn:
        assert wide == bn and -(-nv // bn) * bn < -(-nv // 64) * 64
    ref = _reference(x, w, y, a, b, V)
    _within(loss, ref["loss"], "loss")
    _within(dx, ref["dx"], "dx")
    _within(dw, ref["dw"], "dweight", 2.0 ** -8)


@pytest.mark.parametrize("T", [16, 70, 1500])
def test_gradients_of_the_whole_head(gpu, T):
    """151,936 words by 2048 values: the gradients of tokens and rows here and there in 64 bits, from a few tokens to two pieces."""
    import torch
    from vates_amd.head import head_loss, head_loss_grad
    H, V = 2048, 151936
    log(f"case: the whole head T={T}")
    x, w, y, a, b = _inputs(gpu, T, H, V, ignored=T // 7)
    loss, lse = head_loss(x, w, y)
    dx, dw = head_loss_grad(x, w, y, lse, a, b)
    at = torch.arange(0, T, max(1, T // 12), device=gpu)
    ref = _reference(x[at], w, y[at], a[at], b[at], V)
    _within(loss[at], ref["loss"], "loss")
    _within(dx[at], ref["dx"], "dx")
    rows = torch.cat([y[y >= 0][:20], torch.arange(0, V, 9973, device=gpu), torch.arange(V - 20, V, device=gpu)]).unique()
    keep = y >= 0
    xk, wr, ak, bk = x[keep].double(), w[rows].double(), a[keep].double()[:, None], b[keep].double()[:, None]
    p = torch.exp(xk @ wr.t().contiguous() - lse[keep].double()[:, None]) * (ak + bk)
    g = p - torch.where(y[keep][:, None] == rows, ak, 0.0)
    ez = H * U * (xk.abs() @ wr.abs().t().contiguous())
    eg = 2.0 ** -8 * g.abs() + p * (2 * ez + 2.0 ** -15)
    # (lse is the entry's own here: its error is in p's)
    bound = (eg + p * ref["lse"][1].max()).t().contiguous() @ xk.abs() + T * U * (g.abs().t().contiguous() @ xk.abs())
    _within(dw[rows], (g.t().contiguous() @ xk, bound), "dweight", 2.0 ** -8)
