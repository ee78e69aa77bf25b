"""The loss under a head where its numbers are extreme (u = 2^-24).

Logits here are exact: two products a token, x = (A, c, 0 ..) and w = (1, -gap, 0 ..), of few
bits each, so that z = A - c gap has no rounding and the formula's 64-bit value is known.
"""
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def log(msg):
    print(msg, flush=True)


@pytest.mark.parametrize("T", [1, 5, 64, 130])
def test_foreseen_tokens(gpu, T):
    """A token's loss is as exact where the model foresaw it as elsewhere, however large
    the logits: with s = sum of the other words' exp(z - z_target), loss = log(1 + s).

    Bar, written before the first run: every exponent is an exact difference d times log2 e, off by
    (1.5 |d| + 2) u < 2^-17 of the term at |d| <= 50; 1 + s takes at most 32 additions a token (a lane's 16 rows of a
    tile, the lanes', waves' and strips' joins), u (1 + s) each; the logarithm and the last addition 2 u of
    the loss.  Rounded to the logits' size instead, a loss at A = 1000 is off by up to 2^-15, 16 times the bar."""
    import torch
    from vates_amd.head import head_loss
    H, V = 64, 1003
    log(f"case: foreseen tokens T={T}")
    gap = 8.0 + torch.arange(V, device=gpu) % 16              # 8 .. 23
    gap[777] = 0.0                                            # the target
    w = torch.zeros((V, H), dtype=torch.bfloat16, device=gpu)
    w[:, 0], w[:, 1] = 1.0, -gap.to(torch.bfloat16)
    y = torch.full((T,), 777, device=gpu)
    for A in (0.0, 20.0, 100.0, 500.0, 1000.0, -1000.0):
        x = torch.zeros((T, H), dtype=torch.bfloat16, device=gpu)
        x[:, 0] = A
        x[:, 1] = torch.tensor([2.0, 1.5, 1.0, 0.5], device=gpu).repeat(T)[:T].to(torch.bfloat16)
        d = -x[:, 1, None].double() * gap.double()
        d[:, 777] = -float("inf")
        s = torch.exp(d).sum(-1)
        want = torch.log1p(s)
        loss, lse = head_loss(x, w, y)
        bar = 2.0 ** -17 * s + 32 * U * (1 + s) + 2 * U * want
        err = (loss.double() - want).abs()
        log(f"  A={A}: loss {want.min().item():.3g} .. {want.max().item():.3g}, error over bar {(err / bar).max().item():.3f}")
        assert (err <= bar).all() and (loss >= 0).all()
        assert ((lse.double() - (A + want)).abs() <= bar + U * (A + want).abs()).all()


@pytest.mark.parametrize("T", [3, 40, 100])
@pytest.mark.parametrize("V", [1, 5, 300, 1024])
def test_every_logit_minus_infinity(gpu, T, V):
    """A token all of whose logits are minus infinity: lse minus infinity, and NaN for the loss, as
    the formula gives, whether or not the vocabulary ends inside a tile; one word with a
    finite logit among them is certain."""
    import torch
    from vates_amd.head import head_loss
    H = 64
    log(f"case: every logit minus infinity T={T} V={V}")
    x = torch.ones((T, H), dtype=torch.bfloat16, device=gpu)
    w = torch.full((V, H), -float("inf"), dtype=torch.bfloat16, device=gpu)
    y = torch.arange(T, device=gpu) % V
    loss, lse = head_loss(x, w, y)
    assert (lse == -float("inf")).all() and loss.isnan().all()
    w[V - 1] = -0.25
    loss, lse = head_loss(x, w, y)
    assert (lse == -16.0).all()
    assert (loss == torch.where(y == V - 1, 0.0, float("inf"))).all()


@pytest.mark.parametrize("T", [1, 32, 33, 64])
def test_a_few_tokens_none_in_the_loss(gpu, monkeypatch, T):
    """Up to 64 tokens of which none is in the loss: gradients of zeros, and no product of the head with what the
    workspace held, so that it holds the same afterwards."""
    import torch
    import vates_amd.head as head
    H, V = 512, 5003
    log(f"case: none in the loss T={T}")
    held = []

    def scratch(n, dev):
        held.append(torch.full((n,), 17, dtype=torch.uint8, device=dev))
        return held[-1]

    monkeypatch.setattr(head, "scratch", scratch)
    g = torch.Generator(device=gpu).manual_seed(T)
    x = torch.randn((T, H), generator=g, device=gpu).to(torch.bfloat16)
    w = torch.randn((V, H), generator=g, device=gpu).to(torch.bfloat16)
    y = torch.full((T,), -100, device=gpu)
    y[T // 2:] = V                       # outside the vocabulary
    f = torch.ones(T, device=gpu)
    for wants in ({}, {"want_dweight": False}, {"want_dx": False}):
        dx, dw = head.head_loss_grad(x, w, y, f, f, f, **wants)
        assert (dx is None or not dx.any()) and (dw is None or not dw.any())
    loss, lse = head.head_loss(x, w, y)
    assert not loss[:T // 2].any() and loss[T // 2:].isnan().all() and lse[T // 2:].isnan().all()
    assert len(held) == 4 and all((ws == 17).all() for ws in held)
