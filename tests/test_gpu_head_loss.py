"""The loss of tokens under a head and its gradients (vmi_head_loss, vmi_head_loss_grad)
against the same formulas in 64 bits.

Bars, written before the first run (u = 2^-24, S = sum |x w| of a logit):
  logit       |e| <= H u S =: ez (H fp32 additions of exact products)
  lse         ez + u (8 + |lse|) + 2^-17: a probability's exponent is a product and a
              difference of numbers up to 2^8 in powers of two (2^-16 of itself at most, half
              of that on average over a sum of them), the sums add up to V/64/4 terms a lane
  loss        the lse's and the target's logit's
  g           2^-8 |g| (bf16) + a p (2 ez + 2^-15)
  dx, dW      the sums of |g|'s bounds times |w| (|x|), the additions' n u sum |g w|, and the
              output's own rounding, 2^-8 of it (bf16)
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def log(msg):
    print(msg, flush=True)


def _inputs(dev, T, H, V, seed=0, ignored=0, foreseen=8.0):
    import torch
    g = torch.Generator(device=dev).manual_seed(1000 * seed + T + H + V)
    w = (torch.randn((V, H), generator=g, device=dev) * (0.9 / H ** 0.5)).to(torch.bfloat16)
    y = torch.randint(0, V, (T,), generator=g, device=dev)
    x = torch.randn((T, H), generator=g, device=dev) + foreseen * torch.rand((T, 1), generator=g, device=dev) * w[y].float()
    if ignored:
        y[torch.randperm(T, generator=g, device=dev)[:ignored]] = -100
    a = (torch.rand(T, generator=g, device=dev) + 0.5) / T
    b = torch.rand(T, generator=g, device=dev) * 0.1 / T
    return x.to(torch.bfloat16), w, y, a, b


def _reference(x, w, y, d_loss, d_lse, V):
    """64-bit loss, lse, dx, dW and the bounds of each."""
    import torch
    x, w = x.double(), w.double()
    H = x.shape[1]
    keep = (y >= 0) & (y < V)
    z = x @ w.t().contiguous()
    ez = H * U * (x.abs() @ w.abs().t().contiguous())
    lse = torch.logsumexp(z, -1)
    at = torch.where(keep, y, 0)
    zero = torch.zeros_like(lse)
    loss = torch.where(keep, lse - z.gather(1, at[:, None])[:, 0], zero)
    top = ez.amax(-1)
    e_lse = top + U * (8 + lse.abs()) + 2.0 ** -17
    out = {"loss": (loss, e_lse + top), "lse": (torch.where(keep, lse, zero), e_lse)}
    a = torch.where(keep, d_loss.double() + d_lse.double(), zero)[:, None]
    p = torch.exp(z - lse[:, None])
    g = a * p
    g.scatter_add_(1, at[:, None], -torch.where(keep, d_loss.double(), zero)[:, None])
    eg = 2.0 ** -8 * g.abs() + a * p * (2 * ez + 2.0 ** -15)
    x = torch.where(keep[:, None], x, torch.zeros_like(x))
    dx, dw = g @ w, g.t().contiguous() @ x
    out["dx"] = (dx, eg @ w.abs() + V * U * (g.abs() @ w.abs()) + 2.0 ** -8 * dx.abs())
    out["dw"] = (dw, eg.t().contiguous() @ x.abs() + len(y) * U * (g.abs().t().contiguous() @ x.abs()))
    return out


def _within(got, want, name, rounding=0.0):
    ref, bound = want
    err = (got.double() - ref).abs()
    bound = bound + rounding * ref.abs() + 1e-30
    worst = (err / bound).max().item() if err.numel() else 0.0
    log(f"  {name}: error over bound {worst:.3f}")
    assert (err <= bound).all(), f"{name}: {worst:.3g} of the bound"


# (one token to few, few in the two sizes of their block, blocks of 128 tokens; the wider ones are below, with more rows of the head)
CASES = [(1, 64, 1), (300, 64, 1), (33, 64, 5000), (150, 128, 5000), (185, 64, 9000), (215, 128, 30000), (1000, 64, 1200), (8192, 64, 300), (1, 512, 16), (3, 64, 257), (5, 512, 4099), (16, 2048, 1601), (63, 192, 1000), (64, 1024, 1003),
         (65, 320, 2048), (130, 512, 777), (256, 64, 70), (257, 2048, 3001), (777, 512, 8200), (300, 8192, 129)]


@pytest.mark.parametrize("T,H,V", CASES)
def test_loss_and_gradients(gpu, T, H, V):
    import torch
    from vates_amd.head import head_loss, head_loss_grad
    log(f"case: head_loss T={T} H={H} V={V}")
    x, w, y, a, b = _inputs(gpu, T, H, V, ignored=T // 5)
    loss, lse = head_loss(x, w, y)
    torch.cuda.synchronize()
    ref = _reference(x, w, y, a, b, V)
    _within(loss, ref["loss"], "loss")
    _within(lse, ref["lse"], "lse")
    dx, dw = head_loss_grad(x, w, y, lse, a, b)
    torch.cuda.synchronize()
    _within(dx, ref["dx"], "dx")
    _within(dw, ref["dw"], "dweight bf16", 2.0 ** -8)
    none, dw32 = head_loss_grad(x, w, y, lse, a, b, want_dx=False, dweight_dtype=torch.float32)
    assert none is None and torch.equal(dw32.to(torch.bfloat16), dw)
    _within(dw32, ref["dw"], "dweight f32")
    dx2, none = head_loss_grad(x, w, y, lse, a, b, want_dweight=False)
    assert none is None and torch.equal(dx2, dx)


@pytest.mark.parametrize("T,V", [(20, 1003), (64, 1003), (150, 5000), (150, 60000), (185, 60000), (215, 60000), (470, 60000),
                                 (777, 60000), (1000, 60000)])
def test_workspaces_that_held_anything(gpu, monkeypatch, T, V):
    """A workspace of NaNs: nothing of it is read before it is written, at every width of a
    block (128 tokens with 5,000 rows, 160 to 256 with 60,000), whole steps of 64 tokens or not."""
    import torch
    import vates_amd.head as head
    log(f"case: workspaces of NaNs T={T} V={V}")
    monkeypatch.setattr(head, "scratch", lambda n, dev: torch.full((n,), 255, dtype=torch.uint8, device=dev))
    x, w, y, a, b = _inputs(gpu, T, 128, V, ignored=0)
    loss, lse = head.head_loss(x, w, y)
    dx, dw = head.head_loss_grad(x, w, y, lse, a, b)
    ref = _reference(x, w, y, a, b, V)
    _within(loss, ref["loss"], "loss")
    _within(lse, ref["lse"], "lse")
    _within(dx, ref["dx"], "dx")
    _within(dw, ref["dw"], "dweight", 2.0 ** -8)


def test_no_tokens(gpu):
    """Without a token: empty outputs and gradients, a head's gradient of zeros; a frozen head too."""
    import torch
    from vates_amd.head import head_loss
    log("case: no tokens")
    for frozen in (False, True):
        x = torch.empty((0, 64), dtype=torch.bfloat16, device=gpu, requires_grad=True)
        w = torch.ones((9, 64), dtype=torch.bfloat16, device=gpu, requires_grad=not frozen)
        loss, lse = head_loss(x, w, torch.empty(0, dtype=torch.int64, device=gpu))
        assert loss.shape == lse.shape == (0,)
        got = torch.autograd.grad(loss.sum() + lse.sum(), (x,) if frozen else (x, w))
        assert got[0].shape == (0, 64) and (frozen or not got[1].any())


def test_several_pieces(gpu, monkeypatch):
    """A vocabulary of several pieces, the last one short: tokens enough that g of all
    of it passes 256 MB."""
    import torch
    from vates_amd.head import head_loss, head_loss_grad
    T, H, V = 4100, 64, 33000
    log(f"case: pieces T={T} H={H} V={V}")
    x, w, y, a, b = _inputs(gpu, T, H, V, ignored=9)
    loss, lse = head_loss(x, w, y)
    dx, dw = head_loss_grad(x, w, y, lse, a, b)
    ref = _reference(x, w, y, a, b, V)
    _within(loss, ref["loss"], "loss")
    _within(dx, ref["dx"], "dx")
    _within(dw, ref["dw"], "dweight", 2.0 ** -8)


def test_largest(gpu):
    """The most tokens, and the largest vocabulary, on narrow heads: loss and gradients of
    tokens and rows here and there in 64 bits."""
    import torch
    from vates_amd.head import head_loss, head_loss_grad
    for T, H, V in ((65536, 64, 400), (3, 64, 1 << 21), (64, 64, 1 << 21), (70, 64, 1 << 21)):
        log(f"case: T={T} V={V}")
        x, w, y, a, b = _inputs(gpu, T, H, V, ignored=T // 7)
        loss, lse = head_loss(x, w, y)
        dx, dw = head_loss_grad(x, w, y, lse, a, b)
        at = torch.arange(0, T, max(1, T // 50), device=gpu)
        ref = _reference(x[at], w, y[at], a[at], b[at], V)
        _within(loss[at], ref["loss"], "loss")
        _within(lse[at], ref["lse"], "lse")
        _within(dx[at], ref["dx"], "dx")
        # rows of the head's gradient: the last ones, and those of some targets
        rows = torch.cat([y[y >= 0][:20], torch.arange(max(0, V - 20), V, device=gpu)]).unique()
        keep = y >= 0
        z = x[keep].double() @ w[rows].double().t().contiguous()
        p = torch.exp(z - lse[keep].double()[:, None]) * (a + b)[keep].double()[:, None]
        g = p - torch.where(y[keep][:, None] == rows, a[keep].double()[:, None], 0.0)
        ez = H * U * (x[keep].double().abs() @ w[rows].double().abs().t().contiguous())
        eg = 2.0 ** -8 * g.abs() + p * (2 * ez + 2.0 ** -15)
        xa = x[keep].double().abs()
        # (lse is the entry's own here: its error is in p's)
        bound = eg.t().contiguous() @ xa + T * U * (g.abs().t().contiguous() @ xa) + (p * ref["lse"][1].max()).t().contiguous() @ xa
        _within(dw[rows], (g.t().contiguous() @ x[keep].double(), bound), "dweight", 2.0 ** -8)


def test_twice_differentiable_is_refused(gpu):
    import torch
    from vates_amd.head import head_loss
    from vates_amd.moe import combine_experts, expert_plan
    x, w, y, _, _ = _inputs(gpu, 5, 64, 100)
    x.requires_grad_()
    g, = torch.autograd.grad(head_loss(x, w, y)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    plan = expert_plan(torch.zeros((5, 1), dtype=torch.int32, device=gpu), 2)
    s = torch.rand((5, 1), device=gpu).requires_grad_()
    g, = torch.autograd.grad(combine_experts(x.detach(), plan, s).float().pow(2).sum(), s, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_whole_vocabulary(gpu):
    import torch
    from vates_amd.head import head_loss, lm_head
    T, H, V = 16, 2048, 151936
    log("case: V=151936 against lm_head's logits")
    x, w, y, _, _ = _inputs(gpu, T, H, V, ignored=2)
    loss, lse = head_loss(x, w, y)
    z = lm_head(x, w)[0].double()
    keep = y >= 0
    want = torch.logsumexp(z, -1)
    hit = z.gather(1, y.clamp(min=0)[:, None])[:, 0]
    # both sides' logits are off by H u S at most; S is below |x| |w| = 0.9 |x|
    bound = 3 * H * U * 0.95 * x.double().norm(dim=-1) + 2.0 ** -17 + 32 * U
    assert ((loss.double() - (want - hit)).abs()[keep] <= bound[keep]).all()
    assert (loss[~keep] == 0).all() and (lse[~keep] == 0).all()


@pytest.mark.parametrize("T", [31, 60, 70, 400])
def test_tokens_left_out(gpu, T):
    """Ignored tokens and targets outside the vocabulary: what their rows hold reaches
    nothing, their gradients are zeros; a batch without any token in the loss."""
    import torch
    from vates_amd._lib import VMI_STATUS_BAD_TARGET
    from vates_amd.head import head_loss, head_loss_grad
    H, V = 512, 1003
    log(f"case: tokens left out T={T}")
    x, w, y, a, b = _inputs(gpu, T, H, V)
    y[::3] = -100
    keep = y >= 0
    loss, lse = head_loss(x, w, y)
    dx, dw = head_loss_grad(x, w, y, lse, a, b)
    x2, a2, b2 = x.clone(), a.clone(), b.clone()
    x2[::3] = float("nan")
    x2[3] = float("inf")
    a2[::3] = float("nan")
    b2[::3] = float("inf")
    got = head_loss(x2, w, y)
    assert torch.equal(got[0], loss) and torch.equal(got[1], lse)
    dx2, dw2 = head_loss_grad(x2, w, y, lse, a2, b2)
    assert torch.equal(dx2, dx) and torch.equal(dw2, dw) and not dx[::3].any()
    # the same tokens without the others: another count of tokens cuts the vocabulary into other strips, so the sums run
    # in another order; both results are within the bars of the 64-bit one, hence within twice that of each other
    few = head_loss(x[keep].contiguous(), w, y[keep].contiguous())
    ref = _reference(x, w, y, a, b, V)
    for got, old, name in zip(few, (loss, lse), ("loss", "lse")):
        assert ((got.double() - old[keep].double()).abs() <= 2 * ref[name][1][keep]).all()
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    bad = y.clone()
    bad[1], bad[2] = V, -7
    l2, s2 = head_loss(x, w, bad, status=status)
    assert status.item() == VMI_STATUS_BAD_TARGET and l2[1:3].isnan().all() and s2[1:3].isnan().all()
    assert not l2[3:].isnan().any()
    dx3, dw3 = head_loss_grad(x, w, bad, s2, a, b)
    assert not dx3[1:3].any() and torch.isfinite(dw3).all()
    # another index to ignore, a token of the vocabulary
    z = head_loss(x, w, y.clamp(min=0), ignore_index=0)
    assert (z[0][~keep] == 0).all() and torch.equal(z[0][keep & (y != 0)], loss[keep & (y != 0)])
    none = torch.full_like(y, -100)
    l4, s4 = head_loss(x2, w, none)
    dx4, dw4 = head_loss_grad(x2, w, none, s4, a2, b2)
    assert not l4.any() and not s4.any() and not dx4.any() and not dw4.any()
    empty = head_loss(x[:0], w, y[:0])
    dx5, dw5 = head_loss_grad(x[:0], w, y[:0], empty[1], a[:0], b[:0])
    assert empty[0].shape == (0,) and dx5.shape == (0, H) and not dw5.any()


@pytest.mark.parametrize("T", [9, 90])
def test_rows_that_are_not_finite(gpu, T):
    """A token whose logits are not finite is NaN, the others' losses and dx are not."""
    import torch
    from vates_amd.head import head_loss, head_loss_grad
    H, V = 512, 1003
    log(f"case: rows that are not finite T={T}")
    x, w, y, a, b = _inputs(gpu, T, H, V)
    loss, lse = head_loss(x, w, y)
    dx, _ = head_loss_grad(x, w, y, lse, a, b)
    x2 = x.clone()
    x2[4, 7] = float("inf")
    x2[6] = float("nan")
    l2, s2 = head_loss(x2, w, y)
    dx2, dw2 = head_loss_grad(x2, w, y, s2, a, b)
    rest = [t for t in range(T) if t not in (4, 6)]
    assert l2[[4, 6]].isnan().all() and torch.equal(l2[rest], loss[rest])
    assert torch.equal(dx2[rest], dx[rest]) and dx2[[4, 6]].isnan().all()
    # equal logits, and logits far apart
    flat = head_loss(x, torch.zeros_like(w), y)
    assert (flat[0] - np.log(V)).abs().max().item() <= 32 * U * np.log(V)
    far = head_loss((x * 1e4), w, y)
    assert torch.isfinite(far[0]).all() and (far[0] >= 0).all()


@pytest.mark.parametrize("T,H,V", [(37, 512, 1003), (300, 320, 2000)])
def test_autograd_and_differences(gpu, T, H, V):
    """The gradients that autograd gives are the entry's, and follow differences of
    the loss: over a step d both ways, sum dx d against the loss's change, within dx's
    bound, the losses' own and the third derivative's h^3."""
    import torch
    from vates_amd.head import head_loss, head_loss_grad
    log(f"case: autograd T={T}")
    x, w, y, a, b = _inputs(gpu, T, H, V, ignored=4)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss, lse = head_loss(xl, wl, y)
    ((loss * a).sum() + (lse * b).sum()).backward()
    dx, dw = head_loss_grad(x, w, y, lse.detach(), a, b)
    assert torch.equal(xl.grad, dx) and torch.equal(wl.grad, dw)
    # the mean over the tokens (gradients with stride 0), only one output, only one leaf
    xl.grad = None
    loss, _ = head_loss(xl, w, y)
    loss.mean().backward()
    ones = torch.full((T,), 1.0 / T, device=gpu)
    assert torch.equal(xl.grad, head_loss_grad(x, w, y, lse.detach(), ones, want_dweight=False)[0])
    _, only = head_loss(x, wl, y.int())
    gw, = torch.autograd.grad(only, wl, b)
    assert torch.equal(gw, head_loss_grad(x, w, y, lse.detach(), torch.zeros_like(a), b, want_dx=False)[1])
    ref = _reference(x, w, y, a, b, V)
    for name, base, grad, other in (("x", x, dx, w), ("w", w, dw, x)):
        d = grad.float().sign() * (2.0 ** -5 if name == "x" else 2.0 ** -9)     # uphill, so that the change is large
        hi, lo = (base.float() + d).to(torch.bfloat16), (base.float() - d).to(torch.bfloat16)
        step = hi.double() - lo.double()

        def total(v):
            out = head_loss(v, w, y) if name == "x" else head_loss(x, v, y)
            return (out[0].double() * a.double() + out[1].double() * b.double()).sum().item()

        change = total(hi) - total(lo)
        along = (grad.double() * step).sum().item()
        wobble = (ref["dx" if name == "x" else "dw"][1] * step.abs()).sum().item() + 2.0 ** -8 * (grad.double() * step).abs().sum().item()
        own = 2 * ((a + b).double() * (ref["loss"][1] + ref["lse"][1])).sum().item()
        dz = (step @ other.double().t().contiguous()).abs().amax(-1) if name == "x" else (other.double() @ step.t().contiguous()).abs().amax(-1)
        # f(+) - f(-) - f' (hi - lo): the third derivative of a log-sum-exp along dz is below dz^3, the second below dz^2
        # (dz over the whole step; the middle of hi and lo, which are bf16, is off base by ez)
        off = (hi.double() + lo.double()) / 2 - base.double()
        ez = (off @ other.double().t().contiguous()).abs().amax(-1) if name == "x" else (other.double() @ off.t().contiguous()).abs().amax(-1)
        curve = ((a + b).double() * (dz ** 3 / 12 + dz * ez)).sum().item()
        log(f"  {name}: change {change:.6g} along {along:.6g} bounds {wobble:.2g} {own:.2g} {curve:.2g}")
        assert abs(change - along) <= wobble + own + curve
        assert wobble + own + curve <= 0.25 * change


@pytest.mark.parametrize("T", [20, 130])
def test_same_bits_streams_and_graphs(gpu, T):
    """The same call gives the same bits: again, on another stream, two at once on two
    streams, and captured and replayed on new inputs."""
    import torch
    from vates_amd.head import head_loss, head_loss_grad
    H, V = 512, 4099
    log(f"case: streams and graphs T={T}")
    sets = [_inputs(gpu, T, H, V, seed=s, ignored=11) for s in range(3)]
    want = []
    for x, w, y, a, b in sets:
        loss, lse = head_loss(x, w, y)
        want.append((loss, lse, *head_loss_grad(x, w, y, lse, a, b)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for s, (x, w, y, a, b) in zip(streams, sets):
            loss, lse = head_loss(x, w, y, stream=s)
            got.append((loss, lse, *head_loss_grad(x, w, y, lse, a, b, stream=s)))
        torch.cuda.synchronize()
        for g, r in zip(got, want):
            assert all(torch.equal(i, j) for i, j in zip(g, r))
    # two captured graphs, each a training step of its own inputs, replayed in turn
    held = [[t.clone() for t in sets[i]] for i in (0, 1)]
    for h in held:
        h[0].requires_grad_()
        h[1].requires_grad_()

    def step(h):
        loss, lse = head_loss(*h[:3])
        return (loss, lse, *torch.autograd.grad((loss, lse), h[:2], h[3:]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for h in held:
            step(h)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for h in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(h))
        graphs.append(g)
    for order in ((0, 1), (1, 2), (2, 0), (0, 0)):
        for h, n in zip(held, order):
            with torch.no_grad():
                for dst, src in zip(h, sets[n]):
                    dst.copy_(src)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o, n in zip(outs, order):
            assert all(torch.equal(i.detach(), j) for i, j in zip(o, want[n]))
