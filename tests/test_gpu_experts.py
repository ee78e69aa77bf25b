"""Routes sorted by expert and combined again (vmi_expert_plan, vmi_expert_rows,
vmi_expert_combine, vmi_expert_combine_grad).

Bars, written before the first run (u = 2^-24): plans and sorted rows exact; a
combined row k + 1 fp32 additions of products, (k + 2) u sum |s y|, and the output's own
rounding (bf16 2^-8 of it); d_y one product and its rounding; d_scores H u sum |d y|.
"""
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def log(msg):
    print(msg, flush=True)


def _dtype(name):
    import torch
    return {"bf16": torch.bfloat16, "f32": torch.float32}[name]


def _ids(dev, T, k, E, dropped=0, seed=0, one=None):
    import torch
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + T * 31 + k + E)
    if one is not None:
        return torch.full((T, k), one, dtype=torch.int32, device=dev)
    if k <= E:
        ids = torch.rand((T, E), generator=g, device=dev).argsort(-1)[:, :k].to(torch.int32).contiguous()
    else:
        ids = torch.randint(0, E, (T, k), generator=g, device=dev, dtype=torch.int32)
    if dropped:
        ids.view(-1)[torch.randperm(T * k, generator=g, device=dev)[:dropped]] = -1
    return ids


def _plan(ids, E):
    import numpy as np
    flat = ids.cpu().numpy().reshape(-1).astype(np.int64)
    expert = np.where((flat >= 0) & (flat < E), flat, E)
    source = np.argsort(expert, kind="stable")
    row = np.empty_like(source)
    row[source] = np.arange(len(source))
    offsets = np.concatenate([[0], np.cumsum(np.bincount(expert, minlength=E + 1)[:E])])
    return offsets, source, np.where(expert < E, row, ~row).reshape(ids.shape)


def _same_plan(plan, ids, E):
    import numpy as np
    for got, want in zip((plan.offsets, plan.source, plan.place), _plan(ids, E)):
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("T,k,E,dropped", [(0, 4, 8, 0), (1, 1, 1, 0), (1, 10, 512, 0), (4, 10, 512, 3), (64, 1, 2, 0),
                                           (65, 2, 3, 130), (777, 10, 512, 640), (819, 10, 1024, 5), (820, 10, 1023, 0),
                                           (8192, 10, 512, 0), (40000, 8, 64, 999), (9000, 32, 8, 17), (65536, 16, 1000, 1)])
def test_plan(gpu, T, k, E, dropped):
    from vates_amd.moe import expert_plan
    log(f"case: plan T={T} k={k} E={E} dropped={dropped}")
    ids = _ids(gpu, T, k, E, dropped)
    plan = expert_plan(ids, E)
    _same_plan(plan, ids, E)
    assert plan.num_experts == E and plan.tokens == T and plan.top_k == k


def test_plan_of_one_expert_and_of_none(gpu):
    import torch
    from vates_amd._lib import VMI_STATUS_BAD_SLOT
    from vates_amd.moe import expert_plan
    log("case: one expert, none, ids outside")
    for T, one in ((5000, 3), (5000, -1), (900, 63)):
        ids = _ids(gpu, T, 4, 64, one=one)
        _same_plan(expert_plan(ids, 64), ids, 64)
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    for T in (300, 5000):
        ids = _ids(gpu, T, 4, 64, 7)
        _same_plan(expert_plan(ids, 64, status=status), ids, 64)
        assert status.item() == 0
    ids[4321, 2], ids[7, 0], ids[8, 1] = 64, -2, 2 ** 31 - 1
    _same_plan(expert_plan(ids, 64, status=status), ids, 64)
    assert status.item() == VMI_STATUS_BAD_SLOT


SHAPES = [(1, 1, 1, 8, "bf16", 0), (1, 10, 512, 2048, "bf16", 0), (4, 10, 512, 2048, "bf16", 4), (3, 3, 5, 4, "f32", 2),
          (33, 4, 16, 1000, "bf16", 50), (130, 2, 8, 1000, "f32", 0), (257, 8, 64, 512, "f32", 100), (777, 10, 512, 2048, "bf16", 640),
          (65, 17, 32, 264, "bf16", 9), (20, 32, 40, 8200, "bf16", 1), (2000, 8, 64, 64, "bf16", 16000),
          (9000, 16, 64, 1024, "bf16", 5), (9000, 16, 64, 512, "f32", 5)]   # (rows of more than 256 MB)


@pytest.mark.parametrize("T,k,E,H,dt,dropped", SHAPES)
def test_sort_and_combine(gpu, T, k, E, H, dt, dropped):
    """Forward and backward of both, rows without an expert full of NaN."""
    import torch
    from vates_amd.moe import combine_experts, expert_plan, sort_by_expert
    log(f"case: rows T={T} k={k} E={E} H={H} {dt} dropped={dropped}")
    g = torch.Generator(device=gpu).manual_seed(T + H)
    dtype = _dtype(dt)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=gpu).to(dtype)

    ids = _ids(gpu, T, k, E, dropped)
    plan = expert_plan(ids, E)
    n = int(plan.offsets[-1])
    src, place = plan.source.long(), plan.place.long()
    live = place >= 0
    x = randn(T, H).requires_grad_()
    rows = sort_by_expert(x, plan)
    assert torch.equal(rows[:n].detach(), x.detach()[src[:n] // k]) and not rows[n:].any()
    assert torch.equal(sort_by_expert(x.detach(), plan), rows.detach())
    d_rows = randn(T * k, H)
    d_rows[n:] = float("nan")
    dx, = torch.autograd.grad(rows, x, d_rows)
    picked = torch.where(live[..., None], d_rows.double()[place.clamp(min=0)], 0.0)   # [T, k, H]
    want = picked.sum(1)
    assert ((dx.double() - want).abs() <= (k + 2) * U * picked.abs().sum(1) + HALF[dt] * want.abs()).all()

    y = randn(T * k, H)
    y[n:] = float("nan")
    y.requires_grad_()
    scores = torch.rand((T, k), generator=g, device=gpu)
    scores[~live] = float("nan")
    scores.requires_grad_()
    residual = randn(T, H).requires_grad_()
    out = combine_experts(y, plan, scores, residual=residual)
    terms = torch.where(live[..., None], scores.detach().double()[..., None] * y.detach().double()[place.clamp(min=0)], 0.0)
    want = terms.sum(1) + residual.detach().double()
    size = terms.abs().sum(1) + residual.detach().double().abs()
    assert ((out.double() - want).abs() <= (k + 2) * U * size + HALF[dt] * want.abs()).all()
    d_out = randn(T, H)
    dy, ds, dr = torch.autograd.grad(out, (y, scores, residual), d_out)
    assert torch.equal(dr, d_out)
    p = scores.detach().double().reshape(-1)[src[:n], None]
    d = d_out.double()[src[:n] // k]
    assert ((dy[:n].double() - p * d).abs() <= (U + HALF[dt]) * (p * d).abs() + 1e-38).all() and not dy[n:].any()
    yy = torch.where(live[..., None], y.detach().double()[place.clamp(min=0)], 0.0)
    prod = d_out.double()[:, None] * yy
    assert ((ds.double() - prod.sum(-1)).abs() <= H * U * prod.abs().sum(-1)).all() and (ds[~live] == 0).all()
    # without scores or a residual; one leaf alone
    plain = combine_experts(y.detach(), plan)
    want = yy.sum(1)
    assert ((plain.double() - want).abs() <= (k + 2) * U * yy.abs().sum(1) + HALF[dt] * want.abs()).all()
    ds2, = torch.autograd.grad(combine_experts(y.detach(), plan, scores), scores, d_out)
    dy2, = torch.autograd.grad(combine_experts(y, plan, scores.detach()), y, d_out)
    assert torch.equal(ds2, ds) and torch.equal(dy2, dy)
    dy3, = torch.autograd.grad(combine_experts(y, plan), y, d_out)
    assert torch.equal(dy3[:n], d_out[src[:n] // k]) and not dy3[n:].any()
    dr2, = torch.autograd.grad(combine_experts(y.detach(), plan, residual=residual), residual, d_out)
    assert torch.equal(dr2, d_out)


def test_gradients_with_strides(gpu):
    """Gradients that autograd hands over expanded or transposed."""
    import torch
    from vates_amd.moe import combine_experts, expert_plan, sort_by_expert
    log("case: strides")
    plan = expert_plan(_ids(gpu, 50, 4, 16, 6), 16)
    x = torch.randn((50, 64), device=gpu).requires_grad_()
    rows = sort_by_expert(x, plan)
    dx, = torch.autograd.grad(rows.sum(), x, retain_graph=True)
    assert torch.equal(dx, (plan.place >= 0).sum(1, keepdim=True).float().expand(50, 64))
    w = torch.randn((64, 200), device=gpu)
    a, = torch.autograd.grad(rows, x, w.t(), retain_graph=True)
    b, = torch.autograd.grad(rows, x, w.t().contiguous())
    assert torch.equal(a, b)
    out = combine_experts(rows.detach().requires_grad_(), plan)
    out.sum().backward()


def test_gradients_off_16_bytes(gpu):
    """Gradients that begin anywhere in their storage, as behind a concatenation."""
    import torch
    from vates_amd.moe import combine_experts, expert_plan, sort_by_expert
    T, k, H = 5, 3, 64
    log("case: gradients off 16 bytes")
    ids = _ids(gpu, T, k, 4, 2)
    plan = expert_plan(ids, 4)
    g = torch.Generator(device=gpu).manual_seed(3)
    for dt in (torch.bfloat16, torch.float32):
        make = lambda *s: torch.randn(s, generator=g, device=gpu).to(dt).requires_grad_()
        x, y, s = make(T, H), make(T * k, H), torch.rand((T, k), generator=g, device=gpu).requires_grad_()
        one = torch.ones(1, dtype=dt, device=gpu)
        for out, leaves in ((sort_by_expert(x, plan), (x,)), (combine_experts(y, plan, s), (y, s))):
            d = torch.randn(out.numel() + 1, generator=g, device=gpu).to(dt)
            got = torch.autograd.grad(torch.cat([one, out.reshape(-1)]), leaves, d, retain_graph=True)
            want = torch.autograd.grad(out, leaves, d[1:].clone().view(out.shape))
            assert all(torch.equal(i, j) for i, j in zip(got, want))


def test_no_tokens(gpu):
    import torch
    from vates_amd.moe import combine_experts, expert_plan, sort_by_expert
    log("case: no tokens")
    plan = expert_plan(torch.empty((0, 3), dtype=torch.int32, device=gpu), 4)
    x = torch.empty((0, 64), dtype=torch.bfloat16, device=gpu, requires_grad=True)
    s = torch.empty((0, 3), device=gpu, requires_grad=True)
    out = combine_experts(sort_by_expert(x, plan), plan, s, residual=x)
    dx, ds = torch.autograd.grad(out.sum(), (x, s))
    assert out.shape == dx.shape == (0, 64) and ds.shape == (0, 3)


def test_a_plan_changed_before_backward_is_refused(gpu):
    import torch
    from vates_amd.moe import combine_experts, expert_plan, sort_by_expert
    log("case: plan changed")
    for call, n in ((sort_by_expert, 4), (combine_experts, 8)):
        plan = expert_plan(_ids(gpu, 4, 2, 3), 3)
        x = torch.ones((n, 64), dtype=torch.bfloat16, device=gpu, requires_grad=True)
        out = call(x, plan)
        plan.place.copy_(plan.place.flip(0))
        with pytest.raises(RuntimeError):
            out.sum().backward()


def test_past_32_bits(gpu):
    """Rows whose elements' numbers pass 2^32."""
    import torch
    from vates_amd.moe import combine_experts, expert_plan, sort_by_expert
    T, k, H = 40000, 16, 8192
    log("case: past 32 bits")
    ids = _ids(gpu, T, k, 64, 5)
    plan = expert_plan(ids, 64)
    x = torch.randn((T, H), device=gpu, dtype=torch.bfloat16)
    rows = sort_by_expert(x, plan)
    n = int(plan.offsets[-1])
    at = torch.arange(0, n, 997, device=gpu)
    assert torch.equal(rows[at], x[plan.source[at].long() // k]) and torch.equal(rows[n - 1], x[plan.source[n - 1].long() // k])
    out = combine_experts(rows, plan)
    t = torch.arange(0, T, 499, device=gpu)
    want = x[t].double() * (plan.place[t] >= 0).sum(1, keepdim=True)
    assert ((out[t].double() - want).abs() <= (16 * U * k + HALF["bf16"]) * want.abs()).all()


def test_streams_and_graphs(gpu):
    import torch
    from vates_amd.moe import combine_experts, expert_plan, sort_by_expert
    T, k, E, H = 1000, 10, 64, 256
    log("case: experts on streams and in graphs")
    g = torch.Generator(device=gpu).manual_seed(5)
    sets = []
    for s in range(3):
        sets.append((_ids(gpu, T, k, E, 40 * s, seed=s), torch.randn((T, H), generator=g, device=gpu).to(torch.bfloat16),
                     torch.rand((T, k), generator=g, device=gpu), torch.randn((T, H), generator=g, device=gpu).to(torch.bfloat16)))

    def step(ids, x, scores, d_out, stream=None):
        plan = expert_plan(ids, E, stream=stream)
        rows = sort_by_expert(x, plan, stream=stream)
        out = combine_experts(rows, plan, scores, residual=x, stream=stream)
        return (plan.offsets, plan.place, rows, out, *torch.autograd.grad(out, (x, scores), d_out))

    leaves = lambda s: (s[0], s[1].clone().requires_grad_(), s[2].clone().requires_grad_(), s[3])
    want = [step(*leaves(s)) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    held = [leaves(s) for s in sets[:2]]
    torch.cuda.synchronize()
    for _ in range(3):
        got = [step(*h, stream=s) for h, s in zip(held, streams)]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(i, j) for i, j in zip(a, b))
    held = [tuple(t.detach().clone().requires_grad_(t.requires_grad) for t in h) for h in held]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for h in held:
            step(*h)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for h in held:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(*h))
        graphs.append(gr)
    for order in ((0, 1), (2, 0), (1, 2), (1, 1)):
        for h, n in zip(held, order):
            with torch.no_grad():
                for dst, src in zip(h, sets[n]):
                    dst.copy_(src)
        torch.cuda.synchronize()
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for o, n in zip(outs, order):
            assert all(torch.equal(i, j) for i, j in zip(o, want[n]))


def test_between_a_router_and_the_loss(gpu):
    """A drafter's last steps as they are used together: a router's choice, rows by
    expert, experts of the caller's own, the rows combined onto the residual, the loss
    under the head; the same in plain torch."""
    import torch
    from vates_amd.head import head_loss
    from vates_amd.moe import combine_experts, expert_plan, sort_by_expert
    T, k, E, H, V = 96, 2, 4, 128, 1003
    log("case: router to loss")
    g = torch.Generator(device=gpu).manual_seed(9)
    make = lambda *s, scale=1.0: (torch.randn(s, generator=g, device=gpu) * scale).to(torch.bfloat16).requires_grad_()
    x, experts, head = make(T, H), make(E, H, H, scale=H ** -0.5), make(V, H, scale=H ** -0.5)
    logits = torch.randn((T, E), generator=g, device=gpu)
    top = torch.topk(logits, k, -1)
    ids = top.indices.to(torch.int32)
    scores = torch.softmax(top.values, -1).requires_grad_()
    y = torch.randint(0, V, (T,), generator=g, device=gpu)
    y[:7] = -100
    live = int((y >= 0).sum())

    plan = expert_plan(ids, E)
    rows = sort_by_expert(x, plan)
    at = plan.offsets.tolist()
    out = torch.cat([rows[at[e]:at[e + 1]] @ experts[e] for e in range(E)])
    h = combine_experts(out, plan, scores, residual=x)
    loss = head_loss(h, head, y)[0].sum() / live
    got = torch.autograd.grad(loss, (x, scores, experts, head))

    d = [t.detach().double().requires_grad_() for t in (x, scores, experts, head)]
    hh = d[0] + sum(d[1][:, j, None] * torch.stack([d[0][t] @ d[2][ids[t, j]] for t in range(T)]) for j in range(k))
    ref = torch.nn.functional.cross_entropy(hh @ d[3].t(), y, ignore_index=-100)
    want = torch.autograd.grad(ref, d)
    # five bf16 roundings in a row, each 2^-8 at most, of numbers whose signs are mixed: 2^-5 of the norm
    assert abs(loss.item() - ref.item()) <= 2.0 ** -7 * abs(ref.item())
    for a, b, name in zip(got, want, ("x", "scores", "experts", "head")):
        rel = ((a.double() - b).norm() / b.norm()).item()
        log(f"  {name} {rel:.4f}")
        assert rel <= 2.0 ** -5
