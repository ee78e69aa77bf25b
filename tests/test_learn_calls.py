"""Refusals and workspaces of the head's loss and of the expert rows, on the CPU."""
import pytest

import vates_amd._lib as L


@pytest.fixture(scope="module")
def lib():
    return L.load()


P = 4096   # an aligned address that no refused call reads


def _loss(lib, x=P, T=4, H=512, w=P, V=1000, y=P, loss=P, lse=P, ws=P, n=1 << 40):
    return lib.vmi_head_loss(x, T, H, w, V, y, -100, loss, lse, None, ws, n, None)


def _grad(lib, x=P, T=4, H=512, w=P, V=1000, y=P, lse=P, d=P, dx=P, dw=P, dt=L.VMI_BF16, ws=P, n=1 << 40):
    return lib.vmi_head_loss_grad(x, T, H, w, V, y, -100, lse, d, None, dx, dw, dt, ws, n, None)


@pytest.mark.parametrize("call", [_loss, _grad])
def test_loss_refusals(lib, call):
    for T in (-1, 65537):
        assert call(lib, T=T) == L.VMI_ERR_UNSUPPORTED
    for H in (0, -64, 63, 100, 8256):
        assert call(lib, H=H) == L.VMI_ERR_UNSUPPORTED and b"hidden" in lib.vmi_last_error()
    for V in (0, -1, (1 << 21) + 1):
        assert call(lib, V=V) == L.VMI_ERR_UNSUPPORTED
    for name in ("x", "w", "y"):
        assert call(lib, **{name: None}) == L.VMI_ERR_INVALID
        assert call(lib, **{name: P + 4}) == L.VMI_ERR_INVALID
    assert call(lib, lse=None) == L.VMI_ERR_INVALID
    for ws, n in ((None, 1 << 40), (P, 16), (P + 16, 1 << 40)):
        assert call(lib, ws=ws, n=n) == L.VMI_ERR_WORKSPACE


def test_loss_refusals_of_one(lib):
    assert _loss(lib, loss=None) == L.VMI_ERR_INVALID
    assert _grad(lib, d=None) == L.VMI_ERR_INVALID
    assert _grad(lib, dx=None, dw=None) == L.VMI_ERR_INVALID
    assert _grad(lib, dt=7) == L.VMI_ERR_UNSUPPORTED
    assert _grad(lib, dx=P + 8) == L.VMI_ERR_INVALID and _grad(lib, dw=P + 8) == L.VMI_ERR_INVALID
    assert _loss(lib, T=0, x=None, y=None, loss=None, lse=None, ws=None) == L.VMI_OK


def test_loss_workspaces(lib):
    for q in (lib.vmi_head_loss_workspace_bytes, lib.vmi_head_loss_grad_workspace_bytes):
        for bad in ((-1, 512, 1000), (65537, 512, 1000), (4, 100, 1000), (4, 8256, 1000), (4, 512, 0), (4, 512, (1 << 21) + 1)):
            assert q(*bad) == 0
        assert q(0, 512, 1000) > 0
    # no logits (2.5 GB of bf16 at 8192 tokens): the loss takes a few MB, its gradients a piece of half a GB beside x and dx
    assert lib.vmi_head_loss_workspace_bytes(8192, 2048, 151936) < 8 << 20
    assert lib.vmi_head_loss_grad_workspace_bytes(8192, 2048, 151936) < 768 << 20
    assert lib.vmi_head_loss_grad_workspace_bytes(65536, 2048, 151936) < 3 << 30


def test_expert_refusals(lib):
    plan = lambda T=4, k=2, E=8, ids=P, o=P, s=P, p=P, ws=P, n=1 << 20: lib.vmi_expert_plan(ids, T, k, E, o, s, p, None, ws, n, None)
    for kw in ({"T": -1}, {"k": 0}, {"k": 33}, {"T": 65537}, {"ids": None}, {"o": None}, {"s": None}, {"p": None}):
        assert plan(**kw) == L.VMI_ERR_INVALID, kw
    for E in (0, -1, 1025):
        assert plan(E=E) == L.VMI_ERR_UNSUPPORTED and lib.vmi_expert_plan_workspace_bytes(4, 2, E) == 0
    assert plan(T=4097, ws=None) == L.VMI_ERR_WORKSPACE and plan(T=4097, n=4) == L.VMI_ERR_WORKSPACE
    assert lib.vmi_expert_plan_workspace_bytes(4, 33, 8) == 0

    def rows(T=4, k=2, H=64, dt=L.VMI_BF16, x=P, p=P, r=P):
        return lib.vmi_expert_rows(x, dt, T, k, H, p, r, None)

    def combine(T=4, k=2, H=64, dt=L.VMI_BF16, x=P, p=P, r=P):
        return lib.vmi_expert_combine(x, dt, T, k, H, p, None, None, r, None)

    def grad(T=4, k=2, H=64, dt=L.VMI_BF16, x=P, p=P, r=P, ds=None):
        return lib.vmi_expert_combine_grad(x, None, dt, T, k, H, p, None, r, ds, None)

    for call in (rows, combine, grad):
        for kw in ({"T": -1}, {"k": 0}, {"k": 33}, {"T": 65537}, {"x": None}, {"p": None}, {"x": P + 8}, {"r": P + 4}, {"r": None}):
            assert call(**kw) == L.VMI_ERR_INVALID, (call, kw)
        for kw in ({"H": 0}, {"H": 12}, {"H": 6, "dt": L.VMI_F32}, {"dt": 2}, {"H": (1 << 20) + 8}):
            assert call(**kw) == L.VMI_ERR_UNSUPPORTED, (call, kw)
        assert call(T=0, x=None, p=None) == L.VMI_OK
    assert grad(ds=P) == L.VMI_ERR_INVALID   # y is needed


def test_python_refusals():
    """The wrappers refuse what is not on the current HIP device before anything else."""
    import torch
    from vates_amd.head import head_loss, head_loss_grad
    from vates_amd.moe import ExpertPlan, combine_experts, expert_plan, sort_by_expert
    x, w, y = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((9, 64), dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    f = torch.zeros(4)
    plan = ExpertPlan(torch.zeros(3, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros((4, 2), dtype=torch.int32))
    for call in (lambda: head_loss(x, w, y), lambda: head_loss_grad(x, w, y, f, f), lambda: expert_plan(plan.place, 2),
                 lambda: sort_by_expert(x, plan), lambda: combine_experts(x, plan)):
        with pytest.raises(L.VmiError):
            call()
    assert plan.num_experts == 2 and plan.tokens == 4 and plan.top_k == 2


@pytest.mark.gpu
def test_python_refusals_on_the_device(gpu):
    import torch
    from vates_amd.head import head_loss, head_loss_grad
    from vates_amd.moe import combine_experts, expert_plan, sort_by_expert
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device=gpu)
    x, w, y, f = z(4, 64), z(9, 64), z(4, dt=torch.int64), z(4, dt=torch.float32)
    plan = expert_plan(z(4, 2, dt=torch.int32), 3)
    other = expert_plan(z(5, 2, dt=torch.int32), 3)
    calls = [lambda: head_loss(x.float(), w, y), lambda: head_loss(x, w.float(), y), lambda: head_loss(x, w, y.float()),
             lambda: head_loss(x, w, y[:3]), lambda: head_loss(x, z(9, 128), y), lambda: head_loss(z(4, 100), z(9, 100), y),
             lambda: head_loss(z(64, 4).t(), w, y), lambda: head_loss(x, z(64, 9).t(), y), lambda: head_loss(x, w, y.cpu()),
             lambda: head_loss(x, w, y, status=f), lambda: head_loss_grad(x, w, y, f, f, want_dx=False, want_dweight=False),
             lambda: head_loss_grad(x, w, y, f[:2], f), lambda: head_loss_grad(x, w, y, f, f.double()),
             lambda: head_loss_grad(x, w, y, f, None), lambda: head_loss_grad(x, w, y, f, f, dweight_dtype=torch.float16),
             lambda: expert_plan(z(4, 2, dt=torch.int64), 3), lambda: expert_plan(z(4, dt=torch.int32), 3),
             lambda: expert_plan(z(4, 0, dt=torch.int32), 3), lambda: expert_plan(z(4, 2, dt=torch.int32), 0),
             lambda: expert_plan(z(4, 2, dt=torch.int32), 1025), lambda: expert_plan(z(4, 33, dt=torch.int32), 64),
             lambda: sort_by_expert(x, other), lambda: sort_by_expert(x.half(), plan), lambda: sort_by_expert(z(4, 12), plan),
             lambda: sort_by_expert(z(64, 4).t(), plan), lambda: sort_by_expert(x, None),
             lambda: combine_experts(x, plan), lambda: combine_experts(z(8, 64), plan, z(4, 2)),
             lambda: combine_experts(z(8, 64), plan, z(4, 3, dt=torch.float32)),
             lambda: combine_experts(z(8, 64), plan, residual=z(4, 32)),
             lambda: combine_experts(z(8, 64), plan, residual=z(4, 64, dt=torch.float32))]
    for i, call in enumerate(calls):
        with pytest.raises(L.VmiError):
            call()
            pytest.fail(f"call {i} was taken")


def test_calls_without_tokens(lib):
    """Empty tensors have null pointers: no token is no error, whichever gradient is wanted."""
    assert _grad(lib, T=0, x=None, y=None, lse=None, d=None, dx=None, dw=None, ws=None, n=0) == L.VMI_OK
    assert lib.vmi_expert_combine_grad(None, None, L.VMI_BF16, 0, 2, 64, None, None, None, None, None) == L.VMI_OK


def test_hidden_sizes_past_a_launch(lib):
    """65,536 rows of these would pass the threads of one launch."""
    for H in ((1 << 16) + 8, 1 << 20):
        assert lib.vmi_expert_rows(P, L.VMI_BF16, 4, 2, H, P, P, None) == L.VMI_ERR_UNSUPPORTED
        assert lib.vmi_expert_combine(P, L.VMI_BF16, 4, 2, H, P, None, None, P, None) == L.VMI_ERR_UNSUPPORTED


def test_a_tiled_head_is_refused():
    from vates_amd.head import TiledHead, head_loss, head_loss_grad
    head = object.__new__(TiledHead)
    for call in (lambda: head_loss(None, head, None), lambda: head_loss_grad(None, head, None, None, None)):
        with pytest.raises(L.VmiError, match="row-major"):
            call()


def test_a_plan_workspace_off_16_bytes(lib):
    assert lib.vmi_expert_plan(P, 4097, 2, 8, P, P, P, None, P + 2, 1 << 20, None) == L.VMI_ERR_WORKSPACE


@pytest.mark.gpu
def test_forward_mode_is_refused(gpu):
    """Tensors with a tangent, in whichever argument, and gradients with one: refused, where a result
    without its tangent would be a wrong derivative. Plain calls inside a dual level go on."""
    import torch
    import torch.autograd.forward_ad as ad
    from vates_amd.head import head_loss, head_loss_grad
    from vates_amd.moe import combine_experts, expert_plan, sort_by_expert
    r = lambda *s, dt=torch.bfloat16: torch.ones(s, dtype=dt, device=gpu)
    x, w, t, f = r(4, 64), r(9, 64), torch.zeros(4, dtype=torch.int64, device=gpu), r(4, dt=torch.float32)
    plan = expert_plan(torch.zeros((4, 2), dtype=torch.int32, device=gpu), 3)
    y, s = r(8, 64), r(4, 2, dt=torch.float32)
    lse = head_loss(x, w, t)[1]
    with ad.dual_level():
        dual = lambda v: ad.make_dual(v, torch.ones_like(v))
        calls = [lambda: head_loss(dual(x), w, t), lambda: head_loss(x, dual(w), t),
                 lambda: head_loss_grad(dual(x), w, t, lse, f), lambda: head_loss_grad(x, dual(w), t, lse, f),
                 lambda: head_loss_grad(x, w, t, dual(lse), f), lambda: head_loss_grad(x, w, t, lse, dual(f)),
                 lambda: head_loss_grad(x, w, t, lse, f, dual(f)), lambda: sort_by_expert(dual(x), plan),
                 lambda: combine_experts(dual(y), plan), lambda: combine_experts(y, plan, dual(s)),
                 lambda: combine_experts(y, plan, s, residual=dual(x))]
        for i, call in enumerate(calls):
            with pytest.raises(L.VmiError, match="forward-mode"):
                call()
                pytest.fail(f"call {i} was taken")
        leaf = x.clone().requires_grad_()
        for out in (head_loss(leaf, w, t)[0], sort_by_expert(leaf, plan), combine_experts(y, plan, s, residual=leaf)):
            with pytest.raises(L.VmiError, match="forward-mode"):
                torch.autograd.grad(out, leaf, dual(torch.ones_like(out)), retain_graph=True)
            torch.autograd.grad(out, leaf, torch.ones_like(out))
        assert torch.equal(head_loss(x, w, t)[1], lse) and combine_experts(y, plan, s).shape == (4, 64)


def test_streams_of_another_device_are_refused(monkeypatch):
    """A stream that is not on the tensors' device, which is the current one: the call would
    go to that device's own stream, not to the one asked for."""
    import torch
    from vates_amd.moe import _on_stream
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)

    class Stream:
        device_index = 1

    ran = []
    with pytest.raises(L.VmiError, match="stream"):
        _on_stream(Stream(), ran.append, 1)
    assert not ran
    _on_stream(None, ran.append, 1)
    assert ran == [1]
