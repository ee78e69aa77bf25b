"""The loss under a head and the expert rows behind the framework's own layers: a layer's
choice of experts, and a model's hidden rows.
"""
import pytest

pytestmark = pytest.mark.gpu


def log(msg):
    print(msg, flush=True)


def test_experts_behind_a_layers_router(gpu, orc):
    """The experts that a MoELayer's router chose (ids_out, scores_out), its weights
    multiplied as experts of the caller's own on the sorted rows: the fused operator's result, at that operator's bar of
    1e-5 for f32 rows."""
    import torch
    from oracle.torch_bridge import pool_np
    from vates_amd.moe import combine_experts, expert_plan, fused_moe_slots, sort_by_expert
    from vates_amd.synth import synth_bf16
    from vates_amd.workload import make_layer, synth_layer
    T, k, H, I, E = 7, 4, 512, 128, 64
    log("case: a layer's router, experts of the caller's own")
    w = synth_layer(5, 0, hidden=H, inter=I, num_experts=E, zipf_alpha=0.5, device=gpu)
    layer = make_layer(w, top_k=k)
    x = synth_bf16(5, 77, (T, H), std=1.0, device=gpu)
    ids = torch.empty((T, k), dtype=torch.int32, device=gpu)
    scores = torch.empty((T, k), dtype=torch.float32, device=gpu)
    layer(x, ids_out=ids, scores_out=scores)
    slots = w.table[ids.long()].to(torch.int32)
    xf = x.float()
    ref = layer.reference_weights()
    want = fused_moe_slots(xf, slots, scores, *[t for n in ("gate", "up", "down") for t in (ref[n].weight, ref[n].scales, ref[n].biases)],
                           H, I, 64, 4)

    pool = pool_np(ref["gate"], ref["up"], ref["down"])

    def weights(name, slot, rows, cols):
        full = orc.dequant(pool[name + "_w"][slot], pool[name + "_s"][slot], pool[name + "_b"][slot], rows, cols)
        return torch.from_numpy(full).to(gpu).double()

    plan = expert_plan(ids, E)
    rows = sort_by_expert(xf, plan)
    at = plan.offsets.tolist()
    y = torch.zeros_like(rows)
    for e in range(E):
        if at[e] < at[e + 1]:
            slot = int(w.table[e])
            r = rows[at[e]:at[e + 1]].double()
            h = torch.nn.functional.silu(r @ weights("gate", slot, I, H).t()) * (r @ weights("up", slot, I, H).t())
            y[at[e]:at[e + 1]] = (h @ weights("down", slot, H, I).t()).float()
    got = combine_experts(y, plan, scores)
    rel = ((got - want).norm(dim=-1) / want.norm(dim=-1)).max().item()
    log(f"  largest relative difference of a token {rel:.3g}")
    assert rel <= 1e-5


def test_a_models_rows_scored(gpu):
    """The tokens of a verify batch scored from the model's pre-norm hidden rows, as a
    user scores a text: final norm, then the loss under the model's head; against the log-sum-exp of the
    logits that the same forward gives, within their bar of 1e-4 sum |x w| each."""
    import torch
    from vates_amd.head import head_loss
    from vates_amd.mtp import rmsnorm
    from vates_amd.workload import synth_spec_model
    V = 5003
    log("case: a model's rows scored")
    model = synth_spec_model(3, n_layers=4, attn_every=4, hidden=512, inter=128, num_experts=64, top_k=4, vocab=V,
                             n_heads=4, n_kv_heads=2, n_k_heads=4, n_v_heads=8, device=gpu)
    caches = model.new_caches(64)
    ids = torch.randint(0, V, (9,), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(gpu)
    _, hidden, logits = model.forward(ids[:8], caches, 0, want_logits=True)
    x = rmsnorm(hidden, model.final_norm, eps=model.eps)
    loss, lse = head_loss(x, model.head, ids[1:])
    z = logits.double()
    want = torch.logsumexp(z, -1)
    hit = z.gather(1, ids[1:].long()[:, None])[:, 0]
    bar = 1e-4 * (x.double().abs() @ model.head.double().abs().t().contiguous()).amax(-1)
    log(f"  error over bar {((lse.double() - want).abs() / bar).max().item():.3f}")
    assert ((lse.double() - want).abs() <= bar).all()
    assert ((loss.double() - (want - hit)).abs() <= 2 * bar).all()
