"""Performance cases of learning next to the framework's layers: the loss of a
head over a large vocabulary with its gradients, and the rows of a
mixture-of-experts block sorted by expert and combined again, with theirs.

Head sizes are the ones the repository's head, tests and benchmark use (a
vocabulary of 151,936 over hidden 2048, and smaller ones), experts and top-k
those of its MoE layers (10 of 512 over hidden 2048, and smaller ones); token
counts run from one to the 8192 of its longest prompt block.  Kinds of case:

  score   the loss and log-sum-exp of every token (``head_loss``)
  learn   the same and the gradients of hidden rows and, unless the head is
          frozen, of the head
  sort    routes sorted by expert, the tokens' rows in that order
          (``expert_plan``, ``sort_by_expert``), the gradient of the tokens
  back    the experts' rows weighted and added per token
          (``combine_experts``), the gradients of rows and weights
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
IGNORE = -100
PIECE = 1 << 28         # logits of one piece of the plain loss
TOP = 4096 * 151936 * 2048 * 3   # products of the largest listed case


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token scored over the benchmark's vocabulary: the smallest call that reads the whole head
        {"name": "score 1", "kind": "score", "T": 1, "V": 151936, "H": 2048, "ignored": 0},
        # the answer of a conversation scored, its prompt masked out
        {"name": "score 777", "kind": "score", "T": 777, "V": 151936, "H": 2048, "ignored": 130},
        # a long text scored, a block of it
        {"name": "score 8192", "kind": "score", "T": 8192, "V": 151936, "H": 2048, "ignored": 0},
        # a step of a small head on a few tokens: latency
        {"name": "learn 5 small", "kind": "learn", "T": 5, "V": 4099, "H": 512, "ignored": 1, "frozen": False},
        # a drafter taught under the main model's frozen head, its prompt masked out
        {"name": "learn 777 frozen", "kind": "learn", "T": 777, "V": 151936, "H": 2048, "ignored": 130, "frozen": True},
        # a training step of the hidden rows and the head
        {"name": "learn 4096", "kind": "learn", "T": 4096, "V": 151936, "H": 2048, "ignored": 0, "frozen": False},
        # the verify batch's tokens handed to experts of one's own
        {"name": "sort 4", "kind": "sort", "T": 4, "k": 10, "E": 512, "H": 2048, "type": "bf16", "dropped": 0, "grad": False},
        # a short prompt with padding, odd sizes, in training
        {"name": "sort 777", "kind": "sort", "T": 777, "k": 10, "E": 512, "H": 2048, "type": "bf16", "dropped": 640, "grad": True},
        # the longest prompt block
        {"name": "sort 8192", "kind": "sort", "T": 8192, "k": 10, "E": 512, "H": 2048, "type": "bf16", "dropped": 0, "grad": True},
        # the verify batch's experts added
        {"name": "back 4", "kind": "back", "T": 4, "k": 10, "E": 512, "H": 2048, "type": "bf16", "dropped": 0, "grad": False},
        # a small layer's training step in fp32, some routes over the experts' capacity
        {"name": "back 1001 f32", "kind": "back", "T": 1001, "k": 8, "E": 64, "H": 1024, "type": "f32", "dropped": 77, "grad": True},
        # the longest prompt block in training
        {"name": "back 8192", "kind": "back", "T": 8192, "k": 10, "E": 512, "H": 2048, "type": "bf16", "dropped": 0, "grad": True},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["score", "learn", "learn", "sort", "back"])
    if kind in ("score", "learn"):
        T, V = _spread(rng, 1, 8192), rng.choice([151936, 151936, _spread(rng, 1000, 151936)])
        H = rng.choice([2048, 2048, 1024, 512, 64 * rng.randint(1, 32)])
        frozen = rng.random() < 0.5
        while T * V * H * (1 if kind == "score" else 2 if frozen else 3) > TOP:
            T //= 2
        case = {"kind": kind, "T": T, "V": V, "H": H, "ignored": rng.choice([0, 0, int(T * rng.random())])}
        if kind == "learn":
            case["frozen"] = frozen
        return case
    k, E, H = rng.choice([(10, 512, 2048), (10, 512, 2048), (8, 64, 1024), (4, 64, 512), (1, 16, 2048), (2, 8, 1000)])
    T = _spread(rng, 1, 8192)
    return {"kind": kind, "T": T, "k": k, "E": E, "H": H, "type": rng.choice(["bf16", "bf16", "f32"]),
            "dropped": rng.choice([0, 0, int(T * k * rng.random() / 2)]), "grad": rng.random() < 0.7}


# ------------------------------------------------------------------ the inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + 29)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _head_inputs(case, seed):
    """Hidden rows behind the final norm, a head, and the tokens that came next:
    common words more often than rare ones, some foreseen and some not."""
    g = _gen(seed)
    T, V, H = case["T"], case["V"], case["H"]
    w = torch.empty((V, H), dtype=torch.bfloat16, device=DEV)
    for v0 in range(0, V, 16384):
        n = min(16384, V - v0)
        w[v0:v0 + n] = (_randn(g, n, H) * (0.9 / math.sqrt(H))).to(torch.bfloat16)
    u = torch.rand(T, generator=g, device=DEV, dtype=torch.float64)
    target = (torch.exp(u * math.log(V + 1)) - 1).long().clamp(0, V - 1)      # rank r about as often as 1 / r
    target = target * 7919 % V
    want = torch.rand((T, 1), generator=g, device=DEV) * 16.0
    x = _randn(g, T, H) + want * w[target].float() / 0.81
    target[:case["ignored"]] = IGNORE
    n = max(1, T - case["ignored"])
    out = {"x": x.to(torch.bfloat16), "w": w, "target": target}
    if case["kind"] == "learn":      # the mean over the tokens with a weight each, and a pull of the log-sum-exp to zero
        out["d_loss"] = (0.5 + torch.rand(T, generator=g, device=DEV)) / n
        out["d_lse"] = torch.rand(T, generator=g, device=DEV) * (2e-3 / n)
    return out


def _route_inputs(case, seed):
    """Routes as a router gives them (k experts a token, some experts far more
    often than others), routes without an expert as -1, and rows."""
    g = _gen(seed)
    T, k, E, H = case["T"], case["k"], case["E"], case["H"]
    dt = torch.bfloat16 if case["type"] == "bf16" else torch.float32
    bias = -0.5 * torch.log(1.0 + torch.randperm(E, generator=g, device=DEV).float())
    logits = _randn(g, T, E) + bias
    top = torch.topk(logits, k, dim=-1)
    ids = top.indices.to(torch.int32)
    if case["dropped"]:
        at = torch.randperm(T * k, generator=g, device=DEV)[:case["dropped"]]
        ids.view(-1)[at] = -1
    out = {"ids": ids}
    if case["kind"] == "sort":
        out["x"] = _randn(g, T, H).to(dt)
        if case["grad"]:
            out["d_rows"] = _randn(g, T * k, H).to(dt)
        return out
    y = _randn(g, T * k, H) * torch.exp(0.5 * _randn(g, T * k, 1))
    out["y"] = y.to(dt)
    p = torch.exp(top.values - top.values[:, :1])
    out["scores"] = p / p.sum(-1, keepdim=True)
    out["residual"] = _randn(g, T, H).to(dt)
    if case["grad"]:
        out["d_out"] = _randn(g, T, H).to(dt)
    return out


def _inputs(case, seed):
    return (_head_inputs if case["kind"] in ("score", "learn") else _route_inputs)(case, seed)


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    kind = case["kind"]
    if own:
        if kind == "learn":
            state["x"].requires_grad_()
            state["w"].requires_grad_(not case["frozen"])
        elif kind == "sort":
            state["x"].requires_grad_(case["grad"])
        elif kind == "back":
            state["y"].requires_grad_(case["grad"])
            state["scores"].requires_grad_(case["grad"])
    if kind == "back":      # the plan that sorted the tokens
        if own:
            from vates_amd.moe import expert_plan
            state["plan"] = expert_plan(state["ids"], case["E"])
        else:
            state["plan"] = _plain_plan(state["ids"], case["E"])
    return state


# ------------------------------------------------------------- the plain forms
def _plain_loss(case, s):
    T, V = case["T"], case["V"]
    keep = s["target"] != IGNORE
    x = s["x"].float()
    at = torch.where(keep, s["target"], torch.zeros_like(s["target"]))
    step = max(1, PIECE // T)
    m = torch.full((T,), float("-inf"), device=x.device)
    total = torch.zeros(T, device=x.device)
    hit = torch.zeros(T, device=x.device)
    for v0 in range(0, V, step):
        z = x @ s["w"][v0:v0 + step].float().t()
        new = torch.maximum(m, z.amax(-1))
        total = total * torch.exp(m - new) + torch.exp(z - new[:, None]).sum(-1)
        m = new
        inside = (at >= v0) & (at < v0 + z.shape[1])
        hit = torch.where(inside, z.gather(1, (at - v0).clamp(0, z.shape[1] - 1)[:, None])[:, 0], hit)
    lse = m + torch.log(total)
    none = torch.zeros_like(lse)
    loss = torch.where(keep, lse - hit, none)
    if case["kind"] == "score":
        return loss, torch.where(keep, lse, none)
    a = torch.where(keep, s["d_loss"] + s["d_lse"], none)
    b = torch.where(keep, s["d_loss"], none)
    dx = torch.zeros_like(x)
    dw = None if case["frozen"] else torch.empty_like(s["w"])
    row = torch.arange(T, device=x.device)
    for v0 in range(0, V, step):
        w = s["w"][v0:v0 + step].float()
        g = torch.exp(x @ w.t() - lse[:, None]) * a[:, None]
        inside = (at >= v0) & (at < v0 + w.shape[0])
        g[row, (at - v0).clamp(0, w.shape[0] - 1)] -= torch.where(inside, b, none)
        dx += g @ w
        if dw is not None:
            dw[v0:v0 + step] = (g.t() @ x).to(dw.dtype)
    out = (loss, torch.where(keep, lse, none), dx.to(torch.bfloat16))
    return out if dw is None else (*out, dw)


def _plain_plan(ids, E):
    """(first row of each expert and the end, route of each row, row of each
    route; ~row where the route has no expert, whose rows come last)."""
    flat = ids.reshape(-1)
    expert = torch.where((flat >= 0) & (flat < E), flat, torch.full_like(flat, E)).long()
    source = torch.argsort(expert, stable=True)
    row = torch.empty_like(source)
    row[source] = torch.arange(source.numel(), device=ids.device)
    first = torch.zeros(E + 1, dtype=torch.long, device=ids.device)
    first[1:] = torch.cumsum((expert[:, None] == torch.arange(E, device=ids.device)).sum(0), 0)
    place = torch.where(expert < E, row, -1 - row).view(ids.shape)
    return first.int(), source.int(), place.int()


def _plain_sum(rows, place, scores):
    """Per token its routes' rows times their weights, in the routes' order, fp32."""
    out = torch.zeros((place.shape[0], rows.shape[1]), device=rows.device)
    for j in range(place.shape[1]):
        p = place[:, j].long()
        r = rows[p.clamp(min=0)].float()
        if scores is not None:
            r = r * scores[:, j, None]
        out += torch.where((p >= 0)[:, None], r, torch.zeros_like(r))
    return out


def _plain_routes(case, s):
    k = case["k"]
    if case["kind"] == "sort":
        first, source, place = _plain_plan(s["ids"], case["E"])
        x = s["x"]
        live = torch.arange(source.numel(), device=x.device)[:, None] < first[-1]
        rows = torch.where(live, x[source.long() // k], torch.zeros((), dtype=x.dtype, device=x.device))
        out = (rows, first, source, place)
        if case["grad"]:
            out += (_plain_sum(s["d_rows"], place, None).to(x.dtype),)
        return out
    first, source, place = s["plan"]
    y, scores = s["y"], s["scores"]
    res = (_plain_sum(y, place, scores) + s["residual"].float()).to(y.dtype)
    if not case["grad"]:
        return res
    d = s["d_out"].float()
    src = source.long()
    live = torch.arange(src.numel(), device=y.device)[:, None] < first[-1]
    dy = d[src // k] * scores.reshape(-1)[src][:, None]
    dy = torch.where(live, dy, torch.zeros_like(dy)).to(y.dtype)
    ds = torch.zeros_like(scores)
    for j in range(k):
        p = place[:, j].long()
        ds[:, j] = torch.where(p >= 0, (d * y[p.clamp(min=0)].float()).sum(-1), torch.zeros_like(ds[:, j]))
    return res, dy, ds


# ------------------------------------------------------------ the framework's
def _own(s):
    case = s["case"]
    kind = case["kind"]
    if kind in ("score", "learn"):
        from vates_amd.head import head_loss
        loss, lse = head_loss(s["x"], s["w"], s["target"])
        if kind == "score":
            return loss, lse
        leaves = (s["x"],) if case["frozen"] else (s["x"], s["w"])
        grads = torch.autograd.grad((loss, lse), leaves, (s["d_loss"], s["d_lse"]))
        return (loss.detach(), lse.detach(), *grads)
    from vates_amd.moe import combine_experts, expert_plan, sort_by_expert
    if kind == "sort":
        plan = expert_plan(s["ids"], case["E"])
        rows = sort_by_expert(s["x"], plan)
        out = (rows.detach(), plan.offsets, plan.source, plan.place)
        return (*out, *torch.autograd.grad(rows, s["x"], s["d_rows"])) if case["grad"] else out
    out = combine_experts(s["y"], s["plan"], s["scores"], residual=s["residual"])
    if not case["grad"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, (s["y"], s["scores"]), s["d_out"]))


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    return (_plain_loss if case["kind"] in ("score", "learn") else _plain_routes)(case, state)


# ---------------------------------------------------------------------- counts
def work(case):
    T = case["T"]
    if case["kind"] in ("score", "learn"):
        V, H, live = case["V"], case["H"], max(1, T - case["ignored"])
        nbytes, flops = 2 * (live * H + V * H) + 16 * T, 2 * live * V * H
        if case["kind"] == "learn":
            nbytes, flops = nbytes + 2 * T * H + 8 * T, 2 * flops
            if not case["frozen"]:
                nbytes, flops = nbytes + 2 * V * H, flops + 2 * live * V * H
        return {"bytes": nbytes, "flops": flops}
    k, H = case["k"], case["H"]
    n, live, e = T * k, T * k - case["dropped"], 2 if case["type"] == "bf16" else 4
    if case["kind"] == "sort":
        nbytes = e * H * (T + n) + 12 * n + 4 * case["E"]
        if case["grad"]:
            nbytes += e * H * (live + T)
        return {"bytes": nbytes, "flops": live * H if case["grad"] else 0}
    nbytes = e * H * (live + 2 * T) + 8 * n
    if case["grad"]:
        nbytes += e * H * (T + n) + 4 * n
    return {"bytes": nbytes, "flops": live * H * (5 if case["grad"] else 2)}


# ------------------------------------------------------------- 64-bit results
def _exact_head(case, seed):
    d = _head_inputs(case, seed)
    T, V = case["T"], case["V"]
    live = torch.nonzero(d["target"] != IGNORE)[:, 0]
    x, t = d["x"][live].double(), d["target"][live]
    wide = max(1, (1 << 27) // max(1, len(live)))
    sums, hit = [], torch.zeros(len(live), dtype=torch.float64, device=DEV)
    for lo in range(0, V, wide):
        z = torch.matmul(x, d["w"][lo:lo + wide].double().t().contiguous())
        sums.append(torch.logsumexp(z, dim=1))
        here = torch.nonzero((t >= lo) & (t < lo + wide))[:, 0]
        hit[here] = z[here, t[here] - lo]
    lse = torch.logsumexp(torch.stack(sums), dim=0)
    full = lambda v: torch.zeros((T, *v.shape[1:]), dtype=torch.float64, device=DEV).index_copy_(0, live, v)
    if case["kind"] == "score":
        return full(lse - hit), full(lse)
    pull, hold = (d["d_loss"].double() + d["d_lse"].double())[live], d["d_loss"].double()[live]
    dx = torch.zeros_like(x)
    dw = None if case["frozen"] else torch.empty(d["w"].shape, dtype=torch.float64, device=DEV)
    for lo in range(0, V, wide):
        w = d["w"][lo:lo + wide].double()
        p = torch.exp(torch.matmul(x, w.t().contiguous()) - lse.unsqueeze(1)).mul_(pull.unsqueeze(1))
        here = torch.nonzero((t >= lo) & (t < lo + wide))[:, 0]
        p[here, t[here] - lo] -= hold[here]
        dx.addmm_(p, w)
        if dw is not None:
            dw[lo:lo + wide] = torch.matmul(p.t().contiguous(), x)
    out = [full(lse - hit), full(lse), full(dx)]
    return out if dw is None else [*out, dw]


def _exact_routes(case, seed):
    d = _route_inputs(case, seed)
    T, k, E = case["T"], case["k"], case["E"]
    flat = d["ids"].reshape(-1).long()
    expert = flat.masked_fill(flat < 0, E)
    # every route's rank: routes of lower experts, and earlier ones of its own
    source = torch.sort(expert * (T * k) + torch.arange(T * k, device=DEV)).indices
    rank = torch.empty_like(source).scatter_(0, source, torch.arange(T * k, device=DEV))
    first = torch.searchsorted(expert[source].contiguous(), torch.arange(E + 1, device=DEV))
    place = torch.where(expert < E, rank, ~rank).view(T, k)
    n = int(first[E])
    token = source[:n] // k
    if case["kind"] == "sort":
        rows = torch.zeros((T * k, case["H"]), dtype=torch.float64, device=DEV)
        rows[:n] = d["x"].double()[token]
        out = [rows, first.int(), source.int(), place.int()]
        if case["grad"]:
            dx = torch.zeros((T, case["H"]), dtype=torch.float64, device=DEV)
            out.append(dx.index_add_(0, token, d["d_rows"][:n].double()))
        return out
    p = d["scores"].double().reshape(-1)[source[:n]].unsqueeze(1)
    y = d["y"][:n].double()
    res = d["residual"].double().index_add_(0, token, p * y)
    if not case["grad"]:
        return res
    do = d["d_out"].double()[token]
    dy = torch.zeros((T * k, case["H"]), dtype=torch.float64, device=DEV)
    dy[:n] = p * do
    ds = torch.zeros(T * k, dtype=torch.float64, device=DEV)
    ds[source[:n]] = (do * y).sum(1)
    return res, dy, ds.view(T, k)


def exact(case, seed):
    return (_exact_head if case["kind"] in ("score", "learn") else _exact_routes)(case, seed)
