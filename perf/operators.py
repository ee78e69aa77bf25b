"""Performance cases of the 8-bit KV cache: storing, reading back, the pass that
forms a batch's heads, and attention over it.

The cache holds keys and values of one attention layer in 8 bits: for every
position and kv head a row of 256 codes c in [-127, 127] and one scale s, so
that the row stands for s c.  Head dimension 256 and the head counts are those
of the repository's own attention layer (16 query heads over 2 kv heads) and of
its tests; contexts run from a first token to 262,144 positions.  Kinds of case:

  store   rows written into the cache and read back (``KVCache8.write``, ``.read``)
  load    rows read back (``KVCache8.read``)
  heads   q and k RMSNorm, rotary embedding, keys and values into the cache
          (``norm_rope_append``), and the appended rows read back
  attend  softmax attention of T query tokens over the cache (``attend``)

What the cache holds is returned as the values it stands for.
"""
from __future__ import annotations

import math

import torch

own = False

DIM = 256
EPS, THETA = 1e-6, 1e7
DEV = "cuda:0"
ROWS = 1 << 28          # scores of one piece of the plain attention


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a draft's key and value kept from another source: the smallest write
        {"name": "store 1", "kind": "store", "n": 1, "pos": 4095, "n_kv": 2, "order": "heads"},
        # part of a prefix moved in from token-major rows, at odd places
        {"name": "store 777 token-major", "kind": "store", "n": 777, "pos": 1235, "n_kv": 2, "order": "tokens"},
        # a whole 32,768-position prefix moved in
        {"name": "store 32768", "kind": "store", "n": 32768, "pos": 0, "n_kv": 2, "order": "heads"},
        # a short stretch read back, for a program that inspects or moves a prefix
        {"name": "load 1001", "kind": "load", "n": 1001, "pos": 517, "n_kv": 4, "out": "f32"},
        # a whole long prefix read back as bf16
        {"name": "load 131072", "kind": "load", "n": 131072, "pos": 0, "n_kv": 2, "out": "bf16"},
        # the heads of the verify batch [x, d1, d2, d3] across a block of positions
        {"name": "heads T=4", "kind": "heads", "T": 4, "pos": 8190, "n_heads": 16, "n_kv": 2, "rope": 64},
        # the heads of a long prompt's block
        {"name": "heads T=2048", "kind": "heads", "T": 2048, "pos": 0, "n_heads": 16, "n_kv": 2, "rope": 64},
        # a decoded token of a short conversation: latency
        {"name": "attend T=1 at 1000", "kind": "attend", "T": 1, "pos": 1000, "n_heads": 16, "n_kv": 2, "gate": True},
        # the verify batch over the benchmark's context
        {"name": "attend T=4 at 32764", "kind": "attend", "T": 4, "pos": 32764, "n_heads": 16, "n_kv": 2, "gate": True},
        # a decoded token of a very long document
        {"name": "attend T=1 at 262143", "kind": "attend", "T": 1, "pos": 262143, "n_heads": 16, "n_kv": 2, "gate": False},
        # a short prompt from its start
        {"name": "attend T=777 at 0", "kind": "attend", "T": 777, "pos": 0, "n_heads": 16, "n_kv": 2, "gate": True},
        # a block of a long prompt behind two others
        {"name": "attend T=4096 at 8192", "kind": "attend", "T": 4096, "pos": 8192, "n_heads": 16, "n_kv": 2, "gate": True},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["store", "load", "heads", "attend", "attend", "attend"])
    n_heads, n_kv = rng.choice([(16, 2), (16, 2), (8, 2), (16, 4), (8, 1), (4, 4), (6, 2), (5, 1)])
    if kind in ("store", "load"):
        case = {"kind": kind, "n": _spread(rng, 1, 32768), "pos": rng.choice([0, _spread(rng, 1, 8192)]), "n_kv": n_kv}
        if kind == "store":
            case["order"] = rng.choice(["heads", "tokens"])
        else:
            case["out"] = rng.choice(["f32", "bf16"])
        return case
    if kind == "heads":
        return {"kind": kind, "T": _spread(rng, 1, 2048), "pos": rng.choice([0, _spread(rng, 1, 200000)]),
                "n_heads": n_heads, "n_kv": n_kv, "rope": rng.choice([64, 64, 128, 256, 32])}
    if rng.random() < 0.5:      # decode and verify batches
        T, pos = rng.randint(1, 8), _spread(rng, 1, 262136)
    else:                       # prompts and their blocks
        T, pos = _spread(rng, 9, 4096), rng.choice([0, _spread(rng, 1, 65536)])
    while n_heads * T * (pos + T / 2) > 16 * 4096 * (8192 + 2048):
        pos //= 2
    return {"kind": "attend", "T": T, "pos": pos, "n_heads": n_heads, "n_kv": n_kv, "gate": rng.random() < 0.5}


# ------------------------------------------------------------------ the inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)


def _cached_rows(g, n_kv, n):
    """Keys and values as a layer's cache holds them, bf16 [n_kv, n, 256]: keys
    of RMS about 1 with a few strong channels and first positions that most
    queries look at, values whose size varies from token to token."""
    gain = torch.ones(DIM, device=DEV)
    gain[torch.randint(0, DIM, (6,), generator=g, device=DEV)] = 4.0
    k = torch.randn((n_kv, n, DIM), generator=g, device=DEV) * gain
    k[:, :min(n, 4)] += 1.5
    v = torch.randn((n_kv, n, DIM), generator=g, device=DEV)
    v *= torch.exp(0.5 * torch.randn((n_kv, n, 1), generator=g, device=DEV))
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _queries(g, T, n_heads):
    q = torch.randn((T, n_heads, DIM), generator=g, device=DEV) + 0.15
    return q.to(torch.bfloat16)


def _inputs(case, seed):
    """The case's tensors, the same whatever computes on them."""
    g = _gen(seed)
    kind = case["kind"]
    if kind == "store":
        k, v = _cached_rows(g, case["n_kv"], case["n"])
        if case["order"] == "tokens":   # [n, n_kv, 256] rows seen as [n_kv, n, 256]
            k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
        return {"k": k, "v": v}
    if kind == "load":
        k, v = _cached_rows(g, case["n_kv"], case["pos"] + case["n"])
        return {"k": k, "v": v}
    if kind == "heads":
        T, nh, nkv = case["T"], case["n_heads"], case["n_kv"]
        # what the projections emit: [q | gate] per head, then the keys, then the values
        qkv = torch.randn((T, (2 * nh + 2 * nkv) * DIM), generator=g, device=DEV)
        qkv *= torch.exp(0.7 * torch.randn((T, 1), generator=g, device=DEV))
        w = [(1.0 + 0.2 * torch.randn(DIM, generator=g, device=DEV)).to(torch.bfloat16) for _ in range(2)]
        return {"qkv": qkv, "q_norm": w[0], "k_norm": w[1]}
    k, v = _cached_rows(g, case["n_kv"], case["pos"] + case["T"])
    out = {"k": k, "v": v, "q": _queries(g, case["T"], case["n_heads"]), "gate": None}
    if case["gate"]:
        out["gate"] = 2.0 * torch.randn((case["T"], case["n_heads"], DIM), generator=g, device=DEV)
    return out


def prepare(case, seed):
    kind = case["kind"]
    data = _inputs(case, seed)
    length = case["pos"] + case.get("n", case.get("T"))
    state = {"case": case}
    if own:
        from vates_amd.attention import KVCache8
        cache = KVCache8(case["n_kv"], length, DEV)
        if kind in ("load", "attend"):
            cache.write(0, data.pop("k"), data.pop("v"))
            cache.length = length
        state["cache"] = cache
    elif kind in ("load", "attend"):
        state["k"], state["v"] = _plain_store(data.pop("k")), _plain_store(data.pop("v"))
    elif kind == "store":
        shape = (case["n_kv"], length)
        for name in ("kc", "vc"):
            state[name] = (torch.zeros((*shape, DIM), dtype=torch.int8, device=DEV),
                           torch.zeros((*shape, 1), device=DEV))
    state.update(data)
    return state


# ------------------------------------------------------------- the plain forms
def _plain_store(x):
    """(codes int8, scales f32) of rows of 256."""
    x = x.float()
    a = x.abs().amax(-1, keepdim=True)
    c = torch.round((x * (127.0 / 128.0)) / (a / 128.0))
    c = torch.where(a > 0, c, torch.zeros_like(c))
    return c.to(torch.int8), a / 127.0


def _plain_heads(case, state):
    T, nh, nkv, rd = case["T"], case["n_heads"], case["n_kv"], case["rope"]
    rows = state["qkv"]
    qg = rows[:, :2 * nh * DIM].view(T, nh, 2, DIM)[:, :, 0]
    k, v = rows[:, 2 * nh * DIM:].view(T, 2, nkv, DIM).unbind(1)
    i = torch.arange(rd // 2, dtype=torch.float64, device=rows.device)
    pos = torch.arange(case["pos"], case["pos"] + T, dtype=torch.float64, device=rows.device)
    ang = pos[:, None] * THETA ** (-2.0 * i / rd)
    cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]

    def form(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rd:]], -1)

    q = form(qg, state["q_norm"]).to(torch.bfloat16)
    out = []
    for x in (form(k, state["k_norm"]), v):
        c, s = _plain_store(x.transpose(0, 1))
        out.append((c.float() * s).to(torch.bfloat16))
    return q, out[0], out[1]


def _plain_attend(case, state):
    T, nh, nkv, pos = case["T"], case["n_heads"], case["n_kv"], case["pos"]
    G, L = nh // nkv, case["pos"] + T
    q = state["q"].float()
    out = torch.empty((T, nh, DIM), device=q.device)
    keys = torch.arange(L, device=q.device)
    for g in range(nkv):
        kc, ks = state["k"]
        vc, vs = state["v"]
        k, v = kc[g].float() * ks[g], vc[g].float() * vs[g]
        step = max(1, ROWS // (L * G))
        for t0 in range(0, T, step):
            t1 = min(T, t0 + step)
            seen = pos + t1
            x = q[t0:t1, g * G:(g + 1) * G].reshape(-1, DIM) @ k[:seen].t() / 16.0
            last = pos + torch.arange(t0, t1, device=q.device).repeat_interleave(G)
            x = x.masked_fill(keys[None, :seen] > last[:, None], float("-inf"))
            p = torch.exp(x - x.amax(-1, keepdim=True))
            o = (p @ v[:seen]) / p.sum(-1, keepdim=True)
            out[t0:t1, g * G:(g + 1) * G] = o.view(t1 - t0, G, DIM)
    if state["gate"] is not None:
        out = out / (1.0 + torch.exp(-state["gate"]))
    return out.to(torch.bfloat16)


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "store":
        a, b = case["pos"], case["pos"] + case["n"]
        out = []
        for cache, x in ((state["kc"], state["k"]), (state["vc"], state["v"])):
            cache[0][:, a:b], cache[1][:, a:b] = _plain_store(x)
            out.append((cache[0][:, a:b].float() * cache[1][:, a:b]).to(torch.bfloat16))
        return tuple(out)
    if kind == "load":
        a, b = case["pos"], case["pos"] + case["n"]
        dt = torch.float32 if case["out"] == "f32" else torch.bfloat16
        return tuple((c[:, a:b].float() * s[:, a:b]).to(dt) for c, s in (state["k"], state["v"]))
    if kind == "heads":
        return _plain_heads(case, state)
    return _plain_attend(case, state)


# ------------------------------------------------------------ the framework's
def _own(state):
    from vates_amd.attention import attend, norm_rope_append
    case, cache = state["case"], state["cache"]
    kind, pos = case["kind"], case["pos"]
    if kind == "store":
        cache.write(pos, state["k"], state["v"])
        return cache.read(pos, pos + case["n"])
    if kind == "load":
        return cache.read(pos, pos + case["n"], dtype=torch.float32 if case["out"] == "f32" else torch.bfloat16)
    if kind == "heads":
        q = norm_rope_append(state["qkv"], cache, state["q_norm"], state["k_norm"], n_heads=case["n_heads"],
                             rope_dim=case["rope"], rope_theta=THETA, eps=EPS, pos0=pos)
        return (q, *cache.read(pos, pos + case["T"]))
    return attend(state["q"], cache, pos0=pos, gate=state["gate"])


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------- counts
def work(case):
    kind = case["kind"]
    if kind in ("store", "load"):
        rows = 2 * case["n"] * case["n_kv"]          # key and value rows
        if kind == "store":                           # bf16 in, codes and scale kept, bf16 back
            return {"bytes": rows * (2 * DIM + DIM + 4 + 2 * DIM), "flops": rows * DIM * 4}
        out = 4 if case["out"] == "f32" else 2
        return {"bytes": rows * (DIM + 4 + out * DIM), "flops": rows * DIM}
    T, nh, nkv = case["T"], case["n_heads"], case["n_kv"]
    if kind == "heads":
        rows = 2 * T * nkv
        return {"bytes": T * DIM * nh * (4 + 2) + rows * (4 * DIM + DIM + 4 + 2 * DIM),
                "flops": T * DIM * (nh + nkv) * 8 + rows * DIM * 4}
    L = case["pos"] + T
    return {"bytes": 2 * L * nkv * (DIM + 4) + T * nh * DIM * (4 + (4 if case["gate"] else 0)),
            "flops": 4 * DIM * nh * (T * case["pos"] + T * (T + 1) // 2)}


# ------------------------------------------------------------- 64-bit results
def _held64(x):
    """The values that rows of 256 are held as."""
    x = x.double()
    a = x.abs().max(dim=-1, keepdim=True).values
    code = torch.round(127.0 * x / torch.where(a == 0, torch.ones_like(a), a))
    return code * (a / 127.0)


def exact(case, seed):
    data = _inputs(case, seed)
    kind = case["kind"]
    if kind == "store":
        return _held64(data["k"]), _held64(data["v"])
    if kind == "load":
        n0 = case["pos"]
        return _held64(data["k"][:, n0:]), _held64(data["v"][:, n0:])
    T, nh, nkv = case["T"], case["n_heads"], case["n_kv"]
    if kind == "heads":
        x = data["qkv"].double().view(T, -1, DIM)     # rows of 256: q, gate, q, gate, .., keys, values
        half = case["rope"] // 2
        where = case["pos"] + torch.arange(T, dtype=torch.float64, device=DEV)
        freq = torch.exp(torch.arange(half, dtype=torch.float64, device=DEV) * (-math.log(THETA) / half))
        turn = torch.polar(torch.ones((T, half), dtype=torch.float64, device=DEV), where[:, None] * freq[None])

        def rotated(y, w):
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / DIM + EPS) * w.double()
            z = torch.complex(y[..., :half], y[..., half:2 * half]) * turn[:, None]
            return torch.cat((z.real, z.imag, y[..., 2 * half:]), dim=-1)

        q = rotated(x[:, 0:2 * nh:2], data["q_norm"])
        k = rotated(x[:, 2 * nh:2 * nh + nkv], data["k_norm"])
        return q, _held64(k.permute(1, 0, 2)), _held64(x[:, 2 * nh + nkv:].permute(1, 0, 2))
    k, v, q = _held64(data["k"]), _held64(data["v"]), data["q"].double()
    G, res = nh // nkv, torch.zeros((T, nh, DIM), dtype=torch.float64, device=DEV)
    piece = max(1, (1 << 26) // (case["pos"] + T))
    at = torch.arange(case["pos"] + T, device=DEV)
    for h in range(nh):
        for t0 in range(0, T, piece):
            t1 = min(T, t0 + piece)
            w = torch.matmul(q[t0:t1, h], k[h // G].t().contiguous()) * 0.0625
            w[at[None] > case["pos"] + torch.arange(t0, t1, device=DEV)[:, None]] = -math.inf
            res[t0:t1, h] = torch.matmul(torch.softmax(w, dim=-1), v[h // G])
    if data["gate"] is not None:
        res *= torch.sigmoid(data["gate"].double())
    return res
