"""Measured cases of the expert router, its gradient and the products with 4-bit weights.

Four operators of a mixture-of-experts layer:

  route_experts            scores of all experts -> the top_k experts of each token and their weights
  route_experts_backward   gradient of those weights with respect to the logits
  linear_w4                y = x . W^T with 4-bit weights and one scale (and zero point) per group
  experts_w4               the routed experts' two products with 4-bit weights, SwiGLU between them,
                           summed with the routing weights

``run`` computes them in plain torch operations in 32 bits (``own`` false) or through the package's
entry points (``own`` true). Both work on the same state.

4-bit weights: ``codes`` uint8 [N, ceil(K / 2)] holds two codes per byte, the even column in the low
nibble; ``scale`` [N, ceil(K / group)] has the activations' type; ``zero`` uint8 of the same shape, or
None for 8. The weight is ``scale * (code - zero)``.
"""
import importlib
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def _pkg():
    return importlib.import_module("15642_moe_b200")


# ------------------------------------------------------------------------------------------ cases
def listed():
    v3 = dict(E=256, k=8, score="sigmoid", bias=True, groups=8, topk_groups=4, group_score="top2",
              renormalize=True, scale=2.5, dtype="f32")
    flat = dict(E=64, k=6, score="softmax", bias=False, groups=1, topk_groups=1, group_score="max",
                renormalize=False, scale=1.0, dtype="bf16")
    return [
        # One decoded token through the 256-expert router of the package's layer: latency.
        dict(name="route_t1", op="route", T=1, **v3),
        # The largest prompt of the package's configurations.
        dict(name="route_t16384", op="route", T=16384, **v3),
        # A router with softmax scores limited to the best groups, bf16 logits, odd counts.
        dict(name="route_softmax_t4097_e60", op="route", T=4097, E=60, k=6, score="softmax", bias=False,
             groups=4, topk_groups=2, group_score="max", renormalize=True, scale=1.0, dtype="bf16"),
        # Training step of the 256-expert router: only the picked experts have a gradient.
        dict(name="route_grad_t16384", op="route_grad", T=16384, **v3),
        # Training step of a softmax router without renormalisation: every expert has a gradient.
        dict(name="route_grad_softmax_t2049", op="route_grad", T=2049, **flat),
        # One decoded token through a gate/up projection (4096 x 7168).
        dict(name="linear_m1", op="linear", M=1, N=4096, K=7168, group=128, zero=False, dtype="bf16"),
        # A few decoded tokens, fp16 with zero points, through a down projection (7168 x 2048).
        dict(name="linear_m7_f16", op="linear", M=7, N=7168, K=2048, group=64, zero=True, dtype="f16"),
        # A speculative batch on a head of odd width.
        dict(name="linear_m13_odd", op="linear", M=13, N=1001, K=1999, group=32, zero=True, dtype="bf16"),
        # A prompt through the gate/up projection.
        dict(name="linear_m512", op="linear", M=512, N=4096, K=7168, group=128, zero=False, dtype="bf16"),
        # One decoded token, all eight picked experts on this GPU.
        dict(name="experts_t1", op="experts", T=1, E=32, EG=32, k=8, H=7168, I=2048, group=128, zero=False,
             dtype="bf16"),
        # The decode batch of the package's configurations: 32 local experts of 256.
        dict(name="experts_t64", op="experts", T=64, E=32, EG=256, k=8, H=7168, I=2048, group=128, zero=False,
             dtype="bf16"),
        # The prompt of the package's headline configuration: 32 local experts of 256.
        dict(name="experts_t4096", op="experts", T=4096, E=32, EG=256, k=8, H=7168, I=2048, group=128,
             zero=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _size(rng, lo, hi):
    """An odd multiple of 32 to 256 between lo and hi."""
    unit = rng.choice([32, 64, 128, 256])
    n = _log(rng, -(-lo // unit), hi // unit)
    return unit * (n if n % 2 else max(1, n - 1))


def draw(rng):
    op = rng.choice(["route", "route_grad", "linear", "linear", "experts", "experts"])
    if op in ("route", "route_grad"):
        groups = rng.choice([1, 1, 2, 4, 8])
        per = rng.randint(max(2, -(-16 // groups)), 512 // groups) if rng.random() < 0.5 else max(2, 64 // groups)
        topk_groups = rng.randint(1, groups)
        E = groups * per
        T = min(_log(rng, 1, 16383), 16384 * 256 // E) | 1
        return dict(op=op, T=T, E=E, k=rng.randint(1, min(12, topk_groups * per)),
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups,
                    topk_groups=topk_groups, group_score=rng.choice(["max", "top2"]),
                    renormalize=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]),
                    dtype=rng.choice(["f32", "bf16", "f16"]))
    group, dtype = rng.choice([32, 64, 128]), rng.choice(["bf16", "bf16", "f16"])
    zero = rng.random() < 0.5
    if op == "linear":
        odd = rng.random() < 0.25
        N = _log(rng, 256, 8190) | 1 if odd else _size(rng, 512, 7168)
        K = _log(rng, 256, 4094) | 1 if odd else _size(rng, 512, 7168)
        return dict(op=op, M=_log(rng, 1, 512), N=N, K=K, group=group, zero=zero, dtype=dtype)
    E, T, k = rng.choice([8, 16, 32]), _log(rng, 1, 1024), rng.randint(1, 8)
    # A slice of a larger layer only where it is sure to get some of the tokens.
    return dict(op=op, T=T, E=E, EG=E * (rng.choice([1, 2, 8]) if T * k >= 64 else 1), k=k,
                H=_size(rng, 512, 4096), I=_size(rng, 256, 2048), group=group, zero=zero, dtype=dtype)


# ----------------------------------------------------------------------------------------- inputs
def _weights(g, lead, N, K, group, zero, dtype, std):
    """Codes of normally distributed weights, their scales and zero points."""
    shape = tuple(lead) + (N, (K + 1) // 2)
    scale_shape = tuple(lead) + (N, -(-K // group))
    lo, hi = ((torch.randn(shape, generator=g, device=DEV, dtype=torch.float16) * 2.6 + 8).round_().clamp_(0, 15)
              .to(torch.uint8) for _ in range(2))
    codes = hi.bitwise_left_shift_(4).bitwise_or_(lo)
    scale = ((std / 2.6) * (0.75 + 0.5 * torch.rand(scale_shape, generator=g, device=DEV))).to(dtype)
    z = torch.randint(6, 11, scale_shape, generator=g, device=DEV, dtype=torch.uint8) if zero else None
    return codes, scale, z


def _near_ties(case, logits, bias):
    """Rows whose picks, their order or the kept groups hang on less than 32-bit scores resolve."""
    x = logits.double()
    s = torch.softmax(x, -1) if case["score"] == "softmax" else torch.sigmoid(x)
    pick = s if bias is None else s + bias.double()
    T, E = pick.shape
    size = pick.abs().amax(-1, keepdim=True)
    bad = torch.zeros(T, dtype=torch.bool, device=pick.device)
    if case["groups"] > 1:
        p = pick.view(T, case["groups"], -1)
        gs = p.amax(-1) if case["group_score"] == "max" else p.sort(dim=-1, descending=True).values[..., :2].sum(-1)
        order = gs.sort(dim=-1, descending=True, stable=True)
        if case["topk_groups"] < case["groups"]:
            gap = order.values[:, case["topk_groups"] - 1] - order.values[:, case["topk_groups"]]
            bad |= (gap > 0) & (gap < 4e-6 * size[:, 0])
        keep = torch.zeros_like(gs).scatter_(1, order.indices[:, :case["topk_groups"]], 1.0).bool()
        pick = torch.where(keep[:, :, None], p, -math.inf).view(T, E)
    top = pick.sort(dim=-1, descending=True).values[:, :case["k"] + 1]
    gap = top[:, :-1] - top[:, 1:]
    return bad | ((gap > 0) & (gap < 4e-6 * torch.minimum(size, top[:, :-1].abs()))).any(-1)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    if case["op"] in ("route", "route_grad"):
        T, E, k = case["T"], case["E"], case["k"]
        logits = torch.randn((T, E), generator=g, device=DEV).to(dtype)
        bias = 0.1 * torch.randn(E, generator=g, device=DEV) if case["bias"] else None
        if case["op"] == "route":
            # Rows that 32-bit scores cannot order for certain are drawn again (a few in a hundred).
            for _ in range(5):
                bad = _near_ties(case, logits, bias)
                logits = torch.where(bad[:, None], torch.randn((T, E), generator=g, device=DEV).to(dtype), logits)
            return dict(case=case, logits=logits, bias=bias)
        idx = torch.topk(logits.float() + (0.0 if bias is None else 5.0 * bias), k, dim=-1).indices.to(torch.int32)
        return dict(case=case, logits=logits, idx=idx, grad=torch.randn((T, k), generator=g, device=DEV))
    if case["op"] == "linear":
        codes, scale, zero = _weights(g, (), case["N"], case["K"], case["group"], case["zero"], dtype, 0.02)
        x = torch.randn((case["M"], case["K"]), generator=g, device=DEV).to(dtype)
        return dict(case=case, x=x, codes=codes, scale=scale, zero=zero)
    T, E, EG, k, H, I = (case[n] for n in ("T", "E", "EG", "k", "H", "I"))
    w13, s13, z13 = _weights(g, (E,), 2 * I, H, case["group"], case["zero"], dtype, 0.02)
    w2, s2, z2 = _weights(g, (E,), H, I, case["group"], case["zero"], dtype, 0.02)
    x = torch.randn((T, H), generator=g, device=DEV).to(dtype)
    # Distinct experts of all EG for each token; this GPU holds the first E of them.
    idx = torch.rand((T, EG), generator=g, device=DEV).topk(k, dim=-1).indices.to(torch.int32)
    wt = torch.rand((T, k), generator=g, device=DEV) + 0.2
    wt = 2.5 * wt / wt.sum(-1, keepdim=True)
    return dict(case=case, x=x, idx=idx, wt=wt, w13=w13, s13=s13, z13=z13, w2=w2, s2=s2, z2=z2)


# ------------------------------------------------------------------------------------ plain forms
def _scores(logits, score):
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _route_plain(st):
    c = st["case"]
    x = st["logits"].float()
    T, E = x.shape
    s = _scores(x, c["score"])
    pick = s if st["bias"] is None else s + st["bias"]
    pick = torch.where(torch.isneginf(x), -math.inf, pick)
    if c["groups"] > 1:
        p = pick.view(T, c["groups"], -1)
        gs = p.amax(-1) if c["group_score"] == "max" else p.sort(dim=-1, descending=True).values[..., :2].sum(-1)
        order = gs.sort(dim=-1, descending=True, stable=True).indices[:, :c["topk_groups"]]
        keep = torch.zeros_like(gs).scatter_(1, order, 1.0).bool()
        pick = torch.where(keep[:, :, None], p, -math.inf).view(T, E)
    top = pick.sort(dim=-1, descending=True, stable=True)
    idx, val = top.indices[:, :c["k"]], top.values[:, :c["k"]]
    none = torch.isneginf(val)
    w = torch.where(none, 0.0, s.gather(1, idx))
    if c["renormalize"]:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return torch.where(none, -1, idx).to(torch.int32), w * c["scale"]


def _route_grad_plain(st):
    c = st["case"]
    x, idx, g = st["logits"].float(), st["idx"].long(), c["scale"] * st["grad"]
    s = _scores(x, c["score"])
    sel = s.gather(1, idx)
    if c["renormalize"]:
        total = sel.sum(-1, keepdim=True) + 1e-20
        g = (g - (g * sel).sum(-1, keepdim=True) / total) / total
    ds = torch.zeros_like(s).scatter_(1, idx, g)
    if c["score"] == "sigmoid":
        return (ds * s * (1.0 - s)).to(st["logits"].dtype)
    return (s * (ds - (ds * s).sum(-1, keepdim=True))).to(st["logits"].dtype)


def _unpack(codes, scale, zero, K, group):
    """The weights in 32 bits: scale * (code - zero)."""
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :K].float()
    q -= 8.0 if zero is None else zero.float().repeat_interleave(group, -1)[..., :K]
    return q.mul_(scale.float().repeat_interleave(group, -1)[..., :K])


def _linear_plain(st):
    c = st["case"]
    w = _unpack(st["codes"], st["scale"], st["zero"], c["K"], c["group"])
    return (st["x"].float() @ w.T).to(st["x"].dtype)


def _experts_plain(st):
    """The rows of each used expert side by side, padded to the largest count, as batched products."""
    c = st["case"]
    x, T, k, E, H, I = st["x"].float(), c["T"], c["k"], c["E"], c["H"], c["I"]
    flat = st["idx"].long().reshape(-1)
    route = torch.nonzero((flat >= 0) & (flat < E)).squeeze(-1)
    out = torch.zeros((T, H), device=x.device)
    if route.numel() == 0:
        return out.to(st["x"].dtype)
    used, slot_e, count = torch.unique(flat[route], return_inverse=True, return_counts=True)
    order = torch.argsort(slot_e, stable=True)
    start = torch.cumsum(count, 0) - count
    pos = torch.empty_like(order)
    pos[order] = torch.arange(order.numel(), device=x.device) - start[slot_e[order]]
    token = route // k
    rows = torch.zeros((used.numel(), int(count.max()), H), device=x.device)
    rows[slot_e, pos] = x[token]

    def weights(name, K):
        z = st["z" + name]
        return _unpack(st["w" + name][used], st["s" + name][used], None if z is None else z[used], K, c["group"])

    u = rows @ weights("13", H).transpose(1, 2)
    h = u[..., :I] * (u[..., I:] / (1.0 + torch.exp(-u[..., I:])))
    y = (h @ weights("2", I).transpose(1, 2))[slot_e, pos] * st["wt"].reshape(-1)[route][:, None]
    every = torch.zeros((T * k, H), device=x.device)
    every[route] = y
    return every.view(T, k, H).sum(1).to(st["x"].dtype)


# -------------------------------------------------------------------------------------------- run
def run(st):
    c = st["case"]
    if not own:
        return {"route": _route_plain, "route_grad": _route_grad_plain, "linear": _linear_plain,
                "experts": _experts_plain}[c["op"]](st)
    moe = st.get("pkg") or st.setdefault("pkg", _pkg())
    if c["op"] == "route":
        return moe.route_experts(st["logits"], c["k"], score=c["score"], bias=st["bias"], n_group=c["groups"],
                                 topk_group=c["topk_groups"], group_score=c["group_score"],
                                 renormalize=c["renormalize"], scale=c["scale"])
    if c["op"] == "route_grad":
        return moe.route_experts_backward(st["grad"], st["logits"], st["idx"], score=c["score"],
                                          renormalize=c["renormalize"], scale=c["scale"])
    if c["op"] == "linear":
        return moe.linear_w4(st["x"], st["codes"], st["scale"], st["zero"], group=c["group"])
    return moe.experts_w4(st["x"], st["idx"], st["wt"], st["w13"], st["s13"], st["w2"], st["s2"],
                          w13_zero=st["z13"], w2_zero=st["z2"], group=c["group"])


# ------------------------------------------------------------------------------------------- work
def _weight_bytes(N, K, group, zero):
    return N * ((K + 1) // 2) + N * -(-K // group) * (3 if zero else 2)


def work(case):
    c, op = case, case["op"]
    if op == "route":
        return {"bytes": c["T"] * c["E"] * SIZE[c["dtype"]] + (4 * c["E"] if c["bias"] else 0) + 8 * c["T"] * c["k"],
                "flops": 8 * c["T"] * c["E"]}
    if op == "route_grad":
        # A sigmoid's gradient needs the picked logits only; a softmax's needs them all.
        read = c["E"] if c["score"] == "softmax" else c["k"]
        return {"bytes": c["T"] * (read + c["E"]) * SIZE[c["dtype"]] + 8 * c["T"] * c["k"],
                "flops": 8 * c["T"] * c["E"]}
    if op == "linear":
        return {"bytes": _weight_bytes(c["N"], c["K"], c["group"], c["zero"]) + 2 * c["M"] * (c["K"] + c["N"]),
                "flops": 2 * c["M"] * c["N"] * c["K"]}
    share = c["k"] / c["EG"]                                    # of the tokens that pick a given expert
    active = c["E"] * (1.0 - (1.0 - share) ** c["T"])           # expected experts with a token
    per = _weight_bytes(2 * c["I"], c["H"], c["group"], c["zero"]) + _weight_bytes(c["H"], c["I"], c["group"], c["zero"])
    return {"bytes": active * per + 4 * c["T"] * c["H"] + 8 * c["T"] * c["k"],
            "flops": 6 * c["T"] * share * c["E"] * c["H"] * c["I"]}


# ------------------------------------------------------------------------------------------ exact
def _product64(x, codes, scale, zero, group):
    """x . W^T in 64 bits, group by group: scale * (x . code - zero * sum(x))."""
    M, K = x.shape
    N, G = scale.shape
    even, odd = codes.double() % 16, (codes // 16).double()
    y = torch.zeros((M, N), dtype=torch.float64, device=x.device)
    for n in range(G):
        a, b = n * group, min(K, (n + 1) * group)
        q = torch.empty((N, (b - a + 1) // 2 * 2), dtype=torch.float64, device=x.device)
        q[:, 0::2], q[:, 1::2] = even[:, a // 2:(b + 1) // 2], odd[:, a // 2:(b + 1) // 2]
        z = 8.0 if zero is None else zero[:, n].double()
        y += scale[:, n].double() * (x[:, a:b] @ q[:, :b - a].T - z * x[:, a:b].sum(-1, keepdim=True))
    return y


def exact(case, seed):
    if work(case)["flops"] > 5e13:
        return None
    st = prepare(case, seed)
    c, op = case, case["op"]
    if op in ("route", "route_grad"):
        x = st["logits"].double()
        s = torch.special.expit(x) if c["score"] == "sigmoid" else torch.softmax(x, -1)
        if op == "route":
            key = s.clone() if st["bias"] is None else s + st["bias"].double()
            key[torch.isneginf(x)] = -math.inf
            per = c["E"] // c["groups"]
            if c["groups"] > 1:
                best = torch.topk(key.view(-1, c["groups"], per), 1 if c["group_score"] == "max" else 2, -1).values.sum(-1)
                rank = torch.argsort(torch.argsort(-best, dim=-1, stable=True), dim=-1, stable=True)
                key = key.masked_fill((rank >= c["topk_groups"]).repeat_interleave(per, -1), -math.inf)
            idx = torch.argsort(-key, dim=-1, stable=True)[:, :c["k"]]
            gone = torch.isneginf(key.gather(1, idx))
            w = s.gather(1, idx).masked_fill(gone, 0.0)
            if c["renormalize"]:
                w = w / (w.sum(-1, keepdim=True) + 1e-20)
            return idx.masked_fill(gone, -1).to(torch.int32), c["scale"] * w
        # d weight_j / d logit_e, written out for every pick j and expert e.
        i, g = st["idx"].long(), c["scale"] * st["grad"].double()
        p = s.gather(1, i)
        if c["renormalize"]:
            D = p.sum(-1, keepdim=True) + 1e-20
            g = g / D - (g * p / D ** 2).sum(-1, keepdim=True)
        if c["score"] == "sigmoid":
            return torch.zeros_like(s).scatter_add_(1, i, g * p * torch.special.expit(-x.gather(1, i)))
        return torch.zeros_like(s).scatter_add_(1, i, g * p) - s * (g * p).sum(-1, keepdim=True)
    if op == "linear":
        return _product64(st["x"].double(), st["codes"], st["scale"], st["zero"], c["group"])
    x, out = st["x"].double(), torch.zeros((c["T"], c["H"]), dtype=torch.float64, device=DEV)
    for e in range(c["E"]):
        t, j = torch.nonzero(st["idx"] == e, as_tuple=True)
        if t.numel() == 0:
            continue
        z13, z2 = (None if z is None else z[e] for z in (st["z13"], st["z2"]))
        u = _product64(x[t], st["w13"][e], st["s13"][e], z13, c["group"])
        h = u[:, :c["I"]] * u[:, c["I"]:] * torch.special.expit(u[:, c["I"]:])
        y = _product64(h, st["w2"][e], st["s2"][e], z2, c["group"])
        out.index_add_(0, t, st["wt"][t, j].double()[:, None] * y)
    return out
