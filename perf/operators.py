"""The operators whose rows pick their weights (routing to experts, the experts'
products, the weighted sum of their rows, low-rank adapters of many requests), as
cases that can be measured: inputs, one pass in plain torch operations or through
the library (`own`), the definition in 64 bits, and the work a pass cannot avoid."""
import math
import random

import torch

own = False

_package = _handle = None
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _library():
    """The package and the program's handle, made once as a user's program does."""
    global _package, _handle
    if _handle is None:
        import __graft_entry__
        _package = __graft_entry__.load_package()

        class Handle(_package.Handle):
            def plan_rows(self, index, groups):
                # slots have the shape of the index: a flat one, as the plain form's
                return super().plan_rows(index.reshape(-1), groups)

        _handle = Handle(0)
    return _package.abi, _handle


# ------------------------------------------------------------------------ cases

def listed():
    return [
        # one token of a decode step is routed: pure latency
        dict(name="route_token", op="route", T=1, E=64, k=8, dtype="bf16", score="softmax", bias=False,
             groups=1, top_groups=1, best=1, renorm=True, scale=1.0, train=False, pad=0),
        # a long prompt, biased sigmoid scores, experts in groups, the last rows padding
        dict(name="route_prompt", op="route", T=16384, E=256, k=8, dtype="f32", score="sigmoid", bias=True,
             groups=8, top_groups=4, best=2, renorm=True, scale=2.5, train=False, pad=300),
        # a training step's routing with the gradient of the logits
        dict(name="route_train", op="route", T=8192, E=128, k=8, dtype="bf16", score="softmax", bias=False,
             groups=1, top_groups=1, best=1, renorm=True, scale=1.0, train=True, pad=0),
        # a decode step of 16 sequences: gated first product, nearly all weights streamed once
        dict(name="experts_decode", op="experts", T=16, E=64, k=8, K=4096, N=2048, dtype="bf16", gated=True,
             gather=True, wlayout="kn", skew=0.0, train=False, pad=0),
        # the gated first product of a prompt, rows fetched through the plan
        dict(name="experts_prompt", op="experts", T=8192, E=64, k=8, K=2048, N=1024, dtype="bf16", gated=True,
             gather=True, wlayout="kn", skew=0.5, train=False, pad=0),
        # odd sizes, an uneven load and weights stored [N, K]; rows already in plan order, as in the second product
        dict(name="experts_odd", op="experts", T=1777, E=10, k=3, K=1000, N=999, dtype="f16", gated=False,
             gather=False, wlayout="nk", skew=1.5, train=False, pad=20),
        # a training step: gradients of the rows and of the weights
        dict(name="experts_train", op="experts", T=8192, E=16, k=4, K=2048, N=2048, dtype="bf16", gated=False,
             gather=True, wlayout="kn", skew=0.5, train=True, pad=0),
        # the experts' rows of a prompt summed per token
        dict(name="combine_prompt", op="combine", T=8192, k=8, N=4096, dtype="bf16", train=False, pad=0),
        # the same in training, forward and backward
        dict(name="combine_train", op="combine", T=4096, k=4, N=2048, dtype="bf16", train=True, pad=100),
        # one sequence decoding beside the shared projection
        dict(name="adapters_token", op="adapters", T=1, G=8, K=4096, N=4096, r=16, dtype="bf16", spread="each",
             none=0.0),
        # 64 sequences of 32 tenants in one decode step, some of them without an adapter
        dict(name="adapters_mixed", op="adapters", T=64, G=32, K=8192, N=8192, r=16, dtype="f16", spread="each",
             none=0.1),
        # the prompts of a few requests, one after the other
        dict(name="adapters_prompt", op="adapters", T=8192, G=12, K=4096, N=4096, r=64, dtype="bf16",
             spread="runs", none=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "experts", "experts", "combine", "adapters", "adapters"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        E = groups * _log(rng, 4, 512 // groups if groups > 1 else 300)
        top_groups = rng.randint(max(1, groups // 2), groups)
        k = rng.randint(1, min(16, (E // groups) * top_groups))
        T = _log(rng, 1, 16384)
        return dict(op=op, T=T, E=E, k=k, dtype=rng.choice(["bf16", "f16", "f32"]),
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups,
                    top_groups=top_groups, best=rng.choice([1, 2]), renorm=rng.random() < 0.7,
                    scale=rng.choice([1.0, 2.5]), train=rng.random() < 0.4, pad=rng.randint(0, T // 8))
    if op == "experts":
        E = _log(rng, 2, 96)
        k = rng.randint(1, min(E, 8))
        while True:
            T = _log(rng, 1, 8192)
            K = 8 * _log(rng, 16, 512)
            N = _log(rng, 16, 512)
            layout = rng.choice(["kn", "nk"])
            # rows of [K, N] weights start on 16 bytes; stored [N, K] they may be any number
            N = 8 * N if layout == "kn" else 8 * N - rng.randint(0, 7)
            gated = rng.random() < 0.4
            train = not gated and rng.random() < 0.4
            if layout == "nk" and train:
                N = (N + 7) // 8 * 8
            if gated and layout == "kn":
                N = (N + 7) // 8 * 8
            cost = 2.0 * T * k * K * N * (2 if gated or train else 1)
            if cost <= 5e11 and E * K * N * (2 if gated else 1) <= 1.1e9:
                break
        return dict(op=op, T=T, E=E, k=k, K=K, N=N, dtype=rng.choice(["bf16", "f16"]), gated=gated,
                    gather=rng.random() < 0.6, wlayout=layout, skew=rng.choice([0.0, 0.5, 1.5]), train=train,
                    pad=rng.randint(0, T // 8))
    if op == "combine":
        T, k = _log(rng, 1, 8192), rng.randint(1, 8)
        N = _log(rng, 64, 8192)
        while T * k * N > 8192 * 8 * 4096:
            T = max(1, T // 2)
        return dict(op=op, T=T, k=k, N=N, dtype=rng.choice(["bf16", "f16", "f32"]),
                    train=rng.random() < 0.5, pad=rng.randint(0, T // 8))
    while True:
        T = _log(rng, 1, 8192)
        K, N = 8 * _log(rng, 32, 1024), 8 * _log(rng, 32, 1024)
        if T * K * N <= 8192 * 4096 * 4096:
            break
    return dict(op=op, T=T, G=_log(rng, 1, 64), K=K, N=N, r=rng.choice([8, 16, 32, 64]),
                dtype=rng.choice(["bf16", "f16"]), spread="each" if T <= 96 else "runs",
                none=rng.choice([0.0, 0.1, 0.5]))


# ----------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _choices(g, case):
    """k distinct experts per token, popular ones more often; -1 for padding tokens."""
    T, E, k = case["T"], case["E"], case["k"]
    pop = case["skew"] * torch.randn(E, generator=g, device="cuda")
    noise = -torch.log(-torch.log(torch.rand(T, E, generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)))
    idx = torch.topk(pop + noise, k, dim=1).indices.to(torch.int32)
    if case["pad"]:
        idx[T - case["pad"]:] = -1
    return idx.contiguous()


def _weights(g, case, n_cols):
    """[E, K, n_cols] as the user sees it, stored that way or with K contiguous."""
    E, K, dt = case["E"], case["K"], _DT[case["dtype"]]
    std = 1.0 / math.sqrt(K)
    if case["wlayout"] == "kn":
        w = torch.empty(E, K, n_cols, device="cuda", dtype=dt)
    else:
        w = torch.empty(E, n_cols, K, device="cuda", dtype=dt)
    for e in range(E):
        w[e] = torch.randn(w.shape[1:], generator=g, device="cuda").mul_(std)
    return w if case["wlayout"] == "kn" else w.transpose(1, 2)


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case=case)
    op, dt = case["op"], _DT[case["dtype"]]
    if own:
        abi, st["h"] = _library()
        st["score"] = abi.SCORE_SIGMOID if case.get("score") == "sigmoid" else abi.SCORE_SOFTMAX
        st["activation"] = abi.ACT_SILU if case.get("gated") else abi.ACT_NONE
    if op == "route":
        T, E = case["T"], case["E"]
        x = _randn(g, T, E, std=1.5)
        if case["pad"]:
            x[T - case["pad"]:] = -math.inf
        st["x"] = x.to(dt)
        st["bias"] = _randn(g, E, std=0.05) if case["bias"] else None
        if case["train"]:
            st["g"] = _randn(g, T, case["k"])
    elif op == "experts":
        T, k, K, N = case["T"], case["k"], case["K"], case["N"]
        st["index"] = _choices(g, case)
        n_x = T if case["gather"] else T * k
        st["x"] = _randn(g, n_x, K, dtype=dt)
        st["w"] = _weights(g, case, 2 * N if case["gated"] else N)
        if case["train"]:
            st["dy"] = _randn(g, T * k, N, dtype=dt, std=0.1)
            st["dx"] = torch.zeros(T * k, K, device="cuda", dtype=dt)
        else:
            # rows behind the last planned one keep what the buffer holds
            st["y"] = torch.zeros(T * k, N, device="cuda", dtype=dt)
    elif op == "combine":
        T, k, N = case["T"], case["k"], case["N"]
        st["rows"] = _randn(g, T * k, N, dtype=dt)
        slots = torch.randperm(T * k, generator=g, device="cuda").to(torch.int32).view(T, k)
        if case["pad"]:
            slots[T - case["pad"]:] = -1
        st["slots"] = slots.contiguous()
        st["w"] = torch.softmax(_randn(g, T, k), dim=1)
        if case["train"]:
            st["dout"] = _randn(g, T, N, dtype=dt)
            st["drows"] = torch.zeros(T * k, N, device="cuda", dtype=dt)
    else:
        T, G, K, N, r = case["T"], case["G"], case["K"], case["N"], case["r"]
        st["x"] = _randn(g, T, K, dtype=dt)
        st["w"] = _randn(g, K, N, dtype=dt, std=1.0 / math.sqrt(K))
        st["a"] = _randn(g, G, K, r, dtype=dt, std=1.0 / math.sqrt(K))
        st["b"] = _randn(g, G, r, N, dtype=dt, std=1.0 / math.sqrt(r))
        st["scale"] = torch.rand(G, generator=g, device="cuda") + 0.5
        n_req = T if case["spread"] == "each" else min(T, 16)
        who = torch.randint(0, G, (n_req,), generator=g, device="cuda")
        who[torch.rand(n_req, generator=g, device="cuda") < case["none"]] = -1
        if case["spread"] == "each":
            st["index"] = who.to(torch.int32)
        else:
            cuts = torch.rand(n_req - 1, generator=g, device="cuda").sort().values * T
            st["index"] = who[torch.searchsorted(cuts, torch.arange(T, device="cuda") + 0.5)].to(torch.int32)
    return st


# ------------------------------------------------------------------ plain forms

def _plain_scores(x, score):
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    top = x.max(dim=1, keepdim=True).values
    e = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    z = e.sum(dim=1, keepdim=True)
    return e / torch.where(z == 0, torch.ones_like(z), z)


def _plain_route(st):
    c = st["case"]
    x, k, E = st["x"], c["k"], c["E"]
    masked = torch.isinf(x) & (x < 0)
    wide = x.double()                       # borders between experts are decided in 64 bits
    sel = _plain_scores(wide, c["score"])
    if st["bias"] is not None:
        sel = sel + st["bias"].double()
    sel = torch.where(masked, torch.full_like(sel, -math.inf), sel)
    if c["groups"] > 1:
        per = sel.view(-1, c["groups"], E // c["groups"])
        best = torch.sort(per, dim=2, descending=True, stable=True).values[..., :c["best"]]
        best = torch.where(torch.isinf(best), torch.zeros_like(best), best).sum(dim=2)
        best = torch.where(torch.isinf(per).all(dim=2), torch.full_like(best, -math.inf), best)
        keep = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, keep, True)
        sel = torch.where(kept.unsqueeze(2), per, torch.full_like(per, -math.inf)).reshape(-1, E)
    order = torch.sort(sel, dim=1, descending=True, stable=True)
    idx, none = order.indices[:, :k], torch.isinf(order.values[:, :k])
    s = _plain_scores(x.float(), c["score"])
    w = torch.where(none, torch.zeros_like(s[:, :k]), s.gather(1, idx))
    total = w.sum(dim=1, keepdim=True)
    if c["renorm"]:
        w = w / torch.where(total == 0, torch.ones_like(total), total)
    w = w * c["scale"]
    experts = torch.where(none, torch.full_like(idx, -1), idx).to(torch.int32)
    if not c["train"]:
        return w, experts
    grad = torch.where(none, torch.zeros_like(st["g"]), st["g"]) * c["scale"]
    ds = grad
    if c["renorm"]:
        unit = torch.where(total == 0, torch.ones_like(total), total)
        ds = (grad - (grad * w / c["scale"]).sum(dim=1, keepdim=True)) / unit
    ds = torch.where(none, torch.zeros_like(ds), ds)
    full = torch.zeros_like(s).scatter_add_(1, idx, ds)
    if c["score"] == "sigmoid":
        dx = full * s * (1.0 - s)
    else:
        dx = s * (full - (s * full).sum(dim=1, keepdim=True))
    return w, experts, dx.to(x.dtype)


def _plain_plan(index, groups):
    flat = index.reshape(-1).long()
    key = torch.where((flat < 0) | (flat >= groups), torch.full_like(flat, groups), flat)
    order = torch.sort(key, stable=True).indices
    count = (key.unsqueeze(0) == torch.arange(groups, device=key.device).unsqueeze(1)).sum(dim=1)
    offsets = torch.zeros(groups + 1, dtype=torch.long, device=key.device)
    offsets[1:] = count.cumsum(0)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(order.numel(), device=key.device)
    slots = torch.where(key == groups, torch.full_like(pos, -1), pos)
    order = torch.where(torch.arange(order.numel(), device=key.device) < offsets[groups], order,
                        torch.full_like(order, -1))
    return order.to(torch.int32), offsets.to(torch.int32), slots.to(torch.int32)


def _silu(v):
    return v / (1.0 + torch.exp(-v))


def _plain_experts(st):
    c = st["case"]
    order, offsets, slots = _plain_plan(st["index"], c["E"])
    ends = offsets.tolist()
    src = torch.div(order.long(), c["k"], rounding_mode="floor") if c["gather"] else \
        torch.arange(order.numel(), device=order.device)
    x, w = st["x"], st["w"]
    if c["train"]:
        dw = torch.zeros(w.shape, device=w.device, dtype=torch.float32)
        dx = torch.zeros_like(st["dx"])
        for e in range(c["E"]):
            a, b = ends[e], ends[e + 1]
            if b > a:
                dy = st["dy"][a:b].float()
                dx[a:b] = (dy @ w[e].float().t()).to(dx.dtype)
                dw[e] = x[src[a:b]].float().t() @ dy
        return order, offsets, slots, dx, dw
    y = torch.zeros_like(st["y"])
    for e in range(c["E"]):
        a, b = ends[e], ends[e + 1]
        if b > a:
            v = x[src[a:b]].float() @ w[e].float()
            if c["gated"]:
                v = _silu(v[:, :c["N"]]) * v[:, c["N"]:]
            y[a:b] = v.to(y.dtype)
    return order, offsets, slots, y


def _plain_combine(st):
    c = st["case"]
    rows, slots, w = st["rows"], st["slots"].long(), st["w"]
    live = slots >= 0
    safe = torch.where(live, slots, torch.zeros_like(slots))
    out = torch.zeros(c["T"], c["N"], device=rows.device)
    for j in range(c["k"]):
        v = rows[safe[:, j]].float() * w[:, j:j + 1]
        out = out + torch.where(live[:, j:j + 1], v, torch.zeros_like(v))
    out = out.to(rows.dtype)
    if not c["train"]:
        return out
    drows = torch.zeros_like(st["drows"])
    dw = torch.zeros_like(w)
    dout = st["dout"].float()
    for j in range(c["k"]):
        on = live[:, j]
        drows[slots[on, j]] = (w[on, j:j + 1] * dout[on]).to(drows.dtype)
        dw[on, j] = (rows[slots[on, j]].float() * dout[on]).sum(dim=1)
    return out, drows, dw


def _plain_adapters(st):
    c = st["case"]
    x = st["x"].float()
    out = x @ st["w"].float()
    for i in range(c["G"]):
        on = st["index"] == i
        # a product over all rows, kept where the row names this adapter: no host copy
        if c["T"] <= 96:
            out = out + torch.where(on.unsqueeze(1), (x @ st["a"][i].float()) @ st["b"][i].float()
                                    * st["scale"][i], torch.zeros_like(out))
        else:
            rows = on.nonzero().squeeze(1)
            out[rows] = out[rows] + (x[rows] @ st["a"][i].float()) @ st["b"][i].float() * st["scale"][i]
    return out.to(st["x"].dtype)


def run(st):
    c = st["case"]
    if not own:
        return {"route": _plain_route, "experts": _plain_experts, "combine": _plain_combine,
                "adapters": _plain_adapters}[c["op"]](st)
    h = st["h"]
    if c["op"] == "route":
        w, experts = h.route(st["x"], c["k"], bias=st["bias"], score=st["score"], groups=c["groups"],
                             top_groups=c["top_groups"], group_best=c["best"], renormalize=c["renorm"],
                             scale=c["scale"])
        if not c["train"]:
            return w, experts
        return w, experts, h.route_backward(st["x"], experts, st["g"], score=st["score"],
                                            renormalize=c["renorm"], scale=c["scale"])
    if c["op"] == "experts":
        order, offsets, slots = h.plan_rows(st["index"], c["E"])
        via = dict(order=order, fan=c["k"]) if c["gather"] else {}
        if c["train"]:
            dx = h.matmul_grouped(st["dy"], st["w"].transpose(1, 2), offsets, st["dx"])
            dw = h.matmul_grouped_grad(st["x"], st["dy"], offsets, out_dtype=torch.float32, **via)
            return order, offsets, slots, dx, dw
        y = h.matmul_grouped(st["x"], st["w"], offsets, st["y"], gated=c["gated"],
                             activation=st["activation"], **via)
        return order, offsets, slots, y
    if c["op"] == "combine":
        out = h.combine_rows(st["rows"], st["slots"], weights=st["w"])
        if not c["train"]:
            return out
        drows, dw = h.combine_rows_backward(st["rows"], st["slots"], st["dout"], weights=st["w"],
                                            grad_rows=st["drows"])
        return out, drows, dw
    return h.matmul_adapters(st["x"], st["w"], st["a"], st["b"], st["index"], scale=st["scale"])


# ------------------------------------------------------------------------- work

def work(case):
    op, es = case["op"], {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    if op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        b, f = T * E * es + T * k * 8 + (4 * E if case["bias"] else 0), 6 * T * E
        if case["train"]:
            b, f = b + T * k * 4 + T * E * es, 2 * f
        return {"bytes": b, "flops": f}
    if op == "experts":
        T, E, k, K = case["T"], case["E"], case["k"], case["K"]
        cols = case["N"] * (2 if case["gated"] else 1)
        P = (T - case["pad"]) * k
        # experts that some token names, if the choices were even
        active = E * (1.0 - (1.0 - k / E) ** max(0, T - case["pad"]))
        n_x = (T - case["pad"]) if case["gather"] else P
        b = n_x * K * es + P * case["N"] * es + active * K * cols * es + 12 * T * k
        f = 2.0 * P * K * cols
        if case["train"]:
            b, f = b + P * K * es + E * K * cols * 4, 2 * f
        return {"bytes": int(b), "flops": int(f)}
    if op == "combine":
        T, k, N = case["T"] - case["pad"], case["k"], case["N"]
        b, f = T * k * N * es + case["T"] * (N * es + 8 * k), 2 * T * k * N
        if case["train"]:
            # the rows and the output's gradient are read, the rows' gradient is written
            b, f = b + T * k * N * es + T * N * es + 4 * T * k, 2 * f + T * k * N
        return {"bytes": b, "flops": f}
    T, K, N, r, G = case["T"], case["K"], case["N"], case["r"], case["G"]
    n_req = T if case["spread"] == "each" else min(T, 16)
    touched = G * (1.0 - (1.0 - (1.0 - case["none"]) / G) ** n_req)
    b = es * (T * K + K * N + T * N + touched * r * (K + N)) + 4 * T
    f = 2 * T * K * N + 2 * T * r * (K + N) * (1.0 - case["none"])
    return {"bytes": int(b), "flops": int(f)}


# ------------------------------------------------------- the definition, 64 bits

def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"route": _exact_route, "experts": _exact_experts, "combine": _exact_combine,
            "adapters": _exact_adapters}[case["op"]](st)


def _exact_route(st):
    c = st["case"]
    x = st["x"].to(torch.float64)
    T, E = x.shape
    k = c["k"]
    alive = x > -math.inf
    if c["score"] == "softmax":
        s = torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0)
    else:
        s = torch.sigmoid(x)
    value = s if st["bias"] is None else s + st["bias"].to(torch.float64)
    allowed = alive.clone()
    if c["groups"] > 1:
        size = E // c["groups"]
        score = torch.full((T, c["groups"]), -math.inf, dtype=torch.float64, device=x.device)
        for q in range(c["groups"]):
            v = torch.where(alive, value, -math.inf)[:, q * size:(q + 1) * size]
            top = torch.topk(v, min(c["best"], size), dim=1).values
            some = top[:, 0] > -math.inf
            score[:, q] = torch.where(some, torch.where(top > -math.inf, top, 0.0).sum(dim=1), -math.inf)
        ahead = torch.zeros(T, c["groups"], dtype=torch.long, device=x.device)
        for q in range(c["groups"]):
            for o in range(c["groups"]):
                if o != q:
                    better = score[:, o] >= score[:, q] if o < q else score[:, o] > score[:, q]
                    ahead[:, q] += better
        for q in range(c["groups"]):
            allowed[:, q * size:(q + 1) * size] &= (ahead[:, q] < c["top_groups"]).unsqueeze(1)
    left = torch.where(allowed, value, -math.inf)
    experts = torch.full((T, k), -1, dtype=torch.int32, device=x.device)
    w = torch.zeros(T, k, dtype=torch.float64, device=x.device)
    where = torch.arange(E, device=x.device).expand(T, E)
    for j in range(k):
        top = left.amax(dim=1, keepdim=True)
        e = torch.where(left == top, where, E).amin(dim=1)
        ok = top.squeeze(1) > -math.inf
        experts[:, j] = torch.where(ok, e, -1).to(torch.int32)
        w[:, j] = torch.where(ok, s.gather(1, e.unsqueeze(1)).squeeze(1), 0.0)
        left = left.scatter(1, e.unsqueeze(1), -math.inf)
    total = w.sum(dim=1, keepdim=True) if c["renorm"] else torch.ones(T, 1, dtype=w.dtype, device=w.device)
    total = torch.where(total > 0, total, 1.0)
    out = w / total * c["scale"]
    if not c["train"]:
        return out, experts
    # the formula's Jacobian, applied column by column of the chosen experts
    ok = experts >= 0
    e = experts.clamp(min=0).long()
    g = torch.where(ok, st["g"].to(torch.float64), 0.0)
    d = c["scale"] * g / total
    if c["renorm"]:
        d = d - (c["scale"] * g * w).sum(dim=1, keepdim=True) / total ** 2
    d = torch.where(ok, d, 0.0)
    dx = torch.zeros_like(x)
    for j in range(k):
        if c["score"] == "sigmoid":
            col = (d[:, j] * w[:, j] * (1.0 - w[:, j])).unsqueeze(1)
            dx.scatter_add_(1, e[:, j:j + 1], col)
        else:
            col = (d[:, j] * w[:, j]).unsqueeze(1)
            dx -= col * s
            dx.scatter_add_(1, e[:, j:j + 1], col)
    return out, experts, dx


def _exact_experts(st):
    c = st["case"]
    flat = st["index"].reshape(-1).cpu().tolist()
    rows_of = [[] for _ in range(c["E"])]
    for i, e in enumerate(flat):
        if 0 <= e < c["E"]:
            rows_of[e].append(i)
    order, offsets, slots = [], [0], [-1] * len(flat)
    for rows in rows_of:
        for i in rows:
            slots[i] = len(order)
            order.append(i)
        offsets.append(len(order))
    order += [-1] * (len(flat) - len(order))
    dev = st["x"].device
    ints = [torch.tensor(v, dtype=torch.int32, device=dev) for v in (order, offsets, slots)]
    f64 = torch.float64
    rows = len(flat)
    if c["train"]:
        dx = torch.zeros(rows, c["K"], dtype=f64, device=dev)
        dw = torch.zeros(c["E"], c["K"], c["N"], dtype=f64, device=dev)
    else:
        y = torch.zeros(rows, c["N"], dtype=f64, device=dev)
    for e in range(c["E"]):
        lo, hi = offsets[e], offsets[e + 1]
        if lo == hi:
            continue
        pick = torch.tensor(rows_of[e], device=dev)
        xr = st["x"].index_select(0, pick // c["k"]) if c["gather"] else st["x"][lo:hi]
        xr, we = xr.to(f64), st["w"][e].to(f64)
        if c["train"]:
            d = st["dy"][lo:hi].to(f64)
            dx[lo:hi] = torch.mm(d, we.transpose(0, 1))
            dw[e] = torch.mm(xr.transpose(0, 1), d)
        else:
            v = torch.mm(xr, we)
            if c["gated"]:
                gate, up = v.split(c["N"], dim=1)
                v = gate * torch.sigmoid(gate) * up
            y[lo:hi] = v
    return (*ints, dx, dw) if c["train"] else (*ints, y)


def _exact_combine(st):
    c = st["case"]
    rows = st["rows"].to(torch.float64)
    pad_rows = torch.cat([rows, torch.zeros(1, c["N"], dtype=rows.dtype, device=rows.device)])
    slots = st["slots"].long()
    slots = torch.where(slots < 0, c["T"] * c["k"], slots)
    w = st["w"].to(torch.float64)
    out = torch.zeros(c["T"], c["N"], dtype=rows.dtype, device=rows.device)
    for j in range(c["k"]):
        out.addcmul_(w[:, j:j + 1], pad_rows[slots[:, j]])
    if not c["train"]:
        return out
    dout = st["dout"].to(torch.float64)
    drows = torch.zeros_like(pad_rows)
    dw = torch.empty_like(w)
    for j in range(c["k"]):
        drows.index_copy_(0, slots[:, j], w[:, j:j + 1] * dout)
        dw[:, j] = torch.einsum("tn,tn->t", dout, pad_rows[slots[:, j]])
    return out, drows[:-1], dw


def _exact_adapters(st):
    c = st["case"]
    x = st["x"].to(torch.float64)
    out = torch.mm(x, st["w"].to(torch.float64))
    who = st["index"].cpu()
    for i in sorted(set(who.tolist()) - {-1}):
        rows = torch.nonzero(who == i).flatten().to(x.device)
        low = torch.mm(x.index_select(0, rows), st["a"][i].to(torch.float64))
        out.index_add_(0, rows, torch.mm(low, st["b"][i].to(torch.float64)) * st["scale"][i].to(torch.float64))
    return out


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(s)) for s in range(6)]:
        print(c, work(c))
