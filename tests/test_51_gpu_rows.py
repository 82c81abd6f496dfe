"""The operators whose rows pick their weights against their definitions in 64 bits.

Tolerances.  u = half a step of the output type.  A sum of K products formed in f32 in
any order, with additions that may truncate (the tensor cores'), is off by at most
2 K 2^-24 sum |x w|; a result of value v then by u |v| more.  silu(v) = v / (1 + e^-v)
with ex2.approx (2 ulp) of a product rounded once: (|v| + 8) 2^-22 relative, and its
slope is below 1.1.  Whole numbers and masks are equal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def randn(seed, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=gen(seed)) * std).to(dtype).to(DEV)


def within(got, want, tol):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol) & ~(torch.isnan(got) & torch.isnan(want)) & ~(got == want)
    if bad.any():
        at = bad.nonzero()[0].tolist()
        i = tuple(at)
        t = tol[i].item() if torch.is_tensor(tol) and tol.shape == got.shape else tol
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off, first at {at}: {got[i].item()} for "
                             f"{want[i].item()}, tolerance {t}")


# ------------------------------------------------------------------------ routing

def route_ref(x, k, bias, sigmoid, groups, top_groups, best, renorm, scale):
    x = x.double()
    T, E = x.shape
    masked = x == -math.inf
    if sigmoid:
        s = torch.sigmoid(x)
    else:
        s = torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0)
    c = s if bias is None else s + bias.double()
    if bias is None and (groups == 1 or best == 1):
        c = x
    c = torch.where(masked, -math.inf, c)
    W = torch.zeros(T, k, dtype=torch.float64)
    I = torch.full((T, k), -1, dtype=torch.int32)
    c_l, s_l = c.tolist(), s.tolist()
    for t in range(T):
        left = list(range(E))
        if groups > 1:
            size = E // groups
            rank = []
            for q in range(groups):
                v = sorted((c_l[t][e] for e in range(q * size, (q + 1) * size)), reverse=True)[:best]
                v = [a for a in v if a > -math.inf]
                rank.append(sum(v) if v else -math.inf)
            kept = sorted(range(groups), key=lambda q: (-rank[q], q))[:top_groups]
            left = [e for e in left if e // size in kept]
        left = [e for e in left if not masked[t, e]]
        left = sorted(left, key=lambda e: (-c_l[t][e], e))[:k]
        tot = sum(s_l[t][e] for e in left) if renorm else 1.0
        for j, e in enumerate(left):
            I[t, j] = e
            W[t, j] = scale * s_l[t][e] / tot
    return W.to(DEV), I.to(DEV)


ROUTES = [  # T, E, k, sigmoid, bias, groups, top_groups, best, renorm, scale
    (1, 8, 1, 0, 0, 1, 1, 1, 1, 1.0), (5, 64, 8, 0, 0, 1, 1, 1, 1, 1.0), (33, 60, 4, 0, 1, 1, 1, 1, 0, 2.0),
    (17, 256, 8, 1, 1, 8, 4, 2, 1, 2.5), (9, 256, 8, 1, 0, 8, 3, 1, 1, 1.0), (12, 128, 6, 0, 0, 4, 2, 2, 0, 1.0),
    (40, 7, 7, 1, 1, 7, 3, 2, 0, 1.0), (3, 1024, 32, 1, 1, 32, 9, 2, 1, 1.0), (6, 300, 3, 0, 1, 1, 1, 1, 1, 1.0),
    (4, 512, 16, 0, 0, 2, 1, 1, 0, 16.0), (2, 1, 1, 0, 0, 1, 1, 1, 0, 1.0)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", ROUTES)
def test_route(handle, pkg, case, dt):
    T, E, k, sig, bias, groups, tg, best, renorm, scale = case
    x = randn(100 + E, T, E, dtype=dt, std=2.0)
    if T > 2:
        x[1, ::2] = -math.inf            # half the experts masked
        x[2] = -math.inf                 # a row that names nobody
        x[2, 0] = 0.5 if T > 5 else -math.inf
    b = randn(7 + E, E, std=0.3) if bias else None
    w, e = handle.route(x, k, bias=b, score=sig, groups=groups, top_groups=tg, group_best=best,
                        renormalize=bool(renorm), scale=scale)
    handle.check()
    assert handle.last_kernel == "route"
    W, I = route_ref(x, k, b, sig, groups, tg, best, renorm, scale)
    assert torch.equal(e, I)
    # expf (2 ulp) of a rounded difference up to 2*8, a sum of 1024 terms by a tree of
    # depth 37, a division, a product: below 64 roundings
    within(w, W, 64 * 2.0 ** -24 * W.abs())


def test_route_ties_and_borders(handle, pkg):
    # equal logits: the lowest indices, in order
    w, e = handle.route(torch.zeros(3, 64, device=DEV), 8)
    assert torch.equal(e.cpu(), torch.arange(8, dtype=torch.int32).expand(3, 8))
    assert torch.equal(w.cpu(), torch.full((3, 8), 0.125))
    # scores that 32 bits cannot tell apart: sigmoid(x) + bias equal to within 2^-30,
    # the larger one at the higher index
    x = torch.zeros(2, 32, device=DEV)
    x[:, 20] = 2.0 ** -28
    w, e = handle.route(x, 2, bias=torch.zeros(32, device=DEV), score=pkg.abi.SCORE_SIGMOID)
    assert e[:, 0].tolist() == [20, 20] and e[:, 1].tolist() == [0, 0]
    # the same between groups ranked by a sum of two
    w, e = handle.route(x, 2, score=pkg.abi.SCORE_SIGMOID, groups=4, top_groups=1, group_best=2)
    assert e.tolist() == [[20, 16], [20, 16]]
    # both zeros rank alike; a bias of -inf ranks behind every number but is not a mask
    x = torch.tensor([[-0.0, 0.0, -1.0]], device=DEV)
    assert handle.route(x, 3)[1].tolist() == [[0, 1, 2]]
    b = torch.tensor([0.0, -math.inf, 0.0], device=DEV)
    assert handle.route(x, 3, bias=b)[1].tolist() == [[0, 2, 1]]


@pytest.mark.parametrize("sig", [0, 1])
@pytest.mark.parametrize("groups, tg, best", [(1, 1, 1), (8, 3, 2), (5, 2, 2)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_route_many_rows_of_near_ties(handle, sig, groups, tg, best, dt):
    """Coarse logits and a coarse bias make equal and nearly equal scores common; the
    choice is still that of the scores in 64 bits, ties by index."""
    T, E, k = 700, 40 if groups == 5 else 64, 6
    x = (torch.randn(T, E, generator=gen(E)) * 8).round().div(8).to(dt).to(DEV)
    if dt == torch.float32:  # and scores that differ by less than 32 bits can tell
        x = x + (torch.randint(0, 3, (T, E), generator=gen(1)) * 2.0 ** -27).to(DEV)
    x[5::17, ::3] = -math.inf
    b = (torch.randn(E, generator=gen(2)) * 4).round().div(16).to(DEV)
    w, e = handle.route(x, k, bias=b, score=sig, groups=groups, top_groups=tg, group_best=best)
    handle.check()
    W, I = route_ref(x, k, b, sig, groups, tg, best, 1, 1.0)
    # torch's and the kernel's 64-bit exponentials may differ in the last bit, which can
    # only show where two sums are that close without being equal: allow for it by value
    same = (e == I).all(1)
    assert same.float().mean() > 0.999
    within(w[same], W[same], 64 * 2.0 ** -24 * W[same].abs())


@pytest.mark.parametrize("sig", [0, 1])
def test_route_far_logits(handle, pkg, sig):
    # chosen scores far below what f32 can hold: the ratios are still those of the scores
    x = torch.tensor([[-300.0, -301.0, -400.0, -302.0]], device=DEV)
    w, e = handle.route(x, 3, score=sig)
    assert e.tolist() == [[0, 1, 3]]
    z = sum(math.exp(-i) for i in range(3))
    within(w, torch.tensor([[math.exp(-i) / z for i in range(3)]], device=DEV), 1e-6)
    # a row's biggest logit is not among the chosen: still normalised
    x = torch.tensor([[50.0, -60.0, -61.0, -62.0]], device=DEV)
    b = torch.tensor([-9.0, 0.0, 1.0, 2.0], device=DEV)
    w, e = handle.route(x, 2, bias=b, score=sig)
    assert e.tolist() == [[3, 2]]
    z = 1 + math.exp(1)
    within(w, torch.tensor([[1 / z, math.exp(1) / z]], device=DEV), 1e-6)


def test_route_nan_and_inf_rows_stay_apart(handle, pkg):
    x = randn(3, 4, 40)
    clean = handle.route(x, 4)
    y = x.clone()
    y[1, 5] = math.nan
    y[2, 6] = math.inf
    w, e = handle.route(y, 4)
    handle.check()
    assert torch.isnan(w[1]).all() and torch.isnan(w[2]).any()
    assert torch.equal(w[[0, 3]], clean[0][[0, 3]]) and torch.equal(e[[0, 3]], clean[1][[0, 3]])
    assert ((e >= 0) & (e < 40)).all()
    # a NaN score ranks behind every number, before masked experts
    z = torch.tensor([[math.nan, 1.0, -math.inf, 0.0]], device=DEV)
    for bias in (None, torch.zeros(4, device=DEV)):
        assert handle.route(z, 4, bias=bias, score=pkg.abi.SCORE_SIGMOID)[1].tolist() == [[1, 3, 0, -1]]


def test_route_strides_and_outputs(handle):
    base = randn(9, 50, 120, dtype=torch.bfloat16)
    views = [base[:, 3:99:2], base.t()[5:69, 1:33].t(), base[::5, 7:8]]
    for v in views:
        k = min(4, v.shape[1])
        w, e = handle.route(v, k)
        w2, e2 = handle.route(v.contiguous(), k)
        assert torch.equal(w, w2) and torch.equal(e, e2)
    # into given buffers; nothing outside them
    buf = torch.full((52, 4), 7.0, device=DEV)
    ids = torch.full((52, 4), 9, device=DEV, dtype=torch.int32)
    handle.route(base, 4, weights=buf[1:51], experts=ids[1:51])
    assert (buf[[0, 51]] == 7).all() and (ids[[0, 51]] == 9).all()
    w, e = handle.route(torch.empty(0, 16, device=DEV), 2)
    assert w.shape == (0, 2) and e.shape == (0, 2)


def route_grad_ref(x, e, g, sigmoid, renorm, scale):
    """By automatic differentiation in 64 bits of the weights at a fixed choice."""
    x = x.double().clone().requires_grad_(True)
    live = e >= 0
    idx = e.clamp(min=0).long()
    if sigmoid:
        s = torch.sigmoid(x)
    else:
        z = torch.where(torch.isinf(x) & (x < 0), -1e300, x)
        s = torch.softmax(z, dim=1)
    c = torch.where(live, s.gather(1, idx), 0.0)
    if renorm:
        c = c / torch.where(live.any(1, keepdim=True), c.sum(1, keepdim=True), 1.0)
    (c * scale * torch.where(live, g.double(), 0.0)).sum().backward()
    d = x.grad.clone()
    d[torch.isinf(x.detach())] = 0.0
    return d


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", ROUTES)
def test_route_backward(handle, case, dt):
    T, E, k, sig, bias, groups, tg, best, renorm, scale = case
    x = randn(200 + E, T, E, dtype=dt, std=2.0)
    if T > 2:
        x[1, ::2] = -math.inf
        x[2] = -math.inf
    b = randn(7 + E, E, std=0.3) if bias else None
    w, e = handle.route(x, k, bias=b, score=sig, groups=groups, top_groups=tg, group_best=best,
                        renormalize=bool(renorm), scale=scale)
    g = randn(5, T, k)
    d = handle.route_backward(x, e, g, score=sig, renormalize=bool(renorm), scale=scale)
    handle.check()
    assert d.dtype == dt
    D = route_grad_ref(x, e, g, sig, renorm, scale)
    # every term is a product of factors in [0, 1], g and scale; at most k + 2 of them meet
    tol = U[dt] * D.abs() + 64 * 2.0 ** -24 * scale * (k + 2) * g.abs().double().amax()
    within(d, D, tol)
    if not (sig == 0 and renorm == 0):
        untouched = torch.ones(T, E + 1, dtype=torch.bool, device=DEV)
        untouched.scatter_(1, torch.where(e < 0, E, e).long(), False)
        assert (d[untouched[:, :E]] == 0).all()


def test_route_backward_against_differences(handle, pkg):
    x = randn(11, 3, 24)
    for sig in (0, 1):
        for renorm in (True, False):
            kw = dict(score=sig, renormalize=renorm, scale=1.5)
            w, e = handle.route(x, 5, **kw)
            g = randn(12, 3, 5)
            d = handle.route_backward(x, e, g, **kw)
            for at in [(0, int(e[0, 0])), (1, int(e[1, 4])), (2, int(e[2, 2]))]:
                h = 2.0 ** -6
                hi, lo = x.clone(), x.clone()
                hi[at] += h
                lo[at] -= h
                fh, eh = handle.route(hi, 5, **kw)
                fl, el = handle.route(lo, 5, **kw)
                # by expert: the order of the choice may change
                pick = lambda f, ee: sum((f[at[0]][ee[at[0]] == e[at[0], j]].sum() * g[at[0], j]).item()
                                         for j in range(5))
                if set(eh[at[0]].tolist()) == set(e[at[0]].tolist()) == set(el[at[0]].tolist()):
                    # third derivative of the weights below 4 * 1.5, k = 5 of them
                    assert abs((pick(fh, eh) - pick(fl, el)) / (2 * h) - d[at].item()) < \
                        h * h / 6 * 6 * 5 * g.abs().max().item() + 1e-4


def test_route_backward_takes_any_choice(handle):
    x = randn(21, 2, 16)
    e = torch.tensor([[3, 3, -1], [99, 15, 0]], dtype=torch.int32, device=DEV)
    g = randn(22, 2, 3)
    d = handle.route_backward(x, e, g, score=1, renormalize=False)
    s = torch.sigmoid(x.double())
    want = torch.zeros(2, 16, dtype=torch.float64, device=DEV)
    want[0, 3] = (g[0, 0] + g[0, 1]).double()
    want[1, 15], want[1, 0] = g[1, 1].double(), g[1, 2].double()
    within(d, want * s * (1 - s), 1e-6)


# --------------------------------------------------------------------------- plan

def plan_ref(index, groups):
    flat = index.flatten().tolist()
    rows = [[i for i, g in enumerate(flat) if g == q] for q in range(groups)]
    order = [i for r in rows for i in r]
    offsets = [0]
    for r in rows:
        offsets.append(offsets[-1] + len(r))
    slots = [-1] * len(flat)
    for p, i in enumerate(order):
        slots[i] = p
    order += [-1] * (len(flat) - len(order))
    return order, offsets, slots


@pytest.mark.parametrize("n, groups", [(0, 3), (1, 1), (31, 4), (128, 64), (1000, 7), (2048, 1024), (2049, 5),
                                       (9000, 33), (40000, 256), (70001, 1000)])
def test_plan_rows(handle, n, groups):
    index = torch.randint(-2, groups + 2, (n,), generator=gen(n), dtype=torch.int32).to(DEV)
    order, offsets, slots = handle.plan_rows(index, groups)
    handle.check()
    o, f, s = plan_ref(index.cpu(), groups)
    assert offsets.tolist() == f and order.tolist() == o and slots.tolist() == s
    again = handle.plan_rows(index, groups)
    assert all(torch.equal(a, b) for a, b in zip(again, (order, offsets, slots)))


def test_plan_rows_extremes(handle):
    for index in (torch.full((5000,), 3, dtype=torch.int32), torch.full((5000,), -1, dtype=torch.int32),
                  torch.tensor([2 ** 31 - 1, -2 ** 31, 0, 7], dtype=torch.int32)):
        order, offsets, slots = handle.plan_rows(index.to(DEV), 8)
        o, f, s = plan_ref(index, 8)
        assert offsets.tolist() == f and order.tolist() == o and slots.tolist() == s
    idx = torch.randint(0, 4, (6, 3), generator=gen(1), dtype=torch.int32).to(DEV)
    assert handle.plan_rows(idx, 4)[2].shape == (6, 3)


# ------------------------------------------------------------------------ products

def act_ref(v, act):
    if act == 1:
        return v.clamp(min=0)
    if act == 2:
        return torch.nn.functional.gelu(v, approximate="tanh")
    if act == 3:
        return v * torch.sigmoid(v)
    return v


def plan_of(handle, seed, T, E, k, pad=0, skew=1.0):
    pop = skew * torch.randn(E, generator=gen(seed))
    noise = -torch.log(-torch.log(torch.rand(T, E, generator=gen(seed + 1)).clamp(1e-9, 1 - 1e-6)))
    idx = torch.topk(pop + noise, k, dim=1).indices.to(torch.int32)
    if pad:
        idx[T - pad:] = -1
    return handle.plan_rows(idx.to(DEV), E)


def products_ref(x, w, offsets, order, fan, gated, act, alpha, bias, out_dt, K):
    """(value, tolerance) over the planned rows, in 64 bits."""
    ends = offsets.tolist()
    P = ends[-1]
    N = w.shape[2] // 2 if gated else w.shape[2]
    rows = order[:P].long() // fan if order is not None else torch.arange(P, device=DEV)
    val = torch.zeros(P, N, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(val)
    eps = 2.0 * (K + 4) * 2.0 ** -24
    for g in range(w.shape[0]):
        a, b = ends[g], ends[g + 1]
        if a == b:
            continue
        xr, wg = x[rows[a:b]].double(), w[g].double()
        v = alpha * (xr @ wg)
        e = eps * abs(alpha) * (xr.abs() @ wg.abs())
        if bias is not None:
            v = v + bias[g].double()
            e = e + eps * bias[g].double().abs()
        e = e + 2.0 ** -23 * v.abs()
        def acted(z, d):
            if act == 0:
                return z, d
            r = act_ref(z, act)
            return r, 1.15 * d + ((z.abs() + 8) * 2.0 ** -22 * r.abs() if act >= 2 else 0)
        if gated:
            r, d = acted(v[:, :N], e[:, :N])
            u, du = v[:, N:], e[:, N:]
            val[a:b] = r * u
            tol[a:b] = d * u.abs() + r.abs() * du + d * du + 2.0 ** -24 * (r * u).abs()
        else:
            val[a:b], tol[a:b] = acted(v, e)
    return val, tol + U[out_dt] * (val.abs() + tol) + TINY[out_dt]


PRODUCTS = [  # T, E, k, K, N, weights layout, gather, gated, pad
    (1, 8, 2, 64, 128, "kn", True, False, 0), (1, 1, 1, 8, 8, "kn", False, False, 0),
    (16, 8, 2, 256, 192, "kn", True, True, 0), (5, 4, 1, 72, 40, "nk", False, False, 1),
    (100, 6, 3, 136, 264, "kn", True, False, 7), (257, 3, 2, 200, 129, "nk", True, True, 0),
    (300, 5, 2, 512, 136, "nk", False, False, 30), (700, 2, 1, 320, 384, "kn", True, False, 0),
    (90, 64, 2, 128, 256, "kn", False, True, 0), (640, 3, 3, 64, 33, "nk", False, False, 0)]


def make_products(handle, case, dt, seed=0):
    T, E, k, K, N, layout, gather, gated, pad = case
    order, offsets, slots = plan_of(handle, 40 + E, T, E, k, pad)
    cols = 2 * N if gated else N
    x = randn(seed + 1, T if gather else T * k, K, dtype=dt)
    if layout == "kn":
        w = randn(seed + 2, E, K, cols, dtype=dt, std=K ** -0.5)
    else:
        w = randn(seed + 2, E, cols, K, dtype=dt, std=K ** -0.5).transpose(1, 2)
    via = dict(order=order, fan=k) if gather else {}
    return x, w, order, offsets, slots, via


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", PRODUCTS)
def test_matmul_grouped(handle, pkg, case, dt):
    T, E, k, K, N, layout, gather, gated, pad = case
    x, w, order, offsets, slots, via = make_products(handle, case, dt)
    act = pkg.abi.ACT_SILU if gated else pkg.abi.ACT_NONE
    out = torch.full((T * k, N), 5.0, device=DEV, dtype=dt)
    handle.matmul_grouped(x, w, offsets, out, gated=gated, activation=act, **via)
    handle.check()
    val, tol = products_ref(x, w, offsets, via.get("order"), k, gated, act, 1.0, None, dt, K)
    P = val.shape[0]
    within(out[:P], val, tol)
    assert (out[P:] == 5.0).all()                       # rows behind the plan are left alone
    again = handle.matmul_grouped(x, w, offsets, gated=gated, activation=act, **via)
    assert torch.equal(again[:P], out[:P])              # the same bits on every run


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("out_dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gated", [False, True])
def test_matmul_grouped_epilogue(handle, act, out_dt, gated):
    case = (70, 5, 2, 192, 144, "kn", True, gated, 3)
    x, w, order, offsets, slots, via = make_products(handle, case, torch.bfloat16)
    for bdt in (torch.float32, torch.bfloat16):
        bias = randn(9, 5, w.shape[2], dtype=bdt)
        y = handle.matmul_grouped(x, w, offsets, gated=gated, activation=act, alpha=0.75, bias=bias,
                                  out_dtype=out_dt, **via)
        handle.check()
        val, tol = products_ref(x, w, offsets, order, 2, gated, act, 0.75, bias, out_dt, 192)
        within(y[:val.shape[0]], val, tol)


def test_which_kernels_run(handle):
    """16-bit operands TMA can describe run on the tensor cores, the rest on CUDA cores."""
    ran = lambda call: (call(), handle.last_kernel)[1]
    for dt, want, grad in [(torch.bfloat16, "grouped_pair", "grouped_grad_pair"),
                           (torch.float32, "grouped_simt", "grouped_grad_simt")]:
        w = randn(1, 4, 64, 128, dtype=dt)
        for T in (40, 400):
            order, offsets, _ = plan_of(handle, 3, T, 4, 1)
            x = randn(2, T, 64, dtype=dt)
            assert ran(lambda: handle.matmul_grouped(x, w, offsets, order=order)) == want
            assert ran(lambda: handle.matmul_grouped(x, w, offsets, gated=True)) == want
        assert ran(lambda: handle.matmul_grouped_grad(x, x, offsets)) == grad
        for T, fast in ((256, "adapters_decode"), (257, "adapters_pair")):
            x, wo, a, b, index = make_adapters((T, 2, 64, 64, 8, "each"), dt)
            assert ran(lambda: handle.matmul_adapters(x, wo, a, b, index)) == (
                fast if dt == torch.bfloat16 else "adapter_simt")
    # a row pitch that is not a multiple of 16 bytes
    x = randn(2, 400, 67, dtype=torch.bfloat16)[:, :64]
    assert ran(lambda: handle.matmul_grouped(x, randn(1, 4, 64, 128, dtype=torch.bfloat16), offsets)) == "grouped_simt"


def test_rows_beyond_two_to_the_31_elements(handle):
    """A source, and rows to combine, whose last rows lie behind 2^31 elements."""
    R, K = 550_000, 4096
    x = torch.zeros(R, K, device=DEV, dtype=torch.bfloat16)
    pick = torch.tensor([R - 1, 3, 524_289, R - 2], device=DEV)
    x[pick] = randn(1, 4, K, dtype=torch.bfloat16)
    w = randn(2, 2, K, 64, dtype=torch.bfloat16, std=0.02)
    for P in (4, 300):
        order = pick[torch.arange(P, device=DEV) % 4].to(torch.int32)
        offsets = torch.tensor([0, P // 2, P], dtype=torch.int32, device=DEV)
        y = handle.matmul_grouped(x, w, offsets, order=order)
        handle.check()
        val, tol = products_ref(x, w, offsets, order, 1, False, 0, 1.0, None, torch.bfloat16, K)
        within(y, val, tol)
    d = handle.matmul_grouped_grad(x, randn(3, P, 64, dtype=torch.bfloat16), offsets, order=order)
    e = handle.matmul_grouped_grad(x[order.long()], randn(3, P, 64, dtype=torch.bfloat16), offsets)
    assert torch.equal(d, e)
    slots = pick.to(torch.int32).view(2, 2)
    assert torch.equal(handle.combine_rows(x, slots, out_dtype=torch.float32),
                       x[pick].float().view(2, 2, K).sum(1))
    g = randn(4, 2, K, dtype=torch.bfloat16)
    other = torch.empty_like(x)
    handle.combine_rows_backward(x, slots, g, grad_rows=other)
    handle.check()
    assert torch.equal(other[pick], g.repeat_interleave(2, 0))


def test_matmul_grouped_strides(handle):
    """Operands and outputs that are views: row pitches, a column offset, weights inside a
    larger tensor, and layouts the tensor cores cannot be fed from."""
    T, E, k, K, N = 60, 4, 2, 96, 80
    order, offsets, slots = plan_of(handle, 3, T, E, k)
    big_x = randn(1, T, K + 40, dtype=torch.bfloat16)
    big_w = randn(2, E + 1, K + 8, N + 24, dtype=torch.bfloat16, std=0.1)
    big_o = torch.zeros(T * k, N + 9, device=DEV, dtype=torch.bfloat16)
    for x, w in [(big_x[:, 16:16 + K], big_w[1:, 8:, 16:16 + N]), (big_x[:, 3:3 + K], big_w[:E, 1:1 + K, 5:5 + N]),
                 (big_x[:, :2 * 48:1][:, :K], big_w[:E, :K, :N])]:
        for o in (big_o[:, 8:8 + N], big_o[:, 1:1 + N]):
            big_o.fill_(3.0)
            handle.matmul_grouped(x, w, offsets, o, order=order, fan=k)
            handle.check()
            val, tol = products_ref(x, w, offsets, order, k, False, 0, 1.0, None, torch.bfloat16, K)
            within(o, val, tol)
            assert int((big_o == 3.0).sum()) >= T * k * 9      # the pitch's gap is not written
    xt = randn(4, K, T, dtype=torch.bfloat16).t()              # unit stride on rows
    o = torch.zeros(N, T * k, device=DEV, dtype=torch.bfloat16).t()
    w = big_w[:E, :K, :N]
    handle.matmul_grouped(xt, w, offsets, o, order=order, fan=k)
    handle.check()
    val, tol = products_ref(xt, w, offsets, order, k, False, 0, 1.0, None, torch.bfloat16, K)
    within(o, val, tol)


def test_matmul_grouped_keeps_rows_apart(handle):
    """NaN and infinities in one row, or in another group's weights, reach nobody else."""
    T, E, k, K, N = 50, 3, 1, 128, 128
    order, offsets, slots = plan_of(handle, 5, T, E, k)
    x, w = randn(1, T, K, dtype=torch.bfloat16), randn(2, E, K, N, dtype=torch.bfloat16, std=0.1)
    clean = handle.matmul_grouped(x, w, offsets, order=order, fan=k)
    x2, w2 = x.clone(), w.clone()
    x2[7] = math.nan
    x2[8, 0] = math.inf
    w2[1] = math.nan
    y = handle.matmul_grouped(x2, w2, offsets, order=order, fan=k)
    handle.check()
    ends = offsets.tolist()
    p = torch.arange(T, device=DEV)
    hit = ((p >= ends[1]) & (p < ends[2])) | (order == 7) | (order == 8)
    assert torch.equal(y[~hit], clean[~hit]) and torch.isnan(y[slots[7]]).all()


def test_matmul_grouped_broken_plans(handle):
    """Offsets and orders that lead nowhere: rows of zeros, nothing outside the tensors."""
    x, w = randn(1, 10, 64, dtype=torch.bfloat16), randn(2, 3, 64, 64, dtype=torch.bfloat16)
    order = torch.tensor([0, 9, 10, 2 ** 31 - 1, -5, 3], dtype=torch.int32, device=DEV)
    offsets = torch.tensor([0, 4, 4, 6], dtype=torch.int32, device=DEV)
    out = torch.full((8, 64), 2.0, device=DEV, dtype=torch.bfloat16)
    handle.matmul_grouped(x, w, offsets, out[:6], order=order)
    handle.check()
    assert (out[[2, 3, 4]] == 0).all() and (out[6:] == 2).all()
    val, tol = products_ref(x, w, torch.tensor([0, 2, 2, 2]), torch.tensor([0, 9], device=DEV), 1, False, 0, 1.0,
                            None, torch.bfloat16, 64)
    within(out[:2], val, tol)
    wild = torch.tensor([-7, 2, 900, 1], dtype=torch.int32, device=DEV)     # not even ascending
    out.fill_(2.0)
    handle.matmul_grouped(x, w, wild, out[:6], order=order)
    handle.check()
    assert (out[6:] == 2).all()
    for dt in (torch.bfloat16, torch.float32):  # groups that seem to overlap: the first one has the rows
        big, v = randn(4, 700, 64, dtype=dt), randn(5, 40, 64, 64, dtype=dt, std=0.125)
        over = torch.tensor([0] + [700, 0] * 20, dtype=torch.int32, device=DEV)
        got = handle.matmul_grouped(big, v, over)
        handle.check()
        val, tol = products_ref(big, v, torch.tensor([0] + [700] * 40), None, 1, False, 0, 1.0, None, dt, 64)
        within(got, val, tol)
    d = handle.matmul_grouped_grad(x, randn(3, 6, 64, dtype=torch.bfloat16), wild, order=order)
    handle.check()
    assert d.shape == (3, 64, 64)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", PRODUCTS)
def test_matmul_grouped_gradients(handle, case, dt):
    T, E, k, K, N, layout, gather, gated, pad = case
    x, w, order, offsets, slots, via = make_products(handle, case, dt)
    N = w.shape[2]
    dy = randn(7, T * k, N, dtype=dt)
    # rows: the same call with transposed weights
    dx = handle.matmul_grouped(dy, w.transpose(1, 2), offsets)
    handle.check()
    val, tol = products_ref(dy, w.transpose(1, 2), offsets, None, 1, False, 0, 1.0, None, dt, N)
    P = val.shape[0]
    within(dx[:P], val, tol)
    for out_dt in {dt, torch.float32}:
        dw = handle.matmul_grouped_grad(x, dy, offsets, out_dtype=out_dt, alpha=0.5, **via)
        handle.check()
        ends = offsets.tolist()
        rows = order[:P].long() // k if gather else torch.arange(P, device=DEV)
        want = torch.zeros(E, K, N, dtype=torch.float64, device=DEV)
        slack = torch.zeros_like(want)
        for g in range(E):
            a, b = ends[g], ends[g + 1]
            if b > a:
                xr, d = x[rows[a:b]].double(), dy[a:b].double()
                want[g] = 0.5 * (xr.t() @ d)
                slack[g] = 2.0 * (b - a + 4) * 2.0 ** -24 * 0.5 * (xr.abs().t() @ d.abs())
            else:
                assert (dw[g] == 0).all()
        within(dw, want, slack + U[out_dt] * (want.abs() + slack) + TINY[out_dt])


def test_matmul_grouped_grad_of_long_groups(handle):
    """An f32 gradient over thousands of rows keeps the precision of rounded sums: it is
    accumulated 1024 rows at a time.  A sum of R random terms in which each of the R / 16
    additions loses at most 2^-23 of the running sum is off by at most R / 16 2^-23 of it;
    pieces of 1024 rows lose 64 2^-23, and joining them half a step each."""
    R = [5000, 0, 1024, 1025, 2049, 3100, 7]
    K, N = 264, 392
    off = torch.tensor([0] + R).cumsum(0).to(torch.int32).to(DEV)
    x, dy = randn(1, sum(R), K, dtype=torch.bfloat16), randn(2, sum(R), N, dtype=torch.bfloat16)
    for out_dt in (torch.float32, torch.bfloat16):
        big = torch.full((len(R), K, N + 4), 3.0, device=DEV, dtype=out_dt)
        d = handle.matmul_grouped_grad(x, dy, off, big[:, :, :N])
        handle.check()
        assert (big[:, :, N:] == 3.0).all()
        assert torch.equal(d, handle.matmul_grouped_grad(x, dy, off, out_dtype=out_dt))
        ends = off.tolist()
        for g, r in enumerate(R):
            ref = x[ends[g]:ends[g + 1]].double().t() @ dy[ends[g]:ends[g + 1]].double()
            err = (d[g].double() - ref).norm().item()
            limit = (64 * 2.0 ** -23 + 8 * 2.0 ** -24) if out_dt == torch.float32 else r / 16 * 2.0 ** -23 + 2.0 ** -8
            assert err <= limit * ref.norm().item(), (g, err / ref.norm().item())


def test_matmul_grouped_grad_ignores_other_rows(handle):
    """Rows behind the plan and rows of other groups hold NaN and infinities."""
    T, E, K, N = 100, 4, 72, 136
    idx = torch.randint(-1, 3, (T,), generator=gen(5), dtype=torch.int32).to(DEV)  # group 3 stays empty
    order, offsets, slots = handle.plan_rows(idx, E)
    ends = offsets.tolist()
    x, dy = randn(1, T, K, dtype=torch.bfloat16), randn(2, T, N, dtype=torch.bfloat16)
    clean = handle.matmul_grouped_grad(x, dy, offsets, order=order)
    dy2 = dy.clone()
    dy2[ends[-1]:] = math.nan
    dy2[ends[1]:ends[2]] = math.inf
    x2 = x.clone()
    x2[idx < 0] = math.nan
    d = handle.matmul_grouped_grad(x2, dy2, offsets, order=order)
    handle.check()
    assert torch.equal(d[[0, 2, 3]], clean[[0, 2, 3]]) and (d[3] == 0).all()


# ------------------------------------------------------------------------- combine

@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T, k, N", [(1, 1, 8), (3, 2, 64), (50, 8, 256), (17, 5, 100), (9, 9, 2056), (20, 32, 33),
                                     (7, 3, 1)])
def test_combine_rows(handle, dt, T, k, N):
    R = T * k + 3
    rows = randn(1, R, N, dtype=dt)
    slots = torch.randperm(R, generator=gen(2))[:T * k].to(torch.int32).view(T, k)
    if T > 2:
        slots[1] = -1
        slots[2, 0] = R + 5
    named = slots[(slots >= 0) & (slots < R)].long()
    poison = torch.ones(R, dtype=torch.bool)
    poison[named] = False
    rows[poison.to(DEV)] = math.nan                   # rows nobody names are not read
    slots = slots.to(DEV)
    w = randn(3, T, k)
    live = ((slots >= 0) & (slots < R)).unsqueeze(2)
    pick = torch.where(live, rows[slots.clamp(0, R - 1).long()].double(), 0.0)
    for wt in (w, None):
        ww = torch.ones(T, k, device=DEV).double() if wt is None else wt.double()
        val = (pick * ww.unsqueeze(2)).sum(1)
        slack = 2 * k * 2.0 ** -24 * (pick.abs() * ww.abs().unsqueeze(2)).sum(1)
        out = handle.combine_rows(rows, slots, weights=wt)
        handle.check()
        within(out, val, slack + U[dt] * (val.abs() + slack) + TINY[dt])
        wide = handle.combine_rows(rows, slots, weights=wt, out_dtype=torch.float32)
        within(wide, val, slack + U[torch.float32] * val.abs())
    # gradients
    dout = randn(4, T, N, dtype=dt)
    keep = torch.full((R, N), 4.0, device=DEV, dtype=dt)
    drows, dw = handle.combine_rows_backward(rows, slots, dout, weights=w, grad_rows=keep)
    handle.check()
    want = torch.full((R, N), 4.0, dtype=torch.float64, device=DEV)
    sl = slots[live.squeeze(2)].long()
    want[sl] = (w.double().unsqueeze(2) * dout.double().unsqueeze(1))[live.squeeze(2)]
    within(drows, want, 2.0 ** -24 * want.abs() + U[dt] * (1 + 2.0 ** -23) * want.abs() + TINY[dt])
    wd = (pick * dout.double().unsqueeze(1)).sum(2)
    within(dw, wd, 2 * N * 2.0 ** -24 * (pick.abs() * dout.double().abs().unsqueeze(1)).sum(2) + 2.0 ** -24 * wd.abs())
    ones, none = handle.combine_rows_backward(rows, slots, dout)
    assert none is None and torch.equal(ones[sl], dout.unsqueeze(1).expand(T, k, N)[live.squeeze(2)])


def test_combine_rows_views(handle):
    rows = randn(1, 40, 99, dtype=torch.float16)[:, 2:2 + 64]
    slots = torch.arange(40, dtype=torch.int32, device=DEV).view(10, 4)
    out = torch.zeros(10, 70, device=DEV, dtype=torch.float16)
    handle.combine_rows(rows, slots, out[:, 3:67])
    want = rows.double().view(10, 4, 64).sum(1)
    slack = 8 * 2.0 ** -24 * rows.double().abs().view(10, 4, 64).sum(1)
    within(out[:, 3:67], want, slack + U[torch.float16] * (want.abs() + slack))
    assert (out[:, :3] == 0).all() and (out[:, 67:] == 0).all()
    assert handle.combine_rows(rows, torch.empty(0, 4, dtype=torch.int32, device=DEV)).shape == (0, 64)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N", [127, 129, 300, 1301])
@pytest.mark.parametrize("layout", ["odd", "spread", "columns", "types"])
def test_combine_rows_any_layout(handle, dt, N, layout):
    """Rows that start anywhere, columns apart, rows behind one another column by column, and
    tensors of three types: forward and backward."""
    T, k, other = 11, 5, {torch.bfloat16: torch.float32, torch.float16: torch.bfloat16, torch.float32: torch.float16}

    def view(seed, rows, dt):
        if layout == "spread":
            return randn(seed, rows, 2 * N + 1, dtype=dt)[:, 1::2]
        if layout == "columns":
            return randn(seed, N, rows, dtype=dt).t()
        return randn(seed, rows, N, dtype=dt)

    rows, dout = view(1, T * k, dt), view(2, T, other[dt] if layout == "types" else dt)
    drows = view(3, T * k, other[other[dt]] if layout == "types" else dt)
    slots = torch.randperm(T * k, generator=gen(4)).to(torch.int32).view(T, k).to(DEV)
    slots[3, 2] = -1
    kept = torch.ones(T * k, dtype=torch.bool, device=DEV)
    kept[slots[slots >= 0].long()] = False
    before = drows.clone()
    w = randn(5, T, k)
    out = torch.zeros_like(dout)
    handle.combine_rows(rows, slots, out, weights=w)
    _, dw = handle.combine_rows_backward(rows, slots, dout, weights=w, grad_rows=drows)
    handle.check()
    live = (slots >= 0).unsqueeze(2)
    pick = torch.where(live, rows[slots.clamp(min=0).long()].double(), 0.0)
    ww, g = w.double().unsqueeze(2), dout.double().unsqueeze(1)
    val, slack = (pick * ww).sum(1), 2 * k * 2.0 ** -24 * (pick * ww).abs().sum(1)
    within(out, val, slack + U[out.dtype] * (val.abs() + slack) + TINY[out.dtype])
    want = torch.where(live, ww * g, 0.0)
    got = drows[slots.clamp(min=0).long()]
    within(torch.where(live, got, 0.0), want,
           2.0 ** -24 * want.abs() + U[drows.dtype] * (1 + 2.0 ** -23) * want.abs() + TINY[drows.dtype])
    assert torch.equal(drows[kept], before[kept])
    wd = (pick * g).sum(2)
    within(dw, wd, 2 * N * 2.0 ** -24 * (pick * g).abs().sum(2) + 2.0 ** -24 * wd.abs())


# ------------------------------------------------------------------------ adapters

def adapters_ref(x, w, a, b, index, scale, alpha, bias, bias_axis, act, out_dt):
    K, r = a.shape[1], a.shape[2]
    xd = x.double()
    v = alpha * (xd @ w.double())
    e = 2.0 * (K + 8) * 2.0 ** -24 * abs(alpha) * (xd.abs() @ w.double().abs())
    if bias is not None:
        bb = bias.double() if bias_axis == 1 else bias.double().unsqueeze(1)
        v = v + bb
        e = e + 2.0 ** -22 * bb.abs()
    for i in range(a.shape[0]):
        rows = (index == i).nonzero().flatten()
        if rows.numel() == 0:
            continue
        s = 1.0 if scale is None else scale[i].double()
        low = xd[rows] @ a[i].double()
        low_e = 2.0 * (K + 8) * 2.0 ** -24 * (xd[rows].abs() @ a[i].double().abs())
        # the inner product keeps 16 bits at least (high and low half of the operand
        # type; the low half of an f16 below its smallest step, 2^-24, is lost)
        low_e = low_e + 2.0 ** -16 * low.abs() + 2.0 ** -24
        v[rows] += s * (low @ b[i].double())
        e[rows] += abs(s) * (low_e @ b[i].double().abs() +
                             2.0 * (r + 8) * 2.0 ** -24 * (low.abs() @ b[i].double().abs()))
    e = e + 2.0 ** -22 * v.abs()
    o = act_ref(v, act)
    e = 1.15 * e + ((v.abs() + 8) * 2.0 ** -22 * o.abs() if act >= 2 else 0)
    return o, e + U[out_dt] * (o.abs() + e) + TINY[out_dt]


ADAPTERS = [  # T, G, K, N, r, how the rows choose
    (1, 1, 64, 64, 8, "one"), (1, 4, 256, 136, 16, "none"), (3, 4, 72, 128, 1, "each"), (16, 8, 256, 256, 16, "each"),
    (64, 30, 512, 200, 16, "each"), (65, 5, 128, 264, 32, "each"), (130, 3, 264, 128, 64, "runs"),
    (300, 7, 192, 384, 16, "runs"), (513, 40, 128, 130, 8, "each"), (700, 2, 320, 256, 128, "runs"),
    (260, 6, 136, 72, 20, "runs"), (200, 3, 64, 72, 8, "each"), (256, 9, 640, 264, 16, "each"),
    (257, 4, 64, 256, 8, "each"), (90, 5, 1160, 136, 40, "each")]


def make_adapters(case, dt, up_layout="rn", seed=0):
    T, G, K, N, r, how = case
    x = randn(seed + 1, T, K, dtype=dt)
    w = randn(seed + 2, K, N, dtype=dt, std=K ** -0.5)
    a = randn(seed + 3, G, K, r, dtype=dt, std=K ** -0.5)
    b = randn(seed + 4, G, r, N, dtype=dt)
    if up_layout == "nr":  # stored the other way round
        a = a.transpose(1, 2).contiguous().transpose(1, 2)
        b = b.transpose(1, 2).contiguous().transpose(1, 2)
    if how == "each":
        index = torch.randint(-1, G, (T,), generator=gen(seed + 5))
    elif how == "runs":
        index = torch.randint(-1, G, (9,), generator=gen(seed + 5))[torch.arange(T) * 9 // T]
    else:
        index = torch.full((T,), 0 if how == "one" else G)
    return x, w, a, b, index.to(torch.int32).to(DEV)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["rn", "nr"])
@pytest.mark.parametrize("case", ADAPTERS)
def test_matmul_adapters(handle, case, layout, dt):
    x, w, a, b, index = make_adapters(case, dt, layout)
    scale = torch.rand(a.shape[0], generator=gen(6)).to(DEV) + 0.5
    out = handle.matmul_adapters(x, w, a, b, index, scale=scale)
    handle.check()
    val, tol = adapters_ref(x, w, a, b, index, scale, 1.0, None, 1, 0, dt)
    within(out, val, tol)
    assert torch.equal(out, handle.matmul_adapters(x, w, a, b, index, scale=scale))
    if case[5] == "none":  # nobody has an adapter: the shared projection alone
        val, tol = adapters_ref(x, w, a, b, torch.full_like(index, -1), None, 1.0, None, 1, 0, dt)
        within(out, val, tol)


@pytest.mark.parametrize("T", [5, 200])
@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("axis", [0, 1])
def test_matmul_adapters_epilogue(handle, T, act, axis):
    x, w, a, b, index = make_adapters((T, 4, 128, 144, 16, "each"), torch.bfloat16)
    for out_dt in (torch.float32, torch.bfloat16):
        bias = randn(8, 144 if axis == 1 else T, dtype=out_dt)
        out = handle.matmul_adapters(x, w, a, b, index, alpha=0.5, bias=bias, bias_axis=axis, activation=act,
                                     out_dtype=out_dt)
        handle.check()
        val, tol = adapters_ref(x, w, a, b, index, None, 0.5, bias, axis, act, out_dt)
        within(out, val, tol)


@pytest.mark.parametrize("T", [12, 150])
def test_matmul_adapters_keep_requests_apart(handle, T):
    """A broken adapter or input row spoils its own rows only."""
    x, w, a, b, index = make_adapters((T, 4, 128, 128, 16, "each"), torch.bfloat16)
    clean = handle.matmul_adapters(x, w, a, b, index)
    a2, b2, x2 = a.clone(), b.clone(), x.clone()
    a2[1], b2[2] = math.nan, math.inf
    x2[0] = math.nan
    out = handle.matmul_adapters(x2, w, a2, b2, index)
    handle.check()
    hit = (index == 1) | (index == 2)
    hit[0] = True
    assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("T", [9, 140])
def test_matmul_adapters_strides(handle, T):
    G, K, N, r = 3, 96, 112, 16
    bx = randn(1, T, K + 24, dtype=torch.bfloat16)
    bw = randn(2, K + 3, N + 16, dtype=torch.bfloat16, std=0.1)
    ba = randn(3, G + 1, K, r + 8, dtype=torch.bfloat16, std=0.1)
    bb = randn(4, G, r + 1, N + 8, dtype=torch.bfloat16)
    index = torch.randint(-1, G, (T,), generator=gen(5), dtype=torch.int32).to(DEV)
    o = torch.full((T, N + 5), 3.0, device=DEV, dtype=torch.bfloat16)
    for x, w, a, b in [(bx[:, 8:8 + K], bw[3:, 8:8 + N], ba[1:, :, 8:], bb[:, 1:, 8:]),
                       (bx[:, 1:1 + K], bw[:K, 1:1 + N], ba[:G, :, 1:1 + r], bb[:, :r, 3:3 + N]),
                       (bx[:, :K], bw[:K, :N].t().contiguous().t(), ba[:G, :, :r], bb[:, :r, :N])]:
        for out in (o[:, :N], o[:, 5:]):
            o.fill_(3.0)
            handle.matmul_adapters(x, w, a, b, index, out)
            handle.check()
            val, tol = adapters_ref(x, w, a, b, index, None, 1.0, None, 1, 0, torch.bfloat16)
            within(out, val, tol)
            assert int((o == 3.0).sum()) >= 5 * T


# -------------------------------------------------- the operators as they are used

def test_experts_layer_forward_and_backward(handle, pkg):
    """Routing, plan, gated first product, second product, weighted sum; then all
    gradients, composed from the operators and from kapyb_elementwise's formula for the
    gate, against automatic differentiation of the layer in 64 bits."""
    T, E, k, H, I = 96, 6, 2, 128, 64
    dt = torch.float32           # f32 storage: the composition's own roundings stay small
    x, wr = randn(1, T, H), randn(2, H, E, std=0.3)
    w1, w2 = randn(3, E, H, I, std=H ** -0.5), randn(4, E, I, H, std=I ** -0.5)
    logits = (x.double() @ wr.double()).float()
    w, e = handle.route(logits, k)
    order, offsets, slots = handle.plan_rows(e, E)
    h = handle.matmul_grouped(x, w1, offsets, order=order, fan=k, activation=pkg.abi.ACT_NONE)
    y = handle.matmul_grouped(h, w2, offsets)
    out = handle.combine_rows(y, slots, weights=w)
    dout = randn(5, T, H)
    dy, dw = handle.combine_rows_backward(y, slots, dout, weights=w)
    dh = handle.matmul_grouped(dy, w2.transpose(1, 2), offsets)
    dw2 = handle.matmul_grouped_grad(h, dy, offsets)
    dxr = handle.matmul_grouped(dh, w1.transpose(1, 2), offsets)
    dw1 = handle.matmul_grouped_grad(x, dh, offsets, order=order, fan=k)
    dx = handle.combine_rows(dxr, slots)
    dlogits = handle.route_backward(logits, e, dw)
    handle.check()
    X, W1, W2, L = (t.double().requires_grad_(True) for t in (x, w1, w2, logits))
    p = torch.softmax(L, 1).gather(1, e.long())
    p = p / p.sum(1, keepdim=True)
    ref = torch.zeros(T, H, dtype=torch.float64, device=DEV)
    for j in range(k):
        z = torch.einsum("th,thi->ti", X, W1[e[:, j].long()])
        ref = ref + p[:, j:j + 1] * torch.einsum("ti,tih->th", z, W2[e[:, j].long()])
    (ref * dout.double()).sum().backward()
    # chains of at most four f32 products of sizes up to 128 * T rows
    for got, want in ((out, ref.detach()), (dx, X.grad), (dw1, W1.grad), (dw2, W2.grad), (dlogits, L.grad)):
        within(got, want, 1e-5 * want.abs().max())


@pytest.mark.parametrize("dt", [torch.bfloat16])
def test_experts_layer_in_a_graph_on_another_stream(handle, pkg, dt):
    """The serving sequence captured once and replayed on new inputs gives what eager calls
    give, also beside a second graph of the same handle in flight on another stream."""
    T, E, k, H, I = 24, 8, 2, 256, 128
    w1, w2 = randn(3, E, H, 2 * I, dtype=dt, std=H ** -0.5), randn(4, E, I, H, dtype=dt, std=I ** -0.5)
    a, b = randn(5, 4, H, 16, dtype=dt, std=H ** -0.5), randn(6, 4, 16, H, dtype=dt)
    wo = randn(7, H, H, dtype=dt, std=H ** -0.5)

    def layer(x, logits, who, stream=None):
        w, e = handle.route(logits, k, stream=stream)
        order, offsets, slots = handle.plan_rows(e, E, stream=stream)
        h = handle.matmul_grouped(x, w1, offsets, order=order, fan=k, gated=True, activation=pkg.abi.ACT_SILU,
                                  stream=stream)
        y = handle.matmul_grouped(h, w2, offsets, stream=stream)
        o = handle.combine_rows(y, slots, weights=w, stream=stream)
        return handle.matmul_adapters(o, wo, a, b, who, stream=stream)

    def inputs(seed):
        return (randn(seed, T, H, dtype=dt), randn(seed + 1, T, E, dtype=dt),
                torch.randint(-1, 4, (T,), generator=gen(seed), dtype=torch.int32).to(DEV))

    held, graphs, outs = [inputs(50), inputs(60)], [], []
    for i in range(2):
        layer(*held[i])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(*held[i]))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        fresh = [inputs(100 + 10 * turn), inputs(105 + 10 * turn)]
        for i in range(2):
            for dst, src in zip(held[i], fresh[i]):
                dst.copy_(src)
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                for _ in range(3):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], layer(*fresh[i])), (turn, i)
    handle.check()
    # an explicit stream, while another one is current
    s = torch.cuda.Stream()
    got = layer(*held[0], stream=s)
    s.synchronize()
    assert torch.equal(got, layer(*held[0]))
    got = layer(*held[1], stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(got, layer(*held[1]))


def test_training_step_in_a_graph(handle, pkg):
    """Forward and backward calls, long groups in pieces and adapters of many rows, captured
    once and replayed on new inputs: the bits of eager calls."""
    T, E, k, H, N = 1500, 2, 2, 128, 264
    dt = torch.bfloat16
    w = randn(3, E, H, N, dtype=dt, std=H ** -0.5)
    wo, a, b = randn(5, H, N, dtype=dt, std=H ** -0.5), randn(6, 4, H, 24, dtype=dt), randn(7, 4, 24, N, dtype=dt)

    def step(x, logits, g, who):
        wts, e = handle.route(logits, k)
        order, offsets, slots = handle.plan_rows(e, E)
        y = handle.matmul_grouped(x, w, offsets, order=order, fan=k)
        out = handle.combine_rows(y, slots, weights=wts)
        dy, dwts = handle.combine_rows_backward(y, slots, g, weights=wts)
        dw = handle.matmul_grouped_grad(x, dy, offsets, order=order, fan=k, out_dtype=torch.float32)
        dx = handle.combine_rows(handle.matmul_grouped(dy, w.transpose(1, 2), offsets), slots)
        dl = handle.route_backward(logits, e, dwts)
        return out, dw, dx, dl, handle.matmul_adapters(x, wo, a, b, who)

    def inputs(seed):
        return (randn(seed, T, H, dtype=dt), randn(seed + 1, T, E), randn(seed + 2, T, N, dtype=dt),
                torch.randint(-1, 4, (T,), generator=gen(seed), dtype=torch.int32).to(DEV))

    held = inputs(50)
    step(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held)
    for turn in range(3):
        fresh = inputs(100 + 10 * turn)
        for dst, src in zip(held, fresh):
            dst.copy_(src)
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        for i, (u, v) in enumerate(zip(got, step(*fresh))):
            assert torch.equal(u, v), (turn, i)
    handle.check()


def test_python_refusals(handle, pkg):
    x = randn(1, 4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        handle.route(x.cpu(), 2)
    with pytest.raises(ValueError, match="top_k"):
        handle.route(x, 9)
    with pytest.raises(ValueError, match="bias"):
        handle.route(x, 2, bias=torch.zeros(7, device=DEV))
    with pytest.raises(ValueError, match="element type"):
        handle.plan_rows(torch.zeros(4, device=DEV, dtype=torch.int64), 2)
    with pytest.raises(ValueError, match="contiguous"):
        handle.plan_rows(torch.zeros(8, device=DEV, dtype=torch.int32)[::2], 2)
    off = torch.zeros(3, device=DEV, dtype=torch.int32)
    with pytest.raises(ValueError, match="offsets"):
        handle.matmul_grouped(x, torch.zeros(3, 8, 8, device=DEV), off)
    with pytest.raises(ValueError, match="columns of lhs"):
        handle.matmul_grouped(x, torch.zeros(2, 7, 8, device=DEV), off)
    with pytest.raises(ValueError, match="order"):
        handle.matmul_grouped_grad(x, x, off, order=torch.zeros(3, device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError, match="slots"):
        handle.combine_rows(x, torch.zeros(4, device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError, match="index"):
        handle.matmul_adapters(x, torch.zeros(8, 8, device=DEV), torch.zeros(1, 8, 2, device=DEV),
                               torch.zeros(1, 2, 8, device=DEV), torch.zeros(3, device=DEV, dtype=torch.int32))
