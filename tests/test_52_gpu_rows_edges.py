"""Rows that pick their weights, at the ends of what the calls are documented to take.

Tolerances as in test_51_gpu_rows.  Beyond 256 rows the low-rank part is 2 r more terms
(two halves of each inner product) in the sum of the shared part, so all of it is one sum of
K + 2 r terms.  The inner product is divided by d before it is stored as two 16-bit values and
multiplied by d at the end (bf16: d = alpha; f16: alpha, or below 1 its mantissa, 1 <= d < 2).
The second value is half a step off what the first one left: in bf16 2^-8 of 2^-8 of the
product, in f16 2^-11 of 2^-11, but at least half of f16's smallest step, 2^-25 of what was
stored, d 2^-25 of the product: below 2^-24 for d < 2, else |alpha| 2^-25."""
import math

import pytest
import torch

from test_51_gpu_rows import DEV, TINY, U, act_ref, gen, make_adapters, plan_of, randn, within

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------ adapters

def adapters_want(x, w, a, b, index, scale, alpha, bias, bias_axis, act, out_dt):
    """(value, tolerance) in 64 bits."""
    K, r = a.shape[1], a.shape[2]
    eps = 2.0 * (K + 2 * r + 16) * 2.0 ** -24
    xd, wd, ad, bd = (t.double() for t in (x, w, a, b))
    v = alpha * (xd @ wd)
    size = abs(alpha) * (xd.abs() @ wd.abs())
    low_err = torch.zeros_like(v)
    if bias is not None:
        bb = bias.double() if bias_axis == 1 else bias.double().unsqueeze(1)
        v, size = v + bb, size + bb.abs()
    for i in range(a.shape[0]):
        rows = (index == i).nonzero().flatten()
        s = 1.0 if scale is None else scale[i].double()
        low = s * (xd[rows] @ ad[i])
        e = 2.0 * (K + 8) * 2.0 ** -24 * abs(s) * (xd[rows].abs() @ ad[i].abs()) + \
            2.0 ** -16 * low.abs() + max(2.0 ** -24, abs(alpha) * 2.0 ** -25)
        v[rows] += low @ bd[i]
        size[rows] += low.abs() @ bd[i].abs()
        low_err[rows] += e @ bd[i].abs()
    e = eps * size + low_err + 2.0 ** -22 * v.abs()
    o = act_ref(v, act)
    e = 1.15 * e + ((v.abs() + 8) * 2.0 ** -22 * o.abs() if act >= 2 else 0)
    return o, e + U[out_dt] * (o.abs() + e) + TINY[out_dt]


@pytest.mark.parametrize("T", [256, 257, 700])
@pytest.mark.parametrize("alpha", [1 / 256, -0.5, 1.0, -2.0, 256.0, 1000.0])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_matmul_adapters_any_alpha(handle, T, alpha, dt):
    """Inner products of some 300 beside any scale of the shared part, and one row more or
    less does not change what a call can take."""
    x, w, a, b, index = make_adapters((T, 4, 192, 144, 16, "each"), dt)
    scale = torch.tensor([300.0, 1.0, 2.0 ** -10, 30.0], device=DEV)
    out = handle.matmul_adapters(x, w, a, b, index, scale=scale, alpha=alpha, out_dtype=torch.float32)
    handle.check()
    val, tol = adapters_want(x, w, a, b, index, scale, alpha, None, 1, 0, torch.float32)
    within(out, val, tol)


@pytest.mark.parametrize("T", [200, 300])
@pytest.mark.parametrize("alpha", [1 / 256, 1.0, 2.0, 16.0, 256.0])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_matmul_adapters_small_products(handle, T, alpha, dt):
    """Inner products of 2^-10 and less with nothing else in the sum."""
    x, w, a, b, index = make_adapters((T, 3, 128, 72, 16, "each"), dt)
    scale = torch.tensor([2.0 ** -10, 2.0 ** -14, 1.0], device=DEV)
    w = torch.zeros_like(w)
    out = handle.matmul_adapters(x, w, a, b, index, scale=scale, alpha=alpha, out_dtype=torch.float32)
    handle.check()
    val, tol = adapters_want(x, w, a, b, index, scale, alpha, None, 1, 0, torch.float32)
    within(out, val, tol)


@pytest.mark.parametrize("alpha", [1 / 256, 0.3, 0.5, 0.999, -0.0625])
@pytest.mark.parametrize("axis", [0, 1])
def test_matmul_adapters_f16_scales_below_one(handle, alpha, axis):
    """Rows with an adapter are scaled in two steps, rows without one at once."""
    x, w, a, b, index = make_adapters((600, 4, 128, 144, 16, "each"), torch.float16)
    bias = randn(8, 600 if axis == 0 else 144, dtype=torch.float16)
    out = torch.full((600, 150), 3.0, device=DEV, dtype=torch.float16)
    handle.matmul_adapters(x, w, a, b, index, out[:, 3:147], alpha=alpha, bias=bias, bias_axis=axis, activation=1)
    handle.check()
    assert handle.last_kernel == "adapters_pair"
    val, tol = adapters_want(x, w, a, b, index, None, alpha, bias, axis, 1, torch.float16)
    within(out[:, 3:147], val, tol)
    assert (out[:, :3] == 3.0).all() and (out[:, 147:] == 3.0).all()


@pytest.mark.parametrize("T", [200, 300])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_matmul_adapters_infinite_product(handle, T, dt):
    """An inner product of +inf meets positive factors: +inf, and no other row changes."""
    x, w, a, b, index = make_adapters((T, 3, 128, 72, 8, "each"), dt)
    x[:, 0], b[1] = 1.0, b[1].abs() + 0.125
    clean = handle.matmul_adapters(x, w, a, b, index)
    a2 = a.clone()
    a2[1, 0, 3] = math.inf
    out = handle.matmul_adapters(x, w, a2, b, index)
    handle.check()
    hit = index == 1
    assert hit.any() and (out[hit] == math.inf).all()
    assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("T", [300, 700])
@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("axis", [0, 1, None])
@pytest.mark.parametrize("dt, alpha", [(torch.bfloat16, 0.5), (torch.bfloat16, -2.0), (torch.float16, 1.5)])
def test_matmul_adapters_epilogue_of_many_rows(handle, T, act, axis, dt, alpha):
    x, w, a, b, index = make_adapters((T, 4, 128, 144, 16, "each"), dt)
    for out_dt in (torch.float32, torch.bfloat16, torch.float16):
        bias = None if axis is None else randn(8, 144 if axis == 1 else T, dtype=out_dt)
        out = handle.matmul_adapters(x, w, a, b, index, alpha=alpha, bias=bias, bias_axis=axis or 0, activation=act,
                                     out_dtype=out_dt)
        handle.check()
        assert handle.last_kernel == "adapters_pair"
        val, tol = adapters_want(x, w, a, b, index, None, alpha, bias, axis, act, out_dt)
        within(out, val, tol)


@pytest.mark.parametrize("T", [300, 700])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_matmul_adapters_keep_many_requests_apart(handle, T, dt):
    x, w, a, b, index = make_adapters((T, 4, 128, 128, 16, "each"), dt)
    clean = handle.matmul_adapters(x, w, a, b, index)
    a2, b2, x2 = a.clone(), b.clone(), x.clone()
    a2[1], b2[2] = math.nan, math.inf
    x2[0], x2[T - 1] = math.nan, math.inf
    out = handle.matmul_adapters(x2, w, a2, b2, index)
    handle.check()
    assert handle.last_kernel == "adapters_pair"
    hit = (index == 1) | (index == 2)
    hit[0] = hit[T - 1] = True
    assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("T", [300, 513])
@pytest.mark.parametrize("out_dt", [torch.bfloat16, torch.float32])
def test_matmul_adapters_strides_of_many_rows(handle, T, out_dt):
    """Views TMA can describe, outputs that start anywhere, an odd number of columns (weights
    and up stored the other way round), and views it cannot."""
    G, K, r = 3, 96, 16
    for N in (112, 131):
        bx = randn(1, T, K + 24, dtype=torch.bfloat16)
        bw = randn(2, K + 3, 136, dtype=torch.bfloat16, std=0.1)
        bt = randn(6, 136, K + 8, dtype=torch.bfloat16, std=0.1)
        ba = randn(3, G + 1, K, r + 8, dtype=torch.bfloat16, std=0.1)
        bb = randn(4, G, r + 1, 136, dtype=torch.bfloat16)
        bu = randn(7, G, 136, r + 8, dtype=torch.bfloat16)
        index = torch.randint(-1, G, (T,), generator=gen(5), dtype=torch.int32).to(DEV)
        o = torch.full((T, N + 5), 3.0, device=DEV, dtype=out_dt)
        straight = [(bx[:, 8:8 + K], bw[3:, :N], ba[1:, :, 8:], bb[:, 1:, :N], N % 8 == 0 or "adapters_pair"),
                    (bx[:, :K], bt[:N, 8:].t(), ba[:G, :, :r], bu[:, :N, 8:].transpose(1, 2), "adapters_pair"),
                    (bx[:, 1:1 + K], bw[:K, 1:1 + N], ba[:G, :, 1:1 + r], bb[:, :r, 3:3 + N], "adapter_simt")]
        for x, w, a, b, kernel in straight:
            for out in (o[:, :N], o[:, 5:], o[:, 4:4 + N]):
                o.fill_(3.0)
                handle.matmul_adapters(x, w, a, b, index, out)
                handle.check()
                assert kernel is True or handle.last_kernel == kernel
                val, tol = adapters_want(x, w, a, b, index, None, 1.0, None, 1, 0, out_dt)
                within(out, val, tol)
                out.fill_(3.0)
                assert (o == 3.0).all()


# ----------------------------------------------------------------- weight gradients

def gradient_want(x, dy, offsets, order, fan, out_dt):
    """(value, tolerance): offsets clamped to the positions and made ascending, positions
    whose source does not exist left out on both sides."""
    P, src = dy.shape[0], x.shape[0]
    high, starts, ends = 0, [], []
    raw = [min(max(o, 0), P) for o in offsets.tolist()]
    for g in range(len(raw) - 1):
        high = max(high, raw[g])
        starts.append(high)
        ends.append(max(high, raw[g + 1]))
    val = torch.zeros(len(starts), x.shape[1], dy.shape[1], dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(val)
    rows = torch.arange(P, device=DEV) if order is None else \
        torch.where(order < 0, -1, torch.div(order.long(), fan, rounding_mode="floor"))
    there = (rows >= 0) & (rows < src)
    for g, (a, b) in enumerate(zip(starts, ends)):
        on = there[a:b].nonzero().flatten() + a
        xr, d = x[rows[on]].double(), dy[on].double()
        val[g] = xr.t() @ d
        tol[g] = 2.0 * (b - a + 4) * 2.0 ** -24 * (xr.abs().t() @ d.abs())
    return val, tol + U[out_dt] * (val.abs() + tol) + TINY[out_dt]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offsets", [[0, 10, 5, 20], [0] + [700, 0] * 20, [-7, 2, 900, 1], [30, 20, 10, 700],
                                     [0, 300, 100, 400, 200, 700]])
def test_matmul_grouped_grad_of_falling_offsets(handle, dt, offsets):
    """An offset below the one before it counts as that one: no row in two groups."""
    x, dy = randn(1, 700, 40, dtype=dt), randn(2, 700, 72, dtype=dt)
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    d = handle.matmul_grouped_grad(x, dy, off, out_dtype=torch.float32)
    handle.check()
    val, tol = gradient_want(x, dy, off, None, 1, torch.float32)
    within(d, val, tol)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out_dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fan", [1, 3])
def test_matmul_grouped_grad_of_missing_rows(handle, dt, out_dt, fan):
    """A position whose order names no row counts as zeros, whatever its gradient holds."""
    src, P, E, K, N = 900, 2600, 4, 72, 264
    x = randn(1, src, K, dtype=dt)
    order = torch.randint(0, src * fan, (P,), generator=gen(3), dtype=torch.int32)
    holes = torch.tensor([0, 63, 64, 130, 131, 199, 1000, 1500, 1501, 2400, 2599])
    order[holes] = torch.tensor([-1, src * fan, 2 ** 31 - 1, -2 ** 31, src * fan + 1, -5, -1, -1, src * fan, -3, -1],
                                dtype=torch.int32)
    order = order.to(DEV)
    offsets = torch.tensor([0, 200, 200, 2500, 2600], dtype=torch.int32, device=DEV)
    dy = randn(2, P, N, dtype=dt)
    clean = handle.matmul_grouped_grad(x, dy, offsets, order=order, fan=fan, out_dtype=out_dt)
    val, tol = gradient_want(x, dy, offsets, order, fan, out_dt)
    within(clean, val, tol)
    dy[holes.to(DEV)] = math.nan
    dy[holes[3].item()] = math.inf
    d = handle.matmul_grouped_grad(x, dy, offsets, order=order, fan=fan, out_dtype=out_dt)
    handle.check()
    assert torch.equal(d, clean)
    # a plan without holes is not affected, and a group of holes only has a gradient of zeros
    order[200:2500] = -1
    d = handle.matmul_grouped_grad(x, dy, offsets, order=order, fan=fan, out_dtype=out_dt)
    handle.check()
    assert (d[2] == 0).all() and torch.equal(d[[0, 3]], clean[[0, 3]])


# ------------------------------------------------------------------ chains of calls

@pytest.mark.parametrize("N", [2048, 1032])
def test_weighted_sum_right_behind_the_product(handle, N):
    """The sum is set up while the product in front still writes its rows: it reads what the
    product has written, never what was there before."""
    T, E, k, K = 512, 8, 4, 256
    order, offsets, slots = plan_of(handle, 3, T, E, k)
    w = randn(2, E, K, N, dtype=torch.bfloat16, std=K ** -0.5)
    weights = randn(4, T, k)
    y = torch.zeros(T * k, N, device=DEV, dtype=torch.bfloat16)
    out, xs = torch.empty(T, N, device=DEV, dtype=torch.bfloat16), [randn(10 + i, T, K, dtype=torch.bfloat16)
                                                                     for i in range(4)]
    want = []
    for x in xs:
        handle.matmul_grouped(x, w, offsets, y, order=order, fan=k)
        torch.cuda.synchronize()
        want.append(handle.combine_rows(y, slots, weights=weights))
        torch.cuda.synchronize()
    for turn in range(40):
        got = []
        for x in xs:
            handle.matmul_grouped(x, w, offsets, y, order=order, fan=k)
            handle.combine_rows(y, slots, out, weights=weights)
            got.append(out.clone())
        for i, (u, v) in enumerate(zip(got, want)):
            assert torch.equal(u, v), (turn, i)
    handle.check()
