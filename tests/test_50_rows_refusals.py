"""What the operators whose rows pick their weights refuse, and with which words.
Arguments are checked before the handle is looked at, so all of this runs without a
GPU: a call whose arguments are in order ends at the missing handle."""
import ctypes as C

import pytest

BUF = 1 << 20  # stands in for device addresses; nothing is launched


def t2(abi, rows, cols, dt=1, s0=None, s1=1, at=1, off=0, pad=0):
    return abi.Tensor2d(at * BUF, off, rows, cols, cols if s0 is None else s0, s1, dt, pad, 0, 0)


def call(pkg, name, *args):
    lib = pkg.abi.load()
    st = getattr(lib, name)(None, *[C.byref(a) if isinstance(a, C.Structure) else a for a in args], None)
    return st, lib.kapyb_last_error_string(None).decode()


def refuse(pkg, words, name, *args, status=None):
    st, msg = call(pkg, name, *args)
    assert st == (pkg.abi.INVALID_ARG if status is None else status), (st, msg)
    assert words in msg, msg


def P(at):
    return at * BUF


def routing(abi, **kw):
    r = dict(score=0, top_k=4, n_groups=1, top_groups=1, group_best=1, renormalize=1, scale=1.0)
    r.update(kw)
    return abi.Routing(*[r[f] for f, _ in abi.Routing._fields_])


def test_struct_layout(pkg):
    assert C.sizeof(pkg.abi.Routing) == 28


def test_complete_calls_end_at_the_missing_handle(pkg):
    a = pkg.abi
    x, out = t2(a, 8, 16), t2(a, 8, 16, at=2)
    w = t2(a, 16, 16, at=3)
    up, down = t2(a, 4, 16, at=4), t2(a, 16, 4, at=5)
    ok = "NULL handle"
    refuse(pkg, ok, "kapyb_route", x, None, routing(a), P(3), P(4))
    refuse(pkg, ok, "kapyb_route_backward", x, routing(a), P(3), P(4), out)
    refuse(pkg, ok, "kapyb_plan_rows", P(1), 8, 4, P(2), P(3), P(4))
    refuse(pkg, ok, "kapyb_plan_rows", None, 0, 4, None, P(3), None)
    refuse(pkg, ok, "kapyb_matmul_grouped", x, w, 2, 256, P(6), None, 1, out, None, 0)
    refuse(pkg, ok, "kapyb_matmul_grouped_grad", x, out, 2, P(6), None, 1, w, 256, 1.0, 1)
    refuse(pkg, ok, "kapyb_combine_rows", x, P(3), 2, P(4), t2(a, 4, 16, at=2))
    refuse(pkg, ok, "kapyb_combine_rows_backward", x, P(3), 2, P(4), t2(a, 4, 16, at=2), t2(a, 8, 16, at=5), P(6))
    refuse(pkg, ok, "kapyb_matmul_adapters", x, w, 2, down, 64, up, 64, P(6), None, out, None, P(7), 1 << 19)
    # an empty result needs a handle too
    refuse(pkg, ok, "kapyb_matmul_grouped", t2(a, 0, 16), w, 2, 256, P(6), None, 1, t2(a, 0, 16, at=2), None, 0)


@pytest.mark.parametrize("field, value, words", [
    ("top_k", 0, "top_k"), ("top_k", 33, "top_k"), ("top_k", 17, "top_k"), ("score", 2, "score"),
    ("n_groups", 3, "n_groups"), ("n_groups", 0, "n_groups"), ("top_groups", 2, "top_groups"),
    ("group_best", 3, "group_best"), ("group_best", 0, "group_best")])
def test_route_arguments(pkg, field, value, words):
    a = pkg.abi
    x = t2(a, 8, 16)
    refuse(pkg, words, "kapyb_route", x, None, routing(a, **{field: value}), P(3), P(4))
    refuse(pkg, words, "kapyb_route_backward", x, routing(a, **{field: value}), P(3), P(4), t2(a, 8, 16, at=2))


def test_route_tensors(pkg):
    a = pkg.abi
    refuse(pkg, "experts", "kapyb_route", t2(a, 8, 1025), None, routing(a), P(3), P(4), status=a.UNSUPPORTED)
    refuse(pkg, "element type", "kapyb_route", t2(a, 8, 16, dt=a.F8E4M3), None, routing(a), P(3), P(4))
    refuse(pkg, "overlaps", "kapyb_route", t2(a, 8, 16), None, routing(a), P(3), P(3) + 16)
    refuse(pkg, "overlaps", "kapyb_route", t2(a, 8, 16), None, routing(a), P(1) + 32, P(4))
    refuse(pkg, "aligned", "kapyb_route", t2(a, 8, 16), None, routing(a), P(3) + 2, P(4))
    refuse(pkg, "NULL", "kapyb_route", t2(a, 8, 16), None, routing(a), None, P(4))
    refuse(pkg, "shape", "kapyb_route_backward", t2(a, 8, 16), routing(a), P(3), P(4), t2(a, 8, 15, at=2))
    refuse(pkg, "stride of 0", "kapyb_route_backward", t2(a, 8, 16), routing(a), P(3), P(4), t2(a, 8, 16, s0=0, at=2))
    refuse(pkg, "negative", "kapyb_route", t2(a, 8, 16, s0=-16), None, routing(a), P(3), P(4))


def test_plan_arguments(pkg):
    a = pkg.abi
    refuse(pkg, "groups", "kapyb_plan_rows", P(1), 8, 0, P(2), P(3), P(4))
    refuse(pkg, "groups", "kapyb_plan_rows", P(1), 8, 1025, P(2), P(3), P(4), status=a.UNSUPPORTED)
    refuse(pkg, "negative", "kapyb_plan_rows", P(1), -1, 4, P(2), P(3), P(4))
    refuse(pkg, "NULL", "kapyb_plan_rows", None, 8, 4, P(2), P(3), P(4))
    refuse(pkg, "NULL", "kapyb_plan_rows", P(1), 8, 4, P(2), None, P(4))
    refuse(pkg, "overlap", "kapyb_plan_rows", P(1), 8, 4, P(1) + 16, P(3), P(4))


def test_grouped_arguments(pkg):
    a = pkg.abi
    x, w, out = t2(a, 8, 16), t2(a, 16, 24, at=3), t2(a, 8, 24, at=2)
    g = lambda words, *args, **kw: refuse(pkg, words, "kapyb_matmul_grouped", *args, **kw)
    g("columns of lhs", x, t2(a, 17, 24, at=3), 2, 408, P(6), None, 1, out, None, 0)
    g("columns of out", x, t2(a, 16, 23, at=3), 2, 408, P(6), None, 1, out, None, 0)
    g("twice the columns", x, w, 2, 408, P(6), None, 1, out, None, 1)
    g("same element type", x, t2(a, 16, 24, dt=0, at=3), 2, 384, P(6), None, 1, out, None, 0)
    g("f16, bf16 or f32", x, t2(a, 16, 24, dt=3, at=3), 2, 384, P(6), None, 1, out, None, 0)
    g("groups", x, w, 0, 384, P(6), None, 1, out, None, 0)
    g("groups", x, w, 1025, 384, P(6), None, 1, out, None, 0, status=a.UNSUPPORTED)
    g("offsets", x, w, 2, 384, None, None, 1, out, None, 0)
    g("fan", x, w, 2, 384, P(6), P(7), 0, out, None, 0)
    g("as many rows", t2(a, 7, 16), w, 2, 384, P(6), None, 1, out, None, 0)
    g("zeros only", t2(a, 8, 16, pad=1), w, 2, 384, P(6), None, 1, out, None, 0, status=a.UNSUPPORTED)
    g("stride of 0", x, w, 2, 384, P(6), None, 1, t2(a, 8, 24, s0=0, at=2), None, 0)
    g("overlaps", x, w, 2, 384, P(6), None, 1, t2(a, 8, 24, at=1, off=100), None, 0)
    g("overlaps", x, w, 2, 384, P(6), None, 1, t2(a, 8, 24, at=3, off=500), None, 0)  # second group's weights
    g("negative", x, w, 2, -1, P(6), None, 1, out, None, 0)
    ep = lambda **kw: a.Epilogue(*[{**dict(alpha=1.0, bias=None, bias_dtype=2, bias_axis=1, activation=0,
                                           rounding=1), **kw}[f] for f, _ in a.Epilogue._fields_])
    g("activation", x, w, 2, 384, P(6), None, 1, out, ep(activation=9), 0)
    g("rounding", x, w, 2, 384, P(6), None, 1, out, ep(rounding=2), 0)
    g("bias_axis", x, w, 2, 384, P(6), None, 1, out, ep(bias=P(8), bias_axis=0), 0, status=a.UNSUPPORTED)
    d = lambda words, *args, **kw: refuse(pkg, words, "kapyb_matmul_grouped_grad", *args, **kw)
    gr, dw = t2(a, 8, 24, at=2), t2(a, 16, 24, at=3)
    d("row per column", x, gr, 2, P(6), None, 1, t2(a, 15, 24, at=3), 384, 1.0, 1)
    d("overlap", x, gr, 2, P(6), None, 1, dw, 383, 1.0, 1)
    d("same element type", x, t2(a, 8, 24, dt=2, at=2), 2, P(6), None, 1, dw, 384, 1.0, 1)
    d("rounding", x, gr, 2, P(6), None, 1, dw, 384, 1.0, 7)
    d("overlaps", x, gr, 2, P(6), None, 1, t2(a, 16, 24, at=2), 384, 1.0, 1)


def test_sizes_beyond_the_index_arithmetic(pkg):
    a, big = pkg.abi, (1 << 30) + 1
    no = lambda name, *args: refuse(pkg, "2^30", name, *args, status=a.UNSUPPORTED)
    no("kapyb_route", t2(a, big, 16), None, routing(a), P(3), P(4))
    no("kapyb_matmul_grouped", t2(a, 8, big), t2(a, big, 24, at=3), 1, 0, P(6), None, 1, t2(a, 8, 24, at=2), None, 0)
    no("kapyb_matmul_grouped_grad", t2(a, big, 16), t2(a, big, 24, at=2), 1, P(6), None, 1, t2(a, 16, 24, at=3), 0,
       1.0, 1)
    no("kapyb_combine_rows", t2(a, 8, big), P(3), 2, None, t2(a, 4, big, at=2))
    no("kapyb_combine_rows_backward", None, P(3), 2, None, t2(a, 4, big), t2(a, 8, big, at=2), None)
    no("kapyb_matmul_adapters", t2(a, big, 16), t2(a, 16, 24, at=3), 1, t2(a, 16, 4, at=4), 0, t2(a, 4, 24, at=5), 0,
       P(6), None, t2(a, big, 24, at=2), None, P(7), 1 << 19)


def test_combine_arguments(pkg):
    a = pkg.abi
    rows, out = t2(a, 8, 16), t2(a, 4, 16, at=2)
    c = lambda words, *args: refuse(pkg, words, "kapyb_combine_rows", *args)
    c("k must be", rows, P(3), 0, None, out)
    c("k must be", rows, P(3), 33, None, out)
    c("slots", rows, None, 2, None, out)
    c("columns", rows, P(3), 2, None, t2(a, 4, 15, at=2))
    c("overlaps", rows, P(3), 2, None, t2(a, 4, 16, at=1, off=64))
    b = lambda words, *args: refuse(pkg, words, "kapyb_combine_rows_backward", *args)
    b("needs rows", None, P(3), 2, None, out, t2(a, 8, 16, at=4), P(5))
    b("shape of rows", rows, P(3), 2, None, out, t2(a, 7, 16, at=4), P(5))
    b("overlaps", rows, P(3), 2, None, out, t2(a, 8, 16, at=2), P(5))
    b("overlaps", rows, P(3), 2, None, out, t2(a, 8, 16, at=4), P(4))


def test_adapter_arguments(pkg):
    a = pkg.abi
    x, w, out = t2(a, 8, 16), t2(a, 16, 24, at=3), t2(a, 8, 24, at=2)
    down, up = t2(a, 16, 4, at=4), t2(a, 4, 24, at=5)
    f = lambda words, *args, **kw: refuse(pkg, words, "kapyb_matmul_adapters", *args, **kw)
    tail = (None, P(7), 1 << 19)
    f("down must be", x, w, 2, t2(a, 15, 4, at=4), 64, up, 96, P(6), None, out, *tail)
    f("down must be", x, w, 2, down, 64, t2(a, 5, 24, at=5), 96, P(6), None, out, *tail)
    f("rank", x, w, 2, t2(a, 16, 129, at=4), 2064, t2(a, 129, 24, at=5), 3096, P(6), None, out, *tail,
      status=a.UNSUPPORTED)
    f("same element type", x, w, 2, t2(a, 16, 4, dt=0, at=4), 64, up, 96, P(6), None, out, *tail)
    f("adapters", x, w, 0, down, 64, up, 96, P(6), None, out, *tail)
    f("index", x, w, 2, down, 64, up, 96, None, None, out, *tail)
    f("scratch", x, w, 2, down, 64, up, 96, P(6), None, out, None, None, 0)
    f("scratch", x, w, 2, down, 64, up, 96, P(6), None, out, None, P(7), 4)
    f("scratch", x, w, 2, down, 64, up, 96, P(6), None, out, None, P(7) + 16, 1 << 19)
    f("overlaps", x, w, 2, down, 64, up, 96, P(6), None, t2(a, 8, 24, at=5, off=100), *tail)
    f("overlaps", x, w, 2, down, 64, up, 96, P(6), None, out, None, P(3), 1 << 19)
    f("rows of lhs", x, w, 2, down, 64, up, 96, P(6), None, t2(a, 7, 24, at=2), *tail)
    lib = a.load()
    assert lib.kapyb_matmul_adapters_scratch(0, 2, 4) == 0
    assert lib.kapyb_matmul_adapters_scratch(8, 2, 4) >= 8 * 4 * 4
