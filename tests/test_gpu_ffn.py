"""Feed-forward operators on the GPU against their definition in 64 bits: MATMUL with 4-bit weights, the gated product, its backward
pass, the gated product with 4-bit weights.

Tolerances, from the arithmetic alone.  A sum of C products p_i with S = sum |p_i|: products of the 16-bit types are exact in
fp32; the tensor cores add sixteen at a time and every addition loses at most 2^-23 of a partial sum <= S, twice per step, and a run
of 64 added one by one at most 64 2^-24 S, so the sum is within ACC(C) S with ACC(C) = (C / 8 + 40) 2^-23.  fp32 products are rounded too and
added one by one: (C + 64) 2^-24 S.  A result is rounded once to its type: half a step, eps / 2 of its size (and half the smallest
subnormal step).  Where a path rounds an operand to 16 bits in between (the weights of a product with many rows, dG and dU of
the backward pass), S times eps / 2 is added.  f(G) U with errors eG, eU: |f'| <= 1.13 and |f''| <= 1.2 for every activation.
"""
import math

import numpy as np
import pytest
import torch

import reference_model_b200 as tb
from reference_model_b200 import binding

pytestmark = pytest.mark.gpu

DT = {"fp16": tb.DType.FP16, "bf16": tb.DType.BF16, "fp32": tb.DType.FP32}
TT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
HALF = {k: torch.finfo(v).eps / 2 for k, v in TT.items()}
TINY = {k: torch.finfo(v).smallest_normal * torch.finfo(v).eps for k, v in TT.items()}
ACTS = ["SILU", "GELU", "GELU_TANH", "RELU", "SIGMOID"]


@pytest.fixture(scope="module")
def ctx():
    c = tb.Context(0)
    yield c
    c.close()


def acc(n, dtype):
    return (n + 64) * 2.0 ** -24 if dtype == "fp32" else (n / 8 + 40) * 2.0 ** -23


def rand(seed, dtype, scale, *shape):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float32) * scale).to(TT[dtype])


def put(ctx, t):
    """A torch tensor on the CPU as one of the library's."""
    if t.dtype == torch.bfloat16:
        return ctx.from_numpy(t.view(torch.uint16).numpy(), tb.DType.BF16)
    return ctx.from_numpy(t.numpy())


def get(t, status=tb.Status.OK):
    st, a = t.download(check=False)
    assert st == status, st
    x = torch.from_numpy(a)
    return x.view(torch.bfloat16) if t.dtype == tb.DType.BF16 else x


def blank(ctx, dtype, shape):
    """An output full of NaNs, so that what a kernel leaves out shows."""
    return put(ctx, torch.full(shape, math.nan, dtype=TT[dtype]))


def value(act, g):
    """Activation and derivative in 64 bits."""
    if act == "RELU":
        return g.clamp(min=0), (g > 0).double()
    if act in ("SILU", "SIGMOID"):
        s, r = torch.sigmoid(g), torch.sigmoid(-g)
        return (g * s, s + g * s * r) if act == "SILU" else (s, s * r)
    if act == "GELU":
        p = torch.special.ndtr(g)
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    y = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    t = torch.tanh(y)
    return g * torch.sigmoid(2 * y), torch.sigmoid(2 * y) + 0.5 * g * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * g * g)


def close(got, ref, bound, dtype):
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape
    limit = bound + ref.abs() * (HALF[dtype] * (1 + 2.0 ** -10)) + TINY[dtype]
    off = (got - ref).abs()
    assert torch.isfinite(got).all(), "%d results are not finite" % int((~torch.isfinite(got)).sum())
    worst = (off / limit).max().item() if off.numel() else 0.0
    assert worst <= 1.0, "off by %.3g of the bound at %s" % (worst, np.unravel_index(int((off / limit).argmax()), tuple(off.shape)))


# ------------------------------------------------------------------------------------------------ 4-bit weights
class Four:
    """A random 4-bit matrix, its operands on the device and its values in 64 bits."""

    def __init__(self, ctx, seed, c, w, group, zero, pad, scale_dtype):
        r = np.random.default_rng(seed)
        groups, pitch = -(-c // group), (c + 1) // 2
        if pad:
            pitch = (pitch + 15) // 16 * 16
        data = r.integers(-128, 128, size=(w, pitch)).astype(np.int8)
        u = data.view(np.uint8)
        q = np.stack([u & 15, u >> 4], axis=2).reshape(w, -1)[:, :c].astype(np.float64).T
        q[q > 7] -= 16
        scale = rand(seed + 1, scale_dtype, 0.2 / math.sqrt(c), groups, w)
        self.zero = r.integers(-8, 8, size=(groups, w)).astype(np.int8) if zero else None
        at = np.arange(c) // group
        if zero:
            q = q - self.zero[at].astype(np.float64)
        self.dense = torch.from_numpy(q) * scale.double()[torch.from_numpy(at)]
        self.op = tb.W4(ctx.from_numpy(data), put(ctx, scale), ctx.from_numpy(self.zero) if zero else None, group)

    def free(self):
        for t in (self.op.data, self.op.scale, self.op.zero):
            if t is not None:
                t.free()


def w4_bound(a, dense, rows, c, dtype):
    s = a.abs() @ dense.abs()
    b = acc(c, dtype) * s
    # many rows: the weights are rounded to a's type
    return b + HALF[dtype] * s if rows > 16 else b


W4_CASES = [
    # n, h, c, w, group, zero, pad, dtype, out, scales
    (1, 1, 2048, 1000, 32, False, True, "fp16", "fp16", "fp16"),
    (1, 1, 4096, 4096, 128, True, True, "bf16", "bf16", "bf16"),
    (1, 1, 1, 1, 32, True, True, "bf16", "bf16", "fp32"),
    (1, 1, 31, 7, 32, True, True, "fp16", "fp16", "fp16"),
    (1, 1, 33, 129, 32, True, False, "fp16", "fp32", "fp16"),
    (1, 3, 257, 130, 64, False, True, "bf16", "bf16", "bf16"),
    (2, 2, 1000, 127, 96, True, True, "fp16", "fp16", "bf16"),
    (1, 5, 999, 255, 999, True, False, "bf16", "fp32", "bf16"),
    (1, 8, 2080, 128, 32, True, True, "bf16", "bf16", "fp32"),
    (3, 3, 1312, 640, 128, False, True, "fp16", "fp16", "fp16"),
    (1, 16, 4128, 384, 32, True, True, "fp16", "fp16", "fp16"),
    (1, 17, 512, 200, 256, True, True, "bf16", "bf16", "bf16"),
    (1, 33, 1500, 333, 128, True, False, "fp16", "fp16", "fp16"),
    (1, 64, 768, 512, 64, False, True, "bf16", "bf16", "bf16"),
    (1, 65, 768, 513, 64, True, True, "bf16", "bf16", "bf16"),
    (5, 41, 1001, 264, 512, True, False, "fp16", "fp16", "fp16"),
    (1, 300, 520, 1024, 128, False, True, "bf16", "fp32", "bf16"),
    (1, 513, 1024, 257, 32, True, True, "fp16", "fp16", "fp16"),
    (1, 1, 640, 512, 64, True, True, "fp32", "fp32", "fp32"),
    (1, 2, 1003, 77, 32, False, False, "fp32", "fp32", "fp32"),
    (1, 7, 4096, 130, 128, True, True, "fp32", "fp32", "fp16"),
    (1, 22, 260, 100, 260, True, True, "fp32", "fp32", "fp32"),
    (2, 100, 300, 200, 32, False, True, "fp32", "fp32", "fp32"),
]


@pytest.mark.parametrize("policy", [0, 1])
@pytest.mark.parametrize("case", W4_CASES, ids=lambda c: "x".join(map(str, c)))
def test_matmul_w4(ctx, case, policy):
    n, h, c, w, group, zero, pad, dtype, out, scales = case
    a, m = rand(1, dtype, 1.0, n, h, c), Four(ctx, 2, c, w, group, zero, pad, scales)
    ta, to = put(ctx, a), blank(ctx, out, (n, h, w))
    old = ctx.set_kernel_policy(policy)
    try:
        ctx.matmul_w4(ta, m.op, to)
    finally:
        ctx.set_kernel_policy(old)
    a64 = a.double()
    close(get(to), a64 @ m.dense, w4_bound(a64, m.dense, n * h, c, dtype), out)
    for t in (ta, to):
        t.free()
    m.free()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("case", [
    (1, 1, 2048, 512, 128, True, True, "bf16", "bf16"),
    (1, 4, 1030, 100, 32, False, True, "fp16", "fp16"),
    (2, 9, 511, 65, 64, True, False, "fp16", "fp32"),
    (1, 30, 1024, 192, 1024, True, True, "bf16", "bf16"),
    (1, 140, 640, 300, 128, True, True, "fp16", "fp16"),
    (1, 5, 513, 64, 32, True, True, "fp32", "fp32"),
    (1, 50, 200, 96, 64, False, True, "fp32", "fp32")], ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("policy", [0, 1])
def test_matmul_gated_w4(ctx, case, act, policy):
    n, h, c, w, group, zero, pad, dtype, out = case
    a = rand(1, dtype, 1.0, n, h, c)
    g, u = Four(ctx, 2, c, w, group, zero, pad, dtype), Four(ctx, 4, c, w, group, zero, pad, dtype)
    ta, to = put(ctx, a), blank(ctx, out, (n, h, w))
    old = ctx.set_kernel_policy(policy)
    try:
        ctx.matmul_gated_w4(ta, g.op, u.op, to, act)
    finally:
        ctx.set_kernel_policy(old)
    a64 = a.double()
    eg, eu = (w4_bound(a64, m.dense, n * h, c, dtype) for m in (g, u))
    check_gated(get(to), a64 @ g.dense, a64 @ u.dense, eg, eu, act, out)
    for t in (ta, to):
        t.free()
    g.free()
    u.free()


def check_gated(got, G, U, eg, eu, act, out):
    f, _ = value(act, G)
    # the activation itself in fp32: a few roundings of numbers no larger than its argument
    ef = 1.13 * eg + (G.abs() + 1) * 2.0 ** -21
    close(got, f * U, ef * U.abs() + f.abs() * eu + ef * eu + (f * U).abs() * 2.0 ** -23, out)


@pytest.mark.parametrize("group", (32, 96, 197))
@pytest.mark.parametrize("scales", ("fp16", "bf16"))
@pytest.mark.parametrize("dtype", ("fp16", "bf16"))
@pytest.mark.parametrize("h,w", ((70, 70), (700, 2060)))
def test_w4_values_are_rounded_once(ctx, h, w, dtype, scales, group):
    """More than 32 rows multiply the weights' values, rounded once to a's type (a whole number of at most 15 times a 16-bit scale is exact
    in fp32).  What lies behind a row's last element counts for nothing; a scale that is not finite reaches its own column alone."""
    c = 197
    a = rand(11, dtype, 1.0, 1, h, c)
    m = Four(ctx, 12, c, w, group, True, True, scales)
    ta, to = put(ctx, a), blank(ctx, "fp32", (1, h, w))
    ctx.matmul_w4(ta, m.op, to)
    assert ctx.last_kernel() == "matmul_w4_pair"
    values = m.dense.to(TT[dtype]).double()
    got, a64 = get(to), a.double()
    close(got, a64 @ values, acc(c, dtype) * (a64.abs() @ values.abs()), "fp32")
    s = get(m.op.scale)
    s[-1, 3] = math.inf
    m.op.scale.upload(s.view(torch.uint16).numpy() if scales == "bf16" else s.numpy())
    ctx.matmul_w4(ta, m.op, to)
    again = get(to)
    assert not torch.isfinite(again[..., 3]).any()
    again[..., 3] = got[..., 3]
    assert torch.equal(again, got)
    for t in (ta, to):
        t.free()
    m.free()


@pytest.mark.parametrize("scales", ("fp16", "bf16", "fp32"))
@pytest.mark.parametrize("dtype", ("fp16", "bf16"))
@pytest.mark.parametrize("h,w", ((70, 70), (700, 2060)))
def test_gated_w4_values_are_not_rounded(ctx, h, w, dtype, scales):
    """The gated product takes a value as two numbers, each off by half a step: half a step's square of the value, or half the smallest
    fp16 number (2^-25).  An fp32 scale's value is rounded to fp32 before (2^-24).  Sums have twice the terms."""
    c = 197
    a = rand(15, dtype, 1.0, 1, h, c)
    g, u = Four(ctx, 16, c, w, 96, True, True, scales), Four(ctx, 17, c, w, 96, True, True, scales)
    ta, to = put(ctx, a), blank(ctx, "fp32", (1, h, w))
    ctx.matmul_gated_w4(ta, g.op, u.op, to, "SIGMOID")
    assert ctx.last_kernel() == "gated_w4_pair"
    a64 = a.double()
    least = 2.0 ** -25 * a64.abs().sum(-1, keepdim=True) if dtype == "fp16" else 0.0
    eg, eu = ((acc(2 * c, dtype) + HALF[dtype] ** 2 + 2.0 ** -24) * (a64.abs() @ m.dense.abs()) + least for m in (g, u))
    check_gated(get(to), a64 @ g.dense, a64 @ u.dense, eg, eu, "SIGMOID", "fp32")
    for t in (ta, to):
        t.free()
    g.free()
    u.free()


@pytest.mark.parametrize("scales", ("same", "fp32"))
@pytest.mark.parametrize("h", (5, 70))
@pytest.mark.parametrize("dtype", ("fp16", "bf16"))
def test_gated_w4_infinite_scales(ctx, h, dtype, scales):
    """A group of one element under an infinite scale: the gate's sum is infinite, not a NaN; its sigmoid is 0 or 1."""
    c, w = 33, 70
    a = rand(18, dtype, 1.0, 1, h, c)
    a[a == 0] = 1
    scales = dtype if scales == "same" else scales
    g, u = Four(ctx, 19, c, w, 32, True, True, scales), Four(ctx, 20, c, w, 32, True, True, scales)
    s = get(g.op.scale)
    whole_numbers = g.dense[32] * s[1].double().sign()    # their signs
    s[1, :] = math.inf
    g.op.scale.upload(s.view(torch.uint16).numpy() if scales == "bf16" else s.numpy())
    ta, to = put(ctx, a), blank(ctx, "fp32", (1, h, w))
    ctx.matmul_gated_w4(ta, g.op, u.op, to, "SIGMOID")
    a64, last = a.double(), g.dense[32] != 0    # (zero times infinity is a NaN)
    assert int(last.sum()) > w // 2
    U, S = a64 @ u.dense, a64.abs() @ u.dense.abs()
    one = (a64[..., 32:] * whole_numbers > 0).double()
    got = get(to).double()
    off = (got - one * U).abs() <= (acc(2 * c, dtype) + HALF[dtype] ** 2 + 2.0 ** -23) * S + 2.0 ** -24 * a64.abs().sum(-1, keepdim=True)
    assert off[..., last].all() and torch.isnan(got[..., ~last]).all()
    for t in (ta, to):
        t.free()
    g.free()
    u.free()


@pytest.mark.parametrize("nb", (1, 3))
@pytest.mark.parametrize("c", (1, 63, 300, 2000))
@pytest.mark.parametrize("w", (1, 100, 129, 1002))
def test_gated_f32_one_row(ctx, w, c, nb):
    """Whole numbers, exact; a NaN in one batch's row stays there."""
    h = 1
    a, bg, bu = whole(31, "fp32", -3, 4, nb, h, c), whole(32, "fp32", -3, 4, nb, c, w), whole(33, "fp32", -3, 4, nb, c, w)
    if nb > 1:
        a[1, 0, c // 2] = math.nan
    out = blank(ctx, "fp32", (nb, h, w))
    ts  = [put(ctx, t) for t in (a, bg, bu)]
    ctx.matmul_gated(*ts, out, "RELU")
    assert ctx.last_kernel() == "gated_rows_f32"
    a, got = a.double(), get(out).double()
    if nb > 1:
        assert torch.isnan(got[1]).all()
        a[1], got[1] = 0, 0
    assert torch.equal(got, (a @ bg.double()).clamp(min=0) * (a @ bu.double()))
    for t in ts + [out]:
        t.free()


@pytest.mark.parametrize("rows", (15, 16, 21))
def test_w4_parts_of_fp32_rows(ctx, rows):
    """45 to 63 bf16 parts.  fp32 sums of exact products: as far off as 16-bit operands' (the parts' products are exact too)."""
    c, w = 1001, 150
    a = rand(13, "fp32", 1.0, 1, rows, c)
    m = Four(ctx, 14, c, w, 64, True, True, "fp32")
    ta, to = put(ctx, a), blank(ctx, "fp32", (1, rows, w))
    ctx.matmul_w4(ta, m.op, to)
    assert ctx.last_kernel() == "matmul_w4_rows"
    a64 = a.double()
    close(get(to), a64 @ m.dense, acc(3 * c, "fp16") * (a64.abs() @ m.dense.abs()), "fp32")
    for t in (ta, to):
        t.free()
    m.free()


@pytest.mark.parametrize("nb", (1, 3))
@pytest.mark.parametrize("c", (1, 37, 300, 1500))
@pytest.mark.parametrize("w", (1, 7, 203, 206, 212, 1001))
@pytest.mark.parametrize("h", (1, 9, 30))
def test_gated_rows_of_matrices_at_any_element(ctx, h, w, c, nb):
    """Matrices whose rows do not start at multiples of sixteen bytes, on whole numbers: exact.  NaNs behind the last row and in the next
    batch's rows count for nothing."""
    a, bg, bu = whole(21, "bf16", -1, 2, nb, h, c), whole(22, "bf16", -1, 2, nb, c, w), whole(23, "bf16", -1, 2, nb, c, w)
    out = blank(ctx, "fp32", (nb, h, w))
    ts = [put(ctx, a)]
    if nb > 1:
        bg[1] = bu[1] = math.nan
    ts += [put(ctx, bg), put(ctx, bu)]
    ctx.matmul_gated(*ts, out, "RELU")
    assert ctx.last_kernel() == "gated_rows_f16"
    ref, got = (a.double() @ bg.double()).clamp(min=0) * (a.double() @ bu.double()), get(out).double()
    if nb > 1:
        assert torch.isnan(got[1]).all()
        ref[1] = got[1] = 0
    assert torch.equal(got, ref)
    for t in ts + [out]:
        t.free()


def test_w4_extreme_values(ctx):
    """Lowest and highest elements, zero points at both ends, scales of both signs and zero."""
    c, w = 256, 64
    for q, z in ((-8, 7), (7, -8), (-8, -8), (7, 7)):
        data = np.full((w, c // 2), (q & 15) * 17, dtype=np.uint8)
        scale = np.tile(np.array([1.0, -1.0, 0.0, 2.0], dtype=np.float16), (c // 32, w // 4))
        zero = np.full((c // 32, w), z, dtype=np.int8)
        m = tb.W4(ctx.from_numpy(data), ctx.from_numpy(scale), ctx.from_numpy(zero), 32)
        for dtype in ("fp16", "bf16", "fp32"):
            ta, to = put(ctx, torch.ones((1, 3, c), dtype=TT[dtype])), blank(ctx, "fp32", (1, 3, w))
            ctx.matmul_w4(ta, m, to)
            ref = c * (q - z) * torch.from_numpy(scale[0]).double()
            assert torch.equal(get(to).double()[0], ref.expand(3, w))


def test_w4_zero_point_out_of_range(ctx):
    data, scale = ctx.from_numpy(np.zeros((40, 64), np.int8)), ctx.from_numpy(np.ones((4, 40), np.float16))
    for where, v in (((0, 0), 8), ((3, 39), -9), ((1, 17), 127)):
        z = np.zeros((4, 40), np.int8)
        z[where] = v
        m = tb.W4(data, scale, ctx.from_numpy(z), 32)
        for rows in (1, 20, 100):
            for dtype in ("fp16", "fp32"):
                ta, to = put(ctx, rand(1, dtype, 1.0, 1, rows, 128)), blank(ctx, dtype, (1, rows, 40))
                ctx.matmul_w4(ta, m, to)
                get(to, tb.Status.UNPREDICTABLE)
    assert ctx.sync() == tb.Status.OK


@pytest.mark.parametrize("rows", [1, 3, 12, 40, 200])
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_w4_rows_keep_their_infinities_and_nans(ctx, rows, dtype):
    """What is not finite in one row stays in that row."""
    c, w = 384, 96
    a = rand(1, dtype, 1.0, 1, rows, c)
    m = Four(ctx, 2, c, w, 32, True, True, "fp16")
    bad = {0: math.nan, rows // 2: math.inf, rows - 1: -math.inf}
    for r, v in bad.items():
        a[0, r, 5] = v
    ta, to = put(ctx, a), blank(ctx, dtype, (1, rows, w))
    ctx.matmul_w4(ta, m.op, to)
    got = get(to).double()[0]
    ref = a.double()[0] @ m.dense
    keep = [r for r in range(rows) if r not in bad]
    assert torch.isfinite(got[keep]).all()
    clean = a.double()[0][keep]
    close(got[keep], ref[keep], w4_bound(clean, m.dense, rows, c, dtype), dtype)
    for r in bad:
        assert torch.equal(torch.isnan(got[r]), torch.isnan(ref[r])) and torch.equal(got[r][~torch.isnan(ref[r])], ref[r][~torch.isnan(ref[r])])


# ------------------------------------------------------------------------------------------------ gated product
GATED_CASES = [
    # n, weights' batches, h, c, w, dtype, out
    (1, 1, 1, 1024, 512, "bf16", "bf16"),
    (1, 1, 1, 1, 1, "fp16", "fp16"),
    (1, 1, 1, 4100, 4, "fp16", "fp32"),
    (1, 1, 2, 777, 333, "bf16", "bf16"),
    (1, 1, 3, 2048, 136, "fp16", "fp16"),
    (3, 3, 4, 260, 72, "bf16", "fp32"),
    (2, 1, 2, 256, 260, "bf16", "bf16"),
    (1, 1, 5, 512, 96, "fp16", "fp16"),
    (1, 1, 127, 200, 128, "bf16", "bf16"),
    (1, 1, 128, 64, 129, "fp16", "fp16"),
    (1, 1, 257, 1000, 1416, "bf16", "bf16"),
    (4, 4, 197, 333, 261, "fp16", "fp16"),
    (4, 1, 197, 128, 264, "fp16", "fp32"),
    (1, 1, 300, 72, 2000, "bf16", "fp32"),
    (1, 1, 700, 1032, 520, "fp16", "fp16"),
    (1, 1, 33, 100, 50, "fp32", "fp32"),
    (2, 2, 150, 260, 130, "fp32", "fp32"),
    (3, 1, 1, 512, 64, "fp32", "fp32"),
]


def gated_inputs(n, nb, h, c, w, dtype):
    return (rand(1, dtype, 1.0, n, h, c), rand(2, dtype, 1 / math.sqrt(c), nb, c, w), rand(3, dtype, 1 / math.sqrt(c), nb, c, w),
            rand(4, dtype, 1.0, n, h, w))


@pytest.mark.parametrize("policy", [0, 1])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("case", GATED_CASES, ids=lambda c: "x".join(map(str, c)))
def test_matmul_gated(ctx, case, act, policy):
    n, nb, h, c, w, dtype, out = case
    a, bg, bu, _ = gated_inputs(n, nb, h, c, w, dtype)
    ts = [put(ctx, t) for t in (a, bg, bu)] + [blank(ctx, out, (n, h, w))]
    old = ctx.set_kernel_policy(policy)
    try:
        ctx.matmul_gated(ts[0], ts[1], ts[2], ts[3], act)
    finally:
        ctx.set_kernel_policy(old)
    a, bg, bu = a.double(), bg.double(), bu.double()
    eg, eu = (acc(c, dtype) * (a.abs() @ b.abs()) for b in (bg, bu))
    check_gated(get(ts[3]), a @ bg, a @ bu, eg, eu, act, out)
    for t in ts:
        t.free()


def backward_reference(a, bg, bu, d, act, dtype):
    """Gradients in 64 bits and how far fp32 sums with dG, dU rounded to the type may be off."""
    n, h, c = a.shape
    w, nb = bg.shape[2], bg.shape[0]
    G, U = a @ bg, a @ bu
    eg, eu = (acc(c, dtype) * (a.abs() @ b.abs()) for b in (bg, bu))
    f, s = value(act, G)
    dG, dU = d * U * s, d * f
    r = HALF[dtype]
    # the derivative in fp32: roundings of numbers no larger than 1 + |G|^3 / 4 (the tanh form's polynomial)
    es = 1.2 * eg + (1 + G.abs() + G.abs() ** 3 / 4) * 2.0 ** -21
    ef = 1.13 * eg + (G.abs() + 1) * 2.0 ** -21
    edG = (d * U).abs() * es + (d * s).abs() * eu + d.abs() * es * eu + TINY[dtype]
    edU = d.abs() * ef + TINY[dtype]
    edG, edU = edG + r * (dG.abs() + edG), edU + r * (dU.abs() + edU)
    tg, tu = bg.transpose(1, 2), bu.transpose(1, 2)
    at = a.transpose(1, 2)

    def shared(x):
        return x.sum(0, keepdim=True) if nb == 1 else x

    da = dG @ tg + dU @ tu
    eda = edG @ tg.abs() + edU @ tu.abs() + acc(2 * w, dtype) * ((dG.abs() + edG) @ tg.abs() + (dU.abs() + edU) @ tu.abs())
    rows = n * h if nb == 1 else h
    outs, bounds = [da], [eda]
    for x, e in ((dG, edG), (dU, edU)):
        outs.append(shared(at @ x))
        bounds.append(shared(at.abs() @ e) + acc(rows, dtype) * shared(at.abs() @ (x.abs() + e)))
    return outs, bounds


BACKWARD_CASES = [
    (1, 1, 1, 64, 40, "bf16", ("bf16", "bf16", "bf16")),
    (1, 1, 1, 1, 1, "fp16", ("fp16", "fp16", "fp16")),
    (1, 1, 37, 200, 120, "fp16", ("fp16", "fp32", "fp32")),
    (1, 1, 130, 261, 333, "bf16", ("bf16", "bf16", "bf16")),
    (1, 1, 394, 512, 1024, "fp16", ("fp16", "fp16", "fp16")),
    (2, 1, 100, 136, 264, "bf16", ("fp32", "fp32", "fp32")),
    (3, 3, 70, 128, 200, "fp16", ("fp16", "fp16", "fp16")),
    (2, 2, 77, 99, 65, "bf16", ("bf16", "fp32", "bf16")),
    (1, 1, 600, 72, 328, "bf16", ("bf16", "bf16", "bf16")),
    (1, 1, 45, 100, 60, "fp32", ("fp32", "fp32", "fp32")),
    (2, 2, 33, 130, 70, "fp32", ("fp32", "fp32", "fp32")),
    (2, 1, 50, 64, 128, "fp32", ("fp32", "fp32", "fp32")),
]


@pytest.mark.parametrize("policy", [0, 1])
@pytest.mark.parametrize("act", ["SILU", "GELU", "GELU_TANH", "SIGMOID"])
@pytest.mark.parametrize("case", BACKWARD_CASES, ids=lambda c: "x".join(map(str, c[:6])))
def test_matmul_gated_backward(ctx, case, act, policy):
    n, nb, h, c, w, dtype, outs = case
    a, bg, bu, d = gated_inputs(n, nb, h, c, w, dtype)
    ts = [put(ctx, t) for t in (a, bg, bu, d)]
    grads = [blank(ctx, o, s) for o, s in zip(outs, ((n, h, c), (nb, c, w), (nb, c, w)))]
    old = ctx.set_kernel_policy(policy)
    try:
        ctx.matmul_gated_backward(*ts, *grads, activation=act)
    finally:
        ctx.set_kernel_policy(old)
    refs, bounds = backward_reference(a.double(), bg.double(), bu.double(), d.double(), act, dtype)
    for g, r, b, o in zip(grads, refs, bounds, outs):
        close(get(g), r, b, o)
    for t in ts + grads:
        t.free()


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_backward_of_relu_on_whole_numbers(ctx, dtype):
    """Whole-number operands: every sum is exact, the slope at 0 is 0, and all results are exact."""
    r = np.random.default_rng(5)
    n, h, c, w = 1, 40, 24, 32
    a, bg, bu = (torch.from_numpy(r.integers(-2, 3, size=s).astype(np.float32)) for s in ((n, h, c), (1, c, w), (1, c, w)))
    d = torch.from_numpy(r.integers(-1, 2, size=(n, h, w)).astype(np.float32))
    G, U = a @ bg, a @ bu
    assert (G == 0).any()
    dG, dU = d * U * (G > 0), d * G.clamp(min=0)
    refs = [dG @ bg.transpose(1, 2) + dU @ bu.transpose(1, 2), a.transpose(1, 2) @ dG, a.transpose(1, 2) @ dU]
    ts = [put(ctx, t.to(TT[dtype])) for t in (a, bg, bu, d)]
    grads = [blank(ctx, "fp32", tuple(t.shape)) for t in refs]
    ctx.matmul_gated_backward(*ts, *grads, activation="RELU")
    for g, ref in zip(grads, refs):
        assert torch.equal(get(g), ref)


@pytest.mark.parametrize("act", ACTS)
def test_backward_against_differences(ctx, act):
    """The directional derivative of the fp32 forward pass by central differences."""
    n, h, c, w = 1, 6, 40, 24
    a, bg, bu, d = gated_inputs(n, 1, h, c, w, "fp32")
    ts = [put(ctx, t) for t in (a, bg, bu, d)]
    grads = [blank(ctx, "fp32", tuple(t.shape)) for t in (a, bg, bu)]
    ctx.matmul_gated_backward(*ts, *grads, activation=act)
    grads = [get(g).double() for g in grads]
    steps = [rand(10 + i, "fp32", 1.0, *t.shape) for i, t in enumerate((a, bg, bu))]
    eps = 2.0 ** -7
    sides = []
    for sign in (1, -1):
        out = blank(ctx, "fp32", (n, h, w))
        moved = [put(ctx, (t + sign * eps * s)) for t, s in zip((a, bg, bu), steps)]
        ctx.matmul_gated(moved[0], moved[1], moved[2], out, act)
        sides.append((get(out).double() * d.double()).sum())
    slope = (sides[0] - sides[1]) / (2 * eps)
    want = sum((g * s.double()).sum() for g, s in zip(grads, steps))
    # third derivatives along the step and fp32 results (2^-20 of the sum's size, over 2 eps); RELU's kink may lie in between
    size = sum((g * s.double()).abs().sum() for g, s in zip(grads, steps))
    assert abs(slope - want) <= (0.05 if act == "RELU" else 0.02) * size


@pytest.mark.parametrize("policy", (0, 1))
@pytest.mark.parametrize("dtype", ("bf16", "fp32"))
@pytest.mark.parametrize("act", ("GELU_TANH", "RELU"))
def test_backward_does_not_overflow_beside_a_zero(ctx, act, dtype, policy):
    """Finite gradients stay finite where a square or a partial product on the way to them passes the type's largest number.  Powers
    of two: every product and sum is exact."""
    p = 2.0
    up, d1 = (p ** -33, 1.0) if act == "GELU_TANH" else (p ** 60, p ** 50)
    a, bg = torch.tensor([[[p ** 33]]]), torch.tensor([[[p ** 33, -p ** 33]]])
    bu, d = torch.tensor([[[up, up]]]), torch.tensor([[[1.0, d1]]])
    # G = (2^66, -2^66): values (G, 0), slopes (1, 0)
    dg, du = p ** 33 * up, p ** 66
    want = (dg * p ** 33 + du * up,), (p ** 33 * dg, 0.0), (p ** 33 * du, 0.0)
    ops  = [put(ctx, t.to(TT[dtype])) for t in (a, bg, bu, d)]
    outs = [blank(ctx, dtype, s) for s in ((1, 1, 1), (1, 1, 2), (1, 1, 2))]
    old  = ctx.set_kernel_policy(policy)
    try:
        ctx.matmul_gated_backward(*ops, *outs, activation=act)
    finally:
        ctx.set_kernel_policy(old)
    for t, w in zip(outs, want):
        assert get(t).double().flatten().tolist() == list(w)
    for t in ops + outs:
        t.free()


def test_gradients_that_are_not_asked_for(ctx):
    a, bg, bu, d = gated_inputs(1, 1, 70, 136, 72, "bf16")
    ts = [put(ctx, t) for t in (a, bg, bu, d)]
    shapes = [tuple(t.shape) for t in (a, bg, bu)]
    whole = [blank(ctx, "bf16", s) for s in shapes]
    ctx.matmul_gated_backward(*ts, *whole, activation="GELU")
    whole = [get(t) for t in whole]
    for mask in range(1, 7):
        g = [blank(ctx, "bf16", s) if mask >> i & 1 else None for i, s in enumerate(shapes)]
        ctx.matmul_gated_backward(*ts, *g, activation="GELU")
        for t, ref in zip(g, whole):
            if t is not None:
                assert torch.equal(get(t), ref)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", [2, 150])
def test_gated_rows_keep_their_nans(ctx, rows, dtype):
    a, bg, bu, _ = gated_inputs(1, 1, rows, 264, 136, dtype)
    ts = [put(ctx, t) for t in (a, bg, bu)]
    clean, out = blank(ctx, dtype, (1, rows, 136)), blank(ctx, dtype, (1, rows, 136))
    ctx.matmul_gated(*ts, clean, "SILU")
    b = a.clone()
    b[0, rows // 2, 263] = math.nan
    ctx.matmul_gated(put(ctx, b), ts[1], ts[2], out, "SILU")
    clean, got = get(clean)[0], get(out)[0]
    assert torch.isnan(got[rows // 2]).all()
    keep = [r for r in range(rows) if r != rows // 2]
    assert torch.equal(got[keep], clean[keep])


# ------------------------------------------------------------------------------------------------ empty, refused, captured, together
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_empty_dimensions(ctx, dtype):
    def zeros(*s):
        return put(ctx, torch.zeros(s, dtype=TT[dtype]))

    # no products: sums are zero
    out = blank(ctx, dtype, (2, 3, 5))
    ctx.matmul_gated(zeros(2, 3, 0), zeros(2, 0, 5), zeros(2, 0, 5), out, "SIGMOID")
    assert torch.equal(get(out), torch.zeros((2, 3, 5), dtype=TT[dtype]))
    m = tb.W4(ctx.from_numpy(np.zeros((5, 0), np.int8)), zeros(0, 5), None, 32)
    out = blank(ctx, dtype, (2, 3, 5))
    ctx.matmul_w4(zeros(2, 3, 0), m, out)
    assert torch.equal(get(out), torch.zeros((2, 3, 5), dtype=TT[dtype]))
    # no rows: the weights' gradients are zero
    g = [blank(ctx, dtype, (1, 7, 5)) for _ in range(2)]
    ctx.matmul_gated_backward(zeros(1, 0, 7), zeros(1, 7, 5), zeros(1, 7, 5), zeros(1, 0, 5), zeros(1, 0, 7), g[0], g[1])
    for t in g:
        assert torch.equal(get(t), torch.zeros((1, 7, 5), dtype=TT[dtype]))
    # no columns: grad_a is zero
    da = blank(ctx, dtype, (1, 4, 7))
    ctx.matmul_gated_backward(zeros(1, 4, 7), zeros(1, 7, 0), zeros(1, 7, 0), zeros(1, 4, 0), da, None, None)
    assert torch.equal(get(da), torch.zeros((1, 4, 7), dtype=TT[dtype]))
    # nothing at all
    ctx.matmul_gated(zeros(1, 0, 7), zeros(1, 7, 5), zeros(1, 7, 5), zeros(1, 0, 5), "SILU")


def test_refusals(ctx):
    a, bg, bu, d = (put(ctx, t) for t in gated_inputs(1, 1, 4, 64, 32, "fp16"))
    out = blank(ctx, "fp16", (1, 4, 32))
    for args in ((a, bg, bu, out, 9), (a, bg, a, out, 0), (a, bg, bu, bg, 0)):
        with pytest.raises(tb.Tb200Error):
            ctx.matmul_gated(*args)
    m = Four(ctx, 1, 64, 32, 32, False, True, "fp16").op
    for w in (tb.W4(m.data, m.scale, None, 48), tb.W4(m.data, m.scale, None, 64), tb.W4(m.scale, m.scale, None, 32), tb.W4(m.data, m.scale, m.scale, 32)):
        with pytest.raises(tb.Tb200Error):
            ctx.matmul_w4(a, w, out)
    with pytest.raises(tb.Tb200Error):
        ctx.matmul_gated_backward(a, bg, bu, d)
    lib, null = binding.load_library(), None
    assert lib.tb200_matmul_gated(ctx.handle, a.handle, null, bu.handle, 0, out.handle) == tb.Status.ERROR
    assert lib.tb200_matmul_w4(ctx.handle, a.handle, null, out.handle) == tb.Status.ERROR
    assert lib.tb200_matmul_w4(null, a.handle, m.ref, out.handle) == tb.Status.ERROR
    assert ctx.sync() == tb.Status.OK


@pytest.mark.parametrize("rows", [1, 24, 140])
def test_captured_block(ctx, rows):
    """A decoder's block as it is served (gated product, then the projection back, 4-bit weights), eager, captured and replayed with
    other inputs; another context on another stream gives the same."""
    c, w = 512, 1408
    g, u, down = Four(ctx, 1, c, w, 128, True, True, "bf16"), Four(ctx, 2, c, w, 128, True, True, "bf16"), Four(ctx, 3, w, c, 64, True, True, "bf16")
    x = [rand(20 + i, "bf16", 1.0, 1, rows, c) for i in range(2)]
    ta, mid, out = put(ctx, x[0]), blank(ctx, "bf16", (1, rows, w)), blank(ctx, "bf16", (1, rows, c))

    def block(cx, a, m, o):
        cx.matmul_gated_w4(a, g.op, u.op, m, "SILU")
        cx.matmul_w4(m, down.op, o)

    eager = []
    for t in x:
        ta.upload(t.view(torch.uint16).numpy())
        block(ctx, ta, mid, out)
        eager.append(get(out))
        h = get(mid).double()
        close(eager[-1], h @ down.dense, w4_bound(h, down.dense, rows, w, "bf16"), "bf16")
    ctx.capture_begin()
    block(ctx, ta, mid, out)
    graph = ctx.capture_end()
    for t, ref in zip(x, eager):
        ta.upload(t.view(torch.uint16).numpy())
        out.upload(np.full((1, rows, c), 0x7FC0, np.uint16))
        ctx.graph_launch(graph)
        assert torch.equal(get(out), ref)
    ctx.graph_destroy(graph)
    ctx.sync()
    with tb.Context(0, stream=torch.cuda.Stream().cuda_stream) as other:
        a2, m2, o2 = put(other, x[0]), blank(other, "bf16", (1, rows, w)), blank(other, "bf16", (1, rows, c))
        block(other, a2, m2, o2)
        assert torch.equal(get(o2), eager[0])


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_captured_training_block(ctx, dtype):
    """Gated product, MATMUL back, and the gradients through the block: eager and replayed alike, twice over the same graph, and a
    second graph of other sizes between them (they share the context's workspace)."""
    def build(h, c, w):
        a, bg, bu, d = gated_inputs(1, 1, h, c, w, dtype)
        ts = [put(ctx, t) for t in (a, bg, bu, d)]
        down, mid, y = put(ctx, rand(9, dtype, 0.05, 1, w, c)), blank(ctx, dtype, (1, h, w)), blank(ctx, dtype, (1, h, c))
        grads = [blank(ctx, dtype, tuple(t.shape)) for t in (a, bg, bu)]

        def step():
            ctx.matmul_gated(ts[0], ts[1], ts[2], mid, "GELU_TANH")
            ctx.matmul(mid, down, y)
            ctx.matmul_gated_backward(*ts, *grads, activation="GELU_TANH")

        return step, [mid, y] + grads

    one, outs = build(200, 264, 392)
    two, others = build(90, 131, 77)
    one(), two()
    refs, other_refs = [get(t) for t in outs], [get(t) for t in others]
    graphs = []
    for step in (one, two):
        ctx.capture_begin()
        step()
        graphs.append(ctx.capture_end())
    for _ in range(2):
        for t in outs + others:
            t.upload(np.full(t.shape, 0x7E7E if dtype == "fp16" else 0x7E7E7E7E, np.uint16 if dtype == "fp16" else np.uint32))
        for g in graphs:
            ctx.graph_launch(g)
        for t, ref in zip(outs + others, refs + other_refs):
            assert torch.equal(get(t), ref)
    for g in graphs:
        ctx.graph_destroy(g)


def test_repeated_calls_give_the_same_bits(ctx):
    a, bg, bu, d = gated_inputs(1, 1, 300, 520, 712, "bf16")
    ts = [put(ctx, t) for t in (a, bg, bu, d)]
    grads = [blank(ctx, "bf16", tuple(t.shape)) for t in (a, bg, bu)]
    first = None
    for _ in range(5):
        ctx.matmul_gated_backward(*ts, *grads, activation="SILU")
        got = [get(t) for t in grads]
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(first, got))


# ------------------------------------------------------------------------------------------------ forms, limits, neighbours
def whole(seed, dtype, lo, hi, *shape):
    """Small whole numbers: every product and sum is exact, whatever the order."""
    return torch.randint(lo, hi, shape, generator=torch.Generator().manual_seed(seed)).to(TT[dtype])


def forms(ctx):
    """(name, kernel, call, outputs, exact results) of calls that reach every kernel and shape of it, with exact results."""
    made = []

    def gated(name, kernel, n, nb, h, c, w):
        a, bg, bu = whole(1, "bf16", -1, 2, n, h, c), whole(2, "bf16", -1, 2, nb, c, w), whole(3, "bf16", -1, 2, nb, c, w)
        out = blank(ctx, "fp32", (n, h, w))
        ts = [put(ctx, t) for t in (a, bg, bu)]
        a, bg, bu = a.double(), bg.double(), bu.double()
        made.append((name, kernel, lambda: ctx.matmul_gated(ts[0], ts[1], ts[2], out, "RELU"), [out], [(a @ bg).clamp(min=0) * (a @ bu)]))

    def four(name, kernel, h, c, w, gated_too):
        a = whole(4, "fp16", -1, 2, 1, h, c)
        r = np.random.default_rng(5)
        data = [r.integers(0, 256, size=(w, (c + 31) // 32 * 16)).astype(np.uint8) for _ in range(2)]
        ops, dense = [], []
        for d in data:
            q = np.stack([d & 15, d >> 4], axis=2).reshape(w, -1)[:, :c].astype(np.float64).T
            q[q > 7] -= 16
            dense.append(torch.from_numpy(q))
            ops.append(tb.W4(ctx.from_numpy(d), put(ctx, torch.ones((-(-c // 64), w), dtype=torch.float16)), None, 64))
        ta, out = put(ctx, a), blank(ctx, "fp32", (1, h, w))
        a = a.double()
        if gated_too:
            made.append((name, kernel, lambda: ctx.matmul_gated_w4(ta, ops[0], ops[1], out, "RELU"), [out],
                         [(a @ dense[0]).clamp(min=0) * (a @ dense[1])]))
        else:
            made.append((name, kernel, lambda: ctx.matmul_w4(ta, ops[0], out), [out], [a @ dense[0]]))

    def backward(name, kernel, n, nb, h, c, w):
        # one column of `a` apart, dG and dU are whole numbers below 256: exact in bf16
        a, bg, bu = whole(6, "bf16", 0, 2, n, h, c), whole(7, "bf16", -1, 2, nb, c, w), whole(8, "bf16", -1, 2, nb, c, w)
        a[:, :, 8:] = 0
        d = whole(9, "bf16", -1, 2, n, h, w)
        ts = [put(ctx, t) for t in (a, bg, bu, d)]
        grads = [blank(ctx, "fp32", tuple(t.shape)) for t in (a, bg, bu)]
        a, bg, bu, d = a.double(), bg.double(), bu.double(), d.double()
        G, U = a @ bg, a @ bu
        dG, dU = d * U * (G > 0), d * G.clamp(min=0)
        wg, wu = (a.transpose(1, 2) @ x for x in (dG, dU))
        if nb == 1:
            wg, wu = wg.sum(0, keepdim=True), wu.sum(0, keepdim=True)
        made.append((name, kernel, lambda: ctx.matmul_gated_backward(*ts, *grads, activation="RELU"), grads,
                     [dG @ bg.transpose(1, 2) + dU @ bu.transpose(1, 2), wg, wu]))

    gated("few rows, K over clusters", "gated_rows_f16", 1, 1, 3, 4000, 200)
    gated("few rows, many columns", "gated_rows_f16", 2, 2, 30, 264, 12000)
    gated("few rows, odd columns", "gated_rows_f16", 2, 2, 3, 2000, 203)
    gated("pairs", "gated_pair_f16", 1, 1, 1500, 520, 2000)
    gated("single, K over clusters", "gated_pair_f16", 1, 1, 100, 4000, 72)
    gated("single", "gated_pair_f16", 3, 3, 150, 100, 300)
    four("few rows", "matmul_w4_rows", 1, 9000, 700, False)
    four("few rows, gated", "gated_w4_rows", 20, 3000, 333, True)
    four("30 rows", "matmul_w4_rows", 30, 5000, 129, False)
    four("many rows", "matmul_w4_pair", 200, 1000, 300, False)
    four("many rows, gated", "gated_w4_pair", 90, 2000, 200, True)
    four("many rows, K over clusters", "matmul_w4_pair", 100, 4000, 300, False)
    four("many rows, pairs", "matmul_w4_pair", 600, 700, 4100, False)
    four("many rows, gated pairs", "gated_w4_pair", 700, 520, 2100, True)
    backward("small", "gated_backward_pair_f16", 2, 2, 130, 72, 200)
    backward("long K", "gated_backward_pair_f16", 1, 1, 2600, 64, 40)
    backward("large", "gated_backward_pair_f16", 1, 1, 700, 2100, 1290)
    return made


FORMS = ["few rows, K over clusters", "few rows, many columns", "few rows, odd columns", "pairs", "single, K over clusters", "single", "few rows", "few rows, gated", "30 rows",
         "many rows", "many rows, gated", "many rows, K over clusters", "many rows, pairs", "many rows, gated pairs", "small", "long K", "large"]


@pytest.fixture(scope="module")
def all_forms(ctx):
    return {f[0]: f for f in forms(ctx)}


@pytest.mark.parametrize("name", FORMS)
def test_every_form_is_exact_and_recovers_from_waits_that_give_up(ctx, all_forms, name):
    """Exact results of whole numbers; then the shortest wait limit: every call ends and reports (a short one may well finish within the
    time that a barrier waits by itself), the context stays usable, and the same call is right again."""
    _, kernel, call, outs, refs = all_forms[name]
    call()
    assert ctx.last_kernel() == kernel
    for o, r in zip(outs, refs):
        assert torch.equal(get(o).double(), r)
    ctx.set_wait_limit(1)
    try:
        for _ in range(20):
            call()
            st = ctx.sync(check=False)
            if st == tb.Status.INTERNAL:
                break
    finally:
        ctx.set_wait_limit(4000000000)
    assert st in (tb.Status.OK, tb.Status.INTERNAL)
    for _ in range(2):
        call()
        for o, r in zip(outs, refs):
            assert torch.equal(get(o).double(), r)


@pytest.mark.parametrize("name", FORMS)
def test_plain_launches_give_the_same(ctx, all_forms, name):
    """Without programmatic launches, and with them back to back: calls that follow one another closely share workspaces."""
    _, _, call, outs, refs = all_forms[name]
    for overlap in (0, 1):
        ctx.set_launch_overlap(overlap)
        for _ in range(5):
            call()
        for o, r in zip(outs, refs):
            assert torch.equal(get(o).double(), r)
    ctx.set_launch_overlap(1)


def test_forms_one_after_another(ctx, all_forms):
    """Every form behind every other without a wait between them: none reads what the one before has not written yet, and none
    starts writing into a workspace that is still read."""
    names = list(all_forms)
    for i, a in enumerate(names):
        b = names[(i * 5 + 3) % len(names)]
        for n in (a, b, a):
            all_forms[n][2]()
        for n in (a, b):
            for o, r in zip(all_forms[n][3], all_forms[n][4]):
                assert torch.equal(get(o).double(), r), (a, b)


def test_two_contexts_at_once():
    """The same forms from two contexts (two streams, two threads) at once."""
    import threading
    errors = []

    def work(shift):
        try:
            with tb.Context(0) as c:
                made = forms(c)
                for rep in range(3):
                    for i in range(len(made)):
                        made[(i + shift) % len(made)][2]()
                    for _, _, _, outs, refs in made:
                        for o, r in zip(outs, refs):
                            assert torch.equal(get(o).double(), r)
        except Exception as e:    # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in (0, 6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_more_batches_than_a_grid_has_rows(ctx):
    n, h, c, w = 70000, 1, 8, 8
    a, bg, bu = whole(1, "fp16", -2, 3, n, h, c), whole(2, "fp16", -2, 3, n, c, w), whole(3, "fp16", -2, 3, n, c, w)
    ts, out = [put(ctx, t) for t in (a, bg, bu)], blank(ctx, "fp32", (n, h, w))
    ctx.matmul_gated(*ts, out, "RELU")
    a, bg, bu = a.double(), bg.double(), bu.double()
    assert torch.equal(get(out).double(), (a @ bg).clamp(min=0) * (a @ bu))
    for t in ts + [out]:
        t.free()


def test_operands_inside_larger_tensors(ctx):
    """Contiguous cuts along the first dimension start at any multiple of sixteen bytes; what lies beside an output stays as it was."""
    c, w = 72, 40
    big_a, big_b = put(ctx, whole(1, "fp16", -2, 3, 5, 9, c)), put(ctx, whole(2, "fp16", -2, 3, 4, c, w))
    big_o = put(ctx, torch.full((7, 9, w), 5.0))
    out = big_o.slice([2, 0, 0], [2, 9, w])
    ctx.matmul_gated(big_a.slice([3, 0, 0], [2, 9, c]), big_b.slice([0, 0, 0], [2, c, w]), big_b.slice([2, 0, 0], [2, c, w]), out, "RELU")
    a, b = whole(1, "fp16", -2, 3, 5, 9, c).double()[3:], whole(2, "fp16", -2, 3, 4, c, w).double()
    got = get(big_o).double()
    assert torch.equal(got[2:4], (a @ b[:2]).clamp(min=0) * (a @ b[2:]))
    assert (got[:2] == 5).all() and (got[4:] == 5).all()
    with pytest.raises(tb.Tb200Error):    # a cut that leaves gaps
        ctx.matmul_gated(big_a.slice([0, 0, 0], [2, 8, c]), big_b.slice([0, 0, 0], [2, c, w]), big_b.slice([2, 0, 0], [2, c, w]), out, "RELU")


def test_capture_before_the_first_call():
    """A call that would have to make workspaces is refused while capturing; after it has run once it can be captured, and a workspace that
    grows under a live graph leaves the graph's alone."""
    with tb.Context(0) as c:
        x = whole(1, "fp16", -1, 2, 1, 2, 640)
        m = Four(c, 2, 640, 256, 64, True, True, "fp16")
        a, out, big = put(c, x), blank(c, "fp32", (1, 2, 256)), blank(c, "fp32", (1, 300, 256))
        c.capture_begin()
        with pytest.raises(tb.Tb200Error):
            c.matmul_w4(a, m.op, out)
        c.graph_destroy(c.capture_end())
        c.matmul_w4(a, m.op, out)
        ref = get(out)
        c.capture_begin()
        c.matmul_w4(a, m.op, out)
        graph = c.capture_end()
        c.matmul_w4(put(c, whole(3, "fp16", -1, 2, 1, 300, 640)), m.op, big)    # a larger workspace
        wide = Four(c, 4, 64, 700000, 64, False, True, "fp16")                    # more counters
        c.matmul_w4(put(c, whole(5, "fp16", -1, 2, 1, 1, 64)), wide.op, blank(c, "fp32", (1, 1, 700000)))
        for _ in range(3):
            out.upload(np.full((1, 2, 256), np.nan, np.float32))
            c.graph_launch(graph)
            assert torch.equal(get(out), ref)
        c.graph_destroy(graph)
