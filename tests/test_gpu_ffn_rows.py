"""4-bit weights at the border of 32 rows: up to it weights are never rounded, beyond it tb200_matmul_w4 rounds their values once to a's type.  Bounds are
those of test_gpu_ffn without the rounding of weights, which is hundreds of times wider than the sums'."""
import pytest

import reference_model_b200 as tb    # noqa: F401
from test_gpu_ffn import HALF, Four, acc, blank, check_gated, close, ctx, get, put, rand    # noqa: F401

pytestmark = pytest.mark.gpu

SIZES = [(512, 200, 256, True, True), (1500, 333, 128, True, False), (4096, 520, 64, False, True), (97, 40, 97, True, True)]


@pytest.mark.parametrize("policy", (0, 1))
@pytest.mark.parametrize("scales", ("same", "fp32"))
@pytest.mark.parametrize("dtype", ("fp16", "bf16"))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("n,h", ((1, 9), (1, 17), (2, 12), (1, 24), (1, 25), (1, 32), (8, 4)))
def test_weights_are_not_rounded_up_to_32_rows(ctx, n, h, size, dtype, scales, policy):    # noqa: F811
    c, w, group, zero, pad = size
    a, m = rand(1, dtype, 1.0, n, h, c), Four(ctx, 2, c, w, group, zero, pad, dtype if scales == "same" else scales)
    ta, to = put(ctx, a), blank(ctx, "fp32", (n, h, w))
    old = ctx.set_kernel_policy(policy)
    try:
        ctx.matmul_w4(ta, m.op, to)
    finally:
        ctx.set_kernel_policy(old)
    assert ctx.last_kernel() == ("matmul_w4_direct" if policy else "matmul_w4_rows")
    a64 = a.double()
    # (a scale's product with a group's sum and its addition: within the sums' bound, a group counting as eight terms more at least)
    close(get(to), a64 @ m.dense, acc(c + 8 * (-(-c // group)), dtype) * (a64.abs() @ m.dense.abs()), "fp32")
    for t in (ta, to):
        t.free()
    m.free()


@pytest.mark.parametrize("dtype", ("fp16", "bf16"))
@pytest.mark.parametrize("h", (32, 33))
def test_the_border(ctx, h, dtype):    # noqa: F811
    """The same rows on both sides: apart by no more than the weights' rounding."""
    c, w = 1024, 264
    a, m = rand(1, dtype, 1.0, 1, h, c), Four(ctx, 2, c, w, 128, True, True, dtype)
    g = Four(ctx, 3, c, w, 128, True, True, dtype)
    ta, to = put(ctx, a), blank(ctx, "fp32", (1, h, w))
    a64 = a.double()
    size = a64.abs() @ m.dense.abs()
    ctx.matmul_w4(ta, m.op, to)
    assert ctx.last_kernel() == ("matmul_w4_rows" if h == 32 else "matmul_w4_pair")
    close(get(to), a64 @ m.dense, (acc(c, dtype) + (HALF[dtype] if h > 32 else 0.0)) * size, "fp32")
    # the gated product takes a value as two numbers: half a step's square, and half the smallest fp16 number
    ctx.matmul_gated_w4(ta, m.op, g.op, to, "SILU")
    assert ctx.last_kernel() == ("gated_w4_rows" if h == 32 else "gated_w4_pair")
    more = (HALF[dtype] ** 2, 2.0 ** -25 * a64.abs().sum(-1, keepdim=True) if dtype == "fp16" else 0.0) if h > 32 else (0.0, 0.0)
    eg, eu = ((acc(2 * c, dtype) + more[0]) * (a64.abs() @ x.dense.abs()) + more[1] for x in (m, g))
    check_gated(get(to), a64 @ m.dense, a64 @ g.dense, eg, eu, "SILU", "fp32")
    for t in (ta, to):
        t.free()
    m.free()
    g.free()
