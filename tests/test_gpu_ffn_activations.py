"""Activations of the gated product and their derivatives, alone: G swept over the range where they are not flat, U and the output's gradient
one, against 64 bits, relatively.

Bounds.  G and U are exact.  A result is rounded once to its type (half a step, and half the smallest subnormal step); fp16 and bf16 gradients' dG and
dU once to the operands' type before, whatever type the gradient has.  The functions themselves, in fp32, in units of 2^-23: the argument of SILU's and
SIGMOID's exponential is exact, GELU's is off by two roundings (one unit of it), GELU_TANH's by seven (3.5 units); an exponential turns that
into as many units times the argument's size.  CUDA's exponential adds two units, its erfc four, the sums, products and quotients around them half a
unit each.  The hardware's power of two, for 16-bit results, adds 2 + 1.173 |x| units, and those take the Gaussian's tail by a polynomial
within 2^-16 of it.  A derivative is a sum of two terms that may cancel: its bound counts their sizes.
"""
import math

import pytest
import torch

from test_gpu_ffn import ACTS, HALF, TINY, TT, blank, close, ctx, get, put    # noqa: F401

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -23


def value(act, g):
    """Activation and derivative in 64 bits, without a difference of near numbers on either side."""
    if act == "RELU":
        return g.clamp(min=0), (g > 0).double()
    if act == "GELU":
        p = 0.5 * torch.special.erfc(-g / math.sqrt(2))
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    k = 2 * math.sqrt(2 / math.pi)
    x = k * (g + 0.044715 * g ** 3) if act == "GELU_TANH" else g
    s, r = torch.sigmoid(x), torch.sigmoid(-x)
    if act == "SIGMOID":
        return s, s * r
    return g * s, s + g * s * r * (k * (1 + 0.134145 * g * g) if act == "GELU_TANH" else 1)


def sweep(act, dtype, rows):
    """From far left to far right of where the activations bend, and each sign's neighbourhood of zero."""
    wide = torch.linspace(-80 if act in ("SILU", "SIGMOID") else -12, 30, rows - 2 * (rows // 8))
    near = torch.logspace(-4, 0, rows // 8)
    return torch.cat([wide, near, -near]).to(TT[dtype])


def operands(ctx, dtype, g, c):
    """a, gate and up whose projections are G = g and U = 1, over c elements of K."""
    a, bg, bu = torch.zeros((1, len(g), c)), torch.zeros((1, c, 1)), torch.zeros((1, c, 1))
    a[0, :, 0], a[0, :, c - 1], bg[0, 0, 0], bu[0, c - 1, 0] = g.float(), 1, 1, 1
    return [put(ctx, t.to(TT[dtype])) for t in (a, bg, bu)]


def exponent(act, g):
    """The size of the exponential's argument."""
    if act == "GELU":
        return g * g / 2
    return 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3).abs() if act == "GELU_TANH" else g.abs()


def function_error(act, g, fast):
    """Relative error of the functions in fp32."""
    if act == "RELU":
        return torch.zeros_like(g)
    units = {"SILU": 6, "SIGMOID": 6, "GELU": 8, "GELU_TANH": 8}[act] + {"SILU": 0, "SIGMOID": 0, "GELU": 2, "GELU_TANH": 4}[act] * exponent(act, g)
    if fast:
        units = units + 8 + 2 * exponent(act, g)
    return units * UNIT + (2.0 ** -16 if fast and act == "GELU" else 0.0)


def least(act, g, slope):
    """Where the exponential e is smaller than 2^-126, its steps are 2^-149, of which CUDA's function is off by two at most (its documented two units in
    the last place): relative to e there is no bound.  Values multiply e by no more than |g|, derivatives by no more than |g| k (1 + 0.134145 g^2) + 1."""
    if act in ("RELU", "GELU"):
        return 0.0
    k = 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * g * g) if act == "GELU_TANH" else 1
    return 2.0 ** -148 * (1 + g.abs() * (k if slope else 1))


def terms(act, g):
    """The sizes of a derivative's two terms together."""
    if act in ("RELU", "SIGMOID"):
        return value(act, g)[1].abs()
    f, s = value(act, g)
    p = torch.where(g == 0, torch.full_like(g, 0.5), f / g)
    return p + (s - p).abs()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("c", (2, 1032))
@pytest.mark.parametrize("rows", (32, 600))
@pytest.mark.parametrize("dtype,out", (("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "fp32"), ("fp16", "fp32"), ("fp32", "fp32")))
@pytest.mark.parametrize("policy", (0, 1))
def test_values(ctx, act, c, rows, dtype, out, policy):    # noqa: F811
    g = sweep(act, dtype, rows)
    ts, res = operands(ctx, dtype, g, c), blank(ctx, out, (1, rows, 1))
    old = ctx.set_kernel_policy(policy)
    try:
        ctx.matmul_gated(*ts, res, act)
    finally:
        ctx.set_kernel_policy(old)
    ref = value(act, g.double())[0]
    close(get(res)[0, :, 0], ref, ref.abs() * function_error(act, g.double(), out != "fp32") + least(act, g.double(), False), out)
    for t in ts + [res]:
        t.free()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("c", (2, 1032))
@pytest.mark.parametrize("dtype", ("bf16", "fp16", "fp32"))
@pytest.mark.parametrize("policy", (0, 1))
def test_slopes(ctx, act, c, dtype, policy):    # noqa: F811
    """grad_a holds dG and dU, element by element."""
    rows = 600
    g = sweep(act, dtype, rows)
    ts, d, res = operands(ctx, dtype, g, c), put(ctx, torch.ones((1, rows, 1), dtype=TT[dtype])), blank(ctx, "fp32", (1, rows, c))
    old = ctx.set_kernel_policy(policy)
    try:
        ctx.matmul_gated_backward(*ts, d, res, None, None, activation=act)
    finally:
        ctx.set_kernel_policy(old)
    got, g = get(res)[0], g.double()
    f, s = value(act, g)
    error = function_error(act, g, dtype != "fp32" and policy == 0)
    for column, ref, size, slope in ((0, s, terms(act, g), True), (c - 1, f, f.abs(), False)):
        # (fp32: the growth of the tanh form's derivative and the sum of both terms round a few times more)
        close(got[:, column], ref, size * (error + 8 * UNIT) + least(act, g, slope) + (0.0 if dtype == "fp32" else HALF[dtype] * ref.abs() + TINY[dtype]), "fp32")
    for t in ts + [d, res]:
        t.free()
