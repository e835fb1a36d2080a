"""Gradients of the gated product in FP16 where dG = D U f'(G) or dU = D f(G) are beyond fp16's range between the products: they are
held under one power of two then, and gradients are as good as in its middle.

Bounds: those of test_gpu_ffn, where dG and dU are rounded to fp16 once (half a step, 2^-11), but for the smallest fp16 number: half of it is 2^-25 as they
are, and at most 2^-39 of their largest under a power of two that brings that to 2^14 .. 2^15.
"""
import math

import numpy as np
import pytest
import torch

import reference_model_b200 as tb
from test_gpu_ffn import HALF, acc, blank, close, ctx, get, put, rand, value    # noqa: F401

pytestmark = pytest.mark.gpu


def inputs(n, nb, h, c, w, up, d):
    """Operands whose U and D have about the sizes `up` and `d`."""
    return (rand(1, "fp16", 1.0, n, h, c), rand(2, "fp16", 1 / math.sqrt(c), nb, c, w), rand(3, "fp16", up / math.sqrt(c), nb, c, w), rand(4, "fp16", d, n, h, w))


def reference(a, bg, bu, d, act):
    a, bg, bu, d = (t.double() for t in (a, bg, bu, d))
    n, h, c = a.shape
    nb, w = bg.shape[0], bg.shape[2]
    G, U = a @ bg, a @ bu
    eg, eu = (acc(c, "fp16") * (a.abs() @ b.abs()) for b in (bg, bu))
    f, s = value(act, G)
    dG, dU = d * U * s, d * f
    peak = max(dG[dG.isfinite()].abs().max().item(), dU[dU.isfinite()].abs().max().item())
    floor = 2.0 ** -25 if 2.0 ** -8 <= peak < 65520 else peak * 2.0 ** -38
    # (values and derivatives as in test_gpu_ffn, the hardware's functions and the tail's polynomial beside them)
    es = 1.2 * eg + (1 + G.abs() + G.abs() ** 3 / 4) * 2.0 ** -21 + 2.0 ** -16 * s.abs()
    ef = 1.13 * eg + (G.abs() + 1) * 2.0 ** -21 + 2.0 ** -16 * f.abs()
    edG = (d * U).abs() * es + (d * s).abs() * eu + d.abs() * es * eu
    edU = d.abs() * ef
    edG, edU = edG + HALF["fp16"] * (dG.abs() + edG) + floor, edU + HALF["fp16"] * (dU.abs() + edU) + floor
    tg, tu, at = bg.transpose(1, 2), bu.transpose(1, 2), a.transpose(1, 2)

    def shared(x):
        return x.sum(0, keepdim=True) if nb == 1 else x

    outs = [dG @ tg + dU @ tu]
    bounds = [edG @ tg.abs() + edU @ tu.abs() + acc(2 * w, "fp16") * ((dG.abs() + edG) @ tg.abs() + (dU.abs() + edU) @ tu.abs())]
    rows = n * h if nb == 1 else h
    for x, e in ((dG, edG), (dU, edU)):
        outs.append(shared(at @ x))
        bounds.append(shared(at.abs() @ e) + acc(rows, "fp16") * shared(at.abs() @ (x.abs() + e)))
    return outs, bounds


SIZES = [(1, 1, 37, 200, 120), (3, 3, 70, 128, 200), (1, 1, 394, 512, 1024), (1, 1, 700, 2100, 1290), (2, 1, 300, 72, 328), (2, 2, 77, 99, 65)]
# U's size and D's: dG and dU both large, one of them, both in the middle, small, and as small as fp16's numbers allow
SCALES = [(2.0 ** 13, 2.0 ** 12), (2.0 ** 14, 1.0), (2.0 ** -12, 2.0 ** 13), (1.0, 1.0), (1.0, 2.0 ** -14), (2.0 ** -10, 2.0 ** -10), (2.0 ** -14, 2.0 ** -20)]


@pytest.mark.parametrize("up,d", SCALES)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("act", ("SILU", "GELU"))
def test_gradients_beyond_the_range_of_fp16(ctx, size, act, up, d):    # noqa: F811
    n, nb, h, c, w = size
    ops = inputs(*size, up, d)
    ts = [put(ctx, t) for t in ops]
    grads = [blank(ctx, "fp32", s) for s in ((n, h, c), (nb, c, w), (nb, c, w))]
    ctx.matmul_gated_backward(*ts, *grads, activation=act)
    assert ctx.last_kernel() == "gated_backward_pair_f16"
    refs, bounds = reference(*ops, act)
    whole_set = [get(g) for g in grads]
    for g, r, b in zip(whole_set, refs, bounds):
        close(g, r, b, "fp32")
    # those that are asked for alone, and in fp16 where they are in its range
    for i, g in enumerate(grads):
        if refs[i].abs().max() < 60000:
            half = [blank(ctx, "fp16", g.shape) if k == i else None for k in range(3)]
            ctx.matmul_gated_backward(*ts, *half, activation=act)
            close(get(half[i]), refs[i], bounds[i], "fp16")
            half[i].free()
    for t in ts + grads:
        t.free()


@pytest.mark.parametrize("peak", (65504.0, 65536.0, 2.0 ** 30, 2.0 ** -8, 2.0 ** -8 * (1 - 2.0 ** -10), 2.0 ** -20, 2.0 ** -40))
def test_powers_of_two_are_exact(ctx, peak):    # noqa: F811
    """One row and one element of K: dU = D G with G = peak / D, for RELU; grad_up = a dU exactly, whatever power dU was held under."""
    # peak = g * d with both in fp16
    m, e = math.frexp(peak)
    g, d = math.ldexp(m, e - e // 2), math.ldexp(1.0, e // 2)
    a, bg, bu = torch.ones((1, 1, 1)), torch.full((1, 1, 1), g), torch.zeros((1, 1, 1))
    ts = [put(ctx, t.half()) for t in (a, bg, bu, torch.full((1, 1, 1), d))]
    assert float(torch.tensor(g).half()) * float(torch.tensor(d).half()) == peak
    grads = [blank(ctx, "fp32", (1, 1, 1)) for _ in range(3)]
    ctx.matmul_gated_backward(*ts, *grads, activation="RELU")
    assert get(grads[1]).item() == 0.0 and get(grads[2]).item() == peak
    for t in ts + grads:
        t.free()


@pytest.mark.parametrize("size", ((1, 1, 37, 200, 120), (1, 1, 700, 2100, 1290)), ids=lambda s: "x".join(map(str, s)))
def test_infinities_and_nans_keep_to_their_rows(ctx, size):    # noqa: F811
    """What is not finite has no part in the power of two."""
    ops = list(inputs(*size, 2.0 ** -10, 2.0 ** -10))
    rows = torch.arange(size[2]) % 7 != 3
    refs, bounds = reference(ops[0], ops[1], ops[2], ops[3] * rows.half()[None, :, None], "SILU")
    ops[3][:, 3::7, 5] = math.inf
    ops[3][:, 10::14, 7] = math.nan
    ts = [put(ctx, t) for t in ops]
    grads = [blank(ctx, "fp32", tuple(t.shape)) for t in ops[:3]]
    ctx.matmul_gated_backward(*ts, *grads, activation="SILU")
    st, da = grads[0].download(check=False)
    da = torch.from_numpy(da)
    assert st == tb.Status.OK and not torch.isfinite(da[:, ~rows]).any()
    close(da[:, rows], refs[0][:, rows], bounds[0][:, rows], "fp32")
    for t in ts + grads:
        t.free()


def test_replays_look_at_their_own_values(ctx):    # noqa: F811
    """A captured call takes the power of two that the replay's gradients call for, not the one of its capture."""
    size = (1, 1, 150, 264, 392)
    ops = {s: inputs(*size, *s) for s in SCALES}
    ts = [put(ctx, t) for t in ops[SCALES[3]]]
    grads = [blank(ctx, "fp32", tuple(t.shape)) for t in ops[SCALES[3]][:3]]

    def step():
        ctx.matmul_gated_backward(*ts, *grads, activation="GELU_TANH")

    step()
    ctx.sync()
    ctx.capture_begin()
    step()
    graph = ctx.capture_end()
    for order in (SCALES, SCALES[::-1]):
        for s in order:
            for t, x in zip(ts, ops[s]):
                t.upload(x.numpy())
            for g in grads:
                g.upload(np.full(g.shape, np.nan, np.float32))
            ctx.graph_launch(graph)
            got = [get(g) for g in grads]
            step()
            for g, x in zip(grads, got):
                assert torch.equal(get(g), x)
            for x, r, b in zip(got, *reference(*ops[s], "GELU_TANH")):
                close(x, r, b, "fp32")
    ctx.graph_destroy(graph)
    for t in ts + grads:
        t.free()
