"""Feed-forward operators whose waits give up: every call ends, what it had on its way has landed by then, and neither the same context's
next calls nor another context's kernels beside it are touched by it."""
import numpy as np
import pytest
import torch

import reference_model_b200 as tb
from test_gpu_ffn import blank, get, put, whole

pytestmark = pytest.mark.gpu

SHORTEST, DEFAULT = 1, 4000000000


@pytest.fixture(scope="module")
def two():
    """Two contexts, each with a stream of its own."""
    with tb.Context(0) as a, tb.Context(0) as b:
        yield a, b


class Call:
    """A call on whole numbers, its outputs and their exact values."""

    def __init__(self, ctx, kernel, run, outs, refs, held):
        self.ctx, self.kernel, self.run, self.outs, self.refs, self.held = ctx, kernel, run, outs, refs, held

    def check(self):
        for o, r in zip(self.outs, self.refs):
            assert torch.equal(get(o).double(), r)

    def free(self):
        for t in self.held + self.outs:
            t.free()


def product64(a, b):
    """On the GPU, exactly: whole numbers."""
    return torch.matmul(a.cuda().double(), b.cuda().double())


def gated(ctx, kernel, nb, h, c, w):
    a, bg, bu = whole(1, "bf16", -1, 2, nb, h, c), whole(2, "bf16", -1, 2, nb, c, w), whole(3, "bf16", -1, 2, nb, c, w)
    ts, out = [put(ctx, t) for t in (a, bg, bu)], blank(ctx, "fp32", (nb, h, w))
    ref = (product64(a, bg).clamp(min=0) * product64(a, bu)).cpu()
    return Call(ctx, kernel, lambda: ctx.matmul_gated(*ts, out, "RELU"), [out], [ref], ts)


def four(ctx, kernel, h, c, w, mats, dtype="fp16"):
    a = whole(4, dtype, -1, 2, 1, h, c)
    r = np.random.default_rng(5)
    ops, projections, held = [], [], [put(ctx, a)]
    for _ in range(mats):
        d = r.integers(0, 256, size=(w, (c + 31) // 32 * 16)).astype(np.uint8)
        q = torch.from_numpy(np.stack([d & 15, d >> 4], axis=2).reshape(w, -1)[:, :c].astype(np.float32))
        projections.append(product64(a, torch.where(q > 7, q - 16, q).t()))
        ops.append(tb.W4(ctx.from_numpy(d), put(ctx, torch.ones((-(-c // 64), w), dtype=torch.float16)), None, 64))
        held += [ops[-1].data, ops[-1].scale]
    out = blank(ctx, "fp32", (1, h, w))
    if mats == 2:
        return Call(ctx, kernel, lambda: ctx.matmul_gated_w4(held[0], *ops, out, "RELU"), [out], [(projections[0].clamp(min=0) * projections[1]).cpu()], held)
    return Call(ctx, kernel, lambda: ctx.matmul_w4(held[0], ops[0], out), [out], [projections[0].cpu()], held)


def backward(ctx, nb, h, c, w):
    # a few columns of `a`: dG and dU are whole numbers below 256, exact in bf16
    a, bg, bu, d = whole(6, "bf16", 0, 2, nb, h, c), whole(7, "bf16", -1, 2, nb, c, w), whole(8, "bf16", -1, 2, nb, c, w), whole(9, "bf16", -1, 2, nb, h, w)
    a[:, :, 8:] = 0
    ts = [put(ctx, t) for t in (a, bg, bu, d)]
    grads = [blank(ctx, "fp32", tuple(t.shape)) for t in (a, bg, bu)]
    G, U = product64(a, bg), product64(a, bu)
    dG, dU = d.cuda() * U * (G > 0), d.cuda() * G.clamp(min=0)
    refs = [product64(dG, bg.transpose(1, 2)) + product64(dU, bu.transpose(1, 2)), product64(a.transpose(1, 2), dG), product64(a.transpose(1, 2), dU)]
    return Call(ctx, "gated_backward_pair_f16", lambda: ctx.matmul_gated_backward(*ts, *grads, activation="RELU"), grads, [r.cpu() for r in refs], ts)


# More stages of K to a block than its ring holds, so that copies are asked for in the middle of a call, and fewer, so that all are on their way
# before the first has been used.
CALLS = {
    "gated, few rows": lambda ctx: gated(ctx, "gated_rows_f16", 1, 3, 1200, 9600),
    "gated, few rows, a short ring": lambda ctx: gated(ctx, "gated_rows_f16", 1, 20, 200, 640),
    "gated, few rows at any element": lambda ctx: gated(ctx, "gated_rows_f16", 1, 3, 2500, 9601),
    "gated, few rows at any element, a short ring": lambda ctx: gated(ctx, "gated_rows_f16", 2, 9, 250, 203),
    "4 bits, one row": lambda ctx: four(ctx, "matmul_w4_rows", 1, 8192, 12000, 1),
    "4 bits, one row, a stage a block": lambda ctx: four(ctx, "matmul_w4_rows", 1, 2048, 1000, 1),
    "4 bits, 30 rows": lambda ctx: four(ctx, "matmul_w4_rows", 30, 4096, 12000, 1),
    "4 bits, gated": lambda ctx: four(ctx, "gated_w4_rows", 5, 4096, 6001, 2),
    "4 bits, fp32 rows": lambda ctx: four(ctx, "matmul_w4_rows", 21, 8192, 12000, 1, "fp32"),
    "4 bits, gated, fp32 rows": lambda ctx: four(ctx, "gated_w4_rows", 21, 4096, 12001, 2, "fp32"),
    "pairs": lambda ctx: gated(ctx, "gated_pair_f16", 1, 1500, 2000, 2500),
    "pairs, one stage": lambda ctx: gated(ctx, "gated_pair_f16", 1, 3000, 100, 2500),
    "CTAs by themselves": lambda ctx: gated(ctx, "gated_pair_f16", 3, 150, 500, 300),
    "K over clusters": lambda ctx: gated(ctx, "gated_pair_f16", 1, 100, 4000, 72),
    "4 bits, pairs": lambda ctx: four(ctx, "matmul_w4_pair", 777, 4096, 4096, 1),
    "4 bits, K over clusters": lambda ctx: four(ctx, "matmul_w4_pair", 100, 4000, 300, 1),
    "4 bits, gated, pairs": lambda ctx: four(ctx, "gated_w4_pair", 700, 2000, 2100, 2),
    "4 bits, gated, CTAs by themselves": lambda ctx: four(ctx, "gated_w4_pair", 90, 2000, 200, 2),
    "gradients": lambda ctx: backward(ctx, 1, 1700, 1000, 1290),
    "gradients, small": lambda ctx: backward(ctx, 2, 130, 72, 200),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_waits_that_give_up_leave_others_alone(two, name):
    """One context under the shortest limit, another beside it under its usual one, and copies that keep the memory busy, so that waits are long.  A
    short call may well finish within the time that a barrier waits by itself (few rows against 4-bit weights mostly do)."""
    limited, other = (CALLS[name](c) for c in two)
    copies, side = torch.empty((2, 1 << 29), dtype=torch.uint8, device="cuda"), torch.cuda.Stream()
    for x in (limited, other):
        x.run()
        assert x.ctx.last_kernel() == x.kernel
        x.check()
    limited.ctx.set_wait_limit(SHORTEST)
    try:
        for _ in range(5):
            for o in other.outs:
                o.upload(np.full(o.shape, np.nan, np.float32))
            with torch.cuda.stream(side):
                for _ in range(8):
                    copies[1].copy_(copies[0])
            for _ in range(10):
                limited.run()
                other.run()
            other.check()
            assert limited.ctx.sync(check=False) in (tb.Status.OK, tb.Status.INTERNAL)
    finally:
        limited.ctx.set_wait_limit(DEFAULT)
        side.synchronize()
    for _ in range(2):
        limited.run()
        limited.check()
    for x in (limited, other):
        x.free()
