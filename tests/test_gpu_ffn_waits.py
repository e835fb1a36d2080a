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


# More stages of K to a block than its ring holds, so that copies are asked for in the middle of a call, and fewer, so that all are on their way
# before the first has been used.
CALLS = {
    "gated, few rows": lambda ctx: gated(ctx, "gated_rows_f16", 1, 3, 1200, 9600),
    "gated, few rows, a short ring": lambda ctx: gated(ctx, "gated_rows_f16", 1, 20, 200, 640),
    "gated, few rows at any element": lambda ctx: gated(ctx, "gated_rows_f16", 1, 3, 2500, 9601),
    "gated, few rows at any element, a short ring": lambda ctx: gated(ctx, "gated_rows_f16", 2, 9, 250, 203),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_waits_that_give_up_leave_others_alone(two, name):
    """One context under the shortest limit, another beside it under its usual one.  A short call may well finish within the time that a
    barrier waits by itself."""
    limited, other = (CALLS[name](c) for c in two)
    for x in (limited, other):
        x.run()
        assert x.ctx.last_kernel() == x.kernel
        x.check()
    limited.ctx.set_wait_limit(SHORTEST)
    try:
        for _ in range(5):
            for o in other.outs:
                o.upload(np.full(o.shape, np.nan, np.float32))
            for _ in range(4):
                limited.run()
                other.run()
            other.check()
            assert limited.ctx.sync(check=False) in (tb.Status.OK, tb.Status.INTERNAL)
    finally:
        limited.ctx.set_wait_limit(DEFAULT)
    for _ in range(2):
        limited.run()
        limited.check()
    for x in (limited, other):
        x.free()
