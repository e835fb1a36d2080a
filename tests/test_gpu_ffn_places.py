"""Feed-forward operators on tensors that start at any multiple of sixteen bytes, which is all that a wrapped pointer has to be: every operand and result
at an odd sixteen or at a whole 32 bytes, on whole numbers, exactly; what lies before and behind a result stays as it was."""
import itertools

import numpy as np
import pytest
import torch

import reference_model_b200 as tb
from test_gpu_ffn import TT, ctx, whole    # noqa: F401

pytestmark = pytest.mark.gpu

KIND = {torch.float16: tb.DType.FP16, torch.bfloat16: tb.DType.BF16, torch.float32: tb.DType.FP32, torch.int8: tb.DType.INT8}


class Places:
    """Tensors cut out of torch memory, `odd` sixteens of bytes behind a multiple of 256."""

    def __init__(self, ctx):    # noqa: F811
        self.ctx, self.made = ctx, []

    def put(self, values, odd):
        es = values.element_size()
        room = torch.full((values.numel() + 512 // es,), 77, dtype=values.dtype, device="cuda")
        first = (-room.data_ptr() % 256 + 16 * odd) // es
        place = room[first:first + values.numel()]
        place.copy_(values.flatten())
        t = self.ctx.wrap(KIND[values.dtype], tuple(values.shape), place.data_ptr(), room)
        torch.cuda.synchronize()
        self.made.append(t)
        return t, room, first, place

    def blank(self, dtype, shape, odd):
        return self.put(torch.full(shape, float("nan"), dtype=TT[dtype]), odd)

    def check(self, out, ref):
        _, room, first, place = out
        self.ctx.sync()
        assert torch.equal(place.cpu().double(), ref.double().cpu().flatten())
        rest = torch.cat([room[:first], room[first + place.numel():]])
        assert (rest == 77).all()

    def free(self):
        for t in self.made:
            t.free()


@pytest.fixture
def places(ctx):    # noqa: F811
    p = Places(ctx)
    yield p
    ctx.sync()
    p.free()


def product64(a, b):
    return torch.matmul(a.cuda().double(), b.cuda().double())


ODDS = list(itertools.product((0, 1), repeat=2))


@pytest.mark.parametrize("gate_odd,up_odd", ODDS)
@pytest.mark.parametrize("out_odd", (0, 1))
@pytest.mark.parametrize("dtype,h,c,w", (("fp32", 600, 512, 1024), ("fp32", 1, 512, 1024), ("fp32", 90, 100, 88), ("bf16", 3, 512, 136), ("bf16", 3, 500, 131), ("bf16", 700, 512, 1024),
                                         ("fp16", 100, 2048, 72), ("fp16", 150, 99, 301)))
def test_gated(places, dtype, h, c, w, out_odd, gate_odd, up_odd):
    a, bg, bu = whole(1, dtype, -1, 2, 1, h, c), whole(2, dtype, -1, 2, 1, c, w), whole(3, dtype, -1, 2, 1, c, w)
    ref = product64(a, bg).clamp(min=0) * product64(a, bu)
    out = places.blank("fp32", (1, h, w), out_odd)
    places.ctx.matmul_gated(places.put(a, gate_odd)[0], places.put(bg, gate_odd)[0], places.put(bu, up_odd)[0], out[0], "RELU")
    places.check(out, ref)


@pytest.mark.parametrize("gate_odd,up_odd", ODDS)
@pytest.mark.parametrize("a_odd", (0, 1))
@pytest.mark.parametrize("dtype,h,c,w", (("fp32", 600, 1024, 2048), ("fp32", 90, 100, 88), ("bf16", 300, 512, 1024), ("bf16", 77, 99, 65), ("fp16", 600, 72, 328)))
def test_gradients(places, dtype, h, c, w, a_odd, gate_odd, up_odd):
    """The gradients of gate and up at places of their own: one launch writes both."""
    # a few columns of `a`: dG and dU are small whole numbers, exact in 16 bits
    a, bg, bu, d = whole(6, dtype, 0, 2, 1, h, c), whole(7, dtype, -1, 2, 1, c, w), whole(8, dtype, -1, 2, 1, c, w), whole(9, dtype, -1, 2, 1, h, w)
    a[:, :, 8:] = 0
    G, U = product64(a, bg), product64(a, bu)
    dG, dU = d.cuda() * U * (G > 0), d.cuda() * G.clamp(min=0)
    refs = [product64(dG, bg.transpose(1, 2)) + product64(dU, bu.transpose(1, 2)), product64(a.transpose(1, 2), dG), product64(a.transpose(1, 2), dU)]
    grads = [places.blank("fp32", tuple(t.shape), odd) for t, odd in zip((a, bg, bu), (a_odd, gate_odd, up_odd))]
    ops = [places.put(t, odd)[0] for t, odd in zip((a, bg, bu, d), (a_odd, up_odd, gate_odd, a_odd))]
    places.ctx.matmul_gated_backward(*ops, *[g[0] for g in grads], activation="RELU")
    for g, r in zip(grads, refs):
        places.check(g, r)


@pytest.mark.parametrize("odds", ODDS)
@pytest.mark.parametrize("mats", (1, 2))
@pytest.mark.parametrize("dtype,h,c,w", (("fp16", 1, 1024, 200), ("bf16", 20, 520, 131), ("fp16", 70, 1000, 131), ("bf16", 700, 520, 2056), ("fp32", 5, 300, 100), ("fp32", 80, 512, 264)))
def test_four_bits(places, dtype, h, c, w, mats, odds):
    a = whole(4, dtype, -1, 2, 1, h, c)
    r = np.random.default_rng(5)
    ops, projections = [], []
    for _ in range(mats):
        d = torch.from_numpy(r.integers(-128, 128, size=(w, (c + 31) // 32 * 16)).astype(np.int8))
        zero = torch.from_numpy(r.integers(-2, 3, size=(-(-c // 64), w)).astype(np.int8))
        u = d.numpy().view(np.uint8)
        q = torch.from_numpy(np.stack([u & 15, u >> 4], axis=2).reshape(w, -1)[:, :c].astype(np.float64)).t()
        q = torch.where(q > 7, q - 16, q) - zero.double()[torch.arange(c) // 64]
        projections.append(product64(a, q))
        scale = torch.ones((-(-c // 64), w), dtype=TT[dtype])
        ops.append(tb.W4(places.put(d, odds[0])[0], places.put(scale, odds[1])[0], places.put(zero, odds[0])[0], 64))
    out = places.blank("fp32", (1, h, w), odds[1])
    ta = places.put(a, odds[0])[0]
    if mats == 2:
        places.ctx.matmul_gated_w4(ta, *ops, out[0], "RELU")
        places.check(out, projections[0].clamp(min=0) * projections[1])
    else:
        places.ctx.matmul_w4(ta, ops[0], out[0])
        places.check(out, projections[0])
