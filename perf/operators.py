"""Timed calls of the feed-forward operators: MATMUL with 4-bit weights, the gated product of two projections, its backward
pass, and the gated product with 4-bit weights.

`own` false: the plain forms, elementary torch operations in 32 bits, rounded once to the output's type.  `own` true: the calls
a user of the framework makes on a Context, with operands over torch memory.

Operands.  a [n, rows, C]; 16-bit and 32-bit weights [1, C, W] (shared by the rows) or [n, C, W] (a matrix for each batch);
4-bit weights: bytes [W, pitch], element c of a row in bits 4 (c mod 2) .. 4 (c mod 2) + 3 of byte c / 2, two's complement, and
scales (optionally zero points) [groups, W], group c / G for element c.
"""
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # 4-bit weights.  The classifier behind one image, its weights in groups of 32: the smallest call
        dict(name="w4_classifier", kind="w4", rows=1, c=2048, w=1000, group=32, zero=False, pad=True, dtype="fp16"),
        # one token through a square projection: a decoder's single position
        dict(name="w4_token", kind="w4", rows=1, c=8192, w=8192, group=128, zero=True, pad=True, dtype="bf16"),
        # a serving batch: a token of each of 24 sequences, groups of 64, width that is no multiple of a tile
        dict(name="w4_batch", kind="w4", rows=24, c=4096, w=10250, group=64, zero=True, pad=True, dtype="fp16"),
        # a prompt of odd length
        dict(name="w4_prompt", kind="w4", rows=777, c=4096, w=4096, group=128, zero=False, pad=True, dtype="bf16"),
        # gated product.  One token, weights in 16 bits
        dict(name="gated_token", kind="gated", n=1, rows=1, c=4096, w=16384, act="SILU", dtype="bf16"),
        # a long prompt, or the forward half of a training step
        dict(name="gated_prompt", kind="gated", n=1, rows=4096, c=4096, w=8192, act="SILU", dtype="bf16"),
        # 197 positions of each of four images through weights of their own; sizes that are no multiple of a tile
        dict(name="gated_ragged", kind="gated", n=4, rows=197, c=1000, w=1416, act="GELU", dtype="fp16"),
        # the same operator in full precision
        dict(name="gated_f32", kind="gated", n=1, rows=256, c=1024, w=4096, act="GELU_TANH", dtype="fp32"),
        # backward pass.  A small model's step
        dict(name="gated_backward_small", kind="backward", n=1, rows=394, c=1024, w=2048, act="GELU", dtype="fp16"),
        # a training step's worth of tokens
        dict(name="gated_backward", kind="backward", n=1, rows=4096, c=4096, w=8192, act="SILU", dtype="bf16"),
        # gated product with 4-bit weights.  One token
        dict(name="gated_w4_token", kind="gated_w4", rows=1, c=4096, w=16384, group=128, zero=True, pad=True, act="SILU", dtype="bf16"),
        # a serving batch with fine groups
        dict(name="gated_w4_batch", kind="gated_w4", rows=12, c=2048, w=8192, group=32, zero=False, pad=True, act="GELU_TANH", dtype="fp16"),
    ]


# ------------------------------------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, step):
    """Mostly whole steps, sometimes any size."""
    s = _log(rng, lo, hi)
    return s if rng.random() < 0.2 else max(step, (s + step // 2) // step * step)


def draw(rng):
    most = {k: max(work(c)["flops"] for c in listed() if c["kind"] == k) for k in ("w4", "gated", "backward")}
    most["gated_w4"] = most["w4"]
    while True:
        kind = rng.choice(["w4", "w4", "gated", "gated", "backward", "gated_w4", "gated_w4"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
        act = rng.choice(["SILU", "SILU", "GELU", "GELU_TANH", "RELU", "SIGMOID"])
        if kind in ("w4", "gated_w4"):
            c = dict(kind=kind, rows=rng.choice([1, 1, _log(rng, 1, 64), _log(rng, 1, 777)]), c=_size(rng, 64, 8192, 32),
                     w=_size(rng, 16, 16384 if kind == "w4" else 8192, 8))
            c.update(group=rng.choice([32, 64, 128, 128, c["c"]]), zero=rng.random() < 0.5, pad=rng.random() < 0.8, dtype=dtype)
            if c["c"] * c["w"] > 8192 * 8192:
                continue
        else:
            n = rng.choice([1, 1, 1, _log(rng, 2, 8)])
            c = dict(kind=kind, n=n, rows=rng.choice([1, _log(rng, 1, 4096 // n), _log(rng, 16, 4096 // n)]) if kind == "gated"
                     else _log(rng, 16, 4096 // n), c=_size(rng, 64, 4096, 8), w=_size(rng, 64, 8192, 8), dtype=dtype)
        if kind != "w4":
            # the step of RELU's slope turns the last bit of a sum next to zero into a whole term of a gradient
            c["act"] = "SILU" if kind == "backward" and act == "RELU" else act
        # products in fp32 cost the plain form what they cost in 16 bits, and a 32-bit kernel far more
        if work(c)["flops"] <= most[kind] / (8 if dtype == "fp32" else 1):
            return c


# ------------------------------------------------------------------------------------------------ work
def work(case):
    """Inputs read once, outputs written once; two operations per multiply-add (the backward pass evaluates both projections
    again and has two products for the gradient of a and one for each weight matrix)."""
    n, m, c, w, e = case.get("n", 1), case["rows"], case["c"], case["w"], _SIZE[case["dtype"]]
    kind = case["kind"]
    if kind in ("w4", "gated_w4"):
        mats = 2 if kind == "gated_w4" else 1
        groups = -(-c // case["group"])
        weights = w * (c / 2 + groups * (e + (1 if case["zero"] else 0)))
        return {"bytes": mats * weights + e * m * (c + w), "flops": 2.0 * mats * m * c * w}
    if kind == "gated":
        return {"bytes": e * n * (m * c + 2 * c * w + m * w), "flops": 4.0 * n * m * c * w}
    return {"bytes": e * n * (2 * m * c + 4 * c * w + m * w), "flops": 12.0 * n * m * c * w}


# ------------------------------------------------------------------------------------------------ inputs
class _State:
    pass


def _randn(gen, dtype, scale, *shape):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _weights4(gen, case):
    """Bytes, scales and zero points (or None) of a [C, W] matrix whose elements have about unit variance over sqrt(C)."""
    c, w, dt = case["c"], case["w"], _TYPES[case["dtype"]]
    groups = -(-c // case["group"])
    pitch = (c + 1) // 2
    if case["pad"]:
        pitch = (pitch + 15) // 16 * 16
    data = torch.randint(-128, 128, (w, pitch), generator=gen, device="cuda", dtype=torch.int8)
    spread = torch.rand((groups, w), generator=gen, device="cuda", dtype=torch.float32) + 0.5
    scale = (spread * (0.217 / math.sqrt(c))).to(dt)
    zero = torch.randint(-4, 5, (groups, w), generator=gen, device="cuda", dtype=torch.int8) if case["zero"] else None
    return data, scale, zero


def _inputs(case, seed):
    """The operands of one call as torch tensors, made from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, m, c, w, dt = case.get("n", 1), case["rows"], case["c"], case["w"], _TYPES[case["dtype"]]
    a = _randn(gen, dt, 1.0, n, m, c)
    if case["kind"] == "w4":
        return a, [_weights4(gen, case)], None
    if case["kind"] == "gated_w4":
        return a, [_weights4(gen, case), _weights4(gen, case)], None
    mats = [_randn(gen, dt, 1.0 / math.sqrt(c), n, c, w) for _ in range(2)]
    return a, mats, _randn(gen, dt, 1.0, n, m, w) if case["kind"] == "backward" else None


_CONTEXT = []


def _context():
    """One context per process and device, as a host keeps it."""
    if not _CONTEXT:
        import reference_model_b200 as tb
        _CONTEXT.append(tb.Context(0))
    return _CONTEXT[0]


def _wrapped(state, t):
    import reference_model_b200 as tb
    types = {torch.int8: tb.DType.INT8, torch.float32: tb.DType.FP32, torch.float16: tb.DType.FP16, torch.bfloat16: tb.DType.BF16}
    h = state.ctx.wrap(types[t.dtype], tuple(t.shape), t.data_ptr(), t)
    state.handles.append(h)
    return h


class _Own(_State):
    """Operands as the framework's tensors over torch memory, outputs, and the call."""

    def __init__(self, case, seed):
        import reference_model_b200 as tb
        ctx = _context()
        self.ctx, self.handles = ctx, []
        a, mats, dout = _inputs(case, seed)
        kind = case["kind"]
        n, m, w, dt = case.get("n", 1), case["rows"], case["w"], _TYPES[case["dtype"]]
        ta = _wrapped(self, a)
        if kind in ("w4", "gated_w4"):
            ops = [tb.W4(_wrapped(self, d), _wrapped(self, s), _wrapped(self, z) if z is not None else None, case["group"])
                   for d, s, z in mats]
        else:
            ops = [_wrapped(self, t) for t in mats]
        if kind == "backward":
            grads = [torch.empty_like(t) for t in [a] + mats]
            tg, td = [_wrapped(self, t) for t in grads], _wrapped(self, dout)
            act = case["act"]
            self.call = lambda: (ctx.matmul_gated_backward(ta, ops[0], ops[1], td, tg[0], tg[1], tg[2], act), grads)[1]
        else:
            out = torch.empty((n, m, w), dtype=dt, device="cuda")
            to = _wrapped(self, out)
            if kind == "w4":
                self.call = lambda: (ctx.matmul_w4(ta, ops[0], to), out)[1]
            elif kind == "gated":
                act = case["act"]
                self.call = lambda: (ctx.matmul_gated(ta, ops[0], ops[1], to, act), out)[1]
            else:
                act = case["act"]
                self.call = lambda: (ctx.matmul_gated_w4(ta, ops[0], ops[1], to, act), out)[1]
        torch.cuda.synchronize()

    def __del__(self):
        try:
            self.ctx.sync()
            for h in self.handles:
                h.free()
        except Exception:    # the interpreter is going down
            pass


def prepare(case, seed):
    if own:
        return _Own(case, seed)
    s = _State()
    s.case = case
    s.a, s.mats, s.dout = _inputs(case, seed)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_act(kind, g):
    if kind == "SILU":
        return g / (1.0 + torch.exp(-g))
    if kind == "GELU":
        return 0.5 * g * (1.0 + torch.erf(g * 0.7071067811865476))
    if kind == "GELU_TANH":
        return 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g)))
    if kind == "RELU":
        return torch.where(g < 0, torch.zeros_like(g), g)
    return 1.0 / (1.0 + torch.exp(-g))


def _plain_slope(kind, g):
    """Derivative of the activation."""
    if kind == "SILU":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s * (1.0 + g * (1.0 - s))
    if kind == "GELU":
        return 0.5 * (1.0 + torch.erf(g * 0.7071067811865476)) + g * (0.3989422804014327 * torch.exp(-0.5 * g * g))
    if kind == "GELU_TANH":
        t = torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g))
        return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * 0.7978845608028654 * (1.0 + 3.0 * 0.044715 * g * g)
    if kind == "RELU":
        return (g > 0).to(g.dtype)
    s = 1.0 / (1.0 + torch.exp(-g))
    return s * (1.0 - s)


def _plain_matrix(case, mat):
    """[C, W] in 32 bits from 4-bit weights."""
    data, scale, zero = mat
    low = torch.bitwise_and(data, 15)
    high = torch.bitwise_and(torch.bitwise_right_shift(data, 4), 15)
    q = torch.stack([low, high], dim=2).reshape(data.shape[0], -1)[:, :case["c"]].to(torch.float32)
    q = torch.where(q > 7, q - 16, q).t()
    group = torch.arange(case["c"], device=data.device) // case["group"]
    if zero is not None:
        q = q - zero.to(torch.float32)[group]
    return q * scale.to(torch.float32)[group]


def _plain(s):
    case, dt = s.case, _TYPES[s.case["dtype"]]
    a = s.a.to(torch.float32)
    if case["kind"] in ("w4", "gated_w4"):
        mats = [_plain_matrix(case, m) for m in s.mats]
    else:
        mats = [m.to(torch.float32) for m in s.mats]
    if case["kind"] == "w4":
        return torch.matmul(a, mats[0]).to(dt)
    g, u = torch.matmul(a, mats[0]), torch.matmul(a, mats[1])
    if case["kind"] != "backward":
        return (_plain_act(case["act"], g) * u).to(dt)
    d = s.dout.to(torch.float32)
    du = d * _plain_act(case["act"], g)
    dg = d * u * _plain_slope(case["act"], g)
    da = torch.matmul(dg, mats[0].transpose(1, 2)) + torch.matmul(du, mats[1].transpose(1, 2))
    at = a.transpose(1, 2)
    return [da.to(dt), torch.matmul(at, dg).to(dt), torch.matmul(at, du).to(dt)]


def run(state):
    return state.call() if own else _plain(state)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _value(kind, x):
    """Activation and its derivative at x, in 64 bits."""
    if kind == "RELU":
        return x.clamp(min=0), (x > 0).double()
    if kind in ("SILU", "SIGMOID"):
        p = torch.sigmoid(x)
        q = torch.sigmoid(-x)
        return (x * p, p + x * p * q) if kind == "SILU" else (p, p * q)
    if kind == "GELU":
        phi = 0.5 * torch.erfc(-x / math.sqrt(2.0))
        return x * phi, phi + x * torch.exp(-x * x / 2) / math.sqrt(2.0 * math.pi)
    k = math.sqrt(2.0 / math.pi)
    p = torch.sigmoid(2 * k * (x + 0.044715 * x ** 3))
    return x * p, p + x * p * (1 - p) * 2 * k * (1 + 0.134145 * x ** 2)


def _matrix64(case, mat):
    data, scale, zero = mat
    table = torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, -8, -7, -6, -5, -4, -3, -2, -1], dtype=torch.float64, device=data.device)
    code = data.view(torch.uint8).long()
    c, groups = case["c"], scale.shape[0]
    out = torch.empty((data.shape[0], 2 * data.shape[1]), dtype=torch.float64, device=data.device)
    out[:, 0::2], out[:, 1::2] = table[code % 16], table[code // 16]
    out = out[:, :c]
    for k in range(groups):
        part = out[:, k * case["group"]:(k + 1) * case["group"]]
        if zero is not None:
            part -= zero[k].double()[:, None]
        part *= scale[k].double()[:, None]
    return out.t()


def exact(case, seed):
    a, mats, dout = _inputs(case, seed)
    a = a.double()
    if case["kind"] in ("w4", "gated_w4"):
        mats = [_matrix64(case, m)[None] for m in mats]
    else:
        mats = [m.double() for m in mats]
    first = torch.einsum("nmc,ncw->nmw", a, mats[0].expand(a.shape[0], -1, -1))
    if case["kind"] == "w4":
        return first
    second = torch.einsum("nmc,ncw->nmw", a, mats[1].expand(a.shape[0], -1, -1))
    value, slope = _value(case["act"], first)
    if case["kind"] != "backward":
        return value * second
    dfirst, dsecond = slope * second * dout.double(), value * dout.double()
    da = torch.einsum("nmw,ncw->nmc", dfirst, mats[0]) + torch.einsum("nmw,ncw->nmc", dsecond, mats[1])
    return [da, torch.einsum("nmc,nmw->ncw", a, dfirst), torch.einsum("nmc,nmw->ncw", a, dsecond)]
