"""The operators of 8-bit layers as cases that can be timed and checked.

A layer whose weights and activations are 8-bit integers is a chain of four operators: a norm (with the residual's addition)
or a gated activation or a plain row of numbers is written as 8-bit integers with one float32 scale a row, and a product
multiplies such rows with such weights, whose scales are one for each output channel. Each case is one pass through one of
them. What is held in 8 bits comes back as the numbers it stands for, beside the scales.

    values[r, i] = round(y[r, i] * (127 / m_r)),  scales[r] = m_r / 127,  m_r = max_i |y[r, i]|   (ties to even; zeros: scale 0)
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
EPS = 1e-6


@functools.lru_cache(maxsize=None)
def _int8():
    from openinfer_b200.kernels import int8
    return int8


# ------------------------------------------------------------------------------------------------------------- the cases
def _norm(rows, width, residual=True, dtype="bfloat16"):
    return dict(op="norm", rows=rows, width=width, residual=residual, dtype=dtype)


def _gate(rows, width, act="silu", block=0, dtype="bfloat16"):
    return dict(op="gate", rows=rows, width=width, act=act, block=block, dtype=dtype)


def _rows(rows, width, dtype="bfloat16"):
    return dict(op="rows", rows=rows, width=width, dtype=dtype)


def _product(rows, channels, width, bias=False, dtype="bfloat16"):
    return dict(op="product", rows=rows, channels=channels, width=width, bias=bias, dtype=dtype)


def listed():
    return [dict(case, name=name) for name, case in (
        # decoding for one request: the norm in front of a sublayer, with the branch before it added; latency counts
        ("norm, one token", _norm(1, 4096)),
        # the same for a long prompt: memory bound
        ("norm, long prompt", _norm(8192, 4096)),
        # a 32-bit stream of odd width without a residual, as a final norm or a float32 model has it
        ("norm, float32, odd", _norm(333, 5001, residual=False, dtype="float32")),
        # the activation between a feed-forward's products, for eight decoded tokens and for a prompt portion
        ("gate, eight tokens", _gate(8, 12288)),
        ("gate, prompt", _gate(4096, 12288, block=64)),
        # attention's output in front of its projection, for a step of mixed requests; a weight of a checkpoint, by its output channels
        ("rows, mixed step", _rows(1000, 4096)),
        ("rows, a weight", _rows(6144, 4097, dtype="float32")),
        # one decoded token: the weights' bytes are the bound
        ("product, one token", _product(1, 6144, 4096)),
        # a step of 32 requests on the widest projection of a layer
        ("product, 32 tokens", _product(32, 24576, 4096)),
        # a prompt portion beside decoded tokens on a long sum, neither few rows nor many
        ("product, portion", _product(264, 4096, 12288)),
        # odd everything, with a bias, into float32
        ("product, odd", _product(777, 5003, 2001, bias=True, dtype="float32")),
        # a long prompt on the widest projection: the tensor cores are the bound
        ("product, long prompt", _product(8192, 24576, 4096)),
    )]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most = max(map(_seconds, listed()))
    while True:
        op = rng.choice(("norm", "gate", "rows", "product", "product"))
        dtype = "bfloat16" if rng.random() < 0.75 else "float32"
        width = log(64, 16384)
        if rng.random() < 0.7:
            width = -(-width // 128) * 128
        if op == "norm":
            case = _norm(log(1, 16384), width, rng.random() < 0.7, dtype)
        elif op == "gate":
            case = _gate(log(1, 8192), width, rng.choice(("silu", "silu", "gelu_tanh")), rng.choice((0, 64)) if width % 64 == 0 else 0, dtype)
        elif op == "rows":
            case = _rows(log(1, 16384), width, dtype)
        else:
            channels = log(64, 32768)
            if rng.random() < 0.7:
                channels = -(-channels // 128) * 128
            case = _product(log(1, 8192), channels, width, rng.random() < 0.3, dtype)
        if _seconds(case) <= most:
            return case


def _seconds(case):
    """A rough time of one pass of the plain form, to keep drawn cases below the largest listed one."""
    w = work(case)
    return w["bytes"] / 5e11 + w["flops"] / 5e13


def work(case):
    r, n = case["rows"], case["width"]
    e = DTYPES[case["dtype"]].itemsize
    if case["op"] == "product":
        c = case["channels"]
        return {"bytes": r * n + c * n + 4 * (r + c + (c if case["bias"] else 0)) + r * c * e, "flops": 2.0 * r * c * n}
    values = 2 * r * n + 4 * r       # the numbers that the 8-bit integers stand for come back in bfloat16, and the scales
    if case["op"] == "norm":
        return {"bytes": r * n * e * (3 if case["residual"] else 1) + 2 * n + values, "flops": 8.0 * r * n}
    if case["op"] == "gate":
        return {"bytes": 2 * r * n * e + values, "flops": 12.0 * r * n}
    return {"bytes": r * n * e + values, "flops": 4.0 * r * n}


# ------------------------------------------------------------------------------------------------------ prepare and run
class _State:
    pass


def _random(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _integers(rows, width, gen):
    """Rows of 8-bit integers as a quantiser leaves them (the largest of a row is 127 or close to it), and their scales."""
    room = -(-width // 16) * 16                                   # rows start on 16-byte borders
    held = torch.zeros((rows, room), dtype=torch.int8, device="cuda")[:, :width]
    held.copy_((torch.randn((rows, width), generator=gen, device="cuda") * 32).round_().clamp_(-127, 127))
    return held, torch.rand(rows, generator=gen, device="cuda") * 0.01 + 0.001


def prepare(case, seed):
    s = _State()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s.case = case
    rows, width, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]
    if case["op"] == "product":
        s.x, s.x_scales = _integers(rows, width, gen)
        s.w, s.w_scales = _integers(case["channels"], width, gen)
        s.bias = _random((case["channels"],), gen, torch.float32) if case["bias"] else None
        s.weight = None              # the framework's handle of the weight, made on the first pass as at loading time
        return s
    # a token's numbers are of about one size, with a few channels that are ten times the others
    channels = torch.where(torch.rand(width, generator=gen, device="cuda") < 0.01, 10.0, 1.0)
    if case["op"] == "gate":
        s.x = _random((rows, 2 * width), gen, dtype, 2.0)
        return s
    s.x = (_random((rows, width), gen, torch.float32) * channels).to(dtype)
    if case["op"] == "norm":
        s.weight = (1 + 0.1 * torch.randn(width, generator=gen, device="cuda")).to(torch.bfloat16)
        s.branch = _random((rows, width), gen, dtype, 0.1) if case["residual"] else None
    return s


def run(s):
    case = s.case
    if own:
        return _run_own(s, case)
    if case["op"] == "product":
        sums = s.x.float() @ s.w.float().t()
        y = sums * s.x_scales[:, None] * s.w_scales
        return (y if s.bias is None else y + s.bias).to(DTYPES[case["dtype"]])
    if case["op"] == "norm":
        if s.branch is not None:
            s.x.copy_(s.x.float() + s.branch.float())
        x = s.x.float()
        y = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS) * s.weight.float()
        values, scales = _plain_rows(y)
        return {"values": values, "scales": scales, "stream": s.x} if s.branch is not None else {"values": values, "scales": scales}
    y = s.x.float()
    if case["op"] == "gate":
        gate, up = _halves(case, y)
        t = 1.5957691216057308 * (gate + 0.044715 * gate * gate * gate) if case["act"] == "gelu_tanh" else gate
        y = gate / (1 + torch.exp(-t)) * up
    values, scales = _plain_rows(y)
    return {"values": values, "scales": scales}


def _halves(case, y):
    """Gates and ups: all gates, then all ups, or blocks of `block` gates and the ups of the same indices behind them."""
    rows, width, block = case["rows"], case["width"], case["block"] or case["width"]
    pairs = y.view(rows, width // block, 2, block)
    return pairs[:, :, 0].reshape(rows, width), pairs[:, :, 1].reshape(rows, width)


def _plain_rows(y):
    most = y.abs().amax(dim=1)
    top = torch.full_like(most, 127)      # a tensor: a quotient with a number would be a product with a rounded reciprocal
    scales = most / top
    q = torch.round(y * torch.where(most > 0, top / most, 0)[:, None])
    return (q * scales[:, None]).to(torch.bfloat16), scales


def _run_own(s, case):
    int8 = _int8()
    if case["op"] == "product":
        if s.weight is None:
            s.weight = int8.Int8Weight(s.w, s.w_scales)
        return int8.linear_int8(int8.Int8Rows(s.x, s.x_scales), s.weight, bias=s.bias, out_dtype=DTYPES[case["dtype"]])
    if case["op"] == "norm":
        held = int8.rmsnorm_int8(s.x, s.weight, EPS, delta=s.branch)
    elif case["op"] == "gate":
        held = int8.silu_mul_int8(s.x, block=case["block"] or None, act=case["act"])
    else:
        held = int8.quantize_int8(s.x)
    out = {"values": int8.dequantize_int8(held, torch.bfloat16), "scales": held.scales}
    if case["op"] == "norm" and s.branch is not None:
        out["stream"] = s.x
    return out


# ------------------------------------------------------------------------------------------------------- 64-bit results
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "product":
        y = torch.einsum("mk,nk->mn", s.x.double() * s.x_scales.double()[:, None], s.w.double() * s.w_scales.double()[:, None])
        return y if s.bias is None else y + s.bias.double()
    out = {}
    y = s.x.double()
    if case["op"] == "norm":
        if s.branch is not None:
            out["stream"] = y + s.branch.double()
            y = out["stream"].to(s.x.dtype).double()             # the norm is of the sum as it is stored
        y = y / torch.sqrt(y.pow(2).sum(dim=1, keepdim=True) / case["width"] + EPS) * s.weight.double()
    elif case["op"] == "gate":
        block = case["block"] or case["width"]
        at = torch.arange(case["width"], device="cuda")
        at = at // block * (2 * block) + at % block
        gate, up = y[:, at], y[:, at + block]
        if case["act"] == "gelu_tanh":
            y = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate.pow(3)))) * up
        else:
            y = gate * torch.sigmoid(gate) * up
    steps = y.abs().max(dim=1).values / 127
    out["values"] = torch.round(y / steps.clamp_min(1e-300)[:, None]) * steps[:, None]
    out["scales"] = steps
    return out
