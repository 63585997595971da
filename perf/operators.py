"""The 8-bit operators of a Llama layer: the cases they are measured on, and their plain forms.

Four operators work together: `quantize_fp8` puts rows or 128 x 128 blocks of a matrix into e4m3
with an fp32 scale for each group of 128, `rmsnorm_fp8` adds a residual update, normalises and
quantizes in one pass, `silu_mul_fp8` does the same for the MLP's activation, and `linear_fp8`
multiplies such activations with such weights.

A case names its operator and its sizes. `run` computes the plain form with elementary torch
operations in fp32, or, where `own` is true, calls the engine's entry points
(`specb200.ops`). Quantized values come back as float8_e4m3fn tensors, their scales as fp32.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
GROUP = 128          # elements (or rows and columns) that share a scale
E4M3_MAX = 448.0
MIN_AMAX = 2.0 ** -100  # the largest magnitude of a group counts as at least this
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one verify step of a single request: k + 1 = 5 tokens through the 1.7B architecture
        {"name": "rmsnorm verify 5x2048", "op": "rmsnorm", "rows": 5, "width": 2048, "dtype": "bf16", "delta": True},
        # an odd batch of draft tokens at the 135M architecture's width: its last group has 64 elements
        {"name": "rmsnorm draft 289x576 f32", "op": "rmsnorm", "rows": 289, "width": 576, "dtype": "f32", "delta": False},
        # prompts of 4 requests of 8192 tokens
        {"name": "rmsnorm prompt 32768x2048", "op": "rmsnorm", "rows": 32768, "width": 2048, "dtype": "bf16", "delta": True},
        # the verify step's MLP activation, gate and up in the engine's 64-feature groups
        {"name": "silu_mul verify 5x8192", "op": "silu_mul", "rows": 5, "width": 8192, "dtype": "bf16", "packed": True},
        # a prompt's MLP activation, gate and up as two halves
        {"name": "silu_mul prompt 8192x8192", "op": "silu_mul", "rows": 8192, "width": 8192, "dtype": "bf16",
         "packed": False},
        # attention output of a batch of requests in front of the output projection
        {"name": "quantize rows 321x2048", "op": "quantize", "rows": 321, "width": 2048, "dtype": "bf16",
         "block_rows": 1},
        # gate/up weights of one layer when a model is packed
        {"name": "quantize weight 16384x2048", "op": "quantize", "rows": 16384, "width": 2048, "dtype": "bf16",
         "block_rows": 128},
        # plain decoding: one token through the q/k/v projection
        {"name": "linear decode 1x6144x2048", "op": "linear", "m": 1, "n": 6144, "k": 2048, "dtype": "bf16"},
        # verify of one request: gate/up
        {"name": "linear verify 5x16384x2048", "op": "linear", "m": 5, "n": 16384, "k": 2048, "dtype": "bf16"},
        # an odd batch of draft rows through the 135M architecture's q/k/v, fp32 out; the last group of K is half full
        {"name": "linear draft 33x960x576 f32", "op": "linear", "m": 33, "n": 960, "k": 576, "dtype": "f32"},
        # verify of 64 requests: the down projection
        {"name": "linear batch 320x2048x8192", "op": "linear", "m": 320, "n": 2048, "k": 8192, "dtype": "bf16"},
        # prompts: 8192 tokens through gate/up
        {"name": "linear prompt 8192x16384x2048", "op": "linear", "m": 8192, "n": 16384, "k": 2048, "dtype": "bf16"},
    ]


def _size(rng, low, high):
    """A whole number whose logarithm is spread evenly over the range."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rmsnorm", "silu_mul", "quantize", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "linear":
        while True:
            m, n, k = _size(rng, 1, 8192), _size(rng, 16, 49152), _size(rng, 16, 8192)
            if n * k <= 16384 * 8192 and m * n * k <= 8192 * 16384 * 2048 and m * n <= 8192 * 16384:
                return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype}
    while True:
        rows, width = _size(rng, 1, 32768), _size(rng, 64, 8192)
        if op == "silu_mul":
            packed = rng.random() < 0.5
            if packed:
                width = (width + 63) // 64 * 64
        if rows * width <= 8192 * 8192:
            break
    case = {"op": op, "rows": rows, "width": width, "dtype": dtype}
    if op == "rmsnorm":
        case["delta"] = rng.random() < 0.7
    elif op == "silu_mul":
        case["packed"] = packed
    else:
        case["block_rows"] = rng.choice([1, 128])
    return case


def _groups(width):
    return (width + GROUP - 1) // GROUP


def _size_of(dtype):
    return 2 if dtype == "bf16" else 4


def work(case):
    op, e = case["op"], _size_of(case["dtype"])
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        scales = 4 * _groups(k) * (m + _groups(n))
        return {"bytes": m * k + n * k + scales + m * n * e, "flops": 2 * m * n * k}
    rows, width = case["rows"], case["width"]
    cells = rows * width
    if op == "rmsnorm":
        moved = cells * e * (3 if case["delta"] else 1) + width * e
        return {"bytes": moved + cells + 4 * rows * _groups(width), "flops": 8 * cells}
    if op == "silu_mul":
        return {"bytes": 2 * cells * e + cells + 4 * rows * _groups(width), "flops": 10 * cells}
    blocks = rows if case["block_rows"] == 1 else _groups(rows)
    return {"bytes": cells * e + cells + 4 * blocks * _groups(width), "flops": 4 * cells}


# ---------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _activations(g, rows, width):
    """Hidden states: every feature has a size of its own, a few of them many times the others'."""
    return _normal(g, rows, width) * torch.exp(0.8 * _normal(g, width))


def _in_blocks(x, block_rows):
    """[rows, width] as [row blocks, block_rows, groups, 128], filled up with zeros."""
    rows, width = x.shape
    x = torch.nn.functional.pad(x, (0, -width % GROUP, 0, -rows % block_rows))
    return x.reshape(x.shape[0] // block_rows, block_rows, x.shape[1] // GROUP, GROUP)


def _quantized(y, block_rows=1):
    """(e4m3 values, fp32 scales) of fp32 rows."""
    rows, width = y.shape
    blocks = _in_blocks(y, block_rows)
    scales = blocks.abs().amax(dim=(1, 3)).clamp_min(MIN_AMAX) / E4M3_MAX
    q = blocks / scales[:, None, :, None]
    return q.reshape(-1, q.shape[2] * GROUP)[:rows, :width].to(torch.float8_e4m3fn).contiguous(), scales


def _with_pitch(q):
    """The same values in rows that start on 16-byte boundaries, as the engine's quantizers leave them."""
    rows, width = q.shape
    held = torch.zeros(rows, (width + 15) // 16 * 16, dtype=torch.uint8, device=q.device)
    held[:, :width] = q.view(torch.uint8)
    return held.view(torch.float8_e4m3fn)[:, :width]


def prepare(case, seed):
    g = _generator(seed)
    op, t = case["op"], TYPES[case["dtype"]]
    if op == "linear":
        x, xs = _quantized(_activations(g, case["m"], case["k"]))
        w, ws = _quantized(0.02 * _normal(g, case["n"], case["k"]), GROUP)
        return {"case": case, "x": _with_pitch(x), "x_scales": xs, "w": _with_pitch(w), "w_scales": ws}
    rows, width = case["rows"], case["width"]
    state = {"case": case}
    if op == "rmsnorm":
        state["x"] = _activations(g, rows, width).to(t)
        state["weight"] = (1.0 + 0.2 * _normal(g, width)).to(t)
        state["delta"] = (0.3 * _activations(g, rows, width)).to(t) if case["delta"] else None
    elif op == "silu_mul":
        state["gate_up"] = (1.5 * _normal(g, rows, 2 * width)).to(t)
    elif case["block_rows"] == 1:
        state["x"] = _activations(g, rows, width).to(t)
    else:
        state["x"] = (0.02 * _normal(g, rows, width)).to(t)
    return state


EPS = 1e-5


# ---------------------------------------------------------------- one pass
def run(state):
    return _engine(state) if own else _plain(state)


def _engine(state):
    ops = _ops()
    case = state["case"]
    op = case["op"]
    if op == "rmsnorm":
        return ops.rmsnorm_fp8(state["x"], state["weight"], EPS, delta=state["delta"])
    if op == "silu_mul":
        return ops.silu_mul_fp8(state["gate_up"], packed=case["packed"])
    if op == "quantize":
        return ops.quantize_fp8(state["x"], block_rows=case["block_rows"])
    return ops.linear_fp8(state["x"], state["x_scales"], state["w"], state["w_scales"],
                          out_f32=case["dtype"] == "f32", check=False)


def _ops():
    package = str(Path.cwd() / "speculative-decoder_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from specb200 import ops

    return ops


def _split_gate_up(gate_up, packed):
    rows, both = gate_up.shape
    if packed:  # 64 gate features, then the 64 up features beside them
        pairs = gate_up.reshape(rows, both // 128, 2, 64)
        return pairs[:, :, 0].reshape(rows, both // 2), pairs[:, :, 1].reshape(rows, both // 2)
    return gate_up[:, : both // 2], gate_up[:, both // 2:]


def _plain(state):
    case = state["case"]
    op, t = case["op"], TYPES[case["dtype"]]
    if op == "rmsnorm":
        h = state["x"]
        if case["delta"]:
            h = (h.float() + state["delta"].float()).to(t)
        f = h.float()
        y = f / torch.sqrt(f.square().mean(-1, keepdim=True) + EPS) * state["weight"].float()
        q, scales = _quantized(y)
        return (q, scales, h) if case["delta"] else (q, scales)
    if op == "silu_mul":
        gate, up = (v.float() for v in _split_gate_up(state["gate_up"], case["packed"]))
        return _quantized(gate / (1.0 + torch.exp(-gate)) * up)
    if op == "quantize":
        return _quantized(state["x"].float(), case["block_rows"])
    k, n = case["k"], case["n"]
    x = state["x"].float() * state["x_scales"].repeat_interleave(GROUP, 1)[:, :k]
    ws = state["w_scales"].repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]
    return torch.matmul(x, (state["w"].float() * ws).t()).to(t)


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """What `run` returns, unrounded: the quantized values as quotients before their rounding to e4m3."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        k, n = case["k"], case["n"]
        y = torch.zeros(case["m"], n, dtype=torch.float64, device=DEV)
        for b in range(_groups(k)):  # sum over the groups of K of (x_b w_b^T) * sx_b * sw_b
            at = slice(b * GROUP, min(k, (b + 1) * GROUP))
            xb = s["x"][:, at].double() * s["x_scales"][:, b].double()[:, None]
            row = torch.arange(n, device=DEV) // GROUP
            y += xb @ (s["w"][:, at].double() * s["w_scales"][row, b].double()[:, None]).T
        return y
    more = ()
    if op == "rmsnorm":
        h = s["x"].double()
        if case["delta"]:
            h = h + s["delta"].double()
            more = (h,)
            h = h.to(TYPES[case["dtype"]]).double()  # the norm is defined on the residual stream as it is stored
        y = h * (h.pow(2).sum(-1) / h.shape[1] + EPS).rsqrt()[:, None] * s["weight"].double()
    elif op == "silu_mul":
        gate, up = _split_gate_up(s["gate_up"].double(), case["packed"])
        y = torch.special.expit(gate) * gate * up
    else:
        y = s["x"].double()
    tall = case.get("block_rows", 1)
    rows, width = y.shape
    q = torch.empty_like(y)
    scales = torch.empty((rows + tall - 1) // tall, _groups(width), dtype=torch.float64, device=DEV)
    for b in range(_groups(width)):
        part = y[:, b * GROUP:(b + 1) * GROUP]
        top = part.abs().amax(1)
        if tall > 1:
            top = torch.nn.functional.pad(top, (0, -rows % tall)).reshape(-1, tall).amax(1)
        scales[:, b] = top.clamp(min=MIN_AMAX) / E4M3_MAX
        q[:, b * GROUP:(b + 1) * GROUP] = part / scales[:, b].repeat_interleave(tall)[:rows, None]
    return (q, scales) + more
