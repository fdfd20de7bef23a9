"""The int8 operators of an MLA layer step (per-row quantisation, RMS norm with an int8 output,
int8 projection) in plain form and as calls of this package, for measurement.

``own`` False: ``run`` computes the plain form with elementary torch operations in fp32.
``own`` True: ``run`` calls ``triton_mla.layer_ops``.

Formulas (one row per token, or per output channel of a weight; T is the 16- or 32-bit storage type):

* quantize:   a = max_j |x_j|,  s = max(a / 127, tiny),  q_j = clip(round(x_j / s), -127, 127)
* rms_norm:   h = T(x + r) (h = x without a residual),  y_j = h_j w_j / sqrt(mean(h^2) + eps),
              then y is quantised as above
* linear:     y[i, j] = T(xs[i] ws[j] sum_k xq[i, k] wq[j, k])

int8 rows are returned as the values they stand for, q s, beside their scales: in 16 bits (T, or
bf16 for a 32-bit T), since which of two neighbours a value next to a border goes to is not pinned
in 32 bits.
"""

import math
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
VALUES = {torch.bfloat16: torch.bfloat16, torch.float16: torch.float16, torch.float32: torch.bfloat16}
EPS = 1e-6
TINY = torch.finfo(torch.float32).tiny


def listed():
    return [
        # The attention output of 16 requests (128 heads x 128) before the output projection.
        {"name": "quantize wo input 16", "op": "quantize", "m": 16, "k": 16384, "dtype": "bf16", "pad": 0},
        # The heads of a sharded layer in fp16, an odd number of tokens and an odd width.
        {"name": "quantize ragged 77", "op": "quantize", "m": 77, "k": 2001, "dtype": "fp16", "pad": 47},
        # wq_b's weight quantised per output channel when a checkpoint is loaded (24576 = 128 x 192 rows).
        {"name": "quantize wq_b weight", "op": "quantize", "m": 24576, "k": 1536, "dtype": "bf16", "pad": 0},
        # The layer's input norm for one token.
        {"name": "norm one token", "op": "norm", "m": 1, "k": 7168, "dtype": "bf16", "residual": True, "pad": 0},
        # q_norm: the first 1536 columns of the fused [wq_a; wkv_a] output of a decode batch.
        {"name": "norm q half 64", "op": "norm", "m": 64, "k": 1536, "dtype": "fp16", "residual": False, "pad": 576},
        # An odd batch of a small fp32 layer.
        {"name": "norm fp32 333", "op": "norm", "m": 333, "k": 1003, "dtype": "fp32", "residual": True, "pad": 5},
        # The layer's input norm for a prefill chunk.
        {"name": "norm prefill 8192", "op": "norm", "m": 8192, "k": 7168, "dtype": "bf16", "residual": True, "pad": 0},
        # The fused down-projection [wq_a; wkv_a] for one token.
        {"name": "linear w_a one token", "op": "linear", "m": 1, "n": 2112, "k": 7168, "dtype": "bf16"},
        # The output projection of a decode batch.
        {"name": "linear wo 16", "op": "linear", "m": 16, "n": 7168, "k": 16384, "dtype": "bf16"},
        # An odd batch against odd sizes (rows padded to 16 bytes, as quantize_int8 lays them out).
        {"name": "linear ragged 77", "op": "linear", "m": 77, "n": 4001, "k": 2001, "dtype": "fp16"},
        # wq_b for a batch of several hundred tokens.
        {"name": "linear wq_b 500", "op": "linear", "m": 500, "n": 24576, "k": 1536, "dtype": "fp32"},
        # The output projection of a prefill chunk.
        {"name": "linear wo 8192", "op": "linear", "m": 8192, "n": 7168, "k": 16384, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    k = _log(rng, 64, 16384)
    if op == "linear":
        n = _log(rng, 64, min(24576, 7168 * 16384 // k))
        m = _log(rng, 1, 8192)
        return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype}
    m = _log(rng, 1, min(24576, 8192 * 7168 // k // (2 if dtype == "fp32" else 1)))
    pad = rng.choice([0, 0, 64, rng.randint(1, 100)])
    if op == "quantize":
        return {"op": op, "m": m, "k": k, "dtype": dtype, "pad": pad}
    return {"op": op, "m": m, "k": k, "dtype": dtype, "residual": rng.random() < 0.7, "pad": pad}


def _int8_rows(rows, k, gen):
    """int8 rows as quantisation gives them (a Gaussian row scaled to its largest value), 16-byte aligned."""
    q = torch.empty(rows, -(-k // 16) * 16, dtype=torch.int8, device="cuda")
    step = max(1, (64 << 20) // q.shape[1])
    for i in range(0, rows, step):
        part = q[i:i + step]
        part.copy_(torch.randn(part.shape, device="cuda", generator=gen).mul_(33).clamp_(-127, 127).round_())
    return q[:, :k]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, k, dtype = case["m"], case["k"], TYPES[case["dtype"]]

    def scales(rows, size):
        return torch.rand(rows, device="cuda", generator=gen).add_(0.5).mul_(size)

    if case["op"] == "linear":
        n = case["n"]
        return {"op": "linear", "dtype": dtype, "xq": _int8_rows(m, k, gen), "xs": scales(m, 0.03),
                "wq": _int8_rows(n, k, gen), "ws": scales(n, 0.0005)}
    state = {"op": case["op"], "x": torch.randn(m, k + case["pad"], device="cuda", generator=gen).to(dtype)[:, :k],
             "values": torch.empty(m, k, dtype=VALUES[dtype], device="cuda"), "r": None}
    # A few features of a residual stream are far larger than the others.
    state["x"][:, :: max(1, k // 5)] *= 8
    if case["op"] == "norm":
        state["w"] = torch.randn(k, device="cuda", generator=gen).mul_(0.2).add_(1).to(dtype)
        if case["residual"]:
            state["r"] = torch.randn(m, k, device="cuda", generator=gen).mul_(4).to(dtype)
    return state


def _plain_quantize(y, dtype):
    s = (y.abs().amax(-1, keepdim=True) / 127).clamp_min(TINY)
    q = (y / s).round().clamp(-127, 127)
    return [(q * s).to(VALUES[dtype]), s[:, 0]]


def _plain(state):
    if state["op"] == "linear":
        total = state["xq"].float() @ state["wq"].float().T
        return [(total * state["xs"][:, None] * state["ws"]).to(state["dtype"])]
    x = state["x"]
    if state["op"] == "quantize":
        return _plain_quantize(x.float(), x.dtype)
    h = x if state["r"] is None else (x.float() + state["r"].float()).to(x.dtype)
    f = h.float()
    y = f * state["w"].float() / (f.square().mean(-1, keepdim=True) + EPS).sqrt()
    return _plain_quantize(y, x.dtype) + ([] if state["r"] is None else [h])


def _layer_ops():
    if "triton-mla_b200" not in sys.path:
        sys.path.insert(0, "triton-mla_b200")
    from triton_mla import layer_ops
    return layer_ops


def _own(state):
    ops = _layer_ops()
    if state["op"] == "linear":
        return [ops.linear_int8(state["xq"], state["xs"], state["wq"], state["ws"], state["dtype"])]
    h = None
    if state["op"] == "quantize":
        q, s = ops.quantize_int8(state["x"])
    else:
        q, s, h = ops.rms_norm_int8(state["x"], state["w"], EPS, residual=state["r"])
    out = [torch.mul(q, s[:, None], out=state["values"]), s]
    return out if h is None else out + [h]


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    m, k, size = case["m"], case["k"], TYPES[case["dtype"]].itemsize
    if case["op"] == "linear":
        n = case["n"]
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * size, "flops": 2 * m * n * k}
    # x read, the int8 rows' values and the scales written; the norm's weight, and the residual's two copies.
    nbytes = m * k * (size + 2) + 4 * m
    if case["op"] == "norm":
        nbytes += k * size + (2 * m * k * size if case["residual"] else 0)
    return {"bytes": nbytes, "flops": 6 * m * k}


def exact(case, seed):
    """The definition in 64 bits.  The integers a row stands for are the nearest to y / s."""
    state = prepare(case, seed)
    if case["op"] == "linear":
        out = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
        w = state["wq"].double().mul_(state["ws"].double()[:, None])
        for i in range(0, case["m"], 1024):
            torch.mm(state["xq"][i:i + 1024].double().mul_(state["xs"][i:i + 1024].double()[:, None]), w.T,
                     out=out[i:i + 1024])
        return [out]
    rows = state["x"].double()
    sums = None
    if case["op"] == "norm":
        if state["r"] is not None:
            sums = rows + state["r"].double()
            rows = sums.to(state["x"].dtype).double()  # the norm is of the stored sum
        inv = torch.rsqrt(torch.mean(rows * rows, dim=-1) + EPS)
        rows = rows * inv[:, None] * state["w"].double()
    scale = torch.amax(torch.abs(rows), dim=-1) / 127.0
    scale = torch.maximum(scale, torch.full_like(scale, TINY))
    codes = torch.clamp(torch.round(torch.div(rows, scale[:, None])), -127.0, 127.0)
    out = [codes * scale[:, None], scale]
    return out if sums is None else out + [sums]
