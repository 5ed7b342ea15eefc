"""The linear layers of a decoder in 8-bit integers, as cases to time and to compare.

A decoder's layer whose matrices are kept in 8 bits goes like this: the residual stream takes what the sublayer before left and is
normed, straight into 8-bit rows with a scale each ("norm"); a product of these rows with a matrix of 8-bit channels, each with a
scale, makes q, k and v, or the scores of the vocabulary ("product"), or the gated pair of the feed-forward ("gated"); what the
attention or the gated pair leaves is brought to 8 bits by itself ("quantize"), and a product adds it to the residual stream
("product" with "add"). The plain forms compute them with elementary torch operations in float32; 8-bit rows are returned as the
values that they stand for.
"""
import math

import torch

own = False             # True: the calls of this repository's kernels; False: the plain forms

DEVICE = "cuda:0"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
MOST = 127.0            # the largest magnitude of an 8-bit value
EPS = 1e-5


def _norm(rows, width, delta="bfloat16", gain="float32"):
    return {"op": "norm", "rows": rows, "width": width, "delta": delta, "gain": gain}


def _quantize(rows, width, dtype="bfloat16"):
    return {"op": "quantize", "rows": rows, "width": width, "dtype": dtype}


def _product(rows, k, n, out="bfloat16", add=False):
    return {"op": "product", "rows": rows, "k": k, "n": n, "out": out, "add": add}


def _gated(rows, k, n, out="bfloat16"):
    return {"op": "gated", "rows": rows, "k": k, "n": n, "out": out}


def listed():
    named = {
        # a decode step of eight sequences between two sublayers of an 8B model: all latency
        "norm-8x4096": _norm(8, 4096),
        # rows of an odd width, and a sublayer that leaves float32
        "norm-1001x2049": _norm(1001, 2049, delta="float32", gain="bfloat16"),
        # several long prompts in one step at the width of an 8B model
        "norm-16384x4096": _norm(16384, 4096),
        # what the gated pair of a 32B model left, 33 sequences: before the projection back
        "quantize-33x25600": _quantize(33, 25600),
        # what the gated pair of an 8B model left, two prompts of 4096
        "quantize-8192x14336": _quantize(8192, 14336),
        # one sequence: the attention's output added to the residual stream
        "add-1x4096x4096": _product(1, 4096, 4096, "float32", add=True),
        # 64 sequences: the feed-forward's way back onto the residual stream
        "add-64x14336x4096": _product(64, 14336, 4096, "float32", add=True),
        # no size of it is even
        "product-777x2049x1001": _product(777, 2049, 1001, "float32"),
        # a prompt's q, k and v of an 8B model
        "product-4096x4096x6144": _product(4096, 4096, 6144),
        # eight sequences: gate and up of an 8B model, bound by reading the weights
        "gated-8x4096x14336": _gated(8, 4096, 14336),
        # the next turn of a conversation, 333 tokens, at the sizes of a 32B model
        "gated-333x5120x25600": _gated(333, 5120, 25600),
        # a long prompt's gate and up of an 8B model
        "gated-4096x4096x14336": _gated(4096, 4096, 14336),
    }
    return [dict(case, name=name) for name, case in named.items()]


def draw(rng):
    def spread(low, high):
        return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    op = rng.choice(["norm", "quantize", "product", "product", "gated", "gated"])
    if op == "norm":
        return _norm(spread(1, 8192), spread(64, 8192), rng.choice(["bfloat16", "float32", ""]), rng.choice(["float32", "bfloat16"]))
    if op == "quantize":
        return _quantize(spread(1, 4096), spread(64, 25600), rng.choice(["bfloat16", "float32"]))
    rows, k = spread(1, 4096), spread(64, 14336)
    if rng.random() < 0.5:                      # widths as models have them: whole hundreds
        k = max(64, k // 64 * 64)
    n = spread(64, 28672)
    while 2.0 * rows * k * n > 2.0e11:
        rows = (rows + 1) // 2
    if op == "gated":
        return _gated(rows, k, max(32, n // 2), rng.choice(["bfloat16", "bfloat16", "float32"]))
    if rng.random() < 0.4:
        return _product(rows, k, n, "float32", add=True)
    return _product(rows, k, n, rng.choice(["bfloat16", "float32"]))


def work(case):
    size = {"float32": 4, "bfloat16": 2, "": 0}
    if case["op"] == "norm":
        each = 4 + 2 + size[case["delta"]] + (4 if case["delta"] else 0)        # x in, the values out, the addend, x out again
        count = case["rows"] * case["width"]
        return {"bytes": count * each + case["width"] * size[case["gain"]] + 4 * case["rows"], "flops": 8 * count}
    if case["op"] == "quantize":
        count = case["rows"] * case["width"]
        return {"bytes": count * (size[case["dtype"]] + 2) + 4 * case["rows"], "flops": 4 * count}
    rows, k, n = case["rows"], case["k"], case["n"]
    channels = 2 * n if case["op"] == "gated" else n
    out = rows * n * size[case["out"]] * (2 if case.get("add") else 1)
    return {"bytes": rows * k + channels * k + 4 * (rows + channels) + out, "flops": 2 * rows * k * channels}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------

def _random(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _rows8(rows, k, random):
    """8-bit rows as the operators here leave them, and their scales: normal values whose largest magnitude is 127."""
    x = torch.randn(rows, k, device=DEVICE, generator=random)
    x *= MOST / x.abs().amax(1, keepdim=True)
    return x.round_().to(torch.int8), torch.rand(rows, device=DEVICE, generator=random) * 0.02 + 0.01


def _inputs(case, seed):
    random = _random(seed)
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        x = torch.randn(rows, width, device=DEVICE, generator=random)
        x[:, :: max(1, width // 7)] *= 12.0                                    # a stream has a few channels that stand out
        made = {"x": x, "gain": (torch.randn(width, device=DEVICE, generator=random) * 0.1 + 1.0).to(TYPES[case["gain"]])}
        made["delta"] = (torch.randn(rows, width, device=DEVICE, generator=random) * 0.3).to(TYPES[case["delta"]]) if case["delta"] else None
        return made
    if case["op"] == "quantize":
        x = torch.randn(case["rows"], case["width"], device=DEVICE, generator=random)
        x *= torch.rand(case["rows"], 1, device=DEVICE, generator=random) * 4.0
        return {"x": x.to(TYPES[case["dtype"]])}
    channels = 2 * case["n"] if case["op"] == "gated" else case["n"]
    a, a_scales = _rows8(case["rows"], case["k"], random)
    w, w_scales = _rows8(channels, case["k"], random)
    made = {"a": a, "a_scales": a_scales, "w": w, "w_scales": w_scales * (1.0 / math.sqrt(case["k"]))}
    if case.get("add"):
        made["x"] = torch.randn(case["rows"], case["n"], device=DEVICE, generator=random) * 4.0
    return made


def prepare(case, seed):
    """The inputs; with the kernels also what their user keeps: room for 8-bit rows and results, rows that an operator before left in 8 bits, packed weights."""
    state = dict(_inputs(case, seed), case=case)
    if not own:
        return state
    from xeno_rt_amd.ops import load_ops
    ops = state["ops"] = load_ops()
    if case["op"] in ("norm", "quantize"):
        state["q"] = ops.int8_rows(case["rows"], case["width"], DEVICE)
        state["values"] = torch.empty(case["rows"], case["width"], dtype=torch.bfloat16, device=DEVICE)
        return state

    def as_rows(values, scales):
        made = ops.int8_rows(values.shape[0], values.shape[1], DEVICE)
        made.values.zero_()
        made.values[:, : values.shape[1]] = values
        made.scales.copy_(scales)
        return made

    state["a8"] = as_rows(state.pop("a"), state.pop("a_scales"))
    state["w8"] = ops.pack_int8(as_rows(state.pop("w"), state.pop("w_scales")), gated=case["op"] == "gated")
    if not case.get("add"):
        state["out"] = torch.empty(case["rows"], case["n"], dtype=TYPES[case["out"]], device=DEVICE)
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------------------

def _plain_rows8(y):
    """The 8-bit rows of y (float32): the values that they stand for, and their scales."""
    scale = y.abs().amax(1, keepdim=True) / MOST
    q = torch.where(scale > 0, y / scale, torch.zeros_like(y)).round().clamp(-MOST, MOST).to(torch.int8)
    return (q.float() * scale).to(torch.bfloat16), scale[:, 0]


def _plain(state):
    case = state["case"]
    if case["op"] == "norm":
        x = state["x"]
        if state["delta"] is not None:
            x += state["delta"].float()
        y = x / torch.sqrt((x * x).mean(1, keepdim=True) + EPS) * state["gain"].float()
        values, scales = _plain_rows8(y)
        return {"x": x, "values": values, "scales": scales}
    if case["op"] == "quantize":
        values, scales = _plain_rows8(state["x"].float())
        return {"values": values, "scales": scales}
    sums = state["a"].float() @ state["w"].float().t() * state["a_scales"][:, None] * state["w_scales"]
    if case["op"] == "gated":
        gate, up = sums[:, : case["n"]], sums[:, case["n"]:]
        return {"out": (gate / (1.0 + torch.exp(-gate)) * up).to(TYPES[case["out"]])}
    if case["add"]:
        state["x"] += sums
        return {"out": state["x"]}
    return {"out": sums.to(TYPES[case["out"]])}


def _kernels(state):
    case, ops = state["case"], state["ops"]
    if case["op"] == "norm":
        ops.rmsnorm_int8(state["x"], state["gain"], EPS, state["q"], delta=state["delta"])
        ops.dequantize_int8(state["q"], state["values"])
        return {"x": state["x"], "values": state["values"], "scales": state["q"].scales}
    if case["op"] == "quantize":
        ops.quantize_int8(state["x"], state["q"])
        ops.dequantize_int8(state["q"], state["values"])
        return {"values": state["values"], "scales": state["q"].scales}
    if case["op"] == "gated":
        ops.linear_glu_int8(state["a8"], state["w8"], state["out"])
        return {"out": state["out"]}
    if case["add"]:
        ops.linear_int8(state["a8"], state["w8"], state["x"], accumulate=True)
        return {"out": state["x"]}
    ops.linear_int8(state["a8"], state["w8"], state["out"])
    return {"out": state["out"]}


def run(state):
    return _kernels(state) if own else _plain(state)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------------

def exact(case, seed):
    made = _inputs(case, seed)
    if case["op"] in ("norm", "quantize"):
        given = made["x"].double()
        if made.get("delta") is not None:
            given = given + made["delta"].double()
        y = given
        if case["op"] == "norm":
            mean = given.pow(2).sum(dim=1) / case["width"]
            y = torch.einsum("rc,r,c->rc", given, (mean + EPS).rsqrt(), made["gain"].double())
        scales = y.abs().max(dim=1).values / MOST
        values = torch.round(y / scales.unsqueeze(1)) * scales.unsqueeze(1)
        return {"x": given, "values": values, "scales": scales} if case["op"] == "norm" else {"values": values, "scales": scales}
    a = made["a"].double().mul_(made["a_scales"].double().unsqueeze(1))
    w = made["w"].double().mul_(made["w_scales"].double().unsqueeze(1))
    if case["op"] == "gated":
        gate, up = torch.mm(a, w[: case["n"]].t()), torch.mm(a, w[case["n"]:].t())
        return {"out": gate * torch.sigmoid(gate) * up}
    sums = torch.mm(a, w.t())
    return {"out": made["x"].double() + sums} if case["add"] else {"out": sums}
