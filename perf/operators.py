"""The cases by which the 8-bit and clipping operators are measured, and the operators' plain forms.

Operators (entry points of `distributedes_amd.ops.hip.HipOps`):

- ``quantize_rows(x)``: float rows to 8-bit rows, with one fp32 scale a row.
- ``int8_linear(x, wq, sw, bias, activation, out_dtype)``: quantises x's rows and multiplies them
  with 8-bit weights; ``int8_matmul`` takes rows that are quantised already.
- ``clip_by_global_norm(tensors, max_norm, out)``: the norm over all tensors, and the tensors bounded by it.
"""
import functools
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
_TINY = 2.0 ** -126

# parameter counts of the policies: MLP 4-64-64-2, and the Nature CNN with 18 actions
_MLP = "256,64,4096,64,128,2"
_NATURE = "8192,32,32768,64,36864,64,1605632,512,9216,18"
_LARGE = ",".join(["4194304", "4096", "1048577"] * 16)

_MOST_QUANTIZED = 1024 * 256 * 376
_MOST_PRODUCT = 8192 * 4096 * 4096
_MOST_WEIGHTS = 2048 * 512 * 3136


def listed():
    return [
        # one environment step's observations, a row for each of 10000 members
        {"name": "quantize-observations", "op": "quantize", "lead": 1, "rows": 10000, "cols": 376, "gap": 0, "dtype": "float32"},
        # the second layer of 1024 members, sliced out of their flat parameter rows
        {"name": "quantize-member-layer", "op": "quantize", "lead": 1024, "rows": 256, "cols": 256, "gap": 101137, "dtype": "float32"},
        # a batch of convolution features before the large fully connected layer
        {"name": "quantize-features", "op": "quantize", "lead": 1, "rows": 8192, "cols": 3136, "gap": 0, "dtype": "bfloat16"},
        # the smallest preset's hidden layer: 16 members, one observation each; latency
        {"name": "linear-members-small", "op": "linear", "members": 16, "tokens": 1, "channels": 64, "cols": 64, "dtype": "float32", "out": "float32", "act": "tanh", "packed": False},
        # the first layer of 10000 members, one observation each: every weight is read for one product
        {"name": "linear-members-wide", "op": "linear", "members": 10000, "tokens": 1, "channels": 256, "cols": 376, "dtype": "float32", "out": "float32", "act": "tanh", "packed": False},
        # one policy judged over its usual 16 episodes: the large fully connected layer
        {"name": "linear-episodes", "op": "linear", "members": 0, "tokens": 16, "channels": 512, "cols": 3136, "dtype": "bfloat16", "out": "float32", "act": "relu", "packed": False},
        # one policy over a full batch of 8192 environments
        {"name": "linear-batch", "op": "linear", "members": 0, "tokens": 8192, "channels": 512, "cols": 3136, "dtype": "bfloat16", "out": "bfloat16", "act": "relu", "packed": False},
        # the large fully connected layer with its own weights for each of 2048 members
        {"name": "matmul-members-fc", "op": "matmul", "members": 2048, "tokens": 1, "channels": 512, "cols": 3136, "dtype": "float32", "out": "float32", "act": "none", "packed": False},
        # a large square layer over many tokens: matrix cores
        {"name": "matmul-large", "op": "matmul", "members": 0, "tokens": 8192, "channels": 4096, "cols": 4096, "dtype": "float32", "out": "bfloat16", "act": "none", "packed": False},
        # the smallest preset's gradient, layer by layer; latency
        {"name": "clip-small", "op": "clip", "sizes": _MLP, "dtype": "float32", "clipped": True},
        # the Nature CNN's gradient, layer by layer
        {"name": "clip-policy", "op": "clip", "sizes": _NATURE, "dtype": "float32", "clipped": True},
        # the gradients of a large model: 48 tensors, odd sizes among them
        {"name": "clip-large", "op": "clip", "sizes": _LARGE, "dtype": "bfloat16", "clipped": True},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "linear", "matmul", "matmul", "clip"))
    dtype = rng.choice(("float32", "bfloat16", "float16"))
    if op == "quantize":
        cols = _spread(rng, 1, 8192)
        lead = _spread(rng, 1, 4096)
        rows = _spread(rng, 1, max(1, min(65536, _MOST_QUANTIZED // 2 // (cols * lead))))
        return {"op": op, "lead": lead, "rows": rows, "cols": cols, "gap": rng.choice((0, 0, 5, 1000)), "dtype": dtype}
    if op == "clip":
        count = _spread(rng, 1, 60)
        total = _spread(rng, 64, 50_000_000)
        sizes = [_spread(rng, 1, max(1, total // count)) for _ in range(count)]
        return {"op": op, "sizes": ",".join(map(str, sizes)), "dtype": dtype, "clipped": rng.random() < 0.7}
    case = {"op": op, "dtype": "float32" if op == "matmul" else dtype, "out": rng.choice(("float32", "bfloat16", "float16")),
            "act": rng.choice(("none", "relu", "tanh")), "packed": rng.random() < 0.25}
    if rng.random() < 0.5:
        channels, cols = _spread(rng, 1, 512), _spread(rng, 1, 3136)
        members = _spread(rng, 2, max(2, min(10000, _MOST_WEIGHTS // 2 // (channels * cols))))
        return {**case, "members": members, "tokens": rng.choice((1, 1, 1, 2, 5, 16)), "channels": channels, "cols": cols}
    channels, cols = _spread(rng, 1, 4096), _spread(rng, 1, 4096)
    return {**case, "members": 0, "tokens": _spread(rng, 1, 16384), "channels": channels, "cols": cols}


def _codes(gen, lead, rows, cols, packed):
    """8-bit rows of normal values and their scales, as quantize_rows lays them out: rows begin at
    multiples of 16 bytes (not where `packed`)."""
    step = cols if packed else -(-cols // 16) * 16
    store = torch.zeros(lead, rows, step, dtype=torch.int8, device="cuda")
    scale = torch.empty(lead, rows, device="cuda")
    part = max(1, (1 << 27) // max(1, rows * cols))
    for i in range(0, lead, part):
        x = torch.randn(min(part, lead - i), rows, cols, generator=gen, device="cuda") / math.sqrt(cols)
        s = (x.abs().amax(-1) / 127).clamp_min(_TINY)
        store[i:i + part, :, :cols] = (x / s.unsqueeze(-1)).round().clamp(-127, 127).to(torch.int8)
        scale[i:i + part] = s
    return store[:, :, :cols], scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "quantize":
        lead, rows, cols = case["lead"], case["rows"], case["cols"]
        flat = torch.randn(lead, rows * cols + case["gap"], generator=gen, device="cuda")
        x = flat[:, :rows * cols].unflatten(1, (rows, cols))
        x[:, ::97] = 0  # rows of members that are done
        state["x"] = flat.to(dtype)[:, :rows * cols].unflatten(1, (rows, cols))
        return state
    if case["op"] == "clip":
        state["grads"] = [(torch.randn(int(n), generator=gen, device="cuda") * 1e-2).to(dtype) for n in case["sizes"].split(",")]
        state["out"] = [torch.empty_like(g) for g in state["grads"]]
        total = math.sqrt(sum(g.numel() for g in state["grads"])) * 1e-2
        state["max_norm"] = total * (0.25 if case["clipped"] else 4.0)
        return state
    lead = max(1, case["members"])
    state["wq"], state["sw"] = _codes(gen, lead, case["channels"], case["cols"], case["packed"])
    state["bias"] = torch.randn(lead, case["channels"], generator=gen, device="cuda") * 0.1
    if case["op"] == "matmul":
        state["xq"], state["sx"] = _codes(gen, lead, case["tokens"], case["cols"], case["packed"])
    else:
        x = torch.randn(lead, case["tokens"], case["cols"], generator=gen, device="cuda")
        state["x"] = (x.relu() if case["act"] == "relu" else x.clamp(-5, 5)).to(dtype)
    if not case["members"]:  # one policy: no axis of members
        state.update({k: state[k][0] for k in ("wq", "sw", "bias", "x", "xq", "sx") if k in state})
    return state


@functools.lru_cache(maxsize=None)
def _ops():
    from distributedes_amd.ops.hip import HipOps
    return HipOps()


def _quantize(x):
    """Plain quantize_rows: the quotients in 64 bits, since a value near the border of two codes falls to
    one of them by less than a 32-bit quotient holds."""
    scale = (x.double().abs().amax(-1) / 127).float().clamp_min(_TINY)
    codes = (x.double() / scale.double().unsqueeze(-1)).round().to(torch.int8)
    return codes, scale


def _product(xq, sx, wq, sw, bias, act, out):
    """Plain int8_matmul."""
    if wq.dim() == 2:
        total = xq.float() @ wq.float().t()
    else:
        total = torch.bmm(wq.float(), xq.float().transpose(1, 2).contiguous()).transpose(1, 2)
    y = total * sx.unsqueeze(-1) * sw.unsqueeze(-2) + bias.unsqueeze(-2)
    y = y.clamp_min(0) if act == "relu" else y.tanh() if act == "tanh" else y
    return y.to(out)


def run(state):
    op = state["op"]
    if op == "clip":
        grads, most = state["grads"], state["max_norm"]
        if own:
            clipped, norm = _ops().clip_by_global_norm(grads, most, out=state["out"])
            return {"grads": clipped, "norm": norm}
        norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
        factor = torch.where(norm > most, most / norm, torch.ones_like(norm))
        return {"grads": [(g.float() * factor).to(g.dtype) for g in grads], "norm": norm}
    if op == "quantize":
        codes, scale = _ops().quantize_rows(state["x"]) if own else _quantize(state["x"])
        return {"codes": codes, "scale": scale}  # codes are whole numbers and compared as such
    act, out = state["act"], _DTYPES[state["out"]]
    weights = state["wq"], state["sw"]
    if own:
        how = {"bias": state["bias"], "activation": act, "out_dtype": out}
        if op == "linear":
            return _ops().int8_linear(state["x"], *weights, **how)
        return _ops().int8_matmul(state["xq"], state["sx"], *weights, **how)
    rows = _quantize(state["x"]) if op == "linear" else (state["xq"], state["sx"])
    return _product(*rows, *weights, state["bias"], act, out)


def work(case):
    """Each input read once, each output written once."""
    if case["op"] == "quantize":
        rows = case["lead"] * case["rows"]
        return {"bytes": rows * case["cols"] * (_BYTES[case["dtype"]] + 1) + rows * 4, "flops": 3 * rows * case["cols"]}
    if case["op"] == "clip":
        total = sum(map(int, case["sizes"].split(",")))
        return {"bytes": 2 * total * _BYTES[case["dtype"]] + 4, "flops": 3 * total}
    lead, m, n, k = max(1, case["members"]), case["tokens"], case["channels"], case["cols"]
    rows = m * k * _BYTES[case["dtype"]] if case["op"] == "linear" else m * (k + 4)
    return {"bytes": lead * (n * k + 8 * n + rows + m * n * _BYTES[case["out"]]), "flops": 2 * lead * m * n * k}


def exact(case, seed):
    """The operators' definition in 64 bits. A scale is held in 32 bits, so it is rounded there."""
    state = prepare(case, seed)
    if case["op"] == "clip":
        flat = torch.cat([g.to(torch.float64) for g in state["grads"]])
        norm = torch.linalg.vector_norm(flat)
        share = min(1.0, state["max_norm"] / norm.item())
        return {"grads": list((flat * share).split([g.numel() for g in state["grads"]])), "norm": norm}

    def rounded(x):
        x = x.to(torch.float64)
        top = torch.maximum(x.amax(-1, keepdim=True), -x.amin(-1, keepdim=True))
        step = torch.maximum((top / 127).to(torch.float32).to(torch.float64), torch.full_like(top, _TINY))
        return torch.div(x, step).round(), step

    if case["op"] == "quantize":
        values, step = rounded(state["x"])
        return {"codes": values.to(torch.int8), "scale": step.squeeze(-1)}
    if case["op"] == "linear":
        values, step = rounded(state["x"])
    else:
        values, step = state["xq"].to(torch.float64), state["sx"].to(torch.float64).unsqueeze(-1)
    weights = state["wq"].to(torch.float64) * state["sw"].to(torch.float64).unsqueeze(-1)
    if case["members"]:
        y = torch.stack([(v @ w.T) for v, w in zip(values * step, weights)])
        y = y + state["bias"].to(torch.float64)[:, None, :]
    else:
        y = torch.addmm(state["bias"].to(torch.float64), values * step, weights.T)
    return {"none": y, "relu": torch.relu(y), "tanh": torch.tanh(y)}[case["act"]]
