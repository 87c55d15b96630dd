"""Training and 8-bit operators around the pair stack: LayerNorm and its gradient, 8-bit activation checkpoints, and the
projection in 8-bit floating point with its two gradients.

``prepare`` makes what a program has in hand before the call, ``run`` makes one pass: in plain torch operations, or
(``own``) by the package's public classes.  ``exact`` computes the same from the definitions in 64 bits.

The 8-bit format: 128 consecutive channels of a row (128 x 128 elements of a weight) share a power of two, the least one
that brings the block's largest finite magnitude to 448 (e4m3) or 57344 (e5m2) at most, and not below 2^-126.
"""
import math

import torch

own = False

EPSILON = 1e-5
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
LIMIT_EXPONENT = {"e4m3": 8, "e5m2": 15}      # the largest finite code is 1.75 * 2^this


def listed():
    return [
        # the single track's norm of a short chain: the smallest call, latency counts
        {"name": "norm_single_n76", "op": "norm", "rows": 76, "channels": 384, "dtype": "bf16"},
        # a deep extra-MSA alignment in float32, 64 channels, odd length
        {"name": "norm_extra_msa_f32", "op": "norm", "rows": 1024 * 201, "channels": 64, "dtype": "f32"},
        # a training step through the pair's norm at N = 384: the input is kept in 8 bits for the backward pass
        {"name": "norm_step_pair_n384", "op": "norm_step", "rows": 384 * 384, "channels": 128, "dtype": "bf16", "checkpoint": "e4m3"},
        # ... through the MSA's norm (128 sequences x 256 residues), float32, the input kept whole
        {"name": "norm_step_msa_f32", "op": "norm_step", "rows": 128 * 256, "channels": 256, "dtype": "f32", "checkpoint": ""},
        # ... of an odd width that no vector access divides
        {"name": "norm_step_odd", "op": "norm_step", "rows": 2049, "channels": 1155, "dtype": "bf16", "checkpoint": "e5m2"},
        # a pair tensor at N = 1024 put away in 8 bits and brought back: the largest by bytes
        {"name": "checkpoint_pair_n1024", "op": "checkpoint", "rows": 1024 * 1024, "channels": 128, "dtype": "bf16", "format": "e4m3"},
        # a float32 gradient with its wide range, odd length, a last block of 72 channels
        {"name": "checkpoint_gradient_odd", "op": "checkpoint", "rows": 201 * 203, "channels": 200, "dtype": "f32", "format": "e5m2"},
        # four tokens through a projection of the single track's transition: weights are all that is read
        {"name": "linear_tokens_4", "op": "linear", "rows": 4, "channels": 1536, "outputs": 384, "dtype": "bf16", "format": "e4m3"},
        # the pair transition's first projection at N = 384
        {"name": "linear_pair_n384", "op": "linear", "rows": 384 * 384, "channels": 128, "outputs": 512, "dtype": "bf16", "format": "e4m3"},
        # a square product bound by the tensor cores: the largest by operations
        {"name": "linear_square_4096", "op": "linear", "rows": 4096, "channels": 4096, "outputs": 4096, "dtype": "bf16", "format": "e4m3"},
        # a training step of the pair transition's second projection at N = 256, weights encoded anew as in every step
        {"name": "linear_step_pair_n256", "op": "linear_step", "rows": 256 * 256, "channels": 512, "outputs": 128, "dtype": "bf16",
         "format": "e4m3"},
        # ... in float32 with sizes that no tile divides and gradients in e5m2
        {"name": "linear_step_odd_f32", "op": "linear_step", "rows": 3001, "channels": 449, "outputs": 1283, "dtype": "f32",
         "format": "e5m2"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_step", "checkpoint", "linear", "linear_step"])
    case = {"op": op, "dtype": rng.choice(["f32", "bf16"])}
    if op in ("norm", "norm_step", "checkpoint"):
        case["channels"] = _log_int(rng, 8, 2048)
        case["rows"] = _log_int(rng, 1, 30_000_000 // case["channels"])
        if op == "norm_step":
            case["checkpoint"] = rng.choice(["", "e4m3", "e5m2"])
        if op == "checkpoint":
            case["format"] = rng.choice(["e4m3", "e5m2"])
        return case
    case["format"] = rng.choice(["e4m3", "e5m2"])
    case["channels"] = _log_int(rng, 8, 4096)
    case["outputs"] = _log_int(rng, 8, 4096)
    flops = 6 if op == "linear_step" else 2
    most = min(100_000_000_000 // (flops * case["channels"] * case["outputs"]), 60_000_000 // max(case["channels"], case["outputs"]))
    case["rows"] = _log_int(rng, 1, min(most, 200_000))
    return case


def work(case):
    rows, c = case["rows"], case["channels"]
    size = 4 if case["dtype"] == "f32" else 2
    op = case["op"]
    if op == "norm":
        return {"bytes": rows * c * 2 * size + 8 * c, "flops": 8 * rows * c}
    if op == "norm_step":
        kept = rows * (c + -(-c // 128)) if case["checkpoint"] else 0
        again = kept if case["checkpoint"] else rows * c * size
        # forward: input, output, statistics, checkpoint; backward: gradient, what was kept, statistics, result
        return {"bytes": rows * c * 4 * size + kept + again + 16 * rows + 20 * c, "flops": 20 * rows * c}
    if op == "checkpoint":
        return {"bytes": 2 * rows * (c * size + c + -(-c // 128)), "flops": 4 * rows * c}
    n = case["outputs"]
    if op == "linear":
        return {"bytes": rows * (c + n) * size + n * c + 4 * n, "flops": 2 * rows * c * n}
    # step: input, gradient and weight in; output, input's, weight's and bias' gradients out
    return {"bytes": 2 * rows * (c + n) * size + 8 * n * c + 8 * n, "flops": 6 * rows * c * n}


def _activations(generator, rows, c, dtype):
    """Rows of different size, channels of different gain, a few channels well above the others, as residual streams have them."""
    x = torch.randn(rows, c, generator=generator, device="cuda")
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=generator, device="cuda"))
    gain = torch.exp(0.5 * torch.randn(c, generator=generator, device="cuda"))
    gain[torch.rand(c, generator=generator, device="cuda") < 0.01] *= 20
    x *= gain
    x += 0.3 * torch.randn(c, generator=generator, device="cuda")
    return x.to(dtype)


def _gradient(generator, rows, c, dtype):
    """Small values over some orders of magnitude; the rows of padded residues (the last twentieth) have none."""
    g = torch.randn(rows, c, generator=generator, device="cuda")
    g *= 1e-3 * torch.exp(2.0 * torch.randn(rows, 1, generator=generator, device="cuda"))
    g[rows - rows // 20:] = 0
    return g.to(dtype)


def _inputs(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    rows, c, dtype = case["rows"], case["channels"], DTYPES[case["dtype"]]
    op = case["op"]
    if op == "checkpoint":
        return {"x": (_gradient if case["format"] == "e5m2" else _activations)(generator, rows, c, dtype)}
    state = {"x": _activations(generator, rows, c, dtype)}
    if op in ("norm", "norm_step"):
        state["scale"] = 1 + 0.1 * torch.randn(c, generator=generator, device="cuda")
        state["offset"] = 0.1 * torch.randn(c, generator=generator, device="cuda")
        if op == "norm_step":
            state["dy"] = _gradient(generator, rows, c, dtype)
        return state
    n = case["outputs"]
    state["weight"] = torch.randn(n, c, generator=generator, device="cuda") / math.sqrt(c)
    state["bias"] = 0.1 * torch.randn(n, generator=generator, device="cuda")
    if op == "linear_step":
        state["dy"] = _gradient(generator, rows, n, dtype)
    return state


_devices = {}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        import localfold_b200 as lf
        stream = torch.cuda.current_stream().cuda_stream
        if stream not in _devices:      # a program has one library context for its stream
            _devices[stream] = lf.Device(torch.cuda.current_device(), stream=stream)
        device = state["device"] = _devices[stream]
        if case["op"] in ("norm", "norm_step"):
            state["layer"] = lf.LayerNormGpu(device)
        elif case["op"] in ("linear", "linear_step"):
            state["layer"] = lf.Float8LinearGpu(device)
            state["weights"] = lf.prepare_float8_linear_weights(device, state["weight"], state["bias"])
    elif case["op"] == "linear":
        state["weight8"] = _decoded(state["weight"], "e4m3", 128)      # a serving program encodes its weights once
    return state


# ---- plain form --------------------------------------------------------------


def _decoded(x, name, block_rows=1):
    """The values that the 8-bit form of a matrix stands for, in float32."""
    x = x.float()
    rows, c = x.shape
    padded = torch.nn.functional.pad(x, (0, -c % 128, 0, -rows % block_rows))
    blocks = padded.view(padded.shape[0] // block_rows, block_rows, -1, 128)
    magnitude = torch.where(torch.isfinite(blocks), blocks.abs(), 0.0).amax((1, 3), keepdim=True)
    mantissa, exponent = torch.frexp(magnitude)
    exponent = (exponent - 1 - LIMIT_EXPONENT[name] + (mantissa > 0.875)).clamp(min=-126)
    exponent = torch.where(magnitude > 0, exponent, -126)
    code = torch.ldexp(blocks, -exponent).to(torch.float8_e4m3fn if name == "e4m3" else torch.float8_e5m2)
    return torch.ldexp(code.float(), exponent).view(padded.shape)[:rows, :c]


def _plain_norm(x, scale, offset):
    x = x.float()
    mean = x.mean(1, keepdim=True)
    inverse = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + EPSILON)
    return (x - mean) * inverse * scale + offset, mean, inverse


def _run_plain(state):
    case, x = state["case"], state["x"]
    op = case["op"]
    if op == "checkpoint":
        return {"activations": _decoded(x, case["format"]).to(x.dtype)}
    if op == "norm":
        return {"output": _plain_norm(x, state["scale"], state["offset"])[0].to(x.dtype)}
    if op == "norm_step":
        y, mean, inverse = _plain_norm(x, state["scale"], state["offset"])
        kept = _decoded(x, case["checkpoint"]) if case["checkpoint"] else x.float()
        dy = state["dy"].float()
        unit = (kept - mean) * inverse
        h = dy * state["scale"]
        dx = inverse * (h - h.mean(1, keepdim=True) - unit * (h * unit).mean(1, keepdim=True))
        return {"output": y.to(x.dtype), "activations": dx.to(x.dtype), "scale": (dy * unit).sum(0), "offset": dy.sum(0)}
    x8 = _decoded(x, "e4m3" if op == "linear_step" else case["format"])
    if op == "linear":
        return {"output": (x8 @ state["weight8"].T + state["bias"]).to(x.dtype)}
    w8 = _decoded(state["weight"], "e4m3", 128)
    dy8 = _decoded(state["dy"], case["format"])
    dy = dy8 if case["dtype"] == "f32" else state["dy"].float()      # a bf16 gradient is an exact operand as it is
    return {"output": (x8 @ w8.T + state["bias"]).to(x.dtype), "activations": (dy8 @ w8).to(x.dtype),
            "weight": dy.T @ x8, "bias": dy.sum(0)}


# ---- the package's operators ---------------------------------------------------


def _run_own(state):
    import localfold_b200 as lf
    case, x = state["case"], state["x"]
    op, rows, c = case["op"], case["rows"], case["channels"]
    if op == "checkpoint":
        kept = lf.float8_encode(state["device"], x, rows, c, {"format": case["format"]})
        return {"activations": lf.float8_decode(state["device"], kept, {"output": case["dtype"]})}
    layer = state["layer"]
    if op == "norm":
        return {"output": layer.run({"rows": rows, "channels": c, "activations": x, "scale": state["scale"], "offset": state["offset"],
                                     "epsilon": EPSILON})["output"]}
    if op == "norm_step":
        forward = layer.run({"rows": rows, "channels": c, "activations": x, "scale": state["scale"], "offset": state["offset"],
                             "epsilon": EPSILON}, {"statistics": True, "checkpoint": case["checkpoint"] or None})
        kept = forward["checkpoint"] if case["checkpoint"] else x
        back = layer.backward({"rows": rows, "channels": c, "gradient": state["dy"], "activations": kept, "mean": forward["mean"],
                               "inverseDeviation": forward["inverseDeviation"], "scale": state["scale"]})
        return {"output": forward["output"], "activations": back["activations"], "scale": back["scale"], "offset": back["offset"]}
    weights = state["weights"]
    shape = {"rows": rows, "channels": c, "outChannels": case["outputs"], "weights": weights}
    if op == "linear":
        return {"output": layer.run(dict(shape, activations=x), {"format": case["format"]})["output"]}
    weights.update(state["weight"], state["bias"])
    forward = layer.run(dict(shape, activations=x), {"format": "e4m3", "checkpoint": True})
    back = layer.input_gradient(dict(shape, gradient=state["dy"]), {"format": case["format"], "checkpoint": True})
    operand = back["checkpoint"] if case["dtype"] == "f32" else state["dy"]
    grads = layer.weight_gradient({"rows": rows, "channels": c, "outChannels": case["outputs"], "gradient": operand,
                                   "activations": forward["checkpoint"]})
    return {"output": forward["output"], "activations": back["output"], "weight": grads["weight"], "bias": grads["bias"]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- from the definitions, in 64 bits --------------------------------------------


def _rounded(values, name, block_rows):
    """Float8 by arithmetic on the values: each block's power of two, then the nearest multiple of the value's own step."""
    out = values.double().clone()
    bits, least, top = (3, -6, 448.0) if name == "e4m3" else (2, -14, 57344.0)
    for first in range(0, values.shape[1], 128):
        part = out[:, first:first + 128]
        size = part.abs().amax(1)
        if block_rows > 1:
            size = torch.stack([p.amax() for p in size.split(block_rows)]).repeat_interleave(block_rows)[:len(size)]
        power = torch.ceil(torch.log2(torch.where(size > 0, size, 1.0) / top))
        # log2 is not exact next to a whole number
        power = torch.where(size > top * torch.exp2(power), power + 1, power)
        power = torch.where(size <= top * torch.exp2(power - 1), power - 1, power)
        unit = torch.exp2(torch.where(size > 0, power, -126.0).clamp(min=-126))[:, None]
        scaled = part / unit
        step = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** (least - 1)))).clamp(min=least) - bits)
        part.copy_(torch.round(scaled / step) * step * unit)
    return out


def exact(case, seed):
    state = _inputs(case, seed)
    op, x = case["op"], state["x"].double()
    if op == "checkpoint":
        return {"activations": _rounded(x, case["format"], 1)}
    if op in ("norm", "norm_step"):
        scale, offset = state["scale"].double(), state["offset"].double()
        mean = x.mean(1, keepdim=True)
        deviation = torch.sqrt(x.var(1, unbiased=False, keepdim=True) + EPSILON)
        y = (x - mean) / deviation * scale + offset
        if op == "norm":
            return {"output": y}
        dy = state["dy"].double()
        unit = ((_rounded(x, case["checkpoint"], 1) if case["checkpoint"] else x) - mean) / deviation
        along = dy * scale
        c = case["channels"]
        dx = (along - (along.sum(1, keepdim=True) + unit * (along * unit).sum(1, keepdim=True)) / c) / deviation
        return {"output": y, "activations": dx, "scale": torch.einsum("rc,rc->c", dy, unit), "offset": dy.sum(0)}
    weight = _rounded(state["weight"], "e4m3", 128)
    bias = state["bias"].double()
    if op == "linear":
        return {"output": torch.addmm(bias, _rounded(x, case["format"], 1), weight.T)}
    inputs = _rounded(x, "e4m3", 1)
    gradient = _rounded(state["dy"], case["format"], 1)
    operand = gradient if case["dtype"] == "f32" else state["dy"].double()
    return {"output": torch.addmm(bias, inputs, weight.T), "activations": gradient @ weight,
            "weight": operand.T @ inputs, "bias": operand.sum(0)}
