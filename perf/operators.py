"""Measured cases of the microscaled operators: quantisation to 4 and 8 bits, the RMS norm that feeds it, and the product.

A microscaled tensor holds its last dimension in blocks of 32 elements that share one power of two.  ``mxfp4`` elements
are e2m1 (+-0, .5, 1, 1.5, 2, 3, 4, 6), two to a byte with the even column in the low bits; ``mxfp8`` elements are e4m3.
A scale is one byte e with the value 2^(e - 127), 255 for NaN.  Rows are padded with zeros to whole groups of 128
elements.

``run`` computes one pass of a case: with ``own`` false from elementary tensor operations in fp32, with ``own`` true
through the package's public calls.
"""
import torch

own = False

BLOCK = 32
EMAX = {"mxfp4": 2, "mxfp8": 8}           # exponent of the largest element
LARGEST = {"mxfp4": 6.0, "mxfp8": 448.0}
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # one generated token: its hidden state goes to 4 bits before the next product
        dict(name="quantize_mxfp4_1x4096_bf16", op="quantize", rows=1, cols=4096, dtype="bf16", format="mxfp4"),
        # a weight matrix after an update, laid out in 4 bits for the forward passes of the next step
        dict(name="quantize_mxfp4_4096x4096_fp32", op="quantize", rows=4096, cols=4096, dtype="fp32", format="mxfp4"),
        # activations of a long prompt, with rows that end inside a block
        dict(name="quantize_mxfp8_4099x4111_fp16", op="quantize", rows=4099, cols=4111, dtype="fp16", format="mxfp8"),
        # one generated token: norm in front of a product with 8-bit activations
        dict(name="norm_mxfp8_1x4096_bf16", op="norm", rows=1, cols=4096, dtype="bf16", members=0, residual=True,
             out="mxfp8"),
        # a prompt batch through the same norm
        dict(name="norm_mxfp8_8192x4096_bf16", op="norm", rows=8192, cols=4096, dtype="bf16", members=0, residual=True,
             out="mxfp8"),
        # a population of 1024 members, each with a gain of its own, fp32 throughout as the other layers
        dict(name="norm_population_16384x1000_fp32", op="norm", rows=16384, cols=1000, dtype="fp32", members=1024,
             residual=False, out="fp32"),
        # one generated token through a square layer: bound by the weights' bytes
        dict(name="linear_1x4096x4096_w4a8_bf16", op="linear", rows=1, cols=4096, outs=4096, dtype="bf16",
             weights="mxfp4", activations="mxfp8"),
        # a decode batch through a wide layer
        dict(name="linear_24x8192x8192_w4a4_bf16", op="linear", rows=24, cols=8192, outs=8192, dtype="bf16",
             weights="mxfp4", activations="mxfp4"),
        # odd sizes on every side, fp32 in and out
        dict(name="linear_333x1000x1537_w4a8_fp32", op="linear", rows=333, cols=1000, outs=1537, dtype="fp32",
             weights="mxfp4", activations="mxfp8"),
        # the base product of a 1024-member population layer
        dict(name="linear_1024x1024x1024_w4a4_fp32", op="linear", rows=1024, cols=1024, outs=1024, dtype="fp32",
             weights="mxfp4", activations="mxfp4"),
        # a prompt batch through the layers of a feed-forward block: 8-bit activations, and all in 4 bits
        dict(name="linear_4096x4096x8192_w4a8_bf16", op="linear", rows=4096, cols=4096, outs=8192, dtype="bf16",
             weights="mxfp4", activations="mxfp8"),
        dict(name="linear_8192x4096x16384_w4a4_bf16", op="linear", rows=8192, cols=4096, outs=16384, dtype="bf16",
             weights="mxfp4", activations="mxfp4"),
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], uniform over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "linear"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    while True:
        rows = _spread(rng, 1, 16384)
        cols = _spread(rng, 64, 16384)
        if rng.random() < 0.5:
            cols = max(64, cols // 64 * 64)
        if op != "linear":
            if rows * cols > 8192 * 4096:
                continue
            if op == "quantize":
                return dict(op=op, rows=rows, cols=cols, dtype=dtype, format=rng.choice(["mxfp4", "mxfp8"]))
            members = rng.choice([0, 0, _spread(rng, 1, rows)])
            rows = rows // members * members if members else rows
            return dict(op=op, rows=rows, cols=cols, dtype=dtype, members=members, residual=rng.random() < 0.6,
                        out=rng.choice(["mxfp8", "mxfp8", "mxfp4", dtype]))
        outs = _spread(rng, 64, 16384)
        if rows <= 8192 and rows * cols * outs <= 8192 * 4096 * 16384 and cols * outs <= 8192 * 16384:
            weights, activations = rng.choice([("mxfp4", "mxfp4"), ("mxfp4", "mxfp8"), ("mxfp8", "mxfp8")])
            return dict(op=op, rows=rows, cols=cols, outs=outs, dtype=dtype, weights=weights, activations=activations)


# ------------------------------------------------------------------------------------------------ inputs

def _activations(g, rows, cols, dtype):
    """Hidden states: normal values, a few channels much larger than the rest, rows of different size."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    channel = torch.rand(cols, generator=g, device="cuda")
    x *= torch.where(channel > 0.995, 20.0, 0.5 + channel)
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda"))
    return x.to(DTYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    state["x"] = _activations(g, case["rows"], case["cols"], case["dtype"])
    if case["op"] == "norm":
        state["gain"] = 1.0 + 0.2 * torch.randn(case["cols"], generator=g, device="cuda")
        state["res"] = _activations(g, case["rows"], case["cols"], case["dtype"]) if case["residual"] else None
        state["noise"] = (0.02 * torch.randn(case["members"], case["cols"], generator=g, device="cuda")
                          if case["members"] else None)
    if case["op"] == "linear":
        w = torch.randn(case["outs"], case["cols"], generator=g, device="cuda") / case["cols"] ** 0.5
        state["codes"], state["scales"] = _stored(w, case["weights"])
        state["bias"] = 0.1 * torch.randn(case["outs"], generator=g, device="cuda")
    return state


def _stored(w, form):
    """A matrix in the stored form of the weights: codes and scales as bytes, rows padded to 128 elements."""
    elements, exponents = _blocks(w, form)
    pad = -w.shape[1] % 128
    if form == "mxfp4":
        magnitude = elements.abs()
        code = sum((magnitude >= v).to(torch.uint8) for v in (0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0))
        code |= (elements < 0).to(torch.uint8) << 3
        code = torch.nn.functional.pad(code, (0, pad))
        codes = code[:, 0::2] | (code[:, 1::2] << 4)
    else:
        codes = torch.nn.functional.pad(elements.to(torch.float8_e4m3fn).view(torch.uint8), (0, pad))
    scales = torch.nn.functional.pad((exponents + 127).to(torch.uint8), (0, (w.shape[1] + pad) // BLOCK - exponents.shape[1]))
    return codes.contiguous(), scales.contiguous()


# -------------------------------------------------------------------------------------------- plain forms

def _power(e):
    """2^e as fp32, exactly, for whole e in [-252, 254]: the product of two powers put together from their bits."""
    half = e >> 1
    return ((half + 127) << 23).view(torch.float32) * ((e - half + 127) << 23).view(torch.float32)


def _blocks(x, form):
    """Elements (fp32 values, rows x cols) and block exponents (rows x blocks) of finite fp32 values."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    largest = x.abs().amax(dim=-1)
    exponents = torch.frexp(largest).exponent - 1 - EMAX[form]        # largest = m * 2^e with m in [1/2, 1)
    exponents = torch.where(largest > 0, exponents, -127).clamp_(min=-127)
    scaled = x * _power(-exponents).unsqueeze(-1)
    if form == "mxfp4":
        a = scaled.abs()                                              # ties go to the even code
        steps = (0.5 * (a > 0.25) + 0.5 * (a >= 0.75) + 0.5 * (a > 1.25) + 0.5 * (a >= 1.75)
                 + 1.0 * (a > 2.5) + 1.0 * (a >= 3.5) + 2.0 * (a > 5.0))
        elements = torch.where(scaled < 0, -steps, steps)
    else:
        elements = scaled.clamp(-LARGEST[form], LARGEST[form]).to(torch.float8_e4m3fn).float()
    return elements.view(rows, -1)[:, :cols], exponents


def _returned(x, form):
    elements, exponents = _blocks(x, form)
    return {"elements": elements.to(torch.float8_e4m3fn), "scales": (exponents + 127).to(torch.uint8).view(torch.float8_e8m0fnu)}


def _values(elements, exponents):
    scale = _power(exponents).repeat_interleave(BLOCK, dim=1)
    return elements * scale[:, :elements.shape[1]]


def _plain_norm(s):
    h = s["x"].float()
    if s["res"] is not None:
        h = h + s["res"].float()
    gain = s["gain"]
    if s["noise"] is not None:                                        # row r * members + d has member d's gain
        gain = (gain + s["noise"]).repeat(s["rows"] // s["members"], 1)
    y = h * torch.rsqrt((h * h).mean(dim=-1, keepdim=True) + EPS) * gain
    out = _returned(y, s["out"]) if s["out"] in EMAX else {"y": y.to(DTYPES[s["out"]])}
    if s["res"] is not None:
        out["residual"] = h.to(s["x"].dtype)
    return out


def _plain_linear(s):
    x = _values(*_blocks(s["x"].float(), s["activations"]))
    if s["weights"] == "mxfp4":
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
        table = torch.cat([table, -table])
        code = torch.stack([s["codes"] & 15, s["codes"] >> 4], dim=-1).view(s["outs"], -1)
        elements = table[code.int()]
    else:
        elements = s["codes"].view(torch.float8_e4m3fn).float()
    w = _values(elements, s["scales"].int() - 127)[:, :s["cols"]]
    return (x @ w.t() + s["bias"]).to(s["x"].dtype)


# --------------------------------------------------------------------------------------------------- pass

def run(state):
    if own:
        from nesgpu_b200 import microscaling
        if state["op"] == "quantize":
            q = microscaling.quantize(state["x"], state["format"])
            return {"elements": q.elements(), "scales": q.block_scales()}
        if state["op"] == "norm":
            out = state["out"] if state["out"] in EMAX else DTYPES[state["out"]]
            y = microscaling.rms_norm(state["x"], state["gain"], eps=EPS, residual=state["res"], noise=state["noise"],
                                      output=out)
            y, h = y if state["res"] is not None else (y, None)
            got = {"elements": y.elements(), "scales": y.block_scales()} if state["out"] in EMAX else {"y": y}
            if h is not None:
                got["residual"] = h
            return got
        weight = microscaling.MicroscaledTensor(state["codes"], state["scales"], state["cols"], state["weights"])
        return microscaling.linear(state["x"], weight, state["bias"], activations=state["activations"])
    if state["op"] == "quantize":
        return _returned(state["x"].float(), state["format"])
    return _plain_norm(state) if state["op"] == "norm" else _plain_linear(state)


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2, "mxfp4": 0.5 + 1 / BLOCK, "mxfp8": 1 + 1 / BLOCK}
    n = case["rows"] * case["cols"]
    if case["op"] == "quantize":          # elements come back as one byte each
        unpacked = n if case["format"] == "mxfp4" else 0
        return {"bytes": n * (size[case["dtype"]] + size[case["format"]]) + unpacked, "flops": 4 * n}
    if case["op"] == "norm":
        moved = n * (size[case["dtype"]] * (3 if case["residual"] else 1) + size[case["out"]])
        moved += n if case["out"] == "mxfp4" else 0
        return {"bytes": moved + 4 * case["cols"] * (1 + case["members"]), "flops": 8 * n}
    moved = n * size[case["dtype"]] + case["outs"] * (case["cols"] * size[case["weights"]] + 4)
    moved += case["rows"] * case["outs"] * size[case["dtype"]]
    return {"bytes": moved, "flops": 2 * n * case["outs"]}


# ------------------------------------------------------------------------------------------ in 64 bits

def _binade(v):
    """floor(log2 |v|) from the exponent bits of a 64-bit value (-1023 for zero)."""
    return ((v.view(torch.int64) >> 52 & 2047) - 1023).double()


def _exact_blocks(x, form):
    """The same blocks from the definition, in 64 bits: round(v / step) * step with the step of v's binade."""
    rows, cols = x.shape
    lowest, mantissa = (0, 1) if form == "mxfp4" else (-6, 3)          # smallest normal exponent, fraction bits
    out = torch.zeros(rows, -(-cols // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    out[:, :cols] = x
    out = out.reshape(-1, BLOCK)
    top = out.abs().max(dim=1).values
    e = torch.clamp(_binade(top) - EMAX[form], min=-127)
    out /= torch.exp2(e)[:, None]
    step = torch.exp2(torch.clamp(_binade(out), min=lowest) - mantissa)
    out = torch.clamp(torch.round(out / step) * step, -LARGEST[form], LARGEST[form])
    return out.reshape(rows, -1)[:, :cols], e.reshape(rows, -1)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "quantize":
        elements, e = _exact_blocks(x, case["format"])
        return {"elements": elements, "scales": torch.exp2(e)}
    if case["op"] == "norm":
        h = x if s["res"] is None else x + s["res"].double()
        y = h / torch.sqrt(h.square().sum(dim=1, keepdim=True) / case["cols"] + EPS)
        if s["noise"] is None:
            y = y * s["gain"].double()
        else:
            member = torch.arange(case["rows"], device="cuda") % case["members"]
            y = y * (s["gain"].double() + s["noise"].double()[member])
        if case["out"] in EMAX:
            elements, e = _exact_blocks(y, case["out"])
            got = {"elements": elements, "scales": torch.exp2(e)}
        else:
            got = {"y": y}
        if s["res"] is not None:
            got["residual"] = h
        return got
    elements, e = _exact_blocks(x, case["activations"])
    a = elements.reshape(case["rows"], -1)
    column = torch.arange(case["cols"], device="cuda")
    a = a * torch.exp2(e)[:, column // BLOCK]
    if case["weights"] == "mxfp4":
        nibble = (s["codes"].long()[:, column // 2] >> (4 * (column % 2))) & 15
        exponent, fraction = (nibble >> 1) & 3, (nibble & 1).double()
        w = torch.where(exponent > 0, (2 + fraction) * torch.exp2(exponent.double() - 2), 0.5 * fraction)
        w = torch.where(nibble >= 8, -w, w)
    else:
        w = s["codes"].view(torch.float8_e4m3fn)[:, :case["cols"]].to(torch.float64)
    w = w * torch.exp2(s["scales"].double()[:, column // BLOCK] - 127)
    return torch.matmul(a, w.t()) + s["bias"].double()
