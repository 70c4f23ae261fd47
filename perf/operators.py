"""Operators on microscaled matrices: 4-bit quantisation and product, 8-bit activation checkpoints and the backward pass
that reads them.  One pass through each, in its plain form and through the library's entry points (``own``).

Matrices are column-major, ``rows x columns``; as torch tensors they are therefore ``[columns, rows]``.  A microscaled matrix
has blocks of 32 rows in each column; a block shares the scale 2**X and a value is ``element * 2**X``:

  fp4    elements 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives (codes 0..7, +8 for the sign), two to a byte, the even row low
  int8   elements q / 64 with q = -127..127, one byte

X = floor(log2(largest magnitude of the block)) less 2 (fp4) or 0 (int8), at least -127; elements are rounded to nearest, ties
to even, and held at the largest one.  Columns are padded to whole blocks with zero codes.  A scale is stored as the byte
X + 127; the bytes of 128 columns x 4 blocks lie together in a tile of 512, at (column % 32) * 16 + (column % 128 // 32) * 4 +
block % 4, tiles of one 128 columns one after the other, missing columns and blocks with byte 0.

A case's ``kind``:

  quantize     matrix -> codes and scales -> values again (blocks along the rows, or along the columns: ``transpose``)
  times        Y (outputs x tokens) = W' X + bias, W (inputs x outputs) and X (inputs x tokens) both fp4
  weight_grad  dW (outputs x inputs) = dY X', X (inputs x tokens) an 8- or 4-bit checkpoint: the gradient matrix that the
               aggregator takes
  input_grad   dX (inputs x tokens) = W dY, W (inputs x outputs) as the product has it
  activation   a training step of a pointwise layer: y = f(x) with x kept in 8 bits (codes and scales), dx = dy f'(x kept)

``pad``: values between the end of one column and the start of the next in the dense operands (0: none).
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
FUNCTIONS = ("relu", "sigmoid", "tanh", "gelu", "silu")


# ---- cases --------------------------------------------------------------------------------------------------------------


def listed():
    return [
        # the 512 x 363 weight of the small speech net brought into product form after an update: latency
        {"name": "quantize_fp4_weight_512x363", "kind": "quantize", "rows": 512, "cols": 363, "type": "float32", "format": "fp4", "transpose": True, "pad": 0},
        # a minibatch of hidden activations kept for the backward pass: bandwidth
        {"name": "quantize_int8_2048x16384", "kind": "quantize", "rows": 2048, "cols": 16384, "type": "bfloat16", "format": "int8", "transpose": False, "pad": 0},
        # one token through a 2048 x 2048 layer: the weights are read once, and latency
        {"name": "times_token_2048", "kind": "times", "outputs": 2048, "inputs": 2048, "tokens": 1, "type": "float32", "pad": 0},
        # the first speech layer, 429 inputs, over a ragged minibatch
        {"name": "times_429_ragged", "kind": "times", "outputs": 2048, "inputs": 429, "tokens": 1001, "type": "bfloat16", "pad": 0},
        # a wide layer over a large batch: matrix units
        {"name": "times_4096", "kind": "times", "outputs": 4096, "inputs": 4096, "tokens": 8192, "type": "bfloat16", "pad": 0},
        # output layer of the small speech net, fp32 gradients as that net trains
        {"name": "weight_grad_132x512", "kind": "weight_grad", "outputs": 132, "inputs": 512, "tokens": 256, "type": "float32", "format": "int8", "pad": 0},
        # the first speech layer: 429 inputs, ragged minibatch
        {"name": "weight_grad_2048x429", "kind": "weight_grad", "outputs": 2048, "inputs": 429, "tokens": 4001, "type": "bfloat16", "format": "int8", "pad": 0},
        # the softmax layer of the headline set over a large minibatch
        {"name": "weight_grad_9304x2048", "kind": "weight_grad", "outputs": 9304, "inputs": 2048, "tokens": 8192, "type": "bfloat16", "format": "int8", "pad": 0},
        # 363 -> 512 layer of the small net, half-precision gradients, few samples
        {"name": "input_grad_512x363", "kind": "input_grad", "outputs": 512, "inputs": 363, "tokens": 64, "type": "float16", "pad": 0},
        # the softmax layer of the headline set over a large minibatch
        {"name": "input_grad_9304x2048", "kind": "input_grad", "outputs": 9304, "inputs": 2048, "tokens": 8192, "type": "bfloat16", "pad": 0},
        # sigmoid layer of the small net, a few samples: latency
        {"name": "activation_sigmoid_512x37", "kind": "activation", "rows": 512, "cols": 37, "type": "float32", "function": "sigmoid", "pad": 0},
        # a wide layer with a smooth unit over a large minibatch: bandwidth
        {"name": "activation_gelu_4096x8192", "kind": "activation", "rows": 4096, "cols": 8192, "type": "bfloat16", "function": "gelu", "pad": 0},
    ]


def _log_int(rng, lo, hi):
    """Log-uniform integer of [lo, hi]; every other one a multiple of 8 where that stays in range."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 8:
        v = v // 8 * 8
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["quantize", "times", "weight_grad", "input_grad", "activation"])
    case = {"kind": kind, "type": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), "pad": rng.choice([0, 0, 0, 8, 3])}
    if kind in ("quantize", "activation"):
        while True:
            rows, cols = _log_int(rng, 1, 16384), _log_int(rng, 1, 16384)
            if 64 <= rows * cols <= 1 << 25:
                break
        case |= {"rows": rows, "cols": cols}
        if kind == "quantize":
            case |= {"format": rng.choice(["fp4", "int8"]), "transpose": rng.random() < 0.4}
        else:
            case |= {"function": rng.choice(FUNCTIONS)}
        return case
    while True:
        outputs, inputs, tokens = _log_int(rng, 16, 9304), _log_int(rng, 16, 4096), _log_int(rng, 1, 8192)
        if outputs * inputs * tokens <= 1 << 36:
            break
    case |= {"outputs": outputs, "inputs": inputs, "tokens": tokens}
    if kind == "weight_grad":
        case |= {"format": rng.choice(["int8", "int8", "fp4"])}
    return case


# ---- the microscaled form, from its definition --------------------------------------------------------------------------


def _blocks(x):
    """[columns, rows] -> [columns, blocks, 32] in 32 bits, padded with zeros."""
    n, m = x.shape
    b = -(-m // 32)
    return torch.nn.functional.pad(x.float(), (0, b * 32 - m)).view(n, b, 32)


def _exponents(blocks, fmt):
    """X of each block."""
    largest = blocks.abs().amax(-1, keepdim=True)
    e = torch.frexp(largest).exponent - 1 - (2 if fmt == "fp4" else 0)
    return torch.where(largest > 0, e, -127).clamp(min=-127)


def _power(e):
    """2**e in 32 bits, exactly, for e of -127 to 127: its bit pattern (torch's own power is off by a unit now and then)."""
    return torch.where(e == -127, 1 << 22, (e + 127) << 23).int().view(torch.float32)


def _elements(blocks, exponents, fmt):
    """The rounded elements: multiples of 1/64 (int8), or of what fp4 has."""
    a = blocks * _power(-exponents)
    if fmt == "int8":
        return (a * 64).round().clamp(-127, 127) / 64
    m = a.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    return torch.copysign(((m / step).round() * step).clamp(max=6), a)


def _round_trip(x, fmt):
    """The values that a microscaled x ([columns, rows]) stands for."""
    blocks = _blocks(x)
    e = _exponents(blocks, fmt)
    return (_elements(blocks, e, fmt) * _power(e)).flatten(1)[:, : x.shape[1]].contiguous()


def _tile_at(n, b, device):
    """Where the scale bytes of n columns x b blocks lie, and how many bytes there are."""
    j, k = torch.arange(n, device=device)[:, None], torch.arange(b, device=device)[None, :]
    at = (j // 128 * -(-b // 4) + k // 4) * 512 + j % 32 * 16 + j % 128 // 32 * 4 + k % 4
    return at, -(-n // 128) * -(-b // 4) * 512


def _pack(x, fmt):
    """Codes and scales of x ([columns, rows]), as bytes."""
    blocks = _blocks(x)
    e = _exponents(blocks, fmt)
    el = _elements(blocks, e, fmt)
    if fmt == "int8":
        codes = (el * 64).to(torch.int8).view(torch.uint8).flatten(1)
    else:
        m = el.abs()
        c = torch.where(m < 2, m * 2, torch.where(m < 4, m + 2, m / 2 + 4)).to(torch.uint8)
        c = (c + (el < 0).to(torch.uint8) * 8).flatten(1)
        codes = c[:, 0::2] + c[:, 1::2] * 16
    at, size = _tile_at(e.shape[0], e.shape[1], x.device)
    scales = torch.zeros(size, dtype=torch.uint8, device=x.device)
    scales[at.flatten()] = (e.flatten() + 127).to(torch.uint8)
    return codes.contiguous(), scales


def _values(codes, scales, rows, fmt):
    """[columns, rows] in 32 bits: what codes and scales stand for."""
    n = codes.shape[0]
    if fmt == "int8":
        el = codes.view(torch.int8).float() / 64
    else:
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
        el = table[torch.stack((codes & 15, codes >> 4), -1).flatten(1).int()]
    b = el.shape[1] // 32
    at, _ = _tile_at(n, b, codes.device)
    e = scales[at].int() - 127
    return (el.view(n, b, 32) * _power(e)[..., None]).flatten(1)[:, :rows]


# ---- inputs -------------------------------------------------------------------------------------------------------------


def _random(n, m, case, gen, scale=1.0, pad=0):
    """[n, m] of the case's type, `pad` values between the columns; columns differ in size, as activations do."""
    size = torch.exp2(torch.empty(n, 1, device="cuda").normal_(0.0, 1.0, generator=gen)) * scale
    x = torch.empty(n, m + pad, device="cuda").normal_(0.0, 1.0, generator=gen) * size
    return x.to(TYPES[case["type"]])[:, :m]


def _packed(n, m, case, fmt, gen, scale=1.0):
    return _pack(_random(n, m, dict(case, type="float32"), gen, scale), fmt)


def _empty(n, m, dtype, pad):
    return torch.zeros(n, m + pad, dtype=dtype, device="cuda")[:, :m]


def _bytes(rows, cols, fmt):
    """(bytes of codes, bytes of scales) of a packed matrix."""
    b = -(-rows // 32)
    return cols * b * (32 if fmt == "int8" else 16), -(-cols // 128) * -(-b // 4) * 512


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, pad = case["kind"], case["pad"]
    state = {"case": case}
    if kind in ("quantize", "activation"):
        rows, cols = case["rows"], case["cols"]
        state["x"] = _random(cols, rows, case, gen, 2.0 if kind == "activation" else 0.05, pad)
        fmt = case.get("format", "int8")
        m, n = (cols, rows) if case.get("transpose") else (rows, cols)
        codes, scales = _bytes(m, n, fmt)
        state["codes"] = torch.zeros(codes, dtype=torch.uint8, device="cuda")
        state["scales"] = torch.zeros(scales, dtype=torch.uint8, device="cuda")
        state["kept"] = torch.zeros(n, m, device="cuda")
        if kind == "activation":
            state["dy"] = _random(cols, rows, case, gen, 1e-2, pad)
            state["y"] = _empty(cols, rows, TYPES[case["type"]], pad)
            state["dx"] = _empty(cols, rows, TYPES[case["type"]], pad)
        return state
    outputs, inputs, tokens, dtype = case["outputs"], case["inputs"], case["tokens"], TYPES[case["type"]]
    if kind in ("times", "input_grad"):
        state["w"] = _packed(outputs, inputs, case, "fp4", gen, 0.05)
    if kind in ("times", "weight_grad"):
        state["x"] = _packed(tokens, inputs, case, case.get("format", "fp4"), gen)
    if kind == "times":
        state["bias"] = torch.empty(outputs, device="cuda").normal_(0.0, 0.5, generator=gen)
        state["y"] = _empty(tokens, outputs, dtype, pad)
    else:
        state["dy"] = _random(tokens, outputs, case, gen, 1e-2, pad)
    if kind == "weight_grad":
        state["dw"] = torch.zeros(inputs, outputs, device="cuda")
    if kind == "input_grad":
        state["dx"] = _empty(tokens, inputs, dtype, pad)
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------------


def _function(x, name):
    """f(x) and f'(x) in 32 bits."""
    if name == "relu":
        return x.clamp(min=0), (x > 0).float()
    if name == "sigmoid":
        s = 1 / (1 + torch.exp(-x))
        return s, s * (1 - s)
    if name == "tanh":
        t = torch.tanh(x)
        return t, 1 / torch.cosh(x).square()
    if name == "gelu":
        c = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
        return x * c, c + x * torch.exp(-0.5 * x * x) * (0.5 / math.pi) ** 0.5
    s = 1 / (1 + torch.exp(-x))
    return x * s, s * (1 + x * (1 - s))


def _run_plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "quantize":
        return _round_trip(state["x"].t() if case["transpose"] else state["x"], case["format"])
    if kind == "activation":
        x = state["x"].float()
        kept = _round_trip(x, "int8")
        dx = state["dy"].float() * _function(kept, case["function"])[1]
        return {"y": _function(x, case["function"])[0].to(state["y"].dtype), "kept": kept, "dx": dx.to(state["dx"].dtype)}
    if kind == "times":
        w, x = _values(*state["w"], case["inputs"], "fp4"), _values(*state["x"], case["inputs"], "fp4")
        return (torch.matmul(x, w.t()) + state["bias"]).to(state["y"].dtype)
    if kind == "weight_grad":
        x = _values(*state["x"], case["inputs"], case["format"])
        return torch.matmul(x.t(), state["dy"].float())
    w = _values(*state["w"], case["inputs"], "fp4")
    return torch.matmul(state["dy"].float(), w).to(state["dx"].dtype)


def _run_own(state):
    from cntk_b200 import lib

    case = state["case"]
    kind = case["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    dtype = {"float32": lib.F32, "float16": lib.F16, "bfloat16": lib.BF16}[case["type"]]
    fmt = lib.MXFP4 if case.get("format", "fp4") == "fp4" else lib.MXINT8
    if kind in ("quantize", "activation"):
        x, codes, scales, kept = state["x"], state["codes"], state["scales"], state["kept"]
        rows, cols = case["rows"], case["cols"]
        n, m = kept.shape
        if kind == "quantize":
            lib.mx_quantize(x.data_ptr(), dtype, rows + case["pad"], codes.data_ptr(), scales.data_ptr(), rows, cols, fmt, case["transpose"], stream)
            lib.mx_unquantize(codes.data_ptr(), scales.data_ptr(), kept.data_ptr(), lib.F32, m, m, n, fmt, stream)
            return kept
        function = {"relu": lib.ACT_RELU, "sigmoid": lib.ACT_SIGMOID, "tanh": lib.ACT_TANH, "gelu": lib.ACT_GELU, "silu": lib.ACT_SILU}[case["function"]]
        dy, y, dx, ld = state["dy"], state["y"], state["dx"], rows + case["pad"]
        lib.mx_act_forward(x.data_ptr(), dtype, ld, function, y.data_ptr(), ld, codes.data_ptr(), scales.data_ptr(), rows, cols, stream)
        lib.mx_act_backward(dy.data_ptr(), dtype, ld, codes.data_ptr(), scales.data_ptr(), function, dx.data_ptr(), ld, rows, cols, stream)
        lib.mx_unquantize(codes.data_ptr(), scales.data_ptr(), kept.data_ptr(), lib.F32, rows, rows, cols, lib.MXINT8, stream)
        return {"y": y, "kept": kept, "dx": dx}
    outputs, inputs, tokens, pad = case["outputs"], case["inputs"], case["tokens"], case["pad"]
    if kind == "times":
        (wc, ws), (xc, xs), y = state["w"], state["x"], state["y"]
        lib.mx_times(wc.data_ptr(), ws.data_ptr(), xc.data_ptr(), xs.data_ptr(), state["bias"].data_ptr(), y.data_ptr(), dtype, outputs + pad, outputs, tokens,
                     inputs, stream)
        return y
    if kind == "weight_grad":
        (xc, xs), dy, dw = state["x"], state["dy"], state["dw"]
        lib.mx_weight_grad(dy.data_ptr(), dtype, outputs + pad, xc.data_ptr(), xs.data_ptr(), fmt, dw.data_ptr(), outputs, inputs, tokens, False, stream)
        return dw
    (wc, ws), dy, dx = state["w"], state["dy"], state["dx"]
    lib.mx_input_grad(dy.data_ptr(), dtype, outputs + pad, wc.data_ptr(), ws.data_ptr(), fmt, dx.data_ptr(), dtype, inputs + pad, outputs, inputs, tokens, stream)
    return dx


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    kind, size = case["kind"], TYPES[case["type"]].itemsize
    if kind in ("quantize", "activation"):
        rows, cols = case["rows"], case["cols"]
        v = rows * cols
        m, n = (cols, rows) if case.get("transpose") else (rows, cols)
        packed = sum(_bytes(m, n, case.get("format", "int8")))
        if kind == "quantize":
            # the matrix in, the packed form out and in, the values out
            return {"bytes": v * (size + 4) + 2 * packed, "flops": 4 * v}
        # x and dy in, y and dx out, the packed form out once and in twice, the values out
        return {"bytes": v * (4 * size + 4) + 3 * packed, "flops": 30 * v}
    outputs, inputs, tokens = case["outputs"], case["inputs"], case["tokens"]
    flops = 2 * outputs * inputs * tokens
    if kind == "times":
        return {"bytes": sum(_bytes(inputs, outputs, "fp4")) + sum(_bytes(inputs, tokens, "fp4")) + 4 * outputs + size * outputs * tokens, "flops": flops}
    if kind == "weight_grad":
        return {"bytes": sum(_bytes(inputs, tokens, case["format"])) + size * outputs * tokens + 4 * outputs * inputs, "flops": flops}
    return {"bytes": sum(_bytes(inputs, outputs, "fp4")) + size * outputs * tokens + size * inputs * tokens, "flops": flops}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------


def _exact_power(e):
    """2**e as a double, put together from its exponent field."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_round_trip(x, fmt):
    """Element by element: the nearest of the format's values, a tie to the even code."""
    n, m = x.shape
    x = x.double()
    groups = torch.zeros(n, -(-m // 32) * 32, dtype=torch.float64, device=x.device)
    groups[:, :m] = x
    groups = groups.reshape(-1, 32)
    top = groups.abs().max(dim=1).values
    # floor(log2) by counting powers of two that do not exceed the magnitude
    power = torch.floor(torch.log2(top.clamp(min=2.0 ** -149)))
    power = power + (_exact_power(power + 1) <= top).double() - (_exact_power(power) > top).double()
    power = (power - (2 if fmt == "fp4" else 0)).clamp(min=-127)
    power = torch.where(top > 0, power, -127.0)
    unit = _exact_power(power)[:, None]
    if fmt == "fp4":
        levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
        a = groups.abs() / unit
        below = (torch.searchsorted(levels, a, right=True) - 1).clamp(0, 7)
        above = (below + 1).clamp(max=7)
        dl, du = a - levels[below], levels[above] - a
        up = (du < dl) | ((du == dl) & (below % 2 == 1))
        got = torch.where(up & (above > below), levels[above], levels[below]) * torch.sign(groups)
    else:
        levels = torch.arange(0, 128, dtype=torch.float64, device=x.device) / 64
        a = groups.abs() / unit
        below = torch.floor(a * 64).clamp(max=127)
        rest = a * 64 - below
        up = ((rest > 0.5) | ((rest == 0.5) & (below % 2 == 1))) & (below < 127)
        got = levels[(below + up).long()] * torch.sign(groups)
    return (got * unit).reshape(n, -1)[:, :m]


def _exact_values(codes, scales, rows, fmt):
    n, b = codes.shape[0], -(-rows // 32)
    across = -(-b // 4)
    # undo the tiling: [128 columns, 4 blocks][column % 32][column // 32 % 4][block % 4]
    s = scales.view(-(-n // 128), across, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-n // 128) * 128, across * 4)[:n, :b]
    unit = _exact_power(s.long() - 127).repeat_interleave(32, dim=1)
    if fmt == "int8":
        q = codes.long()
        el = torch.where(q >= 128, q - 256, q).double() / 64
    else:
        c = torch.empty(n, codes.shape[1] * 2, dtype=torch.int64, device=codes.device)
        c[:, 0::2], c[:, 1::2] = codes.long() % 16, codes.long() // 16
        k = c % 8
        # exponent and mantissa bit of the 4-bit element; exponent 0 has no leading one
        el = torch.where(k < 2, 0.5 * k, (1 + 0.5 * (k % 2)) * _exact_power(k // 2 - 1)) * torch.where(c >= 8, -1.0, 1.0).double()
    return (el * unit)[:, :rows]


def _exact_function(x, name):
    if name == "relu":
        return torch.where(x > 0, x, 0.0), torch.where(x > 0, 1.0, 0.0).double()
    if name == "tanh":
        return torch.tanh(x), 1 - torch.tanh(x) ** 2
    if name == "gelu":
        c = 0.5 * torch.erfc(-x / math.sqrt(2.0))
        return x * c, c + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    s = torch.special.expit(x)
    if name == "sigmoid":
        return s, s * torch.special.expit(-x)
    return x * s, s + x * s * torch.special.expit(-x)


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        return _exact_round_trip(state["x"].t() if case["transpose"] else state["x"], case["format"])
    if kind == "activation":
        kept = _exact_round_trip(state["x"], "int8")
        return {"y": _exact_function(state["x"].double(), case["function"])[0], "kept": kept,
                "dx": state["dy"].double() * _exact_function(kept, case["function"])[1]}
    if kind == "weight_grad":
        return _exact_values(*state["x"], case["inputs"], case["format"]).t() @ state["dy"].double()
    w = _exact_values(*state["w"], case["inputs"], "fp4")
    if kind == "times":
        return _exact_values(*state["x"], case["inputs"], "fp4") @ w.t() + state["bias"].double()
    return state["dy"].double() @ w
