"""Cases of the block-scaled 8-bit operators: encode, root-mean-square norm, matrix product.

Storage: a matrix of 8-bit codes (E4M3 or E5M2) with one FP32 scale for each
block of 128 columns, of one row (activations) or of 128 rows (weights).  The
scale of row group R and column block b stands at scales[b, R].  A value is
its code's value times its block's scale.

encode   scale = max(largest finite |x| of the block / F, 2^-126), F the
         largest code value (448 or 57344); code = x / scale rounded to the
         nearest code, ties to even; what is not finite becomes the NaN code.
norm     h = x + residual; y = h / sqrt(mean(h^2) + eps) * weight; y encoded
         by rows as above; h goes back rounded to the type of x.
product  out[i, j] = sum over the blocks b of 128 of k:
         a_scale[b, i] * b_scale[b, j / 128] * sum_{c in b} a[i, c] * b[j, c].
"""
import math

import torch

own = False

EPS = 1e-5
BLOCK = 128
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
TYPE_ID = {"fp32": 0, "bf16": 1, "fp16": 2}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
CODES = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
CODE_ID = {"e4m3": 0, "e5m2": 1}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}


def _blocks(n):
    return -(-n // BLOCK)


def _stride(columns):
    """Row stride of a code matrix: whole 16-byte lines."""
    return -(-columns // 16) * 16


def encode(name, rows, columns, type, code, block_rows):
    return {"name": name, "op": "encode", "rows": rows, "columns": columns, "type": type,
            "code": code, "block_rows": block_rows}


def norm(name, rows, columns, type, code, residual):
    return {"name": name, "op": "norm", "rows": rows, "columns": columns, "type": type,
            "code": code, "residual": residual}


def product(name, m, n, k, type, a_code, b_code):
    return {"name": name, "op": "product", "m": m, "n": n, "k": k, "type": type,
            "a_code": a_code, "b_code": b_code}


def listed():
    return [
        # a few tokens' activations between two products of a decoding step
        encode("encode 4x8192 bf16", 4, 8192, "bf16", "e4m3", 1),
        # a prompt's activations
        encode("encode 4096x8192 bf16", 4096, 8192, "bf16", "e4m3", 1),
        # a weight matrix laid out once from FP32, odd sizes
        encode("encode weight 8191x5001 fp32", 8191, 5001, "fp32", "e4m3", 128),
        # one token of a decoding step
        norm("norm 1x4096 bf16", 1, 4096, "bf16", "e4m3", True),
        # a prompt
        norm("norm 4096x8192 bf16", 4096, 8192, "bf16", "e4m3", True),
        # first layer, no residual, a ragged batch of odd width, wide range codes
        norm("norm 777x5001 fp16", 777, 5001, "fp16", "e5m2", False),
        # one token: the weights are read once
        product("product 1x4096x4096", 1, 4096, 4096, "bf16", "e4m3", "e4m3"),
        # a small batch of single tokens on a large layer
        product("product 8x8192x8192", 8, 8192, 8192, "bf16", "e4m3", "e4m3"),
        # a batch of single tokens
        product("product 64x4096x16384", 64, 4096, 16384, "bf16", "e4m3", "e4m3"),
        # odd sizes, FP32 out, gradients' codes against weights
        product("product 333x1000x1999 fp32", 333, 1000, 1999, "fp32", "e5m2", "e4m3"),
        # a short prompt
        product("product 512x8192x4096", 512, 8192, 4096, "bf16", "e4m3", "e4m3"),
        # a long prompt
        product("product 4096x8192x8192", 4096, 8192, 8192, "bf16", "e4m3", "e4m3"),
    ]


def _log(rng, low, high):
    n = int(math.exp(rng.uniform(math.log(low), math.log(high))))
    return min(high, max(low, n if rng.random() < 0.4 else -(-n // 16) * 16))


def draw(rng):
    op = rng.choice(["encode", "norm", "product", "product"])
    type = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    code = rng.choice(["e4m3", "e4m3", "e4m3", "e5m2"])
    if op == "product":
        m, n, k = _log(rng, 1, 4096), _log(rng, 64, 8192), _log(rng, 64, 8192)
        case = product("", m, n, k, type, code, rng.choice(["e4m3", "e4m3", "e5m2"]))
    elif op == "norm":
        rows, columns = _log(rng, 1, 4096), _log(rng, 64, 8192)
        case = norm("", rows, columns, type, code, rng.random() < 0.75)
    else:
        block_rows = rng.choice([1, 1, 128])
        rows, columns = _log(rng, 1 if block_rows == 1 else 64, 4096), _log(rng, 64, 8192)
        case = encode("", rows, columns, type, code, block_rows)
    del case["name"]
    return case


def _values(g, rows, columns, spread):
    """Normal values, some columns (channels) of them far larger than the rest."""
    v = torch.randn(rows, columns, generator=g, device="cuda")
    gain = torch.exp(spread * torch.randn(columns, generator=g, device="cuda"))
    return v * gain


def _buffers(rows, columns, code, block_rows):
    codes = torch.zeros(rows, _stride(columns), dtype=torch.uint8, device="cuda")
    scales = torch.zeros(_blocks(columns), -(-rows // block_rows), device="cuda")
    return codes, scales


def _operand(g, rows, columns, code, block_rows, gain):
    """Codes and scales that a program has in hand before a product."""
    v = _values(g, rows, columns, 0.5) * gain
    if block_rows == 1 and rows >= 16:
        v[rows - rows // 16:] = 0  # places of a batch that hold no token
    codes, scales = _buffers(rows, columns, code, block_rows)
    c, s = _encode(v, code, block_rows)
    codes[:, :columns] = c.view(torch.uint8)
    scales.copy_(s)
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = {"case": case}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        state["a"], state["a_scales"] = _operand(g, m, k, case["a_code"], 1, 1.0)
        state["b"], state["b_scales"] = _operand(g, n, k, case["b_code"], BLOCK, 0.02)
        state["out"] = torch.zeros(m, n, dtype=TYPES[case["type"]], device="cuda")
        return state
    rows, columns, type = case["rows"], case["columns"], TYPES[case["type"]]
    weights = case["op"] == "encode" and case["block_rows"] == BLOCK
    v = _values(g, rows, columns, 0.5 if not weights else 0.1) * (0.02 if weights else 1.0)
    if not weights and rows >= 16:
        v[rows - rows // 16:] = 0  # places of a batch that hold no token
    state["x"] = v.to(type)
    state["codes"], state["scales"] = _buffers(rows, columns, case["code"],
                                               case.get("block_rows", 1))
    if case["op"] == "norm":
        state["weight"] = (1 + 0.1 * torch.randn(columns, generator=g, device="cuda")).to(type)
        if case["residual"]:
            state["residual"] = _values(g, rows, columns, 0.5).to(type)
            state["stream"] = torch.zeros_like(state["residual"])
    return state


# ---- the plain forms --------------------------------------------------------

def _encode(v, code, block_rows):
    rows, columns = v.shape
    nb, nr = _blocks(columns), -(-rows // block_rows)
    x = torch.nn.functional.pad(v, (0, nb * BLOCK - columns, 0, nr * block_rows - rows))
    x = x.view(nr, block_rows, nb, BLOCK)
    fine = torch.isfinite(x)
    largest = torch.where(fine, x.abs(), 0.0).amax(dim=(1, 3))
    scale = (largest / LARGEST[code]).clamp_min(2.0 ** -126)
    q = (x / scale[:, None, :, None]).clamp(-LARGEST[code], LARGEST[code])
    q = torch.where(fine, q, float("nan"))
    q = q.view(nr * block_rows, nb * BLOCK)[:rows, :columns].contiguous()
    return q.to(CODES[code]), scale.t().contiguous()


def _plain(state):
    case = state["case"]
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a = state["a"][:, :k].contiguous().view(CODES[case["a_code"]]).float()
        b = state["b"][:, :k].contiguous().view(CODES[case["b_code"]]).float()
        a = a * state["a_scales"].t().repeat_interleave(BLOCK, 1)[:, :k]
        bs = state["b_scales"].t().repeat_interleave(BLOCK, 0)[:n]
        b = b * bs.repeat_interleave(BLOCK, 1)[:, :k]
        return (a @ b.t()).to(TYPES[case["type"]])
    x = state["x"].float()
    if case["op"] == "encode":
        return _encode(x, case["code"], case["block_rows"])
    stream = None
    if case["residual"]:
        x = x + state["residual"].float()
        stream = x.to(TYPES[case["type"]])
    y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * state["weight"].float()
    codes, scales = _encode(y, case["code"], 1)
    return (codes, scales) if stream is None else (codes, scales, stream)


# ---- the framework's calls --------------------------------------------------

_workspace = None


def _own(state):
    global _workspace
    if _workspace is None:
        from accessor_universal_test_b200 import Workspace
        _workspace = Workspace(0)
    case, stream = state["case"], torch.cuda.current_stream().cuda_stream
    if case["op"] == "product":
        a, b, out = state["a"], state["b"], state["out"]
        _workspace.gemm_scaled(
            CODE_ID[case["a_code"]], CODE_ID[case["b_code"]], TYPE_ID[case["type"]],
            a.data_ptr(), a.stride(0), state["a_scales"].data_ptr(), state["a_scales"].stride(0),
            b.data_ptr(), b.stride(0), state["b_scales"].data_ptr(), state["b_scales"].stride(0),
            case["m"], case["n"], case["k"], out.data_ptr(), out.stride(0), stream)
        return out
    x, codes, scales = state["x"], state["codes"], state["scales"]
    rows, columns = x.shape
    values = codes.view(CODES[case["code"]])[:, :columns]
    if case["op"] == "encode":
        _workspace.encode_scaled(
            CODE_ID[case["code"]], TYPE_ID[case["type"]], case["block_rows"],
            x.data_ptr(), x.stride(0), rows, columns, codes.data_ptr(), codes.stride(0),
            scales.data_ptr(), scales.stride(0), stream)
        return values, scales
    residual, after = state.get("residual"), state.get("stream")
    _workspace.rms_norm_scaled(
        CODE_ID[case["code"]], TYPE_ID[case["type"]], x.data_ptr(), x.stride(0),
        0 if residual is None else residual.data_ptr(), 0 if after is None else after.data_ptr(),
        0 if residual is None else residual.stride(0), state["weight"].data_ptr(), EPS,
        rows, columns, codes.data_ptr(), codes.stride(0), scales.data_ptr(), scales.stride(0),
        stream)
    return (values, scales) if residual is None else (values, scales, after)


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        scales = 4 * _blocks(k) * (m + _blocks(n))
        return {"bytes": m * k + n * k + scales + m * n * SIZE[case["type"]],
                "flops": 2 * m * n * k}
    rows, columns = case["rows"], case["columns"]
    scales = 4 * _blocks(columns) * -(-rows // case.get("block_rows", 1))
    size = SIZE[case["type"]]
    if case["op"] == "encode":
        return {"bytes": rows * columns * (size + 1) + scales, "flops": 3 * rows * columns}
    streams = 3 if case["residual"] else 1
    return {"bytes": rows * columns * (streams * size + 1) + columns * size + scales,
            "flops": 7 * rows * columns}


# ---- the definitions in 64 bits ---------------------------------------------

def _by_definition(x, code, block_rows):
    """Codes' values and scales of a matrix in 64 bits, a column block at a time."""
    rows, columns = x.shape
    top = LARGEST[code]
    low = -6 if code == "e4m3" else -14  # exponent of the smallest normal code
    digits = 3 if code == "e4m3" else 2
    values = torch.empty_like(x)
    scales = []
    group = torch.arange(rows, device=x.device) // block_rows
    for first in range(0, columns, BLOCK):
        part = x[:, first:first + BLOCK]
        size = part.abs()
        size[~torch.isfinite(part)] = 0
        by_row = size.max(1).values
        by_group = torch.zeros(int(group[-1]) + 1, dtype=x.dtype, device=x.device)
        by_group.scatter_reduce_(0, group, by_row, "amax")
        s = torch.maximum(by_group / top, torch.full_like(by_group, 2.0 ** -126))
        scales.append(s)
        q = part / s[group].unsqueeze(1)
        step = torch.frexp(q).exponent.sub(1).clamp_min(low).sub(digits)
        q = torch.ldexp(torch.round(torch.ldexp(q, -step)), step)  # ties to even
        values[:, first:first + BLOCK] = torch.where(
            torch.isfinite(part), torch.minimum(torch.maximum(q, -top + 0 * q), top + 0 * q),
            float("nan"))
    return values, torch.stack(scales)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        out = torch.zeros(m, n, dtype=torch.float64, device="cuda")
        row_group = torch.arange(n, device="cuda") // BLOCK
        for b in range(_blocks(k)):
            c = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
            left = state["a"][:, c].contiguous().view(CODES[case["a_code"]]).double()
            right = state["b"][:, c].contiguous().view(CODES[case["b_code"]]).double()
            left *= state["a_scales"][b].double().unsqueeze(1)
            right *= state["b_scales"][b].double()[row_group].unsqueeze(1)
            out += left.mm(right.t())
        return out
    x = state["x"].double()
    if case["op"] == "encode":
        return _by_definition(x, case["code"], case["block_rows"])
    if case["residual"]:
        x = x + state["residual"].double()
    mean = torch.sum(x ** 2, 1) / case["columns"]
    y = x / torch.sqrt(mean + EPS).unsqueeze(1) * state["weight"].double()
    values, scales = _by_definition(y, case["code"], 1)
    return (values, scales, x) if case["residual"] else (values, scales)
