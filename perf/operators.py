"""Performance cases of the operators around a quantized linear layer.

A transformer's block on top of this library is a chain of mmt4d products with
row-wise steps in between. Three operators make up what lies between two
products and what a product does with its sums:

  norm     h = x + residual; y = h / sqrt(mean(h^2) + epsilon) * weight, row by
           row, brought into the tiles [M1][K1][M0][K0] of the next product's
           left-hand side: as 8-bit integers or 8-bit floats with a scale per
           row, or in the input's own type.
  gate     y = activation(gate) * up, the same way into the same tiles (without
           `up`: y = activation(gate), without an activation either: x itself,
           quantized as it is packed).
  product  out = residual + activation(lhs * rhs^T * row_scale * col_scale +
           bias), from tiles into a row-major matrix of f32, f16 or bf16.

Each case is one call as a program makes it, on operands in device memory.
`listed()` holds one case for each part of the range, `draw()` picks others from
the same ranges. `run` makes the library's calls where `own` is true, and
computes the plain form in 32-bit floats where it is false; `exact` is the
definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_FLOATS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_TYPES = {**_FLOATS, "s8": torch.int8, "f8": torch.float8_e4m3fn}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "s8": 1, "f8": 1}
_LARGEST = {"s8": 127.0, "f8": 448.0}
EPSILON = 1e-5


def listed():
    return [
        # Decoding of one sequence: the norm in front of a quantized projection, rows as they are (M0 = 1).
        dict(name="norm_token_s8", kind="norm", tin="bf16", tout="s8", rows=1, cols=4096, m0=1, k0=16, residual=True),
        # Decoding of a batch of 16 into the tiles of the decode-shaped quantized layer.
        dict(name="norm_batch_s8", kind="norm", tin="bf16", tout="s8", rows=16, cols=4096, m0=32, k0=8, residual=True),
        # Nothing divides anything; unquantized, for a product in 16-bit floats.
        dict(name="norm_ragged_f16", kind="norm", tin="f16", tout="f16", rows=1000, cols=4097, m0=16, k0=16,
             residual=False),
        # A long prompt in 8-bit floats.
        dict(name="norm_prompt_f8", kind="norm", tin="bf16", tout="f8", rows=2048, cols=8192, m0=16, k0=32,
             residual=True),
        # Decoding: the hidden layer of a batch of 16, gate and up as the halves of one matrix.
        dict(name="gate_batch_s8", kind="gate", tin="bf16", tout="s8", rows=16, cols=14336, m0=32, k0=8, act="silu",
             up=True),
        # A single matrix of f32 through a GELU, odd sizes.
        dict(name="gate_ragged_f32", kind="gate", tin="f32", tout="f8", rows=777, cols=1501, m0=16, k0=16, act="gelu",
             up=False),
        # The hidden layer of a long prompt.
        dict(name="gate_prompt_f8", kind="gate", tin="bf16", tout="f8", rows=2048, cols=28672, m0=16, k0=32, act="silu",
             up=True),
        # Decoding of one sequence: the down projection onto the residual stream.
        dict(name="product_token_f8", kind="product", dtype="f8", tout="bf16", m=1, n=4096, k=14336, m0=1, n0=16, k0=32,
             act="none", bias=False, residual=True),
        # The decode-shaped quantized layer for a batch of 16.
        dict(name="product_batch_s8", kind="product", dtype="s8", tout="bf16", m=16, n=14336, k=4096, m0=32, n0=16,
             k0=8, act="silu", bias=True, residual=False),
        # bf16, nothing divides anything, everything the epilogue has.
        dict(name="product_ragged_bf16", kind="product", dtype="bf16", tout="bf16", m=1000, n=1501, k=777, m0=16, n0=16,
             k0=8, act="gelu", bias=True, residual=True),
        # A square product of the benchmark's chain with bias and GELU.
        dict(name="product_4096_f16", kind="product", dtype="f16", tout="f16", m=4096, n=4096, k=4096, m0=16, n0=16,
             k0=16, act="gelu_tanh", bias=True, residual=False),
        # The largest: the down projection of a long prompt.
        dict(name="product_prompt_f8", kind="product", dtype="f8", tout="bf16", m=2048, n=8192, k=28672, m0=16, n0=16,
             k0=32, act="none", bias=False, residual=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_TILES = {"s8": [(1, 16, 16), (16, 16, 16), (32, 16, 8)], "f8": [(1, 16, 32), (16, 16, 32), (16, 16, 16)],
          "f16": [(1, 16, 8), (16, 16, 8), (16, 16, 16)], "bf16": [(1, 16, 8), (16, 16, 8), (16, 16, 16)],
          "f32": [(16, 16, 4), (16, 16, 1)]}
_ACTIVATIONS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def draw(rng):
    kind = rng.choice(["norm", "gate", "product"])
    if kind == "product":
        dtype = rng.choice(["s8", "f8", "f16", "bf16"])
        m0, n0, k0 = rng.choice(_TILES[dtype])
        m, n, k = _log_int(rng, 1, 2048), _log_int(rng, 64, 28672), _log_int(rng, 64, 28672)
        while float(m) * n * k > 2e11:
            n, k = max(64, n * 3 // 4), max(64, k * 3 // 4)
        return dict(kind=kind, dtype=dtype, tout=rng.choice(["f32", "f16", "bf16", "bf16"]), m=m, n=n, k=k, m0=m0, n0=n0,
                    k0=k0, act=rng.choice(_ACTIVATIONS), bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    tin = rng.choice(["f32", "f16", "bf16", "bf16"])
    tout = rng.choice(["s8", "f8", tin])
    m0, _, k0 = rng.choice(_TILES[tout])
    rows, cols = _log_int(rng, 1, 2048), _log_int(rng, 64, 8192 if kind == "norm" else 28672)
    case = dict(kind=kind, tin=tin, tout=tout, rows=rows, cols=cols, m0=m0, k0=k0)
    if kind == "norm":
        return dict(case, residual=rng.random() < 0.5)
    up = rng.random() < 0.7
    return dict(case, act=rng.choice(_ACTIVATIONS), up=up)


# ------------------------------------------------------------------- inputs
def _ceil(a, b):
    return -(-a // b)


def _channels(rows, cols, gen):
    """Activations as a trained network has them: channels of different widths."""
    t = torch.randn((rows, cols), generator=gen, device="cuda")
    return t * torch.exp(0.5 * torch.randn(cols, generator=gen, device="cuda"))


def _random_tiles(t1, k1, t0, k0, rows, k, dtype, weights, gen):
    """A random rows x k operand in tiles, zeros where tiles reach beyond it."""
    t = torch.randn((t1 * t0, k1 * k0), generator=gen, device="cuda")
    if dtype == "s8":
        t = t.mul_(40.0).round_().clamp_(-127, 127)
    elif dtype == "f8":
        t = t.mul_(100.0).clamp_(-448, 448)
    elif weights:
        t = t.mul_(1.0 / math.sqrt(k))
    t[rows:] = 0
    t[:, k:] = 0
    return t.to(_TYPES[dtype]).view(torch.uint8).view(t1, t0, k1, -1).transpose(1, 2).contiguous().view(_TYPES[dtype])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = dict(case=case)
    if case["kind"] == "product":
        m, n, k, m0, n0, k0 = (case[x] for x in ("m", "n", "k", "m0", "n0", "k0"))
        m1, n1, k1 = _ceil(m, m0), _ceil(n, n0), _ceil(k, k0)
        tout = _FLOATS[case["tout"]]
        state["lhs"] = _random_tiles(m1, k1, m0, k0, m, k, case["dtype"], False, gen)
        state["rhs"] = _random_tiles(n1, k1, n0, k0, n, k, case["dtype"], True, gen)
        width = {"s8": 40.0, "f8": 100.0}.get(case["dtype"])
        state["row_scale"] = state["col_scale"] = state["bias"] = state["residual"] = None
        if width:
            state["row_scale"] = (0.5 + torch.rand(m, generator=gen, device="cuda")) / width
            state["col_scale"] = (0.5 + torch.rand(n, generator=gen, device="cuda")) / (width * math.sqrt(k))
        if case["bias"]:
            state["bias"] = 0.5 * torch.randn(n, generator=gen, device="cuda")
        if case["residual"]:
            state["residual"] = (2.0 * _channels(m, n, gen)).to(tout)
        state["out"] = torch.empty((m, n), dtype=tout, device="cuda")
        return state
    rows, cols, m0, k0 = (case[x] for x in ("rows", "cols", "m0", "k0"))
    tin, tout = _FLOATS[case["tin"]], _TYPES[case["tout"]]
    state["tiles"] = torch.empty((_ceil(rows, m0), _ceil(cols, k0), m0, k0), dtype=tout, device="cuda")
    state["scale"] = torch.empty(rows, device="cuda") if case["tout"] in _LARGEST else None
    if case["kind"] == "norm":
        state["x"] = _channels(rows, cols, gen).to(tin)
        state["weight"] = (1.0 + 0.1 * torch.randn(cols, generator=gen, device="cuda")).to(tin)
        state["residual"] = state["sum"] = None
        if case["residual"]:
            state["residual"] = (2.0 * _channels(rows, cols, gen)).to(tin)
            state["sum"] = torch.empty((rows, cols), dtype=tin, device="cuda")
    else:  # gate and up as the product in front leaves them: two halves of one matrix
        both = _channels(rows, cols * (2 if case["up"] else 1), gen).to(tin)
        state["gate"] = both[:, :cols]
        state["up"] = both[:, cols:] if case["up"] else None
    return state


# ---------------------------------------------------------- the library's calls
_library = None


def _own_calls():
    """The library and its flags, set up as a serving program does once: device operands, torch's stream."""
    global _library
    if _library is None:
        from iree_amd import ukernel as uk
        lib = uk.load()
        lib.set_stream(torch.cuda.current_stream().cuda_stream)
        lib.set_pointer_mode(uk.POINTER_MODE_DEVICE)
        _library = (lib, {
            "in": {"f32": uk.IN_TYPE_F32, "f16": uk.IN_TYPE_F16, "bf16": uk.IN_TYPE_BF16},
            "out": {"f32": uk.OUT_TYPE_F32, "f16": uk.OUT_TYPE_F16, "bf16": uk.OUT_TYPE_BF16, "s8": uk.OUT_TYPE_S8,
                    "f8": uk.OUT_TYPE_F8E4M3FN},
            "act": {"none": uk.ACTIVATION_NONE, "relu": uk.ACTIVATION_RELU, "gelu": uk.ACTIVATION_GELU,
                    "gelu_tanh": uk.ACTIVATION_GELU_TANH, "silu": uk.ACTIVATION_SILU},
            "product": {"s8": uk.MMT4D_TYPE_S8S8S32, "f8": uk.MMT4D_TYPE_F8E4M3FNF8E4M3FNF32,
                        "f16": uk.MMT4D_TYPE_F16F16F32, "bf16": uk.MMT4D_TYPE_BF16BF16F32}})
    return _library


def _at(t):
    return None if t is None else t.data_ptr()


def _run_own(state):
    lib, flags = _own_calls()
    case = state["case"]
    if case["kind"] == "product":
        lhs, rhs, out, residual = (state[x] for x in ("lhs", "rhs", "out", "residual"))
        lib.mmt4d_epilogue_unpack(
            lhs.data_ptr(), 0, lhs.stride(0), rhs.data_ptr(), 0, rhs.stride(0), _at(residual), 0, case["n"],
            out.data_ptr(), 0, case["n"], case["m"], case["n"], _at(state["row_scale"]), _at(state["col_scale"]),
            _at(state["bias"]), lhs.shape[0], rhs.shape[0], lhs.shape[1], case["m0"], case["n0"], case["k0"],
            flags["product"][case["dtype"]], flags["out"][case["tout"]] | flags["act"][case["act"]])
        return out
    rows, cols, tiles, scale = case["rows"], case["cols"], state["tiles"], state["scale"]
    types = flags["in"][case["tin"]] | flags["out"][case["tout"]]
    into = (tiles.data_ptr(), 0, tiles.stride(0), _at(scale), rows, cols, *tiles.shape)
    if case["kind"] == "norm":
        lib.rmsnorm_pack(state["x"].data_ptr(), 0, cols, _at(state["residual"]), 0, cols, _at(state["sum"]), 0, cols,
                         state["weight"].data_ptr(), EPSILON, *into, types)
    else:
        gate, up = state["gate"], state["up"]
        lib.gate_pack(gate.data_ptr(), 0, gate.stride(0), _at(up), 0, gate.stride(0), *into,
                      types | flags["act"][case["act"]])
    return _outputs(tiles, scale, state.get("sum"))


def _outputs(tiles, scale, added):
    """What a call writes; 8-bit integers as the numbers that they stand for beside their scales, all of which
    bfloat16 holds exactly."""
    tiles = tiles.to(torch.bfloat16) if tiles.dtype == torch.int8 else tiles
    return {key: t for key, t in (("tiles", tiles), ("scale", scale), ("sum", added)) if t is not None}


# ---------------------------------------------------------------- the plain form
def _activation(x, act):
    if act == "relu":
        return torch.where(x < 0, torch.zeros_like(x), x)
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return x


def _into_tiles(y, state):
    case, m1, k1 = state["case"], *state["tiles"].shape[:2]
    full = y.new_zeros((m1 * case["m0"], k1 * case["k0"]))
    full[:case["rows"], :case["cols"]] = y
    return full.view(m1, case["m0"], k1, case["k0"]).transpose(1, 2).contiguous()


def _quantize(y, tout):
    largest = _LARGEST[tout]
    scale = y.abs().amax(dim=1) / largest
    q = (y / scale[:, None]).clamp(-largest, largest)
    return q.round() if tout == "s8" else q, scale


def _rows_plain(state):
    case = state["case"]
    added = None
    if case["kind"] == "norm":
        h = state["x"].float()
        if case["residual"]:
            h = h + state["residual"].float()
            added = h.to(_FLOATS[case["tin"]])
        y = h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPSILON) * state["weight"].float()
    else:
        y = _activation(state["gate"].float(), case["act"])
        if case["up"]:
            y = y * state["up"].float()
    scale = None
    if case["tout"] in _LARGEST:
        y, scale = _quantize(y, case["tout"])
    return _outputs(_into_tiles(y, state).to(_TYPES[case["tout"]]), scale, added)


def _matrix(tiles, rows, k):
    t1, k1, t0, k0 = tiles.shape
    return tiles.float().transpose(1, 2).reshape(t1 * t0, k1 * k0)[:rows, :k]


def _product_plain(state):
    case = state["case"]
    y = _matrix(state["lhs"], case["m"], case["k"]) @ _matrix(state["rhs"], case["n"], case["k"]).T
    if state["row_scale"] is not None:
        y = y * state["row_scale"][:, None] * state["col_scale"]
    if case["bias"]:
        y = y + state["bias"]
    y = _activation(y, case["act"])
    if case["residual"]:
        y = y + state["residual"].float()
    return y.to(_FLOATS[case["tout"]])


def run(state):
    if own:
        return _run_own(state)
    return _product_plain(state) if state["case"]["kind"] == "product" else _rows_plain(state)


# ------------------------------------------------------------------ the definition
def _curve(x, act):
    """The activations in the numbers' own type, written by their integrals and sigmoids."""
    if act == "relu":
        return x.clamp(min=0)
    if act == "silu":
        return x * torch.sigmoid(x)
    if act == "gelu":
        return x * torch.special.ndtr(x)
    if act == "gelu_tanh":
        return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))
    return x


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "product":
        def rows_of(t, rows):  # [T1][K1][T0][K0] -> the rows x k matrix in 64 bits
            return torch.cat([t[:, j].double() for j in range(t.shape[1])], dim=2).flatten(0, 1)[:rows, :case["k"]]
        z = torch.matmul(rows_of(state["lhs"], case["m"]), rows_of(state["rhs"], case["n"]).t())
        if state["row_scale"] is not None:
            z *= torch.outer(state["row_scale"].double(), state["col_scale"].double())
        if case["bias"]:
            z += state["bias"].double()
        z = _curve(z, case["act"])
        return z + state["residual"].double() if case["residual"] else z
    rows, cols, m0, k0 = (case[x] for x in ("rows", "cols", "m0", "k0"))
    result = {}
    if case["kind"] == "norm":
        z = state["x"].double()
        if case["residual"]:
            z += state["residual"].double()
            result["sum"] = z.clone()
        rms = (torch.linalg.vector_norm(z, dim=1) ** 2 / cols + EPSILON).sqrt()
        z = torch.einsum("rc,r,c->rc", z, 1 / rms, state["weight"].double())
    else:
        z = _curve(state["gate"].double(), case["act"])
        if case["up"]:
            z *= state["up"].double()
    if case["tout"] in _LARGEST:
        largest = _LARGEST[case["tout"]]
        top = z.abs().max(dim=1).values
        result["scale"] = top / largest
        z = z * (largest / top)[:, None]
        if case["tout"] == "s8":
            z = torch.round(z)
        else:  # three fraction bits, down to steps of 2^-9
            step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
            z = (torch.round(z / step) * step).clamp(-largest, largest)
    m1, k1 = _ceil(rows, m0), _ceil(cols, k0)
    z = torch.nn.functional.pad(z, (0, k1 * k0 - cols, 0, m1 * m0 - rows))
    result["tiles"] = z.unflatten(0, (m1, m0)).unflatten(2, (k1, k0)).permute(0, 2, 1, 3).contiguous()
    return result


def work(case):
    """Every input read once and every output written once; two operations for each product and sum of a matrix
    product, about ten for each element of a row-wise step."""
    if case["kind"] == "product":
        m, n, k, out = case["m"], case["n"], case["k"], _BYTES[case["tout"]]
        scales = 4 * (m + n) if case["dtype"] in _LARGEST else 0
        return {"bytes": (m + n) * k * _BYTES[case["dtype"]] + scales + (4 * n if case["bias"] else 0)
                + m * n * out * (2 if case["residual"] else 1), "flops": 2.0 * m * n * k}
    rows, cols, tin = case["rows"], case["cols"], _BYTES[case["tin"]]
    tiles = _ceil(rows, case["m0"]) * case["m0"] * _ceil(cols, case["k0"]) * case["k0"] * _BYTES[case["tout"]]
    streams = (3 if case["residual"] else 1) if case["kind"] == "norm" else (2 if case["up"] else 1)
    once = (cols * tin if case["kind"] == "norm" else 0) + (4 * rows if case["tout"] in _LARGEST else 0)
    return {"bytes": rows * cols * tin * streams + tiles + once, "flops": 10.0 * rows * cols}
