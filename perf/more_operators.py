"""Performance cases: a layer's products with 8-bit operands on one GPU.

The program holds its tensors in torch and calls the C ABI through
``tensorcx_hip_capi`` with plain pointers, descriptors and one scratch buffer
that it keeps, on torch's current stream:

``quantise``  float32 rows held in 8-bit floating point with a power of two for
              each 128 features, and what they stand for read back
``norm``      a residual added, the root-mean-square norm of the sum, and its
              output in that form
``linear``    the product of activations and weights in that form, with bias and
              activation, as float32
``gated``     the products with gate and up weights, the activated gate times the
              other, and the result in that form

A case is a dict of plain values; ``kind`` picks the path. Where ``own`` is
false, ``run`` computes the same in elementary torch operations.
"""

from __future__ import annotations

import math
import pathlib
import sys

import torch

own = False

BLOCK = 128  # features that share a power of two
LOWEST = -100  # the least exponent of a block
EPSILON = 1e-5

# No drawn case does more than the largest listed ones.
MAX_BYTES = 9e8
MAX_FLOPS = 1.1e12
MAX_VALUES = 6e8  # float32 values of an operand or a result that the plain form holds


def listed():
    return [
        # One decoded token's hidden state: latency.
        {"name": "norm_token", "kind": "norm", "rows": 1, "features": 4096, "residual": True, "weight": True},
        # A batch of prompts, wide.
        {"name": "norm_prompt", "kind": "norm", "rows": 8192, "features": 8192, "residual": True, "weight": True},
        # A few rows whose last block is cut short.
        {"name": "quantise_odd", "kind": "quantise", "rows": 333, "features": 1100},
        # A layer's weights when they are loaded.
        {"name": "quantise_weights", "kind": "quantise", "rows": 11264, "features": 4096},
        # One token through a projection: latency and the weights' bytes.
        {"name": "linear_token", "kind": "linear", "rows": 1, "outputs": 4096, "features": 4096,
         "bias": False, "activation": "none"},
        # A step of 32 sequences through a layer's second, long product.
        {"name": "linear_step", "kind": "linear", "rows": 32, "outputs": 4096, "features": 11264,
         "bias": False, "activation": "none"},
        # Logits of eight sequences over a large vocabulary.
        {"name": "linear_logits", "kind": "linear", "rows": 8, "outputs": 128256, "features": 4096,
         "bias": False, "activation": "none"},
        # Sizes that fit no tile, with bias and activation.
        {"name": "linear_odd", "kind": "linear", "rows": 300, "outputs": 1100, "features": 1000,
         "bias": True, "activation": "gelu"},
        # A chunk of a prompt beside others' steps.
        {"name": "linear_chunk", "kind": "linear", "rows": 512, "outputs": 4096, "features": 4096,
         "bias": False, "activation": "none"},
        # Whole prompts through a wide square projection.
        {"name": "linear_prompt", "kind": "linear", "rows": 8192, "outputs": 8192, "features": 8192,
         "bias": True, "activation": "none"},
        # The first half of a gated layer: a step of 16 sequences, and a prompt.
        {"name": "gated_step", "kind": "gated", "rows": 16, "outputs": 11264, "features": 4096,
         "bias": False, "activation": "silu"},
        {"name": "gated_prompt", "kind": "gated", "rows": 4096, "outputs": 11264, "features": 4096,
         "bias": False, "activation": "silu"},
    ]


# ------------------------------------------------------------------ drawing
def _size(rng, low, high):
    """Spread over the logarithm of [low, high]; one in three a multiple of 128."""
    value = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.33 and value >= 192:
        value = (value + 64) // 128 * 128
    return max(low, min(high, value))


def _draw_rows(rng):
    if rng.random() < 0.4:
        return {"kind": "quantise", "rows": _size(rng, 1, 32768), "features": _size(rng, 1, 32768)}
    return {"kind": "norm", "rows": _size(rng, 1, 16384), "features": _size(rng, 1, 32768), "residual": rng.random() < 0.7,
            "weight": rng.random() < 0.8}


def _draw_product(rng):
    kind = rng.choice(["linear", "linear", "gated"])
    rows = rng.choice([1, _size(rng, 1, 16), _size(rng, 16, 256), _size(rng, 256, 8192), _size(rng, 256, 8192)])
    return {"kind": kind, "rows": rows, "outputs": _size(rng, 16, 131072 if kind == "linear" else 16384),
            "features": _size(rng, 64, 16384), "bias": rng.random() < 0.4,
            "activation": rng.choice(["none", "none", "silu", "gelu"] if kind == "linear" else ["silu", "silu", "gelu", "none"])}


def _held(case):
    """Values of the largest tensor that the plain form holds."""
    if "outputs" not in case:
        return case["rows"] * case["features"]
    n = case["outputs"] * (2 if case["kind"] == "gated" else 1)
    return max(case["rows"] * case["features"], n * case["features"], case["rows"] * n)


def draw(rng):
    """One more case of the listed kinds; sizes too large for one pass are drawn again."""
    pick = rng.choice([_draw_rows, _draw_product, _draw_product])
    while True:
        case = pick(rng)
        needs = work(case)
        if needs["bytes"] <= MAX_BYTES and needs["flops"] <= MAX_FLOPS and _held(case) <= MAX_VALUES:
            return case


# ------------------------------------------------------------------ sizes
def _blocks(features):
    return (features + BLOCK - 1) // BLOCK


def _row_bytes(features):
    """Bytes of a row in 8 bits: whole blocks of codes, and the exponents."""
    return _blocks(features) * (BLOCK + 1)


def work(case):
    """Bytes (each input read once, each output written once) and operations of one pass."""
    rows, features = case["rows"], case["features"]
    if case["kind"] == "quantise":  # float32 in, 8 bits out; and back
        return {"bytes": 2 * rows * (4 * features + _row_bytes(features)), "flops": 5 * rows * features}
    if case["kind"] == "norm":
        floats = 3 if case["residual"] else 1
        return {"bytes": rows * (4 * floats * features + _row_bytes(features)) + (4 * features if case["weight"] else 0),
                "flops": 8 * rows * features}
    n = case["outputs"] * (2 if case["kind"] == "gated" else 1)
    out = rows * _row_bytes(case["outputs"]) if case["kind"] == "gated" else 4 * rows * n
    return {"bytes": (rows + n) * _row_bytes(features) + out + (4 * n if case["bias"] else 0), "flops": 2 * rows * n * features}


# ------------------------------------------------------------------ the 8-bit form
def _quantise(x):
    """(rows, features) float32 to codes (rows, blocks * 128), float8_e4m3fn, and the exponents' bytes (rows,
    blocks). A block's exponent e is the least from -100 on with its largest value at most 448 * 2^e."""
    rows, features = x.shape
    blocks = _blocks(features)
    padded = torch.zeros((rows, blocks * BLOCK), dtype=torch.float32, device=x.device)
    padded[:, :features] = x
    g = padded.reshape(rows, blocks, BLOCK)
    bits = g.abs().amax(-1).view(torch.int32)
    exponent = torch.clamp(((bits + 0x1FFFFF) >> 23) - 127 - 8, min=LOWEST)  # 448 = 1.75 * 2^8
    codes = torch.ldexp(g, -exponent[..., None]).to(torch.float8_e4m3fn)
    return codes.reshape(rows, blocks * BLOCK), (exponent + 127).to(torch.uint8)


def _dequantise(codes, exponents, features):
    g = codes.to(torch.float32).reshape(codes.shape[0], -1, BLOCK)
    x = torch.ldexp(g, exponents.to(torch.int32)[..., None] - 127)
    return x.reshape(codes.shape)[:, :features]


def _words(codes, exponents):
    """The int32 words that hold codes and exponents: four bytes a word, the last word of exponents filled up."""
    rows, blocks = exponents.shape
    held = torch.zeros((rows, (blocks + 3) // 4 * 4), dtype=torch.uint8, device=codes.device)
    held[:, :blocks] = exponents
    return codes.view(torch.uint8).view(torch.int32), held.view(torch.int32)


def _views(codes, scales, features):
    """The values that the words stand for: codes and the blocks' powers of two."""
    return {"codes": codes.view(torch.float8_e4m3fn),
            "scales": scales.view(torch.uint8)[:, :_blocks(features)].view(torch.float8_e8m0fnu)}


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=generator, device="cuda") * scale

    def activations(rows, features):
        """Features of levels of their own, a few of them far larger, as hidden states have."""
        x = normal(rows, features) * torch.exp(normal(features, scale=0.5))
        x[:, ::601] *= 20.0
        return x

    kind, rows, features = case["kind"], case["rows"], case["features"]
    if kind == "quantise":
        return {"x": activations(rows, features) * features ** -0.5}
    if kind == "norm":
        t = {"x": normal(rows, features)}
        if case["residual"]:
            t["residual"] = activations(rows, features)
        if case["weight"]:
            t["weight"] = 1.0 + normal(features, scale=0.2)
        return t
    n = case["outputs"] * (2 if kind == "gated" else 1)
    t = {}
    t["x_codes"], t["x_scales"] = _words(*_quantise(activations(rows, features)))
    t["w_codes"], t["w_scales"] = _words(*_quantise(normal(n, features, scale=features ** -0.5)))
    if case["bias"]:
        t["bias"] = normal(n, scale=0.1)
    return t


def prepare(case, seed):
    """The inputs, and the outputs and the scratch memory that the program keeps."""
    t, kind, rows, features = _inputs(case, seed), case["kind"], case["rows"], case["features"]

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda")

    def empty8(width):
        blocks = _blocks(width)
        return empty(rows, blocks * BLOCK // 4, dtype=torch.int32), empty(rows, (blocks + 3) // 4, dtype=torch.int32)

    state = {"case": dict(case), "tensors": t, "plan": {}, "scratch": empty(32 << 20, dtype=torch.uint8), "out": {}}
    out = state["out"]
    if kind == "linear":
        out["values"] = empty(rows, case["outputs"])
        state["returned"] = out["values"]
        return state
    width = case["outputs"] if kind == "gated" else features
    out["codes"], out["scales"] = empty8(width)
    state["returned"] = _views(out["codes"], out["scales"], width)
    if kind == "quantise":
        out["values"] = state["returned"]["values"] = empty(rows, features)
    elif kind == "norm" and case["residual"]:
        out["sum"] = state["returned"]["sum"] = empty(rows, features)
    return state


# ------------------------------------------------------------------ the framework's operators
def _capi():
    path = str(pathlib.Path(__file__).resolve().parents[1] / "tensor.cx_amd" / "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tensorcx_hip_capi as capi
    return capi


def _own(state):
    case, t, plan, out = state["case"], state["tensors"], state["plan"], state["out"]
    kind, stream = case["kind"], torch.cuda.current_stream().cuda_stream
    if not plan:  # what the program keeps from call to call
        capi = plan["capi"] = _capi()
        plan["at"] = {name: x.data_ptr() for name, x in t.items()}
        plan["to"] = {name: x.data_ptr() for name, x in out.items()}
        if kind == "norm":
            plan["desc"] = capi.rmsnorm8_desc(case["rows"], case["features"], EPSILON)
        elif kind in ("linear", "gated"):
            plan["desc"] = capi.linear8_desc(case["rows"], case["features"], case["outputs"], bias=plan["at"].get("bias"),
                                             activation=case["activation"])
            # The scratch buffer, or one of the size that the library asks for where that is more.
            wanted = capi.linear8_workspace_bytes(plan["desc"], gated=kind == "gated")
            plan["scratch"] = state["scratch"] if wanted <= state["scratch"].numel() else torch.empty(
                wanted, dtype=torch.uint8, device="cuda")
            plan["workspace"] = capi.Workspace(plan["scratch"].data_ptr(), plan["scratch"].numel())
    capi, at, to = plan["capi"], plan["at"], plan["to"]
    if kind == "quantise":
        capi.quantise8(at["x"], to["codes"], to["scales"], case["rows"], case["features"], s=stream)
        capi.dequantise8(to["codes"], to["scales"], to["values"], case["rows"], case["features"], s=stream)
    elif kind == "norm":
        capi.rmsnorm8(at["x"], to["codes"], to["scales"], plan["desc"], residual=at.get("residual"), weight=at.get("weight"),
                      sum=to.get("sum"), s=stream)
    elif kind == "linear":
        capi.linear8(at["x_codes"], at["x_scales"], at["w_codes"], at["w_scales"], to["values"], plan["desc"],
                     workspace=plan["workspace"], s=stream)
    else:
        capi.gated_linear8(at["x_codes"], at["x_scales"], at["w_codes"], at["w_scales"], to["codes"], to["scales"], plan["desc"],
                           workspace=plan["workspace"], s=stream)
    return state["returned"]


# ------------------------------------------------------------------ the plain form
def _activate(x, name):
    if name == "silu":
        return x / (1.0 + torch.exp(-x))
    if name == "gelu":
        return 0.5 * x * (1.0 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    return x


def _product(case, t):
    blocks = _blocks(case["features"])
    x, w = (_dequantise(t[c].view(torch.float8_e4m3fn), t[s].view(torch.uint8)[:, :blocks], blocks * BLOCK)
            for c, s in (("x_codes", "x_scales"), ("w_codes", "w_scales")))
    y = torch.matmul(x, w.T)
    return y + t["bias"] if case["bias"] else y


def _eight(x):
    codes, exponents = _quantise(x)
    return {"codes": codes, "scales": exponents.view(torch.float8_e8m0fnu)}, exponents


def _plain(state):
    case, t = state["case"], state["tensors"]
    kind = case["kind"]
    if kind == "quantise":
        found, exponents = _eight(t["x"])
        return {**found, "values": _dequantise(found["codes"], exponents, case["features"])}
    if kind == "norm":
        x = t["x"] + t["residual"] if case["residual"] else t["x"]
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPSILON)
        found, _ = _eight(y * t["weight"] if case["weight"] else y)
        return {**found, "sum": x} if case["residual"] else found
    y = _product(case, t)
    if kind == "linear":
        return _activate(y, case["activation"])
    n = case["outputs"]
    return _eight(_activate(y[:, :n], case["activation"]) * y[:, n:])[0]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the results in 64 bits
def _values(words, scales, features):
    """What 8-bit rows stand for, from the format's fields: sign, four bits of exponent, three of mantissa."""
    code = words.contiguous().view(torch.uint8).to(torch.int32)
    field, mantissa = (code >> 3) & 15, (code & 7).double()
    size = torch.where(field == 0, mantissa / 512.0, (8.0 + mantissa) * torch.pow(2.0, (field - 10).double()))
    size = torch.where(code >= 128, -size, size)
    shift = scales.contiguous().view(torch.uint8).double() - 127.0
    blocks = code.shape[1] // BLOCK
    return size * torch.pow(2.0, shift[:, :blocks]).repeat_interleave(BLOCK, 1)


def _unrounded(x):
    """A row's values in units of their blocks' powers of two, before they are rounded to a code, and those powers."""
    width = _blocks(x.shape[1]) * BLOCK
    x = torch.nn.functional.pad(x, (0, width - x.shape[1])).reshape(x.shape[0], -1, BLOCK)
    top = x.abs().amax(-1, keepdim=True) / 448.0
    power = torch.where(top > 0, torch.ceil(torch.log2(torch.where(top > 0, top, 1.0))), float(LOWEST)).clamp(min=LOWEST)
    return (x * torch.pow(2.0, -power)).reshape(x.shape[0], width), torch.pow(2.0, power)[..., 0]


def _rounded(u):
    """Values up to 448 rounded to a code's: three bits behind the first, steps of 2^-9 at the least, ties to even."""
    step = torch.pow(2.0, (torch.frexp(u).exponent.double() - 1.0).clamp(min=-6.0) - 3.0)
    return torch.round(u / step) * step


def exact(case, seed):
    """In 64 bits. Computed outputs in 8 bits are given unrounded, without their blocks' powers: a block whose largest
    value is next to 448 of its units may take either of two. What is only quantised has one value."""
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "quantise":
        unrounded, power = _unrounded(t["x"].double())
        codes = _rounded(unrounded)
        return {"codes": codes, "scales": power, "values": (codes * power.repeat_interleave(BLOCK, 1))[:, :case["features"]]}
    if kind == "norm":
        x = t["x"].double()
        if case["residual"]:
            x = x + t["residual"].double()
        y = x / torch.sqrt(torch.square(x).sum(-1, keepdim=True) / case["features"] + EPSILON)
        found = {"codes": _unrounded(y * t["weight"].double() if case["weight"] else y)[0], "scales": None}
        return {**found, "sum": x} if case["residual"] else found
    act = {"none": lambda v: v, "silu": lambda v: v * torch.sigmoid(v),
           "gelu": lambda v: v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))}[case["activation"]]
    x, w = _values(t["x_codes"], t["x_scales"], case["features"]), _values(t["w_codes"], t["w_scales"], case["features"])
    y = x @ w.T
    if case["bias"]:
        y += t["bias"].double()
    if kind == "linear":
        return act(y)
    return {"codes": _unrounded(act(y[:, :case["outputs"]]) * y[:, case["outputs"]:])[0], "scales": None}
