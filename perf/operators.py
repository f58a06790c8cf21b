"""Microscaled 4-bit floating point (quantisation, its inverse, the product) and rotary positions, as measurable cases.

What a program that runs an encoder with 4-bit projections and rotary positions has these operators do:

* ``quantize``: values to 4-bit codes with one power-of-two scale for 32 of them and back to values, which is what the next
  layer sees of an activation or a weight;
* ``product``: D = act(alpha * A.B^T + beta * C) of two matrices that are held that way;
* ``rotary``: the first dimensions of every head turned by position times frequency;
* ``project``: a layer's QKV projection as the layer runs it: activations quantised, the product, queries and keys of the
  packed result turned in place, ready for the attention that reads them.

Where ``own`` is false everything is computed in elementary torch operations, in 32 bits, rounded at the end of each
operator.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = "hands_on_mlir_b200"  # the directory's name has a hyphen: loaded by path
_TYPES = {"f16": torch.float16, "f32": torch.float32}


def _package():
    if _PACKAGE not in sys.modules:
        root = Path.cwd() / "hands-on-mlir_b200"
        spec = importlib.util.spec_from_file_location(_PACKAGE, root / "__init__.py",
                                                      submodule_search_locations=[str(root)])
        module = importlib.util.module_from_spec(spec)
        sys.modules[_PACKAGE] = module
        spec.loader.exec_module(module)
    return sys.modules[_PACKAGE]


# ------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # the activations of one token on their way into a projection: latency
        dict(name="quantize_token", kind="quantize", rows=1, cols=4096, type="f16", transposed=False),
        # a weight stored [K, N], quantised along K when the model is loaded
        dict(name="quantize_weight_kn", kind="quantize", rows=1024, cols=4096, type="f16", transposed=True),
        # fp32 activations whose width is no multiple of the block
        dict(name="quantize_f32_odd", kind="quantize", rows=20011, cols=777, type="f32", transposed=False),
        # FFN1 of one token: bias row and GELU
        dict(name="product_token", kind="product", m=1, n=4096, k=1024, c="row", act=True, alpha=1.0, beta=1.0),
        # ragged everything, scaled, residual
        dict(name="product_odd", kind="product", m=385, n=1001, k=808, c="full", act=False, alpha=0.5, beta=2.0),
        # QKV projection of a batch of 32 sequences of 128
        dict(name="product_qkv_4096", kind="product", m=4096, n=2304, k=768, c="none", act=False, alpha=1.0, beta=0.0),
        # FFN2 of 32 sequences of 512 with the residual added
        dict(name="product_ffn2_16384", kind="product", m=16384, n=1024, k=4096, c="full", act=False, alpha=1.0, beta=1.0),
        # FFN1 of the largest batch, 256 sequences of 512
        dict(name="product_ffn1_131072", kind="product", m=131072, n=4096, k=1024, c="row", act=True, alpha=1.0, beta=1.0),
        # one new token in each of eight sequences, far into a long context
        dict(name="rotary_token_far", kind="rotary", batch=8, seq=1, heads=16, dim=64, turned=64, packed=True, type="f16",
             interleaved=False, backward=False, far=1 << 20, scaling=8.0, magnitude=1.0),
        # the gradient's way back, fp32, neighbouring dimensions as pairs, half of an odd-sized head
        dict(name="rotary_f32_gradient", kind="rotary", batch=3, seq=777, heads=12, dim=80, turned=40, packed=False,
             type="f32", interleaved=True, backward=True, far=0, scaling=1.0, magnitude=1.0),
        # queries and keys of 64 sequences of 512 in their packed buffer
        dict(name="rotary_64x512", kind="rotary", batch=64, seq=512, heads=16, dim=64, turned=64, packed=True, type="f16",
             interleaved=False, backward=False, far=0, scaling=1.0, magnitude=1.1),
        # a layer's QKV projection, ready for the attention
        dict(name="project_32x128", kind="project", batch=32, seq=128, heads=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["quantize", "product", "product", "product", "rotary", "rotary", "project"])
    if kind == "quantize":
        cols = _log_int(rng, 17, 8192)
        return dict(kind=kind, rows=_log_int(rng, 1, (1 << 26) // cols), cols=cols, type=rng.choice(["f16", "f32"]),
                    transposed=rng.random() < 0.3)
    if kind == "product":
        k = _log_int(rng, 32, 4096)
        n = _log_int(rng, 32, 4096)
        n = n if rng.random() < 0.3 else (n + 7) // 8 * 8
        m = _log_int(rng, 1, min(131072, (131072 * 4096 * 1024) // (n * k)))
        c = rng.choice(["none", "row", "full"])
        plain = rng.random() < 0.7
        return dict(kind=kind, m=m, n=n, k=k, c=c, act=rng.random() < 0.4, alpha=1.0 if plain else rng.uniform(0.1, 3.0),
                    beta=0.0 if c == "none" else 1.0 if plain else rng.uniform(0.1, 3.0))
    heads = _log_int(rng, 1, 32)
    seq = _log_int(rng, 1, 4096)
    if kind == "project":
        return dict(kind=kind, batch=_log_int(rng, 1, max(1, 32768 // seq)), seq=seq, heads=min(heads, 16))
    dim = rng.choice([64, 64, 64, 2 * _log_int(rng, 16, 128)])
    batch = _log_int(rng, 1, max(1, min(256, (1 << 25) // (seq * heads * dim))))
    return dict(kind=kind, batch=batch, seq=seq, heads=heads, dim=dim,
                turned=dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2), packed=rng.random() < 0.5,
                type=rng.choice(["f16", "f16", "f32"]), interleaved=rng.random() < 0.4, backward=rng.random() < 0.3,
                far=rng.choice([0, 0, 1 << 17, 1 << 20]), scaling=rng.choice([1.0, 4.0, 16.0]),
                magnitude=rng.choice([1.0, 1.2]))


# ----------------------------------------------------------------------------------------- inputs

def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _normal(gen, shape, dtype=torch.float16, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def _activations(gen, rows, cols, dtype=torch.float16):
    """Normal values whose channels differ in size, a few of them by much, as behind a LayerNorm with learned weights."""
    size = torch.exp(_normal(gen, (cols,), torch.float32, 0.7))
    return (_normal(gen, (rows, cols), torch.float32) * size).to(dtype)


def _frequencies(turned, scaling, base=10000.0):
    """Radians a position for each pair of dimensions, positions stretched over a `scaling` times longer context."""
    i = torch.arange(turned // 2, dtype=torch.float64, device="cuda")
    return base ** (-2.0 * i / turned) / scaling


def prepare(case, seed):
    return {"case": case, "inputs": _inputs(case, seed)}


def _inputs(case, seed):
    gen = _generator(seed)
    kind = case["kind"]
    if kind == "quantize":
        return {"x": _activations(gen, case["rows"], case["cols"], _TYPES[case["type"]])}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a, sa = _encode(_activations(gen, m, k).float())
        b, sb = _encode(_normal(gen, (n, k), torch.float32, k ** -0.5))
        c = None if case["c"] == "none" else _normal(gen, (1, n) if case["c"] == "row" else (m, n))
        return {"a": a, "sa": sa, "b": b, "sb": sb, "c": c}
    batch, seq, heads = case["batch"], case["seq"], case["heads"]
    if kind == "project":
        hidden = 64 * heads
        b, sb = _encode(_normal(gen, (3 * hidden, hidden), torch.float32, hidden ** -0.5))
        return {"x": _activations(gen, batch * seq, hidden).reshape(batch, seq, hidden), "b": b, "sb": sb,
                "frequencies": _frequencies(64, 1.0)}
    dim, dtype = case["dim"], _TYPES[case["type"]]
    x = _normal(gen, (batch, seq, (3 if case["packed"] else 2) * heads, dim), dtype)[:, :, :2 * heads]
    positions = None
    if case["far"]:
        first = torch.randint(0, case["far"], (batch, 1), generator=gen, device="cuda")
        positions = first + torch.arange(seq, device="cuda")
    return {"x": x, "positions": positions, "frequencies": _frequencies(case["turned"], case["scaling"])}


# ------------------------------------------------------- the 4-bit format in elementary operations

def _encode(x):
    """fp32 [rows, cols] -> codes [rows, 16 * blocks] (two to a byte, the first in the low half) and scale bytes as
    [ceil(rows / 128), ceil(blocks / 4), 512]: byte (r % 32) * 16 + (r / 32) % 4 * 4 + b % 4 of a tile belongs to row r,
    block b."""
    rows, cols = x.shape
    blocks = (cols + 31) // 32
    padded = torch.zeros((rows, 32 * blocks), dtype=torch.float32, device=x.device)
    padded[:, :cols] = x
    values = padded.reshape(rows, blocks, 32)
    largest = values.abs().amax(-1)
    exponent = torch.where(largest > 0, (torch.frexp(largest)[1] - 3).clamp(min=-127), torch.full_like(largest, -127).int())
    scaled = values * torch.exp2(-exponent.double()).float()[..., None]
    v = scaled.abs()
    # halfway between two neighbours the even code is taken
    code = ((v > 0.25).int() + (v >= 0.75).int() + (v > 1.25).int() + (v >= 1.75).int() + (v > 2.5).int() +
            (v >= 3.5).int() + (v > 5.0).int())
    code = (code + 8 * (scaled < 0).int()).to(torch.uint8).reshape(rows, 16 * blocks, 2)
    scales = torch.zeros(((rows + 127) // 128 * 128, (blocks + 3) // 4 * 4), dtype=torch.uint8, device=x.device)
    scales[:rows, :blocks] = (exponent + 127).to(torch.uint8)
    tiles = scales.reshape(-1, 4, 32, scales.shape[1] // 4, 4).permute(0, 3, 2, 1, 4)
    return code[..., 0] | (code[..., 1] << 4), tiles.reshape(tiles.shape[0], tiles.shape[1], 512).contiguous()


def _decode(codes, tiles, dtype=torch.float32):
    """The values, [rows, 32 * blocks]."""
    rows, blocks = codes.shape[0], codes.shape[1] // 16
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=dtype, device=codes.device)
    scales = tiles.reshape(tiles.shape[0], tiles.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4)
    scales = scales.reshape(tiles.shape[0] * 128, tiles.shape[1] * 4)[:rows, :blocks]
    values = table[torch.stack((codes & 15, codes >> 4), -1).reshape(rows, blocks, 32).int()]
    return (values * torch.exp2(scales.double() - 127).to(dtype)[..., None]).reshape(rows, 32 * blocks)


def _plain_product(a, sa, b, sb, c, act, alpha, beta):
    v = _decode(a, sa) @ _decode(b, sb).t()
    v = alpha * v
    if c is not None:
        v = v + beta * c.float()
    if act:
        v = 0.5 * v * (1.0 + torch.erf(v * 0.5 ** 0.5))
    return v.half()


def _plain_rotary(x, positions, frequencies, interleaved, backward, magnitude):
    half = frequencies.numel()
    if positions is None:
        positions = torch.arange(x.shape[1], device=x.device)[None]
    angle = positions.double()[..., None] * frequencies
    cos, sin = (magnitude * f(angle).float()[:, :, None] for f in (torch.cos, torch.sin))
    sin = -sin if backward else sin
    turned, rest = x[..., :2 * half].float(), x[..., 2 * half:]
    x0, x1 = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    y0, y1 = x0 * cos - x1 * sin, x1 * cos + x0 * sin
    y = torch.stack((y0, y1), -1).flatten(-2) if interleaved else torch.cat((y0, y1), -1)
    return torch.cat((y.to(x.dtype), rest), -1)


# -------------------------------------------------------------------------------------------- run

def run(state):
    if own:
        return _own(state)
    case, t = state["case"], state["inputs"]
    kind = case["kind"]
    if kind == "quantize":
        x = t["x"].float()
        x = x.t() if case["transposed"] else x
        return _decode(*_encode(x))[:, :x.shape[1]].to(t["x"].dtype)
    if kind == "product":
        return _plain_product(t["a"], t["sa"], t["b"], t["sb"], t["c"], case["act"], case["alpha"], case["beta"])
    if kind == "rotary":
        return _plain_rotary(t["x"], t["positions"], t["frequencies"], case["interleaved"], case["backward"],
                             case["magnitude"])
    batch, seq, hidden = t["x"].shape
    qkv = _plain_product(*_encode(t["x"].reshape(-1, hidden).float()), t["b"], t["sb"], None, False, 1.0, 0.0)
    qkv = qkv.reshape(batch, seq, -1, 64)
    turned = _plain_rotary(qkv[:, :, :2 * case["heads"]], None, t["frequencies"], False, False, 1.0)
    return torch.cat((turned, qkv[:, :, 2 * case["heads"]:]), 2).reshape(batch, seq, 3 * hidden)


def _own(state):
    if "calls" not in state:
        _bind(state)  # buffers and descriptors, which a program makes once and calls with ever after
    for call, args in state["calls"]:
        call(*args)
    return state["out"]


def _codes(rows, cols):
    blocks = (cols + 31) // 32
    return (torch.empty((rows, 16 * blocks), dtype=torch.uint8, device="cuda"),
            torch.empty(((rows + 127) // 128, (blocks + 3) // 4, 512), dtype=torch.uint8, device="cuda"))


def _bind(state):
    hom, ref = _package().runner(), _package().MemRef.of
    case, t = state["case"], state["inputs"]
    kind = case["kind"]
    hom.use_torch_stream()
    if kind == "quantize":
        x, transposed = t["x"], case["transposed"]
        rows, cols = reversed(x.shape) if transposed else x.shape
        q, s = _codes(rows, cols)
        out = torch.empty((rows, cols), dtype=x.dtype, device="cuda")
        there, back = ((hom.homQuantizeMxF4F16, hom.homDequantizeMxF4F16) if x.dtype == torch.float16 else
                       (hom.homQuantizeMxF4F32, hom.homDequantizeMxF4F32))
        q, s = ref(q), ref(s)
        state["calls"] = [(there, (ref(x), q, s, transposed)), (back, (q, s, ref(out)))]
    elif kind == "product":
        out = torch.empty((case["m"], case["n"]), dtype=torch.float16, device="cuda")
        d = ref(out)
        state["calls"] = [(hom.homGemmMxF4F16, (ref(t["a"]), ref(t["sa"]), ref(t["b"]), ref(t["sb"]),
                                                d if t["c"] is None else ref(t["c"]), d, int(case["act"]), case["alpha"],
                                                case["beta"]))]
    elif kind == "rotary":
        out = torch.empty(t["x"].shape, dtype=t["x"].dtype, device="cuda")
        call = hom.homRotaryF16 if t["x"].dtype == torch.float16 else hom.homRotaryF32
        positions = None if t["positions"] is None else ref(t["positions"])
        state["calls"] = [(call, (ref(t["x"]), positions, ref(t["frequencies"]), ref(out), case["interleaved"],
                                  case["backward"], case["magnitude"]))]
    else:
        x = t["x"]
        batch, seq, hidden = x.shape
        q, s = (ref(v) for v in _codes(batch * seq, hidden))
        out = torch.empty((batch, seq, 3 * hidden), dtype=torch.float16, device="cuda")
        rows, turned = ref(out.view(batch * seq, 3 * hidden)), ref(out.view(batch, seq, -1, 64)[:, :, :2 * case["heads"]])
        state["calls"] = [(hom.homQuantizeMxF4F16, (ref(x.view(-1, hidden)), q, s, False)),
                          (hom.homGemmMxF4F16, (q, s, ref(t["b"]), ref(t["sb"]), rows, rows, 0, 1.0, 0.0)),
                          (hom.homRotaryF16, (turned, None, ref(t["frequencies"]), turned, False, False, 1.0))]
    state["out"] = out


# ------------------------------------------------------------------------------------------ exact

def exact(case, seed):
    """What `run` returns, in 64 bits from the operators' definitions."""
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "quantize":
        x = t["x"].double()
        return _nearest64(x.t() if case["transposed"] else x)
    if kind == "product":
        v = case["alpha"] * (_values64(t["a"], t["sa"]) @ _values64(t["b"], t["sb"]).t())
        if t["c"] is not None:
            v += case["beta"] * t["c"].double()
        return v * torch.special.ndtr(v) if case["act"] else v
    if kind == "rotary":
        return _rotary64(t["x"].double(), t["positions"], t["frequencies"], case["interleaved"], case["backward"],
                         case["magnitude"])
    batch, seq, hidden = t["x"].shape
    qkv = _nearest64(t["x"].double().reshape(-1, hidden)) @ _values64(t["b"], t["sb"]).t()[:hidden]
    qkv = qkv.reshape(batch, seq, -1, 64)
    heads = 2 * case["heads"]
    qkv[:, :, :heads] = _rotary64(qkv[:, :, :heads].clone(), None, t["frequencies"], False, False, 1.0)
    return qkv.reshape(batch, seq, 3 * hidden)


def _nearest64(x):
    """Every value of a block replaced by the nearest multiple of the block's scale that four bits express: whole halves
    below 2, whole numbers below 4, even ones up to 6 (`round` goes to the even neighbour of a halfway value)."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x, (0, -cols % 32)).unflatten(-1, (-1, 32))
    # a number with its fraction cleared is the power of two below it
    power = (v.abs().amax(-1, keepdim=True).view(torch.int64) & (0x7FF << 52)).view(torch.float64)
    scale = power.clamp(min=2.0 ** -125) / 4
    v = v / scale
    size = v.abs()
    spacing = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    return ((v / spacing).round() * spacing).clamp(-6, 6).mul(scale).flatten(-2)[:, :cols]


def _values64(codes, tiles):
    rows, blocks = codes.shape[0], codes.shape[1] // 16
    row = torch.arange(rows, device="cuda")[:, None]
    block = torch.arange(blocks, device="cuda")[None]
    scale = tiles[row // 128, block // 4, row % 32 * 16 + row // 32 % 4 * 4 + block % 4].double() - 127
    nibbles = torch.empty((rows, 32 * blocks), dtype=torch.uint8, device="cuda")
    nibbles[:, 0::2], nibbles[:, 1::2] = codes % 16, codes // 16
    exponent, mantissa = (nibbles // 2 % 4).double(), (nibbles % 2).double()
    size = torch.where(exponent > 0, (1 + mantissa / 2) * torch.exp2(exponent - 1), mantissa / 2)
    return torch.where(nibbles < 8, size, -size) * torch.exp2(scale).repeat_interleave(32, 1)


def _rotary64(x, positions, frequencies, interleaved, backward, magnitude):
    half = frequencies.numel()
    if positions is None:
        positions = torch.arange(x.shape[1], device="cuda").expand(x.shape[:2])
    angle = torch.einsum("bs,f->bsf", positions.double(), frequencies) * (-1 if backward else 1)
    turn = torch.polar(torch.full_like(angle, magnitude), angle).unsqueeze(2)
    y = x.clone()
    if interleaved:
        y[..., :2 * half] = torch.view_as_real(torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) * turn).flatten(-2)
    else:
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


# ------------------------------------------------------------------------------------------- work

def _code_bytes(rows, cols):
    return rows * cols * (0.5 + 1 / 32)


def work(case):
    """Bytes: inputs read once, outputs and what travels between two calls written once.  Operations: the product's."""
    kind = case["kind"]
    if kind == "quantize":
        rows, cols = case["rows"], case["cols"]
        return {"bytes": 2 * (2 if case["type"] == "f16" else 4) * rows * cols + _code_bytes(rows, cols), "flops": 0.0}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        c = {"none": 0, "row": 2 * n, "full": 2 * m * n}[case["c"]]
        return {"bytes": _code_bytes(m, k) + _code_bytes(n, k) + c + 2 * m * n, "flops": 2.0 * m * n * k}
    tokens, heads = case["batch"] * case["seq"], case["heads"]
    if kind == "project":
        hidden = 64 * heads
        return {"bytes": 2 * tokens * hidden + _code_bytes(tokens + 3 * hidden, hidden) + 6 * tokens * hidden,
                "flops": 6.0 * tokens * hidden * hidden}
    element = 2 if case["type"] == "f16" else 4
    return {"bytes": 2.0 * element * tokens * 2 * heads * case["dim"] + (8 * tokens if case["far"] else 0),
            "flops": 3.0 * tokens * 2 * heads * case["turned"]}
