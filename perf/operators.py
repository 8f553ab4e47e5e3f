"""The performance cases of the microscaled 4-bit layers and of the channels-last group norm.

`listed()` names the cases; `draw(rng)` gives further ones of the same ranges; `prepare(case, seed)`
builds what a program holds before the call; `run(state)` is one pass, in elementary torch operations
or, where `own` is true, through the operators of `glow_b200.ops`; `exact(case, seed)` is what the
definition gives in 64 bits; `work(case)` what the pass cannot do without.

Every case has a "path":
  round     float rows to the microscaled 4-bit format and back to the values it stands for
  fc        a fully connected layer whose input and weights are both in that format
  dynamic   the same with a float input that the layer quantizes itself
  norm      group norm over channels-last activations with the activation behind it

The format: blocks of 32 neighbours of a row share a power of two 2^e, e = floor(log2(max |x|)) - 2;
an element is the E2M1 number (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives) nearest to x / 2^e, ties
to the even code, beyond 6 it is 6.  Rows are packed two to a byte, the even column in the low half,
filled up with zeros to whole blocks; the scale bytes e + 127 lie in tiles of 128 rows by 4 blocks:
row r, block b at byte (r % 32) * 16 + (r // 32) * 4 + b of its tile, the tiles of a row of tiles one
after the other, bytes of rows and blocks that are not there 0.
"""
import math

import torch

own = False
DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # The tokens of one decoding step on their way into a quantized layer: the smallest call.
        {"name": "round_few_rows", "path": "round", "rows": 4, "cols": 4096, "dtype": "bf16"},
        # The activations of a whole batch, as dynamic quantization sees them.
        {"name": "round_batch", "path": "round", "rows": 8192, "cols": 4096, "dtype": "fp16"},
        # The interaction's 479 float columns: no whole number of blocks, rows off 16-byte boundaries.
        {"name": "round_ragged", "path": "round", "rows": 2048, "cols": 479, "dtype": "fp32"},
        # One token through a square layer: the weights' bytes, and latency.
        {"name": "fc_one_token", "path": "fc", "M": 1, "K": 4096, "N": 4096, "out": "bf16", "bias": True, "relu": False},
        # A recommendation model's top layer at a ragged batch: nothing is a multiple of a tile.
        {"name": "fc_ragged", "path": "fc", "M": 400, "K": 479, "N": 1000, "out": "fp16", "bias": True, "relu": True},
        # The benchmark's int8 layer in this format (2048 x 4096 x 4096).
        {"name": "fc_layer", "path": "fc", "M": 2048, "K": 4096, "N": 4096, "out": "fp16", "bias": True, "relu": False},
        # A whole prompt through the widening layer of a feed-forward block: the largest product.
        {"name": "fc_large", "path": "fc", "M": 4096, "K": 4096, "N": 8192, "out": "bf16", "bias": False, "relu": False},
        # Eight sequences' next tokens, quantized by the layer itself.
        {"name": "dynamic_decode", "path": "dynamic", "M": 8, "K": 4096, "N": 4096, "dtype": "fp16", "out": "fp16", "bias": True},
        # The same layer over a batch of prompts.
        {"name": "dynamic_batch", "path": "dynamic", "M": 2048, "K": 4096, "N": 4096, "dtype": "bf16", "out": "bf16", "bias": True},
        # One image in the deep part of a residual network: few pixels, many channels.
        {"name": "norm_one_image", "path": "norm", "n": 1, "h": 14, "w": 14, "C": 1024, "G": 32, "dtype": "fp16", "act": "relu"},
        # The first stage of ResNet-50 at batch 64, normalised by groups.
        {"name": "norm_batch", "path": "norm", "n": 64, "h": 56, "w": 56, "C": 256, "G": 32, "dtype": "fp16", "act": "relu"},
        # Large images: a sample's 16 MB exceed what a few SMs hold, and Swish behind the norm.
        {"name": "norm_large_images", "path": "norm", "n": 8, "h": 256, "w": 256, "C": 128, "G": 32, "dtype": "bf16", "act": "swish"},
    ]


def _log(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm; every other one is a multiple of 32 where it can be."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(hi, max(lo, v))
    if rng.random() < 0.5 and v >= 64:
        v = v // 32 * 32
    return v


def draw(rng):
    path = rng.choice(["round", "fc", "dynamic", "norm"])
    if path == "round":
        cols = _log(rng, 32, 16384)
        rows = _log(rng, 1, max(1, min(16384, 8192 * 4096 // cols)))
        return {"path": path, "rows": rows, "cols": cols, "dtype": rng.choice(["fp16", "bf16", "fp32"])}
    if path == "norm":
        G = rng.choice([1, 4, 8, 16, 32])
        C = G * rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 24, 32, 64])
        n = _log(rng, 1, 64)
        most = min(256 * 256, 4 * 256 * 256 * 128 // (n * C))
        h = max(1, int(math.sqrt(_log(rng, 1, max(1, most)))))
        w = max(1, min(h + rng.choice([-1, 0, 0, 1, 3]), most // h))
        return {"path": path, "n": n, "h": h, "w": w, "C": C, "G": G, "dtype": rng.choice(["fp16", "bf16", "fp32"]),
                "act": rng.choice(["none", "relu", "swish"])}
    K = _log(rng, 64, 16384)
    N = _log(rng, 64, max(64, min(16384, 4096 * 8192 // K)))
    most = max(1, min(8192, 4096 * 4096 * 8192 // (K * N), 4096 * 8192 // N, 8192 * 4096 // K))
    M = _log(rng, 1, most) if rng.random() < 0.7 else rng.randint(1, min(64, most))
    case = {"path": path, "M": M, "K": K, "N": N, "out": rng.choice(["fp16", "bf16", "fp32"]), "bias": rng.random() < 0.7}
    if path == "fc":
        case["relu"] = rng.random() < 0.5
    else:
        case["dtype"] = rng.choice(["fp16", "bf16", "fp32"])
    return case


# ---- the format, in elementary operations ----
def _power(e):
    """2^e in fp32, exactly, for whole numbers of -127..127."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _blocks(x):
    """fp32 [rows, blocks, 32], zeros behind the last column."""
    rows, cols = x.shape
    return torch.nn.functional.pad(x.float(), (0, -cols % 32)).view(rows, -1, 32)


def _quantized(x):
    """(E2M1 values fp32 [rows, blocks, 32], exponents int32 [rows, blocks])"""
    b = _blocks(x)
    _, e = torch.frexp(b.abs().amax(2))  # max = m * 2^e, m in [0.5, 1)
    e = torch.where(b.abs().amax(2) == 0, torch.full_like(e, -127), (e - 3).clamp(min=-127))
    y = b * _power(-e).unsqueeze(2)
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), y), e


def _packed(x):
    """(bytes uint8 [rows, 16 * blocks], scale tiles uint8 [row tiles, block tiles, 512])"""
    v, e = _quantized(x)
    rows, blocks = e.shape
    a = v.abs()
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) + 8 * torch.signbit(v).to(torch.uint8)
    code = code.view(rows, -1)
    tiles = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, -blocks % 4, 0, -rows % 128))
    tiles = tiles.view(-1, 4, 32, tiles.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, tiles.shape[1] // 4, 512)
    return code[:, 0::2] | code[:, 1::2] << 4, tiles.contiguous()


def _values(data, tiles):
    """The numbers that packed rows stand for, fp32 [rows, 32 * blocks]."""
    rows, blocks = data.shape[0], data.shape[1] // 16
    code = torch.stack((data & 15, data >> 4), 2).view(rows, -1).to(torch.int64)
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device=data.device)
    e = tiles.view(tiles.shape[0], tiles.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiles.shape[0] * 128, -1)
    e = e[:rows, :blocks].to(torch.int32) - 127
    return (table[code].view(rows, blocks, 32) * _power(e).unsqueeze(2)).view(rows, -1)


# ---- inputs ----
def _activations(rows, cols, dtype, g):
    """Rows of different size with a few columns far larger than the rest, and a stretch of zeros."""
    x = torch.randn(rows, cols, device=DEV, generator=g)
    x *= torch.exp(torch.randn(rows, 1, device=DEV, generator=g))
    x *= torch.where(torch.rand(1, cols, device=DEV, generator=g) < 0.01, 20.0, 1.0)
    if cols >= 128:
        x[rows // 2, 32:96] = 0
    return x.to(TYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case)
    if case["path"] == "round":
        s["x"] = _activations(case["rows"], case["cols"], case["dtype"], g)
    elif case["path"] in ("fc", "dynamic"):
        M, K, N = case["M"], case["K"], case["N"]
        s["x"] = _activations(M, K, case.get("dtype", "fp32"), g)
        s["weights"], s["weight_tiles"] = _packed(torch.randn(N, K, device=DEV, generator=g) * (2.0 / math.sqrt(K)))
        s["bias_values"] = torch.randn(N, device=DEV, generator=g) if case["bias"] else None
        if case["path"] == "fc":
            s["input"], s["input_tiles"] = _packed(s.pop("x"))
    else:
        n, h, w, C = case["n"], case["h"], case["w"], case["C"]
        x = torch.randn(n, h, w, C, device=DEV, generator=g)
        x = x * (0.2 + torch.rand(n, 1, 1, C, device=DEV, generator=g)) + torch.randn(n, 1, 1, C, device=DEV, generator=g)
        s["x"] = x.to(TYPES[case["dtype"]])
        s["gamma"] = 1 + 0.2 * torch.randn(C, device=DEV, generator=g)
        s["beta"] = 0.2 * torch.randn(C, device=DEV, generator=g)
    return s


# ---- one pass ----
def _own(s):
    from glow_b200 import ops
    if s["path"] == "round":
        data, scales = ops.microscaled_fp4_quantize(s["x"])
        return {"values": ops.microscaled_fp4_dequantize(data, scales, s["cols"], out_dtype=torch.bfloat16)}
    if s["path"] == "fc":
        return {"out": ops.microscaled_fp4_fc(s["input"], s["input_tiles"], s["weights"], s["weight_tiles"], s["bias_values"],
                                              flags=ops.FC_FUSE_RELU if s["relu"] else 0, out_dtype=TYPES[s["out"]])}
    if s["path"] == "dynamic":
        return {"out": ops.dynamic_microscaled_fp4_fc(s["x"], s["weights"], s["weight_tiles"], s["bias_values"],
                                                      out_dtype=TYPES[s["out"]])}
    act = {"none": ops.NORM_ACT_NONE, "relu": ops.NORM_ACT_RELU, "swish": ops.NORM_ACT_SWISH}[s["act"]]
    return {"out": ops.group_norm(s["x"], s["G"], s["gamma"], s["beta"], 1e-5, activation=act)}


def run(state):
    s = state
    if own:
        return _own(s)
    if s["path"] == "round":
        v, e = _quantized(s["x"])
        return {"values": (v * _power(e).unsqueeze(2)).view(s["rows"], -1)[:, :s["cols"]].to(torch.bfloat16)}
    if s["path"] in ("fc", "dynamic"):
        if s["path"] == "fc":
            a = _values(s["input"], s["input_tiles"])
        else:
            v, e = _quantized(s["x"])
            a = (v * _power(e).unsqueeze(2)).view(s["M"], -1)
        y = torch.matmul(a, _values(s["weights"], s["weight_tiles"]).t())
        if s["bias_values"] is not None:
            y = y + s["bias_values"]
        if s.get("relu"):
            y = torch.maximum(y, torch.zeros_like(y))
        return {"out": y.to(TYPES[s["out"]])}
    n, h, w, C = s["x"].shape
    x = s["x"].float().view(n, h * w, s["G"], C // s["G"])
    d = x - x.mean((1, 3), keepdim=True)
    d = d / torch.sqrt((d * d).mean((1, 3), keepdim=True) + 1e-5)
    y = d.view(n, h * w, C) * s["gamma"] + s["beta"]
    if s["act"] == "relu":
        y = torch.maximum(y, torch.zeros_like(y))
    elif s["act"] == "swish":
        y = y / (1 + torch.exp(-y))
    return {"out": y.view(n, h, w, C).to(s["x"].dtype)}


# ---- the definitions in 64 bits ----
def _exact_rounded(x):
    """What the format makes of float rows, fp64: the nearest of the sixteen numbers, found by comparing with their midpoints."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    b = torch.zeros(rows, blocks * 32, dtype=torch.float64, device=x.device)
    b[:, :cols] = x.double()
    b = b.view(rows, blocks, 32)
    top = b.abs().amax(2, keepdim=True)
    e = torch.floor(torch.log2(top))
    e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e))  # next to a power of two
    e = torch.where(top > 0, torch.clamp(e - 2, min=-127), torch.full_like(top, -127))
    scale = torch.exp2(e)
    a = b.abs() / scale
    # a number on a midpoint goes to the even code: up from the midpoints above odd codes, down from those above even ones
    value = torch.zeros_like(a)
    for mid, to, up in ((.25, .5, False), (.75, 1., True), (1.25, 1.5, False), (1.75, 2., True), (2.5, 3., False),
                        (3.5, 4., True), (5., 6., False)):
        value = torch.where((a >= mid) if up else (a > mid), torch.full_like(a, to), value)
    return (torch.sign(b) * value * scale).view(rows, -1)


def _exact_values(data, tiles):
    """The numbers that packed rows stand for, fp64, element by element from the format's addresses."""
    rows, cols = data.shape[0], 2 * data.shape[1]
    r = torch.arange(rows, device=data.device).view(-1, 1)
    c = torch.arange(cols, device=data.device).view(1, -1)
    code = (data.to(torch.int64).gather(1, (c // 2).expand(rows, cols)) >> (4 * (c % 2))) & 15
    b = c // 32
    at = (r // 128 * tiles.shape[1] + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4
    e = tiles.reshape(-1)[at].to(torch.float64) - 127
    m, p = (code & 1).double(), ((code >> 1) & 3).double()  # one bit of mantissa, two of exponent
    size = torch.where(p > 0, (1 + m / 2) * torch.exp2(p - 1), m / 2)
    return torch.where(code >= 8, -size, size) * torch.exp2(e)


def exact(case, seed):
    s = prepare(case, seed)
    if case["path"] == "round":
        return {"values": _exact_rounded(s["x"])[:, :case["cols"]]}
    if case["path"] in ("fc", "dynamic"):
        if case["path"] == "fc":
            a = _exact_values(s["input"], s["input_tiles"])
        else:
            a = _exact_rounded(s["x"])
        y = a @ _exact_values(s["weights"], s["weight_tiles"]).T
        if s["bias_values"] is not None:
            y += s["bias_values"].double()
        return {"out": y.clamp(min=0) if case.get("relu") else y}
    n, C, G = case["n"], case["C"], case["G"]
    x = s["x"].double().reshape(n, -1, G, C // G).transpose(1, 2).reshape(n, G, -1)
    var, mean = torch.var_mean(x, dim=2, unbiased=False, keepdim=True)
    y = ((x - mean) * torch.rsqrt(var + 1e-5)).view(n, G, -1, C // G).transpose(1, 2).reshape(n, -1, C)
    y = y * s["gamma"].double() + s["beta"].double()
    if case["act"] == "relu":
        y = y.clamp(min=0)
    elif case["act"] == "swish":
        y = y * torch.sigmoid(y)
    return {"out": y.view(s["x"].shape)}


def work(case):
    if case["path"] == "round":
        n = case["rows"] * case["cols"]
        # the rows in, the format out and in again, the bf16 values out
        return {"bytes": n * (BYTES[case["dtype"]] + 2 * 17 / 32 + 2), "flops": 6 * n}
    if case["path"] in ("fc", "dynamic"):
        M, K, N = case["M"], case["K"], case["N"]
        into = M * K * (17 / 32 if case["path"] == "fc" else BYTES[case["dtype"]])
        return {"bytes": into + N * K * 17 / 32 + M * N * BYTES[case["out"]] + (4 * N if case["bias"] else 0), "flops": 2 * M * K * N}
    n = case["n"] * case["h"] * case["w"] * case["C"]
    return {"bytes": 2 * n * BYTES[case["dtype"]] + 8 * case["C"], "flops": 10 * n}
