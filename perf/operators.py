"""What the 8-bit operators of the engine are measured on: quantising rows and weights to e4m3 with a
power-of-two scale for each block of 128, reading them back, and the linear layer over them.

A stored block is 128 consecutive columns of one row (of 128 rows for weights): the values are e4m3,
the block's scale is 2^(E - 127) with E one byte. `run` either computes an operator in elementary torch
operations in 32 bits or calls the package's entry points (`own`)."""
import importlib.util
import math
import os
import sys

import torch

own = False

HIDDEN, QKV, FFN = 768, 2304, 2048  # the encoder's widths
LINES = 33104  # token rows of the benchmark's 251 lines
TEXTS = 67251  # token rows of the text-side workload's 256 sequences
LAYERS = ((QKV, HIDDEN), (HIDDEN, HIDDEN), (FFN, HIDDEN), (HIDDEN, FFN), (512, HIDDEN), (HIDDEN, 128))
MOST_FLOPS = 2.0 * 8192 ** 3
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one token's hidden state quantised and read back: latency
        {"name": "quantize-1x768-f32", "op": "quantize", "rows": 1, "k": HIDDEN, "pad": 0, "type": "f32", "block_rows": 1},
        # one long line's 514-channel concat, held in wider rows: an odd width whose last block is 2 columns
        {"name": "quantize-1041x514-bf16", "op": "quantize", "rows": 1041, "k": 514, "pad": 2, "type": "bf16", "block_rows": 1},
        # the hidden states of the benchmark's 251 lines
        {"name": "quantize-33104x768-f32", "op": "quantize", "rows": LINES, "k": HIDDEN, "pad": 0, "type": "f32", "block_rows": 1},
        # a large layer's weights as they are loaded
        {"name": "quantize-weight-8192", "op": "quantize", "rows": 8192, "k": 8192, "pad": 0, "type": "bf16", "block_rows": 128},
        # one token through the QKV projection: latency
        {"name": "linear-qkv-1", "op": "linear", "m": 1, "n": QKV, "k": HIDDEN, "act": "none", "residual": False, "out": "bf16"},
        # a short line (64 phonemes and the two pads) through the FFN's first layer, kept in 8 bits for the second
        {"name": "linear-ffn-66", "op": "linear", "m": 66, "n": FFN, "k": HIDDEN, "act": "gelu", "residual": False, "out": "e4m3"},
        # the longest line through the FFN's second layer, onto the 32-bit residual rows
        {"name": "linear-ffn-out-512", "op": "linear", "m": 512, "n": HIDDEN, "k": FFN, "act": "none", "residual": True, "out": "f32"},
        # odd sizes on every side: one long line's frames through the decoder's concat widths
        {"name": "linear-odd-1041", "op": "linear", "m": 1041, "n": 1090, "k": 514, "act": "none", "residual": False, "out": "f32"},
        # the benchmark's 251 lines through the QKV projection
        {"name": "linear-qkv-33104", "op": "linear", "m": LINES, "n": QKV, "k": HIDDEN, "act": "none", "residual": False, "out": "bf16"},
        # the same through the FFN's first layer, kept in 8 bits
        {"name": "linear-ffn-33104", "op": "linear", "m": LINES, "n": FFN, "k": HIDDEN, "act": "gelu", "residual": False, "out": "e4m3"},
        # the square product the card's matrix rate is quoted on
        {"name": "linear-8192", "op": "linear", "m": 8192, "n": 8192, "k": 8192, "act": "none", "residual": False, "out": "bf16"},
        # the text-side workload through a whole feed-forward block: quantise, GELU layer, second layer + residual
        {"name": "ffn-67251", "op": "ffn", "m": TEXTS, "n": FFN, "k": HIDDEN, "act": "gelu", "residual": True, "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "linear", "linear", "ffn"))
    if op == "quantize":
        rows, k = _log(rng, 1, TEXTS), _log(rng, 1, 8192)
        rows = max(1, min(rows, 2 ** 26 // k))
        return {"op": op, "rows": rows, "k": k, "pad": rng.choice((0, 0, 1, 2, 8, 64)), "type": rng.choice(("f32", "bf16")),
                "block_rows": rng.choice((1, 1, 128))}
    n, k = rng.choice(LAYERS) if rng.random() < 0.5 else (_log(rng, 16, 8192), _log(rng, 16, 8192))
    if op == "ffn":
        n, k = rng.choice(((FFN, HIDDEN), (_log(rng, 64, 8192), _log(rng, 64, 2048))))
    m = _log(rng, 1, TEXTS)
    m = int(max(1, min(m, MOST_FLOPS / ((4.0 if op == "ffn" else 2.0) * n * k), 1.6e8 / max(n, k))))
    if op == "ffn":
        return {"op": op, "m": m, "n": n, "k": k, "act": "gelu", "residual": True, "out": "bf16"}
    act, out = rng.choice(("none", "none", "gelu")), rng.choice(("f32", "bf16", "bf16", "e4m3"))
    return {"op": op, "m": m, "n": n, "k": k, "act": act, "residual": out != "e4m3" and rng.random() < 0.4, "out": out}


def work(case):
    if case["op"] == "quantize":
        n, size = case["rows"] * case["k"], 4 if case["type"] == "f32" else 2
        blocks = math.ceil(case["rows"] / case["block_rows"]) * math.ceil(case["k"] / 128)
        return {"bytes": n * (size + 1) + blocks + n * (1 + size) + blocks, "flops": 2.0 * n}
    m, n, k = case["m"], case["n"], case["k"]
    size = {"f32": 4, "bf16": 2}
    weights = n * k + 4 * n
    if case["op"] == "ffn":  # 32-bit rows in, residual rows in, both weights, result
        return {"bytes": 8 * m * k + 2 * weights, "flops": 4.0 * m * n * k}
    out = m * n * (1 + 1 + 2) if case["out"] == "e4m3" else m * n * size[case["out"]] * (2 if case["residual"] else 1)
    return {"bytes": m * k + m * math.ceil(k / 128) + weights + out, "flops": 2.0 * m * n * k}


# ---- the stored form, in elementary operations


def _blocks(x, block_rows):
    """x padded with zeros to whole blocks, as [row blocks, block_rows, column blocks, 128]."""
    r, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % 128, 0, -r % block_rows))
    return x.view(x.shape[0] // block_rows, block_rows, x.shape[1] // 128, 128)


def _quantize(x, block_rows=1):
    """(e4m3 values [rows, k], E [row blocks, column blocks]): E is the smallest number with
    max |x| <= 448 * 2^(E - 127), taken from the bits of the maximum (448 = 1.75 * 2^8)."""
    b = _blocks(x.float(), block_rows)
    bits = b.abs().amax(dim=(1, 3)).view(torch.int32)
    e = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp_min(0)
    q = (b * ((254 - e) << 23).view(torch.float32)[:, None, :, None]).to(torch.float8_e4m3fn)
    q = q.view(b.shape[0] * block_rows, -1)[: x.shape[0], : x.shape[1]]
    return q, e.to(torch.uint8)


def _dequantize(q, e, block_rows=1):
    """Each value times 2^(E - 127), the power made of its bits (2^-127 is below the normal numbers)."""
    e = e.int()
    scale = torch.where(e == 0, 1 << 22, e << 23).view(torch.float32)
    scale = scale.repeat_interleave(block_rows, 0)[: q.shape[0]].repeat_interleave(128, 1)[:, : q.shape[1]]
    return q.float() * scale


def _gelu(v):
    return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))


def _linear(x, w, bias, act, residual):
    y = x @ w.t() + bias
    y = _gelu(y) if act == "gelu" else y
    return y + residual.float() if residual is not None else y


# ---- inputs


def _rows(m, k, g):
    """Rows as a LayerNorm leaves them: unit variance, a few channels several times larger."""
    gain = 1.0 + 5.0 * (torch.rand(k, device="cuda", generator=g) < 0.01).float()
    return torch.randn(m, k, device="cuda", generator=g) * gain


def _weights(n, k, g):
    """A layer's initial weights, uniform in +-1/sqrt(k), stored in 8 bits; and its bias."""
    w = (torch.rand(n, k, device="cuda", generator=g) * 2.0 - 1.0) / math.sqrt(k)
    q, e = _quantize(w, 128)
    return _held(q, e) + ((torch.rand(n, device="cuda", generator=g) * 2.0 - 1.0) / math.sqrt(k),)


def _held(q, e):
    """Values and scales as the engine's store holds them: rows of values a multiple of 16 bytes apart,
    rows of scales a multiple of 4."""
    v = torch.zeros(q.shape[0], -(-q.shape[1] // 16) * 16, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.zeros(e.shape[0], -(-e.shape[1] // 4) * 4, device="cuda", dtype=torch.uint8)
    v.view(torch.uint8)[:, : q.shape[1]] = q.view(torch.uint8)
    s[:, : e.shape[1]] = e
    return v[:, : q.shape[1]], s[:, : e.shape[1]]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "quantize":
        rows, k = case["rows"], case["k"]
        x = _rows(rows, k + case["pad"], g).to(TYPES[case["type"]])
        s["x"] = x[:, :k]
        return s
    m, n, k = case["m"], case["n"], case["k"]
    s["w"] = _weights(n, k, g)
    if case["op"] == "ffn":
        s["x"] = _rows(m, k, g)
        s["w2"] = _weights(k, n, g)
        s["residual"] = s["x"].to(TYPES[case["out"]])
        return s
    s["x"] = _held(*_quantize(_rows(m, k, g)))
    s["residual"] = torch.randn(m, n, device="cuda", generator=g).to(TYPES[case["out"]]) if case["residual"] else None
    return s


# ---- one pass


def _package():
    """The package (its directory is not an importable name)."""
    if "kokoro_rust_b200" not in sys.modules:
        d = os.path.join(os.getcwd(), "kokoro-rust_b200")
        spec = importlib.util.spec_from_file_location("kokoro_rust_b200", os.path.join(d, "__init__.py"),
                                                      submodule_search_locations=[d])
        sys.modules["kokoro_rust_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["kokoro_rust_b200"])
    return sys.modules["kokoro_rust_b200"]


def _run_own(s):
    fp8 = _package().fp8
    case = s["case"]
    if case["op"] == "quantize":
        q = fp8.quantize(s["x"], block_rows=case["block_rows"])
        return {"read": fp8.dequantize(q, s["x"].dtype), "e": q.exps}
    w = fp8.Fp8Tensor(s["w"][0], s["w"][1], block_rows=128)
    if case["op"] == "ffn":
        h = fp8.linear(fp8.quantize(s["x"]), w, s["w"][2], act="gelu", out_dtype=torch.float8_e4m3fn)
        w2 = fp8.Fp8Tensor(s["w2"][0], s["w2"][1], block_rows=128)
        return fp8.linear(h, w2, s["w2"][2], residual=s["residual"], out_dtype=TYPES[case["out"]])
    x = fp8.Fp8Tensor(s["x"][0], s["x"][1])
    act = "gelu" if case["act"] == "gelu" else None
    if case["out"] == "e4m3":
        y = fp8.linear(x, w, s["w"][2], act=act, out_dtype=torch.float8_e4m3fn)
        return fp8.dequantize(y, torch.bfloat16)
    return fp8.linear(x, w, s["w"][2], act=act, residual=s["residual"], out_dtype=TYPES[case["out"]])


def run(state):
    if own:
        return _run_own(state)
    s, case = state, state["case"]
    if case["op"] == "quantize":
        q, e = _quantize(s["x"], case["block_rows"])
        return {"read": _dequantize(q, e, case["block_rows"]).to(s["x"].dtype), "e": e}
    w = _dequantize(s["w"][0], s["w"][1], 128)
    if case["op"] == "ffn":
        x = _dequantize(*_quantize(s["x"]))
        h = _dequantize(*_quantize(_linear(x, w, s["w"][2], "gelu", None)))
        return _linear(h, _dequantize(s["w2"][0], s["w2"][1], 128), s["w2"][2], "none", s["residual"]).to(TYPES[case["out"]])
    y = _linear(_dequantize(*s["x"]), w, s["w"][2], case["act"], s["residual"])
    if case["out"] == "e4m3":
        return _dequantize(*_quantize(y)).to(torch.bfloat16)
    return y.to(TYPES[case["out"]])


# ---- the definition in 64 bits, apart from the above


def _power(e):
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_store(x, block_rows):
    """The values that x is held as, and the scales, by arithmetic in 64 bits: the scale exponent from
    the logarithm of the block's maximum (mended where the logarithm rounds across a whole number), each
    value rounded to a multiple of its binade's step (3 fraction bits, no step below 2^-9)."""
    x = x.double()
    r, k = x.shape
    rb, kb = -(-r // block_rows), -(-k // 128)
    p = torch.zeros(rb * block_rows, kb * 128, dtype=torch.float64, device=x.device)
    p[:r, :k] = x
    p = p.reshape(rb, block_rows, kb, 128).transpose(1, 2).reshape(rb, kb, block_rows * 128)
    top = p.abs().max(dim=2).values
    e = torch.ceil(torch.log2(top.clamp_min(2.0 ** -150) / 448.0))
    e = torch.where(top > 448.0 * _power(e), e + 1, e)
    e = torch.where(top <= 448.0 * _power(e - 1), e - 1, e).clamp_min(-127.0)
    scale = _power(e)[:, :, None]
    v = p / scale
    _, binade = torch.frexp(v)  # |v| in [2^(binade - 1), 2^binade)
    step = _power((binade - 1).clamp_min(-6) - 3)
    v = torch.round(v / step) * step * scale
    v = v.reshape(rb, kb, block_rows, 128).transpose(1, 2).reshape(rb * block_rows, kb * 128)[:r, :k]
    return v, (e + 127.0).to(torch.uint8)


def _exact_linear(x, held, bias, gelu, residual):
    q, e = held
    scale = _power(e.long() - 127)
    w = q.double() * torch.kron(scale, torch.ones(128, 128, dtype=torch.float64, device=q.device))[: q.shape[0], : q.shape[1]]
    y = torch.addmm(bias.double(), x, w.T)
    if gelu:  # x * sigmoid(2 u) is the tanh form
        y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
    return y if residual is None else y + residual.double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        v, e = _exact_store(s["x"], case["block_rows"])
        return {"read": v, "e": e}
    if case["op"] == "ffn":
        x, _ = _exact_store(s["x"], 1)
        h, _ = _exact_store(_exact_linear(x, s["w"][:2], s["w"][2], True, None), 1)
        return _exact_linear(h, s["w2"][:2], s["w2"][2], False, s["residual"])
    q, e = s["x"]
    x = q.double() * _power(e.long() - 127).repeat_interleave(128, dim=1)[:, : q.shape[1]]
    y = _exact_linear(x, s["w"][:2], s["w"][2], case["act"] == "gelu", s["residual"])
    return _exact_store(y, 1)[0] if case["out"] == "e4m3" else y
