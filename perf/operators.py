"""The operators over microscaled (MX) blocks, as cases to time: quantising rows into blocks and back, the RMS norm whose rows come
out in 8 bits with scales, the product of such rows with 4-bit weights, and the routed experts' gated FFN over 4-bit weights, for a
chunk of tokens and for single ones.

An MX block is 32 elements along a row that share one E8M0 scale byte s, 2^(s - 127), 255 standing for NaN. Elements are E4M3 (a byte)
or E2M1 (two a byte, the even element in the low half). Quantising takes the largest power of two that the block's largest value holds,
over the format's own, as the scale, and rounds to nearest even, saturating.

Sizes are those of the benchmark's configurations (bench.py) and generic ones inside the operators' documented limits. Weights are
N(0, 0.02) rounded to MX blocks, activations N(0, 1), routes follow a Zipf skew.
"""
from __future__ import annotations

import math
import types

import numpy as np
import torch

own = False

BLOCK = 32
E4M3, E2M1 = 0, 1
BF16, F16, F32 = 0, 1, 2
TYPES = {"f16": (F16, torch.float16), "bf16": (BF16, torch.bfloat16), "f32": (F32, torch.float32)}
FORMATS = {"e4m3": E4M3, "e2m1": E2M1}
GPTOSS = dict(d=2880, f=2880, experts=32, top_k=4, act="clamped", biases=True)   # gpt-oss-20B, whose experts are published in this format
Q35B = dict(d=2048, f=512, experts=256, top_k=8, act="silu", biases=False)       # 35B-A3B
KIMI = dict(d=2304, f=1024, experts=256, top_k=8, act="silu", biases=False)      # Kimi-Linear-48B
MOST_FLOPS = 2000 * 4 * 6 * 2880 * 2880
MOST_BYTES = 92160 * 2880 * 5
MOST_WEIGHTS = 32 * 2880 * 2880


def listed():
    return [
        # the smallest call: one token's fp16 row on its way to an 8-bit product
        dict(name="quantize_f16_e4m3_1x2048", kind="quantize", src="f16", format="e4m3", rows=1, d=2048, pad=0),
        # a model load: one projection of every gpt-oss expert, from bf16 to 4 bits
        dict(name="quantize_bf16_e2m1_92160x2880", kind="quantize", src="bf16", format="e2m1", rows=92160, d=2880, pad=0),
        # a decode step's norm
        dict(name="norm_1x2880", kind="norm", rows=1, d=2880, delta=True, out=True),
        # a long chunk's norm
        dict(name="norm_4096x2304", kind="norm", rows=4096, d=2304, delta=True, out=True),
        # one token through one projection
        dict(name="product_e4m3_1x2880x2880", kind="product", x="e4m3", rows=1, n=2880, k=2880, bias=True, out="f16"),
        # the ragged end of a prompt, an odd number of outputs
        dict(name="product_e4m3_37x2049x2304", kind="product", x="e4m3", rows=37, n=2049, k=2304, bias=False, out="bf16"),
        # a long chunk, 8-bit rows
        dict(name="product_e4m3_4096x4096x2880", kind="product", x="e4m3", rows=4096, n=4096, k=2880, bias=True, out="f16"),
        # a long chunk, both sides in 4 bits
        dict(name="product_e2m1_2048x5760x2880", kind="product", x="e2m1", rows=2048, n=5760, k=2880, bias=False, out="f16"),
        # one token of gpt-oss-20B through its four experts
        dict(GPTOSS, name="decode_gptoss_1", kind="decode", tokens=1, missing=0),
        # sixteen sequences of the Kimi-Linear shape, a token each, some experts not in the pool
        dict(KIMI, name="decode_kimi_16", kind="decode", tokens=16, missing=9),
        # the 512-token chunk over many small experts, unevenly loaded
        dict(Q35B, name="grouped_q35b_512", kind="grouped", tokens=512, skew=1.1),
        # a long chunk of gpt-oss-20B: the largest products, with its biases and activation
        dict(GPTOSS, name="grouped_gptoss_2000", kind="grouped", tokens=2000, skew=0.3),
    ]


def _log(rng, low, high, step=1):
    return max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + step))) // step * step))


def draw(rng):
    kind = rng.choice(["quantize", "norm", "product", "product", "decode", "grouped"])
    if kind == "quantize":
        d = _log(rng, 32, 4096, 32)
        rows = _log(rng, 1, MOST_BYTES // 8 // d)
        return dict(kind=kind, src=rng.choice(["f16", "bf16", "f32"]), format=rng.choice(["e4m3", "e2m1"]), rows=rows, d=d,
                    pad=rng.choice([0, 0, 8, 40]))
    if kind == "norm":
        return dict(kind=kind, rows=_log(rng, 1, 16384), d=_log(rng, 64, 4096, 32), delta=rng.random() < 0.8, out=rng.random() < 0.7)
    if kind == "product":
        n, k = _log(rng, 16, 8192), _log(rng, 32, 8192, 32)
        rows = _log(rng, 1, min(8192, MOST_FLOPS // (2 * n * k)))
        return dict(kind=kind, x=rng.choice(["e4m3", "e4m3", "e2m1"]), rows=rows, n=n, k=k, bias=rng.random() < 0.5,
                    out=rng.choice(["f16", "f16", "bf16"]))
    experts = rng.choice([8, 32, 64, 128, 256])
    d = _log(rng, 256, 4096, 64)
    f = min(_log(rng, 128, 4096, 64), max(64, MOST_WEIGHTS // experts // d // 64 * 64))
    shape = dict(d=d, f=f, experts=experts, top_k=rng.choice([1, 2, 4, 6, 8]), act=rng.choice(["silu", "gelu", "clamped"]),
                 biases=rng.random() < 0.3)
    if kind == "decode":
        return dict(shape, kind=kind, tokens=rng.randint(1, 16), missing=rng.choice([0, 0, experts // 4]))
    most = MOST_FLOPS // (6 * d * f * shape["top_k"])
    return dict(shape, kind=kind, tokens=_log(rng, 17, max(17, min(4096, most))), skew=rng.choice([0.0, 0.5, 1.1]))


def _row_bytes(fmt, d):
    return (d if fmt == "e4m3" else d // 2) + d // BLOCK


def work(case):
    kind = case["kind"]
    if kind == "quantize":
        n, size = case["rows"] * case["d"], 4 if case["src"] == "f32" else 2
        return dict(bytes=n * (size + 2) + 2 * case["rows"] * _row_bytes(case["format"], case["d"]), flops=2 * n)
    if kind == "norm":
        n = case["rows"] * case["d"]
        moved = n * (2 + 2 + (2 if case["out"] else 0) + (4 if case["delta"] else 0))
        return dict(bytes=moved + 2 * case["rows"] * _row_bytes("e4m3", case["d"]) + 2 * case["d"], flops=6 * n)
    if kind == "product":
        rows, n, k = case["rows"], case["n"], case["k"]
        return dict(bytes=n * _row_bytes("e2m1", k) + rows * _row_bytes(case["x"], k) + rows * n * 2,
                    flops=2 * rows * n * k)
    d, f, pairs = case["d"], case["f"], case["tokens"] * case["top_k"]
    used = case["experts"] * (1 - (1 - case["top_k"] / case["experts"]) ** case["tokens"])
    weights = used * (2 * f * _row_bytes("e2m1", d) + d * _row_bytes("e2m1", f))
    out = case["tokens"] * d * 4 if kind == "decode" else pairs * d * 2
    return dict(bytes=weights + case["tokens"] * _row_bytes("e4m3", d) + out, flops=6 * pairs * d * f)


# ---------------------------------------------------------------- the plain forms

def _power(e):
    """2^e for int32 exponents from -127 to 127, from its bits."""
    return torch.where(e < -126, 1 << 22, (e + 127) << 23).to(torch.int32).view(torch.float32)


def _scale_of(s):
    """2^(s - 127) of scale bytes, NaN at 255."""
    return torch.where(s == 255, torch.nan, _power(s.to(torch.int32).clamp(max=254) - 127))


def _quantize(x, fmt):
    """fp32 rows -> (element values, scale bytes): elements as the fp32 values that they stand for, unscaled."""
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    bad = ~torch.isfinite(b).all(-1)
    amax = torch.where(bad, 0.0, b.abs().amax(-1))
    exponent = (amax.view(torch.int32) >> 23) & 255
    s = (exponent - (8 if fmt == "e4m3" else 2)).clamp(min=0)
    v = torch.where(bad[..., None], 0.0, b) * _power(127 - s)[..., None]
    v = v.clamp(-448.0, 448.0) if fmt == "e4m3" else v.clamp(-6.0, 6.0)
    bits, low = (3, -6) if fmt == "e4m3" else (1, 0)  # of the mantissa, and the smallest normal's exponent
    step = _power((torch.frexp(v.abs())[1] - 1).clamp(min=low) - bits)
    v = torch.round(v / step) * step
    return v.reshape(x.shape), torch.where(bad, 255, s).to(torch.uint8)


def _blocks_times(v, s):
    return (v.reshape(*v.shape[:-1], -1, BLOCK) * _scale_of(s)[..., None]).reshape(v.shape)


def _codes4(v):
    """E2M1 values -> two codes a byte."""
    a = v.abs()
    mag = torch.where(a < 2.0, a * 2.0, torch.where(a < 4.0, a + 2.0, a / 2.0 + 4.0)).to(torch.uint8)
    c = mag | (torch.signbit(v).to(torch.uint8) << 3)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _values4(codes):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    m = (c & 7).to(torch.float32)
    a = torch.where(m < 4.0, m * 0.5, torch.where(m < 6.0, m - 2.0, 2.0 * m - 8.0))
    return torch.where(c > 7, -a, a)


def _values(codes, s, fmt):
    """The fp32 values of codes and their scale bytes."""
    return _blocks_times(_values4(codes) if fmt == "e2m1" else codes.view(torch.float8_e4m3fn).to(torch.float32), s)


def _glu(gate, up, act):
    if act == "clamped":
        gate, up = gate.clamp(max=7.0), up.clamp(-7.0, 7.0)
        return gate / (1.0 + torch.exp(-1.702 * gate)) * (up + 1.0)
    if act == "silu":
        return gate / (1.0 + torch.exp(-gate)) * up
    inner = (0.7978845608028654 * (gate + 0.044715 * gate * gate * gate)).clamp(-20.0, 20.0)
    return 0.5 * gate * (1.0 + torch.tanh(inner)) * up


def _experts(st, x, expert):
    """The experts' outputs, fp32[pairs, d], of the rows x[pairs] at expert[pairs]. Rows are laid out by expert in a padded block, `most`
    of them each; where there are fewer pairs than experts, every pair takes a copy of its expert for itself."""
    case, w = st["case"], st["w"]
    pairs, experts, most, cell_of = x.shape[0], case["experts"], st["most"], st["cells"]
    if pairs < experts:
        cell_of, expert, experts, most = cell_of[expert], torch.arange(pairs, device=x.device), pairs, 1
    order = torch.argsort(expert, stable=True)
    e = expert[order]
    place = torch.arange(pairs, device=x.device) - torch.searchsorted(e, torch.arange(experts, device=x.device))[e]
    rows = torch.zeros(experts, most, case["d"], device=x.device)
    rows[e, place] = x[order]
    bias = {p: w[p + "_bias"][cell_of].to(torch.float32)[:, None, :] if case["biases"] else 0.0 for p in ("gate", "up", "down")}

    def times(a, p):
        m = _values(w[p][cell_of], w[p + "_scales"][cell_of], "e2m1")
        return torch.bmm(a, m.transpose(1, 2).contiguous()) + bias[p]

    act = _blocks_times(*_quantize(_glu(times(rows, "gate"), times(rows, "up"), case["act"]), "e4m3"))
    y = torch.empty(pairs, case["d"], device=x.device)
    y[order] = times(act, "down")[e, place]
    return y


# ---------------------------------------------------------------- inputs

def _parts(case):
    """An expert's blob: (name, byte offset, shape, type) of its parts, and its size."""
    d, f = case["d"], case["f"]
    parts, at = [], 0
    for name, rows, n in (("gate", f, d), ("up", f, d), ("down", d, f)):
        for part, size in ((name, n // 2), (name + "_scales", n // BLOCK)):
            parts.append((part, at, (rows, size), torch.uint8))
            at += rows * size
    if case["biases"]:
        for name, n in (("gate_bias", f), ("up_bias", f), ("down_bias", d)):
            parts.append((name, at, (n,), torch.bfloat16))
            at += n * 2
    return parts, at


def _weights(case, rng, dev):
    """The experts' blobs, a cell each, and views of their parts by name."""
    parts, size = _parts(case)
    stride = -(-size // 16384) * 16384
    blobs = torch.zeros(case["experts"], stride, dtype=torch.uint8, device=dev)
    w = {}
    for name, at, shape, dtype in parts:
        n = math.prod(shape) * (2 if dtype == torch.bfloat16 else 1)
        w[name] = blobs[:, at:at + n].view(dtype).view(case["experts"], *shape) if dtype == torch.uint8 else \
            blobs[:, at:at + n].contiguous().view(dtype)
    for name, at, shape, dtype in parts:
        if dtype == torch.bfloat16:
            w[name] = torch.randn(case["experts"], *shape, generator=rng, device=dev).mul_(0.1).to(dtype)
            blobs[:, at:at + 2 * shape[0]] = w[name].view(torch.uint8)
        elif not name.endswith("_scales"):
            for first in range(0, case["experts"], 32):
                cells = slice(first, min(first + 32, case["experts"]))
                v, s = _quantize(torch.randn(cells.stop - first, shape[0], shape[1] * 2, generator=rng, device=dev).mul_(0.02), "e2m1")
                w[name][cells], w[name + "_scales"][cells] = _codes4(v), s
    return blobs, w


def _rows(rows, d, fmt, rng, dev):
    v, s = _quantize(torch.randn(rows, d, generator=rng, device=dev), fmt)
    return (_codes4(v) if fmt == "e2m1" else v.to(torch.float8_e4m3fn).view(torch.uint8)), s


def _routes(case, seed, skew):
    """int64[tokens, top_k] of distinct experts, by a Zipf skew over a shuffled order of them; fp16 weights that sum to one."""
    r = np.random.default_rng(seed)
    popular = -skew * np.log1p(r.permutation(case["experts"]))
    score = popular + r.gumbel(size=(case["tokens"], case["experts"]))
    idx = np.argsort(-score, axis=1)[:, :case["top_k"]]
    e = np.exp(r.standard_normal(idx.shape))
    return np.ascontiguousarray(idx), (e / e.sum(1, keepdims=True)).astype(np.float16)


def prepare(case, seed):
    dev = torch.device("cuda")
    rng = torch.Generator(device=dev).manual_seed(seed)
    kind = case["kind"]
    st = dict(case=case)
    if kind == "quantize":
        t = TYPES[case["src"]][1]
        st["x"] = torch.randn(case["rows"], case["d"] + case["pad"], generator=rng, device=dev).mul_(0.02 if case["format"] == "e2m1" else 1.0).to(t)
        return st
    if kind == "norm":
        shape = (case["rows"], case["d"])
        st["hidden"] = torch.randn(shape, generator=rng, device=dev).to(torch.float16)
        st["delta"] = torch.randn(shape, generator=rng, device=dev).mul_(0.3).to(torch.float16) if case["delta"] else None
        st["weight"] = torch.rand(case["d"], generator=rng, device=dev).add_(0.5).to(torch.bfloat16)
        return st
    if kind == "product":
        st["x"], st["x_scales"] = _rows(case["rows"], case["k"], case["x"], rng, dev)
        v, st["w_scales"] = _quantize(torch.randn(case["n"], case["k"], generator=rng, device=dev).mul_(0.02), "e2m1")
        st["w"] = _codes4(v)
        st["bias"] = torch.randn(case["n"], generator=rng, device=dev).mul_(0.1).to(torch.bfloat16) if case["bias"] else None
        return st
    st["blobs"], st["w"] = _weights(case, rng, dev)
    st["x"], st["x_scales"] = _rows(case["tokens"], case["d"], "e4m3", rng, dev)
    idx, weights = _routes(case, seed, case.get("skew", 0.5))
    st["most"] = int(np.bincount(idx.reshape(-1)).max())  # rows of the busiest expert: the plain form's padding
    st["idx"] = torch.from_numpy(idx.astype(np.int32)).to(dev)
    st["weights"] = torch.from_numpy(weights).to(dev)
    cells = np.random.default_rng(seed + 1).permutation(case["experts"])  # the cell that holds an expert
    st["cells"] = torch.from_numpy(cells).to(dev)
    if kind == "decode":
        st["residual"] = torch.randn(case["tokens"], case["d"], generator=rng, device=dev).to(torch.float16)
        slots = cells[idx]
        slots[idx < case["missing"]] = 0xFFFFFFFF  # these experts are not in the pool
        st["slots"] = torch.from_numpy(slots.astype(np.uint32).view(np.int32)).to(dev)
    else:
        st["residency"] = torch.from_numpy(cells.astype(np.int64) | (2 << 32)).to(dev)
    if own:  # what a program that uses the library keeps: the layer's handle, the pool's place, the route buffers
        from shrike_amd import capi, runtime as rt
        act = {"gelu": capi.ACT_GELU_TANH, "silu": capi.ACT_SILU, "clamped": capi.ACT_CLAMPED_SWIGLU}[case["act"]]
        st["moe"] = rt.MoE(case["d"], case["f"], case["experts"], case["top_k"], activation=act, additive_biases=case["biases"])
        st["offsets"], _ = rt.mx_expert_offsets(case["d"], case["f"], case["biases"])
        bases = capi.PoolBases()
        bases.base[0], bases.cells_per_chunk = st["blobs"].data_ptr(), case["experts"]
        st["pool"] = types.SimpleNamespace(bases=bases, stride=st["blobs"].shape[1])
        if kind == "decode":
            st["workspace"] = rt.DeviceBuffer(st["moe"].mx_decode_workspace_bytes(case["tokens"]))
        else:
            st["prefill"] = rt.Prefill(st["moe"])
            st["routes"] = rt.GroupedRoutesDevice(case["tokens"] * case["top_k"], case["experts"])
            st["workspace"] = rt.DeviceBuffer(st["prefill"].mx_ffn_workspace_bytes(st["routes"].max_row_tiles))
    return st


# ---------------------------------------------------------------- one pass

def _run_own(st):
    from shrike_amd import runtime as rt
    case = st["case"]
    kind = case["kind"]
    new = lambda *shape, dtype=torch.uint8: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    if kind == "quantize":
        x, fmt, rows, d = st["x"], case["format"], case["rows"], case["d"]
        codes, scales, values = new(rows, d if fmt == "e4m3" else d // 2), new(rows, d // BLOCK), new(rows, d, dtype=torch.bfloat16)
        rt.mx_quantize(x.data_ptr(), TYPES[case["src"]][0], x.stride(0), FORMATS[fmt], codes.data_ptr(), scales.data_ptr(), rows, d)
        rt.mx_dequantize(codes.data_ptr(), scales.data_ptr(), FORMATS[fmt], values.data_ptr(), BF16, d, rows, d)
        return dict(values=values, scales=scales)
    if kind == "norm":
        rows, d = case["rows"], case["d"]
        total = new(rows, d, dtype=torch.float16) if case["delta"] else None
        out = new(rows, d, dtype=torch.float16) if case["out"] else None
        codes, scales, values = new(rows, d), new(rows, d // BLOCK), new(rows, d, dtype=torch.bfloat16)
        rt.residual_add_rmsnorm_bf16w_mx8(st["hidden"].data_ptr(), st["delta"].data_ptr() if case["delta"] else None, st["weight"].data_ptr(),
                                          total.data_ptr() if case["delta"] else None, out.data_ptr() if case["out"] else None,
                                          codes.data_ptr(), scales.data_ptr(), d, 1e-6, rows)
        rt.mx_dequantize(codes.data_ptr(), scales.data_ptr(), E4M3, values.data_ptr(), BF16, d, rows, d)
        return dict(total=total, out=out, values=values)
    if kind == "product":
        rows, n, k = case["rows"], case["n"], case["k"]
        code, dtype = TYPES[case["out"]]
        out = new(rows, n, dtype=dtype)
        rt.mx_product(st["x"].data_ptr(), st["x_scales"].data_ptr(), FORMATS[case["x"]], st["w"].data_ptr(), st["w_scales"].data_ptr(),
                      st["bias"].data_ptr() if case["bias"] else None, out.data_ptr(), code, n, rows, n, k)
        return out
    tokens, top_k, d = case["tokens"], case["top_k"], case["d"]
    if kind == "decode":
        y = new(tokens, d, dtype=torch.float16)
        st["moe"].encode_mx_decode_ffn(st["pool"], st["slots"].data_ptr(), st["offsets"], st["x"].data_ptr(), st["x_scales"].data_ptr(),
                                       st["weights"].data_ptr(), st["residual"].data_ptr(), y.data_ptr(), None, st["workspace"], top_k, tokens)
        return y
    partials = new(tokens * top_k, d, dtype=torch.float16)
    st["prefill"].group_pairs(st["idx"].data_ptr(), st["weights"].data_ptr(), tokens, top_k, case["experts"], st["routes"],
                              residency=st["residency"].data_ptr())
    st["prefill"].encode_mx_grouped_expert_gemms(st["pool"], st["offsets"], st["routes"], st["x"].data_ptr(), st["x_scales"].data_ptr(),
                                                 partials.data_ptr(), st["workspace"], tokens, top_k)
    return partials


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    kind = case["kind"]
    if kind == "quantize":
        v, s = _quantize(st["x"][:, :case["d"]].to(torch.float32), case["format"])
        return dict(values=_blocks_times(v, s).to(torch.bfloat16), scales=s)
    if kind == "norm":
        total = None
        h = st["hidden"]
        if case["delta"]:
            h = total = (h.to(torch.float32) + st["delta"].to(torch.float32)).to(torch.float16)
        wide = h.to(torch.float32)
        inv = 1.0 / torch.sqrt((wide * wide).mean(-1, keepdim=True, dtype=torch.float64) + 1e-6)
        out = (wide * inv.to(torch.float32) * st["weight"].to(torch.float32)).to(torch.float16)
        values = _blocks_times(*_quantize(out.to(torch.float32), "e4m3")).to(torch.bfloat16)
        return dict(total=total, out=out if case["out"] else None, values=values)
    if kind == "product":
        y = _values(st["x"], st["x_scales"], case["x"]) @ _values(st["w"], st["w_scales"], "e2m1").t()
        if case["bias"]:
            y = y + st["bias"].to(torch.float32)
        return y.to(TYPES[case["out"]][1])
    x = _values(st["x"], st["x_scales"], "e4m3")
    tokens, top_k = case["tokens"], case["top_k"]
    y = _experts(st, x.repeat_interleave(top_k, 0), st["idx"].reshape(-1).to(torch.int64))
    if kind == "grouped":
        return y.to(torch.float16)
    share = st["weights"].to(torch.float32) * (st["slots"] != -1)
    return (st["residual"].to(torch.float32) + (y.view(tokens, top_k, -1) * share[..., None]).sum(1)).to(torch.float16)


# ---------------------------------------------------------------- the definition, in 64 bits

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _grid(fmt):
    """The format's non-negative values in rising order; a value's index is its code."""
    if fmt == "e2m1":
        return torch.tensor(_E2M1, dtype=torch.float64, device="cuda")
    c = torch.arange(127, dtype=torch.float64, device="cuda")
    e, m = torch.div(c, 8, rounding_mode="floor"), c % 8
    return torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.exp2(e - 7))


def _rounded(x, fmt):
    """float64 -> (the values that the MX blocks of x stand for, scale bytes), by the nearest value of the format's grid."""
    grid = _grid(fmt)
    b = x.reshape(-1, BLOCK)
    top = b.abs().amax(1)
    power = torch.where(top > 0, torch.floor(torch.log2(top)), -200.0)
    power = torch.where(torch.exp2(power) > top, power - 1, torch.where(torch.exp2(power + 1) <= top, power + 1, power))
    power = torch.clamp(power - (8 if fmt == "e4m3" else 2), min=-127.0)
    scale = torch.exp2(power)[:, None]
    v = (b / scale).abs().contiguous()
    up = torch.searchsorted(grid, v).clamp(max=len(grid) - 1)
    down = (up - 1).clamp(min=0)
    a, c = grid[down], grid[up]
    take_up = (v - a > c - v) | ((v - a == c - v) & (up % 2 == 0))
    q = torch.where(take_up, c, a) * torch.sign(b) * scale
    return q.reshape(x.shape), (power + 127).to(torch.uint8).reshape(*x.shape[:-1], -1)


def _wide4(codes, s):
    table = torch.tensor([*_E2M1, *(-v for v in _E2M1)], dtype=torch.float64, device=codes.device)
    v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).flatten(-2)
    return v * torch.exp2(s.double() - 127).repeat_interleave(BLOCK, -1)


def _wide8(codes, s):
    c = codes.long()
    return torch.where(c > 127, -1.0, 1.0) * _grid("e4m3")[c & 127] * torch.exp2(s.double() - 127).repeat_interleave(BLOCK, -1)


def _wide_glu(g, u, act):
    if act == "clamped":
        g = torch.minimum(g, torch.full_like(g, 7.0))
        return g * torch.sigmoid(1.702 * g) * (torch.clamp(u, -7.0, 7.0) + 1)
    if act == "silu":
        return g * torch.sigmoid(g) * u
    return g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)) * u


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        values, scales = _rounded(st["x"][:, :case["d"]].double(), case["format"])
        return dict(values=values, scales=None)
    if kind == "norm":
        h = st["hidden"].double()
        if case["delta"]:
            h = (h + st["delta"].double()).to(torch.float16).double()  # the residual stream is held in fp16
        out = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * st["weight"].double()
        values, _ = _rounded(out.to(torch.float16).double(), "e4m3")
        return dict(total=h if case["delta"] else None, out=out if case["out"] else None, values=values)
    if kind == "product":
        y = (_wide8 if case["x"] == "e4m3" else _wide4)(st["x"], st["x_scales"]) @ _wide4(st["w"], st["w_scales"]).t()
        return y + st["bias"].double() if case["bias"] else y
    x, idx, w = _wide8(st["x"], st["x_scales"]), st["idx"].long(), st["w"]
    y = torch.zeros(case["tokens"], case["top_k"], case["d"], dtype=torch.float64, device=x.device)
    for e, cell in enumerate(st["cells"].tolist()):
        token, rank = torch.nonzero(idx == e, as_tuple=True)
        if len(token) == 0:
            continue
        part = lambda a, p: a @ _wide4(w[p][cell], w[p + "_scales"][cell]).t() + (w[p + "_bias"][cell].double() if case["biases"] else 0)  # noqa: B023, E731
        act, _ = _rounded(_wide_glu(part(x[token], "gate"), part(x[token], "up"), case["act"]), "e4m3")
        y[token, rank] = part(act, "down")
    if kind == "grouped":
        return y.reshape(-1, case["d"])
    share = st["weights"].double() * (st["slots"] != -1)
    return st["residual"].double() + (y * share[..., None]).sum(1)
