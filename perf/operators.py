"""The 8-bit operators of the library as measurable cases: quantisation by blocks of 128, the matrix product of such
operands, and the root-mean-square norm that feeds it, with its gradient.

A case is one pass through one operator.  `prepare` makes its inputs on the GPU, `run` computes it: in elementary torch
operations in 32 bits where `own` is false, by the calls of the C ABI (backup_1_amd/capi.py) where it is true.

Data layout, as the C ABI takes it: matrices are row-major with a pitch, 8-bit codes are OCP e4m3 or e5m2, the scales of
an M x K operand lie as [ceil(K / 128)][pitch], one for each row (block_rows 1) or each 128 rows (block_rows 128), as fp32
or as a biased exponent of two in 8 bits (e8m0).  A value is code * scale.
"""
import math

import torch

own = False

BLOCK = 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FORMATS = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
EPS = 1e-5


def listed():
    return [
        # activations of a few requests on their way into a product, one token each: latency
        {"name": "quantize_16x4096_f16", "op": "quantize", "M": 16, "K": 4096, "type": "f16", "format": "e4m3", "scale": "f32", "block_rows": 1, "both": False},
        # activations of a training step: rows for the forward product and columns for the weight's gradient
        {"name": "quantize_8192x8192_bf16_both", "op": "quantize", "M": 8192, "K": 8192, "type": "bf16", "format": "e4m3", "scale": "e8m0", "block_rows": 1, "both": True},
        # a weight after its fp32 update, square blocks, as it is and transposed for the input's gradient; ragged
        {"name": "quantize_3000x4500_f32_weight", "op": "quantize", "M": 3000, "K": 4500, "type": "f32", "format": "e4m3", "scale": "f32", "block_rows": 128, "both": True},
        # one token through one layer: reading the weight is all the work
        {"name": "gemm_1x4096x4096", "op": "gemm", "M": 1, "N": 4096, "K": 4096, "type": "bf16", "a": "e4m3", "b": "e4m3", "scale": "f32", "b_rows": 128, "add": False},
        # a batch of decoding requests against a wide layer
        {"name": "gemm_48x8192x4096", "op": "gemm", "M": 48, "N": 8192, "K": 4096, "type": "f16", "a": "e4m3", "b": "e4m3", "scale": "e8m0", "b_rows": 128, "add": False},
        # a prompt of odd length, with no size a multiple of the block: the ragged product of bench.py
        {"name": "gemm_3000x4500x1500", "op": "gemm", "M": 3000, "N": 4500, "K": 1500, "type": "f16", "a": "e4m3", "b": "e4m3", "scale": "f32", "b_rows": 128, "add": False},
        # a weight's gradient: e5m2 gradients and e4m3 activations, both scaled along the tokens, added to what is there
        {"name": "gemm_4096x4096x8192_gradient", "op": "gemm", "M": 4096, "N": 4096, "K": 8192, "type": "f32", "a": "e5m2", "b": "e4m3", "scale": "f32", "b_rows": 1, "add": True},
        # the largest product of bench.py
        {"name": "gemm_8192x8192x8192", "op": "gemm", "M": 8192, "N": 8192, "K": 8192, "type": "bf16", "a": "e4m3", "b": "e4m3", "scale": "e8m0", "b_rows": 128, "add": False},
        # the norm before a layer, one token for each of a few requests
        {"name": "norm_16x4096_bf16", "op": "norm", "M": 16, "K": 4096, "type": "bf16", "format": "e4m3", "scale": "f32", "wide": False},
        # the same over the tokens of a long prompt or a training batch; the training step keeps the wide result too
        {"name": "norm_8192x8192_bf16", "op": "norm", "M": 8192, "K": 8192, "type": "bf16", "format": "e4m3", "scale": "f32", "wide": True},
        # its gradient: a small odd one, and a training batch
        {"name": "norm_gradient_200x1500_f32", "op": "norm_gradient", "M": 200, "K": 1500, "type": "f32"},
        {"name": "norm_gradient_8192x8192_bf16", "op": "norm_gradient", "M": 8192, "K": 8192, "type": "bf16"},
    ]


def draw(rng):
    def size(low, high):
        n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        return n if rng.random() < 0.5 else max(1, n // BLOCK * BLOCK) if n >= BLOCK else n

    op = rng.choice(["quantize", "gemm", "gemm", "norm", "norm_gradient"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "quantize":
        return {"op": op, "M": size(1, 8192), "K": size(64, 8192), "type": kind, "format": rng.choice(["e4m3", "e5m2"]),
                "scale": rng.choice(["f32", "e8m0"]), "block_rows": rng.choice([1, 128]), "both": rng.random() < 0.5}
    if op == "gemm":
        return {"op": op, "M": size(1, 8192), "N": size(64, 8192), "K": size(64, 8192), "type": kind,
                "a": rng.choice(["e4m3", "e4m3", "e5m2"]), "b": rng.choice(["e4m3", "e4m3", "e5m2"]),
                "scale": rng.choice(["f32", "e8m0"]), "b_rows": rng.choice([1, 128]), "add": rng.random() < 0.3}
    if op == "norm":
        # fp32 scales: an exponent of two would go by which side of a border the last bit of a sum falls on
        return {"op": op, "M": size(1, 8192), "K": size(64, 8192), "type": kind, "format": "e4m3", "scale": "f32", "wide": rng.random() < 0.5}
    return {"op": op, "M": size(1, 8192), "K": size(64, 8192), "type": kind}


def work(case):
    M, K = case["M"], case["K"]
    wide = 4 if case.get("type") == "f32" else 2
    blocks = -(-K // BLOCK)
    if case["op"] == "quantize":
        scale = 4 if case["scale"] == "f32" else 1
        rows = M if case["block_rows"] == 1 else -(-M // BLOCK)
        out = M * K + blocks * rows * scale
        if case["both"]:
            out += M * K + -(-M // BLOCK) * (K if case["block_rows"] == 1 else blocks) * scale
        return {"bytes": M * K * wide + out, "flops": 2 * M * K}
    if case["op"] == "gemm":
        N = case["N"]
        scale = 4 if case["scale"] == "f32" else 1
        b_rows = N if case["b_rows"] == 1 else -(-N // BLOCK)
        return {"bytes": M * K + N * K + blocks * (M + b_rows) * scale + M * N * wide * (2 if case["add"] else 1), "flops": 2 * M * N * K}
    if case["op"] == "norm":
        # sum with the residual, its squares, the weight, the codes with their scales, each row's factor
        return {"bytes": M * K * wide * (4 if case["wide"] else 3) + K * wide + M * K + blocks * M * 4 + M * 4, "flops": 8 * M * K}
    return {"bytes": M * K * wide * 4 + K * wide + M * 4 + K * 4, "flops": 12 * M * K}


# ---- inputs

def _up(n, to):
    return -(-n // to) * to


def _pitched(rows, cols, dtype):
    """A rows x cols view of storage whose pitch is the next multiple of 16 elements, as the library's containers have it."""
    return torch.zeros(rows, _up(cols, 16), dtype=dtype, device="cuda")[:, :cols]


def _values(gen, rows, cols, spread, dtype):
    """Normal values with a few channels much larger than the rest, as activations and gradients have them."""
    v = torch.randn(rows, cols, generator=gen, device="cuda") * spread
    v *= 1 + 30 * (torch.rand(cols, generator=gen, device="cuda") < 0.01).float()
    out = _pitched(rows, cols, dtype)
    out.copy_(v)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    M, K, op = case["M"], case["K"], case["op"]
    state = {"case": case}
    if op == "gemm":
        N, dtype = case["N"], TYPES[case["type"]]
        for name, rows, spread, block_rows in (("a", M, 1.0, 1), ("b", N, 0.02, case["b_rows"])):
            codes, scales = _quantize(_values(gen, rows, K, spread, torch.float32), case[name], case["scale"], block_rows)
            state[name] = _pitched(rows, K, torch.uint8)
            state[name].copy_(codes.view(torch.uint8))
            state["scales_" + name] = _pitched(scales.shape[0], scales.shape[1], scales.dtype)
            state["scales_" + name].copy_(scales)
        state["c"] = _values(gen, M, N, 1.0, dtype) if case["add"] else None
        state["d"] = _pitched(M, N, dtype)
        return state
    dtype = TYPES[case["type"]]
    if op == "quantize":
        state["x"] = _values(gen, M, K, 0.02 if case["block_rows"] == BLOCK else 1.0, dtype)
        blocks, blocks_m = -(-K // BLOCK), -(-M // BLOCK)
        scale_type = torch.float32 if case["scale"] == "f32" else torch.uint8
        state["codes"] = _pitched(M, K, torch.uint8)
        state["scales"] = _pitched(blocks, M if case["block_rows"] == 1 else blocks_m, scale_type)
        if case["both"]:
            state["codes_t"] = _pitched(K, M, torch.uint8)
            state["scales_t"] = _pitched(blocks_m, K if case["block_rows"] == 1 else blocks, scale_type)
        return state
    state["w"] = (1 + 0.1 * torch.randn(K, generator=gen, device="cuda")).to(dtype)
    if op == "norm":
        state["x"], state["r"] = _values(gen, M, K, 0.5, dtype), _values(gen, M, K, 2.0, dtype)
        state["h"], state["rstd"] = _pitched(M, K, dtype), torch.zeros(M, device="cuda")
        state["y"] = _pitched(M, K, dtype) if case["wide"] else None
        state["codes"], state["scales"] = _pitched(M, K, torch.uint8), _pitched(-(-K // BLOCK), M, torch.float32)
        return state
    state["h"], state["dy"], state["dr"] = _values(gen, M, K, 2.0, dtype), _values(gen, M, K, 1e-2, dtype), _values(gen, M, K, 1e-2, dtype)
    state["rstd"] = torch.rsqrt(state["h"].float().square().mean(1) + EPS)
    state["dx"], state["dw"] = _pitched(M, K, dtype), torch.zeros(K, device="cuda")
    state["work"] = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    return state


# ---- the operators in their plain form

def _blocks(v, block_rows):
    """v, padded with zeros to whole blocks, as [row block][rows of it][column block][128]."""
    M, K = v.shape
    pad = torch.zeros(_up(M, block_rows), _up(K, BLOCK), dtype=v.dtype, device=v.device)
    pad[:M, :K] = v
    return pad.view(-1, block_rows, pad.shape[1] // BLOCK, BLOCK)


def _quantize(x, fmt, scale, block_rows):
    """Codes in 8 bits and the blocks' scales: fp32 amax / largest (in 64 bits, rounded once), or the least power of two
    that is no smaller, as a biased exponent."""
    M, K = x.shape
    blocks = _blocks(x.float(), block_rows)
    amax = blocks.abs().amax((1, 3)).clamp_min(2.0 ** -100)
    if scale == "f32":
        scales = (amax.double() / torch.full_like(amax, LARGEST[fmt]).double()).float()
        factor = (torch.ones_like(scales).double() / scales.double()).float()
        kept = scales
    else:
        mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, 0.5 <= mantissa < 1; largest = 0.875 * 2^top
        power = exponent - math.frexp(LARGEST[fmt])[1] + (mantissa > 0.875).int()
        factor = ((127 - power) << 23).view(torch.float32)  # 2^-power by its bits: a power function may be a bit off
        kept = (power + 127).to(torch.uint8)
    codes = (blocks * factor[:, None, :, None]).to(FORMATS[fmt]).view(torch.uint8)
    codes = codes.reshape(codes.shape[0] * block_rows, -1)[:M, :K].contiguous()
    return codes.view(FORMATS[fmt]), kept.t().contiguous()


def _scale_values(scales):
    return scales if scales.dtype == torch.float32 else (scales.int() << 23).view(torch.float32)


def _dequantize(codes, fmt, scales, block_rows):
    M, K = codes.shape
    s = _scale_values(scales).t().repeat_interleave(block_rows, 0)[:M].repeat_interleave(BLOCK, 1)[:, :K]
    return codes.contiguous().view(FORMATS[fmt]).float() * s


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op == "quantize":
        codes, scales = _quantize(state["x"], case["format"], case["scale"], case["block_rows"])
        out = {"codes": codes, "scales": scales}
        if case["both"]:
            out["codes_t"], out["scales_t"] = _quantize(state["x"].t(), case["format"], case["scale"], case["block_rows"])
        return {k: _as_values(v) for k, v in out.items()}
    if op == "gemm":
        a = _dequantize(state["a"], case["a"], state["scales_a"], 1)
        b = _dequantize(state["b"], case["b"], state["scales_b"], case["b_rows"])
        d = a @ b.t()
        if state["c"] is not None:
            d += state["c"].float()
        return d.to(TYPES[case["type"]])
    if op == "norm":
        h = (state["x"].float() + state["r"].float()).to(TYPES[case["type"]])
        rstd = 1 / torch.sqrt(h.float().square().mean(1) + EPS)
        y = h.float() * rstd[:, None] * state["w"].float()
        codes, scales = _quantize(y, case["format"], case["scale"], 1)
        out = {"h": h, "rstd": rstd, "codes": codes, "scales": scales}
        if case["wide"]:
            out["y"] = y.to(TYPES[case["type"]])
        return out
    h, dy, rstd = state["h"].float(), state["dy"].float(), state["rstd"][:, None]
    n = h * rstd
    g = dy * state["w"].float()
    dx = rstd * (g - n * (g * n).mean(1, keepdim=True)) + state["dr"].float()
    return {"dx": dx.to(TYPES[case["type"]]), "dw": (dy * n).sum(0)}


def _as_values(v):
    """8-bit exponents as the powers of two that they stand for."""
    return v.view(torch.float8_e8m0fnu) if v.dtype == torch.uint8 else v


# ---- the library's calls

def _calls():
    from backup_1_amd import capi
    if not capi.lib().decx_hip_is_init():
        capi.init()
    return capi


def _own(state):
    capi = _calls()
    case = state["case"]
    op, M, K = case["op"], case["M"], case["K"]
    at = lambda name: state[name].data_ptr() if state.get(name) is not None else None  # noqa: E731
    ld = lambda name: state[name].stride(0) if state.get(name) is not None else 0  # noqa: E731
    kind = {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}[case["type"]]
    fmt = {"e4m3": capi.E4M3, "e5m2": capi.E5M2}
    if op == "quantize":
        capi.f8_quantize(at("x"), ld("x"), kind, M, K, case["block_rows"], fmt[case["format"]], capi.SCALE_F32 if case["scale"] == "f32" else capi.SCALE_E8M0,
                         at("codes"), ld("codes"), at("scales"), ld("scales"), at("codes_t"), ld("codes_t"), at("scales_t"), ld("scales_t"), blocking=False)
        return {k: state[k].view(FORMATS[case["format"]]) if k.startswith("codes") else _as_values(state[k]) for k in ("codes", "scales", "codes_t", "scales_t") if k in state}
    if op == "gemm":
        capi.f8gemm(at("a"), ld("a"), fmt[case["a"]], at("scales_a"), ld("scales_a"), at("b"), ld("b"), fmt[case["b"]], at("scales_b"), ld("scales_b"),
                    case["b_rows"], capi.SCALE_F32 if case["scale"] == "f32" else capi.SCALE_E8M0, at("d"), ld("d"), kind, M, case["N"], K, at("c"), ld("c"), blocking=False)
        return state["d"]
    if op == "norm":
        capi.rmsnorm_f8(at("x"), ld("x"), at("r"), ld("r"), at("w"), EPS, kind, M, K, at("h"), ld("h"), at("rstd"), at("y"), ld("y"),
                        at("codes"), ld("codes"), at("scales"), ld("scales"), fmt[case["format"]], capi.SCALE_F32, blocking=False)
        out = {"h": state["h"], "rstd": state["rstd"], "codes": state["codes"].view(FORMATS[case["format"]]), "scales": state["scales"]}
        if case["wide"]:
            out["y"] = state["y"]
        return out
    capi.rmsnorm_backward(at("h"), ld("h"), at("w"), at("rstd"), at("dy"), ld("dy"), at("dr"), ld("dr"), kind, M, K, at("dx"), ld("dx"), at("dw"),
                          at("work"), state["work"].numel(), blocking=False)
    return {"dx": state["dx"], "dw": state["dw"]}


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions in 64 bits

def _power_of_two(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _on_grid(v, fmt):
    """The nearest value that the format holds, ties to even."""
    bits, least = (3, -6) if fmt == "e4m3" else (2, -14)
    step = _power_of_two(torch.frexp(v)[1].sub(1).clamp_min(least) - bits)
    return (torch.round(v / step) * step).clamp(-LARGEST[fmt], LARGEST[fmt])


def _spread(scales, rows, cols, block_rows):
    """One scale for each element, from scales of [column block][row block]."""
    r = torch.arange(rows, device="cuda") // block_rows
    c = torch.arange(cols, device="cuda") // BLOCK
    return scales.t()[r][:, c]


def _exact_codes(v, fmt, scale, block_rows):
    rows, cols = v.shape
    padded = torch.nn.functional.pad(v.abs(), (0, -cols % BLOCK, 0, -rows % block_rows))
    largest = padded.unflatten(1, (-1, BLOCK)).amax(2).unflatten(0, (-1, block_rows)).amax(1).t().clamp_min(2.0 ** -100)
    s = largest / torch.full_like(largest, LARGEST[fmt])
    if scale == "e8m0":
        mantissa, exponent = torch.frexp(s)
        s = _power_of_two(exponent - (mantissa == 0.5).int())
    return {"codes": _on_grid(v / _spread(s, rows, cols, block_rows), fmt), "scales": s}


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        v = state["x"].double()
        out = _exact_codes(v, case["format"], case["scale"], case["block_rows"])
        if case["both"]:
            t = _exact_codes(v.t(), case["format"], case["scale"], case["block_rows"])
            out["codes_t"], out["scales_t"] = t["codes"], t["scales"]
        return out
    if op == "gemm":
        sides = []
        for name, block_rows in (("a", 1), ("b", case["b_rows"])):
            s = state["scales_" + name]
            s = s.double() if s.dtype == torch.float32 else _power_of_two(s.int() - 127)
            codes = state[name].contiguous().view(FORMATS[case[name]]).double()
            sides.append(codes * _spread(s, codes.shape[0], codes.shape[1], block_rows))
        d = torch.matmul(sides[0], sides[1].t())
        return d if state["c"] is None else d + state["c"].double()
    if op == "norm":
        h = (state["x"].double() + state["r"].double()).to(TYPES[case["type"]])
        v = h.double()
        rstd = (v.pow(2).sum(1) / case["K"] + EPS).pow(-0.5)
        y = v * state["w"].double() * rstd[:, None]
        out = _exact_codes(y, case["format"], case["scale"], 1)
        out["h"], out["rstd"] = v, rstd
        if case["wide"]:
            out["y"] = y
        return out
    h, dy, w, rstd = state["h"].double(), state["dy"].double(), state["w"].double(), state["rstd"].double()
    dot = (dy * w * h).sum(1) / case["K"]
    dx = (dy * w - h * (dot * rstd.pow(2))[:, None]) * rstd[:, None] + state["dr"].double()
    return {"dx": dx, "dw": (dy * h * rstd[:, None]).sum(0)}
