"""The microscaled (MX) operators as they are measured: cases, inputs, plain forms and the framework's calls.

An MX matrix holds, for every 32 consecutive values of a row, a scale 2^e (e8m0: the byte e + 127) and the values
over that scale, rounded to e4m3 ("fp8") or e2m1 ("fp4", the even column in the low half of a byte).
e = max(ceil(log2(amax / vmax)), -126) with vmax = 448 or 6.  Rows are padded with zeros to a multiple of 128 columns,
their scales to a multiple of 16 with 2^0; of each 16 scales, that of block 4 s + g is byte 4 g + s.

  norm      s = x + residual, h = s rounded, y = MX of (norm(s) * weight) * (1 + scale[segment]) + shift[segment]
  quantize  MX of a matrix
  linear    epilogue(x w^T + b) of an MX activation and an MX weight, in bf16 or again in MX
  matvec    epilogue(x w^T + b) of a few bf16 rows and a weight in 4 bits

`own` False: plain torch operations.  `own` True: the calls a user makes of ditserve_amd.mx.
"""
import math

import torch

own = False

DEV = "cuda"
VMAX = {"fp8": 448.0, "fp4": 6.0}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6


def listed():
    return [
        # one timestep's conditioning row per branch of a CFG pair: launch latency
        dict(name="norm_2x1536", kind="norm", rows=2, cols=1536, form="rms", residual=True, segments=0),
        # both branches' text tokens of a joint block at SD3.5-Large's width, modulated LayerNorm
        dict(name="norm_666x2432_mod", kind="norm", rows=666, cols=2432, form="ln", residual=False, segments=2),
        # the video tokens of a 480x832x81 CFG pair, residual and RMS norm
        dict(name="norm_65520x1536", kind="norm", rows=65520, cols=1536, form="rms", residual=True, segments=0),
        # one latent frame's attention output before its projection
        dict(name="quantize_1560x1536", kind="quantize", rows=1560, cols=1536),
        # a 480x832x81 video's attention output at Wan2.1-14B's width
        dict(name="quantize_32760x5120", kind="quantize", rows=32760, cols=5120),
        # Wan's text embedding: 512 encoder rows
        dict(name="linear_512x4096_1536", kind="linear", rows=512, k=4096, n=1536, epilogue="gelu", mx_out=False),
        # the joint block's text qkv at SD3.5-Large's width, an odd number of rows
        dict(name="linear_667x2432_7296", kind="linear", rows=667, k=2432, n=7296, epilogue="bias", mx_out=False),
        # one latent frame's feed-forward input, its output in 8 bits for the next product
        dict(name="linear_1560x1536_8960_mx", kind="linear", rows=1560, k=1536, n=8960, epilogue="gelu", mx_out=True),
        # a CFG pair's feed-forward output with the gated residual
        dict(name="linear_65520x8960_1536", kind="linear", rows=65520, k=8960, n=1536, epilogue="gate_res",
             mx_out=False),
        # one timestep's modulation projection
        dict(name="matvec_1x1536_9216", kind="matvec", rows=1, k=1536, n=9216, epilogue="f32"),
        # a square projection of a few rows at Wan2.1-14B's width
        dict(name="matvec_13x5120_5120", kind="matvec", rows=13, k=5120, n=5120, epilogue="silu"),
        # every block's modulations of an SD3.5-Medium step, stacked
        dict(name="matvec_2x1536_499712", kind="matvec", rows=2, k=1536, n=499712, epilogue="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "quantize", "linear", "linear", "matvec", "matvec"])
    if kind in ("norm", "quantize"):
        cols = 32 * _log(rng, 4, 192)
        rows = _log(rng, 1, 65520 * 1536 // cols)
        if kind == "quantize":
            return dict(kind=kind, rows=rows, cols=cols)
        segments = rng.choice([0, 0, 1, 2, 3])
        if segments:
            rows = max(1, rows // segments) * segments
        return dict(kind=kind, rows=rows, cols=cols, form=rng.choice(["rms", "rms", "ln"]),
                    residual=rng.random() < 0.6, segments=segments)
    if kind == "linear":
        k, n = 32 * _log(rng, 4, 448), 32 * _log(rng, 4, 432)
        rows = _log(rng, 1, min(65520, max(2, 65520 * 8960 * 1536 // (k * n))))
        epilogue = rng.choice(["bias", "gelu", "silu", "res", "gate_res"])
        if epilogue == "gate_res":
            rows += rows % 2
        mx_out = epilogue in ("bias", "gelu", "silu") and rng.random() < 0.5
        return dict(kind=kind, rows=rows, k=k, n=n if mx_out else n - rng.choice([0, 0, 8, 16, 24]), epilogue=epilogue,
                    mx_out=mx_out)
    return dict(kind=kind, rows=_log(rng, 1, 48), k=32 * _log(rng, 4, 448), n=8 * _log(rng, 16, 6400),
                epilogue=rng.choice(["bias", "gelu", "silu", "res", "f32"]))


def _up(n, to):
    return (n + to - 1) // to * to


def work(case):
    r = case["rows"]
    if case["kind"] in ("norm", "quantize"):
        d = case["cols"]
        per = 2 + 1 + 1 / 32 + (4 if case.get("residual") else 0)
        flops = (8 if case["kind"] == "norm" else 2) * r * d
        return {"bytes": r * d * per + 8 * d * case.get("segments", 0) + (4 * d if case["kind"] == "norm" else 0),
                "flops": flops}
    k, n, epi = case["k"], case["n"], case["epilogue"]
    if case["kind"] == "matvec":
        return {"bytes": n * k * (1 / 2 + 1 / 32) + 2 * r * k + (4 if epi == "f32" else 2) * r * n + 4 * n
                + (2 * r * n if epi == "res" else 0), "flops": 2 * r * n * k}
    out = 1 + 1 / 32 if case["mx_out"] else 2
    return {"bytes": (r + n) * k * (1 + 1 / 32) + out * r * n + 4 * n + (2 * r * n if "res" in epi else 0),
            "flops": 2 * r * n * k}


# ---------------------------------------------------------------------------------------------
# plain forms (32 bits)
# ---------------------------------------------------------------------------------------------

def _to_mx(x, fmt="fp8"):
    """(data, scales) of fp32 rows: values in e4m3 or two e2m1 a byte, scales e8m0, padded and ordered as above."""
    rows, cols = x.shape
    v = x.reshape(rows, cols // 32, 32)
    amax = v.abs().amax(2)
    m, e = torch.frexp(amax)  # amax = m 2^e with m in [0.5, 1): vmax = 0.875 2^9 or 0.75 2^3
    top, high = (9, 0.875) if fmt == "fp8" else (3, 0.75)
    e = (e - top + (m > high).to(e.dtype)).clamp_min(-126)
    e = torch.where(amax == 0, torch.full_like(e, -126), e)
    v = torch.ldexp(v, -e.unsqueeze(2)).reshape(rows, cols)
    if fmt == "fp8":
        q = v.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
        a = v.abs()
        low = torch.bucketize(a, mid)               # ties down
        high = torch.bucketize(a, mid, right=True)  # ties up
        code = torch.where(low % 2 == 0, low, high)  # ties to the even code
        code = code + 8 * (v < 0)
        q = (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8)
    wide = _up(cols, 128) // (2 if fmt == "fp4" else 1)
    data = torch.zeros((rows, wide), dtype=torch.uint8, device=x.device)
    data[:, :q.shape[1]] = q
    s = torch.full((rows, _up(cols, 512) // 32), 127, dtype=torch.uint8, device=x.device)
    s[:, :cols // 32] = (e + 127).to(torch.uint8)
    s = s.reshape(rows, -1, 4, 4).transpose(2, 3).reshape(rows, -1)
    if fmt == "fp8":
        data = data.view(torch.float8_e4m3fn)
    return data, s.view(torch.float8_e8m0fnu)


def _from_mx(data, scales, cols, dtype=torch.float32):
    """The fp32 values an MX matrix stands for."""
    rows = data.shape[0]
    s = scales.view(torch.uint8).reshape(rows, -1, 4, 4).transpose(2, 3).reshape(rows, -1)[:, :cols // 32]
    if data.dtype == torch.uint8:
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=dtype, device=data.device)
        v = torch.stack([table[(data & 15).int()], table[(data >> 4).int()]], 2).reshape(rows, -1)
    else:
        v = data.to(dtype)
    v = v[:, :cols].reshape(rows, cols // 32, 32)
    return torch.ldexp(v, (s.int() - 127).unsqueeze(2)).reshape(rows, cols)


def _gelu(y):
    return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))


def _epilogue(y, s, epi):
    if epi == "gelu":
        return _gelu(y)
    if epi == "silu":
        return y / (1 + torch.exp(-y))
    if epi == "res":
        return s["residual"].float() + y
    if epi == "gate_res":
        return s["residual"].float() + y * s["gate"].repeat_interleave(y.shape[0] // 2, 0)
    return y


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "quantize":
        data, scales = _to_mx(s["x"].float())
        return {"y": data, "scales": scales}
    if c["kind"] == "norm":
        x = s["x"].float()
        out = {}
        if c["residual"]:
            x = x + s["residual"].float()
            out["h"] = x.to(torch.bfloat16)
        if c["form"] == "ln":
            x = x - x.mean(1, keepdim=True)
        y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s["weight"]
        if c["segments"]:
            per = c["rows"] // c["segments"]
            y = y * (1 + s["scale"].repeat_interleave(per, 0)) + s["shift"].repeat_interleave(per, 0)
        out["y"], out["scales"] = _to_mx(y)
        return out
    if c["kind"] == "matvec":
        y = s["x"].float() @ _from_mx(s["w"], s["w_scales"], c["k"]).T + s["bias"]
        y = _epilogue(y, s, c["epilogue"])
        return {"y": y if c["epilogue"] == "f32" else y.to(torch.bfloat16)}
    y = _from_mx(s["x"], s["x_scales"], c["k"]) @ _from_mx(s["w"], s["w_scales"], c["k"]).T + s["bias"]
    y = _epilogue(y, s, c["epilogue"])
    if c["mx_out"]:
        data, scales = _to_mx(y)
        return {"y": data, "scales": scales}
    return {"y": y.to(torch.bfloat16)}


# ---------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------

def _run_own(s):
    from ditserve_amd import mx, ops

    c = s["case"]
    if c["kind"] == "quantize":
        y = mx.quantize(s["x"])
        return {"y": y.data, "scales": y.scales}
    if c["kind"] == "norm":
        more = {}
        if c["segments"]:
            seg = ops.Segments.uniform(c["segments"], c["rows"] // c["segments"], s["x"].device)
            more = dict(shift=s["shift"], scale=s["scale"], segments=seg)
        y = mx.norm(s["x"], s.get("residual"), weight=s["weight"], eps=EPS, kind=c["form"], **more)
        if c["residual"]:
            y, h = y
            return {"h": h, "y": y.data, "scales": y.scales}
        return {"y": y.data, "scales": y.scales}
    if c["kind"] == "matvec":
        w = mx.MXTensor("fp4", s["w"], s["w_scales"], c["k"])
        return {"y": mx.matvec(s["x"], w, s["bias"], epilogue=c["epilogue"], residual=s.get("residual"))}
    x = mx.MXTensor("fp8", s["x"], s["x_scales"], c["k"])
    w = mx.MXTensor("fp8", s["w"], s["w_scales"], c["k"])
    more = {}
    if c["epilogue"] == "gate_res":
        more = dict(gate=s["gate"], segments=ops.Segments.uniform(2, c["rows"] // 2, s["x"].device))
    y = mx.linear(x, w, s["bias"], epilogue=c["epilogue"], residual=s.get("residual"),
                  out_fmt="fp8" if c["mx_out"] else None, **more)
    return {"y": y.data, "scales": y.scales} if c["mx_out"] else {"y": y}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

def _activation(g, rows, cols):
    """Token rows as a residual stream has them: each token of a size of its own, and a few wide channels."""
    x = torch.randn((rows, cols), generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn((rows, 1), generator=g, device=DEV))
    return x * torch.where(torch.rand((1, cols), generator=g, device=DEV) < 0.01, 8.0, 1.0)


def _weight(g, n, k, fmt):
    data, scales = [], []
    for i in range(0, n, 65536):  # by parts: a stacked weight in 32 bits, several times over, would be large
        w = torch.randn((min(65536, n - i), k), generator=g, device=DEV) / math.sqrt(k)
        d, s = _to_mx(w, fmt)
        data.append(d.view(torch.uint8))
        scales.append(s.view(torch.uint8))
    d, s = torch.cat(data), torch.cat(scales)
    return (d if fmt == "fp4" else d.view(torch.float8_e4m3fn)), s.view(torch.float8_e8m0fnu)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    bf = torch.bfloat16
    s = {"case": case}
    r = case["rows"]
    if case["kind"] in ("norm", "quantize"):
        d = case["cols"]
        s["x"] = _activation(g, r, d).to(bf)
        if case["kind"] == "norm":
            s["weight"] = 1 + 0.1 * torch.randn(d, generator=g, device=DEV)
            if case["residual"]:
                s["residual"] = (2 * _activation(g, r, d)).to(bf)
            if case["segments"]:
                s["shift"] = 0.3 * torch.randn((case["segments"], d), generator=g, device=DEV)
                s["scale"] = 0.3 * torch.randn((case["segments"], d), generator=g, device=DEV)
        return s
    k, n = case["k"], case["n"]
    s["bias"] = 0.1 * torch.randn(n, generator=g, device=DEV)
    if case["kind"] == "matvec":
        s["x"] = _activation(g, r, k).to(bf)
        s["w"], s["w_scales"] = _weight(g, n, k, "fp4")
    else:
        s["x"], s["x_scales"] = _to_mx(_activation(g, r, k))
        s["w"], s["w_scales"] = _weight(g, n, k, "fp8")
    if "res" in case["epilogue"]:
        s["residual"] = torch.randn((r, n), generator=g, device=DEV).to(bf)
    if case["epilogue"] == "gate_res":
        s["gate"] = torch.randn((2, n), generator=g, device=DEV)
    return s


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------

def _exact_mx(y):
    """(values over their scales, scales) of 64-bit rows, laid out as the MX matrix of them."""
    rows, cols = y.shape
    blocks = y.reshape(rows, -1, 32)
    amax = blocks.abs().max(2).values
    e = torch.ceil(torch.log2(amax / 448.0))
    e = torch.where(amax <= torch.exp2(e - 1) * 448.0, e - 1, e)  # a logarithm that rounded up past a power of two
    e = torch.where(amax > torch.exp2(e) * 448.0, e + 1, e).clamp(min=-126.0)
    v = blocks / torch.exp2(e)[:, :, None]
    # e4m3: 8 steps to each octave, the lowest octave's below 2^-6
    octave = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6)))
    octave = torch.where(torch.exp2(octave) > v.abs().clamp_min(2.0 ** -6), octave - 1, octave)
    step = torch.exp2(octave - 3)
    v = (torch.round(v / step) * step).reshape(rows, cols)
    values = torch.nn.functional.pad(v, (0, -cols % 128))
    scales = torch.nn.functional.pad(torch.exp2(e), (0, -(cols // 32) % 16), value=1.0)
    order = [16 * (i // 16) + 4 * (i % 4) + (i % 16) // 4 for i in range(scales.shape[1])]  # byte i's block
    return values, scales[:, order]


def _exact_values(data, scales, cols):
    """What an MX matrix stands for, in 64 bits, from its bytes."""
    b = data.view(torch.uint8).to(torch.int64)
    if data.dtype == torch.uint8:
        b = torch.cat([(b % 16)[:, :, None], (b // 16)[:, :, None]], 2).flatten(1)
        sign, exp, man, low, bits = b // 8, b // 2 % 4, b % 2, 1, 1
    else:
        sign, exp, man, low, bits = b // 128, b // 8 % 16, b % 8, 7, 3
    frac = man.double() / 2 ** bits
    v = torch.where(exp > 0, (1 + frac) * torch.exp2((exp - low).double()), frac * 2.0 ** (1 - low))
    v = torch.where(sign > 0, -v, v)[:, :cols]
    e = scales.view(torch.uint8).double() - 127
    place = [16 * (i // 16) + 4 * (i % 4) + (i % 16) // 4 for i in range(cols // 32)]  # block i's byte
    return v * torch.exp2(e[:, place]).repeat_interleave(32, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        y, scales = _exact_mx(s["x"].double())
        return {"y": y, "scales": scales}
    if case["kind"] == "norm":
        x = s["x"].double()
        out = {}
        if case["residual"]:
            x = x + s["residual"].double()
            out["h"] = x
        mean = x.sum(1, keepdim=True) / x.shape[1] if case["form"] == "ln" else 0.0
        var = ((x - mean) ** 2).sum(1, keepdim=True) / x.shape[1]
        y = (x - mean) / torch.sqrt(var + EPS) * s["weight"].double()
        if case["segments"]:
            seg = torch.arange(case["rows"], device=DEV) // (case["rows"] // case["segments"])
            y = y * (1 + s["scale"].double())[seg] + s["shift"].double()[seg]
        out["y"], out["scales"] = _exact_mx(y)
        return out
    k, epi = case["k"], case["epilogue"]
    x = s["x"].double() if case["kind"] == "matvec" else _exact_values(s["x"], s["x_scales"], k)
    y = torch.empty((case["rows"], case["n"]), dtype=torch.float64, device=DEV)
    for i in range(0, case["n"], 32768):
        w = _exact_values(s["w"][i:i + 32768], s["w_scales"][i:i + 32768], k)
        torch.mm(x, w.T, out=y[:, i:i + 32768]) if case["n"] <= 32768 else y[:, i:i + 32768].copy_(torch.mm(x, w.T))
    y += s["bias"].double()
    if epi == "gelu":
        y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    elif epi == "silu":
        y = y * torch.sigmoid(y)
    elif epi == "res":
        y = y + s["residual"].double()
    elif epi == "gate_res":
        half = case["rows"] // 2
        y[:half] *= s["gate"][0].double()
        y[half:] *= s["gate"][1].double()
        y += s["residual"].double()
    if case.get("mx_out"):
        values, scales = _exact_mx(y)
        return {"y": values, "scales": scales}
    return {"y": y}
