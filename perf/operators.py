"""Cases of the low-precision and block operators for timing and comparison.

Four operators of the acoustic model's serving path, each beside its plain form in elementary
torch operations:

* ``quantize``: rows to microscaled 4-bit floating point (MXFP4: E2M1 elements, one E8M0 power of
  two for every 32 of them) and back to the values that the codes stand for;
* ``linear``: y = act(q(x) q(w)^T + b), both operands in MXFP4, sums in 32 bits;
* ``conv``: the same product over the taps of a 'same'-padded one-dimensional convolution;
* ``norm``: the end of one block and the start of the next,
  y = residual + scale * gate * Norm_post(u), z = Norm_pre(y).

``own`` selects between the two forms.  Weights are quantised once, in `prepare`, as a serving
program does; activations are quantised inside the call.
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_DEVICE = "cuda"


def listed():
    return [
        # one sentence of phonemes at the width of the encoder's convolutions: launch latency
        {"name": "quantize_sentence", "op": "quantize", "rows": 165, "cols": 256, "type": "fp32"},
        # the BiLSTM output of 64 utterances of 865 frames: memory traffic
        {"name": "quantize_batch", "op": "quantize", "rows": 55360, "cols": 1024, "type": "bf16"},
        # a width that is no multiple of the block, rows that are not 16-byte aligned
        {"name": "quantize_ragged", "op": "quantize", "rows": 997, "cols": 1001, "type": "fp16"},
        # the input gates of both directions of a BiLSTM layer (4 x 512 x 2) for a single row
        {"name": "linear_token", "op": "linear", "rows": 1, "cols": 1024, "out": 4096, "type": "bf16",
         "bias": True, "act": "none"},
        # the mel head over one utterance at the reference's padded length
        {"name": "linear_mel_head", "op": "linear", "rows": 865, "cols": 256, "out": 80, "type": "fp32",
         "bias": True, "act": "none"},
        # the gates of a BiLSTM layer over 64 sentences of 165 phonemes
        {"name": "linear_gates", "op": "linear", "rows": 10560, "cols": 1024, "out": 4096, "type": "bf16",
         "bias": True, "act": "none"},
        # a large product of generic size: the matrix cores
        {"name": "linear_large", "op": "linear", "rows": 8192, "cols": 8192, "out": 8192, "type": "bf16",
         "bias": False, "act": "none"},
        # the encoder's first convolution over one sentence
        {"name": "conv_sentence", "op": "conv", "batch": 1, "time": 165, "cols": 256, "out": 256, "taps": 5,
         "dilation": 2, "type": "fp32", "act": "relu"},
        # a convolution of the duration predictor's kind over 64 padded utterances
        {"name": "conv_batch", "op": "conv", "batch": 64, "time": 865, "cols": 256, "out": 256, "taps": 3,
         "dilation": 1, "type": "bf16", "act": "relu"},
        # the norm after a convolution of one sentence, as the encoder's blocks end
        {"name": "norm_sentence", "op": "norm", "batch": 1, "time": 165, "cols": 256, "type": "fp32",
         "kind": "layer", "post": True, "pre": False, "residual": False, "gate": "none", "scale": "none"},
        # a whole block boundary over a batch: norm, element gate, residual with a scale per channel, next norm
        {"name": "norm_batch", "op": "norm", "batch": 64, "time": 865, "cols": 1024, "type": "bf16",
         "kind": "rms", "post": True, "pre": True, "residual": True, "gate": "element", "scale": "channel"},
        # an odd width and a gate for each utterance, broadcast over its frames
        {"name": "norm_ragged", "op": "norm", "batch": 7, "time": 143, "cols": 5003, "type": "fp16",
         "kind": "layer", "post": True, "pre": True, "residual": True, "gate": "batch", "scale": "number"},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "conv", "norm"])
    kind = rng.choice(["fp32", "bf16", "fp16"])
    if op == "quantize":
        cols = _log_uniform(rng, 1, 8192)
        return {"op": op, "rows": _log_uniform(rng, 1, max(1, min(65536, (1 << 25) // cols))), "cols": cols,
                "type": kind}
    if op == "linear":
        cols, out = _log_uniform(rng, 16, 8192), _log_uniform(rng, 8, 8192)
        return {"op": op, "rows": _log_uniform(rng, 1, 8192), "cols": cols, "out": out, "type": kind,
                "bias": rng.random() < 0.5, "act": rng.choice(["none", "relu"])}
    if op == "conv":
        return {"op": op, "batch": _log_uniform(rng, 1, 32), "time": _log_uniform(rng, 1, 1000),
                "cols": _log_uniform(rng, 16, 512), "out": _log_uniform(rng, 8, 512), "taps": rng.randint(1, 7),
                "dilation": rng.randint(1, 4), "type": kind, "act": rng.choice(["none", "relu"])}
    cols, post = _log_uniform(rng, 8, 8192), rng.random() < 0.8
    return {"op": op, "batch": rng.randint(1, 16), "time": _log_uniform(rng, 1, max(1, min(4096, (1 << 20) // cols))),
            "cols": cols, "type": kind, "kind": rng.choice(["layer", "rms"]), "post": post,
            "pre": rng.random() < 0.6 or not post, "residual": rng.random() < 0.7,
            "gate": rng.choice(["none", "element", "batch"]), "scale": rng.choice(["none", "number", "channel"])}


# -- inputs -----------------------------------------------------------------------------
def _activations(gen, rows, cols, dtype):
    """Rows of different loudness, a few channels far above the rest, one row in sixteen zero (padding)."""
    x = torch.randn((rows, cols), generator=gen, device=_DEVICE)
    x *= torch.exp(torch.randn((rows, 1), generator=gen, device=_DEVICE))
    x *= 1 + 15 * (torch.rand((1, cols), generator=gen, device=_DEVICE) < 0.01)
    x *= torch.rand((rows, 1), generator=gen, device=_DEVICE) >= 1 / 16
    return x.to(dtype)


def _inputs(case, seed):
    gen = torch.Generator(device=_DEVICE)
    gen.manual_seed(seed)
    op, dtype = case["op"], _DTYPES[case["type"]]
    if op == "quantize":
        return {"x": _activations(gen, case["rows"], case["cols"], dtype)}
    if op == "linear":
        m, k, n = case["rows"], case["cols"], case["out"]
        return {"x": _activations(gen, m, k, dtype),
                "w": torch.randn((n, k), generator=gen, device=_DEVICE) / math.sqrt(k),
                "b": 0.1 * torch.randn(n, generator=gen, device=_DEVICE) if case["bias"] else None}
    if op == "conv":
        b, t, c, n, j = case["batch"], case["time"], case["cols"], case["out"], case["taps"]
        return {"x": _activations(gen, b * t, c, dtype).reshape(b, t, c),
                "w": torch.randn((n, j, c), generator=gen, device=_DEVICE) / math.sqrt(j * c),
                "b": 0.1 * torch.randn(n, generator=gen, device=_DEVICE)}
    b, t, c = case["batch"], case["time"], case["cols"]

    def rand(*shape):
        return torch.randn(shape, generator=gen, device=_DEVICE)

    def vector(centre):
        return centre + 0.1 * rand(c)

    layer = case["kind"] == "layer"
    return {"u": (0.5 + 2 * rand(b, t, c)).to(dtype),
            "post": (vector(1.0), vector(0.0) if layer else None) if case["post"] else None,
            "pre": (vector(1.0), vector(0.0) if layer else None) if case["pre"] else None,
            "residual": (3 * rand(b, t, c)).to(dtype) if case["residual"] else None,
            "gate": {"none": lambda: None, "element": lambda: rand(b, t, c).to(dtype),
                     "batch": lambda: rand(b, 1, c).to(dtype)}[case["gate"]](),
            "scale": {"none": lambda: None, "number": lambda: 0.5, "channel": lambda: vector(0.5)}[case["scale"]]()}


_EPS = 1e-3  # the epsilon of the acoustic model's norms


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if "w" in state:  # a serving program keeps the weights quantised
        w = state.pop("w")
        if own:
            import tts_amd
            state["weight"] = tts_amd.mxfp4_quantize(w)
        else:
            state["weight"] = _encode(w)
    if own and case["op"] == "norm":
        import tts_amd
        for side in ("post", "pre"):
            if state[side] is not None:
                state[side] = tts_amd.Norm(*state[side], eps=_EPS, kind=case["kind"])
    return state


# -- plain forms ------------------------------------------------------------------------
_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _power_of_two(e):
    """2 ** e in float32 for integers e in [-126, 127]."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _blocks(x):
    cols = x.shape[-1]
    pad = -cols % 32
    if pad:
        x = torch.nn.functional.pad(x, (0, pad))
    return x.reshape(*x.shape[:-1], -1, 32)


def _encode(x):
    """(codes 0..15, one byte each; biased exponents of the blocks' scales; columns)."""
    v = _blocks(x.float())
    top = v.abs().amax(-1, keepdim=True)
    biased = ((top.view(torch.int32) >> 23) - 2).clamp_min(0)
    y = v * _power_of_two(127 - biased)
    m = y.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
    code = code + 8 * (y < 0)
    biased = torch.where(torch.isfinite(top), biased, 255)
    return code.to(torch.uint8), biased.to(torch.uint8), x.shape[-1]


def _decode(q):
    code, biased, cols = q
    table = torch.tensor(_MAGNITUDES + tuple(-v for v in _MAGNITUDES), device=code.device)
    e = biased.to(torch.int32)
    # 2 ** (e - 127) as the product of two normal numbers: e = 0 stands for a subnormal one
    half = e >> 1
    v = table[code.long()] * _power_of_two(half - 63) * _power_of_two(e - half - 64)
    v = torch.where(biased == 255, float("nan"), v)
    return v.reshape(*v.shape[:-2], -1)[..., :cols]


def _activate(y, act):
    return torch.clamp_min(y, 0) if act == "relu" else y


def _shifted(x, offset):
    """Row t of the result is row t + offset of x (B, T, C), zero outside."""
    t = x.shape[1]
    out = torch.zeros_like(x)
    if abs(offset) < t:
        if offset >= 0:
            out[:, :t - offset] = x[:, offset:]
        else:
            out[:, -offset:] = x[:, :t + offset]
    return out


def _norm(x, kind, weight, bias):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight
    return x + bias if bias is not None else x


def _block_end(s, case, upcast):
    u = upcast(s["u"])
    y = _norm(u, case["kind"], *[upcast(v) for v in s["post"]]) if s["post"] is not None else u
    if s["gate"] is not None:
        y = y * upcast(s["gate"])
    if s["scale"] is not None:
        y = y * upcast(s["scale"])
    if s["residual"] is not None:
        y = upcast(s["residual"]) + y
    z = _norm(y, case["kind"], *[upcast(v) for v in s["pre"]]) if s["pre"] is not None else None
    return y, z


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "quantize":
        return _decode(_encode(s["x"])).to(s["x"].dtype)
    if op == "linear":
        y = _decode(_encode(s["x"])) @ _decode(s["weight"]).t()
        if s["b"] is not None:
            y = y + s["b"]
        return _activate(y, case["act"]).to(s["x"].dtype)
    if op == "conv":
        x, w = _decode(_encode(s["x"])), _decode(s["weight"])
        left = case["dilation"] * (case["taps"] - 1) // 2
        b, t, c = x.shape
        y = s["b"].expand(b * t, -1)
        for j in range(case["taps"]):
            y = y + _shifted(x, j * case["dilation"] - left).reshape(b * t, c) @ w[:, j].t()
        return _activate(y, case["act"]).reshape(b, t, -1).to(s["x"].dtype)
    y, z = _block_end(s, case, lambda v: v.float() if isinstance(v, torch.Tensor) else v)
    return y.to(s["u"].dtype) if z is None else (y.to(s["u"].dtype), z.to(s["u"].dtype))


def run(state):
    if not own:
        return _plain(state)
    import tts_amd
    case = state["case"]
    op = case["op"]
    if op == "quantize":
        return tts_amd.mxfp4_quantize(state["x"]).dequantize(state["x"].dtype)
    act = None if case.get("act", "none") == "none" else case["act"]
    if op == "linear":
        return tts_amd.mxfp4_linear(state["x"], state["weight"], state["b"], activation=act)
    if op == "conv":
        return tts_amd.mxfp4_conv1d(state["x"], state["weight"], state["b"], dilation=case["dilation"],
                                    activation=act)
    return tts_amd.block_norm(state["u"], post=state["post"], gate=state["gate"], scale=state["scale"],
                              residual=state["residual"], pre=state["pre"])


# -- costs and exact values -------------------------------------------------------------
def work(case):
    op = case["op"]
    size = 4 if case["type"] == "fp32" else 2
    mx = 17 / 32  # bytes of an element in MXFP4: half a byte and its share of the scale
    if op == "quantize":
        n = case["rows"] * case["cols"]
        # read, codes written, codes read back, values written; about four operations an element and way
        return {"bytes": n * (2 * size + 2 * mx), "flops": 8 * n}
    if op in ("linear", "conv"):
        m = case["rows"] if op == "linear" else case["batch"] * case["time"]
        taps = case.get("taps", 1)
        n, k = case["out"], case["cols"]
        bias = 4 * n if case.get("bias", True) else 0
        return {"bytes": m * k * size + n * taps * k * mx + bias + m * n * size, "flops": 2 * m * n * k * taps}
    m, c = case["batch"] * case["time"], case["cols"]
    streams = 2 + int(case["pre"]) + int(case["residual"]) + int(case["gate"] == "element")
    vectors = (int(case["post"]) + int(case["pre"])) * (2 if case["kind"] == "layer" else 1)
    vectors += int(case["scale"] == "channel")
    gate = case["batch"] * c * size if case["gate"] == "batch" else 0
    return {"bytes": m * c * size * streams + 4 * c * vectors + gate,
            "flops": m * c * (8 * (int(case["post"]) + int(case["pre"])) + 3)}


def _nearest64(x):
    """The values that MXFP4 gives x, in 64 bits: the scale is the largest power of two not above
    the block's largest magnitude, over 4; a value goes to the nearest of the eight magnitudes,
    ties to the one with the even code, and to 6 beyond it."""
    cols = x.shape[-1]
    v = x.double()
    v = torch.cat([v, v.new_zeros(*v.shape[:-1], -cols % 32)], -1)
    v = v.unflatten(-1, (-1, 32))
    top = v.abs().max(-1, keepdim=True).values
    _, e = torch.frexp(torch.where(top > 0, top, torch.ones_like(top)))
    shared = torch.clamp(e - 3, min=-127).long()
    unit = ((shared + 1023) << 52).view(torch.float64)
    m = v.abs() / unit
    _, f = torch.frexp(m)
    step = ((torch.clamp(f - 1, 0, 2).long() - 1 + 1023) << 52).view(torch.float64)
    m = torch.clamp(torch.round(m / step) * step, max=6.0)
    return (torch.sign(v) * m * unit).flatten(-2)[..., :cols]


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "quantize":
        return _nearest64(s["x"])
    if op == "norm":
        y, z = _exact_block_end(s, case)
        return y if z is None else (y, z)
    x, w = _nearest64(s["x"]), _nearest64(s["w"])
    if op == "linear":
        y = torch.mm(x, w.T.contiguous())
    else:
        b, t, c = x.shape
        j, d = case["taps"], case["dilation"]
        left = d * (j - 1) // 2
        padded = torch.zeros((b, t + d * (j - 1), c), dtype=torch.float64, device=x.device)
        padded[:, left:left + t] = x
        taps = torch.stack([padded[:, i * d:i * d + t] for i in range(j)], 2)
        y = torch.mm(taps.reshape(b * t, j * c), w.reshape(-1, j * c).T.contiguous()).reshape(b, t, -1)
    if s["b"] is not None:
        y = y + s["b"].double()
    return torch.where(y > 0, y, torch.zeros_like(y)) if case["act"] == "relu" else y


def _exact_block_end(s, case):
    def normalise(x, vectors):
        weight, bias = vectors
        centre = x.sum(-1, keepdim=True) / x.shape[-1] if case["kind"] == "layer" else 0.0
        power = torch.square(x - centre).sum(-1, keepdim=True) / x.shape[-1]
        x = weight.double() * (x - centre) / torch.sqrt(power + _EPS)
        return x if bias is None else x + bias.double()

    y = s["u"].double()
    if s["post"] is not None:
        y = normalise(y, s["post"])
    factor = 1.0
    if s["gate"] is not None:
        factor = s["gate"].double()
    if s["scale"] is not None:
        factor = factor * (s["scale"].double() if isinstance(s["scale"], torch.Tensor) else s["scale"])
    y = y * factor
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return y, normalise(y, s["pre"]) if s["pre"] is not None else None
