"""Operators of the microscaled (MX) expert path, as a program calls them.

The path is the FFN half of a mixture-of-experts layer with 8-bit activations
and 8- or 4-bit expert weights: residual add + RMSNorm to 8-bit rows with
scales, the token lists of the experts, the experts' gate / up products with
SwiGLU, and their down product, each grouped by expert with ragged sizes.

An MX row holds one power-of-two scale byte per 32 elements (value = element *
2^(scale - 127)); elements are e4m3 ("mxfp8") or e2m1 ("mxfp4", two to a byte,
the first in the low nibble).
"""

import torch

own = False

BLOCK = 32
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # a decode batch's rows, and a long prefill's
        {"name": "norm 64", "op": "norm", "rows": 64, "n": 2048},
        {"name": "norm 16384", "op": "norm", "rows": 16384, "n": 2048},
        # one chunk's activations, and one expert tensor's load from fp16
        {"name": "quantize act", "op": "quantize", "rows": 512, "cols": 768, "src": "f32", "to": "mxfp8"},
        {"name": "quantize weight", "op": "quantize", "rows": 98304, "cols": 2048, "src": "f16", "to": "mxfp4"},
        # the engine's prefill chunk, and a long ragged batch
        {"name": "rows 512", "op": "rows", "tokens": 512, "experts": 128, "used": 8},
        {"name": "rows 8191", "op": "rows", "tokens": 8191, "experts": 128, "used": 8},
        # gate / up products: one decoded token, a prefill chunk, a long prefill
        {"name": "swiglu 1 fp4", "op": "swiglu", "tokens": 1, "experts": 128, "used": 8, "n_in": 2048, "n_out": 768,
         "w": "mxfp4", "skew": 0.0},
        {"name": "swiglu 512 fp8", "op": "swiglu", "tokens": 512, "experts": 128, "used": 8, "n_in": 2048, "n_out": 768,
         "w": "mxfp8", "skew": 0.3},
        {"name": "swiglu 4096 fp8", "op": "swiglu", "tokens": 4096, "experts": 128, "used": 8, "n_in": 2048,
         "n_out": 768, "w": "mxfp8", "skew": 0.3},
        # down products: a decode batch, a prefill chunk, a long prefill with popular experts
        {"name": "matmul 16 fp8", "op": "matmul", "tokens": 16, "experts": 128, "used": 8, "n_in": 768, "n_out": 2048,
         "w": "mxfp8", "out": "f32", "skew": 0.0},
        {"name": "matmul 512 fp4", "op": "matmul", "tokens": 512, "experts": 128, "used": 8, "n_in": 768,
         "n_out": 2048, "w": "mxfp4", "out": "f32", "skew": 0.3},
        {"name": "matmul 4096 fp4", "op": "matmul", "tokens": 4096, "experts": 128, "used": 8, "n_in": 768,
         "n_out": 2048, "w": "mxfp4", "out": "f16", "skew": 1.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "rows", "swiglu", "swiglu", "matmul", "matmul"])
    if op == "norm":
        n = 32 * _log_int(rng, 8, 128)
        return {"op": op, "rows": _log_int(rng, 1, 16384 * 2048 // n), "n": n}
    if op == "quantize":
        cols = 32 * _log_int(rng, 4, 128)
        return {"op": op, "rows": _log_int(rng, 16, 98304 * 2048 // cols), "cols": cols, "src": rng.choice(["f32", "f16"]),
                "to": rng.choice(["mxfp8", "mxfp4"])}
    used = rng.choice([1, 2, 4, 8, 8])
    if op == "rows":
        return {"op": op, "tokens": _log_int(rng, 16, 8191), "experts": rng.choice([8, 60, 64, 128, 128, 256]), "used": used}
    experts = rng.choice([1, 8, 60, 64, 128, 128, 256])
    used = min(experts, used)
    n_in = 128 * _log_int(rng, 2, 16)
    n_out = 32 * _log_int(rng, 2, 24) if op == "swiglu" else _log_int(rng, 64, 2048)
    tokens = _log_int(rng, 1, 4096)
    # no more weights, and no more work, than the largest listed case
    experts = min(experts, max(used, int(128 * 2048 * 768 * 2 / (n_in * n_out * (2 if op == "swiglu" else 1)))))
    case = {"op": op, "tokens": tokens, "experts": experts, "used": used, "n_in": n_in, "n_out": n_out,
            "w": rng.choice(["mxfp8", "mxfp4"]), "skew": rng.choice([0.0, 0.3, 1.0])}
    if op == "matmul":
        case["out"] = rng.choice(["f32", "f16"])
    return case


def _used_experts(case):
    """Experts that get at least one row, for routing without preference."""
    return case["experts"] * (1.0 - (1.0 - case["used"] / case["experts"]) ** case["tokens"])


def work(case):
    op = case["op"]
    if op == "norm":
        e = case["rows"] * case["n"]
        return {"bytes": e * (4 * 4 + 1 + 1 / BLOCK) + 4 * case["n"], "flops": 5 * e}
    if op == "quantize":
        e = case["rows"] * case["cols"]
        mx = (1.0 if case["to"] == "mxfp8" else 0.5) + 1 / BLOCK
        return {"bytes": e * ((4 if case["src"] == "f32" else 2) + 2 * mx + 4), "flops": 3 * e}
    rows = case["tokens"] * case["used"]
    if op == "rows":
        return {"bytes": 4 * (3 * rows + case["experts"] + 1), "flops": 2 * rows}
    pair = 2 if op == "swiglu" else 1
    w = _used_experts(case) * pair * case["n_out"] * case["n_in"] * ((1.0 if case["w"] == "mxfp8" else 0.5) + 1 / BLOCK)
    x = (case["tokens"] if op == "swiglu" else rows) * case["n_in"] * (1 + 1 / BLOCK)
    y = rows * case["n_out"] * (1 + 1 / BLOCK if op == "swiglu" else 4 if case["out"] == "f32" else 2)
    return {"bytes": w + x + y + 8 * rows, "flops": 2.0 * rows * pair * case["n_out"] * case["n_in"]}


# ---------------------------------------------------------------- MX, plainly
def _power(e):
    """2^e for a whole-number tensor e in -127 .. 127, in fp32."""
    return torch.where(e > -127, (e + 127).clamp(min=1) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _quantize(x, to):
    """fp32 [..., n] -> (element bytes [..., n or n/2], scale bytes [..., n/32])."""
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    exponent = b.abs().amax(-1).view(torch.int32) >> 23
    scale = (exponent - (8 if to == "mxfp8" else 2)).clamp(min=0)
    v = b * _power(127 - scale).unsqueeze(-1)
    if to == "mxfp8":
        q = v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).reshape(x.shape).view(torch.uint8)
    else:
        a = v.abs()
        c = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
        c = (c.to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)).reshape(x.shape)
        q = c[..., 0::2] | (c[..., 1::2] << 4)
    return q.contiguous(), scale.to(torch.uint8)


def _values(q, scale, fmt):
    """The fp32 values that MX rows stand for."""
    if fmt == "mxfp8":
        v = q.view(torch.float8_e4m3fn).to(torch.float32)
    else:
        table = torch.tensor(E2M1 + tuple(-t for t in E2M1), device=q.device)
        v = torch.stack((table[(q & 15).int()], table[(q >> 4).int()]), -1)
    return (v.reshape(*scale.shape, BLOCK) * _power(scale.int() - 127).unsqueeze(-1)).reshape(*scale.shape[:-1], -1)


# ------------------------------------------------------------------ the inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _weights(g, case):
    """One expert tensor [experts, n_out, n_in], quantised at load time."""
    shape = (case["experts"], case["n_out"], case["n_in"])
    return _quantize(_normal(g, *shape).mul_(case["n_in"] ** -0.5), case["w"])


def _routing(g, tokens, experts, used, skew=0.0):
    """Top-k ids [tokens, used] of random logits, some experts preferred by `skew`."""
    logits = _normal(g, tokens, experts) + skew * _normal(g, experts)
    return torch.topk(logits, used, dim=1)[1].to(torch.int32)


def _sorted_rows(idx, experts):
    """offsets [experts + 1], entries (flat idx positions sorted by expert), row_of (its inverse)."""
    flat = idx.reshape(-1)
    entries = torch.sort(flat, stable=True)[1]
    # the first sorted row of each expert: how many ids are below it
    bounds = torch.arange(experts + 1, device=idx.device, dtype=torch.int32)
    offsets = (flat[None, :] < bounds[:, None]).sum(1)
    row_of = torch.empty_like(entries)
    row_of[entries] = torch.arange(entries.numel(), device=idx.device)
    return offsets.to(torch.int32), entries.to(torch.int32), row_of.to(torch.int32)


def _bytes(*shape):
    return torch.zeros(*shape, dtype=torch.uint8, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    if op == "norm":
        rows, n = case["rows"], case["n"]
        s["x"], s["residual"] = _normal(g, rows, n), _normal(g, rows, n) * 2.0
        s["weight"] = 1.0 + 0.1 * _normal(g, n)
        s["sum"], s["norm"] = torch.zeros(rows, n, device="cuda"), torch.zeros(rows, n, device="cuda")
        s["q"], s["scales"] = _bytes(rows, n), _bytes(rows, n // BLOCK)
    elif op == "quantize":
        rows, cols = case["rows"], case["cols"]
        s["src"] = (_normal(g, rows, cols) * 0.05).to(torch.float32 if case["src"] == "f32" else torch.float16)
        s["q"] = _bytes(rows, cols if case["to"] == "mxfp8" else cols // 2)
        s["scales"] = _bytes(rows, cols // BLOCK)
        s["values"] = torch.zeros(rows, cols, device="cuda")
    elif op == "rows":
        s["idx"] = _routing(g, case["tokens"], case["experts"], case["used"])
        n = case["tokens"] * case["used"]
        s["offsets"] = torch.zeros(case["experts"] + 1, dtype=torch.int32, device="cuda")
        s["entries"], s["row_of"] = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
    else:
        tokens, used = case["tokens"], case["used"]
        rows = tokens * used
        idx = _routing(g, tokens, case["experts"], used, case["skew"])
        s["offsets"], s["entries"], _ = _sorted_rows(idx, case["experts"])
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
        s["x"], s["x_scales"] = _quantize(_normal(g, tokens if op == "swiglu" else rows, case["n_in"]), "mxfp8")
        s["w"], s["w_scales"] = _weights(g, case)
        if op == "swiglu":
            s["up"], s["up_scales"] = _weights(g, case)
            s["scores"] = torch.softmax(_normal(g, tokens, used), 1)
            s["q"], s["scales"] = _bytes(rows, case["n_out"]), _bytes(rows, case["n_out"] // BLOCK)
        else:
            s["out"] = torch.zeros(rows, case["n_out"], device="cuda",
                                   dtype=torch.float32 if case["out"] == "f32" else torch.float16)
    if own:
        s["h"] = _handles(s)
    return s


_ds3 = _stream = None


def _handles(s):
    """The library's handles of the state's tensors; the first call opens the library and the batch that ops queue in.

    Ops run on the library's own stream, which is not ordered with torch's: here it is put behind the inputs that
    torch is still making, and a program that reads the outputs waits for the device (or lets its stream wait for the
    library's) once behind its last op. What ops report on the device is read here too, behind those of earlier states."""
    global _ds3, _stream
    if _ds3 is None:
        from qw3_b200 import ds3

        if ds3.init() != 0 or ds3.begin_batch() != 0:
            raise RuntimeError(ds3.last_error())
        _ds3, _stream = ds3, torch.cuda.ExternalStream(ds3.stream())
    if _ds3.device_errors() != 0:
        raise RuntimeError("an op on an earlier state reported an error on the device")
    _stream.wait_stream(torch.cuda.current_stream())
    return {k: _ds3.buffer_wrap(t.data_ptr(), t.numel() * t.element_size())
            for k, t in s.items() if isinstance(t, torch.Tensor)}


# --------------------------------------------------------------------- the runs
def run(s):
    op = s["case"]["op"]
    if own:
        rc = {"norm": _own_norm, "quantize": _own_quantize, "rows": _own_rows, "swiglu": _own_swiglu,
              "matmul": _own_matmul}[op](s["case"], s["h"])
        if rc != 0:
            raise RuntimeError(_ds3.last_error())
        return _outputs(s)
    return {"norm": _plain_norm, "quantize": _plain_quantize, "rows": _plain_rows, "swiglu": _plain_swiglu,
            "matmul": _plain_matmul}[op](s)


def _elements(q):
    """e4m3 bytes as the 8-bit floats they are."""
    return q.view(torch.float8_e4m3fn)


def _scale_floats(scales):
    return scales.view(torch.float8_e8m0fnu)


def _outputs(s):
    op = s["case"]["op"]
    if op == "norm":
        return {"sum": s["sum"], "norm": s["norm"], "q": _elements(s["q"]), "scales": _scale_floats(s["scales"])}
    if op == "quantize":
        return {"values": s["values"]}
    if op == "rows":
        return {"offsets": s["offsets"], "entries": s["entries"], "row_of": s["row_of"]}
    if op == "swiglu":
        return {"q": _elements(s["q"]), "scales": _scale_floats(s["scales"])}
    return {"out": s["out"]}


EPS = 1e-6


def _own_norm(c, h):
    return _ds3.add_rms_norm_mx(h["x"], h["residual"], h["weight"], h["sum"], h["norm"], h["q"], h["scales"], c["n"],
                                c["rows"], EPS)


def _own_quantize(c, h):
    to = _ds3.MXFP8 if c["to"] == "mxfp8" else _ds3.MXFP4
    src = _ds3.TYPE_F32 if c["src"] == "f32" else _ds3.TYPE_F16
    return (_ds3.mx_quantize(h["src"], src, h["q"], h["scales"], to, c["rows"], c["cols"])
            or _ds3.mx_dequantize(h["q"], h["scales"], to, h["values"], c["rows"], c["cols"]))


def _own_rows(c, h):
    return _ds3.moe_expert_rows(h["idx"], h["offsets"], h["entries"], h["row_of"], c["tokens"], c["experts"], c["used"])


def _own_swiglu(c, h):
    # token rows through `entries` (entry / used is the token), weighted by the router's scores
    return _ds3.moe_mx_swiglu(h["x"], h["x_scales"], h["entries"], c["used"], h["offsets"], h["w"], h["w_scales"], h["up"],
                              h["up_scales"], _ds3.MXFP8 if c["w"] == "mxfp8" else _ds3.MXFP4, h["scores"], h["q"],
                              h["scales"], c["tokens"], c["tokens"] * c["used"], c["experts"], c["n_in"], c["n_out"])


def _own_matmul(c, h):
    # sorted rows in place, results back in token order through `entries`
    rows = c["tokens"] * c["used"]
    return _ds3.moe_mx_matmul(h["x"], h["x_scales"], None, 1, h["offsets"], h["w"], h["w_scales"],
                              _ds3.MXFP8 if c["w"] == "mxfp8" else _ds3.MXFP4, h["out"],
                              _ds3.TYPE_F32 if c["out"] == "f32" else _ds3.TYPE_F16, h["entries"], rows, rows,
                              c["experts"], c["n_in"], c["n_out"])


def _plain_norm(s):
    total = s["x"] + s["residual"]
    # in 64 bits: an element next to a rounding border follows the last bits
    d = total.double()
    inv = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    norm = (d * inv * s["weight"].double()).to(torch.float32)
    q, scales = _quantize(norm, "mxfp8")
    return {"sum": total, "norm": norm, "q": _elements(q), "scales": _scale_floats(scales)}


def _plain_quantize(s):
    q, scales = _quantize(s["src"].float(), s["case"]["to"])
    return {"values": _values(q, scales, s["case"]["to"])}


def _plain_rows(s):
    offsets, entries, row_of = _sorted_rows(s["idx"], s["case"]["experts"])
    return {"offsets": offsets, "entries": entries, "row_of": row_of}


def _padded(s, rows_of_x):
    """Each expert's token rows as fp32 [experts, most, n_in], and the place of each sorted row in it."""
    n = s["entries"].numel()
    row = torch.arange(n, device="cuda", dtype=torch.int32)
    expert = torch.bucketize(row, s["offsets"][1:], right=True)
    place = expert * s["most"] + (row - s["offsets"][expert])
    x = _values(s["x"], s["x_scales"], "mxfp8")
    padded = torch.zeros(s["case"]["experts"] * s["most"], x.shape[1], device="cuda")
    padded[place] = x if rows_of_x is None else x[rows_of_x]
    return padded.reshape(s["case"]["experts"], s["most"], -1), place


def _plain_swiglu(s):
    c = s["case"]
    x, place = _padded(s, s["entries"].long() // c["used"])
    gate = torch.bmm(x, _values(s["w"], s["w_scales"], c["w"]).transpose(1, 2)).reshape(-1, c["n_out"])[place]
    up = torch.bmm(x, _values(s["up"], s["up_scales"], c["w"]).transpose(1, 2)).reshape(-1, c["n_out"])[place]
    act = gate / (1.0 + torch.exp(-gate)) * up * s["scores"].reshape(-1)[s["entries"].long()].unsqueeze(1)
    q, scales = _quantize(act, "mxfp8")
    return {"q": _elements(q), "scales": _scale_floats(scales)}


def _plain_matmul(s):
    c = s["case"]
    x, place = _padded(s, None)
    y = torch.bmm(x, _values(s["w"], s["w_scales"], c["w"]).transpose(1, 2)).reshape(-1, c["n_out"])[place]
    out = torch.empty_like(y)
    out[s["entries"].long()] = y
    return {"out": out if c["out"] == "f32" else out.to(torch.float16)}


# ------------------------------------------------------------------ in 64 bits
def _table64(fmt):
    """The value of every element code, from the format's definition."""
    if fmt == "mxfp4":
        mag = [(1 + (c & 1) / 2) * 2.0 ** ((c >> 1) - 1) if c >> 1 else (c & 1) / 2 for c in range(8)]
    else:
        mag = [(1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) if c >> 3 else (c & 7) / 8 * 2.0**-6 for c in range(127)]
        mag.append(float("nan"))
    return torch.tensor(mag + [-m for m in mag], dtype=torch.float64, device="cuda")


def _power64(e):
    """2^e for whole e, exactly (a power function may be off in the last bit)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _decode64(q, scales, fmt):
    if fmt == "mxfp4":
        q = torch.stack((q % 16, q // 16), -1).flatten(-2)
    v = _table64(fmt)[q.long()]
    return v * _power64(scales.long() - 127).repeat_interleave(BLOCK, -1)


def _encode64(x, fmt):
    """(element values, scale exponents) of MX rows of 64-bit x, ties to the even code."""
    mags = _table64(fmt)[: 8 if fmt == "mxfp4" else 127]
    b = x.unflatten(-1, (-1, BLOCK))
    top = torch.frexp(b.abs().amax(-1))[1] - 1
    e = (top - (2 if fmt == "mxfp4" else 8)).clamp(min=-127)
    v = b / _power64(e).unsqueeze(-1)
    a = v.abs().clamp(max=float(mags[-1]))
    hi = torch.searchsorted(mags, a.contiguous()).clamp(max=mags.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    down, up = a - mags[lo], mags[hi] - a
    code = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return (mags[code] * torch.sign(v)).flatten(-2), e


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        total = s["x"].double() + s["residual"].double()
        t = total.float().double()  # the stored sum is what is normed
        norm = t * torch.rsqrt(t.pow(2).sum(1, keepdim=True) / case["n"] + EPS) * s["weight"].double()
        q, e = _encode64(norm.float().double(), "mxfp8")
        return {"sum": total, "norm": norm, "q": q, "scales": _power64(e)}
    if op == "quantize":
        q, e = _encode64(s["src"].double(), case["to"])
        return {"values": q * _power64(e).repeat_interleave(BLOCK, -1)}
    if op == "rows":
        return None  # whole numbers
    swiglu = op == "swiglu"
    x = _decode64(s["x"], s["x_scales"], "mxfp8")
    entries = s["entries"].long()
    out = torch.zeros(entries.numel(), case["n_out"], dtype=torch.float64, device="cuda")
    bounds = s["offsets"].tolist()
    for e in range(case["experts"]):
        lo, hi = bounds[e], bounds[e + 1]
        if lo == hi:
            continue
        w = _decode64(s["w"][e], s["w_scales"][e], case["w"]).T
        if swiglu:
            rows = x[torch.div(entries[lo:hi], case["used"], rounding_mode="floor")]
            gate, up = rows @ w, rows @ _decode64(s["up"][e], s["up_scales"][e], case["w"]).T
            out[lo:hi] = gate * torch.sigmoid(gate) * up * s["scores"].double().flatten()[entries[lo:hi], None]
        else:
            out[entries[lo:hi]] = x[lo:hi] @ w
    if not swiglu:
        return {"out": out}
    # The elements before their rounding to 8 bits: which way one next to a
    # border goes hangs on the last bits of a long sum. A scale byte has no
    # such value, for the same reason.
    e = _encode64(out, "mxfp8")[1]
    return {"q": out / _power64(e).repeat_interleave(BLOCK, -1), "scales": None}
