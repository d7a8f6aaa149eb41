"""What the projections around the attention are measured on: the residual addition + RMS norm + 8-bit rows, the matrix
product with 4-bit weights, and the gated feed-forward product, at the sizes of decode steps and prompt passes.

Every operator works on fp32 rows that are held in 8 bits for a product (int8 levels, one fp32 scale per group of `gs` values),
and on weights of 4 bits (levels -8 .. 7, one f16 scale per group).  `own` selects the library's calls instead of the plain form.
"""
import torch

own = False

EPS = 1e-6


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the norm in front of a layer's first product: one decoded token; a ragged batch of an odd width; a prompt chunk
        {"name": "norm_1x4096", "op": "norm", "rows": 1, "k": 4096, "gs": 64, "delta": True, "y": False},
        {"name": "norm_77x2720", "op": "norm", "rows": 77, "k": 2720, "gs": 32, "delta": True, "y": True},
        {"name": "norm_2048x4096", "op": "norm", "rows": 2048, "k": 4096, "gs": 128, "delta": True, "y": False},
        # one token through the attention's output projection (32 heads of 128) and through a vocabulary
        {"name": "mm_1x4096x4096", "op": "mm", "rows": 1, "n": 4096, "k": 4096, "gs": 64},
        {"name": "mm_1x65536x4096", "op": "mm", "rows": 1, "n": 65536, "k": 4096, "gs": 64},
        # a few tokens (a verify segment) through the second product of a feed-forward block, odd sizes
        {"name": "mm_5x4099x11008", "op": "mm", "rows": 5, "n": 4099, "k": 11008, "gs": 32},
        # a batch of decoding sequences through q, k and v at once (32 + 2 x 8 heads of 128)
        {"name": "mm_48x6144x4096", "op": "mm", "rows": 48, "n": 6144, "k": 4096, "gs": 64},
        # prompt chunks
        {"name": "mm_512x4096x12288", "op": "mm", "rows": 512, "n": 4096, "k": 12288, "gs": 128},
        {"name": "mm_2000x6144x4096", "op": "mm", "rows": 2000, "n": 6144, "k": 4096, "gs": 64},
        # the gated product of a feed-forward block: one token; a small batch whose rows go on in 8 bits; a prompt chunk
        {"name": "ffn_1x12288x4096", "op": "ffn", "rows": 1, "n": 12288, "k": 4096, "gs": 64, "quant": False},
        {"name": "ffn_19x5504x2048", "op": "ffn", "rows": 19, "n": 5504, "k": 2048, "gs": 32, "quant": True},
        {"name": "ffn_1024x12288x4096", "op": "ffn", "rows": 1024, "n": 12288, "k": 4096, "gs": 64, "quant": False},
    ]


def _spread(rng, lo, hi):
    """An integer in lo .. hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "mm", "mm", "ffn"])
    gs = rng.choice([32, 64, 128])
    k = gs * max(1, _spread(rng, 512, 12288) // gs)
    if op == "norm":
        return {"op": op, "rows": _spread(rng, 1, 2048), "k": k, "gs": gs, "delta": rng.random() < 0.75, "y": rng.random() < 0.3}
    rows = _spread(rng, 1, 2048)
    most = 1024 * 12288 * 4096  # rows x outputs x inputs of the largest listed case, per projection
    if op == "mm":
        n = min(_spread(rng, 256, 32768), 2 * most // (rows * k))
        return {"op": op, "rows": rows, "n": n, "k": k, "gs": gs}
    n = min(_spread(rng, 512, 12288), most // (rows * k))
    return {"op": op, "rows": rows, "n": gs * max(1, n // gs), "k": k, "gs": gs, "quant": rng.random() < 0.5}


def work(case):
    r, k, gs = case["rows"], case["k"], case["gs"]
    if case["op"] == "norm":
        per = 4 + 4 * case["delta"] + 4 * case["delta"] + 1 + 4 * case["y"]
        return {"bytes": r * k * per + r * (k // gs) * 4 + 4 * k, "flops": 8 * r * k}
    m = 1 if case["op"] == "mm" else 2
    n = case["n"]
    weights = m * (n * k // 2 + n * (k // gs) * 2)
    out = r * n * 4 if not case.get("quant") else r * n + r * (n // gs) * 4
    return {"bytes": weights + r * k + r * (k // gs) * 4 + out, "flops": 2 * m * r * n * k}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _rows8(x, gs):
    """fp32 rows as int8 levels and scales: scale = max / 127, level = the nearest (the framework's rule)."""
    g = x.view(x.shape[0], -1, gs)
    top = g.abs().amax(2, keepdim=True)
    v = g * torch.where(top > 0, torch.full_like(top, 127.0) / top, torch.zeros_like(top))
    level = torch.trunc(v + torch.copysign(torch.full_like(v, 0.49999997), v))
    return level.to(torch.int8).view(x.shape), (top * (1.0 / 127.0)).squeeze(2)


def _weights(n, k, gs, gen):
    """4-bit levels, two in a byte (value + 8; the even input in the low half), and f16 scales, as a quantised matrix has them."""
    packed = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
    for at in range(0, n, 8192):
        w = torch.randn(min(8192, n - at), k, generator=gen, device="cuda").mul_(2.6).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
        packed[at:at + w.shape[0]] = w[:, 0::2] | (w[:, 1::2] << 4)
    scales = (torch.rand(n, k // gs, generator=gen, device="cuda") * 0.006 + 0.004).to(torch.float16)
    return packed, scales


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    r, k, gs = case["rows"], case["k"], case["gs"]
    # rows of a residual stream: unit variance with a few columns that are far larger
    x = torch.randn(r, k, generator=gen, device="cuda")
    x[:, torch.randint(0, k, (4,), generator=gen, device="cuda")] *= 20.0
    s = {"case": dict(case)}
    if case["op"] == "norm":
        s["x"] = x
        s["delta"] = torch.randn(r, k, generator=gen, device="cuda") * 0.3 if case["delta"] else None
        s["w"] = 1.0 + 0.2 * torch.randn(k, generator=gen, device="cuda")
        return s
    s["xq"], s["xs"] = _rows8(x, gs)
    s["mats"] = [_weights(case["n"], k, gs, gen) for _ in range(1 if case["op"] == "mm" else 2)]
    return s


_context = None


def _library():
    """The program's one context; its work goes to the stream that torch uses (1: the handle of the default stream)."""
    global _context
    if _context is None:
        import gwenedeg_b200 as g
        _context = g.Context(torch.cuda.current_device(), n_attn=1, n_heads=32, n_kv_heads=8, head_dim=128, max_rows=2048)
        _context.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    return _context


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # what a program keeps: its context, the laid out weights, the output buffers
        c = s["ctx"] = _library()
        r, k, gs = case["rows"], case["k"], case["gs"]
        new = lambda *shape, t=torch.float32: torch.empty(shape, dtype=t, device="cuda")  # noqa: E731
        if case["op"] == "norm":
            s["x_out"] = new(r, k) if case["delta"] else None
            s["y"] = new(r, k) if case["y"] else None
            s["q"], s["qs"] = new(r, k, t=torch.int8), new(r, k // gs)
        else:
            torch.cuda.synchronize()
            s["q4"] = [c.q4_new_dev(case["n"], k, gs, p.data_ptr(), f.data_ptr()) for p, f in s.pop("mats")]
            if case.get("quant"):
                s["q"], s["qs"] = new(r, case["n"], t=torch.int8), new(r, case["n"] // gs)
                s["values"] = new(r, case["n"] // gs, gs, t=torch.bfloat16)
            else:
                s["out"] = new(r, case["n"])
    return s


# ---- a pass ---------------------------------------------------------------------------------------------------------
def _ptr(t):
    return None if t is None else t.data_ptr()


def _run_own(s):
    case, c = s["case"], s["ctx"]
    r, k, gs = case["rows"], case["k"], case["gs"]
    if case["op"] == "norm":
        c.add_norm_quant_dev(r, k, gs, _ptr(s["x"]), _ptr(s["delta"]), _ptr(s["w"]), EPS, _ptr(s["x_out"]), _ptr(s["y"]), _ptr(s["q"]), _ptr(s["qs"]))
        values = s["q"].view(r, -1, gs) * s["qs"].unsqueeze(2)
        return {"x": s["x_out"], "y": s["y"], "values": values.view(r, k)}
    if case["op"] == "mm":
        c.mm_q4_dev(s["q4"][0], r, _ptr(s["xq"]), _ptr(s["xs"]), _ptr(s["out"]))
        return s["out"]
    if case["quant"]:
        c.ffn_q4_dev(s["q4"][0], s["q4"][1], r, _ptr(s["xq"]), _ptr(s["xs"]), None, _ptr(s["q"]), _ptr(s["qs"]))
        return torch.mul(s["q"].view(r, -1, gs), s["qs"].unsqueeze(2), out=s["values"]).view(r, -1)
    c.ffn_q4_dev(s["q4"][0], s["q4"][1], r, _ptr(s["xq"]), _ptr(s["xs"]), _ptr(s["out"]), None, None)
    return s["out"]


def _plain_weights(packed, scales, gs):
    level = torch.stack((packed & 15, packed >> 4), 2).to(torch.float32) - 8.0
    return (level.view(scales.shape[0], -1, gs) * scales.float().unsqueeze(2)).view(scales.shape[0], -1)


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    r, gs = case["rows"], case["gs"]
    if case["op"] == "norm":
        x = s["x"] if s["delta"] is None else s["x"] + s["delta"]
        inv = 1.0 / torch.sqrt(x.square().mean(1, keepdim=True) + EPS)
        v = x * s["w"]
        level, scale = _rows8(v, gs)
        values = (level.view(r, -1, gs) * (scale * inv).unsqueeze(2)).view(x.shape)
        return {"x": None if s["delta"] is None else x, "y": v * inv if case["y"] else None, "values": values}
    x = (s["xq"].view(r, -1, gs).to(torch.float32) * s["xs"].unsqueeze(2)).view(r, -1)
    out = [x @ _plain_weights(p, f, gs).t() for p, f in s["mats"]]
    if case["op"] == "mm":
        return out[0]
    h = out[0] / (1.0 + torch.exp(-out[0])) * out[1]
    if not case["quant"]:
        return h
    level, scale = _rows8(h, gs)
    return (level.view(r, -1, gs) * scale.unsqueeze(2)).to(torch.bfloat16).view(h.shape)


def exact(case, seed):
    """The definitions in 64 bits, on the same inputs.  The levels of a row are whole numbers that its fp32 values decide (they
    are found in 32 bits here too, from the values alone: x + d and its product with w, each rounded once)."""
    s = _inputs(case, seed)
    r, k, gs = case["rows"], case["k"], case["gs"]
    d = torch.float64
    if case["op"] == "norm":
        x32 = s["x"] if s["delta"] is None else s["x"] + s["delta"]
        x = x32.to(d)
        rms = (x.pow(2).sum(1, keepdim=True) / k + EPS).sqrt()
        v32 = (x32 * s["w"]).view(r, k // gs, gs)
        most = v32.abs().max(2, keepdim=True).values
        t = v32 * torch.div(torch.full_like(most, 127.0), most)
        level = torch.where(most > 0, torch.sign(t) * torch.floor(t.abs() + 0.49999997), torch.zeros_like(t))
        values = (level.to(d) * most.to(d) / 127.0).view(r, k) / rms
        return {"x": None if s["delta"] is None else x, "y": x * s["w"].to(d) / rms if case["y"] else None, "values": values}
    x = s["xq"].to(d) * s["xs"].to(d).repeat_interleave(gs, 1)
    out = []
    for packed, scales in s["mats"]:
        w = torch.empty(packed.shape[0], k, dtype=d, device=packed.device)
        w[:, 0::2] = (packed & 15).to(d) - 8
        w[:, 1::2] = (packed >> 4).to(d) - 8
        w *= scales.to(d).repeat_interleave(gs, 1)
        out.append(torch.mm(x, w.t()))
        del w
    if case["op"] == "mm":
        return out[0]
    h = out[0] * torch.sigmoid(out[0]) * out[1]
    if not case["quant"]:
        return h
    h = h.view(r, -1, gs)
    unit = h.abs().max(2, keepdim=True).values / 127.0
    return (torch.round(h / torch.where(unit > 0, unit, torch.ones_like(unit))) * unit).view(r, -1)
