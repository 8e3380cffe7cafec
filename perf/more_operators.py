"""Performance cases of the 4-bit projections and of the rotary operator: what a program has them do that runs the
layer's matrices in microscaled 4-bit floating point and its positions in a layout or scaling of its own.

A 4-bit matrix holds e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with one power-of-two scale for each 32
of a row: 2^e, the least power of two with max|x| < 7 * 2^e, so that the largest rounds to at most 6. Kinds of call:

* ``quantise``  rows into 4 bits, and the values they stand for read back (``Mx4Matrix.quantise``, ``Mx4Matrix.values``);
* ``product``   Y = X . W^T (+ an f32 residual), X and W in 4 bits (``mx4_gemm``);
* ``weights``   the same with X in bf16 and W in 4 bits (``mx4_gemm``);
* ``rotary``    norm and rotation of q and k heads (``Rotary.apply``);
* ``project``   the three as a layer calls them: quantise the activations, QKV product, rotary of its q and k.

``exact`` restates each in float64.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # the activations of one token: nothing but latency
        {"name": "quantise_token", "kind": "quantise", "T": 1, "K": 5120, "type": "bf16"},
        # attention outputs of the ordinary micro-batch, ahead of the output projection
        {"name": "quantise_packed", "kind": "quantise", "T": 4096, "K": 6144, "type": "f16"},
        # a short question on a cached document: the QKV projection of its tokens
        {"name": "product_question", "kind": "product", "T": 45, "N": 14336, "K": 5120},
        # one request of ordinary length: output projection into the residual
        {"name": "product_residual", "kind": "product", "T": 1160, "N": 5120, "K": 6144, "residual": True},
        # the ordinary micro-batch (4,096 tokens): its QKV projection
        {"name": "product_packed", "kind": "product", "T": 4096, "N": 14336, "K": 5120},
        # the next token of one request: weights are read once, nothing else counts
        {"name": "weights_token", "kind": "weights", "T": 1, "N": 14336, "K": 5120},
        # the next tokens of a batch: output projection into the residual
        {"name": "weights_tokens", "kind": "weights", "T": 61, "N": 5120, "K": 6144, "residual": True},
        # a prompt whose activations stay in bf16
        {"name": "weights_prompt", "kind": "weights", "T": 1300, "N": 10240, "K": 4096},
        # the next tokens of a batch behind long texts, positions scaled by parts
        {"name": "rotary_tokens", "kind": "rotary", "T": 64, "nh": 24, "nkv": 4, "hd": 256, "n_rot": 64, "layout": "half", "axes": 1,
         "type": "bf16", "gated": True, "norm": True, "scaling": "parts", "factor": 8.0, "far": 130000},
        # the ordinary micro-batch in f32, neighbouring dims in pairs, the whole head
        {"name": "rotary_packed", "kind": "rotary", "T": 4096, "nh": 32, "nkv": 4, "hd": 128, "n_rot": 128, "layout": "interleaved", "axes": 1,
         "type": "f32", "gated": False, "norm": False, "scaling": "linear", "factor": 4.0, "far": 65536},
        # eight packed requests with images: three position axes
        {"name": "rotary_axes", "kind": "rotary", "T": 4096, "nh": 24, "nkv": 4, "hd": 256, "n_rot": 64, "layout": "half", "axes": 3,
         "type": "bf16", "gated": True, "norm": True, "scaling": "none", "factor": 1.0, "far": 16384},
        # one layer's way in, for a request of ordinary length
        {"name": "project_request", "kind": "project", "T": 425, "H": 4096, "nh": 16, "nkv": 4, "hd": 256, "n_rot": 64, "layout": "half",
         "axes": 1, "type": "bf16", "gated": True, "norm": True, "scaling": "base", "factor": 4.0, "far": 65536},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantise", "product", "product", "product", "weights", "weights", "weights", "rotary", "rotary", "project"])
    if kind == "quantise":
        return {"kind": kind, "T": _log(rng, 1, 4096), "K": 32 * _log(rng, 2, 300), "type": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if kind in ("product", "weights"):
        c = {"kind": kind, "T": _log(rng, 1, 4096), "N": _log(rng, 100, 14336), "K": 32 * _log(rng, 4, 160)}
        if rng.random() < 0.3:
            c["residual"] = True
        elif rng.random() < 0.3:
            c["out"] = "f32"
        return c
    scaling = rng.choice(["none", "linear", "base", "parts"])
    c = {"kind": kind, "layout": rng.choice(["half", "interleaved"]), "axes": rng.choice([1, 1, 3]), "type": rng.choice(["bf16", "bf16", "f16", "f32"]),
         "norm": rng.random() < 0.6, "scaling": scaling, "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 32.0]),
         "far": _log(rng, 100, 500000)}
    if kind == "rotary":
        hd = rng.choice([64, 72, 80, 128, 128, 192, 256, 256])
        c.update(T=_log(rng, 1, 4096), hd=hd, n_rot=rng.choice([hd, hd, hd // 2, 2 * rng.randint(2, hd // 2)]), gated=rng.random() < 0.5)
        c["nh"], c["nkv"] = rng.choice([(24, 4), (16, 4), (32, 4), (8, 8), (12, 1), (5, 5)])
    else:
        c.update(T=_log(rng, 1, 2048), H=32 * _log(rng, 8, 160), hd=256, n_rot=64, gated=True, type="bf16")
        c["nh"], c["nkv"] = rng.choice([(24, 4), (16, 4), (8, 2)])
    return c


def _row(case):
    return ((2 if case["gated"] else 1) * case["nh"] + 2 * case["nkv"]) * case["hd"]


def work(case):
    kind, T = case["kind"], case["T"]
    if kind == "quantise":
        return {"bytes": T * case["K"] * ((4 if case["type"] == "f32" else 2) + 2), "flops": 0}
    if kind in ("product", "weights"):
        N, K = case["N"], case["K"]
        out = 8 if case.get("residual") else 4 if case.get("out") == "f32" else 2
        x = T * K * 17 // 32 if kind == "product" else 2 * T * K
        return {"bytes": x + N * K * 17 // 32 + T * N * out, "flops": 2 * T * N * K}
    heads = (case["nh"] + case["nkv"]) * case["hd"]
    size = 4 if case["type"] == "f32" else 2
    if kind == "rotary":
        return {"bytes": T * heads * 2 * size + T * case["axes"] * 4, "flops": 0}
    return {"bytes": T * case["H"] * 2 + _row(case) * case["H"] * 17 // 32 + T * (_row(case) + heads) * 2 + T * case["axes"] * 4,
            "flops": 2 * T * case["H"] * _row(case)}


# ---- inputs

def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32)


def _activations(g, T, K):
    """Rows of a normalised residual: a few channels are much larger than the others."""
    return _randn(g, T, K) * torch.where(torch.rand(K, generator=g, device=DEVICE) < 0.02, 8.0, 1.0)


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(1000003 * seed + 31)
    kind, T, x = case["kind"], case["T"], {"case": case}
    if kind == "quantise":
        x["x"] = _activations(g, T, case["K"]).to(TYPES[case["type"]])
    if kind in ("product", "weights", "project"):
        N, K = (_row(case), case["H"]) if kind == "project" else (case["N"], case["K"])
        a = _activations(g, T, K).to(torch.bfloat16)
        # codes [rows][K / 2], the lower four bits first, and scale exponents + 127 [rows][K / 32], as a file stores them
        x["w_codes"], x["w_scales"] = _codes(_randn(g, N, K) / math.sqrt(K))
        if kind == "product":
            x["x_codes"], x["x_scales"] = _codes(a.float())
        else:
            x["x"] = a
        if case.get("residual"):
            x["residual"] = _randn(g, T, N)
    if kind in ("rotary", "project"):
        nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
        if kind == "rotary":
            x["rows"] = _randn(g, T, _row(case)).to(TYPES[case["type"]])
        x["pos"] = torch.randint(0, case["far"], (T, case["axes"]), generator=g, device=DEVICE, dtype=torch.int32)
        x["q_norm"], x["k_norm"] = (1 + 0.1 * _randn(g, hd), 1 + 0.1 * _randn(g, hd)) if case["norm"] else (None, None)
    return x


def _heads(case, rows):
    """The q and k heads of projection rows: [q | gate] of each q head where the model gates, then k, then v."""
    nh, nkv, hd, wide = case["nh"], case["nkv"], case["hd"], 2 if case["gated"] else 1
    q = rows[:, :wide * nh * hd].unflatten(1, (nh, wide * hd))[:, :, :hd]
    return q, rows[:, wide * nh * hd:(wide * nh + nkv) * hd].unflatten(1, (nkv, hd))


def prepare(case, seed):
    x = _inputs(case, seed)
    kind, T = case["kind"], case["T"]
    if kind == "quantise":
        x["values"] = torch.empty(T, case["K"], dtype=torch.bfloat16, device=DEVICE)
    elif kind in ("product", "weights"):
        out = "f32" if case.get("residual") else case.get("out", "bf16")
        x["y"] = torch.empty(T, case["N"], dtype=TYPES[out], device=DEVICE)
    else:
        if kind == "project":
            x["rows"] = torch.empty(T, _row(case), dtype=torch.bfloat16, device=DEVICE)
        x["freq"] = torch.tensor(_freqs(case), dtype=torch.float64, device=DEVICE)
        x["q"], x["k"] = _heads(case, x["rows"])
        x["q_out"] = torch.empty(T, case["nh"], case["hd"], dtype=x["rows"].dtype, device=DEVICE)
        x["k_out"] = torch.empty(T, case["nkv"], case["hd"], dtype=x["rows"].dtype, device=DEVICE)
    if own:
        from cleffa_amd import Mx4Matrix, Rotary
        if kind in ("quantise", "project"):
            x["m"] = Mx4Matrix(T, case["K" if kind == "quantise" else "H"], device=DEVICE)
        if kind == "product":
            x["x"] = Mx4Matrix.from_codes(x["x_codes"], x["x_scales"])
        if kind in ("product", "weights", "project"):
            x["w"] = Mx4Matrix.from_codes(x["w_codes"], x["w_scales"])
        if kind in ("rotary", "project"):
            scaling = None if case["scaling"] == "none" else {"kind": case["scaling"], "factor": case["factor"], "original": 16384}
            x["rotary"] = Rotary(case["n_rot"], theta=1e7, layout=case["layout"], axes=case["axes"], scaling=scaling, eps=EPS, device=DEVICE)
    return x


# ---- the plain forms

def _pow2(e):
    """2^e as float32, for -126 <= e <= 127."""
    return ((e + 127).int() << 23).view(torch.float32)


def _quantised(x):
    """f32 rows [T][K] to whole numbers of halves (-12 .. 12) and exponents [T][K / 32]."""
    b = x.float().unflatten(1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1))            # max = m * 2^e, m in [0.5, 1); 7 = 0.875 * 2^3
    e = torch.where(m < 0.875, e - 3, e - 2).clamp(min=-126)
    v = b / _pow2(e)[..., None]
    size = v.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    return ((torch.round(v / step) * step).clamp(-6, 6) * 2).to(torch.int8), e


def _codes(x):
    halves, e = _quantised(x)
    size = halves.abs()
    code = torch.where(size <= 4, size, torch.where(size == 6, 5, torch.where(size == 8, 6, 7)))
    code = (code + 8 * (halves < 0)).to(torch.uint8).flatten(1)
    return code[:, 0::2] | code[:, 1::2] << 4, (e + 127).to(torch.uint8)


def _values(codes, scales):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=DEVICE)
    table = torch.cat([table, -table])
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(1).int()
    return (table[c].unflatten(1, (-1, 32)) * _pow2(scales.int() - 127)[..., None]).flatten(1)


def _freqs(case):
    """Radians a position for each pair."""
    n, s, theta = case["n_rot"], case["factor"], 1e7
    if case["scaling"] == "base":
        theta *= s ** (n / (n - 2))
    f = theta ** (-np.arange(0, n, 2, dtype=np.float64) / n)
    if case["scaling"] == "linear":
        f = f / s
    if case["scaling"] == "parts":      # pairs that turn over 32 times in the first 16,384 tokens stay, those under once stretch
        keep = np.clip((16384 * f / (2 * math.pi) - 1) / 31, 0, 1)
        f = keep * f + (1 - keep) * f / s
    return f


def _magnitude(case):
    return 0.1 * math.log(case["factor"]) + 1 if case["scaling"] == "parts" else 1.0


def _rotated(x, heads, norm):
    case, n = x["case"], x["case"]["n_rot"]
    h = heads.float()
    if norm is not None:
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * norm
    axis = torch.arange(n // 2, device=DEVICE) % case["axes"]
    angle = (x["pos"].double()[:, axis] * x["freq"])[:, None]
    c, s = (t.float() * _magnitude(case) for t in (angle.cos(), angle.sin()))
    a, b = (h[..., :n // 2], h[..., n // 2:n]) if case["layout"] == "half" else (h[..., :n:2], h[..., 1:n:2])
    a, b = a * c - b * s, b * c + a * s
    turned = torch.cat([a, b], -1) if case["layout"] == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, h[..., n:]], -1).to(x["q_out"].dtype)


def run(x):
    case = x["case"]
    kind = case["kind"]
    if not own:
        if kind == "quantise":
            halves, e = _quantised(x["x"])
            return {"values": (halves.float() * 0.5 * _pow2(e)[..., None]).flatten(1).to(torch.bfloat16)}
        if kind in ("product", "weights"):
            a = _values(x["x_codes"], x["x_scales"]) if kind == "product" else x["x"].float()
            y = a @ _values(x["w_codes"], x["w_scales"]).T
            if case.get("residual"):
                y = y + x["residual"]
            return {"y": y.to(x["y"].dtype)}
        q, k, out = x["q"], x["k"], {}
        if kind == "project":
            halves, e = _quantised(x["x"])
            rows = (halves.float() * 0.5 * _pow2(e)[..., None]).flatten(1) @ _values(x["w_codes"], x["w_scales"]).T
            q, k = _heads(case, rows)
            out["rows"] = rows.to(torch.bfloat16)
        return dict(out, q=_rotated(x, q, x["q_norm"]), k=_rotated(x, k, x["k_norm"]))
    from cleffa_amd import mx4_gemm
    if kind == "quantise":
        x["m"].quantise(x["x"])
        return {"values": x["m"].values(out=x["values"])}
    if kind in ("product", "weights"):
        return {"y": mx4_gemm(x["x"], x["w"], Y=x["y"], residual=x.get("residual"))}
    if kind == "project":
        mx4_gemm(x["m"].quantise(x["x"]), x["w"], Y=x["rows"])
    x["rotary"].apply(x["q"], x["k"], x["pos"], x["q_norm"], x["k_norm"], q_out=x["q_out"], k_out=x["k_out"])
    return {"rows": x["rows"], "q": x["q_out"], "k": x["k_out"]} if kind == "project" else {"q": x["q_out"], "k": x["k_out"]}


# ---- the same in 64 bits

def _nearest64(x):
    """Each value of rows [T][K] as the nearest of its block's grid, in float64: the grid written out, ties to every second of it."""
    b = x.double().unflatten(1, (-1, 32))
    scale = torch.exp2(torch.floor(torch.log2(b.abs().amax(-1, keepdim=True).clamp(min=1e-300) / 7)) + 1)
    v = b / scale
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEVICE)
    size = v.abs().contiguous()
    middle = (grid[1:] + grid[:-1]) / 2
    below, above = torch.searchsorted(middle, size), torch.searchsorted(middle, size, right=True)
    at = torch.where(below == above, below, torch.where(below % 2 == 0, below, above))     # a tie: the even one
    return (grid[at] * torch.sign(v) * scale).flatten(1)


def _decoded64(codes, scales):
    c = torch.stack([codes % 16, codes // 16], -1).flatten(1).long()
    e, f = (c >> 1) & 3, (c & 1).double()      # sign, two exponent bits of bias 1, one fraction bit
    v = torch.where(e > 0, torch.exp2(e.double() - 1) * (1 + f / 2), f / 2) * torch.where(c >= 8, -1.0, 1.0)
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)


def _freq64(case, j):
    n, s = case["n_rot"], case["factor"]
    base = 1e7 * (s ** (n / (n - 2)) if case["scaling"] == "base" else 1)
    f = math.exp(-2 * j / n * math.log(base))
    if case["scaling"] == "linear":
        return f / s
    if case["scaling"] == "parts":
        turns = 16384 * f / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1) / (32 - 1)))
        return f / s + keep * (f - f / s)
    return f


def _turned64(case, heads, pos, norm):
    n = case["n_rot"]
    h = heads.double().clone()
    if norm is not None:
        h = h / (h.pow(2).sum(-1, keepdim=True) / case["hd"] + EPS).sqrt() * norm.double()
    m = 1 + 0.1 * math.log(case["factor"]) if case["scaling"] == "parts" else 1.0
    f = torch.tensor([_freq64(case, j) for j in range(n // 2)], dtype=torch.float64, device=DEVICE)
    ang = pos[:, [j % case["axes"] for j in range(n // 2)]].double() * f
    z = torch.polar(torch.full_like(ang, m), ang)[:, None]
    first, second = (slice(0, n // 2), slice(n // 2, n)) if case["layout"] == "half" else (slice(0, n, 2), slice(1, n, 2))
    y = torch.complex(h[..., first].contiguous(), h[..., second].contiguous()) * z
    h[..., first], h[..., second] = y.real, y.imag
    return h


def exact(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "quantise":
        return {"values": _nearest64(x["x"])}
    if kind in ("product", "weights"):
        a = _decoded64(x["x_codes"], x["x_scales"]) if kind == "product" else x["x"].double()
        y = torch.mm(a, _decoded64(x["w_codes"], x["w_scales"]).t())
        return {"y": y + x["residual"].double() if case.get("residual") else y}
    out = {}
    rows = x.get("rows")
    if kind == "project":
        out["rows"] = rows = torch.mm(_nearest64(x["x"]), _decoded64(x["w_codes"], x["w_scales"]).t())
    q, k = _heads(case, rows)
    return dict(out, q=_turned64(case, q, x["pos"], x["q_norm"]), k=_turned64(case, k, x["pos"], x["k_norm"]))
