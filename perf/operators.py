"""Performance cases of the 8-bit paged prefix cache: what a program that serves from it has it do.

The cache holds keys and values as e4m3 codes in pages of 64 tokens, with one power-of-two scale for each
page and kv head. Per layer: K codes [pages][nkv][4][64][64] (dim group, token, dim), V codes
[pages][nkv][256][64] (dim, token), scales [pages][nkv]. ``tables`` names the pages of each sequence,
``state`` is {free pages, status, (tokens, pages held) of each sequence}, ``free`` the stack of free pages.
Four kinds of call, each alone, and the three of a serving step together:

* ``plan``    page tables, slot map and positions of a pass, on the GPU, from the lengths (``Kv8Plan.update``);
* ``append``  a pass's new keys (norm, rotary) and values into the pages (``TextAttention.forward_kv8``,
              stage "append"), and the pages they went to read back into 16-bit planes;
* ``read``    whole sequences read back into 16-bit planes (``Kv8Cache.read``);
* ``attend``  gated grouped-query attention of the new tokens over the cache (stage "core");
* ``step``    plan, append and attention of one layer.

``exact`` restates each in float64.
"""
import ctypes
import math

import numpy as np
import torch

own = False

HD, N_ROT, THETA, EPS = 256, 64, 1e7, 1e-6    # head dim, rotary dims, frequency base
PAGE = 64
DEVICE = "cuda"
OUT = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    """``seqs``: the sequences of the pass as cached+new tokens; "64~30:8000+1" is 64 sequences of mixed lengths
    between 30 and 8,000. 0 new tokens: the sequence rests; -1: it has ended and gives its pages back."""
    return [
        # a decoding batch's next tokens: nothing but latency
        {"name": "plan_tokens", "kind": "plan", "seqs": "64~30:8000+1", "nh": 24, "nkv": 4},
        # a server's full table: a long prompt comes in, others go on, rest or end
        {"name": "plan_mixed", "kind": "plan", "seqs": "0+16384,300~1:4000+1,100~1:4000+0,60~1:4000+-1,7x100+13", "nh": 16, "nkv": 4},
        # one new token in each of 64 sequences
        {"name": "append_tokens", "kind": "append", "seqs": "64~30:8000+1", "nh": 24, "nkv": 4},
        # the ordinary micro-batch (eight requests, 4,096 tokens) behind cached prefixes of odd lengths
        {"name": "append_packed", "kind": "append", "seqs": "0+1160,37+890,640+730,1+425,4091+472,63+136,64+179,2000+104", "nh": 24, "nkv": 4},
        # a cached document brought back for the 16-bit path
        {"name": "read_document", "kind": "read", "seqs": "4091+0", "nh": 24, "nkv": 4},
        # a long one and a few short ones
        {"name": "read_long", "kind": "read", "seqs": "65000+0,7x2050+0", "nh": 16, "nkv": 4},
        # the next token of one request on a cached document
        {"name": "attend_token", "kind": "attend", "seqs": "4091+1", "nh": 24, "nkv": 4},
        # the next token of one request behind a very long text
        {"name": "attend_token_long", "kind": "attend", "seqs": "130000+1", "nh": 16, "nkv": 4},
        # the next tokens of a batch of mixed lengths
        {"name": "attend_tokens", "kind": "attend", "seqs": "64~30:8000+1", "nh": 24, "nkv": 4},
        # a short question on a cached document
        {"name": "attend_question", "kind": "attend", "seqs": "4091+45", "nh": 24, "nkv": 4},
        # four requests that continue a cached prefix by 512 tokens each
        {"name": "attend_packed", "kind": "attend", "seqs": "4x2048+512", "nh": 16, "nkv": 4},
        # a whole serving step of one layer for a small batch
        {"name": "step_tokens", "kind": "step", "seqs": "32~100:4000+1", "nh": 24, "nkv": 4},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "plan", "append", "append", "read", "attend", "attend", "attend", "attend", "step"])
    nh, nkv = rng.choice([(24, 4), (24, 4), (16, 4), (32, 4), (8, 2), (16, 8), (16, 1), (20, 4)])
    c = {"kind": kind, "nh": nh, "nkv": nkv}
    if kind == "plan":
        parts = ["%d~1:%d+1" % (_log(rng, 1, 400), _log(rng, 10, 8000))]
        if rng.random() < 0.6:
            parts.append("%d+%d" % (rng.randint(0, 5000), _log(rng, 2, 16384)))
        if rng.random() < 0.5:
            parts.append("%d~1:3000+-1" % rng.randint(1, 60))
        if rng.random() < 0.5:
            parts.append("%d~1:3000+0" % rng.randint(1, 60))
        rng.shuffle(parts)
        c["seqs"] = ",".join(parts)
    elif kind == "append":
        if rng.random() < 0.5:
            c["seqs"] = "%d~1:%d+%d" % (_log(rng, 1, 200), _log(rng, 10, 8000), rng.randint(1, 8))
        else:
            n = rng.choice([1, 1, 2, 5, 9])
            c["seqs"] = ",".join("%d+%d" % (rng.choice([0, rng.randint(1, 5000)]), _log(rng, 2, 6000 // n + 2)) for _ in range(n))
    elif kind == "read":
        n = rng.choice([1, 1, 3, 10])
        c["seqs"] = ",".join("%d+0" % _log(rng, 1, 60000 // n) for _ in range(n))
    elif kind == "step" or rng.random() < 0.5:
        n = _log(rng, 1, 64)
        c["seqs"] = "%d~1:%d+%d" % (n, _log(rng, 10, 100000 // n if n < 12 else 8000), rng.choice([1, 1, 1, 2, 3, 5]))
    else:
        n = rng.choice([1, 1, 2, 4])
        c["seqs"] = ",".join("%d+%d" % (_log(rng, 1, 12000 // n), _log(rng, 2, 1000 // n)) for _ in range(n))
    if kind in ("attend", "step"):
        if rng.random() < 0.3:
            c["out"] = "f16"
        if rng.random() < 0.2:
            c["plain"] = True      # no norms, rotary or gate
    return c


# ---- what a case says

def _seqs(case):
    """(cached, new) tokens of each sequence."""
    out = []
    for part in case["seqs"].split(","):
        cached, new = part.split("+")
        if "~" in cached:
            n, span = cached.split("~")
            lo, hi = span.split(":")
            n, r = int(n), np.random.default_rng(len(part))
            out += [(int(round(float(x))), int(new)) for x in np.exp(r.uniform(math.log(int(lo)), math.log(int(hi)), n))]
        else:
            n, _, v = cached.rpartition("x")
            out += [(int(v), int(new))] * int(n or 1)
    return out


def _ceil(a, b):
    return -(-a // b)


def work(case):
    kind, nh, nkv, seqs = case["kind"], case["nh"], case["nkv"], _seqs(case)
    T = sum(max(q, 0) for _, q in seqs)
    plan = {"bytes": 4 * (sum(_ceil(L + q, PAGE) - _ceil(L, PAGE) if q > 0 else 0 for L, q in seqs) * 2
                          + sum(_ceil(L, PAGE) for L, q in seqs if q < 0) * 2 + len(seqs) * 7 + T * 4), "flops": 0}
    if kind == "plan":
        return plan
    touched = sum(_ceil(L + q, PAGE) - L // PAGE for L, q in seqs if q > 0)
    new = {"bytes": T * nkv * HD * 2 * (2 + 1) + T * 12 + touched * nkv * 8, "flops": 0}
    if kind == "append":   # bf16 in, codes out; the pages' rows read back as 16 bits
        rows = sum(L % PAGE + q for L, q in seqs if q > 0)
        return {"bytes": new["bytes"] + rows * nkv * HD * 2 * (1 + 2), "flops": 0}
    if kind == "read":
        return {"bytes": sum(L for L, _ in seqs) * nkv * HD * 2 * (1 + 2), "flops": 0}
    keys = sum(L + q for L, q in seqs if q > 0)
    pairs = sum(q * L + q * (q + 1) // 2 for L, q in seqs if q > 0)
    w = {"bytes": keys * nkv * HD * 2 + T * nh * HD * ((1 if case.get("plain") else 2) * 2 + 2) + T * 12,
         "flops": 4 * HD * nh * pairs}
    if kind == "step":
        w["bytes"] += plan["bytes"] + new["bytes"]
    return w


# ---- inputs

def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(1000003 * seed + 29)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32)


def _inv_freq():
    """1 / theta^(2j / n) in f32: the frequency table is an FP32 input of the model."""
    powf = ctypes.CDLL("libm.so.6").powf
    powf.restype, powf.argtypes = ctypes.c_float, [ctypes.c_float, ctypes.c_float]
    f = [np.float32(1) / np.float32(powf(THETA, np.float32(2 * j) / np.float32(N_ROT))) for j in range(N_ROT // 2)]
    return torch.from_numpy(np.array(f, dtype=np.float32)).to(DEVICE)


def _int(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEVICE)


def _inputs(case, seed):
    """The pass's lengths and rows, and a cache that holds the cached tokens (of ``attend``: the new ones too)."""
    kind, nh, nkv, seqs = case["kind"], case["nh"], case["nkv"], _seqs(case)
    g, rng = _gen(seed), np.random.default_rng(seed)
    L = np.array([a for a, _ in seqs], dtype=np.int64)
    new = np.array([b for _, b in seqs], dtype=np.int64)
    q = np.maximum(new, 0)
    done = kind in ("append", "attend")     # the pages of the new tokens are in the table already
    held = -(-(L + q * done) // PAGE)
    want = -(-(L + q) // PAGE)
    max_pages = int(want.max()) + 1
    n_pages = int(np.maximum(held, want).sum()) + 8
    perm = rng.permutation(n_pages).astype(np.int32)
    tables = np.full((len(seqs), max_pages), -1, dtype=np.int32)
    at = 0
    for r, h in enumerate(held):
        tables[r, :h] = perm[at:at + h]
        at += h
    free = np.full(n_pages, -1, dtype=np.int32)
    free[:n_pages - at] = perm[at:]
    state = np.zeros(2 + 2 * len(seqs), dtype=np.int32)
    state[0], state[2::2], state[3::2] = n_pages - at, L, held
    T = int(q.sum())
    x = {"case": case, "new": _int(new), "tables": _int(tables), "free": _int(free), "state": _int(state),
         "pos_off": _int(rng.integers(-20, 1, len(seqs)) * (L > 100)), "T": T, "n_pages": n_pages, "max_new": int(q.max())}
    if kind == "plan":
        x["T"] = T + 3       # the rows behind the last sequence take no slot
        return x
    seq = np.repeat(np.arange(len(seqs)), q)
    pos = np.concatenate([np.arange(a, a + b) for a, b in zip(L, q)]) if T else np.zeros(0)
    x.update(seq=_int(seq), pos=_int(pos), pos3=_int(np.repeat(pos[:, None], 3, axis=1)))
    if kind != "read":
        scale = torch.where(torch.rand(2 * (nh + nkv) * HD, generator=g, device=DEVICE) < 0.02, 4.0, 1.0)
        x["qkv"] = (_randn(g, T, 2 * (nh + nkv) * HD) * scale).to(torch.bfloat16)
    plain = bool(case.get("plain"))
    x["q_norm"], x["k_norm"] = (None, None) if plain else (1 + 0.1 * _randn(g, HD), 1 + 0.1 * _randn(g, HD))
    # codes over e4m3's whole range (the largest of a page is between 224 and 448), scales around 2^-7
    x["k"] = (_randn(g, n_pages, nkv, 4, 64, 64) * 70).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    x["v"] = (_randn(g, n_pages, nkv, HD, 64) * 70).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    for name in ("k_scale", "v_scale"):
        x[name] = _pow2(torch.randint(-7, -5, (n_pages, nkv), generator=g, device=DEVICE))
    if kind == "append":     # the pages that take new tokens, and the rows they come back to
        first = L // PAGE
        count = np.where(q > 0, -(-(L + q) // PAGE) - first, 0)
        t_seq = np.repeat(np.arange(len(seqs)), count)
        t_page = np.concatenate([np.arange(f, f + c) for f, c in zip(first, count)])
        cu = np.concatenate([[0], np.cumsum(count)])
        x.update(t_seq=_int(t_seq), t_page=_int(t_page), touched=_int(cu[seq] + pos // PAGE - first[seq]),
                 first_page=_int(first), cu=_int(PAGE * cu), rows=int(PAGE * cu[-1]))
    if kind == "read":
        cu = np.concatenate([[0], np.cumsum(-(-L // 8) * 8)])
        x.update(first_page=_int(0 * L), cu=_int(cu), rows=int(cu[-1]), r_seq=_int(np.repeat(np.arange(len(seqs)), L)),
                 r_pos=_int(np.concatenate([np.arange(n) for n in L])),
                 r_row=_int(np.concatenate([c + np.arange(n) for c, n in zip(cu, L)])))
    if kind in ("attend", "step"):
        cu_q = np.concatenate([[0], np.cumsum(q)])
        x.update(cu_q=_int(cu_q), n_keys=_int(L + q), most_pages=int(want.max()))
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    kind, nh, nkv, T = case["kind"], case["nh"], case["nkv"], x["T"]
    x["inv_freq"] = _inv_freq()
    x["state_out"] = torch.empty_like(x["state"])
    if "rows" in x:
        x["k_plane"] = torch.zeros(nkv, x["rows"], HD, dtype=torch.float16, device=DEVICE)
        x["vt_plane"] = torch.zeros(nkv, HD, x["rows"], dtype=torch.bfloat16, device=DEVICE)
    if kind in ("attend", "step"):
        x["out"] = torch.empty(T, nh * HD, dtype=OUT[case.get("out", "bf16")], device=DEVICE)
    if own:
        from cleffa_amd import Kv8Cache, Kv8Plan, TextAttention
        cache = Kv8Cache(1, nkv, x["n_pages"], len(_seqs(case)), x["tables"].shape[1], device=DEVICE, allocate="k" not in x)
        if "k" in x:
            cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0] = x["k"], x["v"], x["k_scale"], x["v_scale"]
        cache.tables, cache.free, cache.state = x["tables"], x["free"], x["state"]
        x["cache"] = cache
        if kind != "read":
            x["att"] = TextAttention(nh, nkv, HD, 0 if case.get("plain") else N_ROT, EPS, THETA, device=DEVICE)
            x["plan"] = Kv8Plan(cache, T, nh, x["max_new"])
            if kind in ("append", "attend"):
                x["plan"].update(x["new"])
    return x


# ---- the plain forms

def _plain_plan(x):
    new, state, tables = x["new"].long(), x["state"].long(), x["tables"].clone()
    L, held, n_free = state[2::2], state[3::2], state[0]
    gone, q = new < 0, new.clamp(min=0)
    col = torch.arange(tables.shape[1], device=DEVICE)
    back = tables[gone[:, None] & (col < held[:, None])]
    free = x["free"].index_copy(0, n_free + torch.arange(back.numel(), device=DEVICE), back)
    n_free = n_free + back.numel()
    add = torch.where(gone, 0, ((L + q + PAGE - 1) // PAGE - held).clamp(min=0))
    take = (col >= held[:, None]) & (col < (held + add)[:, None])
    order = torch.cumsum(take.reshape(-1), 0).reshape(take.shape) - 1
    tables = torch.where(take, free[(n_free - 1 - order).clamp(min=0)], tables)
    after = torch.stack([torch.where(gone, 0, L + q), torch.where(gone, 0, held + add)], 1).reshape(-1)
    state_out = torch.cat([torch.stack([n_free - add.sum(), torch.zeros_like(n_free)]), after]).int()
    cu_q = torch.cat([torch.zeros_like(n_free)[None], torch.cumsum(q, 0)])
    row = torch.arange(x["T"], device=DEVICE)
    r = torch.searchsorted(cu_q, row, right=True) - 1
    there = row < cu_q[-1]
    r = r.clamp(max=len(new) - 1)
    pos = L[r] + row - cu_q[r]
    slots = torch.where(there, tables[r, torch.where(there, pos // PAGE, 0)].long() * PAGE + pos % PAGE, -1).int()
    pos3 = torch.where(there, pos + x["pos_off"].long()[r], 0).int()[:, None].expand(-1, 3).contiguous()
    return {"tables": tables, "free": free, "state": state_out, "cu_q": cu_q.int(), "slots": slots, "pos3": pos3}


def _normed(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _turned(x, ang):
    """Pair i of the first 64 dims is (i, i + 32)."""
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., :32], x[..., 32:64]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 64:]], -1)


def _angles(x):
    """Pair i turns by position axis i % 3; the angle is the FP32 product of position and frequency."""
    return x["pos3"][:, torch.arange(N_ROT // 2, device=DEVICE) % 3].float() * x["inv_freq"]


def _values(codes, scale):
    return codes.view(torch.float8_e4m3fn).float() * scale[..., None, None]


def _pow2(e):
    return ((e + 127).int() << 23).view(torch.float32)


def _page_scale(most, before):
    """The least 2^e, e >= -64, with 448 * 2^e >= most, and no less than the scale before."""
    m, e = torch.frexp(most)      # most = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(most > 0, torch.where(m <= 0.875, e - 9, e - 8), -64).clamp(min=-64)
    return torch.maximum(_pow2(e), before)


def _coded(x, scale):
    return (x / scale).to(torch.float8_e4m3fn).float() * scale


def _plain_append(x, tables):
    """(K, V) [touched pages][nkv][64 tokens][256] as the pages hold them after the pass, and their pages."""
    case = x["case"]
    nh, nkv = case["nh"], case["nkv"]
    k = _normed(x["qkv"][:, 2 * nh * HD:(2 * nh + nkv) * HD].float().view(-1, nkv, HD), x["k_norm"])
    if not case.get("plain"):
        k = _turned(k, _angles(x))
    v = x["qkv"][:, (2 * nh + nkv) * HD:2 * (nh + nkv) * HD].float().view(-1, nkv, HD)
    page = tables[x["t_seq"].long(), x["t_page"].long()].long()
    off, to = (x["pos"] % PAGE).long(), x["touched"].long()
    n = len(page)
    # tokens that the page held before the pass
    before = (x["state"][2::2].long()[x["t_seq"].long()] - x["t_page"].long() * PAGE).clamp(0, PAGE)
    old = torch.arange(PAGE, device=DEVICE) < before[:, None]
    out = []
    for new, codes, scale in ((k, x["k"], x["k_scale"]), (v, x["v"], x["v_scale"])):
        c = codes[page]
        c = c.permute(0, 1, 3, 2, 4).reshape(n, nkv, PAGE, HD) if codes.dim() == 5 else c.transpose(2, 3).contiguous()
        was = torch.where(before[:, None] > 0, scale[page], 0.0)
        most = torch.zeros(n, nkv, device=DEVICE).index_reduce(0, to, new.abs().amax(-1), "amax")
        s = _page_scale(most, was)
        held = _coded(torch.where(old[:, None, :, None], _values(c, was), 0.0), s[..., None, None])
        held = held.transpose(1, 2).contiguous()      # [page][token][nkv][dim]
        held[to, off] = _coded(new, s[to][..., None])
        out.append(held.transpose(1, 2))
    return out[0], out[1], page


def _planes(k, v):
    """[pages][nkv][64][256] to K [nkv][rows][256] f16 and V^T [nkv][256][rows] bf16."""
    k = k.transpose(0, 1).reshape(k.shape[1], -1, HD)
    v = v.transpose(0, 1).reshape(v.shape[1], -1, HD).transpose(1, 2)
    return {"k_plane": k.clamp(-65504, 65504).to(torch.float16).contiguous(), "vt_plane": v.to(torch.bfloat16).contiguous()}


def _plain_read(x):
    page = x["tables"][x["r_seq"].long(), (x["r_pos"] // PAGE).long()].long()
    off, row = (x["r_pos"] % PAGE).long(), x["r_row"].long()
    k = _values(x["k"], x["k_scale"][..., None])[page, :, :, off].reshape(len(row), -1, HD)
    v = _values(x["v"], x["v_scale"])[page, :, :, off]
    k_plane, vt_plane = torch.zeros_like(x["k_plane"]), torch.zeros_like(x["vt_plane"])
    k_plane[:, row] = k.clamp(-65504, 65504).to(torch.float16).transpose(0, 1)
    vt_plane[:, :, row] = v.to(torch.bfloat16).permute(1, 2, 0)
    return {"k_plane": k_plane, "vt_plane": vt_plane}


def _plain_attend(x, tables, k_page, v_page):
    """k_page(pages), v_page(pages): K and V [..., nkv, 64, 256] of the named pages."""
    case = x["case"]
    nh, nkv = case["nh"], case["nkv"]
    G, T, B, n = nh // nkv, x["T"], len(x["new"]), x["max_new"]
    qg = x["qkv"][:, :2 * nh * HD].float().view(T, nh, 2, HD)
    q, gate = _normed(qg[:, :, 0], x["q_norm"]), qg[:, :, 1]
    if not case.get("plain"):
        q = _turned(q, _angles(x))
    pages = tables[:, :x["most_pages"]].long().clamp(min=0)
    keys = pages.shape[1] * PAGE
    k = k_page(pages).permute(0, 2, 1, 3, 4).reshape(B, nkv, keys, HD)
    v = v_page(pages).permute(0, 2, 1, 3, 4).reshape(B, nkv, keys, HD)
    seq, at = x["seq"].long(), torch.arange(T, device=DEVICE) - x["cu_q"].long()[x["seq"].long()]
    qs = torch.zeros(B, n, nkv, G, HD, device=DEVICE)
    qs[seq, at] = q.view(T, nkv, G, HD)
    last = torch.full((B, n), -1, dtype=torch.int32, device=DEVICE)      # the last key a query sees
    last[seq, at] = x["pos"]
    s = (qs.permute(0, 2, 1, 3, 4).reshape(B, nkv, n * G, HD) @ k.transpose(2, 3)) * HD ** -0.5
    seen = torch.arange(keys, device=DEVICE) <= last.clamp(min=0)[:, :, None]
    s = torch.where(seen[:, None, :, None, :], s.view(B, nkv, n, G, keys), -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = (p.view(B, nkv, n * G, keys) @ v).view(B, nkv, n, G, HD) / p.sum(-1, keepdim=True)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, n, nh, HD)[seq, at]
    if not case.get("plain"):
        o = o * torch.sigmoid(gate)
    return o.reshape(T, nh * HD).to(OUT[case.get("out", "bf16")])


def _pool(codes, scale):
    """A lookup of pages, as [..., nkv, 64, 256] values."""
    def pages(at):
        c = _values(codes[at], scale[at][..., None] if codes.dim() == 5 else scale[at])
        return c.transpose(-3, -2).flatten(-2) if codes.dim() == 5 else c.transpose(-2, -1)
    return pages


def _plain_step(x):
    plan = _plain_plan(x)
    first, last = x["state"][2::2].long() // PAGE, (x["state"][2::2].long() + x["new"].long().clamp(min=0) + PAGE - 1) // PAGE
    count = torch.where(x["new"] > 0, last - first, 0)
    at = torch.cumsum(count, 0) - count
    seq = torch.repeat_interleave(torch.arange(len(count), device=DEVICE), count)
    page = first[seq] + torch.arange(len(seq), device=DEVICE) - at[seq]
    token = x["seq"].long()
    y = dict(x, t_seq=seq, t_page=page, touched=at[token] + x["pos"].long() // PAGE - first[token])
    k, v, where = _plain_append(y, plan["tables"])
    k_all, v_all = (_pool(x[n], x[n + "_scale"])(torch.arange(x["n_pages"], device=DEVICE)) for n in ("k", "v"))
    k_all, v_all = k_all.index_copy(0, where, k), v_all.index_copy(0, where, v)
    out = _plain_attend(x, plan["tables"], lambda at: k_all[at], lambda at: v_all[at])
    return {"out": out, "state": plan["state"], "slots": plan["slots"], "tables": plan["tables"]}


def run(x):
    case = x["case"]
    kind = case["kind"]
    if not own:
        if kind == "plan":
            return _plain_plan(x)
        if kind == "append":
            k, v, _ = _plain_append(x, x["tables"])
            return _planes(k, v)
        if kind == "read":
            return _plain_read(x)
        if kind == "attend":
            return {"out": _plain_attend(x, x["tables"], _pool(x["k"], x["k_scale"]), _pool(x["v"], x["v_scale"]))}
        return _plain_step(x)
    cache, plan = x["cache"], x.get("plan")
    if kind == "plan":
        plan.update(x["new"], pos_off=x["pos_off"], state_out=x["state_out"])
        return {"tables": cache.tables, "free": cache.free, "state": x["state_out"], "cu_q": plan.cu_q, "slots": plan.slots, "pos3": plan.pos3}
    if kind == "read":
        cache.read(0, x["cu"], x["k_plane"], x["vt_plane"])
        return {"k_plane": x["k_plane"], "vt_plane": x["vt_plane"]}
    rows = (x["qkv"], x["q_norm"], x["k_norm"], x["pos3"])
    if kind == "append":
        x["att"].forward_kv8(*rows, plan, cache, 0, stage="append")
        cache.read(0, x["cu"], x["k_plane"], x["vt_plane"], first_page=x["first_page"])
        return {"k_plane": x["k_plane"], "vt_plane": x["vt_plane"]}
    if kind == "step":
        plan.update(x["new"], state_out=x["state_out"])
    x["att"].forward_kv8(*rows, plan, cache, 0, out=x["out"], out_dtype=case.get("out", "bf16"), gate=not case.get("plain"),
                         stage="core" if kind == "attend" else "prefill")
    return {"out": x["out"]} if kind == "attend" else {"out": x["out"], "state": x["state_out"], "slots": plan.slots, "tables": cache.tables}


# ---- the same in 64 bits

def _e4m3(x):
    """The nearest e4m3 value (ties to even), |x| <= 448: steps of 2^(e - 3) in [2^e, 2^(e + 1)), of 2^-9 below 2^-6."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def _decode(codes):
    """e4m3 codes to float64: sign, four exponent bits of bias 7, three fraction bits."""
    c = codes.long()
    e, f = (c >> 3) & 15, (c & 7).double()
    x = torch.where(e > 0, torch.exp2(e.double() - 7) * (1 + f / 8), f * 2.0 ** -9)
    return torch.where(c >= 128, -x, x)


def _rows64(x):
    """Normalised, rotated queries and keys, values and gates of the pass, in float64."""
    case = x["case"]
    nh, nkv, T = case["nh"], case["nkv"], x["T"]
    h = x["qkv"].double()
    qg = h[:, :2 * nh * HD].view(T, nh, 2, HD)
    q, k = qg[:, :, 0], h[:, 2 * nh * HD:(2 * nh + nkv) * HD].view(T, nkv, HD)
    if not case.get("plain"):
        q, k = (t / (t.pow(2).sum(-1, keepdim=True) / HD + EPS).sqrt() * w.double() for t, w in ((q, x["q_norm"]), (k, x["k_norm"])))
        ang = (x["pos3"][:, [i % 3 for i in range(32)]].float() * _inv_freq()).double()
        z = torch.polar(torch.ones_like(ang), ang)[:, None]
        for t in (q, k):
            y = torch.complex(t[..., :32].contiguous(), t[..., 32:64].contiguous()) * z
            t[..., :32], t[..., 32:64] = y.real, y.imag
    return q, k, h[:, (2 * nh + nkv) * HD:].view(T, nkv, HD), qg[:, :, 1]


def _cache64(x, r, n, tables):
    """K and V [nkv][n][256] of the first n tokens that sequence r holds."""
    pages = tables[r, :_ceil(n, PAGE)].long()
    k = _decode(x["k"][pages]) * x["k_scale"][pages].double()[..., None, None, None]
    v = _decode(x["v"][pages]) * x["v_scale"][pages].double()[..., None, None]
    k = torch.cat([k[:, :, g] for g in range(4)], -1)                 # [page][nkv][64][256]
    return (torch.cat(list(t), 1)[:, :n] for t in (k, v.transpose(2, 3)))


def _appended64(x, r, tables, k, v, rows):
    """The pages' tokens after the pass: K and V [nkv][64 * pages from the first touched][256], and that page."""
    L, q = _seqs(x["case"])[r]
    first, last = L // PAGE, _ceil(L + q, PAGE)
    out = []
    for new, codes, scale in ((k, "k", "k_scale"), (v, "v", "v_scale")):
        y = torch.zeros(new.shape[1], (last - first) * PAGE, HD, dtype=torch.float64, device=DEVICE)
        n_old = L - first * PAGE
        both = new[rows].transpose(0, 1)
        for p in range(first, last):
            a, b = max(L, p * PAGE), min(L + q, (p + 1) * PAGE)
            t = both[:, a - L:b - L]
            s = torch.exp2(torch.ceil(torch.log2(t.abs().amax((1, 2)) / 448)).clamp(min=-64))
            old = n_old if p == first else 0
            if old:
                page = int(tables[r, p])
                was = _decode(x[codes][page])
                was = torch.cat(list(was.transpose(0, 1)), -1) if codes == "k" else was.transpose(1, 2)
                s = torch.maximum(s, x[scale][page].double())
                was = was[:, :old] * x[scale][page].double()[:, None, None]
                y[:, :old] = _e4m3(was / s[:, None, None]) * s[:, None, None]
            lo = (p - first) * PAGE
            y[:, lo + a - p * PAGE:lo + b - p * PAGE] = _e4m3(t / s[:, None, None]) * s[:, None, None]
        out.append(y)
    return out[0], out[1], first


def _tables64(x):
    """The page tables after a pass that ends no sequence."""
    tables, free, at = x["tables"].cpu().clone(), x["free"].cpu(), int(x["state"][0]) - 1
    for r, (L, q) in enumerate(_seqs(x["case"])):
        for p in range(_ceil(L, PAGE), _ceil(L + q, PAGE)):
            tables[r, p] = free[at]
            at -= 1
    return tables.to(DEVICE)


def exact(case, seed):
    kind, seqs = case["kind"], _seqs(case)
    if kind == "plan":
        return None
    nh, nkv = case["nh"], case["nkv"]
    if 4 * HD * nh * sum(max(q, 0) * (L + q) for L, q in seqs) > 4e12:
        return None
    x = _inputs(case, seed)
    if kind == "read":
        cu = x["cu"].tolist()
        k = torch.zeros(nkv, x["rows"], HD, dtype=torch.float64, device=DEVICE)
        v = torch.zeros_like(k)
        for r, (L, _) in enumerate(seqs):
            k[:, cu[r]:cu[r] + L], v[:, cu[r]:cu[r] + L] = _cache64(x, r, L, x["tables"])
        return {"k_plane": k.clamp(-65504, 65504), "vt_plane": v.transpose(1, 2)}
    q, k, v, gate = _rows64(x)
    tables = _tables64(x) if kind == "step" else x["tables"]
    out, ks, vs, at = torch.empty(x["T"], nh, HD, dtype=torch.float64, device=DEVICE), [], [], 0
    for r, (L, n) in enumerate(seqs):
        rows = slice(at, at + n)
        at += n
        if kind != "attend":
            k_new, v_new, first = _appended64(x, r, tables, k, v, rows)
            ks.append(k_new)
            vs.append(v_new)
        if kind == "append":
            continue
        kc, vc = _cache64(x, r, L + n, tables)
        if kind == "step":
            kc = torch.cat([kc[:, :first * PAGE], k_new], 1)[:, :L + n]
            vc = torch.cat([vc[:, :first * PAGE], v_new], 1)[:, :L + n]
        hide = torch.arange(L + n, device=DEVICE) > torch.arange(L, L + n, device=DEVICE)[:, None]
        for h in range(nh):
            s = (q[rows, h] @ kc[h // (nh // nkv)].T / 16).masked_fill(hide, -math.inf)
            out[rows, h] = torch.softmax(s, -1) @ vc[h // (nh // nkv)]
    if kind == "append":
        return {"k_plane": torch.cat(ks, 1).clamp(-65504, 65504), "vt_plane": torch.cat(vs, 1).transpose(1, 2)}
    if not case.get("plain"):
        out = out * torch.sigmoid(gate)
    res = {"out": out.reshape(x["T"], nh * HD)}
    return res if kind == "attend" else dict(res, state=None, slots=None, tables=None)
