"""The 8-bit paged cache on the GPU against tests/kv8_ref.py: page bookkeeping exactly, codes to half a
step (exactly where no arithmetic comes before them), attention to the bound that kv8_ref.attend derives."""
import numpy as np
import pytest
import torch

from cleffa_amd import AttnPlan, Kv8Cache, Kv8Plan, TextAttention
from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
HD, PAGE = 256, 64
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def _say(*a):
    print("[kv8]", *a, flush=True)


def _int(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _np(t):
    return t.detach().cpu().double().numpy() if t.is_floating_point() else t.detach().cpu().numpy()


def _qkv(T, nh, nkv, seed, extra=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, 2 * (nh + nkv) * HD + extra), generator=g) * scale
    return x.to(torch.bfloat16).cuda(), (1 + 0.1 * torch.randn(HD, generator=g)).cuda(), (1 + 0.1 * torch.randn(HD, generator=g)).cuda()


def _cache_values(cache, layer=0):
    """Host copies of the pages' code values, K and V [n_pages][nkv][64][256], and scales."""
    k, v = ref.page_values(cache.k[layer].cpu().numpy(), cache.v[layer].cpu().numpy())
    return k, v, _np(cache.k_scale[layer]), _np(cache.v_scale[layer])


def _sequence(cache, values, model, r, n):
    """K, V [nkv][n][256] that sequence r's first n tokens hold."""
    pages = model.tables[r, :-(-n // PAGE)]
    k, v, ks, vs = values
    kk = (k[pages] * ks[pages][..., None, None]).transpose(1, 0, 2, 3).reshape(cache.nkv, -1, HD)[:, :n]
    vv = (v[pages] * vs[pages][..., None, None]).transpose(1, 0, 2, 3).reshape(cache.nkv, -1, HD)[:, :n]
    return kk, vv


def _check_attention(out, model_len_before, new, cu, q, gate, cache, model, values, scale, use_gate, out_dtype="bf16"):
    got = _np(out.float())
    worst = 0.0
    for r, n in enumerate(new):
        if n <= 0:
            continue
        L = model_len_before[r]
        kk, vv = _sequence(cache, values, model, r, L + n)
        rows = slice(cu[r], cu[r + 1])
        want, off = ref.attend(q[rows], gate[rows], kk, vv, L, scale, use_gate)
        off = off + HALF_STEP[out_dtype] * (np.abs(want) + off)
        d = np.abs(got[rows].reshape(want.shape) - want)
        assert np.isfinite(d).all(), f"sequence {r}"
        worst = max(worst, float((d / off).max()))
    _say(f"largest error {worst:.3f} of its bound")
    assert worst <= 1.0


def _run(nh, nkv, passes, seed=0, n_rot=64, norm=True, gate=True, out_dtype="bf16", max_pages=80, n_pages=400, max_new="known",
         extra=0, scale=1.0, ovf=False, theta=1e7, spare=2):
    """Runs passes (lists of new tokens per sequence) one after the other and checks each; each pass has spare rows more
    than its tokens need (with many, and of more than 64 rows a sequence and kv head, the form of large passes runs)."""
    n_seq = len(passes[0])
    cache = Kv8Cache(1, nkv, n_pages, n_seq, max_pages)
    model = ref.Cache(n_pages, n_seq, max_pages)
    cache.k[0].fill_(0x7f)      # what no token has been written to is NaN
    cache.v[0].fill_(0xff)
    att = TextAttention(nh, nkv, HD, n_rot, rope_theta=theta)
    for i, new in enumerate(passes):
        T = sum(max(n, 0) for n in new) + spare
        _say(f"heads {nh}/{nkv} pass {i} new {new} T {T}")
        plan = Kv8Plan(cache, T, nh, max(new) if max_new == "known" else max_new)
        before = model.len.copy()
        status, cu, slots, pos3 = model.plan(new, T)
        assert status == 0
        plan.update(_int(new))
        qkv, qn, kn = _qkv(T, nh, nkv, seed + 13 * i, extra, scale)
        if not norm:
            qn = kn = None
        out = torch.full((T, nh * HD), 7.0, dtype={"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[out_dtype], device="cuda")
        att.forward_kv8(qkv, qn, kn, plan.pos3, plan, cache, 0, out=out, out_dtype=out_dtype, gate=gate)
        torch.cuda.synchronize()
        assert plan.status() == 0
        assert np.array_equal(_np(plan.cu_q), cu) and np.array_equal(_np(plan.slots), slots) and np.array_equal(_np(plan.pos3), pos3)
        assert np.array_equal(_np(cache.state), model.state()) and np.array_equal(_np(cache.tables), model.tables)
        assert np.array_equal(_np(cache.free)[:model.n_free], model.free[:model.n_free])
        q, k, v, g = ref.rows(_np(qkv.float()), nh, nkv, n_rot, None if qn is None else _np(qn), None if kn is None else _np(kn), pos3, theta)
        values = _cache_values(cache)
        for r, n in enumerate(new):   # the new tokens' codes: half a step of their page's scale (and f32 arithmetic before them: 2^-12
            # of it, and 2^-19 of the row for the rotation)
            if n <= 0:
                continue
            L = before[r]
            kk, vv = _sequence(cache, values, model, r, L + n)
            page = model.tables[r, np.arange(L, L + n) // PAGE]
            for got, x, s in ((kk[:, L:], k[cu[r]:cu[r + 1]], values[2][page]), (vv[:, L:], v[cu[r]:cu[r + 1]], values[3][page])):
                x = x.transpose(1, 0, 2)
                room = np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s.T[..., None]) * (1 + 2.0 ** -12) + 2.0 ** -19 * np.abs(x).max(-1, keepdims=True)
                assert (np.abs(got - x) <= room).all(), f"codes of sequence {r}"
        _check_attention(out, before, new, cu, q, g, cache, model, values, HD ** -0.5, gate, out_dtype)
        assert (out[T - spare:] == 7.0).all(), "rows behind the last sequence changed"
    return cache, model


@pytest.mark.parametrize("nh,nkv", [(24, 4), (16, 4), (8, 8), (16, 1), (5, 1), (40, 2)])
def test_tokens_and_prompts(nh, nkv):
    """Prompts, then single tokens, then a mix with resting and ended sequences and new ones on their pages."""
    _run(nh, nkv, [[70, 1, 128, 63, 0], [1, 1, 1, 1, 1], [1, 64, 0, 2, -1], [0, 5, 1, 66, 90]], seed=nh)


@pytest.mark.parametrize("nh,nkv", [(24, 4), (16, 4), (8, 8), (16, 1), (5, 1), (40, 2)])
def test_tokens_and_prompts_large(nh, nkv):
    """The same in passes that have the rows of large ones."""
    _run(nh, nkv, [[70, 1, 128, 63, 0], [1, 1, 1, 1, 1], [1, 64, 0, 2, -1], [0, 5, 1, 66, 90]], seed=nh, max_new=None, spare=8192 // nh + 1)


@pytest.mark.parametrize("room", [2, 342])
@pytest.mark.parametrize("max_new", [None, 1, 3, 200])
def test_max_new_is_a_hint(max_new, room):
    _run(24, 4, [[40, 3, 100], [1, 2, 3], [5, 1, 130]], max_new=max_new, seed=3, spare=room)


@pytest.mark.parametrize("max_new,room", [("known", 2), (None, 513)])
@pytest.mark.parametrize("lens", [[1], [63], [64], [65], [300], [1, 2, 3, 4, 5, 6, 7, 8]])
def test_lengths(lens, max_new, room):
    _run(16, 4, [lens, [1] * len(lens)], seed=len(lens) + lens[0], max_new=max_new, spare=room)


@pytest.mark.parametrize("max_new,room", [("known", 2), (None, 1025)])
def test_long_sequence_is_cut(max_new, room):
    """One sequence whose pages are split over many workgroups and joined."""
    _run(8, 2, [[1300], [1], [2], [5]], seed=11, max_new=max_new, spare=room)


@pytest.mark.parametrize("max_new,room", [("known", 2), (None, 1025)])
@pytest.mark.parametrize("out_dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n_rot,norm,gate", [(64, True, True), (0, False, False), (64, False, True)])
def test_variants(out_dtype, n_rot, norm, gate, max_new, room):
    _run(8, 4, [[33, 100], [1, 1]], n_rot=n_rot, norm=norm, gate=gate, out_dtype=out_dtype, seed=5, max_new=max_new, spare=room)


@pytest.mark.parametrize("max_new,room", [("known", 2), (None, 1025)])
def test_sharp_rows_and_row_stride(max_new, room):
    """Keys that dominate their rows (large queries and keys, no norm), and rows wider than needed."""
    _run(8, 4, [[90], [1], [7]], n_rot=0, norm=False, scale=4.0, extra=24, seed=8, max_new=max_new, spare=room)


@pytest.mark.parametrize("n_seq,new,group", [(70, 1, 2), (70, 3, 8), (40, 40, 4), (6, 1, 1)])
def test_items_of_many_pages(n_seq, new, group):
    """Sequences that share 300 pages (read only) and end in a page of their own: items run over hundreds of pages (with
    many sequences) or are cut (with few), in each of the attention's forms."""
    nkv, shared = 8, 300
    nh = nkv * group
    _say("shared pages", n_seq, new, group)
    cache, model = Kv8Cache(1, nkv, shared + n_seq, n_seq, shared + 1), ref.Cache(shared + n_seq, n_seq, shared + 1)
    g = torch.Generator(device="cuda").manual_seed(n_seq)
    for codes, scale in ((cache.k[0], cache.k_scale[0]), (cache.v[0], cache.v_scale[0])):
        codes.copy_(torch.randint(0, 120, codes.shape, generator=g, dtype=torch.uint8, device="cuda")
                    | torch.randint(0, 2, codes.shape, generator=g, dtype=torch.uint8, device="cuda") << 7)
        codes[shared:] = 0x7f
        # scales of 2^-12 to 2^-4: units of the outputs change within a sequence
        scale.copy_(2.0 ** torch.randint(-12, -3, scale.shape, generator=g, device="cuda"))
    model.tables[:, :shared], model.len[:], model.held[:] = np.arange(shared), shared * PAGE, shared
    model.n_free, model.free[:n_seq] = n_seq, shared + np.arange(n_seq)
    cache.tables.copy_(_int(model.tables))
    cache.free.copy_(_int(model.free))
    cache.state.copy_(_int(model.state()))
    T = n_seq * new
    plan = Kv8Plan(cache, T, nh, new)
    plan.update(_int([new] * n_seq))
    status, cu, _, pos3 = model.plan([new] * n_seq, T)
    qkv, qn, kn = _qkv(T, nh, nkv, 3)
    out = TextAttention(nh, nkv).forward_kv8(qkv, qn, kn, plan.pos3, plan, cache, 0)
    torch.cuda.synchronize()
    assert status == plan.status() == 0
    some = [0, n_seq // 2, n_seq - 1]
    q, _, _, gate = ref.rows(_np(qkv.float()), nh, nkv, 64, _np(qn), _np(kn), pos3)
    values = _cache_values(cache)
    for r in some:
        kk, vv = _sequence(cache, values, model, r, shared * PAGE + new)
        tokens = [0, new - 1] if new > 3 else list(range(new))
        for t in sorted(set(tokens)):
            rows = slice(cu[r] + t, cu[r] + t + 1)
            want, off = ref.attend(q[rows], gate[rows], kk, vv, shared * PAGE + t, HD ** -0.5, True)
            off = off + HALF_STEP["bf16"] * (np.abs(want) + off)
            d = np.abs(_np(out[rows].float()).reshape(want.shape) - want)
            assert (d <= off).all(), (r, t, float((d / off).max()))


@pytest.mark.parametrize("new,rows", [([1], 1), ([40], 40), ([40], 4097)])
@pytest.mark.parametrize("where", ["first", "last"])
def test_many_small_weights(new, rows, where):
    """One key outweighs each other one by 2^23, and together they make 0.4% of the output: weights far below the
    largest still count, whether the largest comes before or behind them."""
    nh, nkv, n = 2, 1, 32768
    _say("small weights", new, rows, where)
    cache, model = Kv8Cache(1, nkv, 520, 1, 520), ref.Cache(520, 1, 520)
    att = TextAttention(nh, nkv, HD, 0)
    plan = Kv8Plan(cache, n, nh)
    plan.update(_int([n]))
    model.plan([n], n)
    qkv = torch.zeros(n, att.row, dtype=torch.bfloat16, device="cuda")
    qkv[:, 2 * nh * HD + HD:] = 1.0                                   # every value 1
    at = 5 if where == "first" else n - 3
    qkv[at, 2 * nh * HD] = 16.0                                       # one key of length 16, its value 0
    qkv[at, 2 * nh * HD + HD:] = 0
    att.forward_kv8(qkv, None, None, None, plan, cache, 0, stage="append")
    T = new[0]
    plan = Kv8Plan(cache, rows, nh, T)
    plan.update(_int(new))
    model.plan(new, rows)
    q = torch.zeros(rows, att.row, dtype=torch.bfloat16, device="cuda")
    q[:, 0] = q[:, 2 * HD] = 16.0                                     # scores 16 = 23.08 in log2, and 0
    out = att.forward_kv8(q, None, None, None, plan, cache, 0, gate=False)[:T]
    torch.cuda.synchronize()
    rest = np.arange(T)[:, None] + n - 1                              # other keys of value 1 (the new ones' values are 0)
    w = np.exp(-16.0)
    want = (n - 1) * w / (1 + rest * w + w)
    # each weight w is off by at most 2^-11 of itself (f16), the output by 2^-8
    assert (np.abs(_np(out.float()) - want) <= want * (2.0 ** -11 + 2.0 ** -8 + 2.0 ** -16)).all()


@pytest.mark.parametrize("magnitude", [2.0 ** -90, 2.0 ** -40, 1.0, 2.0 ** 9])
def test_codes_exact(magnitude):
    """Without norm and rotary the codes and scales are those of the definition bit for bit, also of pages that fill
    in pieces: the scale grows with each and the older codes are rounded again."""
    nh = nkv = 2
    _say("codes at", magnitude)
    cache, model = Kv8Cache(1, nkv, 8, 1, 8), ref.Cache(8, 1, 8)
    att = TextAttention(nh, nkv, HD, 0)
    held = {"k": {}, "v": {}}      # page -> (values, scale) by the definition
    for i, n in enumerate([3, 1, 10, 1, 60, 2]):
        plan = Kv8Plan(cache, n, nh)
        plan.update(_int([n]))
        L = model.len[0]
        model.plan([n], n)
        qkv, _, _ = _qkv(n, nh, nkv, 100 + i, scale=magnitude * 1.7 ** i)
        att.forward_kv8(qkv, None, None, None, plan, cache, 0, stage="append")
        torch.cuda.synchronize()
        x = _np(qkv.float())[:, 2 * nh * HD:].reshape(n, 2, nkv, HD)
        for which, name in ((0, "k"), (1, "v")):
            for t in range(n):
                page, at = int(model.tables[0, (L + t) // PAGE]), (L + t) % PAGE
                if at == 0 or page not in held[name]:
                    held[name][page] = (np.zeros((nkv, PAGE, HD)), np.zeros(nkv), 0)
            for page, (val, s, m) in list(held[name].items()):
                mine = [t for t in range(n) if model.tables[0, (L + t) // PAGE] == page]
                if not mine:
                    continue
                new = np.maximum(ref.page_scale(np.abs(x[mine, which]).max((0, 2))), s)
                val = ref.round_e4m3(val / new[:, None, None]) * new[:, None, None]
                for t in mine:
                    val[:, (L + t) % PAGE] = ref.round_e4m3(x[t, which] / new[:, None]) * new[:, None]
                held[name][page] = (val, new, max(m, (L + mine[-1]) % PAGE + 1))
    k, v, ks, vs = _cache_values(cache)
    for name, got, scale in (("k", k, ks), ("v", v, vs)):
        for page, (val, s, m) in held[name].items():
            assert np.array_equal(scale[page], s), (name, page)
            assert np.array_equal((got[page] * scale[page][:, None, None])[:, :m], val[:, :m]), (name, page)


@pytest.mark.parametrize("last,room", [(1, 0), (30, 0), (30, 2049)])
def test_pages_of_very_different_magnitude(last, room):
    """Pages whose keys and values differ by up to 2^75 in one sequence, in both orders: the outputs' units move with them."""
    nh, nkv, mags = 4, 2, [2.0 ** 13, 2.0 ** -60, 1.0, 2.0 ** -20, 2.0 ** 12, 2.0 ** -62, 2.0 ** -3]
    for order in (mags, mags[::-1]):
        _say("magnitudes", order[0], last)
        cache, model = Kv8Cache(1, nkv, 10, 1, 10), ref.Cache(10, 1, 10)
        cache.k[0].fill_(0x7f)
        cache.v[0].fill_(0xff)
        att = TextAttention(nh, nkv, HD, 0)
        for i, n in enumerate([PAGE] * len(order) + [last]):
            before = model.len.copy()
            plan = Kv8Plan(cache, n + room, nh, None if room else n)
            plan.update(_int([n]))
            _, cu, _, _ = model.plan([n], n + room)
            qkv, _, _ = _qkv(n + room, nh, nkv, 60 + i)
            if i < len(order):
                x = qkv.float()
                x[:, 2 * nh * HD:] *= order[i]
                qkv = x.to(torch.bfloat16)
            out = att.forward_kv8(qkv, None, None, None, plan, cache, 0)
            torch.cuda.synchronize()
            q, _, _, g = ref.rows(_np(qkv[:n].float()), nh, nkv, 0, None, None, None)
            _check_attention(out[:n], before, [n], cu, q, g, cache, model, _cache_values(cache), HD ** -0.5, True)


def test_other_pages_and_rows_untouched():
    """An append writes its tokens' codes and its pages' scales, nothing else of the pools."""
    nh, nkv = 4, 2
    cache, model = Kv8Cache(1, nkv, 12, 2, 6), ref.Cache(12, 2, 6)
    for t in (cache.k[0], cache.v[0]):
        t.copy_(torch.randint(0, 120, t.shape, dtype=torch.uint8, device="cuda"))
    before = [t.clone() for t in (cache.k[0], cache.v[0])]
    plan = Kv8Plan(cache, 80, nh)
    plan.update(_int([10, 70]))
    model.plan([10, 70], 80)
    qkv, qn, kn = _qkv(80, nh, nkv, 1)
    TextAttention(nh, nkv).forward_kv8(qkv, qn, kn, plan.pos3, plan, cache, 0, stage="append")
    torch.cuda.synchronize()
    mine = np.zeros((12, PAGE), bool)
    for r, n in enumerate([10, 70]):
        for t in range(n):
            mine[model.tables[r, t // PAGE], t % PAGE] = True
    same_k = (before[0] == cache.k[0]).cpu().numpy().transpose(0, 3, 1, 2, 4).reshape(12, PAGE, -1)
    same_v = (before[1] == cache.v[0]).cpu().numpy().transpose(0, 3, 1, 2).reshape(12, PAGE, -1)
    for same in (same_k, same_v):
        assert same[~mine].all() and not same[mine].all()


@pytest.mark.parametrize("rows", [90, 1025])
def test_bad_values_saturate_and_flag(rows):
    """Infinities, NaN and values beyond the limit in queries, keys and values: finite outputs and one flag at the
    sequence's first row; other sequences' rows keep their results bit for bit."""
    nh, nkv, lens = 8, 2, [20, 30, 40]
    res = []
    for bad in (False, True):
        _say("bad values", bad, rows)
        cache = Kv8Cache(1, nkv, 8, 3, 4)
        plan = Kv8Plan(cache, rows, nh)
        plan.update(_int(lens))
        qkv, _, _ = _qkv(rows, nh, nkv, 4)
        if bad:
            qkv[25, 3] = float("nan")                          # a query of sequence 1
            qkv[30, 2 * nh * HD + 5] = float("inf")            # a key of it
            qkv[31, (2 * nh + nkv) * HD + 9] = -float("inf")   # a value of it
        ovf = torch.zeros(rows, dtype=torch.int32, device="cuda")
        out = TextAttention(nh, nkv, HD, 0).forward_kv8(qkv, None, None, None, plan, cache, 0, ovf=ovf)
        torch.cuda.synchronize()
        flags = np.zeros(rows, np.int32)
        flags[20] = bad
        assert np.array_equal(_np(ovf), flags)
        assert torch.isfinite(out[:90].float()).all()
        res.append(out)
    others = [i for i in range(90) if not 20 <= i < 50]
    assert torch.equal(res[0][others].view(torch.int16), res[1][others].view(torch.int16))


def test_f16_output_saturates():
    nh = nkv = 1
    cache = Kv8Cache(1, 1, 4, 1, 2)
    plan = Kv8Plan(cache, 3, 1)
    plan.update(_int([3]))
    qkv = torch.zeros(3, 4 * HD, dtype=torch.bfloat16, device="cuda")
    qkv[:, 3 * HD:] = 60000.0
    ovf = torch.zeros(3, dtype=torch.int32, device="cuda")
    out = TextAttention(1, 1, HD, 0).forward_kv8(qkv, None, None, None, plan, cache, 0, out_dtype="f16", gate=False, ovf=ovf, f16_lim=50000.0)
    torch.cuda.synchronize()
    assert (out == 65504).all() and _np(ovf).tolist() == [1, 0, 0]


# ---- the plan

def test_plan_over_many_sequences():
    rng = np.random.default_rng(0)
    n, cap, n_pages = 2500, 9, 9000
    cache, model = Kv8Cache(1, 1, n_pages, n, cap), ref.Cache(n_pages, n, cap)
    off = rng.integers(-9, 9, n)
    for i in range(4):
        new = rng.choice([0, 1, 1, 1, 3, 70, -1], n)
        new = np.where(model.len + new > cap * PAGE, 0, new)
        T = int(np.maximum(new, 0).sum())
        _say(f"plan {i}: {T} tokens over {n} sequences")
        plan = Kv8Plan(cache, T, 2)
        plan.update(_int(new), pos_off=_int(off))
        status, cu, slots, pos3 = model.plan(new, T, off)
        assert status == plan.status() == 0
        assert np.array_equal(_np(plan.cu_q), cu) and np.array_equal(_np(plan.slots), slots) and np.array_equal(_np(plan.pos3), pos3)
        assert np.array_equal(_np(cache.state), model.state()) and np.array_equal(_np(cache.tables), model.tables)
        assert np.array_equal(_np(cache.free)[:model.n_free], model.free[:model.n_free])


@pytest.mark.parametrize("new,T,status", [([5, 129, 1], 200, 4), ([64, 64, 64], 191, 2), ([64, 64, 64], 192, 1), ([300, 0, 0], 100, 2),
                                          ([1, -1, 2 ** 31 - 1], 10, 2), ([1400, 200, 0], 1500, 2)])
def test_plan_refuses_whole(new, T, status):
    """A pass that does not fit changes nothing, and append and attention with its plan write nothing."""
    _say("refused plan", new, T)
    nh, nkv = 4, 2
    cache = Kv8Cache(1, nkv, 5, 3, 2)
    plan = Kv8Plan(cache, T, nh)
    plan.update(_int([64, 10, 64][:3]) if T >= 138 else _int([1, 1, 1]))
    plan.check()
    kept = [t.clone() for t in (cache.tables, cache.free, cache.state, cache.k[0], cache.v[0], cache.k_scale[0])]
    plan.update(_int(new))
    torch.cuda.synchronize()
    assert plan.status() & status
    with pytest.raises(RuntimeError, match="could not be planned"):
        plan.check()
    qkv, qn, kn = _qkv(T, nh, nkv, 2)
    out = torch.full((T, nh * HD), 3.0, dtype=torch.bfloat16, device="cuda")
    TextAttention(nh, nkv).forward_kv8(qkv, qn, kn, plan.pos3, plan, cache, 0, out=out)
    torch.cuda.synchronize()
    assert (out == 3.0).all() and (plan.slots == -1).all() and (plan.cu_q == 0).all()
    cache.state[1] = 0
    for a, b in zip(kept, (cache.tables, cache.free, cache.state, cache.k[0], cache.v[0], cache.k_scale[0])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("what", ["tokens", "pages", "stack", "free page", "table page"])
def test_plan_refuses_bad_state(what):
    _say("bad state", what)
    cache = Kv8Cache(1, 1, 6, 2, 3)
    plan = Kv8Plan(cache, 70, 1)
    plan.update(_int([70, 0]))
    plan.check()
    if what == "tokens":
        cache.state[2] = 129
    elif what == "pages":
        cache.state[3] = 4
    elif what == "stack":
        cache.state[0] = 7
    elif what == "free page":
        cache.free.fill_(6)
    else:
        cache.tables[0, 1] = -5
    before = cache.free.clone()
    plan.update(_int([-1, 70]) if what == "table page" else _int([0, 70]))
    assert plan.status() & 8
    assert torch.equal(before, cache.free)


def test_plan_again_from_the_same_state():
    """With state_out elsewhere the same call gives the same plan again."""
    cache = Kv8Cache(1, 1, 40, 3, 9)
    plan = Kv8Plan(cache, 300, 4)
    plan.update(_int([100, 30, 64]))
    after = torch.empty_like(cache.state)
    got = []
    for _ in range(3):
        plan.update(_int([60, -1, 200]), state_out=after)
        got.append([t.clone() for t in (cache.tables, cache.free, cache.state, after, plan.slots, plan.work)])
    torch.cuda.synchronize()
    for again in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], again))


def test_pass_without_rows():
    """A pass of no rows ends sequences and gives their pages back; a layer's call with it does nothing."""
    nh, nkv = 4, 2
    cache, att = Kv8Cache(1, nkv, 8, 2, 4), TextAttention(nh, nkv)
    plan = Kv8Plan(cache, 200, nh)
    plan.update(_int([150, 50]))
    none = Kv8Plan(cache, 0, nh)
    none.update(_int([-1, 0]))
    none.check()
    assert cache.state.tolist() == [7, 0, 0, 0, 50, 1] and sorted(cache.free[:7].tolist()) == sorted(set(range(8)) - {int(cache.tables[1, 0])})
    out = att.forward_kv8(torch.zeros(0, att.row, dtype=torch.bfloat16, device="cuda"), None, None, none.pos3, none, cache, 0)
    assert out.shape == (0, nh * HD)
    none.update(_int([1, 0]))
    assert none.status() == 2


def test_copies_of_a_cache_are_their_own():
    """A deep copy of a cache and its plan works on its own memory, and leaves the first as it was."""
    import copy
    nh, nkv = 4, 2
    cache, att = Kv8Cache(1, nkv, 8, 1, 4), TextAttention(nh, nkv)
    plan = Kv8Plan(cache, 20, nh)
    rows = _qkv(20, nh, nkv, 5)
    plan.update(_int([20]))
    want = att.forward_kv8(*rows, plan.pos3, plan, cache, 0)
    other, other_plan = copy.deepcopy((cache, plan))
    kept = [t.clone() for t in (cache.state, cache.tables, cache.k[0], cache.v[0])]
    other_plan.update(_int([20]))
    att.forward_kv8(*_qkv(20, nh, nkv, 6), other_plan.pos3, other_plan, other, 0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, (cache.state, cache.tables, cache.k[0], cache.v[0])))
    assert int(other.state[2]) == 40 and int(cache.state[2]) == 20
    assert torch.equal(att.forward_kv8(*rows, plan.pos3, plan, cache, 0, stage="core"), want)


# ---- reading back, and the 16-bit path

@pytest.mark.parametrize("lens", [[1], [64], [130, 7, 0, 64], [5, 300]])
def test_read(lens):
    nh = nkv = 2
    n = len(lens)
    cache, model = Kv8Cache(1, nkv, 20, n, 6), ref.Cache(20, n, 6)
    T = sum(lens)
    plan = Kv8Plan(cache, T, nh)
    plan.update(_int(lens))
    model.plan(lens, T)
    qkv, qn, kn = _qkv(T, nh, nkv, 6)
    TextAttention(nh, nkv).forward_kv8(qkv, qn, kn, plan.pos3, plan, cache, 0, stage="append")
    values = _cache_values(cache)
    for first in (None, [m // 100 for m in lens]):
        _say("read", lens, first)
        skip = [0] * n if first is None else [PAGE * f for f in first]
        room = [-(-(m - s) // 8) * 8 for m, s in zip(lens, skip)]
        room[0] = max(room[0] - 8, 0)      # less than the sequence has: the rest is left out
        cu = np.concatenate([[0], np.cumsum(room)])
        kvT = int(cu[-1]) + 16
        k, v = torch.full((nkv, kvT, HD), 9.0, dtype=torch.float16, device="cuda"), torch.full((nkv, HD, kvT), 9.0, dtype=torch.bfloat16, device="cuda")
        cache.read(0, _int(cu), k, v, first_page=None if first is None else _int(first))
        torch.cuda.synchronize()
        wk, wv = np.full((nkv, kvT, HD), 9.0), np.full((nkv, HD, kvT), 9.0)
        for r in range(n):
            kk, vv = _sequence(cache, values, model, r, lens[r])
            m = min(lens[r] - skip[r], room[r])
            wk[:, cu[r]:cu[r] + m] = kk[:, skip[r]:skip[r] + m]
            wv[:, :, cu[r]:cu[r] + m] = vv[:, skip[r]:skip[r] + m].transpose(0, 2, 1)
        assert np.array_equal(_np(k), wk.astype(np.float16).astype(np.float64)) and np.array_equal(_np(v), wv)


def test_read_of_many_pages():
    """A read large enough for two pages a workgroup: odd lengths, rows that start anywhere at multiples of 8."""
    nkv, lens = 16, [5000, 3, 0, 70, 2049, 64, 1500]
    n, n_pages = len(lens), 150
    cache, model = Kv8Cache(1, nkv, n_pages, n, 80), ref.Cache(n_pages, n, 80)
    g = torch.Generator(device="cuda").manual_seed(1)
    cache.k[0].copy_(torch.randint(0, 127, cache.k[0].shape, generator=g, dtype=torch.uint8, device="cuda"))
    cache.v[0].copy_(torch.randint(0, 127, cache.v[0].shape, generator=g, dtype=torch.uint8, device="cuda"))
    cache.k_scale[0].copy_(2.0 ** torch.randint(-9, 9, (n_pages, nkv), generator=g, device="cuda"))
    cache.v_scale[0].copy_(2.0 ** torch.randint(-9, 9, (n_pages, nkv), generator=g, device="cuda"))
    plan = Kv8Plan(cache, sum(lens), nkv)
    plan.update(_int(lens))
    model.plan(lens, sum(lens))
    cu = np.concatenate([[0], np.cumsum([-(-m // 8) * 8 + 8 for m in lens])])
    kvT = int(cu[-1])
    _say("read", lens, "into", kvT)
    k, v = torch.full((nkv, kvT, HD), 9.0, dtype=torch.float16, device="cuda"), torch.full((nkv, HD, kvT), 9.0, dtype=torch.bfloat16, device="cuda")
    cache.read(0, _int(cu), k, v)
    torch.cuda.synchronize()
    values = _cache_values(cache)
    k, v = _np(k), _np(v)
    for r, m in enumerate(lens):
        kk, vv = _sequence(cache, values, model, r, m)
        assert np.array_equal(k[:, cu[r]:cu[r] + m], np.clip(kk, -65504, 65504)) and np.array_equal(v[:, :, cu[r]:cu[r] + m].transpose(0, 2, 1), vv)
        assert (k[:, cu[r] + m:cu[r + 1]] == 9).all() and (v[:, :, cu[r] + m:cu[r + 1]] == 9).all()


def test_against_the_16_bit_path():
    """Pages read back into the planes of a prefix pass: the text core over them and the paged attention agree to
    twice the bound of one and the 2^-8 of each weight that the core's bf16 weights are off."""
    nh, nkv, L, n = 24, 4, 200, 9
    cache, model = Kv8Cache(1, nkv, 8, 1, 8), ref.Cache(8, 1, 8)
    att = TextAttention(nh, nkv)
    for m in (L, n):
        plan = Kv8Plan(cache, m, nh)
        plan.update(_int([m]))
        model.plan([m], m)
        qkv, qn, kn = _qkv(m, nh, nkv, 40 + m)
        out = att.forward_kv8(qkv, qn, kn, plan.pos3, plan, cache, 0)
    kvT = 256
    k, v = torch.zeros(nkv, kvT, HD, dtype=torch.float16, device="cuda"), torch.zeros(nkv, HD, kvT, dtype=torch.bfloat16, device="cuda")
    cache.read(0, _int([0, 216]), k, v)
    aplan = AttnPlan([0, n], [0, L + n])
    want = att.forward(qkv, qn, kn, plan.pos3, aplan, k_plane=k, vt_plane=v, kvT=kvT, stage="core")
    torch.cuda.synchronize()
    q, _, _, g = ref.rows(_np(qkv.float()), nh, nkv, 64, _np(qn), _np(kn), _np(plan.pos3))
    kk, vv = _sequence(cache, _cache_values(cache), model, 0, L + n)
    mid, off = ref.attend(q, g, kk, vv, L, HD ** -0.5, True)
    core = 2.0 ** -8 * ref.attend(q, g, kk, np.abs(vv), L, HD ** -0.5, True)[0]
    off = off + 2.0 ** -8 * (np.abs(mid) + off + core)
    assert (np.abs(_np(out.float()) - _np(want.float())).reshape(mid.shape) <= 2 * off + core).all()


# ---- as a program runs it

def test_shared_prefix_is_read():
    """Two sequences on one document: the second's table row names the first's full pages; each appends to its own."""
    nh, nkv, doc = 8, 2, 128
    cache = Kv8Cache(1, nkv, 12, 2, 6)
    att = TextAttention(nh, nkv)
    plan = Kv8Plan(cache, doc, nh)
    plan.update(_int([doc, 0]))
    rows = _qkv(doc, nh, nkv, 1)
    att.forward_kv8(*rows, plan.pos3, plan, cache, 0)
    cache.tables[1, :2] = cache.tables[0, :2]
    cache.state[4:6] = cache.state[2:4]
    plan = Kv8Plan(cache, 10, nh)
    plan.update(_int([5, 5]))
    plan.check()
    qkv, _, _ = _qkv(5, nh, nkv, 2)
    qkv = torch.cat([qkv, qkv])
    out = att.forward_kv8(qkv, rows[1], rows[2], plan.pos3, plan, cache, 0)
    torch.cuda.synchronize()
    assert torch.equal(out[:5], out[5:])
    assert cache.tables[0, 2] != cache.tables[1, 2]


def test_truncated_sequence_continues():
    """A sequence cut back to fewer tokens keeps its pages and continues as if the rest had never been."""
    nh, nkv = 8, 2
    outs = []
    for cut in (False, True):
        cache, att = Kv8Cache(1, nkv, 8, 1, 6), TextAttention(nh, nkv)
        plan = Kv8Plan(cache, 150 if cut else 64, nh)
        plan.update(_int([plan.T]))
        rows = _qkv(150, nh, nkv, 3)
        att.forward_kv8(rows[0][:plan.T].contiguous(), rows[1], rows[2], plan.pos3, plan, cache, 0)
        if cut:
            cache.state[2] = 64
        plan = Kv8Plan(cache, 20, nh)
        plan.update(_int([20]))
        out = att.forward_kv8(_qkv(20, nh, nkv, 4)[0], rows[1], rows[2], plan.pos3, plan, cache, 0)
        plan.check()
        assert cache.state[2] == 84 and cache.state[3] == (3 if cut else 2)
        outs.append(out)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])


def test_passes_repeat_bitwise():
    nh, nkv = 24, 4
    cache, att = Kv8Cache(1, nkv, 60, 3, 40), TextAttention(nh, nkv)
    plan = Kv8Plan(cache, 2000, nh)
    plan.update(_int([1500, 300, 200]))
    rows = _qkv(2000, nh, nkv, 9)
    att.forward_kv8(*rows, plan.pos3, plan, cache, 0)
    plan = Kv8Plan(cache, 3, nh, 1)
    plan.update(_int([1, 1, 1]))
    q = _qkv(3, nh, nkv, 10)[0]
    outs = [att.forward_kv8(q, rows[1], rows[2], plan.pos3, plan, cache, 0).clone() for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_captured_loop_matches_eager():
    """A graph of plan and two layers, replayed as a decoding loop with work between the replays, against the
    same passes run one by one."""
    nh, nkv, layers, steps = 16, 4, 2, 6
    outs = {}
    for mode in ("eager", "graph"):
        cache, att = Kv8Cache(layers, nkv, 40, 3, 8), TextAttention(nh, nkv)
        fill = Kv8Plan(cache, 260, nh)
        fill.update(_int([120, 62, 78]))
        rows = _qkv(260, nh, nkv, 20)
        for l in range(layers):
            att.forward_kv8(*rows, fill.pos3, fill, cache, l)
        plan, new = Kv8Plan(cache, 3, nh, 1), _int([1, 1, 1])
        qkv = torch.zeros(3, att.row, dtype=torch.bfloat16, device="cuda")
        out = [torch.zeros(3, nh * HD, dtype=torch.bfloat16, device="cuda") for _ in range(layers)]

        def step():
            plan.update(new)
            for l in range(layers):
                att.forward_kv8(qkv, rows[1], rows[2], plan.pos3, plan, cache, l, out=out[l])

        if mode == "graph":
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        got = []
        for i in range(steps):
            qkv.copy_(_qkv(3, nh, nkv, 30 + i)[0])
            graph.replay() if mode == "graph" else step()
            got += [o.clone() for o in out]
            torch.cuda.synchronize()
        plan.check()
        outs[mode] = got + [cache.state.clone(), cache.tables.clone()]
    assert all(torch.equal(a, b) for a, b in zip(outs["eager"], outs["graph"]))


def test_another_stream():
    nh, nkv = 8, 2
    cache, att = Kv8Cache(1, nkv, 20, 2, 10), TextAttention(nh, nkv)
    s = torch.cuda.Stream()
    rows = _qkv(300, nh, nkv, 50)
    new = _int([200, 100])
    torch.cuda.synchronize()
    plan = Kv8Plan(cache, 300, nh)
    torch.cuda.synchronize()
    plan.update(new, stream=s)
    out = att.forward_kv8(*rows, plan.pos3, plan, cache, 0, stream=s, out=torch.empty(300, nh * HD, dtype=torch.bfloat16, device="cuda"))
    s.synchronize()
    other = Kv8Cache(1, nkv, 20, 2, 10)
    plan2 = Kv8Plan(other, 300, nh)
    plan2.update(new)
    want = att.forward_kv8(*rows, plan2.pos3, plan2, other, 0)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("rows,heads,pages,max_new", [(31, 1, 10, None), (30, 2, 10, None), (30, 1, 11, None), (30, 1, 10, 4)])
def test_plan_of_another_shape_is_not_run(rows, heads, pages, max_new):
    """A plan buffer made for other sizes (rows; kv heads of the same group; table rows; another form's blocks) is left
    alone by the kernels: nothing is written."""
    nh, nkv = 8, 2
    _say("plan of", rows, heads, pages, max_new)
    cache, att = Kv8Cache(1, nkv, 20, 2, 10), TextAttention(nh, nkv)
    plan, wrong = Kv8Plan(cache, 30, nh), Kv8Plan(Kv8Cache(1, nkv * heads, 20, 2, pages), rows, nh * heads, max_new)
    wrong.update(_int([20, 10]))
    plan.work[:16].copy_(wrong.work[:16])
    rows = _qkv(30, nh, nkv, 1)
    out = torch.full((30, nh * HD), 5.0, dtype=torch.bfloat16, device="cuda")
    codes = cache.k[0].clone()
    att.forward_kv8(*rows, wrong.pos3[:30].contiguous(), plan, cache, 0, out=out)
    torch.cuda.synchronize()
    assert (out == 5.0).all() and torch.equal(codes, cache.k[0])


def test_refused_tensors():
    nh, nkv = 8, 2
    cache, att = Kv8Cache(1, nkv, 20, 2, 10), TextAttention(nh, nkv)
    plan = Kv8Plan(cache, 30, nh)
    plan.update(_int([20, 10]))
    qkv, qn, kn = _qkv(30, nh, nkv, 1)
    for args, kw, msg in [((qkv[:29], qn, kn, plan.pos3, plan, cache), {}, "qkv has shape"), ((qkv.float(), qn, kn, plan.pos3, plan, cache), {}, "dtype"),
                          ((qkv, qn, None, plan.pos3, plan, cache), {}, "both"), ((qkv, qn, kn, plan.pos3.long(), plan, cache), {}, "pos3"),
                          ((qkv, qn, kn, plan.pos3, plan, Kv8Cache(1, nkv, 20, 2, 10)), {}, "another cache"),
                          ((qkv, qn, kn, plan.pos3, plan, cache), dict(layer=1), "layer 1"), ((qkv, qn, kn, plan.pos3, plan, cache), dict(stage="prep"), "stage"),
                          ((qkv, qn, kn, plan.pos3, plan, cache), dict(out=torch.empty(30, 9, device="cuda")), "out has")]:
        with pytest.raises((ValueError, TypeError), match=msg):
            att.forward_kv8(*args, **kw)
    with pytest.raises(ValueError, match="heads"):
        TextAttention(4, 2).forward_kv8(qkv, qn, kn, plan.pos3, plan, cache)
