"""Plans of more blocks than one round of the plan's threads, or than its LDS holds: their work lists entry by entry, and
attention and append over samples of their sequences."""
import numpy as np
import pytest
import torch

from cleffa_amd import Kv8Cache, Kv8Plan, TextAttention
from tests import kv8_ref as ref
from tests.test_gpu_kv8 import HALF_STEP, HD, PAGE, _int, _np, _qkv, _say

pytestmark = pytest.mark.gpu


def _lists(plan):
    """The plan's lists, by the layout that kv8_params.h gives."""
    c, T, nh = plan.cache, plan.T, plan.nh
    n, G = c.max_seqs, nh // c.nkv
    rows = (plan.max_new if 0 < plan.max_new < T else T) * G
    bm = 16 if rows <= 16 else 32 if rows <= 64 or T * nh <= 8192 else 128
    budget = -(-(2 if bm == 16 else 1) * 256 // c.nkv)
    max_app, max_blk = min(T // PAGE + 2 * n, T), T * G // bm + min(n, T)
    app = -(-(16 + n) // 4) * 4
    tok = app + 4 * max_app
    blk = -(-(tok + 2 * T) // 4) * 4
    items = -(-(blk + 4 * max_blk) // 8) * 8
    w = plan.work.cpu().numpy().astype(np.int64)
    assert len(w) == items + 8 * (max_blk + budget)
    n_tok, n_app, n_items, most = w[5:9]
    assert n_items <= max_blk + budget
    return dict(bm=bm, slots=2 * budget, n_tok=n_tok, most=most, app=w[app:app + 4 * n_app].reshape(-1, 4), tok=w[tok:tok + 2 * n_tok].reshape(-1, 2),
                blk=w[blk:blk + 4 * max_blk].reshape(-1, 4), items=w[items:items + 8 * n_items].reshape(-1, 8))


def _check_lists(plan, lens, new, tables, cu):
    """Every new token in one append entry; every block's items its rows over its pages, each page once; split slots
    apart from each other and within the workspace."""
    x, G = _lists(plan), plan.nh // plan.cache.nkv
    bm = x["bm"]
    want = []
    for r, q in enumerate(new):
        L = int(lens[r])
        for pg in range(L // PAGE, -(-(L + q) // PAGE)) if q > 0 else ():
            lo, hi = max(L, pg * PAGE), min(L + q, (pg + 1) * PAGE)
            want.append((tables[r, pg], cu[r] + lo - L, (lo - pg * PAGE) | (hi - lo) << 8, cu[r]))
    assert np.array_equal(x["app"], np.array(want))
    at = b = slot = cut = 0
    for r, q in enumerate(new):
        if q <= 0:
            continue
        assert (x["tok"][cu[r]:cu[r] + q] == np.stack([np.full(q, b), np.arange(q)], 1)).all(), r
        for row0 in range(0, q * G, bm):
            rows, pages = min(bm, q * G - row0), (int(lens[r]) + (row0 + min(bm, q * G - row0) - 1) // G) // PAGE + 1
            first, n, r0, s0 = x["blk"][b]
            assert (first, r0) == (at, row0) and n >= 1, b
            it = x["items"][at:at + n]
            assert (it[:, :5] == (r, cu[r], lens[r], lens[r] + q, row0)).all() and (it[:, 5] & 0xff == rows).all(), b
            assert it[0, 6] == 0 and it[-1, 7] == pages and (it[1:, 6] == it[:-1, 7]).all() and (it[:, 6] < it[:, 7]).all(), b
            assert (it[:, 5] >> 8 == (slot + 1 + np.arange(n) if n > 1 else 0)).all(), b
            if n > 1:
                assert s0 == slot
                slot, cut = slot + n, max(cut, n)
            at, b = at + n, b + 1
    assert at == len(x["items"]) and slot <= x["slots"] and cut == x["most"] and x["n_tok"] == cu[-1]
    return b, slot


def _held(cache, pages, n):
    """K, V [nkv][n][256] in the named pages, and the pages' scales."""
    at = torch.as_tensor(pages.astype(np.int64), device="cuda")
    k, v = ref.page_values(cache.k[0][at].cpu().numpy(), cache.v[0][at].cpu().numpy())
    ks, vs = _np(cache.k_scale[0][at]), _np(cache.v_scale[0][at])
    flat = lambda x, s: (x * s[..., None, None]).transpose(1, 0, 2, 3).reshape(cache.nkv, -1, HD)[:, :n]
    return flat(k, ks), flat(v, vs), ks, vs


def _case(name):
    """Cached pages and new tokens of each sequence, heads, max_new, and the least number of blocks."""
    rng = np.random.default_rng(7)
    if name == "tokens":                 # blocks of more than one round of 1,024 threads
        return rng.integers(0, 12, 1200), np.ones(1200, np.int64), 4, 2, 1, 1100
    if name == "tokens and a long one":  # and some of them cut
        pages, new = rng.integers(0, 4, 1500), rng.choice([0, 1, 1, 1, 2], 1500)
        pages[700], new[700], pages[1499], new[1499] = 3000, 1, 900, 2
        return pages, new, 4, 2, 1, 1100
    if name == "more than LDS holds":    # 8,192 blocks and more
        pages, new = rng.integers(0, 3, 4096), rng.choice([2, 3], 4096)
        pages[4000] = 2500
        return pages, new, 16, 1, 1, 8192
    if name == "questions":              # blocks of 32 rows
        pages, new = rng.integers(0, 5, 1100), rng.integers(1, 12, 1100)
        pages[5] = 1200
        return pages, new, 12, 2, 10, 1500
    pages, new = rng.integers(0, 5, 1030), rng.integers(1, 40, 1030)   # blocks of 128, and pages past one round of appends
    pages[[3, 1029]] = 1500, 700
    return pages, new, 16, 4, None, 1100


@pytest.mark.parametrize("name", ["tokens", "tokens and a long one", "more than LDS holds", "questions", "prompts"])
@pytest.mark.parametrize("ragged", [False, True])
def test_plans_of_many_blocks(name, ragged):
    """Sequences on shared pages (read only, 2^-12 to 2^-4 scales) that end in pages of their own, which (ragged) hold some tokens
    already."""
    pages, new, nh, nkv, max_new, least = _case(name)
    n, shared, T = len(pages), int(pages.max()), int(new.sum()) + 3
    _say("many blocks", name, ragged, n, "sequences", T, "rows")
    rng = np.random.default_rng(n)
    part = rng.integers(1, PAGE, n) if ragged else np.zeros(n, np.int64)
    n_pages, cap = shared + 3 * n, shared + 3
    cache, model = Kv8Cache(1, nkv, n_pages, n, cap), ref.Cache(n_pages, n, cap)
    g = torch.Generator(device="cuda").manual_seed(3)
    for codes, scale in ((cache.k[0], cache.k_scale[0]), (cache.v[0], cache.v_scale[0])):
        for a in range(0, n_pages, 1024):
            c = codes[a:a + 1024]
            c.copy_(torch.randint(0, 120, c.shape, generator=g, dtype=torch.uint8, device="cuda")
                    | torch.randint(0, 2, c.shape, generator=g, dtype=torch.uint8, device="cuda") << 7)
        scale.copy_(2.0 ** torch.randint(-12, -3, scale.shape, generator=g, device="cuda"))
    order = rng.permutation(shared)
    for r in range(n):
        model.tables[r, :pages[r]] = order[:pages[r]]
        if part[r]:
            model.tables[r, pages[r]] = shared + r
    model.held[:] = pages + (part > 0)
    model.len[:] = pages * PAGE + part
    model.n_free = 2 * n
    model.free[:2 * n] = shared + n + rng.permutation(2 * n)
    cache.tables.copy_(_int(model.tables))
    cache.free.copy_(_int(model.free))
    cache.state.copy_(_int(model.state()))
    before = model.len.copy()
    plan = Kv8Plan(cache, T, nh, max_new)
    plan.update(_int(new))
    status, cu, slots, pos3 = model.plan(new.tolist(), T)
    assert status == 0
    plan.check()
    assert np.array_equal(_np(plan.cu_q), cu) and np.array_equal(_np(plan.slots), slots) and np.array_equal(_np(plan.pos3), pos3)
    assert np.array_equal(_np(cache.state), model.state()) and np.array_equal(_np(cache.tables), model.tables)
    blocks, slots = _check_lists(plan, before, new.tolist(), model.tables, cu)
    _say(blocks, "blocks,", slots, "items of cut ones")
    assert blocks >= least
    qkv, qn, kn = _qkv(T, nh, nkv, 3)
    out = torch.full((T, nh * HD), 7.0, dtype=torch.bfloat16, device="cuda")
    TextAttention(nh, nkv).forward_kv8(qkv, qn, kn, plan.pos3, plan, cache, 0, out=out)
    torch.cuda.synchronize()
    assert (out[T - 3:] == 7.0).all()
    assert torch.isfinite(out.float()).all()
    long = np.argsort(-pages)[:2].tolist()
    for r in sorted({0, 1, 2, n // 3, n // 2, n - 2, n - 1, *long, *rng.integers(0, n, 12).tolist()}):
        if new[r] <= 0:
            continue
        L, m, rows = int(before[r]), int(new[r]), slice(int(cu[r]), int(cu[r + 1]))
        q, k, v, gate = ref.rows(_np(qkv[rows].float()), nh, nkv, 64, _np(qn), _np(kn), pos3[rows])
        kk, vv, ks, vs = _held(cache, model.tables[r, :-(-(L + m) // PAGE)], L + m)
        page = np.arange(L, L + m) // PAGE
        for got, x, s in ((kk[:, L:], k, ks[page]), (vv[:, L:], v, vs[page])):
            x = x.transpose(1, 0, 2)
            room = np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s.T[..., None]) * (1 + 2.0 ** -12) + 2.0 ** -19 * np.abs(x).max(-1, keepdims=True)
            assert (np.abs(got - x) <= room).all(), f"codes of sequence {r}"
        got = _np(out[rows].float()).reshape(q.shape)
        for t in range(m) if L < 4000 else sorted({0, m - 1}):
            want, off = ref.attend(q[t:t + 1], gate[t:t + 1], kk, vv, L + t, HD ** -0.5, True)
            off = off + HALF_STEP["bf16"] * (np.abs(want) + off)
            d = np.abs(got[t] - want[0])
            assert (d <= off[0]).all(), (r, t, float((d / off[0]).max()))
