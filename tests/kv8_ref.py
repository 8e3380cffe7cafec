"""The 8-bit paged cache restated in plain numpy (float64, one sequence at a time), for the tests."""
import numpy as np

from cleffa_amd import rope_inv_freq

HD, PAGE = 256, 64


def decode(codes):
    """e4m3 codes (uint8) to float64."""
    c = np.asarray(codes).astype(np.int64)
    e, f = (c >> 3) & 15, c & 7
    x = np.where(e > 0, 2.0 ** (e - 7) * (1 + f / 8), f * 2.0 ** -9)
    x = np.where((c & 127) == 127, np.nan, x)
    return np.where(c >= 128, -x, x)


def round_e4m3(x):
    """The nearest e4m3 value, ties to even, |x| <= 448."""
    _, e = np.frexp(x)
    step = 2.0 ** (np.maximum(e - 1, -6) - 3)
    return np.rint(x / step) * step


def page_scale(most):
    """2^e, e the least integer from -64 on with most <= 448 * 2^e."""
    m, e = np.frexp(np.asarray(most, dtype=np.float64))
    e = np.where(m <= 0.875, e - 9, e - 8)
    return 2.0 ** np.maximum(np.where(np.asarray(most) > 0, e, -64), -64)


def page_values(k, v):
    """[..., nkv][64][256] code values of K pages [..., nkv, 4, 64, 64] and V pages [..., nkv, 256, 64]."""
    k, v = decode(k), decode(v)
    return np.moveaxis(k, -3, -2).reshape(*k.shape[:-3], PAGE, HD), np.swapaxes(v, -1, -2)


def saturated(x, lim=65504.0):
    """Elements beyond lim or NaN become +-65504; and whether any did."""
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(x) <= lim)
    return np.where(bad, np.copysign(65504.0, x), x), bad


def rows(qkv, nh, nkv, n_rot, q_norm, k_norm, pos3, theta=1e7, eps=1e-6):
    """float64 Q [T][nh][256], K, V [T][nkv][256] and gates of bf16 rows given as float64."""
    T = len(qkv)
    qg = qkv[:, :2 * nh * HD].reshape(T, nh, 2, HD)
    q, gate = qg[:, :, 0], qg[:, :, 1]
    k = qkv[:, 2 * nh * HD:(2 * nh + nkv) * HD].reshape(T, nkv, HD)
    v = qkv[:, (2 * nh + nkv) * HD:(2 * nh + 2 * nkv) * HD].reshape(T, nkv, HD)
    if q_norm is not None:
        q, k = (x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * w for x, w in ((q, q_norm), (k, k_norm)))
    if n_rot:   # the angle is an FP32 product
        inv = rope_inv_freq(theta, n_rot)
        ang = (pos3[:, np.arange(32) % 3].astype(np.float32) * inv).astype(np.float64)[:, None]
        turn = lambda x: np.concatenate([x[..., :32] * np.cos(ang) - x[..., 32:64] * np.sin(ang),
                                         x[..., 32:64] * np.cos(ang) + x[..., :32] * np.sin(ang), x[..., 64:]], -1)
        q, k = turn(q), turn(k)
    return q, k, v, gate


def attend(q, gate, k, v, first, scale, use_gate):
    """Causal attention of queries at tokens first, first + 1, ... ([n][nh][256]) over keys [nkv][N][256]: the outputs
    [n][nh][256], and how far f16 queries and f16 weights may move each: a query element is off by at most half
    a step, 2^-11 of itself (2^-18 more for the f32 norm, rotary and sums), which moves a score by at most
    that share of sum |q k| * scale = d and a weight by exp(2 d); a weight's own rounding is 2^-11 of it, or 2^-28 of
    the row's largest where that is more (half of f16's smallest step, of weights held times 2^3 at least). The output's rounding comes on top."""
    n, nh = q.shape[:2]
    group = nh // k.shape[0]
    out, off = np.zeros_like(q), np.zeros_like(q)
    for h in range(nh):
        kk, vv = k[h // group], v[h // group]
        for i in range(n):
            m = first + i + 1
            s = kk[:m] @ q[i, h] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ vv[:m]
            d = (np.abs(kk[:m]) @ np.abs(q[i, h])).max() * scale * (2.0 ** -11 + 2.0 ** -18)
            off[i, h] = (w @ np.abs(vv[:m])) * (np.expm1(2 * d) + 2.0 ** -11 * np.exp(2 * d) + 2.0 ** -16) \
                + 2.0 ** -28 * w.max() * np.abs(vv[:m]).sum(0)
    if use_gate:
        g = 1 / (1 + np.exp(-gate))
        out, off = out * g, off * g + np.abs(out * g) * 2.0 ** -20
    return out, off


class Cache:
    """Host model of the page bookkeeping: what Kv8Plan.update does."""

    def __init__(self, n_pages, max_seqs, max_pages):
        self.free, self.n_free = np.arange(n_pages - 1, -1, -1, dtype=np.int32), n_pages
        self.tables = np.full((max_seqs, max_pages), -1, dtype=np.int32)
        self.len, self.held = np.zeros(max_seqs, np.int64), np.zeros(max_seqs, np.int64)

    def plan(self, new, T, pos_off=None):
        """Returns (status, cu_q, slots, pos3); changes the bookkeeping where status is 0."""
        n, cap = len(self.len), self.tables.shape[1]
        status, need = 0, np.zeros(n, np.int64)
        for r, q in enumerate(new):
            if q > T:
                status |= 2
            elif q > 0:
                need[r] = -(-(self.len[r] + q) // PAGE)
                status |= 4 if need[r] > cap else 0
        q = np.where((np.array(new) > 0) & (np.array(new) <= T), new, 0)
        status |= 2 if q.sum() > T else 0
        gone = [r for r in range(n) if new[r] < 0]
        if np.maximum(need - self.held, 0).sum() > self.n_free + sum(self.held[r] for r in gone):
            status |= 1
        slots, pos3 = np.full(T, -1, np.int32), np.zeros((T, 3), np.int32)
        if status:
            return status, np.zeros(n + 1, np.int32), slots, pos3
        for r in gone:
            for p in self.tables[r, :self.held[r]]:
                self.free[self.n_free] = p
                self.n_free += 1
            self.len[r] = self.held[r] = 0
        at = 0
        for r in range(n):
            while self.held[r] < need[r]:
                self.n_free -= 1
                self.tables[r, self.held[r]] = self.free[self.n_free]
                self.held[r] += 1
            for i in range(q[r]):
                t = self.len[r] + i
                slots[at] = self.tables[r, t // PAGE] * PAGE + t % PAGE
                pos3[at] = t + (0 if pos_off is None else pos_off[r])
                at += 1
            self.len[r] += q[r]
        return 0, np.concatenate([[0], np.cumsum(q)]).astype(np.int32), slots, pos3

    def state(self, status=0):
        return np.concatenate([[self.n_free, status], np.stack([self.len, self.held], 1).ravel()]).astype(np.int32)
