"""The paged cache's operators in float64 on the host, and batches to run them on: what tests/test_gpu_paged.py and
tests/test_paged.py compare with."""
import numpy as np

T_F32, T_F16, T_BF16 = 0, 1, 30
#: half a step of each cache type, relative to the value
HALF_STEP = {T_F32: 2.0**-24, T_F16: 2.0**-11, T_BF16: 2.0**-8}
U32 = 2.0**-24


def to_bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def encode(x, t):
    """fp32 values as the cache's bytes: an array of uint32 or uint16 codes."""
    x = np.ascontiguousarray(x, np.float32)
    return x.view(np.uint32) if t == T_F32 else to_bf16(x) if t == T_BF16 else x.astype(np.float16).view(np.uint16)


def decode(c, t):
    """The codes' values in float64."""
    if t == T_F32:
        return c.view(np.float32).astype(np.float64)
    return c.view(np.float16).astype(np.float64) if t == T_F16 else (c.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Batch:
    """Sequences of `news` new tokens and `lens` positions over a pool of pages handed out in a random order.
    `pad`: rows of no sequence before and behind the batch; `gap`: values between pages; `spare`: unused table columns,
    filled with page numbers that do not exist."""

    def __init__(self, seed, type_, hd, n_head, n_kv, page, news, lens, pad=(0, 0), gap=0, spare=1, sigma=1.0):
        r = self.rng = np.random.default_rng(seed)
        self.type, self.hd, self.n_head, self.n_kv, self.page = type_, hd, n_head, n_kv, page
        self.news, self.lens, self.pad = list(news), list(lens), pad
        self.tok = (pad[0] + np.concatenate([[0], np.cumsum(news)])).astype(np.int32)
        self.len = np.array(lens, np.int32)
        self.n_tok = int(self.tok[-1]) + pad[1]
        per = [-(-m // page) for m in lens]
        self.stride = max(per + [1]) + spare
        self.n_pages = sum(per) + 2
        order = r.permutation(self.n_pages)
        self.table = np.full((len(news), self.stride), 0x7FFFFFF0, np.int32)
        at = 0
        for s, m in enumerate(per):
            self.table[s, :m] = order[at:at + m]
            at += m
        self.page_values = n_kv * page * hd
        self.page_stride = self.page_values + gap
        total = self.n_pages * self.page_stride
        self.k = encode(r.standard_normal(total) * sigma, type_)
        self.v = encode(r.standard_normal(total), type_)
        self.q = r.standard_normal((self.n_tok, n_head, hd)).astype(np.float32)

    def at(self, s, pos, head, is_v):
        """Offsets of the hd values of a position."""
        base = int(self.table[s, pos // self.page]) * self.page_stride + head * self.hd * self.page
        i = np.arange(self.hd)
        return base + (i * self.page + pos % self.page if is_v else pos % self.page * self.hd + i)

    def rows(self, s, head, is_v):
        """[len][hd] values of a sequence's head, float64."""
        buf = self.v if is_v else self.k
        idx = np.array([self.at(s, p, head, is_v) for p in range(self.lens[s])], np.int64).reshape(-1, self.hd)
        return decode(buf[idx], self.type)

    def tokens(self):
        """(row, sequence, position) of every new token."""
        for s, (n, m) in enumerate(zip(self.news, self.lens)):
            for i in range(n):
                yield int(self.tok[s]) + i, s, m - n + i


def store(b, qkv, norm=None, n_rot=0, halves=False, base=10000.0, scale=1.0, factors=None, eps=1e-5):
    """float64 q' [n_tok][n_head][hd], k' and v [n_tok][n_kv][hd], and a bound on the fp32 arithmetic's error of q' and
    k': products, the sum of squares and the root of hd values, two products and a sum of the rotation, and
    its cosines to fp32, 20 roundings of the pair's size."""
    x = qkv.astype(np.float64)
    q, k, v = x[:, :b.n_head].copy(), x[:, b.n_head:b.n_head + b.n_kv].copy(), x[:, b.n_head + b.n_kv:]
    if norm is not None:
        for y, w in ((q, norm[0]), (k, norm[1])):
            if w is not None:
                y /= np.sqrt((y * y).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
                y *= w.astype(np.float64)
    half = n_rot // 2
    eq, ek = np.abs(q), np.abs(k)
    if n_rot:
        f = np.float64(np.float32(base)) ** (-2.0 * np.arange(half) / n_rot) * np.float64(np.float32(scale))
        if factors is not None:
            f = f / factors.astype(np.float64)
        ia = np.arange(half) if halves else 2 * np.arange(half)
        ib = ia + (half if halves else 1)
        for t, _, p in b.tokens():
            c, s = np.cos(p * f), np.sin(p * f)
            for y, e in ((q, eq), (k, ek)):
                u, w = y[t][:, ia].copy(), y[t][:, ib].copy()
                y[t][:, ia], y[t][:, ib] = u * c - w * s, u * s + w * c
                e[t][:, ia] = e[t][:, ib] = np.abs(u) + np.abs(w)
    return q, k, v, 20 * U32 * eq, 20 * U32 * ek


def attention(b, q, scale, softcap=0.0, window=0, slopes=None, prefix=None):
    """float64 outputs [n_tok][n_head][hd] (rows of no sequence: None in `mine`) and a bound on their error in fp32.

    A score is a sum of products rounded in fp32 and of 16-bit parts that hold q to 22 bits: off by at most
    8 u sum |q k| scale (u = 2^-24), the cap (a contraction) and its tanh 4 u softcap, the bias 2 u |bias|, its change to
    powers of two 4 u |s|. With every score off by d, weights are off by a factor of exp(2 d), and their own rounding and
    the sums' are 16 u more: |o - o'| <= (2 d + 16 u) 2 sum w |v|."""
    out = np.zeros((b.n_tok, b.n_head, b.hd))
    tol = np.zeros_like(out)
    mine = np.zeros(b.n_tok, bool)
    g = b.n_head // b.n_kv
    keys = {(s, h): (b.rows(s, h, False), b.rows(s, h, True)) for s in range(len(b.news)) for h in range(b.n_kv) if b.news[s]}
    j = np.arange(max(b.lens + [1]))
    for t, s, p in b.tokens():
        mine[t] = True
        see = j[:b.lens[s]] <= p
        if prefix is not None:
            see = see | (j[:b.lens[s]] < prefix[s])
        if window:
            see = see & (p - j[:b.lens[s]] < window)
        idx = np.nonzero(see)[0]
        for h in range(b.n_head):
            k, v = keys[s, h // g]
            k, v, x = k[idx], v[idx], q[t, h].astype(np.float64)
            z = (k @ x) * scale
            d = 8 * U32 * (np.abs(k) @ np.abs(x)) * abs(scale)
            if softcap:
                z = softcap * np.tanh(z / softcap)
                d = d + 4 * U32 * softcap
            if slopes is not None:
                bias = np.float64(slopes[h]) * np.abs(p - idx)
                z, d = z - bias, d + 2 * U32 * bias
            d = (d + 4 * U32 * np.abs(z)).max()
            w = np.exp(z - z.max())
            w /= w.sum()
            out[t, h] = w @ v
            tol[t, h] = (2 * d + 16 * U32) * 2 * (w @ np.abs(v))
    return out, tol, mine


def of_vectors(o, want):
    """The largest error of a row and head, relative to that vector's length."""
    return float((np.linalg.norm(o - want, axis=-1) / np.linalg.norm(want, axis=-1)).max())


def cut(x, bits):
    """fp32 values without the bits behind the first `bits` of their 24: what is left of a value taken apart, a part short."""
    return (np.ascontiguousarray(x, np.float32).view(np.uint32) & np.uint32(-(1 << 24 - bits) & 0xFFFFFFFF)).view(np.float32)


def plain32(b, q, scale, bits_q=24, bits_w=24):
    """The causal attention of a batch in fp32 throughout (rows of no sequence: 0), q and the weights to so many bits."""
    out = np.zeros((b.n_tok, b.n_head, b.hd), np.float32)
    q, scale = cut(q, bits_q), np.float32(scale)
    for s in range(len(b.news)):
        rows = [(t, p) for t, x, p in b.tokens() if x == s]
        for h in range(b.n_head if rows else 0):
            k, v = (b.rows(s, h * b.n_kv // b.n_head, is_v).astype(np.float32) for is_v in (False, True))
            for t, p in rows:
                z = (k[:p + 1] @ q[t, h]) * scale
                w = cut(np.exp(z - z.max()), bits_w)
                out[t, h] = (w @ v[:p + 1]) / w.sum(dtype=np.float32)
    return out


def vector_bound(b, q, scale, want, mine):
    """What a result may be off by, of a vector's length: 4 times the worst of plain32, which rounds as often in another order, and
    2^-22 for the rounding of q, of the weights and of the result, that do not depend on the sums' order."""
    return 4 * of_vectors(plain32(b, q, scale)[mine], want[mine]) + 2.0**-22
