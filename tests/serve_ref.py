"""The calls around the paged cache on the host, in 64 bits: what tests/test_serve.py and tests/test_gpu_serve.py compare with."""
import numpy as np
from paged_ref import T_BF16, T_F16, T_F32, U32, decode, encode


class Pool:
    """Sequences, their pages and the ring of free ones, as the call's inputs and outputs hold them."""

    def __init__(self, seed, n_seq, page, lens, n_free, stride, extra=3, first=None):
        r = np.random.default_rng(seed)
        self.page, self.stride = page, stride
        self.held = np.array([-(-m // page) for m in lens], np.int32)
        used = int(self.held.sum())
        self.n_pages = used + n_free + extra
        order = r.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((n_seq, stride), -7, np.int32)
        at = 0
        for s, h in enumerate(self.held):
            self.table[s, :h] = order[at:at + h]
            at += h
        self.first = int(r.integers(self.n_pages)) if first is None else first
        self.free = np.array([self.first, n_free], np.int32)
        self.queue = np.full(self.n_pages, -9, np.int32)
        self.queue[(self.first + np.arange(n_free)) % self.n_pages] = order[used:used + n_free]
        self.len = np.array(lens, np.int32)

    def pages(self):
        """Every page that some sequence holds or the ring has, in no order."""
        held = [self.table[s, :h] for s, h in enumerate(self.held)]
        return np.concatenate(held + [self.queue[(int(self.free[0]) + np.arange(int(self.free[1]))) % self.n_pages]])


def reserve(p, keep, add, n_tok, max_tok, max_len):
    """The call, one sequence after the other; p's table, held, queue and free become what they are after it. Returns tok,
    len, and the rows' seq, pos and slot."""
    n, P = len(keep), p.page
    cap = min(max_len, p.stride * P)
    max_tok = min(max_tok, n_tok)
    first, count = int(p.free[0]), int(p.free[1])
    if not (0 <= first < p.n_pages and 0 <= count <= p.n_pages):
        first = count = 0
    ring = [int(p.queue[(first + i) % p.n_pages]) for i in range(count)]
    keep, add, held = [int(v) for v in keep], [int(v) for v in add], [int(v) for v in p.held]
    fine = [0 <= k <= h * P and 0 <= h <= p.stride for k, h in zip(keep, held)]
    asks = [f and 0 <= a <= max_tok and k + a <= cap for f, k, a in zip(fine, keep, add)]
    want = [-(-(k + a) // P) if q else -(-k // P) if f else h for k, a, h, f, q in zip(keep, add, held, fine, asks)]
    given = [int(p.table[s, i]) for s in range(n) if fine[s] for i in range(want[s], held[s])]
    for i, page in enumerate(given):
        if count + i < p.n_pages:
            p.queue[(first + count + i) % p.n_pages] = page
    ring += given
    took = asked_pages = asked_rows = 0
    tok, length = [0], []
    for s in range(n):
        more = max(0, want[s] - held[s])
        asked_pages += more
        asked_rows += add[s] if asks[s] else 0
        ok = asks[s] and (more == 0 or asked_pages <= len(ring)) and (add[s] == 0 or asked_rows <= n_tok)
        if ok:
            for i in range(held[s], want[s]):
                p.table[s, i] = ring[took]
                took += 1
        tok.append(tok[-1] + (add[s] if ok else 0))
        length.append(keep[s] + (add[s] if ok else 0) if fine[s] else 0)
        if fine[s]:
            p.held[s] = want[s] if ok or want[s] < held[s] else held[s]
    p.free[:] = (first + took) % p.n_pages, min(p.n_pages, len(ring) - took)
    seq, pos, slot = np.full(n_tok, -1, np.int32), np.full(n_tok, -1, np.int32), np.full(n_tok, -1, np.int64)
    for s in range(n):
        for r in range(tok[s], tok[s + 1]):
            seq[r], pos[r] = s, keep[s] + r - tok[s]
            page = int(p.table[s, pos[r] // P])
            if 0 <= page < p.n_pages:
                slot[r] = page * P + pos[r] % P
    return np.array(tok, np.int32), np.array(length, np.int32), seq, pos, slot


def lse_of(x, temp):
    """log sum exp(x / temp), NaN and infinities as the formula has them."""
    if np.isnan(x).any() or np.isnan(temp) or temp < 0:
        return np.nan
    x = x[x != -np.inf].astype(np.float64) / (np.float64(temp) if temp else 1.0)
    if not x.size:
        return -np.inf
    m = x.max()
    return float(m + np.log(np.exp(x - m).sum())) if np.isfinite(m) else float(m)


def weights(x, temp):
    """Probabilities of a row with a finite largest logit."""
    with np.errstate(invalid="ignore"):
        w = np.where(x == -np.inf, 0.0, np.exp((x - x.max()) / temp))
    return w / w.sum()


def verify(logits, tok, tokens, u, v, vocab, max_tok, temp=None, q=None, q_lse=None, length=None):
    """n_ok, next, keep, and lse of the rows that are in a sequence (NaN elsewhere)."""
    n, n_tok = len(tok) - 1, len(logits)
    n_ok, nxt, keep = np.zeros(n, np.int32), np.full(n, -1, np.int32), None if length is None else np.array(length, np.int32)
    lse = np.full(n_tok, np.nan)
    for s in range(n):
        b, e = int(tok[s]), int(tok[s + 1])
        if b < 0 or e > n_tok or e <= b or e - b > min(max_tok, n_tok):
            continue
        t = 1.0 if temp is None else float(np.float32(temp[s]))
        stop = None
        for i in range(b, e):
            x = logits[i, :vocab].astype(np.float64)
            lse[i] = lse_of(logits[i, :vocab], t)
            if stop is not None:
                continue
            broken = np.isnan(lse[i]) or not np.isfinite(x.max())
            last, d = i == e - 1, -1 if i == e - 1 else int(tokens[i + 1])
            word = 0 <= d < vocab
            if not last and word and not broken:
                if t == 0:
                    good = d == int(np.argmax(x))
                else:
                    with np.errstate(invalid="ignore", over="ignore"):
                        chance = 1.0 if q is None else np.exp(np.float64(q[i, d]) / t - np.float64(q_lse[i]))
                    good = np.float64(u[i]) * chance < weights(x, t)[d]
                if good:
                    n_ok[s] += 1
                    continue
            stop = i
            if broken:
                continue
            if t == 0:
                nxt[s] = int(np.argmax(x))
                continue
            w = weights(x, t)
            left = w
            if not last and word:
                if q is None:
                    left = w.copy()
                    left[d] = 0.0
                else:
                    with np.errstate(invalid="ignore", over="ignore"):
                        taken = np.exp(q[i, :vocab].astype(np.float64) / t - np.float64(q_lse[i]))
                        left = np.maximum(w - np.where(np.isnan(taken), 0.0, taken), 0.0)
                if not left.sum() > 0:
                    left = w
            c = np.cumsum(left)
            past = np.nonzero(c > np.float64(v[s]) * c[-1])[0]
            nxt[s] = past[0] if len(past) else np.nonzero(left > 0)[0][-1]
        if keep is not None:
            keep[s] = max(0, int(length[s]) - (e - b - 1 - n_ok[s]))
    return n_ok, nxt, keep, lse


#: bf16 products of parts that make one of fp32, by the adapters' type
PRODUCTS = {T_F32: 6, T_F16: 6, T_BF16: 3}


class Adapters:
    """n adapters; what stands behind an adapter's rank is NaN."""

    def __init__(self, seed, type_, n, max_rank, cols, rows, ranks=None):
        r = np.random.default_rng(seed)
        self.type, self.n, self.max_rank, self.cols, self.rows = type_, n, max_rank, cols, rows
        self.rank = np.full(n, max_rank, np.int32) if ranks is None else np.array(ranks, np.int32)
        self.scale = r.uniform(-2, 2, n).astype(np.float32)
        a, b = r.standard_normal((n, max_rank, cols)) / np.sqrt(cols), r.standard_normal((n, rows, max_rank))
        for i, k in enumerate(self.rank):
            if 0 <= k < max_rank:
                a[i, k:], b[i, :, k:] = np.nan, np.nan
        self.a, self.b = encode(a, type_), encode(b, type_)

    def of(self, i):
        k = int(self.rank[i])
        return decode(self.a[i, :k], self.type), decode(self.b[i, :, :k], self.type)


def lora(ad, tok, ids, x, y_in):
    """float64 outputs (rows of no sequence: NaN in `mine` False) and a bound on their error.

    h is a sum of 32 exact products an instruction, at most 8 roundings of partial sums each, over PRODUCTS instructions for every
    32 columns, and 8 more where wavefronts' and workgroups' sums meet; F32 adapters leave out products of up to 2^-21 of each.
    Each is off by at most u = 2^-24 of sum |a x|. The same over the ranks for y, and two roundings for the scale and the sum
    with y_in."""
    out, tol = np.full(y_in.shape, np.nan), np.zeros(y_in.shape)
    mine = np.zeros(len(y_in), bool)
    lost = 2.0**-21 if ad.type == T_F32 else 0.0
    per = 8 * PRODUCTS[ad.type]
    down, up = (per * -(-ad.cols // 32) + 40) * U32 + lost, (per * -(-ad.max_rank // 32) + 8) * U32 + lost
    for s, i in enumerate(ids):
        rows = slice(int(tok[s]), int(tok[s + 1]))
        mine[rows] = True
        base = y_in[rows].astype(np.float64)
        if i == -1:
            out[rows] = base
            continue
        if not (0 <= i < ad.n and 0 <= ad.rank[i] <= ad.max_rank):
            continue
        a, b = ad.of(i)
        xs, f = x[rows].astype(np.float64), np.float64(ad.scale[i])
        h, size = xs @ a.T, np.abs(xs) @ np.abs(a).T
        d = h @ b.T
        out[rows] = base + f * d
        tol[rows] = abs(f) * ((down + up) * (size @ np.abs(b).T)) + 2 * U32 * (np.abs(base) + 2 * abs(f) * np.abs(d))
    return out, tol, mine


def lora32(ad, tok, ids, x, y_in):
    """The same in fp32 throughout."""
    out = y_in.copy()
    for s, i in enumerate(ids):
        rows = slice(int(tok[s]), int(tok[s + 1]))
        if 0 <= i < ad.n and 0 <= ad.rank[i] <= ad.max_rank:
            a, b = (z.astype(np.float32) for z in ad.of(i))
            out[rows] = y_in[rows] + ad.scale[i] * ((x[rows] @ a.T) @ b.T)
    return out


TYPES = (T_F32, T_F16, T_BF16)
