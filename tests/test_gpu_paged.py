"""The paged KV cache on the device against float64 (tests/paged_ref.py): the append with head norms and rotation, and
the attention over the pages, at the sizes, masks and damaged inputs where they can go wrong.

Tolerances are per value, from the inputs: half a step of the cache's type for what is stored, and the
bounds that paged_ref derives for the fp32 arithmetic."""
import numpy as np
import pytest
from paged_ref import HALF_STEP, T_BF16, T_F16, T_F32, Batch, attention, decode, encode, of_vectors, store, vector_bound

from fastgguf_amd.backend import ERR_ARG, BackendError, PagedBatch, PagedCache, PagedMask, PagedRope

pytestmark = pytest.mark.gpu


class Dev:
    """Device copies of host arrays, freed together."""

    def __init__(self, backend):
        self.be, self.at, self.ptr = backend, [], {}

    def put(self, a):
        a = np.ascontiguousarray(a)
        p = self.be.dev_alloc(max(16, a.nbytes))
        self.at.append(p)
        self.be.h2d(p, a)
        return p

    def get(self, p, like):
        out = np.empty_like(like)
        self.be.d2h(out, p)
        return out

    def __enter__(self):
        return self

    def __exit__(self, *a):
        for p in self.at:
            self.be.dev_free(p)


def put_batch(d, b, max_len=None, max_tok=None):
    """The cache and batch descriptors of b, its arrays on the device."""
    cache = PagedCache(b.type, d.put(b.k), d.put(b.v), d.put(b.table), n_pages=b.n_pages, page=b.page, table_stride=b.stride,
                       n_head_kv=b.n_kv, hd=b.hd, page_stride=b.page_stride)
    batch = PagedBatch(d.put(b.tok), d.put(b.len), n_seq=len(b.news), n_tok=b.n_tok, max_tok=max_tok or max(b.news + [1]),
                       max_len=max_len or max(b.lens + [1]))
    return cache, batch


def run_attention(be, b, q=None, scale=None, max_len=None, max_tok=None, slopes=None, prefix=None, extra=0, **kw):
    """o [n_tok][n_head][hd] from rows `extra` values apart; o's rows are 777 before the call."""
    q = b.q if q is None else q
    scale = b.hd**-0.5 if scale is None else scale
    row = b.n_head * b.hd
    with Dev(be) as d:
        cache, batch = put_batch(d, b, max_len, max_tok)
        wide = np.full((b.n_tok, row + extra), 777.0, np.float32)
        wide[:, :row] = q.reshape(b.n_tok, row)
        qd, od = d.put(wide), d.put(np.full_like(wide, 777.0))
        mask = PagedMask(scale, slopes=d.put(slopes) if slopes is not None else 0,
                         prefix=d.put(np.asarray(prefix, np.int32)) if prefix is not None else 0, **kw)
        be.paged_attention_dev(cache, batch, mask, b.n_head, qd, row + extra, od, row + extra)
        o = d.get(od, wide)
    assert (o[:, row:] == 777.0).all()
    return o[:, :row].reshape(b.n_tok, b.n_head, b.hd)


def check_attention(be, b, scale=None, max_len=None, max_tok=None, extra=0, **kw):
    scale = b.hd**-0.5 if scale is None else scale
    scale = float(np.float32(scale))
    o = run_attention(be, b, scale=scale, max_len=max_len, max_tok=max_tok, extra=extra, **kw)
    want, tol, mine = attention(b, b.q, scale, **kw)
    assert (o[~mine] == 777.0).all()  # rows of no sequence
    off = np.abs(o[mine] - want[mine])
    assert (off <= tol[mine]).all(), (float((off / tol[mine]).max()), np.argwhere(~(off <= tol[mine]))[:4])
    return o


# ---- the append ----

STORES = [  # type, hd, heads, K / V heads, page, news, lens, norms, n_rot, halves
    (T_F16, 128, 8, 2, 16, [1], [1], False, 128, False),
    (T_F16, 128, 8, 2, 16, [1], [4096], True, 128, True),
    (T_BF16, 64, 4, 4, 32, [1, 1, 0, 1], [17, 64, 0, 100], True, 64, True),
    (T_F16, 80, 5, 1, 64, [70, 0, 3], [70, 5, 131], True, 20, True),
    (T_F32, 96, 4, 2, 16, [33, 16, 1], [40, 16, 300], False, 96, False),
    (T_BF16, 256, 4, 2, 128, [129, 2], [129, 260], True, 256, True),
    (T_F32, 256, 2, 1, 256, [3], [300], True, 64, False),
    (T_F16, 64, 4, 1, 64, [200, 7], [451, 7], False, 0, False),
    (T_F16, 128, 32, 8, 16, [5], [70], False, 126, True),
    (T_BF16, 80, 3, 3, 16, [64], [64], True, 80, False),
]


@pytest.mark.parametrize("i", range(len(STORES)))
@pytest.mark.parametrize("form", ["fused", "apart", "in place"])
def test_store(backend, i, form):
    t, hd, nh, nkv, page, news, lens, normed, n_rot, halves = STORES[i]
    b = Batch(100 + i, t, hd, nh, nkv, page, news, lens, pad=(i % 3, 2 * (i % 2)), gap=8 * (i % 4))
    r = b.rng
    qkv = (r.standard_normal((b.n_tok, nh + 2 * nkv, hd)) * np.exp(r.uniform(-3, 3, (1, nh + 2 * nkv, 1)))).astype(np.float32)
    norm = [(1 + 0.3 * r.standard_normal(hd)).astype(np.float32) for _ in range(2)] if normed else None
    factors = np.exp(r.uniform(0, 2, max(1, n_rot // 2))).astype(np.float32) if i % 2 else None
    base, scale = (500000.0, 0.25) if i % 3 == 0 else (10000.0, 1.0)
    q, k, v, eq, ek = store(b, qkv, norm, n_rot, halves, base, scale, factors)
    row = (nh + 2 * nkv) * hd
    with Dev(backend) as d:
        cache, batch = put_batch(d, b)
        rope = PagedRope(n_rot=n_rot, halves=halves, freq_base=base, freq_scale=scale,
                         freq_factors=d.put(factors) if factors is not None else 0, q_norm=d.put(norm[0]) if norm else 0,
                         k_norm=d.put(norm[1]) if norm else 0)
        if form == "apart":
            qd, ldq = d.put(qkv[:, :nh]), nh * hd
            wide = np.full((2, b.n_tok, nkv * hd + 12), 3.0, np.float32)
            wide[0, :, :nkv * hd] = qkv[:, nh:nh + nkv].reshape(b.n_tok, -1)
            wide[1, :, :nkv * hd] = qkv[:, nh + nkv:].reshape(b.n_tok, -1)
            kd, vd, ldkv = d.put(wide[0]), d.put(wide[1]), nkv * hd + 12
        else:
            qd, ldq = d.put(qkv), row
            kd, vd, ldkv = qd + 4 * nh * hd, qd + 4 * (nh + nkv) * hd, row
        before = np.full((b.n_tok, nh * hd + 4), 777.0, np.float32)
        od, ldo = (qd, row) if form == "in place" else (d.put(before), nh * hd + 4)
        backend.paged_store_dev(cache, batch, rope, nh, qd, ldq, kd, vd, ldkv, od, ldo)
        if form == "in place":
            got = d.get(od, qkv)
            assert np.array_equal(got[:, nh:], qkv[:, nh:])
            got, before = got[:, :nh], qkv[:, :nh]
        else:
            got = d.get(od, before)
            assert (got[:, nh * hd:] == 777.0).all()
            got, before = got[:, :nh * hd].reshape(b.n_tok, nh, hd), before[:, :nh * hd].reshape(b.n_tok, nh, hd)
        kc, vc = d.get(cache.k, b.k), d.get(cache.v, b.v)
    touched = {False: np.zeros(b.k.shape, bool), True: np.zeros(b.k.shape, bool)}
    mine = np.zeros(b.n_tok, bool)
    for tok, s, pos in b.tokens():
        mine[tok] = True
        assert (np.abs(got[tok] - q[tok]) <= eq[tok] + 1e-30).all()
        for h in range(nkv):
            for is_v, code, want, err in ((False, kc, k[tok, h], ek[tok, h]), (True, vc, v[tok, h], 0.0)):
                at = b.at(s, pos, h, is_v)
                touched[is_v][at] = True
                step = HALF_STEP[t] if t != T_F32 or is_v else 0.0
                # half a step of the stored value, itself off by err (F16 below 2^-14: half of 2^-24)
                assert (np.abs(decode(code[at], t) - want) <= step * (np.abs(want) + err) + err + 2.0**-25 * (t == T_F16)).all()
                if is_v:
                    assert np.array_equal(code[at], encode(v[tok, h].astype(np.float32), t))
    assert np.array_equal(got[~mine], before[~mine])
    for is_v, code, old in ((False, kc, b.k), (True, vc, b.v)):  # nothing else changes
        assert np.array_equal(code[~touched[is_v]], old[~touched[is_v]])


def test_store_far_positions(backend):
    """Angles at positions where 32 bits would hold no fraction of a turn."""
    b = Batch(7, T_F16, 64, 2, 1, 256, [3], [3])
    far = 1 << 20
    b.lens, b.len, b.stride = [far], np.array([far], np.int32), far // 256
    b.table = np.full((1, b.stride), -1, np.int32)
    b.table[0, -1] = 0
    qkv = b.rng.standard_normal((3, 4, 64)).astype(np.float32)
    q, k, _, eq, ek = store(b, qkv, None, 64, True, 5e6)
    with Dev(backend) as d:
        cache, batch = put_batch(d, b)
        qd, od = d.put(qkv), d.put(np.zeros((3, 2, 64), np.float32))
        backend.paged_store_dev(cache, batch, PagedRope(n_rot=64, halves=True, freq_base=5e6), 2, qd, 256, qd + 512, qd + 768, 256, od, 128)
        got, kc = d.get(od, np.zeros((3, 2, 64), np.float32)), d.get(cache.k, b.k)
    assert (np.abs(got - q) <= eq).all()
    for i in range(3):
        at = b.at(0, far - 3 + i, 0, False)
        assert (np.abs(decode(kc[at], T_F16) - k[i, 0]) <= 2.0**-11 * (np.abs(k[i, 0]) + ek[i, 0]) + ek[i, 0] + 2.0**-25).all()


def test_store_without_queries(backend):
    b = Batch(8, T_BF16, 64, 2, 2, 16, [5], [20])
    kv = b.rng.standard_normal((2, 5, 2, 64)).astype(np.float32)
    with Dev(backend) as d:
        cache, batch = put_batch(d, b)
        backend.paged_store_dev(cache, batch, PagedRope(), 0, 0, 0, d.put(kv[0]), d.put(kv[1]), 128, 0, 0)
        kc, vc = d.get(cache.k, b.k), d.get(cache.v, b.v)
    for tok, s, pos in b.tokens():
        for h in range(2):
            assert np.array_equal(kc[b.at(s, pos, h, False)], encode(kv[0, tok, h], T_BF16))
            assert np.array_equal(vc[b.at(s, pos, h, True)], encode(kv[1, tok, h], T_BF16))


def test_store_decreasing_starts(backend):
    """Starts that decrease: rows of one sequence are appended, rows of two may not be read or written out of range."""
    b = Batch(10, T_F16, 64, 2, 1, 16, [5, 0, 5], [5, 0, 9])
    b.tok, b.n_tok = np.array([0, 5, 3, 8], np.int32), 8
    qkv = b.rng.standard_normal((8, 4, 64)).astype(np.float32)
    with Dev(backend) as d:
        cache, batch = put_batch(d, b, max_tok=5)
        qd, od = d.put(qkv), d.put(np.full((8, 2, 64), 777.0, np.float32))
        backend.paged_store_dev(cache, batch, PagedRope(), 2, qd, 256, qd + 512, qd + 768, 256, od, 128)
        got, kc = d.get(od, np.zeros((8, 2, 64), np.float32)), d.get(cache.k, b.k)
    for t in (0, 1, 2, 5, 6, 7):
        assert np.array_equal(got[t], qkv[t, :2])
        s, pos = (0, t) if t < 3 else (2, 9 - 5 + t - 3)
        assert np.array_equal(kc[b.at(s, pos, 0, False)], encode(qkv[t, 2], T_F16))


def test_store_overflow_and_specials(backend):
    """F16 rounds to nearest even, past 65504 to infinity; NaN stays NaN."""
    b = Batch(9, T_F16, 64, 1, 1, 16, [1], [1])
    kv = np.zeros((2, 1, 1, 64), np.float32)
    kv[:, 0, 0, :10] = [65504, 65519.9, 65520, -1e30, np.inf, np.nan, 2.0**-24, 2.0**-25, 1 + 2.0**-11, 1 + 3 * 2.0**-11]
    with Dev(backend) as d:
        cache, batch = put_batch(d, b)
        backend.paged_store_dev(cache, batch, PagedRope(), 0, 0, 0, d.put(kv[0]), d.put(kv[1]), 64, 0, 0)
        kc, vc = d.get(cache.k, b.k), d.get(cache.v, b.v)
    with np.errstate(over="ignore"):
        want = kv[0, 0, 0].astype(np.float16)
    for c in (kc[b.at(0, 0, 0, False)], vc[b.at(0, 0, 0, True)]):
        assert np.array_equal(c.view(np.float16), want, equal_nan=True)


# ---- damaged batches: in-bounds, named by NaN, nothing appended ----

def damaged(b, how):
    """Makes sequence 1 of 3 break a bound; (max_len, max_tok) of the call."""
    if how == "longer than max_len":
        return max(b.lens[0], b.lens[2]), None
    if how == "more than max_tok":
        return None, max(b.news[0], b.news[2])
    if how == "shorter than its tokens":
        b.len[1] = b.news[1] - 1
    if how == "longer than the table":
        b.len[1] = b.stride * b.page + 1
        return b.stride * b.page * 4, None
    if how == "negative":
        b.len[1] = -5
    return None, None


HOWS = ["longer than max_len", "more than max_tok", "shorter than its tokens", "longer than the table", "negative"]


@pytest.mark.parametrize("how", HOWS)
@pytest.mark.parametrize("news", [[2, 3, 1], [40, 70, 30]])
def test_damaged_sequences(backend, how, news):
    b = Batch(20, T_F16, 64, 4, 2, 16, news, [news[0] + 9, news[1] + 100, news[2]])
    max_len, max_tok = damaged(b, how)
    o = run_attention(backend, b, max_len=max_len, max_tok=max_tok)
    want, tol, _ = attention(b, b.q, float(np.float32(0.125)))
    bad = np.arange(b.tok[1], b.tok[2])
    assert np.isnan(o[bad]).all()
    fine = np.setdiff1d(np.arange(b.n_tok), bad)
    assert (np.abs(o[fine] - want[fine]) <= tol[fine]).all()
    qkv = b.rng.standard_normal((b.n_tok, 8, 64)).astype(np.float32)
    with Dev(backend) as d:
        cache, batch = put_batch(d, b, max_len, max_tok)
        qd, od = d.put(qkv), d.put(np.zeros((b.n_tok, 4, 64), np.float32))
        backend.paged_store_dev(cache, batch, PagedRope(n_rot=64), 4, qd, 512, qd + 1024, qd + 1536, 512, od, 256)
        got, kc, vc = d.get(od, np.zeros((b.n_tok, 4, 64), np.float32)), d.get(cache.k, b.k), d.get(cache.v, b.v)
    assert np.isnan(got[bad]).all() and np.isfinite(got[fine]).all()
    changed = np.zeros(b.k.shape, bool)
    for s in (0, 2):
        for pos in range(b.lens[s] - b.news[s], b.lens[s]):
            for h in range(2):
                changed[b.at(s, pos, h, False)] = True
    assert np.array_equal(kc != b.k, changed & (kc != b.k)) and (kc != b.k).sum() > 0.9 * changed.sum()
    assert (vc != b.v).sum() <= changed.sum()


@pytest.mark.parametrize("page_no", [-1, 0x7FFFFFFF, -0x80000000, "n_pages"])
@pytest.mark.parametrize("news", [[1, 1], [40, 5], [40, 5] + [9] * 130])
def test_bad_pages(backend, page_no, news):
    """A page that does not exist: the rows that see one of its positions are NaN, the others as they are; an append into it
    writes nothing."""
    b, b_good = [Batch(21, T_BF16, 64, 4, 2, 16, news, [news[0] + 70, 60] + news[2:]) for _ in range(2)]
    bad_pos = (b.lens[0] - 10) // 16 * 16  # page of the last positions: early new tokens do not see it
    b.table[0, bad_pos // 16] = b.n_pages if page_no == "n_pages" else page_no
    want, tol, _ = attention(b_good, b.q, 0.125)
    o = run_attention(backend, b)
    for t, s, p in b.tokens():
        if s == 0 and p >= bad_pos:
            assert np.isnan(o[t]).all()
        else:
            assert (np.abs(o[t] - want[t]) <= tol[t]).all()
    kv = b.rng.standard_normal((b.n_tok, 2, 64)).astype(np.float32)
    with Dev(backend) as d:
        cache, batch = put_batch(d, b)
        kd = d.put(kv)
        backend.paged_store_dev(cache, batch, PagedRope(), 0, 0, 0, kd, kd, 128, 0, 0)
        kc = d.get(cache.k, b.k)
    changed = np.zeros(b.k.shape, bool)
    for t, s, p in b.tokens():
        if not (s == 0 and b.table[0, p // 16] != b_good.table[0, p // 16]):
            for h in range(2):
                changed[b.at(s, p, h, False)] = True
    assert not (kc != b.k)[~changed].any()


# ---- attention ----

SHAPES = [  # type, hd, heads, K / V heads, page, news, lens
    (T_F16, 128, 8, 2, 16, [1], [1]),
    (T_F16, 128, 8, 2, 16, [1, 1, 1], [2, 15, 16]),
    (T_F16, 128, 32, 8, 64, [1, 1, 0, 1], [1000, 33, 0, 257]),
    (T_BF16, 128, 4, 4, 32, [1, 1], [700, 31]),
    (T_F32, 128, 8, 1, 16, [1, 1], [129, 515]),
    (T_F16, 64, 16, 1, 128, [1], [2049]),
    (T_F16, 64, 17, 1, 16, [1, 1], [100, 63]),  # 17 rows a K / V head
    (T_BF16, 80, 5, 5, 16, [1, 3, 2], [200, 65, 2]),
    (T_F32, 80, 4, 2, 256, [2], [700]),
    (T_F16, 96, 6, 3, 32, [1, 2, 5], [64, 128, 300]),
    (T_F32, 96, 2, 1, 16, [3], [50]),
    (T_BF16, 256, 4, 2, 32, [1, 1], [300, 64]),
    (T_F16, 256, 8, 4, 16, [2], [600]),
    (T_F32, 256, 2, 2, 64, [1], [130]),
    (T_F16, 128, 8, 2, 16, [17, 33, 4], [17, 50, 400]),
    (T_F16, 128, 4, 1, 64, [200], [200]),
    (T_F16, 128, 3, 1, 16, [64, 1, 0, 130], [700, 90, 40, 131]),
    (T_BF16, 128, 2, 2, 32, [150], [333]),
    (T_F32, 128, 2, 1, 16, [70, 40], [70, 300]),
    (T_BF16, 64, 4, 4, 16, [100, 65, 64], [100, 65, 64]),
    (T_F16, 80, 2, 1, 64, [90], [190]),
    (T_F32, 80, 2, 2, 16, [65], [80]),
    (T_BF16, 96, 4, 2, 128, [129], [400]),
    (T_BF16, 256, 4, 2, 16, [70], [150]),
    (T_F16, 256, 2, 1, 32, [100, 30], [100, 200]),
    (T_F32, 256, 1, 1, 16, [40], [100]),
]


def crowd(news, lens):
    """The sequences and 130 short prompts: with two K / V heads too many workgroups for the prompt kernel's form of half the rows."""
    return list(news) + [9] * 130, list(lens) + [9] * 130


def shape(i, seed=0, **kw):
    t, hd, nh, nkv, page, news, lens = SHAPES[i]
    return Batch(300 + i + 1000 * seed, t, hd, nh, nkv, page, news, lens, **kw)


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_attention(backend, i):
    check_attention(backend, shape(i, pad=(i % 2, i % 3), gap=16 * (i % 3)), extra=4 * (i % 4))


@pytest.mark.parametrize("i", range(len(SHAPES)))
@pytest.mark.parametrize("how", ["cap", "bias", "window", "prefix", "all"])
def test_attention_forms(backend, i, how):
    b = shape(i, seed=1)
    kw = {}
    if how in ("cap", "all"):
        kw["softcap"] = 5.0
        b.q *= 4
    if how in ("bias", "all"):
        kw["slopes"] = np.exp2(-np.linspace(0.3, 8, b.n_head)).astype(np.float32)
    if how in ("window", "all"):
        kw["window"] = [1, 7, 16, 40, 64, 129, 1000][i % 7]
    if how in ("prefix", "all"):
        kw["prefix"] = np.array([[0, m, m // 2, -3, 1, m + 100][(i + s) % 6] for s, m in enumerate(b.lens)], np.int32)
    check_attention(backend, b, **kw)


@pytest.mark.parametrize("t,hd", [(t, hd) for t in (T_F16, T_BF16, T_F32) for hd in (64, 80, 96, 128, 256)])
@pytest.mark.parametrize("how", ["plain", "all"])
def test_attention_crowded(backend, t, hd, how):
    """Enough rows for whole workgroups of them, ranges in one part and in several, few-row sequences among them."""
    b = Batch(51, t, hd, 4, 2, 32, *crowd([200, 1, 70, 0, 3, 130], [200, 90, 640, 0, 3, 333]), gap=8)
    kw = {}
    if how == "all":
        kw = dict(softcap=5.0, slopes=np.exp2(-np.linspace(0.3, 8, 4)).astype(np.float32), window=129,
                  prefix=np.resize([0, 50, 9, 300, 4, 20], len(b.news)).astype(np.int32))
        b.q *= 4
    check_attention(backend, b, **kw)


@pytest.mark.parametrize("t", [T_F16, T_BF16, T_F32])
@pytest.mark.parametrize("news", [1, 4, 40])
def test_attention_sharp_scores(backend, t, news):
    """Scores of up to some hundreds, large maxima late in the range, and a scale that is not hd^-0.5."""
    b = Batch(40, t, 64, 4, 2, 16, [news], [400], sigma=3.0)
    b.q *= 20
    check_attention(backend, b, scale=0.31)
    check_attention(backend, b, scale=-0.31)
    check_attention(backend, b, scale=0.0)


@pytest.mark.parametrize("t,tiny,huge", [(T_F16, 2.0**-12, 3e4), (T_BF16, 1e-25, 1e25), (T_F32, 1e-25, 1e25)])
@pytest.mark.parametrize("news", [1, 40])
def test_attention_ranges(backend, t, tiny, huge, news):
    """Queries far outside 16-bit range, and values of the cache at the ends of its type's."""
    for k_size, q_size, v_size in ((1.0, 1e6, 1.0), (1.0, 1e-9, huge), (tiny, 1.0 / tiny, tiny)):
        b = Batch(41, t, 128, 4, 2, 16, [news], [100])
        b.k, b.v = encode(decode(b.k, t) * k_size, t), encode(decode(b.v, t) * v_size / 8, t)
        b.q = (b.q * q_size).astype(np.float32)
        scale = 0.088 / (k_size * q_size)
        o = run_attention(backend, b, scale=scale)
        want, tol, _ = attention(b, b.q, float(np.float32(scale)))
        assert (np.abs(o - want) <= tol).all()


@pytest.mark.parametrize("news", [1, 40])
def test_attention_outlier_channels(backend, news):
    """A channel whose K is large and whose q is small beside the row's others: it counts as much as they do."""
    b = Batch(48, T_F16, 64, 4, 2, 16, [news], [100])
    size = np.ones(64)
    size[7] = 2.0**13
    for s, m in enumerate(b.lens):
        for pos in range(m):
            for h in range(2):
                at = b.at(s, pos, h, False)
                b.k[at] = encode(decode(b.k[at], T_F16) * size / 8, T_F16)
    b.q = (b.q / size).astype(np.float32)
    check_attention(backend, b)


@pytest.mark.parametrize("news", [[1, 1, 1], [40, 1, 2]])
def test_attention_prefix_limits(backend, news):
    """A prefix is taken as 0 .. len, whatever it holds."""
    b = Batch(49, T_F16, 64, 4, 2, 16, news, [n + 30 for n in news])
    check_attention(backend, b, prefix=np.array([-2**31, 2**31 - 1, -1], np.int32))


SPLITS = [(T_BF16, 80, 4), (T_F32, 96, 2), (T_F16, 256, 2), (T_F32, 256, 1), (T_BF16, 128, 4), (T_F32, 80, 2), (T_F16, 96, 3)]


@pytest.mark.parametrize("t,hd,nh", SPLITS)
@pytest.mark.parametrize("news,lens", [([1], [2500]), ([3, 1], [2500, 700]), ([40], [2500]), ([40, 1, 0, 3], [2100, 1500, 9, 3])])
def test_attention_splits(backend, t, hd, nh, news, lens):
    """Both kernels' split ranges and their joins, one launch with both included, for each way a head's values are laid out."""
    b = Batch(50, t, hd, nh, 1, 32, news, lens, pad=(1, 2))
    check_attention(backend, b)
    check_attention(backend, b, window=1000, softcap=9.0)


@pytest.mark.parametrize("lens", [[5000], [3, 5000, 1200, 64]])
@pytest.mark.parametrize("news", [1, 4])
def test_attention_long_split(backend, lens, news):
    """Ranges that are split over workgroups, lengths far apart, a bound far above them."""
    b = Batch(42, T_F16, 64, 4, 1, 16, [min(news, m) for m in lens], lens)
    check_attention(backend, b)
    b.stride += 2000  # a table for 32000 positions more
    b.table = np.concatenate([b.table, np.full((len(lens), 2000), -1, np.int32)], 1)
    check_attention(backend, b, max_len=b.stride * 16)


@pytest.mark.parametrize("news", [1, 3, 50, 200])
@pytest.mark.parametrize("t", [T_F16, T_BF16, T_F32])
def test_attention_stale_positions(backend, t, news):
    """What positions behind a sequence's end, behind its window and in free pages hold does not matter."""
    b = Batch(43, t, 128, 4, 2, 64, [news, 1], [news + 90, 30])
    for kw in ({}, {"window": 20}):
        for s, m in enumerate(b.lens):
            first = max(0, m - b.news[s] - (20 if kw else 10**6) + 1)
            for pos in list(range(m, -(-m // 64) * 64)) + list(range(first)):
                for h in range(2):
                    for is_v, buf in ((False, b.k), (True, b.v)):
                        at = b.at(s, pos, h, is_v)
                        buf[at] = encode(np.where(np.arange(128) % 2, np.nan, np.inf), t)
        with np.errstate(invalid="ignore"):
            o = run_attention(backend, b, scale=0.0884, **kw)
        clean = Batch(43, t, 128, 4, 2, 64, [news, 1], [news + 90, 30])
        want, tol, _ = attention(clean, clean.q, float(np.float32(0.0884)), **kw)
        assert (np.abs(o - want) <= tol).all()
    b.table[0, :max(0, b.lens[0] - news - 20 + 1) // 64] = -7  # pages that the window has left
    o = run_attention(backend, b, scale=0.0884, window=20)
    assert (np.abs(o - want) <= tol).all()


@pytest.mark.parametrize("what", ["k", "v", "q"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("news,crowded", [(4, False), (90, False), (90, True)])
def test_attention_non_finite(backend, what, value, news, crowded):
    """A new token's value that is not finite: the tokens before it do not see it, whatever tile they share."""
    t, hd = T_F16, 128
    batch = crowd([news], [news + 20]) if crowded else ([news], [news + 20])
    b, clean = [Batch(44, t, hd, 4, 2, 16, *batch) for _ in range(2)]
    at = news // 2  # of the new tokens
    if what == "q":
        b.q[at, 1, 5] = value
    else:
        (b.k if what == "k" else b.v)[b.at(0, 20 + at, 1, what == "v")[7]] = encode(np.float32([value]), t)[0]
    with np.errstate(invalid="ignore"):
        o = run_attention(backend, b, scale=0.0884)
    want, tol, _ = attention(clean, clean.q, float(np.float32(0.0884)))
    for r in range(news):
        for h in range(4):
            hit = (r == at and h == 1) if what == "q" else (r >= at and h // 2 == 1)
            if not hit:
                assert (np.abs(o[r, h] - want[r, h]) <= tol[r, h]).all(), (r, h)
            elif what == "v":  # value 7 of the head is not finite, the others as they were
                assert not np.isfinite(o[r, h, 7])
                rest = np.arange(hd) != 7
                assert (np.abs(o[r, h] - want[r, h]) <= tol[r, h])[rest].all()
            elif np.isnan(value):
                assert np.isnan(o[r, h]).all()


def test_attention_64_bit_offsets(backend):
    """Pages past 2^32 bytes from the start of the cache."""
    b = Batch(45, T_F16, 64, 4, 2, 16, [2], [40])
    stride, n = (1 << 30) + 64, 4
    with Dev(backend) as d:
        big = [backend.dev_alloc(2 * n * stride) for _ in range(2)]
        try:
            pages = [3, 1, 2]
            for j in range(3):
                old = int(b.table[0, j]) * b.page_stride
                for p, src in zip(big, (b.k, b.v)):
                    backend.h2d(p + 2 * pages[j] * stride, src[old:old + b.page_values])
            cache = PagedCache(T_F16, big[0], big[1], d.put(np.array([pages], np.int32)), n_pages=n, page=16, table_stride=3,
                               n_head_kv=2, hd=64, page_stride=stride)
            batch = PagedBatch(d.put(b.tok), d.put(b.len), n_seq=1, n_tok=2, max_tok=2, max_len=48)
            od = d.put(np.zeros((2, 4, 64), np.float32))
            backend.paged_attention_dev(cache, batch, PagedMask(0.125), 4, d.put(b.q), 256, od, 256)
            o = d.get(od, np.zeros((2, 4, 64), np.float32))
            kv = b.rng.standard_normal((2, 2, 64)).astype(np.float32)
            kd = d.put(kv)
            backend.paged_store_dev(cache, batch, PagedRope(), 0, 0, 0, kd, kd, 128, 0, 0)
            k2, v2 = np.empty(b.page_values, np.uint16), np.empty(b.page_values, np.uint16)
            backend.d2h(k2, big[0] + 2 * 2 * stride)
            backend.d2h(v2, big[1] + 2 * 2 * stride)
        finally:
            for p in big:
                backend.dev_free(p)
    want, tol, _ = attention(b, b.q, 0.125)
    assert (np.abs(o - want) <= tol).all()
    for t, pos in ((0, 38), (1, 39)):
        for h in range(2):
            at = h * 64 * 16
            assert np.array_equal(k2[at + pos % 16 * 64:][:64], encode(kv[t, h], T_F16))
            assert np.array_equal(v2[at + pos % 16:at + 64 * 16:16], encode(kv[t, h], T_F16))


def test_attention_many_sequences(backend):
    """More sequences than a wavefront has lanes, empty ones among them."""
    rng = np.random.default_rng(5)
    news = [int(v) for v in rng.choice([0, 1, 1, 1, 2], 150)]
    lens = [n + int(v) for n, v in zip(news, rng.integers(0, 40, 150))]
    check_attention(backend, Batch(46, T_F16, 64, 2, 1, 16, news, lens))
    news = [int(v) for v in rng.choice([0, 1, 9, 20], 150)]
    lens = [n + int(v) for n, v in zip(news, rng.integers(0, 40, 150))]
    check_attention(backend, Batch(47, T_F16, 64, 2, 1, 16, news, lens))


def test_same_results_twice(backend):
    """No order of arrival in the results."""
    for i in (2, 5, 16):
        b = shape(i, seed=2)
        first = run_attention(backend, b)
        for _ in range(3):
            assert np.array_equal(first.view(np.uint32), run_attention(backend, b).view(np.uint32))


# ---- together ----

@pytest.mark.parametrize("t", [T_F32, T_F16])
def test_prompt_then_decode(backend, t):
    """Two sequences: their prompts appended and read in a batch, then tokens one by one from a recorded graph whose
    lengths move on, against float64 over everything appended."""
    hd, nh, nkv, page, steps = 64, 4, 2, 16, 6
    prompts = [37, 5]
    b = Batch(60, t, hd, nh, nkv, page, prompts, [p + steps for p in prompts])
    b.lens, b.len = prompts, np.array(prompts, np.int32)
    row = (nh + 2 * nkv) * hd
    kw = dict(n_rot=hd, halves=True)
    r = np.random.default_rng(61)
    norm = [(1 + 0.2 * r.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    with Dev(backend) as d:
        cache, batch = put_batch(d, b, max_len=b.stride * page)
        rope = PagedRope(q_norm=d.put(norm[0]), k_norm=d.put(norm[1]), **kw)
        mask = PagedMask(hd**-0.5)

        def step(be, x, q, o):
            be.paged_store_dev(cache, batch, rope, nh, x, row, x + 4 * nh * hd, x + 4 * (nh + nkv) * hd, row, q, nh * hd)
            be.paged_attention_dev(cache, batch, mask, nh, q, nh * hd, o, nh * hd)

        def check(qkv, o, k_codes):
            q, _, _, eq, _ = store(b, qkv, norm, **kw)
            b.k, b.v = k_codes
            want, tol, mine = attention(b, q.astype(np.float32), float(np.float32(hd**-0.5)))
            # q' is off by eq: scores by eq |k| / 8
            k = np.abs(decode(b.k, t)).max()
            tol = tol + 4 * eq.sum(-1).max() * k * hd**-0.5 * np.abs(decode(b.v, t)).max()
            assert (np.abs(o - want)[mine] <= tol[mine]).all()

        def codes():
            return d.get(cache.k, b.k), d.get(cache.v, b.v)

        n = sum(prompts)
        qkv = r.standard_normal((n, nh + 2 * nkv, hd)).astype(np.float32)
        like = np.zeros((n, nh, hd), np.float32)
        x, q, o = d.put(qkv), d.put(like), d.put(like)
        step(backend, x, q, o)
        check(qkv, d.get(o, like), codes())

        # decode: the same descriptors' arrays, new contents, one graph
        b.news, b.tok, b.n_tok = [1, 1], np.array([0, 1, 2], np.int32), 2
        batch.n_tok, batch.max_tok = 2, 1
        backend.h2d(batch.tok, b.tok)
        like = np.zeros((2, nh, hd), np.float32)

        def next_token(i):
            b.lens = [p + i + 1 for p in prompts]
            b.len = np.array(b.lens, np.int32)
            backend.h2d(batch.len, b.len)
            qkv = r.standard_normal((2, nh + 2 * nkv, hd)).astype(np.float32)
            backend.h2d(x, qkv)
            return qkv

        qkv = next_token(0)
        step(backend, x, q, o)  # sizes the scratch
        check(qkv, d.get(o, like), codes())
        backend.graph_begin()
        step(backend, x, q, o)
        g = backend.graph_end()
        try:
            for i in range(1, steps):
                qkv = next_token(i)
                backend.graph_launch(g)
                check(qkv, d.get(o, like), codes())
                replay = d.get(o, like)
                step(backend, x, q, o)  # the eager calls, on the same inputs
                assert np.array_equal(replay, d.get(o, like))
        finally:
            backend.graph_destroy(g)


def test_graphs_share_scratch(backend):
    """Recorded calls with split ranges, of generation, of a prompt and of both, replayed in turn with eager calls
    between them: each gives the eager call's values for the queries that are there then."""
    shapes = [([1, 1], [3000, 2000]), ([40], [2500]), ([40, 1, 3], [1000, 2500, 700])]
    r = np.random.default_rng(64)
    with Dev(backend) as d:
        runs = []
        for i, (news, lens) in enumerate(shapes):
            b = Batch(65 + i, T_F16, 128, 8, 2, 64, news, lens)
            cache, batch = put_batch(d, b)
            q, o = d.put(b.q), d.put(b.q)

            def call(cache=cache, batch=batch, q=q, o=o):
                backend.paged_attention_dev(cache, batch, PagedMask(128**-0.5), 8, q, 1024, o, 1024)

            runs.append([b, q, o, call, None])
        for x in runs:  # sizes the scratch
            x[3]()
        backend.sync()
        for x in runs:
            backend.graph_begin()
            x[3]()
            x[4] = backend.graph_end()
        try:
            for turn in range(4):
                for b, q, o, call, g in runs[turn % 3:] + runs[:turn % 3]:
                    b.q = r.standard_normal(b.q.shape).astype(np.float32)
                    backend.h2d(q, b.q)
                    backend.h2d(o, np.zeros_like(b.q))
                    backend.graph_launch(g)
                    got = d.get(o, b.q)
                    call()
                    assert np.array_equal(got.view(np.uint32), d.get(o, b.q).view(np.uint32))
                    if turn == 3:
                        want, tol, _ = attention(b, b.q, float(np.float32(128**-0.5)))
                        assert (np.abs(got - want) <= tol).all()
        finally:
            for x in runs:
                backend.graph_destroy(x[4])


def test_scratch_and_graphs():
    """Scratch that would grow while a call is recorded is refused, and a recorded call keeps its own when a larger eager
    call takes more."""
    from fastgguf_amd.backend import Backend
    be = Backend(0)
    try:
        with Dev(be) as d:
            small = Batch(70, T_F16, 64, 4, 1, 16, [1], [900])
            large = Batch(71, T_F16, 128, 8, 8, 16, [1, 60], [3000, 2000])
            calls = []
            for b in (small, large):
                cache, batch = put_batch(d, b)
                q, o, row = d.put(b.q), d.put(np.zeros_like(b.q)), b.n_head * b.hd
                calls.append((lambda cache=cache, batch=batch, b=b, q=q, o=o, row=row: be.paged_attention_dev(
                    cache, batch, PagedMask(0.125), b.n_head, q, row, o, row), b, o))

            def check(b, o):
                want, tol, _ = attention(b, b.q, 0.125)
                assert (np.abs(d.get(o, b.q) - want) <= tol).all()
                be.h2d(o, np.zeros_like(b.q))

            calls[0][0]()
            check(*calls[0][1:])
            be.graph_begin()
            calls[0][0]()
            with pytest.raises(BackendError, match="grow"):
                calls[1][0]()
            g = be.graph_end()
            for _ in range(2):
                be.graph_launch(g)
                check(*calls[0][1:])
                calls[1][0]()  # takes more
                check(*calls[1][1:])
            be.graph_destroy(g)
    finally:
        be.close()


def test_agrees_with_ring_attention(backend):
    """An fp32 paged cache against fgh_attention over the same positions in its ring."""
    b = Batch(62, T_F32, 128, 8, 2, 16, [5], [300])
    ring = [np.stack([np.concatenate([b.rows(0, h, is_v)[p] for h in range(2)]) for p in range(300)]).astype(np.float32)
            for is_v in (False, True)]
    en = np.arange(295, 300)
    want = backend.attention(b.q, ring[0], ring[1], np.zeros(5), en, 2, 128**-0.5)
    o = run_attention(backend, b)
    _, tol, _ = attention(b, b.q, 128**-0.5)
    assert (np.abs(o - want) <= 2 * tol).all()


def test_refusals(backend):
    b = Batch(63, T_F16, 64, 4, 2, 16, [1], [5])
    with Dev(backend) as d:
        cache, batch = put_batch(d, b)
        p = d.put(np.zeros(1024, np.float32))
        rope, mask = PagedRope(n_rot=64), PagedMask(0.125)

        def refused(call, word):
            with pytest.raises(BackendError) as e:
                call()
            assert e.value.status == ERR_ARG and word in str(e.value)

        st = lambda q=p, k=p + 1024, v=p + 1536, o=p + 2048, rope=rope, ldq=256, ldo=256, n=4: backend.paged_store_dev(  # noqa: E731
            cache, batch, rope, n, q, ldq, k, v, 128, o, ldo)
        at = lambda q=p, o=p + 2048, mask=mask, n=4, ldq=256, ldo=256: backend.paged_attention_dev(  # noqa: E731
            cache, batch, mask, n, q, ldq, o, ldo)
        st()
        at()
        refused(lambda: st(q=0), "null")
        refused(lambda: st(k=0), "null")
        refused(lambda: st(k=p + 4), "aligned")
        refused(lambda: st(o=p + 8), "aligned")
        refused(lambda: st(ldq=255), "ldq")
        refused(lambda: st(q=p, o=p, ldo=260), "stride")
        refused(lambda: st(rope=PagedRope(n_rot=3)), "n_rot")
        refused(lambda: st(rope=PagedRope(q_norm=p + 2)), "aligned")
        refused(lambda: at(q=0), "null")
        refused(lambda: at(o=p + 4), "aligned")
        refused(lambda: at(n=3), "n_head")
        refused(lambda: at(mask=PagedMask(float("nan"))), "scale")
        refused(lambda: at(mask=PagedMask(1.0, prefix=p + 1)), "aligned")
        for field, value, word in (("type", 8, "type"), ("hd", 72, "hd"), ("page", 24, "page"), ("k", 0, "null"), ("v", cache.v + 2, "aligned"),
                                   ("table", 0, "null"), ("page_stride", 8, "page_stride")):
            old = getattr(cache, field)
            setattr(cache, field, value)
            refused(at, word)
            refused(st, word)
            setattr(cache, field, old)
        at()


# ---- weights far below the row's largest ----

def with_null_key(t, news, lens, gap, at, hd=128, n_kv=2, group=2):
    """A batch whose rows all see one key (position `at` of every sequence long enough) that scores `gap` above the others and whose V is 0,
    so that the others, exp(-gap) of it, make the output. q and that key are few-bit numbers: their product is exact."""
    b = Batch(80 + news[0], t, hd, group * n_kv, n_kv, 16, news, lens, sigma=0.1)
    sign = np.where(b.rng.random(hd) < 0.5, -1.0, 1.0)
    b.q[:] = sign
    scale = 0.125 if hd < 256 else 0.0625
    size = round(gap / (hd * scale) * 256) / 256
    for s, (n, m) in enumerate(zip(news, lens)):
        if m - n < at:
            continue
        for h in range(n_kv):
            b.k[b.at(s, at, h, False)] = encode(sign * size, t)
            b.v[b.at(s, at, h, True)] = 0
    return b, scale


NULL_KEYS = [  # new tokens, lengths, position of the key
    ([1], [120], 0), ([1], [120], 100), ([1], [600], 37), ([4], [300], 2),  # few rows
    ([1] * 140, [130] * 140, 5), ([1] * 140, [130] * 140, 64),  # so many that no range is split
    ([40], [100], 0), ([40], [600], 33), ([20], [64], 40),  # prompts
    ([20] * 260, [64] * 260, 40), ([20] * 260, [64] * 260, 3), ([20] * 260, [60] * 260, 36),  # that fill the device: 128 rows, ranges whole
]


@pytest.mark.parametrize("gap", [12, 14, 16, 18, 20, 22])
@pytest.mark.parametrize("i", range(len(NULL_KEYS)))
def test_attention_null_key(backend, i, gap):
    """Weights of a row's output at 2^-17 to 2^-32 of its largest: 1e-5 per output vector, as everywhere. (Of the 1e-5: a weight at
    2^-31.7 of the largest is off by at most 2^-48 of it, evenly spread, which is 2^-16.3 / sqrt(3) = 7.3e-6 of a sum over
    many; the factor of a score of 31.7 powers of two rounded to fp32 is 31.7 ln 2 2^-24 = 1.3e-6.)"""
    b, scale = with_null_key(T_F16, *NULL_KEYS[i][:2], gap, NULL_KEYS[i][2])
    o = run_attention(backend, b, scale=scale)
    want, _, _ = attention(b, b.q, scale)
    assert of_vectors(o, want) <= 1e-5


NULL_TYPES = [([1], [200], 7), ([40], [150], 7), ([40], [200], 7), ([40], [600], 7), ([20] * 260, [64] * 260, 40)]


@pytest.mark.parametrize("t", [T_F16, T_BF16, T_F32])
@pytest.mark.parametrize("hd", [64, 80, 96, 128, 256])
@pytest.mark.parametrize("news,lens,at", NULL_TYPES)
def test_attention_null_key_types(backend, t, hd, news, lens, at):
    """The same for every type and head size, at a gap of 20."""
    b, scale = with_null_key(t, news, lens, 20, at, hd=hd)
    o = run_attention(backend, b, scale=scale)
    want, _, _ = attention(b, b.q, scale)
    assert of_vectors(o, want) <= 1e-5


# ---- starts that decrease ----

def falling(t, tok, pasts, hd=64, n_head=2, n_kv=1):
    """A batch of these starts, and of every row whether it is in one sequence only."""
    n_tok = max(tok)
    news = [max(0, e - s) for s, e in zip(tok, tok[1:])]
    b = Batch(90, t, hd, n_head, n_kv, 32, news, [n + p for n, p in zip(news, pasts)])
    b.tok, b.n_tok, b.q = np.array(tok, np.int32), n_tok, b.q[:n_tok]
    times = np.zeros(n_tok, int)
    for s, e in zip(tok, tok[1:]):
        times[s:e] += 1
    once = times == 1
    once[tok[-1]:] = False
    return b, once


FALLS = [  # starts, cached positions, query heads
    ([0, 900, 100, 1000], [0, 0, 0], 2),  # more tiles of rows and of positions than 1000 tokens have otherwise
    ([0, 40, 30, 50, 46, 70], [0, 0, 100, 0, 5], 1),  # the third sequence's 20 rows, 10 of them its own
    ([0, 40, 30, 50, 46, 70], [2000, 0, 1500, 0, 5], 1),  # in several splits
    ([v + 70 * i for i in range(30) for v in (0, 40, 30, 50, 46)] + [2100], [3, 0, 40, 0, 5] * 30, 1),  # more than 64 sequences
]


@pytest.mark.parametrize("i", range(len(FALLS)))
@pytest.mark.parametrize("broken", [False, True])
def test_falling_starts(backend, i, broken):
    """Rows that are in one sequence are appended, keys and values, and attended, however many tiles the others make; a broken
    sequence's are NaN and not appended."""
    tok, pasts, nh = FALLS[i]
    b, once = falling(T_F16, tok, pasts, n_head=nh)
    max_len = max(b.lens)
    want, tol, _ = attention(b, b.q, 0.125)
    bad = np.zeros(b.n_tok, bool)
    if broken:
        bad[b.tok[2]:b.tok[3]] = True
        b.len[2] = max_len + 1
    o = run_attention(backend, b, scale=0.125, max_len=max_len)
    assert np.isnan(o[once & bad]).all()
    fine = once & ~bad
    assert (np.abs(o - want)[fine] <= tol[fine]).all()
    qkv = b.rng.standard_normal((b.n_tok, nh + 2, 64)).astype(np.float32)
    with Dev(backend) as d:
        cache, batch = put_batch(d, b, max_len=max_len)
        x, od, row = d.put(qkv), d.put(np.full((b.n_tok, nh, 64), 777.0, np.float32)), (nh + 2) * 64
        backend.paged_store_dev(cache, batch, PagedRope(), nh, x, row, x + 256 * nh, x + 256 * (nh + 1), row, od, 64 * nh)
        got, kc, vc = d.get(od, np.zeros((b.n_tok, nh, 64), np.float32)), d.get(cache.k, b.k), d.get(cache.v, b.v)
    assert np.array_equal(got[fine], qkv[fine][:, :nh]) and np.isnan(got[once & bad]).all()
    for t, s, pos in b.tokens():
        if once[t]:
            for h, is_v, code, old in ((nh, False, kc, b.k), (nh + 1, True, vc, b.v)):
                at = b.at(s, pos, 0, is_v)
                assert np.array_equal(code[at], old[at] if bad[t] else encode(qkv[t, h], T_F16)), (t, s, pos, is_v)


# ---- scores of millions and more ----

@pytest.mark.parametrize("t", [T_F16, T_BF16, T_F32])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("news,lens", [([1, 3], [70, 3000]), ([40], [90]), ([20] * 260, [64] * 260)])
def test_attention_huge_scores(backend, t, size, news, lens):
    """Scores whose fp32 steps are powers of two apart: a row is the value at its largest score, as it is in fp32, where the next one is
    out of the scores' rounding (72 roundings of the largest sum of products, for 64 and the forms) and 30 more away.
    Its weight times that value, over the weight: 2^-21 for the products that an F32 cache leaves out (parts of w and v of 2^-7 and 2^-15
    of them: 2 x 2^-22), 8 roundings of the 6 products' sum, the weights' sum, its reciprocal and the last product: 2^-20 in all."""
    b = Batch(95, t, 64, 4, 2, 16, news, lens)
    b.q = (b.q * (size / 8)).astype(np.float32)
    rows = [r for r in b.tokens() if r[0] % 7 == 0 or len(news) < 3]
    keys = {(s, h): (b.rows(s, h, False), b.rows(s, h, True)) for s in {r[1] for r in rows} for h in range(2)}
    for kw in ({}, {"slopes": np.float32([0.0, size / 100, size, size * 10])}, {"softcap": 1e15}):
        o = run_attention(backend, b, scale=1.0, **kw)
        assert np.isfinite(o).all()
        if "softcap" in kw and size > 1e12:
            continue  # all at the cap: any of them
        clear = 0
        for row, s, p in rows:
            for h in range(4):
                k, v = (x[:p + 1] for x in keys[s, h // 2])
                z = k @ b.q[row, h].astype(np.float64)
                off = 72 * 2.0**-24 * (np.abs(k) @ np.abs(b.q[row, h])).max()
                if "softcap" in kw:
                    z = 1e15 * np.tanh(z / 1e15)
                if "slopes" in kw:
                    z = z - np.float64(kw["slopes"][h]) * (p - np.arange(p + 1))
                    off += 72 * 2.0**-24 * np.abs(z).max()
                order = np.argsort(z)
                if p == 0 or z[order[-1]] - z[order[-2]] > 2 * off + 30:
                    clear += 1
                    want = v[order[-1]]
                    assert (np.abs(o[row, h] - want) <= 2.0**-20 * np.abs(want) + 1e-9).all(), (row, h)
        assert clear > len(rows)


# ---- scales at the ends of their range ----

@pytest.mark.parametrize("t,k_size", [(T_F16, 1e4), (T_BF16, 1e18), (T_F32, 1e18)])
@pytest.mark.parametrize("scale", [0.0, 1e-36, -1e-37, 1e-39, -2e-42])
@pytest.mark.parametrize("news,lens", [([1, 3], [70, 3000]), ([40], [90]), ([20] * 260, [64] * 260)])
def test_attention_tiny_scales(backend, t, k_size, scale, news, lens):
    """Products near an fp32's largest, by scales near or below its smallest normal number, and by 0."""
    b = Batch(96, t, 64, 4, 2, 16, news, lens)
    b.k = encode(decode(b.k, t) * k_size, t)
    b.q = (b.q * (1e36 / k_size)).astype(np.float32)
    check_attention(backend, b, scale=scale)
    check_attention(backend, b, scale=scale, softcap=0.5)


@pytest.mark.parametrize("t", [T_F16, T_BF16, T_F32])
@pytest.mark.parametrize("news,lens", [([1, 3], [70, 3000]), ([40], [90])])
@pytest.mark.parametrize("softcap", [0.0, 1e-15])
def test_attention_zero_products(backend, t, softcap, news, lens):
    """Products that are 0 are scores of 0 at the largest scale and queries too: beside others that the cap makes +-1e-15, or alone."""
    b = Batch(97, t, 64, 4, 2, 16, news, lens)
    for s, m in enumerate(lens):
        for pos in range(m):
            for h in range(2):
                if pos % 3 == 0 or not softcap:
                    b.k[b.at(s, pos, h, False)] = 0
    b.q = (b.q * 1e30).astype(np.float32) if t == T_F16 else b.q
    o = run_attention(backend, b, scale=1e15, softcap=softcap)
    for row, s, p in b.tokens():
        for h in range(4):
            v = b.rows(s, h // 2, True)[:p + 1]
            # all weights the same: off by 16 roundings as in the others' bound
            assert (np.abs(o[row, h] - v.mean(0)) <= 32 * 2.0**-24 * np.abs(v).mean(0)).all()


# ---- results as vectors, values in bad pages, values that are not finite in every type ----

VECTORS = [([1], [4096]), ([1, 3], [700, 600]), ([40], [600]), ([9] * 130 + [40], [60] * 130 + [300])]


def ordinary(t, i, hd=128):
    return Batch(110 + i, t, hd, 4, 2, 32, *VECTORS[i])


@pytest.mark.parametrize("t", [T_F16, T_BF16, T_F32])
@pytest.mark.parametrize("hd", [64, 80, 128, 256])
@pytest.mark.parametrize("i", range(len(VECTORS)))
def test_attention_vectors(backend, t, hd, i):
    """Ordinary scores: an error per output vector as small as a plain fp32 form's (test_paged.py: a part of q or of the weights
    less would be more)."""
    b = ordinary(t, i, hd)
    scale = float(np.float32(hd**-0.5))
    want, _, mine = attention(b, b.q, scale)
    off = of_vectors(run_attention(backend, b, scale=scale)[mine], want[mine])
    assert off <= vector_bound(b, b.q, scale, want, mine) and off <= 1e-5


@pytest.mark.parametrize("page_no", [-1, 0x7FFFFFFF, "n_pages"])
@pytest.mark.parametrize("t", [T_F16, T_BF16, T_F32])
@pytest.mark.parametrize("news", [[1, 1], [40, 5], [150, 70, 1]])
def test_bad_pages_values(backend, t, news, page_no):
    """An append into a page that does not exist: values as well as keys go nowhere, the others to their places."""
    b = Batch(22, t, 64, 4, 2, 16, news, [n + 33 for n in news])
    there = b.table.copy()
    bad = {(0, (b.lens[0] - 1) // 16), (1, (b.lens[1] - news[1]) // 16)}
    for s, at in bad:
        b.table[s, at] = b.n_pages if page_no == "n_pages" else page_no
    kv = b.rng.standard_normal((2, b.n_tok, 2, 64)).astype(np.float32)
    with Dev(backend) as d:
        cache, batch = put_batch(d, b)
        backend.paged_store_dev(cache, batch, PagedRope(), 0, 0, 0, d.put(kv[0]), d.put(kv[1]), 128, 0, 0)
        got = d.get(cache.k, b.k), d.get(cache.v, b.v)
    b.table = there
    for is_v, old in ((False, b.k), (True, b.v)):
        want = old.copy()
        for row, s, p in b.tokens():
            for h in range(2):
                if (s, p // 16) not in bad:
                    want[b.at(s, p, h, is_v)] = encode(kv[int(is_v), row, h], t)
        assert np.array_equal(got[is_v], want)


@pytest.mark.parametrize("t", [T_F16, T_BF16, T_F32])
@pytest.mark.parametrize("hd", [80, 128, 256])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("news,lens", [([4], [24]), ([4], [2000]), ([90], [110]), ([90] + [9] * 130, [110] + [9] * 130)])
def test_attention_non_finite_values(backend, t, hd, value, news, lens):
    """Values that are not finite at a few new positions, in every type: the rows that see one get it in that value of theirs, the
    others and their other values are as they were."""
    b, clean = [Batch(112, t, hd, 4, 2, 16, news, lens) for _ in range(2)]
    marks = [(news[0] // 2, 1, 7), (news[0] - 1, 0, hd - 1), (news[0] // 3, 0, 0)]  # new token, K / V head, value
    for at, h, x in marks:
        b.v[b.at(0, lens[0] - news[0] + at, h, True)[x]] = encode(np.float32([value]), t)[0]
    scale = float(np.float32(hd**-0.5))
    o = run_attention(backend, b, scale=scale)
    want, tol, _ = attention(clean, clean.q, scale)
    hit = np.zeros(o.shape, bool)
    for at, h, x in marks:
        hit[at:news[0], 2 * h:2 * h + 2, x] = True
    assert not np.isfinite(o[hit]).any()
    assert (np.abs(o - want)[~hit] <= tol[~hit]).all()


# ---- starts that are no starts ----

LOW, HIGH = -2**31, 2**31 - 1


@pytest.mark.parametrize("tok,nan,fine", [
    ([0, LOW, 7, 9], range(7), range(7, 9)),
    ([5, LOW, 7, 9], range(5, 7), range(7, 9)),
    ([0, 3, LOW, HIGH], range(3, 9), ()),
    ([0, HIGH, HIGH, HIGH], range(9), ()),
    ([0, 4, 4, HIGH], range(4, 9), range(4)),
    ([HIGH, LOW, HIGH, LOW], (), ()),
    ([LOW, 2, 5, 9], range(2), range(2, 9)),
    ([-1, -1, LOW, LOW], (), ()),
    ([HIGH, HIGH, HIGH, HIGH], (), ()),
])
@pytest.mark.parametrize("heads", [1, 32])
def test_wild_starts(backend, tok, nan, fine, heads):
    """Starts at the ends of an int: the rows in 0 .. n_tok of a sequence that reaches out of it are NaN, those of others as ever, and
    nothing around them is written. (Rows in two sequences or before tok[0] hold anything.)"""
    b = Batch(120, T_F16, 64, heads, 1, 16, [3, 3, 3], [30, 31, 32])
    b.tok = np.array(tok, np.int32)
    n, pad, row = 9, 64, heads * 64
    with Dev(backend) as d:
        cache, batch = put_batch(d, b, max_len=40, max_tok=9)
        q = np.full((n + 2 * pad, row), 777.0, np.float32)
        q[pad:pad + n] = b.q.reshape(n, row)
        qd, od, kv = d.put(q), d.put(np.full_like(q, 777.0)), d.put(np.zeros((n, 64), np.float32))
        at = pad * row * 4
        for call in (lambda: backend.paged_attention_dev(cache, batch, PagedMask(0.125), heads, qd + at, row, od + at, row),
                     lambda: backend.paged_store_dev(cache, batch, PagedRope(), heads, qd + at, row, kv, kv, 64, od + at, row)):
            backend.h2d(od, np.full_like(q, 777.0))
            call()
            o = d.get(od, q)
            assert (o[:pad] == 777.0).all() and (o[pad + n:] == 777.0).all()
            o = o[pad:pad + n]
            assert np.isnan(o[list(nan)]).all() and np.isfinite(o[list(fine)]).all() and (o[list(fine)] != 777.0).all()


# ---- the largest batches and head counts ----

@pytest.mark.parametrize("most", [1, 9])
def test_most_sequences(backend, most):
    """65535 sequences, few of them with tokens; single tokens, and a prompt of the last one."""
    n_seq, page = 65535, 16
    b = Batch(130, T_F16, 64, 2, 1, page, [1, 1, 20 if most > 1 else 1], [5, 40, 50])
    at = [0, 30000, n_seq - 1]
    rows = np.zeros(n_seq, np.int32)
    rows[at] = b.news
    lens, table = np.zeros(n_seq, np.int32), np.full((n_seq, b.stride), -1, np.int32)
    lens[at], table[at] = b.lens, b.table
    qkv = b.rng.standard_normal((b.n_tok, 4, 64)).astype(np.float32)
    want, tol, _ = attention(b, b.q, 0.125)
    with Dev(backend) as d:
        cache, batch = put_batch(d, b)
        cache.table = d.put(table)
        batch = PagedBatch(d.put(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)), d.put(lens), n_seq=n_seq, n_tok=b.n_tok,
                           max_tok=max(b.news), max_len=50)
        q, o = d.put(b.q), d.put(np.full_like(b.q, 777.0))
        backend.paged_attention_dev(cache, batch, PagedMask(0.125), 2, q, 128, o, 128)
        got = d.get(o, b.q)
        assert (np.abs(got - want) <= tol).all()
        x = d.put(qkv)
        backend.paged_store_dev(cache, batch, PagedRope(), 2, x, 256, x + 512, x + 768, 256, o, 128)
        got, kc, vc = d.get(o, b.q), d.get(cache.k, b.k), d.get(cache.v, b.v)
    assert np.array_equal(got, qkv[:, :2])
    for t, s, pos in b.tokens():
        assert np.array_equal(kc[b.at(s, pos, 0, False)], encode(qkv[t, 2], T_F16))
        assert np.array_equal(vc[b.at(s, pos, 0, True)], encode(qkv[t, 3], T_F16))


@pytest.mark.parametrize("heads,kv_heads", [(4000, 1), (16383, 1), (4096, 4096), (8192, 4096)])
def test_most_heads(backend, heads, kv_heads):
    """One token of very many heads over one K / V head, and of very many K / V heads."""
    b = Batch(131, T_F16, 64, heads, kv_heads, 16, [1], [20])
    check_attention(backend, b)
    qkv = b.rng.standard_normal((1, heads + 2 * kv_heads, 64)).astype(np.float32)
    with Dev(backend) as d:
        cache, batch = put_batch(d, b)
        x, o, row = d.put(qkv), d.put(np.zeros((1, heads, 64), np.float32)), (heads + 2 * kv_heads) * 64
        backend.paged_store_dev(cache, batch, PagedRope(), heads, x, row, x + 256 * heads, x + 256 * (heads + kv_heads), row, o, heads * 64)
        got, kc, vc = d.get(o, qkv[:, :heads]), d.get(cache.k, b.k), d.get(cache.v, b.v)
    assert np.array_equal(got, qkv[:, :heads])
    for h in range(kv_heads):
        assert np.array_equal(kc[b.at(0, 19, h, False)], encode(qkv[0, heads + h], T_F16))
        assert np.array_equal(vc[b.at(0, 19, h, True)], encode(qkv[0, heads + kv_heads + h], T_F16))


@pytest.mark.parametrize("news", [1, 40])
def test_attention_rising_bias(backend, news):
    """Slopes below 0 raise what is far away; 0 leaves a head without a bias."""
    b = Batch(132, T_BF16, 64, 4, 2, 16, [news], [news + 300])
    check_attention(backend, b, slopes=np.float32([-0.25, 0.0, 0.125, -1.0]), prefix=np.array([200], np.int32))
    check_attention(backend, b, slopes=np.float32([-0.25, 0.0, 0.125, -1.0]), softcap=3.0)


@pytest.mark.parametrize("t", [T_F16, T_BF16, T_F32])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("news", [[4], [90], [20] * 260])
def test_infinite_key_of_a_later_row(backend, t, value, news):
    """A key that is not finite leaves the rows that do not see it as they are, bit for bit, also where it makes infinite scores."""
    b = Batch(133, t, 64, 4, 2, 16, news, [n + 40 for n in news])
    before = run_attention(backend, b)
    at = news[0] // 2
    b.k[b.at(0, 40 + at, 1, False)[3]] = encode(np.float32([value]), t)[0]
    after = run_attention(backend, b)
    same = np.ones(after.shape[:2], bool)
    same[at:news[0], 2:] = False
    assert np.array_equal(after[same].view(np.uint32), before[same].view(np.uint32))


@pytest.mark.parametrize("past", [0, 2000])
def test_most_sequences_and_one_prompt(backend, past):
    """One tile of a prompt beside 65535 sequences: the most rows of workgroups that a launch can have."""
    n_seq = 65535
    b = Batch(134, T_F16, 64, 1, 1, 256, [1, 20, 1], [5, 20 + past, 9])
    at = [1, 40000, n_seq - 1]
    rows, lens, table = np.zeros(n_seq, np.int32), np.zeros(n_seq, np.int32), np.full((n_seq, b.stride), -1, np.int32)
    rows[at], lens[at], table[at] = b.news, b.lens, b.table
    with Dev(backend) as d:
        cache, _ = put_batch(d, b)
        cache.table = d.put(table)
        batch = PagedBatch(d.put(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)), d.put(lens), n_seq=n_seq, n_tok=b.n_tok,
                           max_tok=20, max_len=20 + past)
        q, o = d.put(b.q), d.put(np.full_like(b.q, 777.0))
        backend.paged_attention_dev(cache, batch, PagedMask(0.125), 1, q, 64, o, 64)
        got = d.get(o, b.q)
    want, tol, _ = attention(b, b.q, 0.125)
    assert (np.abs(got - want) <= tol).all()
