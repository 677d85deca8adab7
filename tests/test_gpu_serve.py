"""The calls around the paged cache on the device against 64 bits on the host (tests/serve_ref.py): a batch's pages and rows, drafted
tokens checked, adapters of many requests, and all of them together with the cache's append and attention.

Whole numbers are equal; a logarithm is off by half a step of fp32 and 1e-10 for its 64-bit sum; adapters' outputs are within the bound
that serve_ref derives, and within 4 times what an fp32 form is off by."""
import numpy as np
import pytest
import serve_ref as R
from paged_ref import T_BF16, T_F16, T_F32, U32, Batch, attention, encode, of_vectors, store
from test_gpu_paged import Dev

from fastgguf_amd.backend import ERR_ARG, BackendError, Drafts, Lora, PagedBatch, PagedCache, PagedMask, PagedPool, PagedRope

pytestmark = pytest.mark.gpu


# ---- pages and rows of a batch ----

class DevPool:
    """A pool's arrays on the device, and the descriptors of its call."""

    def __init__(self, d, p, n_seq, n_tok, max_tok, max_len, in_place=False, maps=True):
        self.d, self.n, self.n_tok = d, n_seq, n_tok
        n = np.zeros(n_seq, np.int32)
        self.keep, self.add, self.held, self.free = d.put(n), d.put(n), d.put(p.held), d.put(p.free)
        self.held_out, self.free_out = (self.held, self.free) if in_place else (d.put(n), d.put(np.zeros(2, np.int32)))
        self.len = self.keep if in_place else d.put(n)
        self.table, self.queue, self.tok = d.put(p.table), d.put(p.queue), d.put(np.zeros(n_seq + 1, np.int32))
        rows = np.full(n_tok, 77, np.int64)
        self.maps = [d.put(rows.astype(np.int32)), d.put(rows.astype(np.int32)), d.put(rows)] if maps else [0, 0, 0]
        self.cache = PagedCache(T_F16, 0, 0, self.table, n_pages=p.n_pages, page=p.page, table_stride=p.stride, n_head_kv=1, hd=64)
        self.batch = PagedBatch(self.tok, self.len, n_seq=n_seq, n_tok=n_tok, max_tok=max_tok, max_len=max_len)
        self.pool = PagedPool(self.keep, self.add, self.held, self.held_out, self.queue, self.free, self.free_out, seq=self.maps[0],
                              pos=self.maps[1], slot=self.maps[2])

    def ask(self, keep, add):
        self.d.be.h2d(self.keep, np.asarray(keep, np.int32))
        self.d.be.h2d(self.add, np.asarray(add, np.int32))

    def check(self, p, want, maps=True):
        """Against the host's pool and outputs after the same call."""
        tok, length, seq, pos, slot = want
        get = self.d.get
        assert np.array_equal(get(self.tok, tok), tok)
        assert np.array_equal(get(self.len, length), length)
        assert np.array_equal(get(self.held_out, p.held), p.held)
        assert np.array_equal(get(self.free_out, p.free), p.free)
        assert np.array_equal(get(self.table, p.table), p.table)
        assert np.array_equal(get(self.queue, p.queue), p.queue)
        if maps:
            for at, w in zip(self.maps, (seq, pos, slot)):
                assert np.array_equal(get(at, w), w)


RESERVES = [  # sequences, page, positions before, new tokens up to, free pages, rows
    (1, 16, (0, 1), 1, 1, 1),
    (1, 16, (4095, 4096), 1, 3, 1),
    (1, 64, (0, 1), 5000, 90, 5000),
    (2, 256, (0, 600), 300, 2, 700),
    (31, 16, (0, 400), 6, 10, 200),
    (64, 32, (1, 2000), 1, 3, 64),
    (65, 16, (0, 50), 40, 60, 1000),
    (300, 16, (0, 900), 9, 400, 1500),
    (1024, 16, (0, 300), 3, 2000, 2048),
    (1025, 128, (0, 1000), 5, 100, 3001),
    (3000, 16, (0, 120), 30, 1500, 9000),
    (9000, 16, (0, 60), 4, 30000, 20011),
    (65535, 16, (0, 20), 2, 9000, 70000),
]


def requests(r, p, most):
    """What is kept and added: some sequences ended, some lost drafts, some have nothing new."""
    n = len(p.len)
    keep = np.where(r.random(n) < 0.15, 0, np.maximum(0, p.len - r.integers(0, 4, n)))
    return keep, np.where(r.random(n) < 0.1, 0, r.integers(0 if most > 1 else 1, most + 1, n))


@pytest.mark.parametrize("form", ["apart", "in place", "without maps"])
@pytest.mark.parametrize("i", range(len(RESERVES)))
def test_reserve(backend, i, form):
    """Three steps, one after the other."""
    n, page, lens, most, free, rows = RESERVES[i]
    r = np.random.default_rng(i)
    stride = -(-(lens[1] + 3 * most) // page)
    p = R.Pool(i, n, page, r.integers(*lens, n), free, stride)
    with Dev(backend) as d:
        dev = DevPool(d, p, n, rows, most, stride * page - 3, form == "in place", form != "without maps")
        for _ in range(3):
            keep, add = requests(r, p, most)
            dev.ask(keep, add)
            backend.paged_reserve_dev(dev.cache, dev.batch, dev.pool)
            want = R.reserve(p, keep, add, rows, most, stride * page - 3)
            dev.check(p, want, form != "without maps")
            if form != "in place":
                backend.h2d(dev.held, p.held)
                backend.h2d(dev.free, p.free)
            p.len = want[1]


MANY = [  # sequences, page, positions before, new tokens up to, free pages, rows, share of sequences that end
    (250, 16, (10, 9000), 60, 90, 11000, 0.0),     # more than 4096 rows: several workgroups; a ring that runs out
    (250, 16, (10, 9000), 60, 0, 11000, 0.004),    # no free pages: those of the same call
    (9, 64, (0, 1), 4000, 400, 20000, 0.1),
    (1024, 16, (0, 300), 12, 800, 5000, 0.1),      # rows run out
    (1000, 32, (0, 300), 60, 40, 25001, 0.3),
    (600, 16, (1000, 9000), 2, 20, 900, 0.0),      # few rows, more than 2^17 pages
    (600, 16, (1000, 9000), 40, 3, 24001, 0.002),
]


@pytest.mark.parametrize("form", ["apart", "in place", "without maps"])
@pytest.mark.parametrize("i", range(len(MANY)))
def test_reserve_by_many(backend, i, form):
    """Up to 1024 sequences whose rows or pages take several workgroups: one launch where outputs are apart from inputs, two where they are not."""
    n, page, lens, most, free, rows, ends = MANY[i]
    r = np.random.default_rng(300 + i)
    stride = -(-(lens[1] + 3 * most) // page)
    p = R.Pool(300 + i, n, page, r.integers(*lens, n), free, stride)
    assert rows > 4096 or min(p.n_pages, n * stride) > 1 << 17
    short = False
    with Dev(backend) as d:
        dev = DevPool(d, p, n, rows, most, stride * page, form == "in place", form != "without maps")
        for _ in range(3):
            keep = np.where(r.random(n) < ends, 0, np.maximum(0, p.len - r.integers(0, 4, n)))
            add = r.integers(0, most + 1, n)
            dev.ask(keep, add)
            backend.paged_reserve_dev(dev.cache, dev.batch, dev.pool)
            want = R.reserve(p, keep, add, rows, most, stride * page)
            short |= bool((np.diff(want[0]) < add).any())
            dev.check(p, want, form != "without maps")
            if form != "in place":
                backend.h2d(dev.held, p.held)
                backend.h2d(dev.free, p.free)
            p.len = want[1]
    assert short or rows < 4096  # where rows or pages are many, some find none


def test_reserve_again(backend):
    """The same inputs give the same outputs again, also where pages moved."""
    r = np.random.default_rng(5)
    p = R.Pool(5, 40, 16, r.integers(0, 300, 40), 30, 40)
    keep, add = requests(r, p, 60)
    with Dev(backend) as d:
        dev = DevPool(d, p, 40, 900, 60, 600)
        dev.ask(keep, add)
        want = R.reserve(p, keep, add, 900, 60, 600)
        for _ in range(3):
            backend.paged_reserve_dev(dev.cache, dev.batch, dev.pool)
            dev.check(p, want)


@pytest.mark.parametrize("what", ["keep below 0", "keep past its pages", "held below 0", "held past the table", "add below 0", "add past max_tok", "past max_len",
                                  "past the table", "largest numbers"])
def test_reserve_bad_sequences(backend, what):
    """A sequence whose numbers mean nothing gets nothing, and the others what they would."""
    r = np.random.default_rng(6)
    p = R.Pool(6, 9, 16, [20, 33, 5, 64, 100, 16, 0, 48, 17], 20, 8)
    keep, add = p.len.copy(), np.array([3, 1, 0, 9, 2, 1, 7, 0, 5])
    max_len = 120
    if what == "keep below 0":
        keep[[0, 4]] = -1, -2**31
    elif what == "keep past its pages":
        keep[[1, 4]] = 49, 2**31 - 1
    elif what == "held below 0":
        p.held[[2, 3]] = -1, -2**31
    elif what == "held past the table":
        p.held[[2, 3]] = 9, 2**31 - 1
    elif what == "add below 0":
        add[[0, 3]] = -1, -2**31
    elif what == "add past max_tok":
        add[[0, 3]] = 13, 2**31 - 1
    elif what == "past max_len":
        add[4] = 12
        max_len = 111
    elif what == "past the table":
        add[4] = 12
        p.stride, p.table = 6, np.ascontiguousarray(p.table[:, :6])
        p.held[4], keep[4] = 6, 96
        max_len = 2**31 - 1
    else:
        keep[:3], add[3:6], p.held[6:] = 2**31 - 1, 2**31 - 1, 2**31 - 1
    with Dev(backend) as d:
        dev = DevPool(d, p, 9, 40, 12, max_len)
        dev.ask(keep, add)
        backend.paged_reserve_dev(dev.cache, dev.batch, dev.pool)
        dev.check(p, R.reserve(p, keep, add, 40, 12, max_len))


@pytest.mark.parametrize("free", [(-1, 5), (2**31 - 1, 5), (3, -1), (3, 10**6), (3, 0)])
def test_reserve_bad_ring(backend, free):
    p = R.Pool(7, 4, 16, [20, 33, 5, 64], 6, 10)
    p.free[:] = free
    keep, add = [20, 0, 5, 64], [1, 30, 20, 1]
    with Dev(backend) as d:
        dev = DevPool(d, p, 4, 60, 30, 160)
        dev.ask(keep, add)
        backend.paged_reserve_dev(dev.cache, dev.batch, dev.pool)
        dev.check(p, R.reserve(p, keep, add, 60, 30, 160))


@pytest.mark.parametrize("first, tok", [(512, [0, 0, 0, 0, 0]), (0, [0, 0, 1, 2, 3]), (160, [0, 160, 161, 162, 163]), (161, [0, 0, 1, 2, 3])])
def test_reserve_rows_of_one_that_waits(backend, first, tok):
    """A prompt without pages keeps the rows it asked for from those behind it, which need no page."""
    p = R.Pool(1, 4, 16, [0, 5, 20, 35], 10, 64)
    with Dev(backend) as d:
        dev = DevPool(d, p, 4, 512, 512, 1024, True)
        dev.ask(p.len, [first, 1, 1, 1])
        backend.paged_reserve_dev(dev.cache, dev.batch, dev.pool)
        want = R.reserve(p, p.len, [first, 1, 1, 1], 512, 512, 1024)
        assert want[0].tolist() == tok
        dev.check(p, want)


def test_reserve_full_ring(backend):
    """Pages given back to a ring that has them already: nothing is written past it, and its number stays that of the pages."""
    p = R.Pool(8, 3, 16, [40, 16, 90], 6, 10)
    p.free[1] = p.n_pages
    p.queue[:] = np.arange(p.n_pages)
    with Dev(backend) as d:
        dev = DevPool(d, p, 3, 10, 10, 160)
        dev.ask([0, 16, 17], [0, 1, 0])
        backend.paged_reserve_dev(dev.cache, dev.batch, dev.pool)
        dev.check(p, R.reserve(p, [0, 16, 17], [0, 1, 0], 10, 10, 160))


def test_reserve_bad_pages(backend):
    """What stands in the ring is handed out as it is; a row there has no slot."""
    p = R.Pool(9, 2, 16, [16, 30], 6, 10)
    p.queue[(p.first + np.arange(2)) % p.n_pages] = p.n_pages, -5
    with Dev(backend) as d:
        dev = DevPool(d, p, 2, 50, 40, 160)
        dev.ask([16, 30], [20, 20])
        backend.paged_reserve_dev(dev.cache, dev.batch, dev.pool)
        want = R.reserve(p, [16, 30], [20, 20], 50, 40, 160)
        assert (want[4][:40] == -1).any() and (want[4][:40] >= 0).any()
        dev.check(p, want)


def test_reserve_captured(backend):
    """A recorded step, its state in place, replayed among eager ones of another size."""
    r = np.random.default_rng(10)
    p, other = R.Pool(10, 50, 16, r.integers(0, 300, 50), 300, 40), R.Pool(11, 2000, 16, r.integers(0, 60, 2000), 900, 40)
    with Dev(backend) as d:
        dev, wide = DevPool(d, p, 50, 200, 6, 640, True), DevPool(d, other, 2000, 9000, 6, 640, True)
        dev.ask(p.len, np.zeros(50))
        backend.paged_reserve_dev(dev.cache, dev.batch, dev.pool)
        R.reserve(p, p.len, np.zeros(50), 200, 6, 640)
        backend.graph_begin()
        backend.paged_reserve_dev(dev.cache, dev.batch, dev.pool)
        g = backend.graph_end()
        try:
            for step in range(5):
                keep, add = requests(r, p, 6)
                dev.ask(keep, add)
                backend.graph_launch(g)
                if step % 2:
                    k2, a2 = requests(r, other, 6)
                    wide.ask(k2, a2)
                    backend.paged_reserve_dev(wide.cache, wide.batch, wide.pool)
                    want2 = R.reserve(other, k2, a2, 9000, 6, 640)
                    wide.check(other, want2)
                    other.len = want2[1]
                want = R.reserve(p, keep, add, 200, 6, 640)
                dev.check(p, want)
                p.len = want[1]
        finally:
            backend.graph_destroy(g)


# ---- drafted tokens ----

class Case:
    """Sequences of rows[s] rows, logits as a language model has them, drafts of which most are likely."""

    def __init__(self, seed, rows, vocab, drafter, pad=(0, 0), extra=0, temps=(1.0, 0.7, 0.0, 1.3), forbidden=0.02):
        r = self.r = np.random.default_rng(seed)
        self.vocab, self.ld, self.n = vocab, vocab + extra, len(rows)
        self.tok = (pad[0] + np.concatenate([[0], np.cumsum(rows)])).astype(np.int32)
        self.n_tok = int(self.tok[-1]) + pad[1]
        self.max_tok = max(list(rows) + [1])
        x = 2 * r.standard_normal((self.n_tok, self.ld))
        for t in range(self.n_tok):
            x[t, r.integers(0, vocab, 6)] = 6 + 2 * r.standard_normal(6)
        x[:, :vocab][:, r.random(vocab) < forbidden] = -np.inf
        x[:, r.integers(0, vocab)] = 1.0  # one word at least
        self.logits = x.astype(np.float32)
        self.logits[:, vocab:] = np.nan
        self.temp = np.array([temps[s % len(temps)] for s in range(self.n)], np.float32)
        heat = np.ones(self.n_tok)
        for s in range(self.n):
            heat[self.tok[s]:self.tok[s + 1]] = self.temp[s] or 1.0
        self.u, self.v = r.random(self.n_tok).astype(np.float32), r.random(self.n).astype(np.float32)
        self.q = self.q_lse = None
        source = self.logits[:, :vocab]
        if drafter:
            self.q = (x + 0.7 * r.standard_normal(x.shape)).astype(np.float32)
            self.q[:, vocab:] = np.nan
            self.q_lse = np.array([R.lse_of(self.q[t, :vocab], heat[t]) for t in range(self.n_tok)]).astype(np.float32)
            source = self.q[:, :vocab]
        guess = np.array([np.argmax(source[t] / heat[t] + r.gumbel(size=vocab)) for t in range(self.n_tok)])
        self.tokens = np.roll(guess, 1).astype(np.int32)
        self.len = (50 + np.arange(self.n)).astype(np.int32)

    def want(self):
        return R.verify(self.logits, self.tok, self.tokens, self.u, self.v, self.vocab, self.max_tok, self.temp, self.q, self.q_lse, self.len)

    def put(self, d):
        q = dict(q=d.put(self.q), q_lse=d.put(self.q_lse), ldq=self.ld) if self.q is not None else {}
        return Drafts(d.put(self.logits), d.put(self.tok), d.put(self.tokens), d.put(self.u), d.put(self.v), n_seq=self.n, n_tok=self.n_tok,
                      max_tok=self.max_tok, vocab=self.vocab, ld=self.ld, len=d.put(self.len), **q,
                      **(dict(temp=d.put(self.temp)) if self.temp is not None else {}))

    def outputs(self, d):
        n = np.full(self.n, 77, np.int32)
        return [d.put(n), d.put(n), d.put(n), d.put(np.full(self.n_tok, 77.0, np.float32))]

    def check(self, d, out):
        n_ok, nxt, keep, lse = self.want()
        got = [d.get(out[0], n_ok), d.get(out[1], nxt), d.get(out[2], keep)]
        for g, w in zip(got, (n_ok, nxt, keep)):
            assert np.array_equal(g, w), (np.nonzero(g != w)[0][:5], g[g != w][:5], w[g != w][:5])
        l = d.get(out[3], np.zeros(self.n_tok, np.float32))
        for s in range(self.n):
            b, e = int(self.tok[s]), int(self.tok[s + 1])
            if e <= b or e - b > self.max_tok:
                continue
            x, w = l[b:e].astype(np.float64), lse[b:e]
            fine = np.isfinite(w)
            assert np.array_equal(np.isnan(x), np.isnan(w)) and np.array_equal(x[~fine & ~np.isnan(w)], w[~fine & ~np.isnan(w)])
            assert (np.abs(x - w)[fine] <= U32 * np.abs(w[fine]) + 1e-10).all()
        assert (l[:self.tok[0]] == 77.0).all() and (l[self.tok[-1]:] == 77.0).all()
        return n_ok, nxt

    def run(self, be):
        with Dev(be) as d:
            out = self.outputs(d)
            be.draft_verify_dev(self.put(d), out[0], out[1], keep_dev=out[2], lse_dev=out[3])
            return self.check(d, out)


VERIFIES = [  # rows of each sequence, vocabulary, rows before and behind, columns behind
    ([1], 1, (0, 0), 0),
    ([3], 2, (0, 0), 0),
    ([1], 1000, (0, 0), 0),
    ([6], 32000, (0, 0), 0),
    ([1, 4, 0, 2, 7], 1023, (1, 2), 1),
    ([1] * 70, 777, (0, 3), 0),
    ([5, 1, 3] * 9, 4097, (2, 0), 3),
    ([9, 2], 50021, (0, 0), 0),
    ([2, 6], 131073, (0, 1), 0),
    ([3], 262147, (0, 0), 5),
    ([17, 33], 300, (0, 0), 0),
    ([4] * 300, 2050, (0, 0), 0),
]


@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("i", range(len(VERIFIES)))
def test_verify(backend, i, drafter):
    rows, vocab, pad, extra = VERIFIES[i]
    c = Case(100 + i, rows, vocab, drafter, pad, extra)
    n_ok, _ = c.run(backend)
    if sum(rows) > 40 and max(rows) > 1:  # some accepted, some rejected
        assert 0 < n_ok.sum() < sum(max(0, n - 1) for n in rows)


@pytest.mark.parametrize("drafter", [False, True])
def test_verify_many_rows(backend, drafter):
    """More rows than fill the device: each part of one takes two blocks, each workgroup two parts."""
    c = Case(113, [6] * 190 + [1, 0, 11], 9001, drafter, (1, 2), 3)
    n_ok, _ = c.run(backend)
    assert 0 < n_ok.sum() < c.n_tok - c.n


@pytest.mark.parametrize("drafter", [False, True])
def test_verify_padded(backend, drafter):
    """Many rows of no sequence before the first and behind the last."""
    Case(115, [3, 1, 4], 5000, drafter, (130, 600)).run(backend)


@pytest.mark.parametrize("drafter", [False, True])
def test_verify_widest(backend, drafter):
    """2^24 words, the most that a row may have: parts of 262144."""
    c = Case(114, [2], 1 << 24, drafter, temps=(30.0,))
    c.run(backend)


def test_verify_long_rows(backend):
    """A vocabulary whose parts take several blocks of a workgroup."""
    c = Case(20, [2], 1000003, True)
    c.run(backend)


@pytest.mark.parametrize("temp", [1e-30, 1e-3, 30.0, 1e30, float("inf"), 0.0, -1.0, float("nan")])
@pytest.mark.parametrize("drafter", [False, True])
def test_verify_temperatures(backend, temp, drafter):
    Case(21, [4, 1, 3], 5000, drafter, temps=(temp,)).run(backend)


def test_verify_without_temperatures(backend):
    c = Case(22, [4, 1, 3], 5000, True, temps=(1.0,))
    with Dev(backend) as d:
        x = c.put(d)
        x.temp, x.len = None, None
        out = c.outputs(d)
        backend.draft_verify_dev(x, out[0], out[1])
        n_ok, nxt, _, _ = c.want()
        assert np.array_equal(d.get(out[0], n_ok), n_ok) and np.array_equal(d.get(out[1], nxt), nxt)
        assert (d.get(out[2], n_ok) == 77).all() and (d.get(out[3], c.u) == 77.0).all()


def even(rows, vocab, **kw):
    """Rows whose words are all as likely: probabilities and sums are exact."""
    c = Case(23, rows, vocab, False, temps=(1.0,), **kw)
    c.logits[:, :vocab] = 3.0
    return c


def test_verify_borders(backend):
    """u q(d) = p(d) rejects; a running sum equal to v times the whole does not pass it."""
    c = even([2] * 6, 8)
    c.tokens[:] = 5
    c.u[0::2] = [0.125, np.nextafter(np.float32(0.125), np.float32(0)), 0.0, 1.0, 0.125, 0.9]
    c.v[:] = [0.0, 0.25, 0.25, 0.0, np.nextafter(np.float32(1), np.float32(0)), 4 / 7]
    n_ok, nxt = c.run(backend)
    assert n_ok.tolist() == [0, 1, 1, 0, 0, 0]
    # without word 5: 7 words; v = 0 the first, 0.25 of 8 the third
    assert nxt.tolist()[:5] == [0, 2, 2, 0, 7]


@pytest.mark.parametrize("vocab", [1, 64, 1000, 4096, 131072])
def test_verify_every_word(backend, vocab):
    """v in the middle of each of 64 words' parts, among them the first and the last word."""
    words = np.unique(np.linspace(0, vocab - 1, 64).astype(np.int64))
    c = even([1] * len(words), vocab)
    c.v[:] = ((words + 0.5) / vocab).astype(np.float32)
    _, nxt = c.run(backend)
    assert np.abs(nxt - words).max() <= vocab * U32 + 0.5


def test_verify_largest(backend):
    """Temperature 0: the lowest of equal largest words, wherever they stand."""
    r = np.random.default_rng(24)
    c = Case(24, [3] * 40, 9000, False, temps=(0.0,))
    for t in range(c.n_tok):
        c.logits[t, r.integers(0, 9000, 5)] = 50.0
    best = np.argmax(c.logits[:, :9000], 1)
    c.tokens[1:] = best[:-1]
    c.tokens[7::9] += 1
    n_ok, nxt = c.run(backend)
    assert n_ok.max() == 2 and n_ok.min() < 2
    assert (c.logits[np.array([c.tok[s] + n_ok[s] for s in range(40)]), nxt] == 50.0).all()


@pytest.mark.parametrize("drafter", [False, True])
def test_verify_special_rows(backend, drafter):
    """NaN, infinities, rows with no word, drafts that are no words or have no probability: defined, and no other sequence's matter."""
    c = Case(25, [3] * 14, 3001, drafter, temps=(1.0, 0.0))
    x = c.logits
    x[0, 100], x[4, 3000], x[7, 0] = np.nan, np.inf, np.nan
    x[9, :3001], x[13, :3001] = -np.inf, -np.inf
    x[15, 5], x[15, 6] = np.nan, np.inf
    x[18, :3001] = -np.inf
    x[18, 77] = -2.0                       # one word
    c.tokens[19] = 77                      # and it is the draft: nothing would be left
    x[24, :3001], x[27, :3001] = 3e38, -3e38
    c.tokens[22], c.tokens[25], c.tokens[31], c.tokens[34] = -1, 3001, 2**31 - 1, -2**31
    x[36, 11] = -np.inf
    c.tokens[37] = 11                      # a draft that cannot be
    if drafter:
        c.q[30, 5], c.q[33, :50], c.q_lse[39] = np.nan, np.inf, np.nan
        c.q[36, :3001] = -np.inf
    c.u[18] = 1.0
    n_ok, nxt = c.run(backend)
    assert nxt[0] == -1 and n_ok[0] == 0


def test_verify_all_rejected_by_u(backend):
    """u of 1 and more, where p is all on the draft: what is left is nothing, and p decides."""
    c = Case(26, [2, 2], 500, False, temps=(1.0,))
    c.logits[:] = -np.inf
    c.logits[:, 321] = 1.0
    c.tokens[:] = 321
    c.u[:] = 1.0, 0.5, 0.999, 0.5
    n_ok, nxt = c.run(backend)
    assert n_ok.tolist() == [0, 1] and nxt.tolist() == [321, 321]


@pytest.mark.parametrize("tok", [[0, 3, 2, 6], [-2, 1, 3, 6], [0, 2, 5, 2**31 - 1], [-2**31, 2, 4, 6], [6, 6, 6, 6], [0, 0, 0, 6]])
def test_verify_wild_starts(backend, tok):
    """Row starts that mean nothing: sequences outside the buffers have no token, and nothing is read there."""
    c = Case(27, [2, 2, 2], 900, True)
    c.tok = np.array(tok, np.int32)
    c.max_tok = 4
    with Dev(backend) as d:
        out = c.outputs(d)
        backend.draft_verify_dev(c.put(d), out[0], out[1], keep_dev=out[2], lse_dev=out[3])
        n_ok, nxt, keep, _ = c.want()
        falls = [tok[s + 1] < tok[s] for s in range(3)]
        for s in range(3):
            if not any(falls):
                assert d.get(out[0], n_ok)[s] == n_ok[s] and d.get(out[1], nxt)[s] == nxt[s] and d.get(out[2], keep)[s] == keep[s]
            elif falls[s]:
                assert d.get(out[0], n_ok)[s] == 0 and d.get(out[1], nxt)[s] == -1


def test_verify_keep_in_place(backend):
    c = Case(28, [4, 0, 1, 6, 2], 700, False)
    c.len[:] = 9, 5, 1, 2, 0
    with Dev(backend) as d:
        x = c.put(d)
        out = c.outputs(d)
        out[2] = x.len
        backend.draft_verify_dev(x, out[0], out[1], keep_dev=out[2], lse_dev=out[3])
        c.check(d, out)


def test_verify_captured(backend):
    """Two recorded calls of different sizes share the scratch with eager ones: every replay gives what it did."""
    a, b = Case(29, [3, 1, 4], 9001, True), Case(30, [1] * 40, 3000, False)
    wide = Case(31, [6] * 30, 20000, True)
    with Dev(backend) as d:
        xa, xb, oa, ob = a.put(d), b.put(d), a.outputs(d), b.outputs(d)
        call = [lambda: backend.draft_verify_dev(xa, oa[0], oa[1], keep_dev=oa[2], lse_dev=oa[3]),
                lambda: backend.draft_verify_dev(xb, ob[0], ob[1], keep_dev=ob[2], lse_dev=ob[3])]
        graphs = []
        try:
            for f in call:
                f()
                backend.graph_begin()
                f()
                graphs.append(backend.graph_end())
            wide.run(backend)  # the scratch grows
            for _ in range(4):
                for c, o, g in ((a, oa, graphs[0]), (b, ob, graphs[1])):
                    c.u[:], c.v[:] = c.r.random(c.n_tok), c.r.random(c.n)
                    x = xa if c is a else xb
                    backend.h2d(x.u, c.u)
                    backend.h2d(x.v, c.v)
                    backend.graph_launch(g)
                    c.check(d, o)
                call[1]()
                b.check(d, ob)
        finally:
            for g in graphs:
                backend.graph_destroy(g)


# ---- adapters ----

def run_lora(be, ad, tok, ids, x, y_in, pad=0, form="apart", n_tok=None):
    """y of a call whose rows are `pad` values apart; rows of no sequence are 777 before it (y_in's in place)."""
    n_tok = len(x) if n_tok is None else n_tok
    with Dev(be) as d:
        wx, wi = np.full((n_tok, ad.cols + pad), 3.0, np.float32), np.full((n_tok, ad.rows + pad), 5.0, np.float32)
        wx[:, :ad.cols], wi[:, :ad.rows] = x, y_in
        before = np.full((n_tok, ad.rows + 2 * pad), 777.0, np.float32)
        set_ = Lora(ad.type, d.put(ad.a), d.put(ad.b), n_adapter=ad.n, max_rank=ad.max_rank, cols=ad.cols, rows=ad.rows, rank=d.put(ad.rank),
                    scale=d.put(ad.scale))
        xd, yi, tk, idd = d.put(wx), d.put(wi), d.put(np.asarray(tok, np.int32)), d.put(np.asarray(ids, np.int32))
        if form == "in place":
            be.lora_dev(set_, tk, idd, len(ids), n_tok, xd, ad.cols + pad, yi, ad.rows + pad, y_in_dev=yi, ldyi=ad.rows + pad)
            got, out = d.get(yi, wi), wi
        else:
            y = d.put(before)
            given = dict(y_in_dev=yi, ldyi=ad.rows + pad) if form == "apart" else {}
            be.lora_dev(set_, tk, idd, len(ids), n_tok, xd, ad.cols + pad, y, ad.rows + 2 * pad, **given)
            got, out = d.get(y, before), before
    assert np.array_equal(got[:, ad.rows:], out[:, ad.rows:])
    return got[:, :ad.rows], out[:, :ad.rows]


def check_lora(be, ad, tok, ids, x, y_in, **kw):
    if kw.get("form") == "alone":
        y_in = np.zeros_like(y_in)
    got, before = run_lora(be, ad, tok, ids, x, y_in, **kw)
    want, tol, mine = R.lora(ad, tok, ids, x, y_in)
    assert np.array_equal(got[~mine], before[~mine])
    bad = mine & np.isnan(want).any(1)
    assert np.isnan(got[bad]).all()
    fine = mine & ~bad
    off = np.abs(got[fine] - want[fine])
    assert (off <= tol[fine]).all(), (float((off - tol[fine]).max()), np.argwhere(off > tol[fine])[:4])
    if fine.any():
        delta = want[fine] - y_in[fine]
        moved = np.abs(delta).max(1) > 0
        if moved.any():  # y_in 0: the adapters' part alone
            plain = R.lora32(ad, tok, ids, x, y_in)[fine][moved]
            assert of_vectors(got[fine][moved], want[fine][moved]) <= 4 * of_vectors(plain, want[fine][moved]) + 2.0**-22


def lora_case(seed, t, n, max_rank, cols, rows, news, ids, ranks=None, pad=(0, 0)):
    r = np.random.default_rng(seed)
    ad = R.Adapters(seed, t, n, max_rank, cols, rows, ranks)
    tok = pad[0] + np.concatenate([[0], np.cumsum(news)])
    n_tok = int(tok[-1]) + pad[1]
    x = r.standard_normal((n_tok, cols)).astype(np.float32)
    x[:, r.integers(0, cols, 2)] *= 30
    return ad, tok, ids, x, r.standard_normal((n_tok, rows)).astype(np.float32)


LORAS = [  # adapters, max_rank, cols, rows, new tokens, ids, ranks, rows before and behind
    (1, 8, 8, 1, [1], [0], None, (0, 0)),
    (2, 16, 128, 64, [1], [1], None, (0, 0)),
    (3, 16, 4096, 300, [1, 1, 1], [2, 0, 2], [16, 16, 5], (0, 0)),
    (4, 64, 520, 1001, [1] * 40, [0, 1, 2, 3, -1] * 8, [64, 1, 33, 17], (1, 2)),
    (2, 8, 136, 70, [3, 0, 1, 16, 2, 17], [0, 1, -1, 1, 1, 0], [8, 3], (0, 5)),
    (3, 32, 1000, 515, [100, 37, 250, 1], [0, 2, 1, 1], [32, 31, 9], (3, 0)),
    (2, 128, 256, 384, [65, 63, 130], [1, 0, 0], [128, 100], (0, 0)),
    (2, 512, 512, 256, [20, 5], [1, 0], [512, 300], (0, 1)),
    (5, 24, 264, 2049, [2] * 33, [s % 5 for s in range(33)], [24, 0, 7, 24, 20], (0, 0)),
    (2, 16, 2048, 256, [700], [1], None, (0, 0)),
    (9, 16, 96, 130, [5, 70, 3, 1, 64, 128, 2], [8, 8, 8, 2, 2, -1, 8], None, (7, 9)),
    (3, 8, 64, 8, [0, 0, 1, 0, 0], [9, -5, 1, 2, 2], None, (0, 0)),
]


@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("i", range(len(LORAS)))
def test_lora(backend, i, t):
    n, max_rank, cols, rows, news, ids, ranks, pad = LORAS[i]
    form = ["apart", "in place", "alone"][i % 3]
    check_lora(backend, *lora_case(40 + i, t, n, max_rank, cols, rows, news, ids, ranks, pad), pad=i % 4, form=form)


PROMPTS = [  # the same, of prompts long enough to have workgroups of 64 rows
    (3, 8, 200, 130, [700, 1, 1, 1, 1, 400], [0, 1, 2, 0, 1, 2], [8, 3, 5], (3, 9)),
    (2, 32, 1000, 515, [600, 499], [1, 0], [32, 9], (0, 0)),
    (3, 64, 136, 70, [301] * 4, [0, 1, 2, -1], [64, 33, 1], (0, 2)),
    (2, 128, 320, 384, [513, 0, 600], [1, 7, 0], [128, 100], (1, 0)),
    (2, 200, 264, 65, [1025, 40], [1, 0], [200, 140], (0, 0)),
    (1, 512, 72, 64, [1100], [0], None, (0, 0)),
    (2, 16, 2048, 3, [1500, 20], [0, 1], [16, 10], (0, 0)),
    (1, 24, 8, 1, [2000], [0], [17], (5, 0)),
    (4, 16, 64, 200, [16] * 70, [s % 6 - 1 for s in range(70)], [16, 0, 2, 11], (0, 0)),
    (2, 40, 448, 1030, [64, 63, 65, 1000], [0, 1, 1, 0], [40, 24], (0, 0)),
]


@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("i", range(len(PROMPTS)))
def test_lora_prompts(backend, i, t):
    n, max_rank, cols, rows, news, ids, ranks, pad = PROMPTS[i]
    form = ["in place", "apart", "alone"][i % 3]
    check_lora(backend, *lora_case(140 + i, t, n, max_rank, cols, rows, news, ids, ranks, pad), pad=i % 4, form=form)


@pytest.mark.parametrize("news", [[4, 1, 1, 1, 1, 1100], [4, 1, 1, 1, 1, 300], [4, 1, 1, 1, 1, 1] * 300])
@pytest.mark.parametrize("rank", [1, 2, 4, 9])
def test_lora_beside_nan(backend, news, rank):
    """A tile's rows whose results are NaN leave nothing to others of the same tile, whose ranks end inside the next eight."""
    ids = [s % 6 for s in range(len(news))]
    ad, tok, ids, x, y_in = lora_case(160 + rank, T_F16, 6, 64, 128, 128, news, ids, [64, 0, 64, rank, rank, rank])
    spoilt = np.isin(np.repeat(ids, news), (0, 2))
    x[spoilt, 3] = np.nan
    got, _ = run_lora(backend, ad, tok, ids, x, y_in)
    want, tol, _ = R.lora(ad, tok, ids, np.where(np.isfinite(x), x, 0).astype(np.float32), y_in)
    assert np.isnan(got[spoilt]).all()
    assert (np.abs(got - want) <= tol)[~spoilt].all()


MIXED = [  # adapters, max_rank, cols, rows, new tokens: more runs in a tile than workgroups for them
    (40, 16, 72, 70, [1] * 2000),
    (40, 24, 64, 130, [1, 2, 1, 0, 1] * 500),
    (9, 8, 64, 66, [1] * 33000),                   # a workgroup for all of a tile's runs
    (24, 64, 264, 200, [4100] + [1] * 63),         # a prompt beside single tokens
    (24, 16, 136, 130, [1] * 40 + [1500] + [1] * 23 + [600]),
    (30, 32, 200, 70, [512] + [1] * 255),
    (5, 136, 72, 70, [300] + [1] * 90),
]


@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("i", range(len(MIXED)))
def test_lora_mixed(backend, i, t):
    """Tiles of many adapters, without one, with ids and ranks that mean nothing among them."""
    n, max_rank, cols, rows, news = MIXED[i]
    r = np.random.default_rng(180 + i)
    ids = r.integers(-2, n, len(news)).tolist()
    ranks = r.integers(0, max_rank + 1, n)
    ranks[:2] = max_rank, max_rank + 1
    check_lora(backend, *lora_case(180 + i, t, n, max_rank, cols, rows, news, ids, ranks.tolist(), (i % 3, 5)), pad=i % 4, form=["apart", "in place", "alone"][i % 3])


@pytest.mark.parametrize("news, few, rows", [([1] * 63 + [1500], 63, 70), ([3, 1, 0, 4] * 10 + [600, 70], 40, 130)])
def test_lora_in_two_calls(backend, news, few, rows):
    """Single tokens first, prompts behind them, a call for each over the same starts: together what one call gives."""
    ad, tok, ids, x, y_in = lora_case(190, T_BF16, 6, 16, 136, rows, news, [s % 7 - 1 for s in range(len(news))], [16, 3, 0, 9, 16, 5], (0, 4))
    want, tol, mine = R.lora(ad, tok, ids, x, y_in)
    most = 4 * few  # rows that the first call may have
    with Dev(backend) as d:
        set_ = Lora(ad.type, d.put(ad.a), d.put(ad.b), n_adapter=ad.n, max_rank=ad.max_rank, cols=ad.cols, rows=ad.rows, rank=d.put(ad.rank), scale=d.put(ad.scale))
        td, idd, xd, y = d.put(tok.astype(np.int32)), d.put(np.array(ids, np.int32)), d.put(x), d.put(y_in)
        for at, n, n_tok in ((0, few, most), (few, len(ids) - few, len(x))):
            backend.lora_dev(set_, td + 4 * at, idd + 4 * at, n, n_tok, xd, ad.cols, y, rows, y_in_dev=y, ldyi=rows)
        got = d.get(y, y_in)
    assert (np.abs(got - want) <= tol)[mine].all() and np.array_equal(got[~mine], y_in[~mine])


@pytest.mark.parametrize("form", ["apart", "in place", "alone"])
@pytest.mark.parametrize("pad", [0, 1, 4])
def test_lora_forms(backend, form, pad):
    check_lora(backend, *lora_case(60, T_F16, 3, 16, 200, 130, [1, 90, 4], [2, 0, 1], [16, 3, 8], (2, 1)), pad=pad, form=form)


@pytest.mark.parametrize("news", [[1] * 6, [50] * 6])
def test_lora_bad_adapters(backend, news):
    """Ids and ranks that mean nothing make NaN rows, and leave the others alone."""
    case = lora_case(61, T_BF16, 4, 16, 64, 50, news, [0, 4, -2, 2**31 - 1, 2, 3], [16, 16, -1, 17])
    check_lora(backend, *case)


def test_lora_defaults(backend):
    """No ranks and no scales: max_rank and 1."""
    ad, tok, ids, x, y_in = lora_case(62, T_F16, 2, 16, 64, 50, [2, 3], [1, 0])
    ad.scale[:] = 1.0
    want, tol, _ = R.lora(ad, tok, ids, x, y_in)
    with Dev(backend) as d:
        set_ = Lora(T_F16, d.put(ad.a), d.put(ad.b), n_adapter=2, max_rank=16, cols=64, rows=50)
        y = d.put(np.zeros_like(y_in))
        backend.lora_dev(set_, d.put(tok.astype(np.int32)), d.put(np.array(ids, np.int32)), 2, 5, d.put(x), 64, y, 50, y_in_dev=d.put(y_in), ldyi=50)
        assert (np.abs(d.get(y, y_in) - want) <= tol).all()


@pytest.mark.parametrize("t", R.TYPES)
def test_lora_ranges(backend, t):
    """Small and large values side by side keep their bits: x, A and B over 2^40."""
    ad, tok, ids, x, y_in = lora_case(63, t, 2, 16, 256, 64, [3, 20], [0, 1])
    r = np.random.default_rng(63)
    x *= np.exp2(r.integers(-20, 20, x.shape)).astype(np.float32)
    check_lora(backend, ad, tok, ids, x, y_in, form="alone")


@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("news", [[3, 20], [1100, 40]])
@pytest.mark.parametrize("e", [-100, -116, -124])
def test_lora_smallest(backend, t, news, e):
    """x near the smallest numbers: a value's bits below 2^-133 are cut, of x and of A x, and no more."""
    ad, tok, ids, x, y_in = lora_case(69, t, 2, 16, 256, 64, news, [0, 1])
    x, y_in = np.ldexp(x, e).astype(np.float32), np.zeros_like(y_in)
    ad.scale[:] = 2.0**100
    got, _ = run_lora(backend, ad, tok, ids, x, y_in, form="alone")
    want, tol, _ = R.lora(ad, tok, ids, x, y_in)
    for s, i in enumerate(ids):
        a, b = (np.abs(w) for w in ad.of(i))
        # every x and every h off by 2^-133; sums' own roundings, fewer than 2^10 of up to 2^-150 each, where they are subnormal
        tol[tok[s]:tok[s + 1]] += 2.0**100 * (b @ (2.0**-133 * (a.sum(1) + 1) + 2.0**-140) + 2.0**-140)
    assert (np.abs(got - want) <= tol).all()


def test_lora_non_finite(backend):
    """A row with an infinity or a NaN, and NaN in an adapter that others do not use, stay with themselves."""
    ad, tok, ids, x, y_in = lora_case(64, T_F16, 3, 16, 128, 40, [1, 1, 20, 1], [0, 1, 1, 2])
    x[0, 5], x[10, 7] = np.inf, np.nan
    ad.a[2] = encode(np.full(ad.a[2].shape, np.nan), T_F16)
    got, _ = run_lora(backend, ad, tok, ids, x, y_in)
    want, tol, _ = R.lora(ad, tok, ids, np.where(np.isfinite(x), x, 0).astype(np.float32), y_in)
    for t in range(len(x)):
        if t in (0, 10, 22):
            assert not np.isfinite(got[t]).any()
        else:
            assert (np.abs(got[t] - want[t]) <= tol[t]).all()


@pytest.mark.parametrize("tok", [[0, 3, 2, 6], [-2, 1, 3, 6], [0, 2, 5, 2**31 - 1], [-2**31, 2, 4, 6], [6, 6, 6, 6], [0, 0, 0, 6], [-9, -5, -2, -1], [2**31 - 1] * 4])
def test_lora_wild_starts(backend, tok):
    """Row starts that mean nothing: nothing is read or written outside the buffers, and rows that are in one sequence get theirs."""
    ad, _, ids, x, y_in = lora_case(65, T_F16, 3, 16, 128, 40, [2, 2, 2], [0, 1, 2])
    got, before = run_lora(backend, ad, tok, ids, x, y_in)
    if all(b <= e for b, e in zip(tok, tok[1:])):
        clear = np.clip(tok, 0, 6)
        want, tol, mine = R.lora(ad, clear, ids, x, y_in)
        assert np.array_equal(got[~mine], before[~mine])
        assert (np.abs(got[mine] - want[mine]) <= tol[mine]).all()


def test_lora_many_sequences(backend):
    """65535 sequences, most of them empty, of one row each where they are not."""
    news = np.zeros(65535, np.int64)
    news[[0, 70, 71, 4000, 65534]] = 1, 2, 1, 3, 1
    ids = [s % 3 for s in range(65535)]
    check_lora(backend, *lora_case(66, T_BF16, 3, 8, 64, 30, news, ids, None, (1, 1)))


@pytest.mark.parametrize("news, pad", [([1] * 300, (0, 800)), ([1] * 20, (70, 300)), ([400, 3], (0, 1500)), ([5], (1100, 40))])
def test_lora_padded(backend, news, pad):
    """Whole tiles before the first row and behind the last are left as they were."""
    check_lora(backend, *lora_case(78, T_BF16, 3, 24, 72, 70, news, [s % 4 - 1 for s in range(len(news))], None, pad), form="apart")


def test_lora_far_adapters(backend):
    """Adapters more than 2^32 bytes away."""
    n, rank, cols, rows = 70, 512, 65536, 65536
    r = np.random.default_rng(67)
    a, b = encode(r.standard_normal((rank, cols)) / 256, T_F16), encode(r.standard_normal((rows, rank)), T_F16)
    x = r.standard_normal((2, cols)).astype(np.float32)
    with Dev(backend) as d:
        big = [backend.dev_alloc(n * rank * cols * 2) for _ in range(2)]
        d.at += big
        backend.h2d(big[0] + (n - 1) * rank * cols * 2, a)
        backend.h2d(big[1] + (n - 1) * rank * cols * 2, b)
        set_ = Lora(T_F16, big[0], big[1], n_adapter=n, max_rank=rank, cols=cols, rows=rows)
        y = np.zeros((2, rows), np.float32)
        yd = d.put(y)
        backend.lora_dev(set_, d.put(np.array([0, 2], np.int32)), d.put(np.array([n - 1], np.int32)), 1, 2, d.put(x), cols, yd, rows)
        got = d.get(yd, y)
    ad = R.Adapters.__new__(R.Adapters)
    ad.type, ad.n, ad.max_rank, ad.cols, ad.rows = T_F16, 1, rank, cols, rows
    ad.rank, ad.scale, ad.a, ad.b = np.array([rank]), np.ones(1, np.float32), a[None], b[None]
    want, tol, _ = R.lora(ad, [0, 2], [0], x, y)
    assert (np.abs(got - want) <= tol).all()
    assert of_vectors(got, want) <= 1e-5


def test_lora_captured(backend):
    """Two recorded calls of different sizes share the scratch with eager ones."""
    cases = [lora_case(68, T_F16, 3, 16, 512, 200, [1, 2, 1], [0, 1, 2]), lora_case(69, T_BF16, 2, 32, 256, 130, [80, 30], [1, 0])]
    with Dev(backend) as d:
        calls, ys, xs, graphs = [], [], [], []
        for ad, tok, ids, x, y_in in cases:
            set_ = Lora(ad.type, d.put(ad.a), d.put(ad.b), n_adapter=ad.n, max_rank=ad.max_rank, cols=ad.cols, rows=ad.rows, rank=d.put(ad.rank),
                        scale=d.put(ad.scale))
            args = (set_, d.put(tok.astype(np.int32)), d.put(np.array(ids, np.int32)), len(ids), len(x), d.put(x), ad.cols, d.put(np.zeros_like(y_in)), ad.rows)
            yi = d.put(y_in)
            calls.append(lambda args=args, yi=yi, ldyi=ad.rows: backend.lora_dev(*args, y_in_dev=yi, ldyi=ldyi))
            ys.append(args[7])
            xs.append(args[5])
        try:
            for f in calls:
                f()
                backend.graph_begin()
                f()
                graphs.append(backend.graph_end())
            check_lora(backend, *lora_case(70, T_F16, 2, 64, 2048, 300, [300, 200], [0, 1]))  # the scratch grows
            for step in range(4):
                for i, (ad, tok, ids, x, y_in) in enumerate(cases):
                    x += 1.0
                    backend.h2d(xs[i], x)
                    backend.graph_launch(graphs[i])
                    want, tol, _ = R.lora(ad, tok, ids, x, y_in)
                    assert (np.abs(d.get(ys[i], y_in) - want) <= tol).all()
                calls[step % 2]()
        finally:
            for g in graphs:
                backend.graph_destroy(g)


def test_lora_prompt_captured(backend):
    """A recorded call of a prompt, beside eager ones of few rows."""
    ad, tok, ids, x, y_in = lora_case(74, T_BF16, 2, 32, 264, 190, [1000, 90], [1, 0])
    with Dev(backend) as d:
        set_ = Lora(ad.type, d.put(ad.a), d.put(ad.b), n_adapter=ad.n, max_rank=ad.max_rank, cols=ad.cols, rows=ad.rows, rank=d.put(ad.rank),
                    scale=d.put(ad.scale))
        xd, yd, yi = d.put(x), d.put(np.zeros_like(y_in)), d.put(y_in)
        args = (set_, d.put(tok.astype(np.int32)), d.put(np.array(ids, np.int32)), len(ids), len(x), xd, ad.cols, yd, ad.rows)
        backend.lora_dev(*args, y_in_dev=yi, ldyi=ad.rows)
        backend.graph_begin()
        backend.lora_dev(*args, y_in_dev=yi, ldyi=ad.rows)
        graph = backend.graph_end()
        try:
            for step in range(3):
                x += 1.0
                backend.h2d(xd, x)
                check_lora(backend, *lora_case(75 + step, T_F16, 3, 16, 512, 200, [1, 2, 1], [0, 1, 2]))
                backend.graph_launch(graph)
                want, tol, _ = R.lora(ad, tok, ids, x, y_in)
                assert (np.abs(d.get(yd, y_in) - want) <= tol).all()
        finally:
            backend.graph_destroy(graph)


def test_same_results_twice(backend):
    """Adapters and logarithms bit for bit, whatever else the scratch held."""
    case = lora_case(71, T_F32, 3, 32, 1000, 515, [100, 1, 37], [0, 2, 1])
    c = Case(72, [4, 2, 5], 20001, True)
    first = run_lora(backend, *case)[0]
    with Dev(backend) as d:
        x, out = c.put(d), c.outputs(d)
        lse = []
        for _ in range(3):
            backend.draft_verify_dev(x, out[0], out[1], keep_dev=out[2], lse_dev=out[3])
            lse.append(d.get(out[3], c.u))
            check_lora(backend, *lora_case(73, T_F16, 1, 8, 64, 20, [5], [0]))
            assert np.array_equal(run_lora(backend, *case)[0].view(np.uint32), first.view(np.uint32))
    assert np.array_equal(lse[0], lse[1]) and np.array_equal(lse[0], lse[2])


# ---- refusals ----

def test_refusals(backend):
    with Dev(backend) as d:
        p = R.Pool(1, 2, 16, [3, 4], 4, 4)
        dev = DevPool(d, p, 2, 8, 4, 64)
        bad = PagedPool(dev.keep, dev.add, dev.held, dev.held_out, 0, dev.free, dev.free_out)
        c = Case(1, [2, 1], 50, False)
        x, out = c.put(d), c.outputs(d)
        no_len = c.put(d)
        no_len.len = None
        ad, tok, ids, xs, y_in = lora_case(1, T_F16, 1, 8, 16, 4, [1], [0])
        set_ = Lora(T_F16, d.put(ad.a), d.put(ad.b), n_adapter=1, max_rank=12, cols=16, rows=4)
        some = d.put(np.zeros(64, np.float32))
        for call, word in ((lambda: backend.paged_reserve_dev(dev.cache, dev.batch, bad), "paged_reserve: null pointer"),
                           (lambda: backend.draft_verify_dev(x, 0, out[1]), "draft_verify: null pointer"),
                           (lambda: backend.draft_verify_dev(no_len, out[0], out[1], keep_dev=out[2]), "draft_verify: null pointer"),
                           (lambda: backend.draft_verify_dev(x, out[0] + 1, out[1]), "aligned"),
                           (lambda: backend.lora_dev(set_, some, some, 1, 1, some, 16, some, 4), "lora: max_rank")):
            with pytest.raises(BackendError) as e:
                call()
            assert e.value.status == ERR_ARG and word in str(e.value)


def test_scratch_does_not_grow_in_a_graph():
    """A capture whose scratch has no size yet is refused, and the context goes on."""
    from fastgguf_amd.backend import ERR, Backend
    c = Case(2, [2, 1], 50, False)
    ad, tok, ids, x, y_in = lora_case(2, T_F16, 1, 8, 16, 4, [1], [0])
    p = R.Pool(2, 2, 16, [3, 4], 4, 4)
    with Backend(0) as be, Dev(be) as d:
        dx, out = c.put(d), c.outputs(d)
        set_ = Lora(T_F16, d.put(ad.a), d.put(ad.b), n_adapter=1, max_rank=8, cols=16, rows=4)
        args = (set_, d.put(tok.astype(np.int32)), d.put(np.array(ids, np.int32)), 1, 1, d.put(x), 16, d.put(y_in), 4)
        for call in (lambda: be.draft_verify_dev(dx, out[0], out[1], keep_dev=out[2], lse_dev=out[3]), lambda: be.lora_dev(*args)):
            be.graph_begin()
            with pytest.raises(BackendError) as e:
                call()
            assert e.value.status == ERR
            be.graph_destroy(be.graph_end())
            call()
        c.check(d, out)
        dev = DevPool(d, p, 2, 8, 4, 64)
        dev.ask([3, 4], [1, 1])
        be.paged_reserve_dev(dev.cache, dev.batch, dev.pool)
        dev.check(p, R.reserve(p, [3, 4], [1, 1], 8, 4, 64))


# ---- together ----

@pytest.mark.parametrize("captured", [False, True])
def test_a_server_steps(backend, captured):
    """Steps of a server of many sequences as they would run: pages for the batch, a projection with adapters, the append, the
    attention, logits, drafts checked, and what stays for the next step; all on the device, the host only looks. Against the host's
    forms, step by step."""
    n, heads, kv, hd, page, vocab, cols, drafts = 6, 4, 2, 64, 16, 260, 128, 3
    row, n_tok, stride = (heads + 2 * kv) * hd, n * (drafts + 1) + 2, 12
    r = np.random.default_rng(80)
    p = R.Pool(80, n, page, [0] * n, 40, stride)
    ad = R.Adapters(81, T_F16, 3, 16, cols, row)
    ids = [0, 0, -1, 2, 1, 1]
    head = (r.standard_normal((heads * hd, vocab)) / 4).astype(np.float32)
    scale = float(np.float32(hd**-0.5))
    with Dev(backend) as d:
        dev = DevPool(d, p, n, n_tok, drafts + 1, stride * page, True)
        values = p.n_pages * kv * page * hd
        kp, vp = np.zeros(values, np.float32), np.zeros(values, np.float32)
        kd, vd = d.put(kp), d.put(vp)
        cache = PagedCache(T_F32, kd, vd, dev.table, n_pages=p.n_pages, page=page, table_stride=stride, n_head_kv=kv, hd=hd)
        set_ = Lora(T_F16, d.put(ad.a), d.put(ad.b), n_adapter=3, max_rank=16, cols=cols, rows=row, scale=d.put(ad.scale))
        idd = d.put(np.array(ids, np.int32))
        x, base = d.put(np.zeros((n_tok, cols), np.float32)), d.put(np.zeros((n_tok, row), np.float32))
        qkv, q, o = d.put(np.zeros((n_tok, row), np.float32)), d.put(np.zeros((n_tok, heads * hd), np.float32)), d.put(np.zeros((n_tok, heads * hd), np.float32))
        logits = d.put(np.zeros((n_tok, vocab), np.float32))
        lm = backend.upload(T_F32, heads * hd, np.ascontiguousarray(head.T).view(np.uint8))
        case = Case(82, [1] * n, vocab, False, temps=(1.0, 0.0))
        case.n_tok, case.max_tok = n_tok, drafts + 1
        case.u, case.tokens = np.zeros(n_tok, np.float32), np.zeros(n_tok, np.int32)
        ud, vdev, tokens = d.put(case.u), d.put(case.v), d.put(case.tokens)
        checks = Drafts(logits, dev.tok, tokens, ud, vdev, n_seq=n, n_tok=n_tok, max_tok=drafts + 1, vocab=vocab, temp=d.put(case.temp), len=dev.len)
        n_ok, nxt = d.put(np.zeros(n, np.int32)), d.put(np.zeros(n, np.int32))

        def step():
            backend.paged_reserve_dev(cache, dev.batch, dev.pool)
            backend.lora_dev(set_, dev.tok, idd, n, n_tok, x, cols, qkv, row, y_in_dev=base, ldyi=row)
            backend.paged_store_dev(cache, dev.batch, PagedRope(n_rot=hd, halves=True), heads, qkv, row, qkv + 4 * heads * hd,
                                    qkv + 4 * (heads + kv) * hd, row, q, heads * hd)
            backend.paged_attention_dev(cache, dev.batch, PagedMask(scale), heads, q, heads * hd, o, heads * hd)
            backend.matmul_dev(lm, o, logits, n_tok)
            backend.draft_verify_dev(checks, n_ok, nxt, keep_dev=dev.keep)

        graph, keep, hidden = None, np.zeros(n, np.int64), np.zeros((n_tok, cols), np.float32)
        try:
            for i in range(8):
                if i == 5:
                    keep[1] = 0  # a sequence has ended
                    backend.h2d(dev.keep, keep.astype(np.int32))
                add = r.integers(1, drafts + 2, n) if i else np.array([drafts + 1] * n)
                add[1] = 0 if i == 5 else add[1]
                backend.h2d(dev.add, add.astype(np.int32))
                hidden, projected = r.standard_normal((n_tok, cols)).astype(np.float32), r.standard_normal((n_tok, row)).astype(np.float32)
                case.u, case.v = r.random(n_tok).astype(np.float32), r.random(n).astype(np.float32)
                case.tokens = r.integers(0, vocab, n_tok).astype(np.int32)
                if i:
                    case.tokens[1::2] = np.argmax(last_logits, 1)[:len(case.tokens[1::2])]
                for at, a in ((x, hidden), (base, projected), (ud, case.u), (vdev, case.v), (tokens, case.tokens)):
                    backend.h2d(at, a)
                if not captured or i == 0:
                    step()
                else:
                    if graph is None:
                        backend.graph_begin()
                        step()
                        graph = backend.graph_end()
                    backend.graph_launch(graph)
                # the host's forms
                tok, length, seq, pos, slot = R.reserve(p, keep, add, n_tok, drafts + 1, stride * page)
                assert np.array_equal(d.get(dev.tok, tok), tok) and np.array_equal(d.get(dev.table, p.table), p.table)
                assert np.array_equal(d.get(dev.held, p.held), p.held) and np.array_equal(d.get(dev.free, p.free), p.free)
                for at, w in zip(dev.maps, (seq, pos, slot)):
                    assert np.array_equal(d.get(at, w), w)
                total = int(tok[-1])
                want, tol, mine = R.lora(ad, tok, ids, hidden, projected)
                got = d.get(qkv, want.astype(np.float32))
                assert (np.abs(got[mine] - want[mine]) <= tol[mine]).all()
                b = Batch.__new__(Batch)
                b.type, b.hd, b.n_head, b.n_kv, b.page = T_F32, hd, heads, kv, page
                b.news, b.lens, b.tok, b.len, b.n_tok = np.diff(tok).tolist(), length.tolist(), tok, length, n_tok
                b.table, b.stride, b.page_values, b.page_stride = p.table, stride, kv * page * hd, kv * page * hd
                b.k, b.v = d.get(kd, kp.view(np.uint32)), d.get(vd, vp.view(np.uint32))
                got_q = d.get(q, np.zeros((n_tok, heads * hd), np.float32)).reshape(n_tok, heads, hd)
                want_q, _, _, eq, _ = store(b, got.reshape(n_tok, heads + 2 * kv, hd), None, hd, True)
                assert (np.abs(got_q - want_q)[:total] <= eq[:total] + 1e-30).all()
                want_o, tol_o, _ = attention(b, got_q, scale)
                got_o = d.get(o, np.zeros((n_tok, heads * hd), np.float32)).reshape(n_tok, heads, hd)
                assert (np.abs(got_o - want_o)[:total] <= tol_o[:total]).all()
                last_logits = d.get(logits, np.zeros((n_tok, vocab), np.float32))
                want_n, want_next, keep, _ = R.verify(last_logits, tok, case.tokens, case.u, case.v, vocab, drafts + 1, case.temp, length=length)
                assert np.array_equal(d.get(n_ok, want_n), want_n) and np.array_equal(d.get(nxt, want_next), want_next)
                assert np.array_equal(d.get(dev.keep, want_n), keep)
                keep = keep.astype(np.int64)
        finally:
            if graph is not None:
                backend.graph_destroy(graph)
            lm.free()
