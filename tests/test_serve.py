"""The calls around the paged cache without a device: what they refuse, and what the host's forms of them, which the GPU tests compare
with, hold to."""
import numpy as np
import pytest
import serve_ref as R
from paged_ref import T_F16, T_F32

from fastgguf_amd import backend as B

P = 1 << 20  # an address that is never read


def pool(**kw):
    c = dict(type_=T_F16, k_dev=0, v_dev=0, table_dev=P, n_pages=8, page=16, table_stride=4, n_head_kv=0, hd=0)
    b = dict(tok_dev=P, len_dev=P, n_seq=2, n_tok=5, max_tok=3, max_len=60)
    p = dict(keep_dev=P, add_dev=P, held_dev=P, held_out_dev=P, queue_dev=P, free_dev=P, free_out_dev=P, seq=P, pos=P, slot=P)
    for d in (c, b, p):
        d.update({k: v for k, v in kw.items() if k in d})
    return B.PagedCache(**c), B.PagedBatch(**b), B.PagedPool(**p)


@pytest.mark.parametrize("kw", [{}, dict(seq=0, pos=0, slot=0), dict(page=256), dict(n_seq=65535), dict(n_tok=1 << 30), dict(max_tok=1 << 30),
                                dict(slot=P + 8), dict(seq=P + 4)])
def test_reserve_accepted(kw):
    assert B.paged_reserve_check(*pool(**kw)) == ""


@pytest.mark.parametrize("kw", [dict(page=8), dict(page=0), dict(page=48), dict(page=512), dict(n_pages=0), dict(table_stride=0), dict(n_seq=0),
                                dict(n_seq=65536), dict(n_tok=0), dict(max_tok=0), dict(max_len=0), dict(slot=P + 4), dict(keep_dev=P + 2)]
                         + [{k: 0} for k in ("table_dev", "tok_dev", "len_dev", "keep_dev", "add_dev", "held_dev", "held_out_dev", "queue_dev",
                                             "free_dev", "free_out_dev")])
def test_reserve_refused(kw):
    assert B.paged_reserve_check(*pool(**kw)) != ""


@pytest.mark.parametrize("most", ["n_tok", "n_pages"])
def test_reserve_largest(most):
    """Rows and pages are counted in 32 bits, by steps of up to 131072 past the last one."""
    assert B.paged_reserve_check(*pool(**{most: 1 << 30})) == ""
    for n in ((1 << 30) + 1, 2**31 - 131072, 2**31 - 1):
        assert most in B.paged_reserve_check(*pool(**{most: n}))


def test_rows_of_one_that_waits():
    """A prompt without pages keeps the rows it asked for from those behind it, call after call; with add 0, or for a piece of the prompt that
    there are pages for, they are served."""
    def step(first, times=1):
        p = R.Pool(1, 4, 16, [0, 5, 20, 35], 10, 64)
        keep = p.len
        for _ in range(times):
            tok, keep, *_ = R.reserve(p, keep, [first, 1, 1, 1], 512, 512, 1024)
        return tok.tolist()

    assert step(512) == step(512, 3) == [0, 0, 0, 0, 0]
    assert step(0) == [0, 0, 1, 2, 3]
    assert step(160) == [0, 160, 161, 162, 163]
    assert step(161) == [0, 0, 1, 2, 3]  # no pages, but few rows


def drafts(**kw):
    d = dict(logits_dev=P, tok_dev=P, tokens_dev=P, u_dev=P, v_dev=P, n_seq=2, n_tok=5, max_tok=3, vocab=100)
    d.update(kw)
    return B.Drafts(**d)


@pytest.mark.parametrize("kw", [{}, dict(q=P, q_lse=P), dict(temp=P, len=P), dict(ld=101, logits_dev=P + 4), dict(vocab=1), dict(vocab=1 << 24),
                                dict(n_tok=(1 << 18) - 1), dict(n_seq=65535)])
def test_drafts_accepted(kw):
    assert B.draft_check(drafts(**kw)) == ""


@pytest.mark.parametrize("kw", [dict(vocab=0), dict(vocab=(1 << 24) + 1, ld=1 << 25), dict(ld=99), dict(ld=1 << 40), dict(q=P, q_lse=P, ldq=99), dict(q=P),
                                dict(n_tok=0), dict(n_tok=1 << 18), dict(n_seq=0), dict(n_seq=65536), dict(max_tok=0), dict(logits_dev=P + 2),
                                dict(u_dev=P + 1), dict(q=P + 2, q_lse=P)]
                         + [{k: 0} for k in ("logits_dev", "tok_dev", "tokens_dev", "u_dev", "v_dev")])
def test_drafts_refused(kw):
    assert B.draft_check(drafts(**kw)) != ""


def lora_check(**kw):
    d = dict(type_=T_F16, a_dev=P, b_dev=P, n_adapter=3, max_rank=16, cols=64, rows=33)
    e = dict(tok_dev=P, id_dev=P, n_seq=2, n_tok=5, x_dev=P, ldx=64, y_dev=P, ldy=33, y_in_dev=2 * P, ldyi=33)
    d.update({k: v for k, v in kw.items() if k in d or k in ("rank", "scale")})
    e.update({k: v for k, v in kw.items() if k in e})
    return B.lora_check(B.Lora(**d), **e)


@pytest.mark.parametrize("kw", [{}, dict(type_=T_F32), dict(type_=30), dict(y_in_dev=0, ldyi=0), dict(y_in_dev=P), dict(rank=P, scale=P), dict(max_rank=512),
                                dict(cols=8, ldx=9), dict(rows=1, ldy=1, ldyi=5), dict(x_dev=P + 4, y_dev=P + 4), dict(n_tok=1 << 20)])
def test_lora_accepted(kw):
    assert lora_check(**kw) == ""


@pytest.mark.parametrize("kw", [dict(type_=2), dict(cols=60, ldx=64), dict(cols=0), dict(cols=128), dict(rows=0), dict(rows=34), dict(max_rank=12), dict(max_rank=0),
                                dict(max_rank=520), dict(n_adapter=0), dict(n_seq=0), dict(n_seq=65536), dict(n_tok=0), dict(n_tok=(1 << 30) + 1),
                                dict(ldx=63), dict(ldy=32), dict(ldyi=32), dict(ldy=1 << 40), dict(a_dev=P + 8), dict(b_dev=P + 4), dict(x_dev=P + 2),
                                dict(y_in_dev=P, ldyi=34), dict(a_dev=0), dict(b_dev=0), dict(tok_dev=0), dict(id_dev=0), dict(x_dev=0), dict(y_dev=0),
                                dict(rank=P + 1), dict(scale=P + 2), dict(n_tok=1 << 28, rows=1 << 20, ldy=1 << 20, ldyi=1 << 20)])
def test_lora_refused(kw):
    assert lora_check(**kw) != ""


def test_lora_largest():
    """A tile's offsets in 32 bits."""
    most = dict(cols=1 << 20, ldx=1 << 24, ldy=1 << 24, ldyi=1 << 24)
    assert lora_check(**most) == ""
    for kw in (dict(n_adapter=(1 << 30) + 1), dict(cols=(1 << 20) + 8), dict(ldx=(1 << 24) + 1), dict(ldy=(1 << 24) + 1), dict(ldyi=(1 << 24) + 1)):
        assert lora_check(**{**most, **kw}) != ""


@pytest.mark.parametrize("seed", range(8))
def test_pages_are_never_lost(seed):
    """After any steps of the host's form, every page is held once or free once, and sequences hold what their lengths take."""
    r = np.random.default_rng(seed)
    n, page = int(r.integers(1, 9)), int(r.choice([16, 32]))
    p = R.Pool(seed, n, page, r.integers(0, 200, n), int(r.integers(0, 12)), 20)
    every = np.sort(p.pages())
    for _ in range(12):
        keep = np.where(r.random(n) < 0.2, 0, np.maximum(0, p.len - r.integers(0, 4, n)))
        add = r.integers(0, 60, n)
        tok, length, seq, pos, slot = R.reserve(p, keep, add, 150, 150, 400)
        assert np.array_equal(np.sort(p.pages()), every)
        assert np.array_equal(p.held[np.diff(tok) > 0], -(-length[np.diff(tok) > 0] // page))
        assert (p.held * page >= length).all()
        assert ((np.diff(tok) == add) | (np.diff(tok) == 0)).all() and tok[-1] <= 150
        used = slot[slot >= 0]
        assert len(set(used.tolist())) == len(used) == tok[-1]
        p.len = length


@pytest.mark.parametrize("kind", ["drafter", "lookup"])
def test_verified_tokens_are_the_targets(kind):
    """Over all u and v of a fine grid, and drafts as the drafter draws them, the first token has the target's distribution."""
    r = np.random.default_rng(3)
    vocab, grid = 5, 400
    logits = r.standard_normal((2, vocab)).astype(np.float32)
    logits[0, 1] = -np.inf
    q = r.standard_normal((2, vocab)).astype(np.float32)
    q_lse = np.log(np.exp(q.astype(np.float64)).sum(1)).astype(np.float32)
    p = np.exp(logits[0].astype(np.float64))
    p /= p.sum()
    got = np.zeros(vocab)
    middle = (np.arange(grid) + 0.5) / grid
    for d in range(vocab):
        share = float(np.exp(q[0, d] - q_lse[0])) if kind == "drafter" else float(d == 2)
        if share == 0.0:
            continue
        for x in middle:
            # v matters only where the draft goes: one v on a coarser grid
            n_ok, nxt, _, _ = R.verify(logits, [0, 2], [0, d], [x, 0.0], [0.5], vocab, 2, q=q if kind == "drafter" else None, q_lse=q_lse)
            if n_ok[0]:
                got[d] += share / grid
            else:
                for y in middle[::20]:
                    got[R.verify(logits, [0, 2], [0, d], [x, 0.0], [y], vocab, 2, q=q if kind == "drafter" else None, q_lse=q_lse)[1][0]] += share / grid / len(middle[::20])
    assert np.abs(got - p).max() < 1 / 20  # a step of v's grid


def test_lora_bound_holds_every_part():
    """The bound on a vector's error that the GPU tests take is passed by x without its last 8 of 24 bits."""
    from paged_ref import cut, of_vectors
    ad = R.Adapters(1, T_F16, 2, 16, 512, 96)
    x = np.random.default_rng(2).standard_normal((6, 512)).astype(np.float32)
    y_in = np.zeros((6, 96), np.float32)
    tok, ids = [0, 3, 6], [1, 0]
    want, _, _ = R.lora(ad, tok, ids, x, y_in)
    bound = 4 * of_vectors(R.lora32(ad, tok, ids, x, y_in), want) + 2.0**-22
    assert bound < 5e-6 < of_vectors(R.lora32(ad, tok, ids, cut(x, 16), y_in), want)
