"""The paged KV cache without a device: what its calls refuse, and where its kernels read and write."""
import numpy as np
import pytest

from fastgguf_amd import backend as B
from paged_ref import Batch, T_BF16, T_F16, T_F32, attention, of_vectors, plain32, vector_bound


def descriptors(**kw):
    c = dict(type_=T_F16, k_dev=1 << 20, v_dev=1 << 21, table_dev=1 << 22, n_pages=8, page=16, table_stride=4, n_head_kv=2, hd=64)
    b = dict(tok_dev=64, len_dev=64, n_seq=2, n_tok=5, max_tok=3, max_len=60)
    c.update({k: v for k, v in kw.items() if k in c or k == "page_stride"})
    b.update({k: v for k, v in kw.items() if k in b})
    return B.PagedCache(**c), B.PagedBatch(**b)


GOOD_ROPE = dict(n_rot=64, halves=True)


@pytest.mark.parametrize("kw", [{}, dict(type_=T_F32), dict(type_=T_BF16), dict(hd=80), dict(hd=256), dict(page=256),
                                dict(page_stride=2 * 16 * 64 + 8), dict(max_len=1), dict(max_tok=1000), dict(n_tok=1)])
def test_accepted(kw):
    c, b = descriptors(**kw)
    rot = min(64, c.hd)
    assert B.paged_check(c, b, 4, rope=B.PagedRope(n_rot=rot)) == ""
    assert B.paged_check(c, b, 4, mask=B.PagedMask(0.125, softcap=30.0, window=7)) == ""
    assert B.paged_check(c, b, 0, rope=B.PagedRope(), ldq=0, ldo=0) == ""


@pytest.mark.parametrize("kw", [dict(type_=2), dict(type_=8), dict(hd=32), dict(hd=100), dict(hd=512), dict(page=8), dict(page=48),
                                dict(page=512), dict(page=0), dict(page=-16), dict(n_pages=0), dict(table_stride=0), dict(n_head_kv=0),
                                dict(page_stride=2 * 16 * 64 - 8), dict(page_stride=2 * 16 * 64 + 4), dict(page_stride=-8),
                                dict(n_seq=0), dict(n_tok=0), dict(max_tok=0), dict(max_len=0), dict(n_seq=65536), dict(n_tok=-1)])
def test_refused_descriptors(kw):
    c, b = descriptors(**kw)
    assert B.paged_check(c, b, 4, rope=B.PagedRope()) != ""
    assert B.paged_check(c, b, 4, mask=B.PagedMask(0.125)) != ""


def test_refused_rope():
    c, b = descriptors()
    for kw in (dict(n_rot=63), dict(n_rot=66), dict(n_rot=-2), dict(n_rot=64, freq_base=0.0), dict(n_rot=64, freq_base=float("nan")),
               dict(n_rot=64, freq_scale=0.0), dict(n_rot=64, freq_scale=float("inf")), dict(q_norm=64, eps=-1.0),
               dict(k_norm=64, eps=float("nan"))):
        assert B.paged_check(c, b, 4, rope=B.PagedRope(**kw)) != "", kw
    r = B.PagedRope(n_rot=64)
    r.rope = 2
    assert B.paged_check(c, b, 4, rope=r) != ""
    for kw in (dict(ldq=255), dict(ldq=258), dict(ldo=252), dict(ldkv=124), dict(ldkv=130), dict(ldkv=1 << 40)):
        assert B.paged_check(c, b, 4, rope=B.PagedRope(), **kw) != "", kw
    assert B.paged_check(c, b, -1, rope=B.PagedRope()) != ""


def test_refused_mask():
    c, b = descriptors()
    for kw in (dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1.0, softcap=-1.0), dict(scale=1.0, softcap=float("inf")),
               dict(scale=1.0, window=-1)):
        assert B.paged_check(c, b, 4, mask=B.PagedMask(**kw)) != "", kw
    for n_head in (0, 1, 3, -2):  # none, or no multiple of the two K / V heads
        assert B.paged_check(c, b, n_head, mask=B.PagedMask(1.0), ldq=512, ldo=512) != ""
    assert B.paged_check(c, b, 4, mask=B.PagedMask(1.0), ldq=252) != ""
    assert B.paged_check(c, b, 4, mask=B.PagedMask(1.0), ldo=257) != ""
    c, b = descriptors(n_head_kv=1, n_tok=1 << 29, max_tok=1 << 29)
    assert B.paged_check(c, b, 4, mask=B.PagedMask(1.0)) == "too many rows"


def test_refused_sizes():
    """More workgroups than a launch takes, offsets past 64 bits, scales at which fp32 scores would not be finite."""
    mask = B.PagedMask(0.125)
    c, b = descriptors(n_head_kv=4096, n_seq=65535)
    assert "too many" in B.paged_check(c, b, 4096, mask=mask)
    c, b = descriptors(n_head_kv=4096, n_seq=65535, n_tok=65535)
    assert "too many" in B.paged_check(c, b, 0, rope=B.PagedRope())
    c, b = descriptors(n_tok=1 << 24)
    assert "too many" in B.paged_check(c, b, 4, rope=B.PagedRope())
    c, b = descriptors(n_head_kv=255, n_seq=65535, n_tok=1 << 15)
    assert B.paged_check(c, b, 255, mask=mask) == "" and B.paged_check(c, b, 255, rope=B.PagedRope()) == "too many rows, sequences or K / V heads"
    c, b = descriptors(n_head_kv=257, n_seq=65535, n_tok=1)  # decode workgroups: one above 2^24 - 1 with fewer prompt tiles
    assert "too many" in B.paged_check(c, b, 257, mask=mask)
    c, b = descriptors(n_pages=1 << 20, page_stride=1 << 30)
    assert "page_stride" in B.paged_check(c, b, 4, mask=mask)
    c, b = descriptors(n_pages=1 << 20, page_stride=1 << 28)
    assert B.paged_check(c, b, 4, mask=mask) == ""
    for kw in (dict(scale=1e20), dict(scale=-1e20), dict(scale=1.0, softcap=1e-30), dict(scale=1.0, softcap=1e30)):
        assert B.paged_check(c, b, 4, mask=B.PagedMask(**kw)) != "", kw
    assert B.paged_check(c, b, 0, rope=B.PagedRope(), ldq=3, ldo=-1) == ""  # not used without queries


@pytest.mark.parametrize("page,hd,gap", [(16, 64, 0), (64, 80, 8), (256, 128, 24)])
def test_slots(page, hd, gap):
    """Every value of every position has a place of its own, inside its page."""
    x = Batch(1, T_F16, hd, 3, 3, page, [1, 1, 1], [page, 2 * page + 3, 1], gap=gap)
    c, _ = descriptors(n_pages=x.n_pages, page=page, table_stride=x.stride, n_head_kv=3, hd=hd, page_stride=x.page_stride)
    for is_v in (False, True):
        seen = set()
        for s, m in enumerate(x.lens):
            for pos in range(m):
                for h in range(3):
                    want = x.at(s, pos, h, is_v)
                    got = [B.paged_slot(c, x.table, s, pos, h, d, is_v) for d in (0, 1, hd - 1)]
                    assert got == [want[0], want[1], want[hd - 1]]
                    seen.update(want.tolist())
        assert len(seen) == sum(x.lens) * 3 * hd
        assert max(seen) < x.n_pages * x.page_stride


def test_slots_of_bad_pages():
    """Page numbers outside the cache and positions outside the table are read and written nowhere."""
    c, _ = descriptors()
    table = np.array([[0, 7, 8, -1], [0x7FFFFFFF, -0x80000000, 3, 0]], np.int32)
    for s, pos, there in ((0, 15, True), (0, 16, True), (0, 32, False), (0, 63, False), (1, 0, False), (1, 16, False), (1, 47, True),
                          (1, 63, True), (0, 64, False), (0, -1, False)):
        for is_v in (False, True):
            got = B.paged_slot(c, table, s, pos, 1, 5, is_v)
            assert (got >= 0) == there and got < 8 * 2 * 16 * 64


def test_slots_of_bad_caches():
    for page in (0, 8, 24, 48):
        c, _ = descriptors(page=page)
        assert B.paged_slot(c, np.zeros((1, 4), np.int32), 0, 1, 0, 0) == -1


def test_slots_are_64_bit():
    c, _ = descriptors(n_pages=1 << 20, page_stride=1 << 20)
    table = np.array([[(1 << 20) - 1] * 4], np.int32)
    assert B.paged_slot(c, table, 0, 17, 1, 3) == ((1 << 20) - 1 << 20) + 64 * 16 + 64 + 3
    assert B.paged_slot(c, table, 0, 17, 1, 3, True) == ((1 << 20) - 1 << 20) + 64 * 16 + 3 * 16 + 1


def plan(b, **kw):
    """What the attention of a batch of paged_ref launches on 256 compute units."""
    c = B.PagedCache(b.type, 16, 16, 16, n_pages=b.n_pages, page=b.page, table_stride=b.stride, n_head_kv=b.n_kv, hd=b.hd, page_stride=b.page_stride)
    batch = B.PagedBatch(16, 16, n_seq=len(b.news), n_tok=b.n_tok, max_tok=max(b.news + [1]), max_len=max(b.lens + [1]))
    return B.paged_plan(c, batch, b.n_head, B.PagedMask(0.125, **kw))


def test_plan():
    """Few rows, prompts, and both: which kernels, over how many splits, in which rows."""
    def of(news, lens, hd=128, heads=8, kv=2, t=T_F16, **kw):
        return plan(Batch(1, t, hd, heads, kv, 16, news, lens, sigma=0.0), **kw)

    assert of([1], [4096]) == (33, 0, 0, False)              # a step for every wavefront
    assert of([1] * 300, [40] * 300) == (1, 0, 0, False)     # more workgroups than fit: whole ranges
    assert of([4], [300], kv=2) == (3, 0, 0, False)          # 16 rows a K / V head
    assert of([5], [300], kv=2) == (0, 2, 64, True)          # 20
    assert of([64], [4096]) == (0, 8, 64, True)
    assert of([64], [4096], t=T_F32, hd=256) == (0, 8, 128, True)  # no form of half the rows
    assert of([64], [4096], window=100) == (0, 1, 64, True)  # 163 positions
    assert of([64], [4096], window=100, prefix=16) == (0, 8, 64, True)
    ds, ps, rows, alone = of([900] * 8, [900] * 8)
    assert (ds, ps, rows) == (8, 1, 128) and not alone
    assert of([40, 1, 0, 3], [2100, 1500, 9, 3])[:3] == (17, 8, 64)
    # a compute unit each only for as many workgroups as there are: 256, and 320, which would take two turns
    assert of([64, 64], [4064, 4064], heads=32, kv=8) == (32, 8, 128, True)
    assert of([150], [2150], heads=32, kv=8) == (0, 8, 128, False)
    assert of([40] * 4, [1040] * 4, heads=16, kv=8, hd=64, t=T_BF16) == (9, 5, 64, False)
    with pytest.raises(B.BackendError):
        of([1], [16], hd=100)


def test_gpu_tests_take_every_form():
    """The batches of the GPU tests reach every kernel form that there is, for every head size and type."""
    import test_gpu_paged as G
    seen = set()

    def add(b, **kw):
        ds, ps, rows, alone = plan(b, **kw)
        for form in (("few rows", "split" if ds > 1 else "whole") if ds else None, (rows, "split" if ps > 1 else "whole") if ps else None):
            if form:
                seen.add((b.type, b.hd) + form)
        if ds and ps:
            seen.add((b.type, b.hd, "both"))
        if alone:
            seen.add("alone")

    types, hds = (T_F16, T_BF16, T_F32), (64, 80, 96, 128, 256)
    for t in types:
        for hd in hds:
            for news, lens, at in G.NULL_TYPES:
                add(G.with_null_key(t, news, lens, 20, at, hd=hd)[0])
            add(Batch(51, t, hd, 4, 2, 32, *G.crowd([200, 1, 70, 0, 3, 130], [200, 90, 640, 0, 3, 333]), sigma=0.0))
    for i in range(len(G.SHAPES)):
        add(G.shape(i))
    for t, hd, nh in G.SPLITS:
        for news, lens in (([1], [2500]), ([3, 1], [2500, 700]), ([40], [2500]), ([40, 1, 0, 3], [2100, 1500, 9, 3])):
            add(Batch(50, t, hd, nh, 1, 32, news, lens, sigma=0.0))
    want = {(t, hd) + f for t in types for hd in hds for f in (("few rows", "whole"), ("few rows", "split"), (128, "whole"), (128, "split"),
                                                              (64, "whole"), (64, "split"), ("both",))}
    want -= {(T_F32, 256, 64, w) for w in ("whole", "split")}
    assert "alone" in seen
    assert not want - seen, sorted(want - seen, key=str)


@pytest.mark.parametrize("i", range(4))
def test_vector_bound_holds_every_part(i):
    """The bound of the GPU tests' output vectors is passed by q or weights that lack their last 8 of 24 bits."""
    import test_gpu_paged as G
    b = G.ordinary(T_BF16, i)
    scale = float(np.float32(128**-0.5))
    want, _, mine = attention(b, b.q, scale)
    bound = vector_bound(b, b.q, scale, want, mine)
    assert of_vectors(plain32(b, b.q, scale)[mine], want[mine]) < bound < 5e-6
    for bits in ({"bits_q": 16}, {"bits_w": 16}):
        assert of_vectors(plain32(b, b.q, scale, **bits)[mine], want[mine]) > bound
