"""The paged KV cache without a device: what its calls refuse, and where its kernels read and write."""
import numpy as np
import pytest

from fastgguf_amd import backend as B
from paged_ref import Batch, T_BF16, T_F16, T_F32


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
