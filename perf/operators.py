"""The paged KV cache's operators as measurable cases: the append of a batch's keys and values with the
head norms and the position rotation, and the attention over the pages.

Operators (the `op` of a case):
  store      `Backend.paged_store_dev`: one pass over the fused QKV rows of a batch of sequences; the
             rotated queries in fp32, the new keys and values in their pages
  attention  `Backend.paged_attention_dev`: a batch of sequences over their pages, causal, with a score
             cap, a distance bias, a window or a prefix where the case has them

A batch is `seqs` sequences; `news` and `pasts` give each one's new tokens and the positions already in its
pages, as "a" (all the same) or "a..b" (spread over a..b, the same for a given case whatever the seed).
K pages are [page][K / V head][position][hd], V pages [page][K / V head][hd][position].
"""
from __future__ import annotations

import math

import torch

own = False

GGML = {"f32": 0, "f16": 1, "bf16": 30}
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6

_backend = None


def backend():
    """The process's device context: a program opens one and keeps it."""
    global _backend
    if _backend is None:
        from fastgguf_amd.backend import Backend
        _backend = Backend(0)
    return _backend


# ---- the cases ----

def _store(name, **kw):
    return dict(name=name, op="store", **kw)


def _attend(name, **kw):
    d = dict(cap=0.0, window=0, bias=False, prefix=0)
    d.update(kw)
    return dict(name=name, op="attention", **d)


def listed():
    return [
        # generation of one sequence: one token's QKV row into its page, pairs rotated, no norms
        _store("store_token", type="f16", heads=32, kv_heads=8, hd=128, page=16, seqs=1, news="1", pasts="4095", norm=False,
               halves=False, rot=128),
        # generation of 48 sequences, heads normed, halves rotated
        _store("store_decode", type="bf16", heads=32, kv_heads=8, hd=128, page=64, seqs=48, news="1", pasts="100..4000", norm=True,
               halves=True, rot=128),
        # five ragged prompts read in one batch, behind cached prefixes
        _store("store_prompts", type="f16", heads=32, kv_heads=8, hd=128, page=32, seqs=5, news="37..1100", pasts="0..500", norm=True,
               halves=True, rot=128),
        # one long prompt, an fp32 cache, a quarter of each head rotated
        _store("store_long", type="f32", heads=32, kv_heads=4, hd=64, page=128, seqs=1, news="16384", pasts="0", norm=False,
               halves=True, rot=16),
        # generation of one sequence at 4096 positions
        _attend("decode_one", type="f16", heads=32, kv_heads=8, hd=128, page=16, seqs=1, news="1", pasts="4095"),
        # generation of 32 sequences of very different lengths
        _attend("decode_batch", type="f16", heads=32, kv_heads=8, hd=128, page=64, seqs=32, news="1", pasts="64..8191"),
        # generation with capped scores in a sliding-window layer, hd 256
        _attend("decode_window", type="bf16", heads=16, kv_heads=8, hd=256, page=32, seqs=8, news="1", pasts="500..8000", cap=50.0,
                window=4096),
        # four drafted tokens a sequence checked at once over an fp32 cache
        _attend("decode_drafts", type="f32", heads=32, kv_heads=8, hd=128, page=16, seqs=6, news="4", pasts="300..3000"),
        # a 64-token prompt batch late in a long prompt
        _attend("prompt_batch", type="f16", heads=32, kv_heads=8, hd=128, page=16, seqs=1, news="64", pasts="4032"),
        # a whole prompt of 8192 tokens
        _attend("prompt_long", type="f16", heads=32, kv_heads=8, hd=128, page=128, seqs=1, news="8192", pasts="0"),
        # ragged documents in one batch, distance bias, one K / V head per query head
        _attend("prompt_docs", type="bf16", heads=12, kv_heads=12, hd=64, page=64, seqs=7, news="51..900", pasts="0", bias=True),
        # capped scores, 256 positions before the text that all tokens see, hd 256
        _attend("prompt_prefix", type="bf16", heads=8, kv_heads=4, hd=256, page=32, seqs=3, news="300..700", pasts="0", cap=30.0,
                prefix=256),
    ]


def _log(rng, lo, hi):
    """An integer of lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["store", "decode", "decode", "decode", "prompt", "prompt"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 8] if kv_heads < 8 else [1, 2, 4])
    hd = rng.choice([64, 80, 96, 128, 128, 256])
    if hd == 256:
        heads = min(heads, 16)
    case = dict(type=rng.choice(["f16", "f16", "bf16", "f32"]), heads=heads, kv_heads=kv_heads, hd=hd, page=rng.choice([16, 16, 32, 64, 128, 256]))
    if kind == "store":
        seqs = _log(rng, 1, 64)
        top = rng.choice([1, 1, _log(rng, 2, max(2, 4096 // seqs))])
        past = _log(rng, 1, 8000)
        rot = rng.choice([hd, hd, hd // 4 // 2 * 2])
        return dict(case, op="store", seqs=seqs, news="1" if top == 1 else f"1..{top}", pasts=f"0..{past}", norm=rng.random() < 0.5,
                    halves=rng.random() < 0.5, rot=rot)
    case.update(op="attention", cap=rng.choice([0.0, 0.0, 30.0, 50.0]), window=rng.choice([0, 0, 0, _log(rng, 16, 2048)]),
                bias=rng.random() < 0.2, prefix=0)
    if kind == "decode":
        seqs = _log(rng, 1, 32)
        past = _log(rng, 16, 16384 // (1 + seqs // 8))
        news = rng.choice(["1", "1", "1", str(rng.randint(2, 5)), "1..4"])
        return dict(case, seqs=seqs, news=news, pasts=f"{past // 8}..{past}")
    if heads > 16:
        case["heads"] = 16
    seqs = rng.choice([1, 1, _log(rng, 2, 6)])
    top = _log(rng, 17, 2048 if seqs == 1 else 700)
    case["prefix"] = rng.choice([0, 0, rng.randint(1, top)])
    past = rng.choice([0, _log(rng, 1, 3000)])
    return dict(case, seqs=seqs, news=str(top) if seqs == 1 else f"{max(1, top // 10)}..{top}", pasts=str(past) if seqs == 1 else f"0..{past}")


def _spread(text, n, salt):
    """n numbers of "a" or "a..b", both ends among them where n allows; the same for the same arguments."""
    lo, _, hi = text.partition("..")
    lo, hi = int(lo), int(hi or lo)
    at = [lo + (hi - lo) * ((i * 2654435761 + salt * 40503) % 1009) // 1008 for i in range(n)]
    if n > 1:
        at[salt % n], at[(salt + 1) % n] = hi, lo
    elif n:
        at[0] = hi
    return at


def _lengths(case):
    """(new tokens, positions in the cache with them) of every sequence."""
    news = [max(1, v) for v in _spread(case["news"], case["seqs"], 3)]
    return news, [p + n for p, n in zip(_spread(case["pasts"], case["seqs"], 8), news)]


# ---- inputs ----

def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000 + what)
    return g


def _inputs(case, seed):
    news, lens = _lengths(case)
    heads, kv, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    n, per = sum(news), [-(-v // page) for v in lens]
    stride, used = max(per), sum(per)
    pages = used + 3  # a pool with some pages free
    order = torch.randperm(pages, generator=_gen(seed, 1), device="cuda").int()
    table = torch.zeros(case["seqs"], stride, dtype=torch.int32, device="cuda")
    at = 0
    for s, m in enumerate(per):
        table[s, :m] = order[at:at + m]
        at += m
    normal = lambda what, *shape: torch.randn(*shape, generator=_gen(seed, what), device="cuda")  # noqa: E731
    i = {"table": table, "tok": torch.tensor([0] + news, device="cuda").cumsum(0).int(), "len": torch.tensor(lens, device="cuda").int(),
         "k": normal(2, pages, kv, page, hd).to(DTYPE[case["type"]]), "v": normal(3, pages, kv, hd, page).to(DTYPE[case["type"]])}
    if case["op"] == "store":
        # rows of a QKV projection: heads of different sizes, a few outlying values
        i["qkv"] = normal(4, n, heads + 2 * kv, hd) * (0.3 + 3 * torch.rand(1, heads + 2 * kv, 1, generator=_gen(seed, 5), device="cuda"))
        if case["norm"]:
            i["qw"], i["kw"] = 1 + 0.3 * normal(6, hd), 1 + 0.3 * normal(7, hd)
        return i
    i["q"] = normal(4, n, heads, hd)
    if case["cap"]:
        i["q"] *= 4  # scores that the cap bends
    if case["bias"]:
        i["slopes"] = torch.exp2(-8 * torch.arange(1, heads + 1, device="cuda", dtype=torch.float32) / heads)
    if case["prefix"]:
        i["prefix"] = torch.minimum(torch.full_like(i["len"], case["prefix"]), i["len"])
    return i


class State:
    def __init__(self, case, i):
        self.case, self.i, self.call, self.most = case, i, None, max(_lengths(case)[0])
        n = int(i["tok"][-1])
        self.out = torch.empty(n, case["heads"], case["hd"], device="cuda")
        if own:  # the descriptors of its cache, batch and model that a program keeps
            from fastgguf_amd.backend import PagedBatch, PagedCache, PagedMask, PagedRope
            be, p = backend(), {k: v.data_ptr() for k, v in i.items()}
            news, lens = _lengths(case)
            heads, kv, hd, page, out = case["heads"], case["kv_heads"], case["hd"], case["page"], self.out.data_ptr()
            cache = PagedCache(GGML[case["type"]], p["k"], p["v"], p["table"], n_pages=i["k"].shape[0], page=page,
                               table_stride=i["table"].shape[1], n_head_kv=kv, hd=hd)
            batch = PagedBatch(p["tok"], p["len"], n_seq=case["seqs"], n_tok=n, max_tok=max(news), max_len=max(lens))
            if case["op"] == "store":
                rope = PagedRope(n_rot=case["rot"], halves=case["halves"], freq_base=10000.0, q_norm=p.get("qw", 0), k_norm=p.get("kw", 0),
                                 eps=EPS)
                row, q = (heads + 2 * kv) * hd, p["qkv"]
                k, v = q + 4 * heads * hd, q + 4 * (heads + kv) * hd
                self.call = lambda: be.paged_store_dev(cache, batch, rope, heads, q, row, k, v, row, out, heads * hd)
            else:
                mask = PagedMask(1.0 / math.sqrt(hd), softcap=case["cap"], window=case["window"], slopes=p.get("slopes", 0),
                                 prefix=p.get("prefix", 0))
                q = p["q"]
                self.call = lambda: be.paged_attention_dev(cache, batch, mask, heads, q, heads * hd, out, heads * hd)
            torch.cuda.synchronize()


def prepare(case, seed):
    return State(case, _inputs(case, seed))


# ---- one pass ----

def run(state):
    i = state.i
    if own:
        state.call()
        return {"q": state.out, "k": i["k"], "v": i["v"]} if state.case["op"] == "store" else state.out
    return _plain_store(state) if state.case["op"] == "store" else _plain_attention(state)


def _rows(i):
    """Of every token of the batch: its sequence, its position, its place in its sequence."""
    t = torch.arange(int(i["q" if "q" in i else "qkv"].shape[0]), device="cuda")
    tok = i["tok"].long()
    seq = torch.searchsorted(tok[1:].contiguous(), t, right=True)
    nth = t - tok[seq]
    return seq, i["len"].long()[seq] - (tok[seq + 1] - tok[seq]) + nth, nth


def _normed(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _rotated(x, cos, sin, rot, halves):
    y = x.clone()
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if halves else (x[..., :rot:2], x[..., 1:rot:2])
    u, w = a * cos - b * sin, a * sin + b * cos
    if halves:
        y[..., :rot // 2], y[..., rot // 2:rot] = u, w
    else:
        y[..., :rot:2], y[..., 1:rot:2] = u, w
    return y


def _plain_store(state):
    case, i = state.case, state.i
    heads, kv, rot, page = case["heads"], case["kv_heads"], case["rot"], case["page"]
    seq, pos, _ = _rows(i)
    q, k, v = i["qkv"].split([heads, kv, kv], 1)
    if case["norm"]:
        q, k = _normed(q, i["qw"]), _normed(k, i["kw"])
    angle = pos.double()[:, None, None] * 10000.0 ** (-2.0 * torch.arange(rot // 2, device="cuda", dtype=torch.float64) / rot)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q, k = _rotated(q, cos, sin, rot, case["halves"]), _rotated(k, cos, sin, rot, case["halves"])
    state.out.copy_(q)
    where, off = i["table"][seq, pos // page].long(), pos % page
    i["k"][where, :, off] = k.to(i["k"].dtype)
    i["v"][where, :, :, off] = v.to(i["v"].dtype)
    return {"q": state.out, "k": i["k"], "v": i["v"]}


def _plain_attention(state):
    case, i = state.case, state.i
    heads, kv, hd, n = case["heads"], case["kv_heads"], case["hd"], state.out.shape[0]
    seq, pos, nth = _rows(i)
    seqs, most, group = case["seqs"], state.most, case["heads"] // case["kv_heads"]
    # every sequence's pages side by side, its new tokens' queries padded to the longest's
    k = i["k"][i["table"].long()].float().permute(0, 2, 1, 3, 4).reshape(seqs * kv, -1, hd)
    v = i["v"][i["table"].long()].float().permute(0, 2, 1, 4, 3).reshape(seqs * kv, -1, hd)
    q = torch.zeros(seqs, most, heads, hd, device="cuda")
    q[seq, nth] = i["q"] / math.sqrt(hd)
    q = q.reshape(seqs, most, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(seqs * kv, group * most, hd)
    s = torch.bmm(q, k.transpose(1, 2).contiguous()).reshape(seqs, kv, group, most, -1)
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    j = torch.arange(k.shape[1], device="cuda")
    p = i["len"].long()[:, None] - (i["tok"][1:] - i["tok"][:-1])[:, None] + torch.arange(most, device="cuda")  # [seqs, most]
    gap = p[:, :, None] - j
    if case["bias"]:
        s = s - i["slopes"].reshape(1, kv, group, 1, 1) * gap.abs().float()[:, None, None]
    see = gap >= 0
    if case["prefix"]:
        see = see | (j < i["prefix"][:, None, None])
    see = see & (j < i["len"][:, None, None])
    if case["window"]:
        see = see & (gap < case["window"])
    s = s.masked_fill_(~see[:, None, None], -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True))
    s = s / s.sum(-1, keepdim=True)
    o = torch.bmm(s.reshape(seqs * kv, group * most, -1), v).reshape(seqs, kv, group, most, hd)
    return o.permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, hd)[seq, nth].reshape(n, heads, hd)


# ---- work ----

def _seen(case):
    """Of every sequence: (cached positions that some new token sees, (token, position) pairs)."""
    got = []
    for n, m in zip(*_lengths(case)):
        lo, hi, pairs, pre = m, 0, 0, min(case["prefix"], m)
        for p in range(m - n, m):
            a, b = max(0, p - case["window"] + 1) if case["window"] else 0, max(p, pre - 1)
            lo, hi, pairs = min(lo, a), max(hi, b), pairs + b - a + 1
        got.append((hi - lo + 1, pairs))
    return got


def work(case):
    news, _ = _lengths(case)
    heads, kv, hd, n, size = case["heads"], case["kv_heads"], case["hd"], sum(news), 4 if case["type"] == "f32" else 2
    if case["op"] == "store":
        row = (8 if case["norm"] else 0) + 3 * case["rot"] / hd
        return {"bytes": n * hd * (4 * (2 * heads + 2 * kv) + 2 * size * kv), "flops": n * hd * (heads + kv) * row}
    seen = _seen(case)
    return {"bytes": 2 * size * kv * hd * sum(a for a, _ in seen) + 8 * n * heads * hd, "flops": 4 * heads * hd * sum(b for _, b in seen)}


# ---- float64 ----

def exact(case, seed):
    i = _inputs(case, seed)
    news, lens = _lengths(case)
    heads, kv, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    group, at = heads // kv, 0
    if case["op"] == "store":
        rot, half = case["rot"], case["rot"] // 2
        x = i["qkv"].double()
        q, k, v = x[:, :heads].clone(), x[:, heads:heads + kv].clone(), x[:, heads + kv:]
        kp, vp = i["k"].double(), i["v"].double()
        for y, w in ((q, "qw"), (k, "kw")):
            if case["norm"]:
                y /= (y.square().sum(-1, keepdim=True) / hd + EPS).sqrt()
                y *= i[w].double()
        for s, (n, m) in enumerate(zip(news, lens)):
            where = torch.arange(m - n, m, device="cuda")
            turn = torch.polar(torch.ones(n, half, device="cuda", dtype=torch.float64),
                               torch.outer(where.double(), torch.pow(10000.0, torch.arange(0, rot, 2, device="cuda").double() / -rot)))
            for y in (q, k):
                z = y[at:at + n, :, :rot]
                z = z.unflatten(-1, (2, half)).transpose(-1, -2) if case["halves"] else z.unflatten(-1, (half, 2))
                z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn[:, None])
                y[at:at + n, :, :rot] = (z.transpose(-1, -2) if case["halves"] else z).flatten(-2)
            pg = i["table"][s].long().repeat_interleave(page)[where]
            kp[pg, :, where % page] = k[at:at + n]
            vp[pg, :, :, where % page] = v[at:at + n]
            at += n
        return {"q": q, "k": kp, "v": vp}
    out = torch.empty(sum(news), heads, hd, device="cuda", dtype=torch.float64)
    for s, (n, m) in enumerate(zip(news, lens)):
        pg = i["table"][s, :-(-m // page)].long()
        p, j = torch.arange(m - n, m, device="cuda")[:, None], torch.arange(m, device="cuda")[None]
        hide = j > p
        if case["prefix"]:
            hide &= j >= int(i["prefix"][s])
        if case["window"]:
            hide |= j <= p - case["window"]
        for h in range(heads):
            keys = i["k"][pg, h // group].double().reshape(-1, hd)[:m]
            vals = i["v"][pg, h // group].double().transpose(1, 2).reshape(-1, hd)[:m]
            x = i["q"][at:at + n, h].double() @ keys.T.contiguous() / math.sqrt(hd)
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            if case["bias"]:
                x += -i["slopes"][h].double() * (p - j).abs()
            out[at:at + n, h] = torch.softmax(x.masked_fill(hide, -math.inf), 1) @ vals
        at += n
    return out
