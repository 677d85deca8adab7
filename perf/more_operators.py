"""What a server of many sequences does around the paged cache, as measurable cases.

Operators (the `op` of a case):
  reserve  `Backend.paged_reserve_dev`: the pages of a batch's new tokens from a ring of free ones, pages that are no longer
           needed back to it, and the batch's row starts, lengths and the sequence, position and slot of each row
  verify   `Backend.draft_verify_dev`: drafted tokens against the target's logits from given random numbers, and the
           token that follows the accepted ones; with one row a sequence, the sampling of a token
  lora     `Backend.lora_dev`: low-rank adapters, one of many for each sequence, added to the outputs of a projection

Ranges are "a" (all the same) or "a..b" (spread over a..b, the same for a given case whatever the seed; the seed
says which sequence gets which).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

GGML = {"f32": 0, "f16": 1, "bf16": 30}
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

_backend = None


def backend():
    """The process's device context: a program opens one and keeps it."""
    global _backend
    if _backend is None:
        from fastgguf_amd.backend import Backend
        _backend = Backend(0)
    return _backend


# ---- the cases ----

def _reserve(name, **kw):
    d = dict(starts="0", prompts="1", ends=0, tight=False)
    d.update(kw)
    return dict(name=name, op="reserve", **d)


def _verify(name, **kw):
    return dict(name=name, op="verify", **kw)


def _lora(name, **kw):
    return dict(name=name, op="lora", **kw)


def listed():
    return [
        # generation: 32 sequences, one token each, a new page for one in 16
        _reserve("pages_decode", seqs=32, page=16, adds="1", pasts="100..4000", rows=32),
        # drafted tokens taken back and new ones added, every tenth sequence a new prompt, too few pages for all: in order until
        # they are spent
        _reserve("pages_serving", seqs=250, page=16, adds="1..6", pasts="10..9000", rows=11000, starts="10", prompts="50..700", tight=True),
        # a batch of prompts, one slot a row
        _reserve("pages_prompts", seqs=9, page=64, adds="300..4000", pasts="0", rows=20000),
        # a large server: every sixteenth sequence ended, every twentieth a new prompt, more rows asked for than a batch holds
        _reserve("pages_many", seqs=4100, page=16, adds="1..5", pasts="1..12000", rows=60000, starts="20", prompts="100..900", ends=16),
        # the next token of one sequence from its logits
        _verify("sample_one", seqs=1, rows="1", vocab=32000, drafter="none"),
        # five drafted tokens of one sequence, against the drafter's probabilities
        _verify("verify_one", seqs=1, rows="6", vocab=128256, drafter="logits"),
        # drafts looked up in the text, without probabilities, a vocabulary of odd size
        _verify("verify_lookup", seqs=24, rows="1..9", vocab=50021, drafter="none"),
        # generation of 64 sequences with up to five drafts each
        _verify("verify_batch", seqs=64, rows="1..6", vocab=128256, drafter="logits"),
        # one token of one sequence
        _lora("lora_one", type="f16", seqs=1, news="1", cols=4096, rows=4096, rank=16, ranks="16", adapters=8),
        # generation of 64 sequences with 24 adapters of different ranks
        _lora("lora_decode", type="bf16", seqs=64, news="1", cols=4096, rows=14336, rank=64, ranks="8..64", adapters=24),
        # ragged prompts, an fp32 adapter each
        _lora("lora_prompts", type="f32", seqs=5, news="37..1100", cols=4096, rows=6144, rank=32, ranks="32", adapters=6),
        # one long prompt
        _lora("lora_long", type="f16", seqs=1, news="8192", cols=4096, rows=14336, rank=64, ranks="64", adapters=3),
    ]


def _log(rng, lo, hi):
    """An integer of lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["reserve", "verify", "lora"])
    if op == "reserve":
        seqs = _log(rng, 1, 4000)
        top = rng.choice([1, rng.randint(2, 9), _log(rng, 10, 2000)])
        return dict(op=op, seqs=seqs, page=rng.choice([16, 16, 32, 64, 128, 256]), adds=str(top) if seqs == 1 else f"{max(1, top // 10)}..{top}",
                    pasts=f"0..{_log(rng, 1, 12000)}", rows=min(60000, max(16, int(seqs * top * rng.uniform(0.4, 1.2)))),
                    starts=str(rng.choice([0, 0, rng.randint(3, 20)])), prompts=f"1..{_log(rng, 2, 900)}", ends=rng.choice([0, rng.randint(3, 20)]),
                    tight=rng.random() < 0.3)
    if op == "verify":
        seqs = _log(rng, 1, 64)
        top = rng.choice([1, rng.randint(2, 6), rng.randint(2, 6)])
        return dict(op=op, seqs=seqs, rows=str(top) if rng.random() < 0.5 else f"1..{top}", vocab=_log(rng, 200, 128256 if seqs * top > 200 else 262144),
                    drafter="none" if top == 1 else rng.choice(["none", "logits", "logits"]))
    kind = rng.choice(["decode", "decode", "prompt"])
    rank = rng.choice([8, 16, 16, 32, 64, 128])
    case = dict(op=op, type=rng.choice(["f16", "f16", "bf16", "f32"]), cols=8 * _log(rng, 32, 1792), rows=_log(rng, 200, 14336), rank=rank,
                ranks=rng.choice([str(rank), f"1..{rank}"]))
    if kind == "decode":
        seqs = _log(rng, 1, 96)
        return dict(case, seqs=seqs, news=rng.choice(["1", "1", "1..4"]), adapters=_log(rng, 1, 32))
    seqs = rng.choice([1, _log(rng, 2, 8)])
    top = _log(rng, 10, min(4000, 250000 // rank) // seqs)
    return dict(case, seqs=seqs, news=str(top) if seqs == 1 else f"{max(1, top // 8)}..{top}", adapters=_log(rng, 1, 8))


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


# ---- inputs ----

def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000 + what)
    return g


def _normal(seed, what, *shape):
    return torch.randn(*shape, generator=_gen(seed, what), device="cuda")


def _uniform(seed, what, *shape):
    return torch.rand(*shape, generator=_gen(seed, what), device="cuda")


def _order(seed, what, n):
    return torch.randperm(n, generator=_gen(seed, what), device="cuda")


def _requests(case):
    """(positions in the pages, positions that stay, new tokens) of every sequence."""
    n, got, every = case["seqs"], [], int(case["starts"])
    for i, (past, add, prompt) in enumerate(zip(_spread(case["pasts"], n, 3), _spread(case["adds"], n, 5), _spread(case["prompts"], n, 7))):
        if every and i % every == every - 1:
            got.append((0, 0, prompt))                                   # a new request
        elif case["ends"] and i % case["ends"] == 2:
            got.append((past, 0, 0))                                     # one that ended
        else:
            got.append((past, max(0, past - i % 4 if past > 4 else past), add))  # up to 3 drafts rejected
    return got


def _per(positions, page):
    return -(-positions // page)


def _reserve_sizes(case):
    """(table_stride, n_pages, free pages) of a case's pool."""
    req, page = _requests(case), case["page"]
    held = sum(_per(a, page) for a, _, _ in req)
    take = sum(max(0, _per(k + n, page) - _per(a, page)) for a, k, n in req)
    give = sum(max(0, _per(a, page) - _per(k + n, page)) for a, k, n in req)
    free = max(0, take - give) * 2 // 3 if case["tight"] else take + 64
    return max(_per(max(a, k + n), page) for a, k, n in req) + 1, held + free + 1, free


def _reserve_inputs(case, seed):
    req, n, page = torch.tensor(_requests(case), device="cuda")[_order(seed, 1, case["seqs"])], case["seqs"], case["page"]
    stride, pages, free = _reserve_sizes(case)
    held = (req[:, 0] + page - 1) // page
    pool = _order(seed, 2, pages).int()
    used = int(held.sum())
    table = torch.full((n, stride), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(stride, device="cuda") < held[:, None]] = pool[:used]
    first = int(_order(seed, 3, pages)[0])
    queue = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    queue[(first + torch.arange(free, device="cuda")) % pages] = pool[used:used + free]
    return {"keep": req[:, 1].int(), "add": req[:, 2].int(), "held": held.int(), "table": table, "queue": queue,
            "free": torch.tensor([first, free], dtype=torch.int32, device="cuda")}


def _verify_inputs(case, seed):
    vocab, n = case["vocab"], case["seqs"]
    rows = torch.tensor([max(1, r) for r in _spread(case["rows"], n, 3)], device="cuda")[_order(seed, 1, n)]
    tok = torch.cat([rows.new_zeros(1), rows.cumsum(0)]).int()
    total = int(tok[-1])
    # logits of a language model: most words unlikely, a few far above them, some forbidden
    logits = 2 * _normal(seed, 2, total, vocab)
    best = torch.randint(vocab, (total, 12), generator=_gen(seed, 3), device="cuda")
    logits.scatter_(1, best, 9 + 2.5 * _normal(seed, 4, total, 12))
    logits[:, torch.randint(vocab, (max(1, vocab // 50),), generator=_gen(seed, 5), device="cuda")] = -math.inf
    temp = torch.tensor([1.0, 0.7, 0.0, 1.2, 0.9], device="cuda")[torch.arange(n, device="cuda") % 5][_order(seed, 6, n)]
    heat = temp.repeat_interleave(rows)[:, None]
    i = {"logits": logits, "tok": tok, "temp": temp, "u": _uniform(seed, 7, total), "v": _uniform(seed, 8, n),
         "len": (100 + rows + torch.arange(n, device="cuda")).int()}
    noise = -torch.log(-torch.log(_uniform(seed, 9, total, vocab).clamp_(1e-30, 0.99999994)))
    if case["drafter"] == "logits":  # a smaller model: the same words, less sure
        i["q"] = logits + 0.8 * _normal(seed, 10, total, vocab)
        x = i["q"].double() / torch.where(heat > 0, heat, 1.0)
        top = x.amax(1, keepdim=True)
        i["q_lse"] = (top[:, 0] + torch.log(torch.exp(x - top).sum(1))).float()
        guess = torch.where(heat > 0, i["q"] + noise * heat, i["q"]).argmax(1)
    else:  # words found in the text: often the likely one
        likely = torch.where(heat > 0, logits + noise * heat, logits).argmax(1)
        guess = torch.where(_uniform(seed, 11, total) < 0.75, likely, torch.randint(vocab, (total,), generator=_gen(seed, 12), device="cuda"))
    i["tokens"] = torch.roll(guess, 1).int()  # a row's guess is the next row's token
    return i


def _lora_lengths(case):
    return [max(1, v) for v in _spread(case["news"], case["seqs"], 3)]


def _lora_ids(case):
    """The adapter of every sequence: every ninth has none."""
    return [-1 if s % 9 == 8 else (s * 7 + s // 3) % case["adapters"] for s in range(case["seqs"])]


def _lora_inputs(case, seed):
    cols, rows, rank, n = case["cols"], case["rows"], case["rank"], case["adapters"]
    news = torch.tensor(_lora_lengths(case), device="cuda")
    tok = torch.cat([news.new_zeros(1), news.cumsum(0)]).int()
    total = int(tok[-1])
    x = _normal(seed, 1, total, cols)
    x[:, torch.randint(cols, (4,), generator=_gen(seed, 2), device="cuda")] *= 20  # outlying channels
    ids = torch.tensor(_lora_ids(case), device="cuda").int()
    ids = torch.where(ids >= 0, _order(seed, 3, n)[ids.long().clamp_min(0)].int(), ids)
    a = (_normal(seed, 4, n, rank, cols) / math.sqrt(cols)).to(DTYPE[case["type"]])
    b = (_normal(seed, 5, n, rows, rank) * 0.5).to(DTYPE[case["type"]])
    ranks = torch.tensor([max(1, r) for r in _spread(case["ranks"], n, 5)], device="cuda").int()
    return {"x": x, "y_in": _normal(seed, 6, total, rows), "a": a, "b": b, "tok": tok, "id": ids, "rank": ranks,
            "scale": 0.25 + _uniform(seed, 7, n)}


class State:
    """Inputs, outputs, and (made with the first pass) the descriptors that a program keeps."""

    def __init__(self, case, i, **out):
        self.case, self.i, self.out, self.call = case, i, out, None


def _ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    n = case["seqs"]
    if case["op"] == "reserve":
        i, rows = _reserve_inputs(case, seed), case["rows"]
        return State(case, i, tok=_ints(n + 1), len=_ints(n), held=_ints(n), free=_ints(2), seq=_ints(rows), pos=_ints(rows),
                     slot=torch.zeros(rows, dtype=torch.int64, device="cuda"), table=i["table"], queue=i["queue"])
    if case["op"] == "verify":
        i = _verify_inputs(case, seed)
        return State(case, i, n_ok=_ints(n), next=_ints(n), keep=_ints(n), lse=torch.zeros(i["logits"].shape[0], device="cuda"))
    i = _lora_inputs(case, seed)
    return State(case, i, y=torch.empty_like(i["y_in"]))


def _bind(state):
    """The framework's call on the state's buffers."""
    from fastgguf_amd.backend import Drafts, Lora, PagedBatch, PagedCache, PagedPool
    be, case = backend(), state.case
    p = {k: v.data_ptr() for k, v in state.i.items()}
    o = {k: v.data_ptr() for k, v in state.out.items()}
    if case["op"] == "reserve":
        stride, pages = state.i["table"].shape[1], state.i["queue"].shape[0]
        cache = PagedCache(GGML["f16"], 0, 0, p["table"], n_pages=pages, page=case["page"], table_stride=stride, n_head_kv=1, hd=64)
        batch = PagedBatch(o["tok"], o["len"], n_seq=case["seqs"], n_tok=case["rows"], max_tok=case["rows"], max_len=stride * case["page"])
        pool = PagedPool(p["keep"], p["add"], p["held"], o["held"], p["queue"], p["free"], o["free"], seq=o["seq"], pos=o["pos"], slot=o["slot"])
        return lambda: be.paged_reserve_dev(cache, batch, pool)
    if case["op"] == "verify":
        total, vocab = state.i["logits"].shape
        most = max(1, max(_spread(case["rows"], case["seqs"], 3)))
        drafts = Drafts(p["logits"], p["tok"], p["tokens"], p["u"], p["v"], n_seq=case["seqs"], n_tok=total, max_tok=most, vocab=vocab,
                        temp=p["temp"], len=p["len"], q=p.get("q", 0), q_lse=p.get("q_lse", 0))
        return lambda: be.draft_verify_dev(drafts, o["n_ok"], o["next"], keep_dev=o["keep"], lse_dev=o["lse"])
    lora = Lora(GGML[case["type"]], p["a"], p["b"], n_adapter=case["adapters"], max_rank=case["rank"], cols=case["cols"], rows=case["rows"],
                rank=p["rank"], scale=p["scale"])
    total = state.i["x"].shape[0]
    return lambda: be.lora_dev(lora, p["tok"], p["id"], case["seqs"], total, p["x"], case["cols"], o["y"], case["rows"], y_in_dev=p["y_in"],
                               ldyi=case["rows"])


# ---- one pass ----

def run(state):
    if own:
        if state.call is None:
            state.call = _bind(state)
        state.call()
        return state.out
    return {"reserve": _plain_reserve, "verify": _plain_verify, "lora": _plain_lora}[state.case["op"]](state)


def _upto(x):
    """Sums of the values before each, and of all."""
    c = x.cumsum(0)
    return c - x, c[-1]


def _plain_reserve(state):
    case, i, o = state.case, state.i, state.out
    page, rows = case["page"], case["rows"]
    n, stride = i["table"].shape
    pages = i["queue"].shape[0]
    keep, add, held = i["keep"].long(), i["add"].long(), i["held"].long()
    first, count = i["free"].long()
    fine = (keep >= 0) & (held >= 0) & (held <= stride) & (keep <= held * page)
    asks = fine & (add >= 0) & (add <= rows) & (keep + add <= stride * page)
    want = torch.where(asks, (keep + add + page - 1) // page, torch.where(fine, (keep + page - 1) // page, held))
    take, give = (want - held).clamp_min(0), (held - want).clamp_min(0)
    wish = torch.where(asks, add, 0)
    given, all_given = _upto(give)
    granted = asks & ((take == 0) | (take.cumsum(0) <= count + all_given)) & ((add == 0) | (wish.cumsum(0) <= rows))
    new, take = torch.where(granted, add, 0), torch.where(granted, take, 0)
    start, total = _upto(new)
    # pages given back, in order, to the ring's end
    s = torch.repeat_interleave(torch.arange(n, device="cuda"), give)
    k = torch.arange(s.shape[0], device="cuda")
    back = i["table"][s, want[s] + k - given[s]]
    i["queue"][(first + count + k) % pages] = back
    # pages taken, from the ring's front
    taken, all_taken = _upto(take)
    s = torch.repeat_interleave(torch.arange(n, device="cuda"), take)
    k = torch.arange(s.shape[0], device="cuda")
    i["table"][s, held[s] + k - taken[s]] = i["queue"][(first + k) % pages]
    o["tok"].copy_(torch.cat([start, total[None]]))
    o["len"].copy_(torch.where(fine, keep + new, 0))
    o["held"].copy_(held - torch.where(fine, give, 0) + take)
    o["free"].copy_(torch.stack([(first + all_taken) % pages, count + all_given - all_taken]))
    r = torch.arange(rows, device="cuda")
    s = torch.searchsorted(o["tok"][1:].long(), r, right=True).clamp_max(n - 1)
    pos = keep[s] + r - start[s]
    slot = i["table"][s, (pos // page).clamp(0, stride - 1)].long() * page + pos % page
    o["seq"].copy_(torch.where(r < total, s, -1))
    o["pos"].copy_(torch.where(r < total, pos, -1))
    o["slot"].copy_(torch.where(r < total, slot, -1))
    return o


def _plain_verify(state):
    i, o = state.i, state.out
    tok, temp, tokens = i["tok"].long(), i["temp"].double(), i["tokens"].long()
    total, vocab = i["logits"].shape
    n, t = tok.shape[0] - 1, torch.arange(i["logits"].shape[0], device="cuda")
    seq = torch.searchsorted(tok[1:].contiguous(), t, right=True)
    greedy, last = (temp == 0)[seq], t == tok[seq + 1] - 1
    heat = torch.where(greedy, 1.0, temp[seq])[:, None]
    # 64 bits: a number's place among sums of all words decides the token
    x = i["logits"].double() / heat
    top, at = x.max(1, keepdim=True)
    at = (i["logits"] == i["logits"].amax(1, keepdim=True)).int().argmax(1)
    p = torch.exp(x - top)
    z = p.sum(1, keepdim=True)
    p = p / z
    draft = torch.roll(tokens, -1)
    chance = torch.ones(total, dtype=torch.float64, device="cuda")
    if "q" in i:
        chance = torch.exp(i["q"].gather(1, draft[:, None]).double() / heat - i["q_lse"].double()[:, None])[:, 0]
    fits = torch.where(greedy, draft == at, i["u"].double() * chance < p.gather(1, draft[:, None])[:, 0])
    stop = torch.where(fits & ~last, total, t)  # rows that end their sequence's run
    stop = torch.full((n,), total, device="cuda").scatter_reduce_(0, seq, stop, "amin")
    o["n_ok"].copy_(stop - tok[:-1])
    rejected = ~last[stop]
    w = p[stop]
    if "q" in i:
        q = torch.exp(i["q"][stop].double() / heat[stop] - i["q_lse"][stop].double()[:, None])
    else:
        q = torch.zeros_like(w).scatter_(1, draft[stop][:, None], 1.0)
    w = torch.where(rejected[:, None], (w - q).clamp_min(0), w)
    c = w.cumsum(1)
    word = (c <= i["v"].double()[:, None] * c[:, -1:]).sum(1)
    o["next"].copy_(torch.where(temp == 0, at[stop], word))
    o["keep"].copy_(i["len"].long() - (tok[1:] - 1 - stop))
    o["lse"].copy_((top + torch.log(z))[:, 0])
    return o


def _plain_lora(state):
    case, i = state.case, state.i
    n, tok, ids = case["seqs"], i["tok"].long(), i["id"].long()
    t = torch.arange(i["x"].shape[0], device="cuda")
    seq = torch.searchsorted(tok[1:].contiguous(), t, right=True)
    nth, most = t - tok[seq], max(_lora_lengths(case))
    # every sequence's tokens padded to the longest's, its adapter beside it, zeros behind its rank
    x = torch.zeros(n, most, case["cols"], device="cuda")
    x[seq, nth] = i["x"]
    own_id = ids.clamp_min(0)
    used = torch.arange(case["rank"], device="cuda") < torch.where(ids >= 0, i["rank"].long()[own_id], 0)[:, None]
    a = i["a"][own_id].float() * used[:, :, None]
    b = i["b"][own_id].float() * used[:, None, :]
    h = torch.bmm(x, a.transpose(1, 2).contiguous())
    d = torch.bmm(h, b.transpose(1, 2).contiguous())
    state.out["y"].copy_(i["y_in"] + i["scale"][own_id][seq, None] * d[seq, nth])
    return state.out


# ---- work ----

def work(case):
    n = case["seqs"]
    if case["op"] == "reserve":
        page, req = case["page"], _requests(case)
        moved = sum(abs(_per(k + m, page) - _per(a, page)) for a, k, m in req)
        return {"bytes": 24 * n + 8 * moved + 16 * case["rows"], "flops": 0}
    if case["op"] == "verify":
        rows = [max(1, r) for r in _spread(case["rows"], n, 3)]
        drafted = sum(r > 1 for r in rows) if case["drafter"] == "logits" else 0
        return {"bytes": 4 * case["vocab"] * (sum(rows) + drafted) + 12 * sum(rows), "flops": 20 * case["vocab"] * (sum(rows) + 2 * drafted)}
    ids, news, ranks = _lora_ids(case), _lora_lengths(case), [max(1, r) for r in _spread(case["ranks"], case["adapters"], 5)]
    size, both = 4 if case["type"] == "f32" else 2, case["cols"] + case["rows"]
    mine = [(m, ranks[a]) for a, m in zip(ids, news) if a >= 0]
    adapters = sum(ranks[a] for a in set(ids) if a >= 0)
    return {"bytes": 4 * sum(news) * (case["cols"] + 2 * case["rows"]) + size * adapters * both, "flops": sum(2 * m * r * both for m, r in mine)}


# ---- float64 ----

def exact(case, seed):
    if case["op"] == "reserve":
        return None  # whole numbers throughout
    if case["op"] == "verify":
        return {"n_ok": None, "next": None, "keep": None, "lse": _exact_lse(case, seed)}
    i = _lora_inputs(case, seed)
    y = i["y_in"].double()
    at = i["tok"].tolist()
    for s, a in enumerate(i["id"].tolist()):
        if a < 0:
            continue
        r = int(i["rank"][a])
        x = i["x"][at[s]:at[s + 1]].double()
        y[at[s]:at[s + 1]] += (x @ i["a"][a, :r].double().T.contiguous()) @ i["b"][a, :, :r].double().T.contiguous() * i["scale"][a].double()
    return {"y": y}


def _exact_lse(case, seed):
    """Every row's logarithm of the sum of exp(logit / temperature), temperature 1 where a sequence takes the largest."""
    i = _verify_inputs(case, seed)
    got, at, heat = [], i["tok"].tolist(), i["temp"].double().cpu().numpy()
    for s in range(case["seqs"]):
        x = i["logits"][at[s]:at[s + 1]].cpu().numpy().astype(np.float64) / (heat[s] if heat[s] > 0 else 1.0)
        got.append(np.logaddexp.reduce(x, axis=1) if x.size < 1 << 16 else x.max(1) + np.log(np.exp(x - x.max(1, keepdims=True)).sum(1)))
    return torch.from_numpy(np.concatenate(got))
