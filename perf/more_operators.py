"""Beam search over a paged key/value cache: representative calls of its three operators.

A request that is searched with several beams keeps its prompt's keys and values once, in pages that all its beams read.

* ``select``: of all continuations of a request's beams (beams x vocabulary), the best ones by running score + log softmax.
* ``tables``: every sequence goes on from the cached tokens of its parent.  Block tables, lengths and use counts of the pages are
  rearranged on the GPU: whole pages are shared, the rows of a page that is not full are copied in every layer's cache, pages that
  nobody holds any more are free, and those that the new tokens need are taken, the lowest numbers first.
* ``attend``: attention of a step's new tokens where groups of sequences have their first tokens in the same pages, which are read
  once for a group.

``own`` chooses between the plain form (elementary torch operations) and the framework's kernels
(``sensenova_u1_b200.ops.beam``, ``.ops.page_tables``, ``.ops.paged``).  A case fixes all lengths; a seed fixes values, orders and
parents.  Head counts and vocabularies are those of the released models and of the test models, prompt lengths those of the workloads
beside this file (conversations of up to 1500 tokens, pictures, a document of 32001 tokens).
"""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128                     # width of a head
SCALE = D ** -0.5
E4M3_MAX = 448.0
INF = float("inf")


def listed():
    return [
        # one short answer searched with four beams: latency
        _select("select_four", 1, 4, 151936, 8, "fp32"),
        # a batch of requests, as a server searches them
        _select("select_batch", 16, 8, 151936, 16, "fp32"),
        # many beams for a caption, the first step: only one beam has a score
        _select("select_first", 2, 32, 151936, 64, "fp32", first=True),
        # the test models' vocabulary, logits kept in bf16
        _select("select_small", 5, 3, 1024, 6, "bf16"),
        # one request, four beams, a short prompt, as many layers as the workloads beside this file run
        _tables("tables_four", "bf16", 64, 8, 12, requests=1, beams=4, keys=840, tail=24),
        # a batch of requests over e4m3 caches with small pages
        _tables("tables_batch", "e4m3", 16, 8, 12, requests=16, beams=8, keys=1500, tail=70),
        # a long document, many beams, few heads
        _tables("tables_long", "bf16", 128, 4, 4, requests=1, beams=32, keys=32001, tail=300),
        # a question about a picture and its text, eight beams
        _attend("beams", "bf16", 64, 32, 8, groups=1, seqs=8, new=1, shared=4200, tail=60),
        # a server's decode step: conversations that begin with the same instructions and examples
        _attend("instructions", "e4m3", 16, 32, 8, groups=1, seqs=48, new=1, shared=6000, tail=1500),
        # several requests of eight beams each
        _attend("requests", "e4m3", 64, 32, 4, groups=6, seqs=8, new=1, shared=8000, tail=130),
        # many questions about one long document
        _attend("document", "bf16", 128, 32, 8, groups=1, seqs=64, new=1, shared=32001, tail=400),
        # drafted tokens of several answers to each of two documents are verified together
        _attend("drafts", "e4m3", 32, 32, 8, groups=2, seqs=12, new=5, shared=16000, tail=90),
    ]


def _select(name, requests, beams, vocab, keep, dtype, first=False):
    c = dict(op="select", requests=requests, beams=beams, vocab=vocab, keep=keep, dtype=dtype, first=first)
    return dict(name=name, **c) if name else c


def _tables(name, fmt, page, kv_heads, layers, *, requests, beams, keys, tail):
    c = dict(op="tables", fmt=fmt, page=page, kv_heads=kv_heads, layers=layers, requests=requests, beams=beams, keys=keys, tail=tail)
    return dict(name=name, **c) if name else c


def _attend(name, fmt, page, heads, kv_heads, *, groups, seqs, new, shared, tail):
    c = dict(op="attend", fmt=fmt, page=page, heads=heads, kv_heads=kv_heads, groups=groups, seqs=seqs, new=new, shared=shared, tail=tail)
    return dict(name=name, **c) if name else c


def draw(rng):
    op = rng.choice(("select", "tables", "attend", "attend"))
    if op == "select":
        beams, vocab = _log(rng, 1, 32), _log(rng, 500, 151936)
        requests = _log(rng, 1, 32)
        while requests * beams * vocab > 128 * 151936:
            requests = max(1, requests // 2)
        return _select("", requests, beams, vocab, rng.choice((beams, 2 * beams, beams + 1)), rng.choice(("fp32", "fp32", "bf16")),
                       first=rng.random() < 0.2)
    fmt, page = rng.choice(("bf16", "e4m3")), rng.choice((16, 32, 64, 128))
    if op == "tables":
        kv_heads, layers = rng.choice((8, 4, 2)), rng.choice((1, 2, 4, 12))
        requests, beams, keys, tail = _log(rng, 1, 24), _log(rng, 1, 32), _log(rng, 20, 32001), _log(rng, 1, 300)
        while requests * (keys + beams * (tail + page)) * layers * kv_heads > 16 * (1500 + 8 * 86) * 12 * 8:
            requests, keys, tail = max(1, requests // 2), max(20, keys * 2 // 3), max(1, tail * 2 // 3)
        return _tables("", fmt, page, kv_heads, layers, requests=requests, beams=beams, keys=keys, tail=tail)
    heads, kv_heads = rng.choice(((32, 8), (32, 8), (32, 4), (16, 2), (4, 2), (8, 8), (12, 4)))
    groups, seqs, shared = _log(rng, 1, 8), _log(rng, 1, 64), _log(rng, 16, 32001)
    new, tail = rng.choice((1, 1, 1, rng.randint(2, 6))), _log(rng, 8, 1500)
    while groups * seqs * new * (shared + tail) * heads > 64 * 32400 * 32 or groups * seqs * tail > 64 * 1500:
        groups, seqs = max(1, groups // 2), max(1, seqs * 2 // 3)
    return _attend("", fmt, page, heads, kv_heads, groups=groups, seqs=seqs, new=new, shared=shared, tail=max(new, tail))


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _kept(case):
    """Tables: tokens of every request's prompt, and tokens that its sequences keep, the prompt's among them."""
    rng = _rng(case)
    prompt = [case["keys"] if i == 0 else rng.randint(max(1, case["keys"] // 3), case["keys"]) for i in range(case["requests"])]
    return prompt, [p + (case["tail"] if i == 0 else rng.randint(0, case["tail"])) for i, p in enumerate(prompt)]


def _lens(case):
    """Attend: shared pages of every group, and all tokens of its sequences."""
    rng, page = _rng(case), case["page"]
    pages = [(case["shared"] if i == 0 else rng.randint(max(1, case["shared"] // 2), case["shared"])) // page for i in range(case["groups"])]
    return pages, [[p * page + (case["tail"] if i == 0 else rng.randint(max(case["new"], case["tail"] // 8), case["tail"]))
                    for i in range(case["seqs"])] for p in pages]


def _held(case):
    """Bytes of a cached token."""
    return case["kv_heads"] * 2 * (2 * D if case["fmt"] == "bf16" else D + 4)


def work(case):
    if case["op"] == "select":
        n = case["requests"] * case["beams"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + case["requests"] * (4 * case["beams"] + 12 * case["keep"]), "flops": 3 * n}
    if case["op"] == "tables":
        prompt, kept = _kept(case)
        page, b = case["page"], case["beams"]
        # the tables' entries and the lengths, in and out; rows of pages that are not full, for one child in two (parents are drawn at random)
        entries = sum(-(-(k + 1) // page) for k in kept) * b
        rows = sum(k % page for k in kept) * b // 2
        return {"bytes": 8 * entries + 16 * len(kept) * b + 2 * rows * case["layers"] * _held(case), "flops": 0}
    pages, lens = _lens(case)
    held, rows = _held(case), case["new"] * case["heads"]
    tokens = sum(p * case["page"] + sum(n - p * case["page"] for n in seqs) for p, seqs in zip(pages, lens))
    pairs = sum(n * case["new"] - case["new"] * (case["new"] - 1) // 2 for seqs in lens for n in seqs)
    return {"bytes": tokens * held + 4 * sum(len(s) for s in lens) * rows * D, "flops": 4 * D * case["heads"] * pairs}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _fill(pages, page, hk, fmt, g):
    """Caches as a step finds them: keys differ in size from channel to channel, values less."""
    gain = 0.5 + torch.rand(2, hk, 1, D, generator=g, device="cuda")
    data = torch.empty(pages, 2, hk, page, D, device="cuda", dtype=torch.bfloat16 if fmt == "bf16" else torch.float8_e4m3fn)
    scales = None if fmt == "bf16" else torch.empty(pages, 2, hk, page, device="cuda")
    step = max(1, (1 << 28) // (2 * hk * page * D))
    for a in range(0, pages, step):
        x = (torch.randn(min(step, pages - a), 2, hk, page, D, generator=g, device="cuda") * gain).to(torch.bfloat16)
        if scales is None:
            data[a:a + step] = x
        else:
            top = x.float().abs().amax(-1).clamp_min(2.0 ** -110)
            data[a:a + step], scales[a:a + step] = (x.float() * (E4M3_MAX / top)[..., None]).to(torch.float8_e4m3fn), top / E4M3_MAX
    return data, scales


def _select_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r, k, v = case["requests"], case["beams"], case["vocab"]
    # most tokens are unlikely, a few stand out, in some rows more than in others
    logits = torch.randn(r * k, v, generator=g, device="cuda").mul_(2.5)
    some = torch.randint(0, v, (r * k, 24), generator=g, device="cuda")
    logits.scatter_add_(1, some, 4 + 10 * torch.rand(r * k, 1, generator=g, device="cuda") * torch.rand(r * k, 24, generator=g, device="cuda"))
    scores = -torch.rand(r, k, generator=g, device="cuda").mul_(3).cumsum(1)
    if case["first"]:
        scores[:, 1:] = -INF
        scores[:, 0] = 0
    return logits.to(torch.bfloat16) if case["dtype"] == "bf16" else logits, scores


def _tables_inputs(case, seed):
    page, b, n = case["page"], case["beams"], case["requests"] * case["beams"]
    prompt, kept = _kept(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = max(-(-(k + 1) // page) for k in kept) + 1
    full = [p // page for p in prompt]
    need = [f + b * (-(-(k + 1) // page) - f) for f, k in zip(full, kept)]
    pages = sum(need) + n + max(4, sum(need) // 16)
    order = torch.randperm(pages, generator=g, device="cuda").cpu().tolist()
    tables, at = [], 0
    for f, k in zip(full, kept):
        head, at = order[at:at + f], at + f
        for _ in range(b):
            own_pages = -(-(k + 1) // page) - f
            tables.append(head + order[at:at + own_pages])
            at += own_pages
    lens = torch.tensor([k + 1 for k in kept for _ in range(b)], dtype=torch.int32)
    first = torch.arange(case["requests"], device="cuda").repeat_interleave(b) * b
    parents = (first + torch.randint(0, b, (n,), generator=g, device="cuda")).to(torch.int32)
    caches = [_fill(pages, page, case["kv_heads"], case["fmt"], g) for _ in range(case["layers"])]
    return tables, lens, width, parents, (lens - 1).cuda(), caches


def _attend_inputs(case, seed):
    page, hk = case["page"], case["kv_heads"]
    shared, lens = _lens(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = sum(p + sum(-(-n // page) - p for n in seqs) for p, seqs in zip(shared, lens))
    pages = need + max(4, need // 16)
    order = torch.randperm(pages, generator=g, device="cuda").cpu().tolist()
    width = max(-(-n // page) for seqs in lens for n in seqs)
    table, at = torch.zeros(case["groups"] * case["seqs"], width, dtype=torch.int32), 0
    for i, (p, seqs) in enumerate(zip(shared, lens)):
        head, at = order[at:at + p], at + p
        for j, n in enumerate(seqs):
            m = -(-n // page)
            table[i * case["seqs"] + j, :m] = torch.tensor(head + order[at:at + m - p], dtype=torch.int32)
            at += m - p
    data, scales = _fill(pages, page, hk, case["fmt"], g)
    rows = case["groups"] * case["seqs"] * case["new"]
    # queries are slices of one projection's output; peaked enough that some keys stand out
    q = torch.randn(rows, case["heads"] + 2 * hk, D, generator=g, device="cuda").mul_(2).to(torch.bfloat16)[:, :case["heads"]]
    return shared, lens, table, data, scales, q


def prepare(case, seed):
    s = dict(case=case)
    if case["op"] == "select":
        s["logits"], s["scores"] = _select_inputs(case, seed)
        return s
    if case["op"] == "tables":
        tables, lens, width, s["parents"], s["keep"], caches = _tables_inputs(case, seed)
        s["caches"] = caches
        if own:
            from sensenova_u1_b200.ops import page_tables, paged
            s["tables"] = page_tables.PageTables([paged.PagedCache(*c) for c in caches], len(tables), width * case["page"])
            s["tables"].load(lens.tolist(), tables)
            return s
        table = torch.full((len(tables), width), -1, dtype=torch.int32)
        for i, t in enumerate(tables):
            table[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        refs = torch.bincount(table[table >= 0].long(), minlength=caches[0][0].shape[0])
        s.update(table=table.cuda(), lens=lens.cuda(), refs=refs.to(torch.int32).cuda())
        return s
    shared, lens, table, data, scales, s["q"] = _attend_inputs(case, seed)
    flat = [n for seqs in lens for n in seqs]
    if own:
        from sensenova_u1_b200.ops import paged
        s["cache"] = paged.PagedCache(data, scales)
        groups = [(i * case["seqs"], case["seqs"], p * case["page"]) for i, p in enumerate(shared)]
        s["plan"] = paged.build_plan(s["cache"], case["heads"], [case["new"]] * len(flat), flat, table, shared=groups)
        return s
    top, n = max(shared), torch.tensor(shared)
    first = torch.arange(case["groups"]) * case["seqs"]
    tail = torch.zeros(len(flat), max(-(-x // case["page"]) - p for p, seqs in zip(shared, lens) for x in seqs), dtype=torch.long)
    for i, x in enumerate(flat):
        p = shared[i // case["seqs"]]
        tail[i, :-(-x // case["page"]) - p] = table[i, p:-(-x // case["page"])]
    kv = torch.tensor(flat)
    s.update(data=data, scales=scales, head=table[first, :top].long().cuda(), tail=tail.cuda(), shared=(n * case["page"]).cuda(),
             tail_len=(kv - (n * case["page"]).repeat_interleave(case["seqs"])).cuda())
    return s


# ------------------------------------------------------------------------------------------------------------- plain forms
def run(state):
    op = state["case"]["op"]
    if own:
        if op == "select":
            from sensenova_u1_b200.ops import beam
            return _named(*beam.beam_select(state["logits"], state["scores"], state["case"]["keep"]))
        if op == "tables":
            t = state["tables"]
            t.step(1, parents=state["parents"], keep=state["keep"])
            return _tabled(t.table, t.lens, t.refs, state["caches"])
        from sensenova_u1_b200.ops import paged
        return paged.paged_attention(state["q"], state["cache"], state["plan"], SCALE)
    return {"select": _run_select, "tables": _run_tables, "attend": _run_attend}[op](state)


def _named(scores, beams, tokens):
    return {"scores": scores, "beams": beams, "tokens": tokens}


def _tabled(table, lens, refs, caches):
    return {"table": table, "lens": lens, "refs": refs, "data": [c[0] for c in caches], "scales": [c[1] for c in caches if c[1] is not None]}


def _run_select(s):
    c = s["case"]
    # 64 bits: candidates of different beams may be closer to one another than 32 bits of a sum over the vocabulary tell
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    x = (x - top) - (x - top).exp().sum(-1, keepdim=True).log()
    x = x.view(c["requests"], c["beams"], c["vocab"]) + s["scores"].double()[..., None]
    best, at = torch.sort(x.flatten(1), dim=-1, descending=True, stable=True)
    best, at = best[:, :c["keep"]], at[:, :c["keep"]]
    at = torch.where(best == -INF, 0, at)
    return _named(best.float(), (at // c["vocab"]).to(torch.int32), (at % c["vocab"]).to(torch.int32))


def _run_tables(s):
    page, table, refs, parents = s["case"]["page"], s["table"], s["refs"], s["parents"].long()
    n, width = table.shape
    pages = refs.numel()
    seq, place = torch.arange(n, device="cuda"), torch.arange(width, device="cuda")
    kept = torch.minimum(s["lens"][parents], s["keep"])
    full, part = kept // page, kept % page
    new = torch.where(place < full[:, None], table[parents], -1)
    count = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    one = torch.ones((), dtype=torch.int32, device="cuda")
    count.index_put_((new.flatten().long(),), one, accumulate=True)             # (-1 counts in the last place)
    # a page that is not full stays with the first sequence that has its rows, if nobody holds it whole; the others get copies
    src = torch.where(part > 0, table[parents].gather(1, full.long().clamp_max(width - 1)[:, None])[:, 0].long(), pages)
    claim = torch.full((pages + 1,), n, device="cuda").scatter_reduce_(0, src, seq, "amin")
    stays = (part > 0) & (count[src] == 0) & (claim[src] == seq)
    copied = (part > 0) & ~stays
    count[torch.where(stays, src, pages)] = 1
    new.scatter_(1, torch.where(stays, full, 0).long()[:, None], torch.where(stays, src.to(torch.int32), new[:, 0])[:, None])
    lens = kept + 1
    begin, end = full + stays, (lens + page - 1) // page
    need = (end - begin).clamp_min(0)
    free = torch.argsort((count[:pages] > 0).to(torch.int32), stable=True)        # the free ones first, lowest numbers first
    before = need.cumsum(0) - need
    taken = (place >= begin[:, None]) & (place < end[:, None])
    which = (before[:, None] + place - begin[:, None]).clamp(0, pages - 1)
    new = torch.where(taken, free[which].to(torch.int32), new)
    count[:pages].index_put_((free,), (torch.arange(pages, device="cuda") < need.sum()).to(torch.int32), accumulate=True)
    dst = new.gather(1, full.long().clamp_max(width - 1)[:, None])[:, 0].long()
    where = (copied[:, None] & (torch.arange(page, device="cuda") < part[:, None]))[:, None, None]
    # whoever copies nothing writes a page of its own, as it is
    to = torch.where(copied, dst, new[:, 0].long())
    rows = torch.where(copied, src, to)
    for data, scales in s["caches"]:
        raw = data.view(torch.uint8) if scales is not None else data
        raw[to] = torch.where(where[..., None], raw[rows], raw[to])
        if scales is not None:
            scales[to] = torch.where(where, scales[rows], scales[to])
    table.copy_(new)
    s["lens"].copy_(lens)
    refs.copy_(count[:pages])
    return _tabled(table, s["lens"], refs, s["caches"])


def _run_attend(s):
    c = s["case"]
    n, m, hk, g, new, page = c["groups"], c["seqs"], c["kv_heads"], c["heads"] // c["kv_heads"], c["new"], c["page"]

    def rows_of(table):                                                            # [2, tables, heads, keys, D]
        x = s["data"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * s["scales"][table][..., None] if s["scales"] is not None \
            else s["data"][table].float()
        return x.permute(2, 0, 3, 1, 4, 5).reshape(2, table.shape[0], hk, table.shape[1] * page, D)

    head, tail = rows_of(s["head"]), rows_of(s["tail"])
    q = s["q"].float().view(n, m, new, hk, g, D).permute(0, 3, 1, 4, 2, 5) * SCALE     # [groups, heads, sequences, group, new, D]
    a = (q.reshape(n, hk, m * g * new, D) @ head[0].transpose(-1, -2)).view(n, hk, m, g, new, -1).transpose(1, 2)
    b = (q.transpose(1, 2).reshape(n * m, hk, g * new, D) @ tail[0].transpose(-1, -2)).view(n, m, hk, g, new, -1)
    dev = q.device
    a = a.masked_fill(torch.arange(a.shape[-1], device=dev) >= s["shared"].view(n, 1, 1, 1, 1, 1), -INF)
    limit = s["tail_len"].view(n, m, 1, 1, 1, 1) - (new - 1 - torch.arange(new, device=dev)).view(new, 1)
    b = b.masked_fill(torch.arange(b.shape[-1], device=dev) >= limit, -INF)
    p = torch.cat([a, b], -1)
    p = (p - p.amax(-1, keepdim=True)).exp()
    total = p.sum(-1, keepdim=True)
    keys = a.shape[-1]
    o = (p[..., :keys].transpose(1, 2).reshape(n, hk, m * g * new, keys) @ head[1]).view(n, hk, m, g, new, D).transpose(1, 2)
    o = o + (p[..., keys:].reshape(n * m, hk, g * new, -1) @ tail[1]).view(n, m, hk, g, new, D)
    return (o / total).permute(0, 1, 4, 2, 3, 5).reshape(n * m * new, hk * g, D).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    return {"select": _exact_select, "tables": _exact_tables, "attend": _exact_attend}[case["op"]](case, seed)


def _exact_select(case, seed):
    logits, scores = _select_inputs(case, seed)
    v, out = case["vocab"], []
    for i in range(case["requests"]):
        rows = torch.log_softmax(logits[i * case["beams"]:(i + 1) * case["beams"]].double(), -1)
        best = []
        for b, row in enumerate(rows):                                             # a beam gives at most as many as are kept
            values, tokens = torch.topk(row, min(v, case["keep"] + 64))
            base = float(scores[i, b])
            best += [(-(base + x), b, t) for x, t in zip(values.tolist(), tokens.tolist())]
        best = sorted(best)[:case["keep"]]
        out.append([(-x, b, t) if x < INF else (-INF, 0, 0) for x, b, t in best])
    x = torch.tensor([[e[0] for e in o] for o in out], dtype=torch.float64, device="cuda")
    return {"scores": x, "beams": None, "tokens": None}


def _exact_tables(case, seed):
    tables, lens, width, parents, keep, caches = _tables_inputs(case, seed)
    page, parents, keep, pages = case["page"], parents.tolist(), keep.tolist(), caches[0][0].shape[0]
    kept = [min(int(lens[p]), k) for p, k in zip(parents, keep)]
    new, uses, owner = [tables[p][:k // page] for p, k in zip(parents, kept)], [0] * pages, {}
    for t in new:
        for pg in t:
            uses[pg] += 1
    whole = list(uses)
    move = []
    for i, (p, k) in enumerate(zip(parents, kept)):
        if k % page:
            pg = tables[p][k // page]
            if whole[pg] == 0 and pg not in owner:
                owner[pg] = i
                uses[pg] = 1
                new[i] = new[i] + [pg]
            else:
                move.append((i, pg, k % page))
    free = iter([pg for pg in range(pages) if uses[pg] == 0])
    todo = {i: (pg, n) for i, pg, n in move}
    jobs = []
    for i, k in enumerate(kept):
        while len(new[i]) * page < k + 1:
            pg = next(free)
            if i in todo and len(new[i]) == k // page:
                jobs.append((todo[i][0], pg, todo[i][1]))
            uses[pg] = 1
            new[i] = new[i] + [pg]
    whole = [None] * case["layers"]
    if sum(c[0].numel() for c in caches) <= 1 << 28:
        for j, (data, scales) in enumerate(caches):
            data, scales = data.double(), None if scales is None else scales.double()
            for src, dst, n in jobs:
                data[dst, :, :, :n] = data[src, :, :, :n]
                if scales is not None:
                    scales[dst, :, :, :n] = scales[src, :, :, :n]
            whole[j] = (data, scales)
    table = torch.full((len(new), width), -1, dtype=torch.int32)
    for i, t in enumerate(new):
        table[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
    return {"table": table, "lens": torch.tensor([k + 1 for k in kept], dtype=torch.int32), "refs": torch.tensor(uses, dtype=torch.int32),
            "data": [None if w is None else w[0] for w in whole],
            "scales": [] if case["fmt"] == "bf16" else [None if w is None else w[1] for w in whole]}


def _exact_attend(case, seed):
    _, lens, table, data, scales, q = _attend_inputs(case, seed)
    page, new, g, out = case["page"], case["new"], case["heads"] // case["kv_heads"], []
    for i, n in enumerate(x for seqs in lens for x in seqs):
        held = table[i, :-(-n // page)].long().cuda()
        x = data.index_select(0, held).double() if scales is None else data.view(torch.uint8).index_select(0, held).view(
            torch.float8_e4m3fn).double() * scales.index_select(0, held).double().unsqueeze(-1)
        x = torch.cat(list(x), dim=2)[:, :, :n].repeat_interleave(g, dim=1)        # [2, heads, keys, D]
        score = torch.einsum("rhd,hkd->hrk", q[i * new:(i + 1) * new].double(), x[0]) / math.sqrt(D)
        hidden = torch.arange(n, device="cuda") > torch.arange(n - new, n, device="cuda")[:, None]
        out.append(torch.einsum("hrk,hkd->rhd", torch.softmax(score.masked_fill(hidden, -INF), -1), x[1]))
    return torch.cat(out)
