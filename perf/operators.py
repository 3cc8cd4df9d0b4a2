"""Paged key/value cache: representative calls of writing it, reading it back, and attention over it.

A cache holds the keys and values of one layer in pages of 16 to 128 tokens that sequences own in any order, as bf16 or
as e4m3 codes with one fp32 scale per token and head.  Three operators:

* ``write``: new keys and values go into the pages of their sequences (quantised on the way).
* ``read``: the cached rows of a batch come back as packed bf16 rows.
* ``attend``: new tokens of several sequences attend to their sequences' pages: one token each, chunks, or both.

``own`` chooses between the plain form (elementary torch operations in fp32) and the framework's kernels
(``sensenova_u1_b200.ops.paged``).  A case fixes all lengths; a seed fixes values and the order of the pages.

Head counts are those of the released models (32 query heads over 8 or 4 key/value heads, 128 wide) and of the test
models; batch and prompt lengths are those of the chat workloads beside this file (24 conversations of up to 1500 tokens,
a prompt of 32001 tokens) and what a server makes of them: longer histories, chunks of a long prompt, drafted tokens.
"""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128                     # width of a head
TINY = 2.0 ** -110          # smallest row maximum that a scale is made of
E4M3_MAX = 448.0
SCALE = D ** -0.5


def listed():
    return [
        # decode step of a batch of conversations: one new row per sequence; latency of a launch
        _case("write_step", "write", "e4m3", 16, 32, 8, seqs=24, new=1, keys=1500),
        # chunks of several prompts, kept in bf16
        _case("write_chunks", "write", "bf16", 32, 32, 4, seqs=12, new=700, keys=5000),
        # a whole long prompt written at once
        _case("write_prompt", "write", "e4m3", 64, 32, 8, seqs=1, new=32001, keys=32001, even=True),
        # conversations leave the cache for bf16 attention or for another device
        _case("read_batch", "read", "e4m3", 16, 32, 8, seqs=24, new=0, keys=1500),
        # the same for one long document of the mixture-of-experts model
        _case("read_long", "read", "e4m3", 128, 32, 4, seqs=1, new=0, keys=32001, even=True),
        # one conversation, one token: latency
        _case("step_one", "attend", "bf16", 16, 32, 8, seqs=1, new=1, keys=840, even=True),
        # decode step of a batch of conversations
        _case("step_batch", "attend", "e4m3", 16, 32, 8, seqs=24, new=1, keys=4096),
        # decode step of long documents, the bytes of the cache count
        _case("step_long", "attend", "e4m3", 64, 32, 4, seqs=48, new=1, keys=32700),
        # a few drafted tokens per sequence are verified together
        _case("drafts", "attend", "bf16", 32, 32, 8, seqs=8, new=5, keys=12000),
        # second chunk of two prompts
        _case("chunk", "attend", "bf16", 64, 32, 8, seqs=2, new=512, keys=8300, even=True),
        # a server's mixed step: 20 conversations decode while the prompts of four others (with pictures, whose tokens
        # see one another) are read
        _case("mixed", "attend", "e4m3", 16, 32, 8, seqs=24, new=700, keys=6000, single=20, picture=196),
        # last chunk of a long document
        _case("prompt_end", "attend", "e4m3", 128, 32, 8, seqs=1, new=4096, keys=32001, even=True),
    ]


def _case(name, op, fmt, page, heads, kv_heads, *, seqs, new, keys, even=False, single=0, picture=0):
    c = dict(op=op, fmt=fmt, page=page, heads=heads, kv_heads=kv_heads, seqs=seqs, new=new, keys=keys, even=even, single=single,
             picture=picture)
    return dict(name=name, **c) if name else c


def draw(rng):
    op = rng.choice(("write", "read", "attend", "attend", "attend"))
    fmt, page = rng.choice(("bf16", "e4m3", "e4m3")), rng.choice((16, 32, 64, 128))
    heads, kv_heads = rng.choice(((32, 8), (32, 8), (32, 4), (16, 2), (4, 2), (8, 8), (12, 4)))
    seqs, keys = _log(rng, 1, 48), _log(rng, 1, 32768)
    if op == "write":
        new = min(keys, _log(rng, 1, 32768))
        while seqs * new * kv_heads > 32001 * 8:
            seqs, new = max(1, seqs * 2 // 3), max(1, new * 3 // 4)
        while seqs * keys * kv_heads > 2 * 32001 * 8 and keys > new:
            keys = max(new, keys * 3 // 4)
        return _case("", op, fmt, page, heads, kv_heads, seqs=seqs, new=new, keys=keys)
    if op == "read":
        while seqs * keys * kv_heads > 32001 * 8:
            seqs, keys = max(1, seqs * 2 // 3), max(1, keys * 3 // 4)
        return _case("", op, fmt, page, heads, kv_heads, seqs=seqs, new=0, keys=keys)
    kind = rng.choice(("step", "few", "chunk", "mixed"))
    new = min(keys, {"step": 1, "few": rng.randint(2, 24)}.get(kind) or _log(rng, 16, 4096))
    while (seqs * heads * new * keys > 4096 * 32001 * 32 or seqs * keys * kv_heads > 48 * 32700 * 4) and seqs > 1:
        seqs = max(1, seqs * 2 // 3)
    return _case("", op, fmt, page, heads, kv_heads, seqs=seqs, new=new, keys=keys, single=rng.randint(0, seqs) if kind == "mixed" else 0,
                 picture=rng.choice((0, 0, 64, 196)) if kind in ("chunk", "mixed") else 0)


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def _lens(case):
    """New tokens and cached tokens (the new ones among them) of every sequence."""
    rng = random.Random(repr([case[k] for k in ("op", "fmt", "page", "seqs", "new", "keys", "single")]))
    q, kv = [], []
    for i in range(case["seqs"]):
        n = case["new"] if case["even"] or case["new"] <= 1 else rng.randint(max(1, case["new"] // 3), case["new"])
        q.append(min(1, n) if i < case["single"] else n)
        kv.append(max(q[-1], case["keys"] if case["even"] or i == 0 else rng.randint(max(1, case["keys"] // 24), case["keys"])))
    return q, kv


def _limits(case):
    """How many keys of its sequence every new token may read: up to itself, or to the end of the picture that it belongs to."""
    out = []
    for n, k in zip(*_lens(case)):
        p = case["picture"] if n > 1 else 0
        for i in range(n):
            at = i
            if p and i >= n // 4 and (i - n // 4) // p % 2 == 0:      # blocks of p tokens, every other one a picture
                at = min(n - 1, n // 4 + ((i - n // 4) // p + 1) * p - 1)
            out.append(k - n + at + 1)
    return out


def work(case):
    q, kv = _lens(case)
    row = case["kv_heads"] * 2 * D                                     # values of a cached token
    held = 2 * row if case["fmt"] == "bf16" else row + 8 * case["kv_heads"]
    if case["op"] == "write":
        return {"bytes": sum(q) * (2 * row + held), "flops": 0}
    if case["op"] == "read":
        return {"bytes": sum(kv) * (2 * row + held), "flops": 0}
    return {"bytes": sum(kv) * held + 4 * sum(q) * case["heads"] * D, "flops": 4 * D * case["heads"] * sum(_limits(case))}


def _quantise(x):
    """fp32 rows as e4m3 codes and their scales."""
    amax = x.abs().amax(-1).clamp_min(TINY)
    return (x * (E4M3_MAX / amax)[..., None]).to(torch.float8_e4m3fn), amax / E4M3_MAX


def _inputs(case, seed):
    q_lens, kv_lens = _lens(case)
    page, hk, dev = case["page"], case["kv_heads"], "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-k // page) for k in kv_lens]
    pages = sum(need) + max(4, sum(need) // 16)                        # a few belong to nobody
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(need), max(need), dtype=torch.int32)
    at = 0
    host = order.cpu()
    for i, n in enumerate(need):
        table[i, :n] = host[at:at + n]
        at += n
    # keys differ in size from channel to channel, values less; pages nobody has written hold what was there before
    gain = 0.5 + torch.rand(2, hk, 1, D, generator=g, device=dev)
    data = torch.empty(pages, 2, hk, page, D, device=dev, dtype=torch.bfloat16 if case["fmt"] == "bf16" else torch.float8_e4m3fn)
    scales = None if case["fmt"] == "bf16" else torch.empty(pages, 2, hk, page, device=dev)
    step = max(1, (1 << 28) // (2 * hk * page * D))
    for a in range(0, pages, step):
        x = torch.randn(min(step, pages - a), 2, hk, page, D, generator=g, device=dev) * gain
        if scales is None:
            data[a:a + step] = x.to(torch.bfloat16)
        else:
            data[a:a + step], scales[a:a + step] = _quantise(x.to(torch.bfloat16).float())
    rows = sum(q_lens)
    # one projection's output, queries, keys and values of a token in a row; peaked enough that some keys stand out
    qkv = torch.randn(max(rows, 1), case["heads"] + 2 * hk, D, generator=g, device=dev).to(torch.bfloat16)[:rows]
    qkv[:, :case["heads"]] *= 2
    return q_lens, kv_lens, table, data, scales, qkv


def prepare(case, seed):
    q_lens, kv_lens, table, data, scales, qkv = _inputs(case, seed)
    h, hk = case["heads"], case["kv_heads"]
    limits = torch.tensor(_limits(case), dtype=torch.int32)
    s = dict(case=case, q=qkv[:, :h], k=qkv[:, h:h + hk], v=qkv[:, h + hk:], data=data, scales=scales)
    if own:
        from sensenova_u1_b200.ops import paged
        s["cache"] = paged.PagedCache(data, scales)
        s["plan"] = paged.build_plan(s["cache"], h, q_lens, kv_lens, table, limits=limits if case["picture"] else None)
        return s
    dev = data.device
    seq = torch.repeat_interleave(torch.arange(len(q_lens)), torch.tensor(q_lens))
    place = torch.cat([torch.arange(n) for n in q_lens])                # of a new token among its sequence's
    s.update(table=table.to(dev).long(), kv_len=torch.tensor(kv_lens, device=dev), q_max=max(q_lens), k_max=max(kv_lens),
             seq=seq.to(dev), place=place.to(dev), limits=limits.to(dev),
             position=(torch.tensor(kv_lens)[seq] - torch.tensor(q_lens)[seq] + place).to(dev),
             key_seq=torch.repeat_interleave(torch.arange(len(kv_lens)), torch.tensor(kv_lens)).to(dev),
             key_place=torch.cat([torch.arange(n) for n in kv_lens]).to(dev))
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        from sensenova_u1_b200.ops import paged
        if op == "write":
            paged.paged_write(state["cache"], state["k"], state["v"], state["plan"])
            return _held(state)
        if op == "read":
            k, v = paged.paged_read(state["cache"], state["plan"])
            return {"k": k, "v": v}
        return paged.paged_attention(state["q"], state["cache"], state["plan"], SCALE)
    return {"write": _write, "read": _read, "attend": _attend}[op](state)


def _held(s):
    return {"data": s["data"]} if s["scales"] is None else {"data": s["data"], "scales": s["scales"]}


def _write(s):
    page = s["case"]["page"]
    at, off = s["table"][s["seq"], s["position"] // page], s["position"] % page
    kv = torch.stack([s["k"], s["v"]], 1)                               # [rows, 2, heads, D]
    if s["scales"] is None:
        s["data"][at, :, :, off] = kv
    else:
        codes, scale = _quantise(kv.float())
        s["data"].view(torch.uint8)[at, :, :, off] = codes.view(torch.uint8)
        s["scales"][at, :, :, off] = scale
    return _held(s)


def _read(s):
    page = s["case"]["page"]
    at, off = s["table"][s["key_seq"], s["key_place"] // page], s["key_place"] % page
    x = s["data"][at, :, :, off].float()
    if s["scales"] is not None:
        x = x * s["scales"][at, :, :, off][..., None]
    return {"k": x[:, 0].to(torch.bfloat16), "v": x[:, 1].to(torch.bfloat16)}


def _attend(s):
    c = s["case"]
    b, hk, g = c["seqs"], c["kv_heads"], c["heads"] // c["kv_heads"]
    x = s["data"][s["table"]].float()                                   # [sequences, pages, 2, heads, page, D]
    if s["scales"] is not None:
        x = x * s["scales"][s["table"]][..., None]
    x = x.permute(2, 0, 3, 1, 4, 5).reshape(2, b, hk, -1, D)[..., :s["k_max"], :]
    q = torch.zeros(b, s["q_max"], hk, g, D, device=x.device)
    q[s["seq"], s["place"]] = s["q"].float().unflatten(1, (hk, g))
    limit = torch.zeros(b, s["q_max"], dtype=torch.long, device=x.device)
    limit[s["seq"], s["place"]] = s["limits"].long()
    q = q.permute(0, 2, 3, 1, 4).reshape(b, hk, g * s["q_max"], D) * SCALE
    p = (q @ x[0].transpose(-1, -2)).view(b, hk, g, s["q_max"], s["k_max"])
    hidden = torch.arange(s["k_max"], device=x.device) >= limit[..., None]
    p.masked_fill_(hidden[:, None, None], float("-inf"))
    p.sub_(p.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(b, hk, g * s["q_max"], s["k_max"]) @ x[1]
    o = o.view(b, hk, g, s["q_max"], D) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4)[s["seq"], s["place"]].flatten(1, 2).to(torch.bfloat16)


def _e4m3(y):
    """Values in 64 bits rounded to the nearest e4m3 value, ties to even: a step is an eighth of the power of two below."""
    e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(e - 3)
    return (torch.round(y / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact(case, seed):
    q_lens, kv_lens, table, data, scales, qkv = _inputs(case, seed)
    h, hk, page = case["heads"], case["kv_heads"], case["page"]
    if case["op"] == "write":
        held, factor = data.double(), None if scales is None else scales.double()
        r = 0
        for i, (n, k) in enumerate(zip(q_lens, kv_lens)):
            if not n:
                continue
            rows = qkv[r:r + n, h:].double().view(n, 2, hk, D)
            at = torch.arange(k - n, k)
            pages, off = table[i, at // page].long().to(data.device), (at % page).to(data.device)
            if factor is None:
                held[pages, :, :, off] = rows
            else:
                top = rows.abs().amax(-1).clamp_min(TINY)
                held[pages, :, :, off] = _e4m3(rows * E4M3_MAX / top[..., None])
                factor[pages, :, :, off] = top / E4M3_MAX
            r += n
        return {"data": held} if factor is None else {"data": held, "scales": factor}

    def rows_of(i):
        """Keys and values of a sequence in 64 bits: [2, heads, keys, D]."""
        k = kv_lens[i]
        pages = table[i, :-(-k // page)].long().to(data.device)
        x = data.index_select(0, pages).double() if scales is None else data.view(torch.uint8).index_select(0, pages).view(
            torch.float8_e4m3fn).double() * scales.index_select(0, pages).double().unsqueeze(-1)
        return torch.cat(list(x), dim=2)[:, :, :k]

    if case["op"] == "read":
        x = [rows_of(i).transpose(1, 2) for i in range(len(kv_lens))]
        return {"k": torch.cat([t[0] for t in x]), "v": torch.cat([t[1] for t in x])}
    out = torch.empty(sum(q_lens), h, D, dtype=torch.float64, device=data.device)
    limits, r, g = torch.tensor(_limits(case), device=data.device), 0, h // hk
    for i, n in enumerate(q_lens):
        kv = rows_of(i)
        for a in range(r, r + n, 512):
            e = min(a + 512, r + n)
            hidden = torch.arange(kv_lens[i], device=data.device)[None] >= limits[a:e, None]
            for j in range(h):
                s = qkv[a:e, j].double() @ kv[0, j // g].T / math.sqrt(D)
                out[a:e, j] = torch.softmax(s.masked_fill(hidden, float("-inf")), -1) @ kv[1, j // g]
        r += n
    return out
