"""Attention of sequences that share their first tokens (csrc/attn_prefix_sm100.cu, attn_paged.cu) against plain arithmetic in 64 bits."""
import pytest
import torch

from test_paged_gpu import BF16, D, E4M3, SCALE, causal, exact, near, quantised

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def always(monkeypatch):
    """Shared however short it is."""
    from sensenova_u1_b200.ops import paged
    monkeypatch.setattr(paged, "SHARE_TOKENS", (0, 0))


def setup(groups, page, hk, dtype, seed=0, room=0, stretch=True):
    """``groups``: (shared tokens, lengths of the sequences).  The cache, tables, what every sequence holds in 64 bits, and the argument ``shared``."""
    from sensenova_u1_b200.ops import paged
    need = sum(s // page + sum(-(-(k + room) // page) - s // page for k in lens) for s, lens in groups)
    pages = need + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(pages, 2, hk, page, D, device="cuda", generator=g).to(BF16)
    if dtype == E4M3:
        if stretch:
            x = x * torch.exp2(torch.randint(-3, 4, x.shape[:4] + (1,), device="cuda", generator=g)).to(BF16)
        codes, scales = quantised(x)
        cache, held = paged.PagedCache(codes, scales), codes.double() * scales.double()[..., None]
    else:
        cache, held = paged.PagedCache(x), x.double()
    tables, shared, kv = [], [], []
    for s, lens in groups:
        head, order = order[:s // page], order[s // page:]
        shared.append((len(kv), len(lens), s))
        for k in lens:
            n = -(-(k + room) // page) - len(head)
            tables.append(head + order[:n])
            order = order[n:]
            kv.append(k)
    # (tokens of a page that is not whole are each sequence's own: only whole pages are alike, and what the caller names must be)
    shared = [(a, n, s // page * page) for a, n, s in shared]
    return cache, tables, kv, rows_of(held, tables, kv), shared


def rows_of(held, tables, kv):
    return [torch.cat([held[p] for p in t[:-(-k // held.shape[3])]], 2)[:, :, :k] if k else held[0, :, :, :0] for t, k in zip(tables, kv)]


def queries(n, hq, seed=1, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n + 2, hq + 3, D, device="cuda", generator=g) * scale).to(BF16)[:, 1:hq + 1]


def wider(room, q, q_lens, rows, limits, plan):
    """Runs of more than 64 rows over e4m3 go to the kernel for chunks, which rounds code times scale of a key to fp16: 2^-11 of it, so a score
    moves by 2^-11 of the sum of |q k| at most and a probability by exp of that, before and after the sum is divided by (see ``near``)."""
    if plan._args.many_count == 0 or rows[0].dtype != torch.float64 or plan.dtype != E4M3:
        return room
    room, r = room.clone(), 0
    for n, kv in zip(q_lens, rows):
        if n and kv.shape[2]:
            k = kv[0].repeat_interleave(q.shape[1] // kv.shape[1], 0)
            hidden = torch.arange(kv.shape[2], device=q.device)[None] >= limits[r:r + n, None]
            most = (torch.einsum("rhd,hkd->hrk", q[r:r + n].double().abs(), k.abs()) * SCALE).masked_fill(hidden, 0.0).amax(-1)
            room[r:r + n] *= 1 + 2 * 2.0 ** -11 * most.T[..., None] / (2.0 ** -8 + 2.0 ** -11)
        r += n
    return room


def check(groups, q_lens, hq, hk, page, dtype, limits=None, seed=0, scale=1.0):
    from sensenova_u1_b200.ops import paged
    cache, tables, kv, rows, shared = setup(groups, page, hk, dtype, seed)
    n = sum(q_lens)
    q = queries(n, hq, seed + 1, scale)
    plan = paged.build_plan(cache, hq, q_lens, kv, tables, limits=limits, shared=shared)
    out = torch.full((n + 2, hq, D), 7.0, device="cuda", dtype=BF16)
    paged.paged_attention(q, cache, plan, SCALE, out=out)
    lim = causal(q_lens, kv) if limits is None else torch.as_tensor(limits, device="cuda")
    ref, room = exact(q[:n], q_lens, rows, lim, dtype)
    assert near(out[:n], ref, wider(room, q[:n], q_lens, rows, lim, plan))
    assert (out[n:] == 7).all()
    assert (out[:n][lim == 0] == 0).all()
    assert torch.equal(paged.paged_attention(q, cache, plan, SCALE), out[:n])
    return plan


BOTH = pytest.mark.parametrize("dtype", [BF16, E4M3])


@BOTH
@pytest.mark.parametrize("hq,hk", [(8, 2), (4, 4), (8, 1), (10, 2), (12, 1), (32, 8)])
@pytest.mark.parametrize("n", [2, 3, 17])
def test_one_token_each(n, hq, hk, dtype):
    plan = check([(700, [700 + 1 + 13 * i for i in range(n)])], [1] * n, hq, hk, 64, dtype)
    assert plan._args.tail_count > 0


@BOTH
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("shared", [128, 129, 255, 256, 1000, 6001])
def test_pages_and_lengths(shared, page, dtype):
    check([(shared, [shared + 1, shared + 5, shared + 130, shared + 64])], [1] * 4, 8, 2, page, dtype, seed=shared)


@BOTH
@pytest.mark.parametrize("q_lens", [[5, 5, 5], [1, 8, 3, 0, 2], [0, 0, 1, 1], [8] * 20, [2, 1, 8, 7, 1, 1, 1, 1]])
def test_drafts(q_lens, dtype):
    check([(1300, [1300 + 8 + 31 * i for i in range(len(q_lens))])], q_lens, 8, 2, 32, dtype)
    check([(1300, [1300 - 20 + 8 * q for q in q_lens])] if all(1300 - 20 + 8 * q >= 1300 for q in q_lens) else [(1280, [1280 + q for q in q_lens])],
          q_lens, 8, 2, 32, dtype)


@BOTH
def test_groups_with_chunks_and_others(dtype):
    groups = [(900, [950, 901, 1300]), (0, [40, 500]), (2000, [2001] * 9), (300, [310]), (640, [700, 900, 641, 800]), (129, [129 + 60, 200])]
    q = [1, 1, 2, 1, 3, *[1] * 9, 1, 1, 150, 2, 1, 60, 1]
    plan = check(groups, q, 8, 2, 16, dtype)
    assert plan._args.tail_count > 0 and plan._args.few_count > 0 and plan._args.chunk_count + plan._args.one_count > 0


@BOTH
def test_long_and_wide(dtype):
    check([(20000, [20001 + 7 * i for i in range(40)])], [1] * 40, 16, 2, 64, dtype)
    check([(9000, [9003] * 33), (4000, [5000] * 5)], [3] * 38, 32, 4, 128, dtype)


@BOTH
def test_limits(dtype):
    """Rows that read part of the shared tokens, or nothing."""
    kv = [820, 900, 769, 1500]
    limits = [820, 100, 0, 900, 769, 768, 767, 300, 1500, 640]
    check([(768, kv)], [2, 2, 3, 3], 8, 2, 64, dtype, limits=limits)
    check([(768, kv)], [2, 2, 3, 3], 8, 2, 64, dtype, limits=[0] * 10)
    check([(768, kv)], [2, 2, 3, 3], 8, 2, 64, dtype, limits=[130] * 10)


@BOTH
def test_limits_of_many_rows(dtype):
    """The same where a run has more rows than a CTA of 64: some read part of the shared tokens, some nothing."""
    g = torch.Generator().manual_seed(4)
    kv = [900 + 17 * i for i in range(24)]
    q = [1 + i % 3 for i in range(24)]
    limits = [int(torch.randint(0, k + 1, (), generator=g)) if i % 3 else k for k, n in zip(kv, q) for i in range(n)]
    plan = check([(896, kv)], q, 8, 2, 64, dtype, limits=limits)
    assert plan._args.tail_count > 0
    check([(896, kv)], q, 8, 2, 64, dtype, limits=[0] * sum(q))
    check([(896, kv)], [1] * 24, 32, 4, 16, dtype, limits=[min(k, 128 * i) for i, k in enumerate(kv)])


@BOTH
@pytest.mark.parametrize("n", [5, 40])
def test_in_place_and_two_streams(n, dtype):
    """The output over the queries, and calls of one plan side by side."""
    from sensenova_u1_b200.ops import paged
    cache, tables, kv, _, shared = setup([(1500, [1501 + 9 * i for i in range(n)]), (0, [300, 90])], 64, 2, dtype)
    q = queries(n + 3, 8)
    plan = paged.build_plan(cache, 8, [1] * n + [2, 1], kv, tables, shared=shared)
    want = paged.paged_attention(q, cache, plan, SCALE)
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for i in range(9):
        s = streams[i % 3]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(paged.paged_attention(q, cache, plan, SCALE))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)
    x = q[:n + 3].clone()
    paged.paged_attention(x, cache, plan, SCALE, out=x)
    assert torch.equal(x, want)


@BOTH
def test_tables_that_have_been_cut(dtype):
    """Sequences of a device's tables that are shorter than the plan says: they read what they have, one that is empty reads nothing."""
    from sensenova_u1_b200.ops import _lib, page_tables, paged
    for n in (4, 30):
        cache, tables, kv, _, shared = setup([(640, [700 + i for i in range(n)])], 64, 2, dtype)
        t = page_tables.PageTables(cache, n, 800)
        t.load(kv, tables)
        plan = paged.build_plan(cache, 8, [1] * n, kv, t, shared=shared)
        keep = [k if i % 3 == 0 else 0 if i % 3 == 1 else 333 for i, k in enumerate(kv)]
        t.step(0, keep=torch.tensor(keep, dtype=torch.int32, device="cuda"))
        _lib.check_status()
        q = queries(n, 8)
        out = paged.paged_attention(q, cache, plan, SCALE)
        _lib.check_status()
        held = cache.data.double() if dtype == BF16 else cache.data.double() * cache.scales.double()[..., None]      # (rows have been copied)
        rows = rows_of(held, t.table.tolist(), keep)
        ref, room = exact(q[:n], [1] * n, rows, torch.tensor(keep, device="cuda"), dtype)
        some = [i for i in range(n) if i % 3 != 1]
        full = [r if r.shape[2] else rows[0][:, :, :1] for r in rows]
        room = wider(room, q[:n], [1] * n, full, torch.tensor([max(k, 1) for k in keep], device="cuda"), plan)
        assert near(out[some], ref[some], room[some])
        assert not out[[i for i in range(n) if i % 3 == 1]].any()


@BOTH
def test_no_tokens_beyond_the_shared(dtype):
    check([(512, [512, 512, 513])], [1, 3, 1], 8, 2, 64, dtype)


@BOTH
@pytest.mark.parametrize("scale", [1e-6, 8.0, 300.0])
def test_sizes_of_scores(scale, dtype):
    """Uniform, peaked, and one key that takes all."""
    cache, tables, kv, rows, shared = setup([(1500, [1501 + i for i in range(6)])], 64, 2, dtype, stretch=False)
    from sensenova_u1_b200.ops import paged
    q = queries(6, 8, scale=scale)
    out = paged.paged_attention(q, cache, paged.build_plan(cache, 8, [1] * 6, kv, tables, shared=shared), SCALE)
    ref, room = exact(q[:6], [1] * 6, rows, causal([1] * 6, kv), dtype)
    if scale < 100:
        assert near(out, ref, room)
    else:
        # scores of up to 2^13 log2 units have an fp32 error of 2^-11 and more: neighbours within it may change places
        assert torch.isfinite(out).all() and float((out.double() - ref).norm() / ref.norm()) < 0.05


def test_scales_far_apart():
    """Values (keys) of one token up to 2^40 (2^10) times those of another: the large value decides where its probability is not tiny, and where
    it is hidden the small ones keep their bits."""
    from sensenova_u1_b200.ops import paged
    cache, tables, kv, rows, shared = setup([(1024, [1030 + i for i in range(5)])], 64, 2, E4M3, stretch=False)
    q = queries(5, 8)
    for values, at in [(2.0 ** 40, 5), (2.0 ** -40, 700), (2.0 ** 100, 1000), (2.0 ** -100, 3)]:
        held = cache.scales.clone()
        held[tables[0][at // 64], 1, :, at % 64] *= values
        c2 = paged.PagedCache(cache.data, held)
        r2 = rows_of(cache.data.double() * held.double()[..., None], tables, kv)
        out = paged.paged_attention(q, c2, paged.build_plan(c2, 8, [1] * 5, kv, tables, shared=shared), SCALE)
        assert near(out, *exact(q[:5], [1] * 5, r2, causal([1] * 5, kv), E4M3))
    # the same value for rows that may not read it
    held = cache.scales.clone()
    held[tables[0][900 // 64], 1, :, 900 % 64] *= 2.0 ** 60
    held[tables[0][901 // 64], :, :, 901 % 64] = float("nan")
    c2 = paged.PagedCache(cache.data, held)
    limits = [900, 300, 900, 10, 899]
    out = paged.paged_attention(q, c2, paged.build_plan(c2, 8, [1] * 5, kv, tables, limits=limits, shared=shared), SCALE)
    assert near(out, *exact(q[:5], [1] * 5, rows, torch.tensor(limits, device="cuda"), E4M3))
    out = paged.paged_attention(q, c2, paged.build_plan(c2, 8, [1] * 5, kv, tables, limits=[901, 1000, 902, 300, 1034], shared=shared), SCALE)
    assert torch.isnan(out[1]).all() and torch.isnan(out[2]).all() and torch.isnan(out[4]).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[3]).all()


def test_a_sink_and_many_small():
    """One key has nearly all of the probability, 20000 others 2^-19 of it each: together they count."""
    from sensenova_u1_b200.ops import paged
    for dtype in (BF16, E4M3):
        n = 20096
        x = torch.zeros(n // 64 + 4, 2, 1, 64, D, device="cuda")
        x[:, 0, :, :, 0] = -13.1                               # scores: 0 and -13.1
        x[0, 0, :, 0, 0] = 0
        x[:, 1, :, :, 1] = 1
        x[0, 1, :, 0, 1] = 0
        x = x.to(BF16)
        codes, scales = quantised(x)
        cache = paged.PagedCache(x) if dtype == BF16 else paged.PagedCache(codes, scales)
        held = x.double() if dtype == BF16 else codes.double() * scales.double()[..., None]
        tables = [list(range(n // 64)) + [n // 64 + i] for i in range(4)]
        kv = [n + 1 + i for i in range(4)]
        q = torch.zeros(4, 4, D, device="cuda", dtype=BF16)
        q[:, :, 0] = 1
        out = paged.paged_attention(q, cache, paged.build_plan(cache, 4, [1] * 4, kv, tables, shared=[(0, 4, n)]), 1.0)
        k, v = held[:, 0, 0].flatten(0, 1), held[:, 1, 0].flatten(0, 1)
        for i, t in enumerate(tables):
            at = torch.tensor([p * 64 + o for p in t for o in range(64)][:kv[i]], device="cuda")
            want = torch.softmax(k[at, 0], 0) @ v[at]
            # p of the small ones rounded to fp16: normal numbers (2^-19 of 2^7), so 2^-11 of themselves; the sum and the result 2^-8
            assert ((out[i].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-9).all()


@BOTH
def test_not_finite(dtype):
    """A row that may read a key or value that is not finite is NaN; the others are as if it were not there."""
    from sensenova_u1_b200.ops import paged
    cache, tables, kv, rows, shared = setup([(640, [650, 700, 641, 660])], 64, 2, dtype, stretch=False)
    q = queries(6, 8)
    limits = [600, 650, 500, 641, 10, 559]
    q_lens = [2, 1, 1, 2]
    ref = exact(q[:6], q_lens, rows, torch.tensor(limits, device="cuda"), dtype)
    for side in (0, 1):
        for bad in (float("nan"), float("inf")):
            if dtype == E4M3:
                if bad == float("inf"):
                    continue
                held = cache.scales.clone()
                held[tables[0][560 // 64], side, :, 560 % 64] = bad
                c2 = paged.PagedCache(cache.data, held)
            else:
                data = cache.data.clone()
                data[tables[0][560 // 64], side, :, 560 % 64, 7] = bad
                c2 = paged.PagedCache(data)
            out = paged.paged_attention(q, c2, paged.build_plan(c2, 8, q_lens, kv, tables, limits=limits, shared=shared), SCALE)
            clean = [2, 4, 5]
            assert near(out[clean], ref[0][clean], ref[1][clean])
            if not (side == 0 and bad == float("inf")):        # (a key of infinity gives scores of either sign)
                assert (torch.isnan(out[[0, 1, 3]]).flatten(1).any(1)).all()
    # a query that is not finite is that row's alone
    q2 = q.clone()
    q2[1, 2, 5] = float("nan")
    plan = paged.build_plan(cache, 8, q_lens, kv, tables, limits=limits, shared=shared)
    a, b = paged.paged_attention(q2, cache, plan, SCALE), paged.paged_attention(q, cache, plan, SCALE)
    assert torch.isnan(a[1, 2]).all()
    a[1, 2] = b[1, 2] = 0
    assert torch.equal(a, b)


@BOTH
def test_what_lies_behind_does_not_matter(dtype):
    """Pages of nobody, and rows behind a sequence's last token, hold NaN."""
    from sensenova_u1_b200.ops import paged
    cache, tables, kv, rows, shared = setup([(300, [301, 310, 333])], 128, 2, dtype)
    q = queries(3, 8)
    used = torch.zeros(cache.pages, 128, dtype=torch.bool)
    for t, k in zip(tables, kv):
        for i in range(k):
            used[t[i // 128], i % 128] = True
    raw = cache.data.view(torch.uint8 if dtype == E4M3 else torch.int16)
    raw[:] = torch.where(used.cuda()[:, None, None, :, None], raw, torch.tensor(0x7f if dtype == E4M3 else 0x7fc0, dtype=raw.dtype, device="cuda"))
    if dtype == E4M3:
        cache.scales[:] = torch.where(used.cuda()[:, None, None], cache.scales, float("nan"))
    plan = paged.build_plan(cache, 8, [1] * 3, kv, tables, shared=shared)
    assert near(paged.paged_attention(q, cache, plan, SCALE), *exact(q[:3], [1] * 3, rows, causal([1] * 3, kv), dtype))
    limits = [200, 130, 333]
    plan = paged.build_plan(cache, 8, [1] * 3, kv, tables, limits=limits, shared=shared)
    assert near(paged.paged_attention(q, cache, plan, SCALE), *exact(q[:3], [1] * 3, rows, torch.tensor(limits, device="cuda"), dtype))


@BOTH
def test_growing_in_a_graph(dtype):
    from sensenova_u1_b200.ops import _lib, paged
    cache, tables, kv, _, shared = setup([(700, [701, 760, 720])], 16, 2, dtype, room=40)
    held = cache.data.double() if dtype == BF16 else cache.data.double() * cache.scales.double()[..., None]
    plan = paged.build_plan(cache, 8, [1] * 3, kv, tables, grow=40, shared=shared)
    q = queries(3, 8)
    paged.paged_attention(q, cache, plan, SCALE)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.advance()
        out = paged.paged_attention(q, cache, plan, SCALE)
    for step in range(1, 41):
        graph.replay()
        if step in (1, 9, 40):
            now = [k + step for k in kv]
            assert near(out, *exact(q[:3], [1] * 3, rows_of(held, tables, now), causal([1] * 3, now), dtype))
    _lib.check_status()
    graph.replay()
    with pytest.raises(_lib.NativeLibraryError):
        _lib.check_status()


@BOTH
def test_tables_on_the_device(dtype):
    """Forks, growth and attention without a look by the host: eight beams of one prompt and three of another."""
    from sensenova_u1_b200.ops import _lib, page_tables, paged
    hk, hq, page, beams, lens = 2, 8, 16, (8, 3), (405, 290)
    caches = [paged.PagedCache.empty(300, page, hk, dtype) for _ in range(2)]
    n = sum(beams)
    t = page_tables.PageTables(caches, n, 500)
    first = [0, beams[0]]
    more = torch.zeros(n, dtype=torch.int32)
    more[first] = torch.tensor(lens, dtype=torch.int32)
    t.step(more.cuda(), parents=torch.full((n,), -1, dtype=torch.int32, device="cuda"))
    g = torch.Generator(device="cuda").manual_seed(3)
    kv = [torch.randn(sum(lens), 2 * hk, D, device="cuda", generator=g).to(BF16) for _ in caches]
    prompt = paged.build_plan(caches[0], hq, more.tolist(), more.tolist(), t)
    for c, x in zip(caches, kv):
        paged.paged_write(c, x[:, :hk], x[:, hk:], prompt)
    # what every beam has seen, as rows of kv
    seen = [[list(x.split(lens)[r]) for r, b in enumerate(beams) for _ in range(b)] for x in kv]
    parents = torch.tensor([0] * 8 + [8] * 3, dtype=torch.int32, device="cuda")
    plan = paged.build_plan(caches[0], hq, [1] * n, [lens[0] + 1] * 8 + [lens[1] + 1] * 3, t, grow=30, shared=[(0, 8, lens[0]), (8, 3, lens[1])])
    assert plan._args.tail_count > 0
    with pytest.raises(RuntimeError):
        plan.advance()
    new, q = torch.empty(2, n, 2 * hk, D, device="cuda", dtype=BF16), queries(n, hq)
    outs = []

    def step():
        t.step(1, parents=parents)
        outs.clear()
        for c, x in zip(caches, new):
            paged.paged_write(c, x[:, :hk], x[:, hk:], plan)
            outs.append(paged.paged_attention(q, c, plan, SCALE))

    graph = None
    for i in range(20):
        new.copy_(torch.randn(new.shape, device="cuda", generator=g))
        if i == 1:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        step() if graph is None else graph.replay()
        p = parents.tolist()
        for s, x in zip(seen, new):
            s[:] = [s[p[b]] + [x[b].clone()] for b in range(n)]
        parents.copy_(torch.tensor([torch.randint(0, 8, ()).item() for _ in range(8)] + [8 + torch.randint(0, 3, ()).item() for _ in range(3)]))
    _lib.check_status()
    for s, out in zip(seen, outs):
        rows = []
        for b in range(n):
            x = torch.stack([y for part in s[b] for y in (part if part.dim() == 3 else part[None])])
            if dtype == E4M3:
                codes, scales = quantised(x)
                x = codes.double() * scales.double()[..., None]
            rows.append(x.double().view(-1, 2, hk, D).permute(1, 2, 0, 3))
        lens_now = [r.shape[2] for r in rows]
        assert t.lens.tolist() == lens_now
        assert near(out, *exact(q[:n], [1] * n, rows, causal([1] * n, lens_now), dtype))


def test_bad_page_is_reported():
    from sensenova_u1_b200.ops import _lib, page_tables, paged
    cache = paged.PagedCache(torch.zeros(8, 2, 2, 64, D, device="cuda", dtype=BF16))
    t = page_tables.PageTables(cache, 2, 512)
    plan = paged.build_plan(cache, 8, [1, 1], [400, 400], t, shared=[(0, 2, 384)])
    t.lens.fill_(400)                                        # and no page
    paged.paged_attention(queries(2, 8), cache, plan, SCALE)
    with pytest.raises(_lib.NativeLibraryError, match="page table"):
        _lib.check_status()


def test_tables_that_do_not_fit():
    from sensenova_u1_b200.ops import page_tables, paged
    cache, other, small = (paged.PagedCache.empty(n, p, 2) for n, p in ((8, 64), (8, 32), (4, 64)))
    t = page_tables.PageTables(cache, 2, 512)
    for c, q, kv, kw in [(other, [1, 1], [5, 5], {}), (small, [1, 1], [5, 5], {}), (cache, [1], [5], {}), (cache, [1, 1], [5, 513], {}), (cache, [1, 1], [5, 500], dict(grow=13)),
                         (cache, [1, 1], [5, 5], dict(shared=[(0, 2, 6)]))]:
        with pytest.raises(ValueError):
            paged.build_plan(c, 8, q, kv, t, **kw)
