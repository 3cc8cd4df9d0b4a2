"""Block tables on the device (csrc/page_tables.cu) against the same rules in Python."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


class Plain:
    """The rules, sequence by sequence; a page's rows are named by where they were written."""

    def __init__(self, pages, page, seqs):
        self.page, self.tables, self.lens, self.refs = page, [[] for _ in range(seqs)], [0] * seqs, [0] * pages

    def step(self, tokens, parents=None, keep=None):
        n, page = len(self.lens), self.page
        parents = list(range(n)) if parents is None else parents
        kept = [0 if p < 0 else min(self.lens[p], self.lens[p] if keep is None else max(0, keep[i])) for i, p in enumerate(parents)]
        new = [self.tables[p][:k // page] if p >= 0 else [] for p, k in zip(parents, kept)]
        refs = [0] * len(self.refs)
        for t in new:
            for p in t:
                refs[p] += 1
        whole, taken, jobs = list(refs), {}, []
        for i, (p, k) in enumerate(zip(parents, kept)):
            if k % page:
                src = self.tables[p][k // page]
                if whole[src] == 0 and src not in taken:
                    taken[src] = i
                    refs[src] = 1
                    new[i] = new[i] + [src]
                else:
                    jobs.append((i, src, k % page))
        free = iter([p for p, r in enumerate(refs) if r == 0])
        todo, copies = {i: (src, m) for i, src, m in jobs}, []
        for i, k in enumerate(kept):
            more = tokens if isinstance(tokens, int) else tokens[i]
            self.lens[i] = k + more
            while len(new[i]) * page < k + more:
                p = next(free)
                if i in todo and len(new[i]) == k // page:
                    copies.append((todo[i][0], p, todo[i][1]))
                refs[p] = 1
                new[i] = new[i] + [p]
        self.tables, self.refs = new, refs
        return copies


def caches(pages, page, hk, dtype, layers, seed=0):
    from sensenova_u1_b200.ops import paged
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for _ in range(layers):
        x = torch.randn(pages, 2, hk, page, 128, generator=g, device="cuda")
        out.append(paged.PagedCache(x.to(dtype), torch.rand(x.shape[:4], generator=g, device="cuda") if dtype == E4M3 else None))
    return out


def same(t, plain):
    want = torch.full((t.seqs, t.width), -1, dtype=torch.int32)
    for i, p in enumerate(plain.tables):
        want[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
    assert torch.equal(t.table.cpu(), want)
    assert t.lens.tolist() == plain.lens and t.refs.tolist() == plain.refs


def on(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def raw(x):
    return x.view(torch.uint8) if x.dtype == E4M3 else x.view(torch.int16)


@pytest.mark.parametrize("page,hk,dtype,layers", [(16, 3, BF16, 2), (64, 1, E4M3, 3), (128, 2, BF16, 1), (32, 4, E4M3, 1)])
@pytest.mark.parametrize("seqs,most", [(1, 300), (5, 700), (33, 260), (600, 90), (1024, 40)])
def test_random_walks(page, hk, dtype, layers, seqs, most):
    from sensenova_u1_b200.ops import _lib, page_tables
    rng = random.Random(seqs * page)
    pages = seqs * (-(-most // page) + 1) + 5
    cs = caches(pages, page, hk, dtype, layers)
    t, plain = page_tables.PageTables(cs, seqs, most), Plain(pages, page, seqs)
    for step in range(14):
        kind = rng.choice(("grow", "ragged", "beams", "drafts", "come and go", "all"))
        if step == 0 or kind == "come and go":
            parents = [rng.choice((-1, i)) if step else -1 for i in range(seqs)]
            tokens = [rng.choice((0, 1, rng.randint(0, most))) if p < 0 else rng.randint(0, most - plain.lens[p]) // 4 for p in parents]
            args = (tokens, parents, None)
        elif kind in ("grow", "ragged"):
            room = most - max(plain.lens)
            args = (min(room, 1), None, None) if kind == "grow" else ([rng.randint(0, most - n) // 3 for n in plain.lens], None, None)
        elif kind == "beams":
            parents = [rng.randint(0, i) for i in range(seqs)]
            args = ([min(1, most - plain.lens[p]) for p in parents], parents, None)
        elif kind == "drafts":
            args = (0, None, [max(0, n - rng.randint(0, 40)) for n in plain.lens])
        else:
            parents = [rng.randint(-1, seqs - 1) for _ in range(seqs)]
            keep = [rng.randint(-3, most + 5) for _ in range(seqs)]
            kept = [0 if p < 0 else max(0, min(plain.lens[p], k)) for p, k in zip(parents, keep)]
            args = ([rng.randint(0, most - k) // 2 for k in kept], parents, keep)
        tokens, parents, keep = args
        before = [(raw(c.data).clone(), None if c.scales is None else c.scales.clone()) for c in cs]
        copies = plain.step(tokens, parents, keep)
        t.step(tokens if isinstance(tokens, int) else on(tokens), parents=None if parents is None else on(parents), keep=None if keep is None else on(keep))
        _lib.check_status()
        same(t, plain)
        for c, (data, scales) in zip(cs, before):
            for src, dst, n in copies:
                data[dst, :, :, :n] = raw(c.data)[src, :, :, :n]
                if scales is not None:
                    scales[dst, :, :, :n] = c.scales[src, :, :, :n]
            assert torch.equal(raw(c.data), data)                      # the copies and nothing else
            assert scales is None or torch.equal(c.scales, scales)
        # no page that is not full is held twice
        for p, n in zip(plain.tables, plain.lens):
            assert n % page == 0 or plain.refs[p[-1]] == 1


def test_load_and_fork_of_a_prompt():
    from sensenova_u1_b200.ops import page_tables
    cs = caches(40, 16, 2, BF16, 2)
    t, plain = page_tables.PageTables(cs, 6, 200), Plain(40, 16, 6)
    plain.tables, plain.lens = [[7, 3, 11], [7, 3, 20], [], [5], [7], []], [40, 48, 0, 16, 16, 0]
    for p in sum(plain.tables, []):
        plain.refs[p] += 1
    t.load(plain.lens, plain.tables)
    same(t, plain)
    parents = [0, 0, 0, 0, 1, 3]
    plain.step(1, parents)
    t.step(1, parents=on(parents))
    same(t, plain)
    for lens, tables in [([1] * 5, [[0]] * 5), ([17] + [0] * 5, [[1]] + [[]] * 5), ([1, 1, 0, 0, 0, 0], [[4], [4], [], [], [], []]),
                         ([33, 0, 0, 0, 0, 0], [[4, 5, 4], [], [], [], [], []]), ([16, 0, 0, 0, 0, 0], [[40], [], [], [], [], []]),
                         ([209, 0, 0, 0, 0, 0], [list(range(14)), [], [], [], [], []]), ([-1] + [0] * 5, [[]] * 6), ([1.5] + [0] * 5, [[1]] + [[]] * 5)]:
        with pytest.raises(ValueError):
            t.load(lens, tables)
    same(t, plain)


def test_captured_and_on_another_stream():
    from sensenova_u1_b200.ops import page_tables
    cs = caches(100, 16, 2, E4M3, 2)
    t, plain = page_tables.PageTables(cs, 8, 300), Plain(100, 16, 8)
    parents = on([-1] * 8)
    t.step(21, parents=parents)
    plain.step(21, [-1] * 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t.step(1, parents=parents)
    rng = random.Random(3)
    side = torch.cuda.Stream()
    for i in range(20):
        p = [rng.randint(0, 7) for _ in range(8)]
        parents.copy_(on(p))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        plain.step(1, p)
        same(t, plain)


def test_what_is_reported():
    from sensenova_u1_b200.ops import _lib, page_tables
    cs = caches(6, 16, 1, BF16, 1)
    t = page_tables.PageTables(cs, 3, 64)
    t.step(33)                                      # nine pages of six: in order, then none
    with pytest.raises(_lib.NativeLibraryError):
        _lib.check_status()
    assert t.table.tolist() == [[0, 1, 2, -1], [3, 4, 5, -1], [-1] * 4] and t.refs.tolist() == [1] * 6
    t.step(0, keep=on([5, 16, 33]))                 # the one that has none keeps none, and nothing is out of range
    _lib.check_status() if t.refs.tolist() == [1, 0, 0, 1, 0, 0] else None
    t.step(0, parents=on([-1] * 3))
    try:
        _lib.check_status()
    except _lib.NativeLibraryError:
        pass
    assert t.refs.tolist() == [0] * 6 and t.lens.tolist() == [0] * 3 and (t.table == -1).all()
    t.step(65)                                      # more than a table has room for
    with pytest.raises(_lib.NativeLibraryError):
        _lib.check_status()
    t = page_tables.PageTables(cs, 3, 64)
    t.step(1, parents=on([0, 3, -2]))               # nobody's children
    with pytest.raises(_lib.NativeLibraryError):
        _lib.check_status()
    assert t.lens.tolist() == [1, 1, 1]


def test_refusals():
    from sensenova_u1_b200.ops import page_tables
    cs = caches(6, 16, 1, BF16, 2)
    for args in [([], 3, 64), (cs, 0, 64), (cs, 1025, 64), (cs, 3, 0), (cs + caches(7, 16, 1, BF16, 1), 3, 64), (cs + caches(6, 32, 1, BF16, 1), 3, 64),
                 (cs + caches(6, 16, 1, E4M3, 1), 3, 64), (cs + cs[:1], 3, 64)]:
        with pytest.raises(ValueError):
            page_tables.PageTables(*args)
    t = page_tables.PageTables(cs[0], 3, 64)
    for kw in [dict(tokens=-1), dict(tokens=1.0), dict(tokens=on([1, 1])), dict(tokens=torch.ones(3, dtype=torch.int32)), dict(tokens=1, parents=on([0, 1])),
               dict(tokens=1, parents=torch.zeros(3, dtype=torch.int64, device="cuda")), dict(tokens=1, keep=on([[1, 2, 3]])), dict(tokens=1, keep=[1, 2, 3]),
               dict(tokens=1, parents=on([0, 0, 1, 0, 2, 0])[::2])]:
        with pytest.raises(ValueError):
            t.step(**kw)
    assert t.lens.tolist() == [0, 0, 0]


def test_a_large_pool_and_long_tables():
    """Free pages far apart in a pool of 70000, tables of 2048 pages."""
    from sensenova_u1_b200.ops import _lib, page_tables, paged
    pages, page, seqs = 70000, 16, 33
    cache = paged.PagedCache.empty(pages, page, 1)
    t, plain = page_tables.PageTables(cache, seqs, 2048 * page), Plain(pages, page, seqs)
    parents = [-1] * seqs
    lens = [2048 * page - 20 - 16 * i for i in range(seqs)]
    for args in [(lens, parents, None), ([0] * seqs, [i if i % 3 else -1 for i in range(seqs)], None), ([5] * seqs, [1, 1] + [2] * 20 + list(range(22, 33)), None),
                 ([17] * seqs, list(range(seqs)), [1000 * i for i in range(seqs)])]:
        plain.step(*args)
        t.step(on(args[0]), parents=on(args[1]), keep=None if args[2] is None else on(args[2]))
        _lib.check_status()
        same(t, plain)
