"""Host side of attention to shared tokens (ops/paged.py): refusals, and that the work covers every row and key once."""
import random

import numpy as np
import pytest

from sensenova_u1_b200.ops import paged


@pytest.fixture(autouse=True)
def always(monkeypatch):
    """Shared however short it is."""
    monkeypatch.setattr(paged, "SHARE_TOKENS", (0, 0))


def lay(q, kv, tables, shared, page=16, group=4, heads=2, fp8=False, limits=None, grow=0, pages=1 << 20):
    return paged._lay_out(list(q), list(kv), tables, page, pages, group, heads, fp8, limits, grow, shared)


def alike(kv, tokens, page):
    """Tables of sequences with the same first pages."""
    head = list(range(tokens // page))
    at = len(head)
    out = []
    for k in kv:
        n = max(0, -(-k // page) - len(head))
        out.append(head[:-(-k // page)] + list(range(at, at + n)))
        at += n
    return out


def test_runs_and_skips():
    kv = [300, 400, 500, 280, 290]
    t = alike(kv, 272, 16)
    a, c = lay([1, 1, 40, 1, 0], kv, t, [(0, 5, 272)])             # the third is a chunk: the first two are together
    assert a["runs"].tolist() == [[0, 2, 0, 256]] and a["skip"].tolist() == [256, 256, 0, 0, 0]
    assert c["few_count"] > 0 and c["chunk_count"] > 0
    a, _ = lay([1, 0, 2, 1, 0], kv, t, [(0, 5, 272)])              # sequences without rows are no hindrance
    assert a["runs"].tolist() == [[0, 4, 0, 256]] and a["skip"].tolist() == [256, 0, 256, 256, 0]
    for q, shared in [([1] * 5, [(0, 5, 127)]), ([1, 0, 0, 0, 0], [(0, 5, 272)]), ([1] * 5, [(0, 1, 272)]), ([40] * 5, [(0, 5, 272)]), ([1] * 5, [])]:
        a, c = lay(q, kv, t, shared)
        assert c["prefix_count"] == c["tail_count"] == c["join_count"] == 0 and a["skip"] is None
    a, c = lay([1] * 5, kv, t, [(3, 2, 256), (0, 2, 272)])
    assert a["runs"].tolist() == [[3, 2, 3, 256], [0, 2, 0, 256]] and a["skip"].tolist() == [256, 256, 0, 256, 256]


@pytest.mark.parametrize("shared", [[(-1, 2, 16)], [(0, 0, 16)], [(0, 6, 16)], [(0, 2, -1)], [(0, 3, 16), (2, 2, 16)], [(0, 2, 301)], [(0, 2.0, 16)], [(0, 2)]])
def test_refusals(shared):
    kv = [300, 400, 500, 280, 290]
    with pytest.raises(ValueError):
        lay([1] * 5, kv, alike(kv, 272, 16), shared)


def test_other_pages_are_refused():
    kv = [300, 300]
    t = alike(kv, 288, 16)
    t[1][3] = 70
    with pytest.raises(ValueError):
        lay([1, 1], kv, t, [(0, 2, 272)])
    t[1][3], t[1][17] = 3, 70                                        # behind the shared tiles it does not matter
    lay([1, 1], kv, t, [(0, 2, 272)])


@pytest.mark.parametrize("seed", range(40))
def test_every_row_and_key_once(seed):
    rng = random.Random(seed)
    page, group, heads = rng.choice((16, 32, 64, 128)), rng.choice((1, 2, 3, 4, 5, 8, 16)), rng.choice((1, 2, 4, 8))
    q, kv, tables, shared, at = [], [], [], [], 0
    for _ in range(rng.randint(1, 4)):
        n, tokens = rng.randint(1, 20), rng.choice((0, 128, 300, 5000))
        lens = [tokens + rng.randint(0, 200) for _ in range(n)]
        new = [min(k, rng.choice((0, 1, 1, 2, 5, 40))) for k in lens]
        shared.append((len(q), n, tokens))
        q, kv = q + new, kv + lens
        for t in alike(lens, tokens // page * page, page):
            tables.append([p + at for p in t])
        at += 4096
    grow = rng.choice((0, 0, 100))
    if grow:
        tables = [t + list(range(at + 100 * i, at + 100 * i + 100)) for i, t in enumerate(tables)]
    fp8 = rng.random() < 0.5
    a, c = lay(q, kv, tables, shared, page, group, heads, fp8, grow=grow)
    rows, n = sum(q), len(q)
    q_start = np.concatenate([[0], np.cumsum(q)])
    direct = np.zeros(rows * group, dtype=int)                       # by few rows and chunks
    tile = {"few": c["few_rows"], "one": 128 // group * group if group <= 128 else 1}
    for name, m in (("few", tile["few"]), ("one", tile["one"]), ("chunk", 2 * tile["one"])):
        for b, row0, z, _ in a[name].tolist():
            if z & 0xffff == 0:
                r = q_start[b] * group + row0
                direct[r:min(r + m, q_start[b + 1] * group)] += 1
    if c["tail_count"] == 0:
        assert c["prefix_count"] == c["many_count"] == 0
        assert (direct == 1).all()
        return
    used = np.zeros(c["partial_rows"], dtype=int)
    where = {}
    for i, (r, row0, z, first) in enumerate(a["prefix"].tolist()):
        part, parts = z & 0xffff, z >> 16
        t0, tokens, seq, skip = a["runs"][r].tolist()
        count = min(64, tokens * group - row0)
        assert count > 0 and skip % 128 == 0 and skip > 0 and 0 <= part < parts <= skip // 128
        used[first:first + 64] += 1
        for k in range(count):
            where.setdefault(t0 * group + row0 + k, []).append(("prefix", part, parts, first + k))
    wide = (128 // group * group) * (1 if fp8 else 2)
    for r, row0, z, first in a["many"].tolist():
        part, parts = z & 0xffff, z >> 16
        t0, end = a["run_start"][r:r + 2].tolist()
        assert r % 2 == 0 and a["run_len"][r] % 128 == 0 and 0 <= part < parts <= a["run_len"][r] // 128 and row0 % group == 0
        used[first:first + wide] += 1
        assert end > t0 and (end - t0) * group > 64 and q_start[a["run_seq"][r]] == t0
        for k in range(min(wide, (end - t0) * group - row0)):
            where.setdefault(t0 * group + row0 + k, []).append(("many", part, parts, first + k))
    for b, row0, z, first in a["tail"].tolist():
        part, parts = z & 0xffff, z >> 16
        m = c["tail_rows"]
        used[first:first + m] += 1
        assert a["skip"][b] > 0 and a["skip"][b] <= kv[b]
        for k in range(min(m, q[b] * group - row0)):
            where.setdefault(q_start[b] * group + row0 + k, []).append(("tail", part, parts, first + k))
    assert used.max() <= 1
    joined = a["joins"].reshape(-1, 8)
    for t, g, pre, parts, tail, tparts, m, mpre in joined.tolist():
        have = sorted(where.pop(t * group + g))
        name = have[0][0]
        assert mpre == (64 if name == "prefix" else wide)
        assert have == sorted([(name, s, parts, pre + mpre * s) for s in range(parts)] + [("tail", s, tparts, tail + m * s) for s in range(tparts)])
        direct[t * group + g] += 1
    assert not where and (direct == 1).all()
    for seq, t0 in zip(a["runs"][:, 2], a["runs"][:, 0]):
        assert q_start[seq] == t0


def test_tables_on_the_device_are_not_looked_at():
    a, c = lay([1, 1], [300, 290], 20, [(0, 2, 288)])
    assert a["table"] is None and a["kv_len"] is None and c["width"] == 20 and c["prefix_count"] > 0
    with pytest.raises(ValueError):
        lay([1, 1], [300, 330], 20, [])


def test_shared_where_it_is_faster(monkeypatch):
    monkeypatch.undo()
    for fp8, n, tokens, heads, want in [(False, 2, 1920, 8, False), (False, 2, 2048, 8, True), (True, 2, 2048, 8, False), (True, 2, 2560, 4, True),
                                        (False, 16, 1024, 8, False), (False, 33, 1024, 8, True), (True, 64, 256, 8, False)]:
        kv = [tokens + 5 + i for i in range(n)]
        a, c = lay([1] * n, kv, alike(kv, tokens, 64), [(0, n, tokens)], page=64, heads=heads, fp8=fp8)
        assert (c["tail_count"] > 0) == want and (c["few_count"] == 0) == want
    kv = [1030] * 20                                                 # several runs together
    t = alike(kv[:10], 1024, 64)
    t += [[p + 10000 for p in x] for x in t]
    assert lay([1] * 20, kv, t, [(0, 10, 1024), (10, 10, 1024)], page=64, heads=16)[1]["tail_count"] > 0
    assert lay([1] * 20, kv, t, [(0, 10, 1024), (10, 10, 1024)], page=64, heads=8)[1]["tail_count"] == 0
