"""Attention of sequences that share their first tokens: values of any size, what is not finite far below, tables that change behind a plan."""
import pytest
import torch

from test_paged_gpu import BF16, D, E4M3, causal, exact, near, quantised
from test_paged_shared_gpu import queries, rows_of, setup, wider

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("dtype", [BF16, E4M3])


@pytest.fixture(autouse=True)
def always(monkeypatch):
    """Shared however short it is."""
    from sensenova_u1_b200.ops import paged
    monkeypatch.setattr(paged, "SHARE_TOKENS", (0, 0))


def as_chunks(monkeypatch, wanted):
    """Runs of more than 64 rows go to the kernel for chunks, whatever is faster."""
    from sensenova_u1_b200.ops import paged
    if wanted:
        monkeypatch.setattr(paged, "MANY_COST", ((0.0, 0.01), (0.0, 0.01)))


def caches(x, dtype):
    """A cache of pages ``x``, and what it holds in 64 bits."""
    from sensenova_u1_b200.ops import paged
    if dtype == BF16:
        return paged.PagedCache(x.to(BF16)), x.to(BF16).double()
    codes, scales = quantised(x.to(BF16))
    return paged.PagedCache(codes, scales), codes.double() * scales.double()[..., None]


def ramp(n, shared, page, score, g):
    """Pages of ``n`` sequences: random values, and keys whose first number is ``score`` (nats) of their place; tables and lengths."""
    whole = shared // page
    x = torch.zeros(whole + n, 2, 1, page, D, device="cuda")
    x[:, 1] = torch.randn(whole + n, 1, page, D, device="cuda", generator=g)
    for p in range(whole):
        for i in range(page):
            x[p, 0, :, i, 0] = score(p * page + i)
    x[whole:, 0, :, :, 0] = score(shared)
    return x, [list(range(whole)) + [whole + i] for i in range(n)], [shared + 1 + i % page for i in range(n)]


@BOTH
@pytest.mark.parametrize("n", [4, 24])
@pytest.mark.parametrize("side", ["shared", "own", "part"])
def test_not_finite_far_below(side, n, dtype, monkeypatch):
    """A value that is not finite makes the row NaN however small its probability is, with and without shared reads."""
    from sensenova_u1_b200.ops import paged
    as_chunks(monkeypatch, n > 16)
    g = torch.Generator(device="cuda").manual_seed(1)
    shared = 4096
    score = {"shared": lambda t: 0.0 if t < shared else 200.0, "own": lambda t: 200.0 if t < shared else 0.0, "part": lambda t: 200.0 if 3000 <= t < 3010 else 0.0}[side]
    x, tables, kv = ramp(n, shared, 64, score, g)
    at = (0, 5) if side != "own" else (tables[1][-1], 0)                     # a page and a place
    cache, _ = caches(x, dtype)
    if dtype == BF16:
        cache.data[at[0], 1, 0, at[1], 3] = float("nan")
    else:
        cache.scales[at[0], 1, 0, at[1]] = float("nan")
    q = torch.zeros(n, 4, D, device="cuda", dtype=BF16)
    q[..., 0] = 1
    for plan in (paged.build_plan(cache, 4, [1] * n, kv, tables, shared=[(0, n, shared)]), paged.build_plan(cache, 4, [1] * n, kv, tables)):
        assert (plan._args.many_count > 0) == (plan._args.tail_count > 0 and n > 16)
        bad = torch.isnan(paged.paged_attention(q, cache, plan, 1.0)).flatten(1).any(1)
        assert bad.tolist() == [side != "own" or i == 1 for i in range(n)]


@BOTH
@pytest.mark.parametrize("n", [4, 24, 25])
@pytest.mark.parametrize("rise", [5, 10, 20, 31, 33, 50, 100])
def test_large_values(rise, n, dtype, monkeypatch):
    """Values of up to 2^100 (e4m3: 2^110 of scale), where the largest score is ``rise`` log2 units above those that the maxima begin at."""
    from sensenova_u1_b200.ops import _lib, paged
    as_chunks(monkeypatch, n > 24)
    g = torch.Generator(device="cuda").manual_seed(rise)
    x, tables, kv = ramp(n, 2048, 64, lambda t: 0.0 if t != 700 and t < 2048 else rise * 0.6931, g)
    x[:, 1] *= 2.0 ** 100
    cache, held = caches(x, dtype)
    if dtype == E4M3:                                       # the largest code is 448
        up = 2.0 ** 110 / cache.scales[:, 1].amax()
        cache.scales[:, 1] *= up
        held[:, 1] *= up.double()
    q = torch.zeros(n, 4, D, device="cuda", dtype=BF16)
    q[..., 0] = 1
    plan = paged.build_plan(cache, 4, [1] * n, kv, tables, shared=[(0, n, 2048)])
    assert plan._args.tail_count > 0 and (plan._args.many_count > 0) == (n > 24)
    out = paged.paged_attention(q, cache, plan, 1.0)
    _lib.check_status()
    assert torch.isfinite(out).all()
    q = q / D ** -0.5                                       # (exact has a scale of its own)
    rows = rows_of(held, tables, kv)
    ref, room = exact(q, [1] * n, rows, causal([1] * n, kv), dtype)
    room = wider(room, q, [1] * n, rows, causal([1] * n, kv), plan)
    assert near(out * 2.0 ** -60, ref * 2.0 ** -60, room * 2.0 ** -60)


@BOTH
@pytest.mark.parametrize("n", [5, 30, 31])
def test_requests_that_come_and_go_behind_a_plan(n, dtype, monkeypatch):
    """The first sequence of a run ends and another request takes its place; others are cut inside the shared tokens and grow again.  Every one reads
    its own tokens, as the tables are."""
    from sensenova_u1_b200.ops import _lib, page_tables, paged
    as_chunks(monkeypatch, n > 30)
    cache, tables, kv, _, shared = setup([(640, [700 + i for i in range(n)])], 64, 2, dtype, room=400, stretch=False)
    t = page_tables.PageTables(cache, n, 1000)
    t.load(kv, tables)
    plan = paged.build_plan(cache, 8, [1] * n, [1000] * n, t, shared=shared)
    assert plan._args.tail_count > 0 and (plan._args.many_count > 0) == (n > 30)
    q = queries(n, 8)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")

    def look():
        _lib.check_status()
        out = paged.paged_attention(q, cache, plan, 128 ** -0.5)
        _lib.check_status()
        held = cache.data.double() if dtype == BF16 else cache.data.double() * cache.scales.double()[..., None]
        lens = t.lens.tolist()
        some = [i for i in range(n) if lens[i]]
        rows = rows_of(held, t.table.tolist(), lens)
        ref, room = exact(q[:n], [1] * n, rows, ints(lens), dtype)
        full = [r if r.shape[2] else rows[some[0]][:, :, :1] for r in rows]
        room = wider(room, q[:n], [1] * n, full, ints([max(k, 1) for k in lens]), plan)
        assert near(out[some], ref[some], room[some])
        assert not out[[i for i in range(n) if not lens[i]]].any()

    look()
    own = list(range(n))
    t.step(0, parents=ints([-1] + own[1:]))                                  # the first one ends
    look()
    t.step(ints([300] + [1] * (n - 1)), parents=ints([-1] + own[1:]), keep=ints([0, 1000, 333, 128, 0] + [1000] * (n - 5)))
    look()                                                                   # 333 and 128 are 334 and 129 now, with a token of their own
    for more in (1, 60, 200):
        t.step(more if more < 200 else ints([200] * 4 + [1] * (n - 4)))
        look()


@BOTH
def test_cut_and_grown_all_together(dtype):
    """All sequences are cut to the same place and go on differently."""
    from sensenova_u1_b200.ops import _lib, page_tables, paged
    n = 4
    cache, tables, kv, _, shared = setup([(640, [700 + i for i in range(n)])], 32, 2, dtype, room=400, stretch=False)
    t = page_tables.PageTables(cache, n, 1000)
    t.load(kv, tables)
    plan = paged.build_plan(cache, 8, [1] * n, [1000] * n, t, shared=shared)
    t.step(100, keep=torch.full((n,), 270, dtype=torch.int32, device="cuda"))
    q = queries(n, 8)
    out = paged.paged_attention(q, cache, plan, 128 ** -0.5)
    _lib.check_status()
    held = cache.data.double() if dtype == BF16 else cache.data.double() * cache.scales.double()[..., None]
    rows = rows_of(held, t.table.tolist(), [370] * n)
    assert near(out, *exact(q[:n], [1] * n, rows, torch.full((n,), 370, device="cuda"), dtype))
