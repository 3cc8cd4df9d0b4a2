"""Host side of the paged cache (ops/paged.py): refusals, page tables, and how the work is split."""
import numpy as np
import pytest
import torch

from sensenova_u1_b200.ops import paged


def lay(q=(1, 3), kv=(5, 40), tables=((0,), (1, 2, 3)), page=16, pages=4, group=4, heads=2, limits=None, grow=0):
    return paged._lay_out(list(q), list(kv), [list(t) for t in tables], page, pages, group, heads, False, limits, grow)


def test_arrays():
    a, c = lay()
    assert a["q_start"].tolist() == [0, 1, 4] and a["k_start"].tolist() == [0, 5, 45] and a["row_seq"].tolist() == [0, 1, 1, 1]
    assert a["table"].tolist() == [[0, 0, 0], [1, 2, 3]] and a["behind"] is None
    assert a["read_pages"].tolist() == [[0, 0], [1, 0], [1, 1], [1, 2]]
    assert c["rows"] == 4 and c["read_count"] == 4 and c["width"] == 3


def test_limits_are_kept_from_the_end():
    a, _ = lay(limits=[5, 0, 40, 39])
    assert a["behind"].tolist() == [0, 40, 0, 1]


@pytest.mark.parametrize("change", [
    dict(q=(1, 41)),                                     # more new tokens than tokens
    dict(q=(-1, 3)),
    dict(kv=(5,)),
    dict(grow=-1),
    dict(tables=((0,),)),                                # a table missing
    dict(tables=((0,), (1, 2))),                         # a page missing
    dict(grow=9, tables=((0,), (1, 2, 3))),              # no page for what may be added
    dict(tables=((0,), (1, 2, 4))),                      # a page that does not exist
    dict(tables=((0,), (1, -1, 3))),
    dict(limits=[5, 0, 40]),                             # a limit missing
    dict(limits=[5, 0, 40, 41]),                         # beyond the sequence
    dict(limits=[5, -1, 40, 39]),
    dict(limits=[5, 0, 40, 39], grow=1, tables=((0,), (1, 2, 3))),
    dict(kv=(1 << 30, 40)),
])
def test_refusals(change):
    with pytest.raises(ValueError):
        lay(**change)


def test_page_tables_as_a_tensor():
    a, _ = lay(tables=torch.tensor([[0, 77, 99], [1, 2, 3]]))          # what a table holds beyond its pages is ignored
    assert a["table"].tolist() == [[0, 0, 0], [1, 2, 3]]
    with pytest.raises(ValueError):
        paged._lay_out([1], [1], torch.zeros(1, dtype=torch.int32), 16, 4, 1, 1, False, None, 0)


def test_sequences_without_rows_or_keys():
    a, c = lay(q=(0, 0, 0), kv=(0, 7, 0), tables=((), (2,), ()))
    assert c["rows"] == 0 and c["few_count"] == 0 and c["merge_count"] == 0 and c["read_count"] == 1
    a, c = paged._lay_out([], [], [], 16, 4, 1, 1, False, None, 0)
    assert c["seqs"] == 0 and c["rows"] == 0


@pytest.mark.parametrize("group,heads", [(1, 1), (4, 8), (3, 5), (8, 4), (100, 1)])
@pytest.mark.parametrize("q,kv", [([1], [840]), ([1] * 24, [62 + 60 * i for i in range(24)]), ([1] * 700, [17] * 700),
                                  ([5, 0, 17, 1], [12000, 3, 17, 1]), ([300], [30000]), ([1] * 3, [0 + 1, 64, 65])])
def test_every_row_meets_every_key_once(q, kv, group, heads):
    page, n = 16, len(q)
    need = [-(-k // page) for k in kv]
    tables = [list(range(sum(need[:i]), sum(need[:i + 1]))) for i in range(n)]
    a, c = paged._lay_out(q, kv, tables, page, sum(need), group, heads, True, None, 0)
    parts, written = {}, set()
    for name, m in (("few", c["few_rows"]), ("chunk", 2 * (128 // group) * group), ("one", 128 // group * group)):
        if a[name] is None:
            continue
        for b, row0, z, at in a[name].tolist():
            part, count = z & 0xffff, z >> 16
            parts.setdefault((b, row0, m, count), []).append(part)
            assert (at < 0) == (count == 1 or name == "few" and c["few_cluster"] > 1)
            if at >= 0:                                               # nobody else's scratch
                rows = set(range(at, at + m))
                assert not rows & written and at + m <= c["partial_rows"]
                written |= rows
    seen = {}
    for (b, row0, m, count), got in parts.items():
        assert sorted(got) == list(range(count))
        for r in range(row0, min(row0 + m, q[b] * group)):
            assert (b, r) not in seen
            seen[(b, r)] = count
    assert len(seen) == sum(q) * group
    joined = {}
    for b, row0, z, at in a["merge"].tolist():                        # up to four rows each
        assert 1 <= (z >> 12 & 15) <= 4
        for r in range(row0, row0 + (z >> 12 & 15)):
            assert (b, r) not in joined
            joined[(b, r)] = (z & 0xfff, z >> 16, at + r - row0)
    if c["few_cluster"] > 1:                                          # the parts of every tile of rows side by side
        k = c["few_cluster"]
        assert len(a["few"]) % k == 0 and len(a["few"]) * heads <= 444
        assert [z for _, _, z, _ in a["few"].tolist()] == [i % k | k << 16 for i in range(len(a["few"]))]
        assert all(len({tuple(x) for x in a["few"][i:i + k, :2].tolist()}) == 1 for i in range(0, len(a["few"]), k))
    assert set(joined) == {(b, r) for (b, r), count in seen.items() if count > 1 and (
        c["few_rows"] > paged.FEW_JOIN and c["few_cluster"] == 1 or q[b] * group > paged.CHUNK_FROM and group <= 128)}
    first = {(b, row0): at for b, row0, z, at in a["few"].tolist() if at >= 0 and z & 0xffff == 0}
    for b, row0, z, at in a["few"].tolist():                          # joined by the parts themselves: side by side, in whole parts
        assert at < 0 or at == first[(b, row0)] + (z & 0xffff) * c["few_rows"] and at % c["few_rows"] == 0
        assert at < 0 or c["few_rows"] > paged.FEW_JOIN or at < c["few_parts"] * c["few_rows"]
    for b, row0, z, at in a["chunk"].tolist() + a["one"].tolist():
        if at >= 0:
            for r in range(row0, q[b] * group):
                count, m, first = joined[(b, r)]
                assert count == z >> 16 and (r - row0 >= m or at + r - row0 == first + (z & 0xffff) * m)
                if r - row0 + 1 >= m:
                    break
    if c["unpack_count"]:                                             # every key of a chunk's sequence has its place
        wide = [-(-k // 128) if any(b == i for b, *_ in a["chunk"].tolist()) else 0 for i, k in enumerate(kv)]
        assert c["unpack_count"] == sum(wide) and a["unpack_first"].tolist() == [sum(wide[:i]) for i in range(n)]
        assert a["unpack"].tolist() == [[i, y] for i in range(n) for y in range(wide[i])]


def test_parts_fill_one_wave():
    """Parts are as short as they can be while their CTAs run at once."""
    for tiles, heads in ((np.array([500]), 8), (np.array([64, 3, 200]), 8), (np.array([10] * 48), 4)):
        parts = paged._shares(tiles, heads, 296, 4)
        assert parts.sum() * heads <= 296
        share = -(-tiles // parts).max()
        assert share <= 4 or (-(-tiles // (share - 1))).sum() * heads > 296


def test_a_cache_is_refused_in_host_memory():
    data = torch.zeros(2, 2, 1, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        paged.PagedCache(data)
    for bad in (data[..., :64], data[:, :1], data.float(), data.view(2, 2, 2, 8, 128), data.transpose(2, 3)):
        with pytest.raises(ValueError):
            paged.PagedCache(bad)
    with pytest.raises(ValueError):
        paged.PagedCache(data, torch.zeros(2, 2, 1, 16))                # bf16 has no scales
    with pytest.raises(ValueError):
        paged.PagedCache(data.to(torch.float8_e4m3fn))                  # e4m3 has
    with pytest.raises(ValueError):
        paged.PagedCache(data.to(torch.float8_e4m3fn), torch.zeros(2, 2, 16))


def test_the_plan_has_the_fields_of_the_kernels():
    """ops/paged.py hands ``Plan`` of csrc/paged.cuh over by address: the same fields in the same order, or nothing is where it should be."""
    import re
    from pathlib import Path
    src = (Path(paged.__file__).parent.parent / "csrc" / "paged.cuh").read_text()
    body = src[src.index("struct Plan {"):]
    names = []
    for line in body[:body.index("};")].splitlines()[1:]:
        m = re.match(r"\s*(const int\d?\*|int)\s+([^;]*);", line)
        if m:
            kind = paged.c_void_p if "*" in m.group(1) else paged.c_int
            names += [(x.strip(), kind) for x in m.group(2).split(",")]
    assert names == paged._Args._fields_
    assert f"PLAN_LAYOUT = {paged.PLAN_LAYOUT:#x}" in src


@pytest.mark.parametrize("tables", [torch.tensor([[0, 0, 0], [1, 2, (1 << 32) + 3]]),           # would be page 3 in 32 bits
                                    torch.tensor([[0, 0, 0], [1, 2, -(1 << 32)]]), torch.zeros(2, 3)])
def test_page_numbers_that_are_none(tables):
    with pytest.raises(ValueError):
        paged._lay_out([1, 3], [5, 40], tables, 16, 4, 4, 2, False, None, 0)


def test_rows_of_a_tile():
    rows = lambda n, fp8, keys=100: paged._lay_out([n], [keys], [range(-(-keys // 64))], 64, 2000, 1, 8, fp8, None, 0)[1]["few_rows"]
    for fp8 in (False, True):
        assert [rows(n, fp8) for n in (1, 8, 9, 16, 25, 32)] == [8, 8, 16, 16, 32, 32]
    assert [rows(n, True) for n in (17, 24)] == [24, 24]
    assert [rows(n, False) for n in (17, 24)] == [32, 32] and [rows(n, False, 40000) for n in (16, 17, 24, 25)] == [16, 24, 24, 32]


def test_a_captured_step_has_buffers_of_its_own(monkeypatch):
    """The engine's buffers are replaced by larger ones; a graph must not have been captured with them."""
    from types import SimpleNamespace
    from sensenova_u1_b200.inference.engine import InferenceEngine
    eng = InferenceEngine.__new__(InferenceEngine)
    eng.cfg, eng.dev, eng.ws = SimpleNamespace(num_layers=1, hidden_size=8), torch.device("cpu"), object()
    eng.p = {"embed_tokens": torch.zeros(4, 8, dtype=torch.bfloat16)}
    used = []
    eng.layers = lambda x, *a, ws=None, **k: (used.append(ws), x)[1]
    plan = SimpleNamespace(rows=2, positions=lambda: torch.zeros(2, dtype=torch.int32))
    for capturing in (False, True, True):
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
        eng.paged_step(plan, [None], ids=torch.tensor([1, 2]))
    assert used[0] is None and used[1] is not None and used[2] is not None and len({id(x) for x in [*used, eng.ws]}) == 4


@pytest.mark.parametrize("change", [dict(q=(1.0, 3)), dict(kv=(5, 40.5)), dict(kv=(5, float("nan"))), dict(tables=((0,), (1, 2.9, 3))), dict(limits=[5, 0, 40, 39.5]),
                                    dict(tables=((0,), (1, 2, float("inf"))))])
def test_numbers_that_are_not_whole_are_refused(change):
    """(Not cut to whole ones: page 2.9 is not page 2.)"""
    with pytest.raises(ValueError, match="whole"):
        lay(**change)


@pytest.mark.parametrize("tables", [np.array([[0, 0, 0], [1, 2.5, 3]]), torch.zeros(2, 3, dtype=torch.bool), [np.array([0.0]), np.array([1, 2, 3])]])
def test_page_tables_that_are_not_whole_numbers(tables):
    with pytest.raises(ValueError):
        paged._lay_out([1, 3], [5, 40], tables, 16, 4, 4, 2, False, None, 0)


def test_whole_numbers_of_any_type():
    want, _ = lay(limits=[5, 0, 40, 39])
    for kind in (np.int32, np.uint8, np.int64):
        a, _ = paged._lay_out(np.array([1, 3], kind), torch.tensor([5, 40]), [np.array([0], kind), torch.tensor([1, 2, 3])], 16, 4, 4, 2, False,
                              np.array([5, 0, 40, 39], kind), 0)
        assert all(np.array_equal(a[n], want[n]) for n in ("q_start", "kv_len", "table", "behind"))


def test_a_capture_on_the_cache_s_device_counts(monkeypatch):
    """The plan's arrays go up on the current stream of the cache's device, whichever device is current."""
    from types import SimpleNamespace
    current = [0]

    class Device:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *a):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[0] == 1)
    monkeypatch.setattr(paged, "_lay_out", lambda *a: (_ for _ in ()).throw(KeyError("laid out")))
    cache = SimpleNamespace(kv_heads=1, device=torch.device("cuda:1"), page=16, pages=1, scales=None)
    with pytest.raises(RuntimeError, match="captured"):
        paged.build_plan(cache, 1, [1], [1], [[0]])
    cache.device, current[0] = torch.device("cuda:0"), 1
    with pytest.raises(KeyError):
        paged.build_plan(cache, 1, [1], [1], [[0]])
    assert current == [1]


def test_a_library_with_plans_of_another_size_is_refused(monkeypatch):
    from types import SimpleNamespace
    from sensenova_u1_b200.ops import _lib
    if _lib.available():
        assert _lib.load().snu1_paged_plan_bytes() == paged.ctypes.sizeof(paged._Args)
    old = SimpleNamespace(snu1_paged_plan_bytes=lambda: paged.ctypes.sizeof(paged._Args) - 8)
    monkeypatch.setattr(paged, "_ENTRY", {})
    monkeypatch.setattr(_lib, "load", lambda: old)
    with pytest.raises(_lib.NativeLibraryError, match="build"):
        paged._library()
    assert not paged._ENTRY
