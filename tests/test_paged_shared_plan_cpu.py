"""Host side of attention to shared tokens (ops/paged.py): runs of different lengths in one plan."""
import numpy as np
import pytest

from sensenova_u1_b200.ops import paged
from test_paged_shared_cpu import alike, lay


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("short,count", [(256, 20), (2560, 18), (2560, 60)])
def test_a_long_run_beside_many_short_ones_is_split(short, count, fp8):
    """However many CTAs the short ones take: it was left whole, and one CTA per head read all of it."""
    kv, tables, shared, at = [], [], [], 0
    for n, tokens in [(8, 40000)] + [(4, short)] * count:
        shared.append((len(kv), n, tokens))
        kv += [tokens + 60] * n
        tables += [[p + at for p in t] for t in alike([tokens + 60] * n, tokens, 64)]
        at += 4096
    a, c = lay([1] * len(kv), kv, tables, shared, page=64, heads=8, fp8=fp8)
    runs, prefix = a["runs"], a["prefix"]
    parts = {int(r): z >> 16 for r, _, z, _ in prefix.tolist()}
    first = int(np.argmax(runs[:, 3]))
    assert parts[first] >= 8
    # no item much longer than all the work over all SMs
    tiles = max(runs[r, 3] // 128 / n for r, n in parts.items())
    assert tiles <= max(2 * 8 * sum(runs[r, 3] // 128 for r in parts) / 148, 25)


@pytest.mark.parametrize("kind", ["array", "tensor", "list", "none"])
def test_shared_as_an_array(monkeypatch, kind):
    """``shared`` as lengths and tables may be given: several entries in one array had no truth value."""
    import torch
    seen = []
    monkeypatch.setattr(paged, "_lay_out", lambda *a: seen.append(a[-1]) or 1 / 0)

    class Cache:
        kv_heads, page, pages, scales, device = 2, 64, 8, None, torch.device("cpu")

    entries = [[0, 2, 128], [2, 2, 256]]
    shared = {"array": np.array(entries), "tensor": torch.tensor(entries), "list": entries, "none": None}[kind]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "device", lambda d: __import__("contextlib").nullcontext())
    with pytest.raises(ZeroDivisionError):
        paged.build_plan(Cache, 8, [1] * 4, [300] * 4, [[0]] * 4, shared=shared)
    runs, _ = paged._shared_runs(seen[0], 4, np.ones(4, int), np.full(4, 300), np.ones(4, bool), None, 64)
    assert runs == ([] if kind == "none" else [(0, 2, 128), (2, 2, 256)])
