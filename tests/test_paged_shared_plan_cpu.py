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
