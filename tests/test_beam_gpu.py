"""Beam search (csrc/beam.cu) against plain arithmetic in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")
# A term of a row's sum has an error of up to 2^-22 of itself (ex2.approx), and so has the sum (from there on 64 bits, before that 32 fp32
# additions of one sign: 5 * 2^-24 on average, 32 * 2^-24 at most): the normaliser is off by at most 2^-22 + 2^-19.
LSE = 2.0 ** -22 + 2.0 ** -19


def exact(logits, scores):
    """Scores of all candidates in 64 bits [requests, beams * vocab]; -inf where there is none."""
    r, k = scores.shape
    x = logits.double()
    good = ~(torch.isnan(x).any(1) | (x == INF).any(1) | (x == -INF).all(1))
    x = torch.where(good[:, None], x, 0.0)
    c = scores.double()[..., None] + torch.log_softmax(x, -1).view(r, k, -1)
    c[~good.view(r, k) | ~torch.isfinite(scores)] = -INF
    return torch.nan_to_num(c, nan=-INF, posinf=-INF, neginf=-INF).flatten(1)


def check(logits, scores, keep, ties=False):
    from sensenova_u1_b200.ops import beam
    got, beams, tokens = beam.beam_select(logits, scores, keep)
    keep = 2 * scores.shape[1] if keep is None else keep
    assert got.dtype == torch.float32 and beams.dtype == tokens.dtype == torch.int32 and got.shape == beams.shape == tokens.shape == (len(scores), keep)
    c, vocab = exact(logits, scores), logits.shape[1]
    want, at = torch.sort(c, dim=1, descending=True, stable=True)
    want, at = want[:, :keep], at[:, :keep]
    have = want > -INF
    flat = beams.long() * vocab + tokens.long()
    assert torch.equal(got > -INF, have)
    assert not flat[~have].any()
    mine = c.gather(1, flat)
    off = (mine - want).abs()[have]
    assert off.numel() == 0 or off.max() <= 2 * LSE                       # no better one was left out
    near = torch.where(have, got.double() - mine, 0.0).abs()
    assert (near <= LSE + want.abs().nan_to_num(posinf=0) * 2.0 ** -24).all()
    for f, h in zip(flat, have):
        assert f[h].unique().numel() == int(h.sum())
    if ties:
        assert torch.equal(flat[have], at[have])
    else:
        # where neighbours are further apart than the error, the order is the exact one
        clear = torch.ones_like(have)
        gap = (want[:, :-1] - want[:, 1:]).nan_to_num(nan=1.0, posinf=1.0) > 2 * LSE
        clear[:, 1:] &= gap
        clear[:, :-1] &= gap
        clear[:, -1] = False
        assert torch.equal(flat[have & clear], at[have & clear])
    return got, beams, tokens


def some(r, k, v, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(r * k, v, generator=g, device="cuda") * 3).to(dtype)
    return x, -torch.rand(r, k, generator=g, device="cuda").cumsum(1) * 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("r,k,v,keep", [(1, 1, 1, 1), (3, 2, 5, 10), (2, 4, 1000, None), (1, 4, 151936, 8), (5, 3, 4099, 6), (2, 64, 700, 128),
                                        (4, 8, 32001, 16), (1, 1, 2048, 17), (7, 5, 8193, 33), (40, 4, 8191, 1), (3, 32, 20000, 64), (1, 2, 300000, 128), (2, 3, 1 << 21, 12)])
def test_best_of_all(r, k, v, keep, dtype):
    check(*some(r, k, v, dtype, seed=v), keep)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("beams,v", [(4, 2048), (8, 2048), (8, 2049), (64, 256), (33, 257), (33, 256), (16, 4096), (16, 4097), (64, 4096), (64, 4097), (3, 33000), (26, 40000)])
def test_lists_that_are_just_full(beams, v, dtype):
    """One launch or two (64 groups of 256); groups and quarters of them that can hold one of the best: few, as many as a list holds, more."""
    zeros = torch.zeros(2, beams, device="cuda")
    for keep in (1, 40, 128):
        check(torch.ones(2 * beams, v, device="cuda", dtype=dtype), zeros, keep, ties=True)
    x, s = some(2, beams, v, dtype, seed=beams + v)
    check(x / 64, s / 64, 100)
    check(x, s, 100)
    x[:, ::256] += 20                           # one in every group
    check(x, s, 100)


@pytest.mark.parametrize("off", [0, 1, 3, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_wider_ones(off, dtype):
    x, s = some(3, 4, 5003, dtype)
    wide = torch.full((12, 5003 + 21), 50.0, device="cuda", dtype=dtype)
    wide[:, off:off + 5003] = x
    a = check(wide[:, off:off + 5003], s, 8)
    b = check(x, s, 8)
    for i in range(3):
        assert torch.equal(a[i], b[i])


@pytest.mark.parametrize("v", [100, 2048, 30000, 20001])
def test_equal_ones_in_order(v):
    x = torch.zeros(6, v, device="cuda")
    check(x, torch.zeros(2, 3, device="cuda"), 20, ties=True)
    x[:, 7] = x[:, v - 1] = 2
    check(x, torch.zeros(2, 3, device="cuda"), 20, ties=True)
    g = torch.Generator(device="cuda").manual_seed(1)                     # few values, each many times, the same in every beam
    x = torch.randint(0, 4, (2, 1, v), generator=g, device="cuda").float().expand(2, 3, v).reshape(6, v)
    check(x, torch.zeros(2, 3, device="cuda"), 64, ties=True)


def test_many_lists_with_the_same_best():
    check(torch.zeros(64, 25000, device="cuda"), torch.zeros(1, 64, device="cuda"), 128, ties=True)
    x = torch.randn(1, 25000, device="cuda").expand(64, -1).contiguous()
    check(x, torch.zeros(1, 64, device="cuda"), 128, ties=True)


@pytest.mark.parametrize("dtype,run", [(torch.float32, 4), (torch.bfloat16, 8)])
@pytest.mark.parametrize("keep", [17, 32, 33, 64, 65, 128])
def test_large_values_side_by_side(keep, dtype, run):
    """Large values in a few places only: more pass the first bound than there is room for."""
    x, s = some(2, 3, 16384, dtype)
    tok = torch.arange(16384, device="cuda")
    check(x + torch.where(tok // run % 4 == 0, 40, 0).to(dtype), s, keep)
    check(x + torch.where(tok // 2048 == 3, 40, 0).to(dtype), s, keep)
    check((x.float() * 0.01).to(dtype) + torch.where(tok < 6000, 40, 0).to(dtype), s, keep)
    x[:, 2000:] = -INF
    check(x, s, keep)


def test_masked_and_broken_rows():
    x, s = some(4, 5, 3001)
    x[0, 10:] = -INF                       # a few tokens are allowed
    x[1] = -INF                            # none
    x[2, 5] = float("nan")
    x[3, 6] = INF
    x[5:10] = -INF                         # a request without any
    x[10:15, 3:] = -INF                    # fewer than are kept
    s[0, 4] = -INF
    s[3, 1] = float("nan")
    s[3, 2] = INF
    got = check(x, s, 20)
    assert (got[0][1] == -INF).all() and not got[1][1].any() and not got[2][1].any()
    assert int((got[0][2] > -INF).sum()) == 15
    assert not (got[1][0][got[0][0] > -INF] == 4).any()


def test_first_step_and_large_values():
    x, s = some(3, 4, 9000)
    s[:, 1:] = -INF
    s[:, 0] = 0
    got = check(x, s, 8)
    assert not got[1].any()
    check(x * 1e30, s, 8)
    check(x * 1e-30, s, 8, ties=False)
    check(x, torch.full_like(s, -1e30), 8)


def test_refusals():
    from sensenova_u1_b200.ops import beam
    x, s = some(2, 3, 50)
    for logits, scores, keep in [(x[:5], s, 6), (x.double(), s, 6), (x, s.double(), 6), (x, s, 0), (x, s, 129), (x, s, 151), (x, s, 2.0), (x.cpu(), s.cpu(), 6), (x, s[0], None), (x, s.view(-1), None),
                                 (x, s.t(), 6), (x.t().contiguous().t(), s, 6), (x[:, None], s, 6), (x[:1].expand(6, 50), s, 6),
                                 (torch.zeros(65, 50, device="cuda"), torch.zeros(1, 65, device="cuda"), 6)]:
        with pytest.raises(ValueError):
            beam.beam_select(logits, scores, keep)
    assert [t.shape for t in beam.beam_select(x[:0], s[:0], 6)] == [(0, 6)] * 3


def test_streams_and_graphs():
    from sensenova_u1_b200.ops import beam
    x, s = some(2, 4, 20011)
    want = beam.beam_select(x, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = beam.beam_select(x, s)
    graph, held = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = beam.beam_select(held, s)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (0, 1, 2):
        held.copy_(some(2, 4, 20011, seed=seed)[0])
        graph.replay()
        for a, b in zip(out, beam.beam_select(held, s)):
            assert torch.equal(a, b)
    for a, b in zip(want, other):
        assert torch.equal(a, b)


class Plain:
    """The search in Python, 64 bits."""

    def __init__(self, requests, beams, steps, eos, penalty, early):
        self.k, self.steps, self.eos, self.penalty, self.early = beams, steps, eos, penalty, early
        self.live = [[(0.0, [], 0)] for _ in range(requests)]              # score, tokens, row of the step before
        self.pool, self.done, self.t = [[] for _ in range(requests)], [False] * requests, 0

    def advance(self, logp):                                               # [requests, beams, vocab]
        for r, live in enumerate(self.live):
            if self.done[r]:
                continue
            cand = [(s + float(logp[r, b, v]), -b, -v) for b, (s, _, _) in enumerate(live) for v in range(logp.shape[2])]
            cand = [(s, -b, -v) for s, b, v in sorted((c for c in cand if c[0] > -INF), reverse=True)[:2 * self.k]]
            new, length = [], (self.t + 1) ** self.penalty
            for i, (s, b, v) in enumerate(cand):
                if len(new) == self.k:
                    break
                if v not in self.eos:
                    new.append((s, live[b][1] + [v], b))
                elif i < self.k:
                    x = (s / length, live[b][1] + [v])
                    if len(self.pool[r]) < self.k:
                        self.pool[r].append(x)
                    else:
                        w = min(range(self.k), key=lambda j: self.pool[r][j][0])
                        if x[0] > self.pool[r][w][0]:
                            self.pool[r][w] = x
            self.live[r] = new
            if not new:
                self.done[r] = True
            elif len(self.pool[r]) == self.k:
                at = self.steps ** self.penalty if self.early == "never" and self.penalty > 0 else length
                self.done[r] = self.early is True or min(p[0] for p in self.pool[r]) >= new[0][0] / at
        self.t += 1

    def result(self, best):
        out = []
        for r in range(len(self.live)):
            found = list(self.pool[r])
            if not self.done[r]:
                found += [(s / self.t ** self.penalty, tokens) for s, tokens, _ in self.live[r]]
            out.append(sorted(found, key=lambda f: -f[0])[:best])
        return out


@pytest.mark.parametrize("early", [False, True, "never"])
@pytest.mark.parametrize("beams,penalty,eos", [(1, 1.0, (3,)), (4, 1.0, (3, 9)), (4, 0.0, (3,)), (5, -0.5, (0, 7, 8)), (3, 2.0, ()), (64, 1.0, (3, 5))])
@pytest.mark.parametrize("captured", [False, True])
def test_search(beams, penalty, eos, early, captured):
    from sensenova_u1_b200.ops import _lib, beam
    requests, steps, vocab = 3, 11, 150
    g = torch.Generator(device="cuda").manual_seed(beams)
    table = torch.randn(requests, vocab, vocab, generator=g, device="cuda") * 2          # logits by the last token
    if eos:
        table[0, :, list(eos)] += 3
    table[2, :, 60:] = -INF
    search, plain = beam.BeamSearch(requests, beams, steps, eos, penalty, early), Plain(requests, beams, steps, eos, penalty, early)
    rows = torch.arange(requests, device="cuda").repeat_interleave(beams)

    def step():
        search.advance(table[rows, search.tokens])

    graph = None
    for t in range(steps):
        if captured and t == 1:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        graph.replay() if graph is not None else step()
        logp = torch.full((requests, beams, vocab), -INF, dtype=torch.float64)
        for r in range(requests):
            for b, (_, tokens, _) in enumerate(plain.live[r]):
                logp[r, b] = torch.log_softmax(table[r, tokens[-1] if tokens else 0].double(), -1).cpu()
        plain.advance(logp)
        done = [d or t + 1 == steps for d in plain.done]
        assert search.done.tolist() == [int(d) for d in plain.done]
        assert search.finished() == all(done)
        tokens, parents = search.tokens.view(requests, beams).tolist(), search.parents.view(requests, beams).tolist()
        for r in range(requests):
            if plain.done[r]:
                assert tokens[r] == [eos[0] if eos else 0] * beams and parents[r] == [r * beams + b for b in range(beams)]
                continue
            for b, (s, path, parent) in enumerate(plain.live[r]):
                assert (tokens[r][b], parents[r][b]) == (path[-1], r * beams + parent)
                assert abs(float(search.scores[r, b]) - s) <= (t + 1) * (LSE + abs(s) * 2.0 ** -24) + 1e-9
    want = plain.result(beams)
    got = search.result(beams)
    for a, b in zip(got, want):
        assert [x[0] for x in a] == [x[1] for x in b]
        for (_, x), (y, _) in zip(a, b):
            assert abs(x - y) <= 1e-4 * max(1, abs(y))
    _lib.check_status()
    search.advance(table[rows, search.tokens])                              # one too many
    with pytest.raises(_lib.NativeLibraryError):
        _lib.check_status()
    assert search.result(beams) == got


def test_search_refusals():
    from sensenova_u1_b200.ops import beam
    for kw in [dict(requests=0), dict(beams=0), dict(beams=65), dict(steps=0), dict(eos=range(9)), dict(eos=(-1,)), dict(early_stopping="soon"),
               dict(length_penalty=math.inf), dict(requests=2000, beams=64)]:
        with pytest.raises(ValueError):
            beam.BeamSearch(**{**dict(requests=2, beams=3, steps=4), **kw})
    search = beam.BeamSearch(2, 3, 4)
    with pytest.raises(ValueError):
        search.advance(torch.zeros(5, 10, device="cuda"))
    with pytest.raises(ValueError):
        search.result(4)
