"""Beam search (csrc/beam.cu): calls over and over, several ending tokens, requests that run out of continuations."""
import pytest
import torch

from test_beam_gpu import INF, LSE, Plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("r,k,v,keep", [(3, 4, 1000, 8), (2, 1, 5, 5), (150, 4, 5000, 8), (2, 8, 40000, 16), (1, 64, 700, 128)])
def test_over_and_over(r, k, v, keep):
    """Short lists and long ones, many requests at a time: every call gives the same."""
    from sensenova_u1_b200.ops import beam
    g = torch.Generator(device="cuda").manual_seed(v)
    x, s = torch.randn(r * k, v, generator=g, device="cuda") * 3, -torch.rand(r, k, generator=g, device="cuda")
    want = beam.beam_select(x, s, keep)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [beam.beam_select(x, s, keep) for _ in range(50)]
    for _ in range(40):
        graph.replay()
        assert all(torch.equal(a, b) for o in out for a, b in zip(o, want))


@pytest.mark.parametrize("eos", [(50,), (1 << 20, 3), (49,), ()])
def test_next_tokens_are_of_the_vocabulary(eos):
    """Rows that nobody goes on with, also where the ending token is none of the vocabulary (they look up an embedding all the same)."""
    from sensenova_u1_b200.ops import beam
    x = torch.randn(12, 50, device="cuda")
    x[6:] = float("nan")                                    # a request that ends at once
    x[:6, 3:] = -INF                                        # and one with fewer continuations than beams
    search = beam.BeamSearch(2, 6, 3, eos)
    for _ in range(3):
        search.advance(x)
        assert 0 <= int(search.tokens.min()) and int(search.tokens.max()) < 50


class All(Plain):
    """The search with all candidates of a step looked at; one without any is over, and its beams count as they are.

    ``sure``: no decision of a request was between scores that are as good as equal.  Logits by the last token give equal sums in another order
    (a, b, b after a, a, b: the same steps), which the device's fp32 scores need not see as equal: after t steps a score is off by up to
    t (LSE + 2^-24 |s|), the difference of two by twice that.  Either order is right then, and what follows is another search."""

    def __init__(self, requests, *args):
        super().__init__(requests, *args)
        self.sure = [True] * requests

    def compare(self, r, x, y, by=1.0):
        """Two scores divided by ``by`` are about to be compared."""
        if abs(x - y) * by <= 2 * (self.t + 1) * (LSE + max(abs(x), abs(y)) * by * 2.0 ** -24):
            self.sure[r] = False

    def advance(self, logp):
        for r, live in enumerate(self.live):
            if self.done[r]:
                continue
            table = logp[r].tolist()
            cand = sorted(((s + x, -b, -v) for b, (s, _, _) in enumerate(live) for v, x in enumerate(table[b]) if s + x > -INF), reverse=True)
            new, length = [], (self.t + 1) ** self.penalty
            for i, (s, b, v) in enumerate(cand):
                if len(new) == self.k:
                    break
                if i + 1 < len(cand):
                    self.compare(r, s, cand[i + 1][0])
                if -v not in self.eos:
                    new.append((s, live[-b][1] + [-v], -b))
                elif i < self.k:
                    self.put(r, (s / length, live[-b][1] + [-v]))
            if not cand and self.t:
                for s, tokens, _ in live:
                    self.put(r, (s / self.t ** self.penalty, tokens))
            self.live[r] = new
            if not new:
                self.done[r] = True
            elif len(self.pool[r]) == self.k:
                at = self.steps ** self.penalty if self.early == "never" and self.penalty > 0 else length
                worst = min(p[0] for p in self.pool[r])
                self.compare(r, worst, new[0][0] / at, min(at, length))
                self.done[r] = self.early is True or worst >= new[0][0] / at
        self.t += 1

    def put(self, r, x):
        pool = self.pool[r]
        if len(pool) < self.k:
            pool.append(x)
            return
        w = min(range(self.k), key=lambda j: pool[j][0])
        self.compare(r, x[0], pool[w][0], min(1.0, (self.t + 1) ** self.penalty))
        if x[0] > pool[w][0]:
            pool[w] = x


def run(table, beams, steps, eos, penalty, early, logits=None):
    """A search over logits by the last token [requests, vocab, vocab], step by step beside the plain one."""
    from sensenova_u1_b200.ops import _lib, beam
    requests, vocab = table.shape[:2]
    search, plain = beam.BeamSearch(requests, beams, steps, eos, penalty, early), All(requests, beams, steps, eos, penalty, early)
    rows = torch.arange(requests, device="cuda").repeat_interleave(beams)
    exact = torch.log_softmax(table.double(), -1).cpu()
    exact[(torch.isnan(table) | (table == INF)).any(-1).cpu() | (table == -INF).all(-1).cpu()] = -INF
    short = compared = 0
    for t in range(steps):
        x = table[rows, search.tokens]
        logp = torch.full((requests, beams, vocab), -INF, dtype=torch.float64)
        for r in range(requests):
            for b, (_, tokens, _) in enumerate(plain.live[r]):
                logp[r, b] = exact[r, tokens[-1] if tokens else 0]
        if logits is not None:
            logits(t, x, logp)
        search.advance(x)
        plain.advance(logp)
        tokens, parents = search.tokens.view(requests, beams).tolist(), search.parents.view(requests, beams).tolist()
        for r in range(requests):
            here = int((search.scores[r] > -INF).sum())
            short += not search.done[r] and here < beams
            if plain.sure[r]:
                assert search.done[r] == int(plain.done[r])
                compared += 1
            if not plain.sure[r] or plain.done[r]:
                continue
            assert here == len(plain.live[r])
            for b, (s, path, parent) in enumerate(plain.live[r]):
                assert (tokens[r][b], parents[r][b]) == (path[-1], r * beams + parent)
                assert abs(float(search.scores[r, b]) - s) <= (t + 1) * (LSE + abs(s) * 2.0 ** -24) + 1e-9
    for a, b, sure in zip(search.result(beams), plain.result(beams), plain.sure):
        if not sure:
            continue
        assert [x[0] for x in a] == [x[1] for x in b]
        for (_, x), (y, _) in zip(a, b):
            assert abs(x - y) <= 1e-4 * max(1, abs(y))
    _lib.check_status()
    return short, compared


@pytest.mark.parametrize("early", [False, True, "never"])
@pytest.mark.parametrize("beams,vocab,eos,penalty", [(4, 20, (3, 7), 2.0), (4, 20, (3, 7, 11), 2.0), (4, 20, tuple(range(8)), 1.0), (2, 30, (1, 2, 3, 4, 5), 0.0), (3, 400, (0, 399, 9, 9, 0), 1.0),
                                                     (1, 12, tuple(range(8)), 1.0), (40, 300, (3, 5), 1.0), (64, 500, (1, 2, 3, 4), 1.0), (64, 700, tuple(range(8)), 1.0)])
def test_several_ending_tokens(beams, vocab, eos, penalty, early):
    """Each of the beams may end in each of them: as many as there are beams go on all the same."""
    compared = 0
    for seed in range(8 if beams < 16 else 1):
        g = torch.Generator(device="cuda").manual_seed(seed)
        table = torch.randn(3, vocab, vocab, generator=g, device="cuda")
        table[:2, :, list(eos)] += 3                            # often all of the best
        short, n = run(table, beams, 7, eos, penalty, early)
        compared += n
        if vocab - len(set(eos)) >= beams:
            assert short == 0
    assert compared >= 3


@pytest.mark.parametrize("when", [0, 1, 3])
@pytest.mark.parametrize("beams,eos", [(1, ()), (4, (2, 5)), (64, (3,))])
def test_no_continuation_is_left(when, beams, eos):
    """From some step on a request's logits are NaN: its beams count as they are, beside what had ended."""
    g = torch.Generator(device="cuda").manual_seed(beams)
    table = torch.randn(3, 200, 200, generator=g, device="cuda") * 2

    def broken(t, x, logp):
        if t >= when:
            x[beams:2 * beams] = float("nan")
            logp[1] = -INF

    run(table, beams, 6, eos, 1.0, "never", broken)


def test_generate_without_a_continuation():
    from sensenova_u1_b200.inference.api import ByteTokenizer, NEOChatModel
    from test_beam_search_gpu import model, prompts
    cfg, store, eng = model()
    store.p["lm_head"].fill_(float("nan"))
    docs = prompts(cfg, [40, 150])
    assert eng.beam_search(docs, 4, 6, stop_ids=(5,)) == [[], []]
    m, tok = NEOChatModel(cfg, store), ByteTokenizer(cfg.vocab_size)
    with pytest.raises(RuntimeError, match="no continuation"):
        m.chat(tok, None, "hello", generation_config={"num_beams": 4, "max_new_tokens": 6})
    with pytest.raises(RuntimeError, match="no continuation"):
        m.generate(input_ids=torch.tensor([tok.encode("what is shown?")]), max_new_tokens=6, num_beams=4, num_return_sequences=2)


def test_sizes_that_another_thread_forgets(monkeypatch):
    """The table of sizes is emptied between a look and the next one."""
    from sensenova_u1_b200.ops import beam

    class Emptied(dict):
        def __contains__(self, key):
            here = super().__contains__(key)
            self.clear()
            return here

        def __setitem__(self, key, value):
            pass

    x, s = torch.randn(8, 40000, device="cuda"), torch.zeros(2, 4, device="cuda")
    want = beam.beam_select(x, s)
    monkeypatch.setattr(beam, "_SCRATCH", Emptied(beam._SCRATCH))
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(beam.beam_select(x, s), want))


def test_penalties_that_leave_fp32_are_refused():
    """(tokens ** penalty was infinite on the device, so hypotheses counted alike, and an OverflowError in the result)"""
    from sensenova_u1_b200.ops import beam
    for penalty in (101.0, -101.0, 1e30):
        with pytest.raises(ValueError, match="fp32"):
            beam.BeamSearch(1, 2, 2, (), penalty)
    for steps, penalty in ((1, 1e30), (2, 100.0), (1024, -10.0)):
        search = beam.BeamSearch(1, 2, steps, (3,), penalty)
        search.advance(torch.randn(2, 9, device="cuda"))
        assert all(abs(s) < INF for _, s in search.result(2)[0])


def test_calls_that_a_search_has_no_place_for():
    """More beams or ending tokens than a search takes, ending tokens that are none: chat and generate answer as they did before there were beams."""
    from sensenova_u1_b200.inference.api import ByteTokenizer, NEOChatModel
    from test_beam_search_gpu import model
    cfg, store, _ = model(8)
    m, tok = NEOChatModel(cfg, store), ByteTokenizer(cfg.vocab_size)
    assert m.chat(tok, None, "hello", generation_config={"num_beams": 4, "max_new_tokens": 0}) == m.chat(tok, None, "hello", generation_config={"max_new_tokens": 0})
    ids = torch.tensor([tok.encode("what is shown in this picture?")])
    for kw, plain in [(dict(num_beams=65), {}), (dict(num_beams=4, eos_token_id=list(range(20, 29))), dict(eos_token_id=list(range(20, 29))))]:
        with pytest.warns(UserWarning, match="left out"):
            got = m.generate(input_ids=ids, max_new_tokens=6, **kw)
        assert torch.equal(got, m.generate(input_ids=ids, max_new_tokens=6, **plain))
    want = m.generate(input_ids=ids, max_new_tokens=6, num_beams=4)
    for eos in (-1, [-1, cfg.vocab_size, cfg.vocab_size + 5]):
        assert torch.equal(m.generate(input_ids=ids, max_new_tokens=6, num_beams=4, eos_token_id=eos), want)
    eos = [int(want[0, 2]), -1, int(want[0, 2]), cfg.vocab_size]
    assert m.generate(input_ids=ids, max_new_tokens=6, num_beams=4, eos_token_id=eos).shape[1] <= 6
