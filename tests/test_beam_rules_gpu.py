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
