"""Beam search through the engine (paged cache, block tables, attention to the shared prompt, selection) against the oracle."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def model(seed=3, **kw):
    from sensenova_u1_b200.config import tiny_mot
    from sensenova_u1_b200.inference.engine import InferenceEngine
    from sensenova_u1_b200.models.params import ParamStore
    cfg = tiny_mot(head_dim=128, patch_size=16, num_layers=2, **kw)
    store = ParamStore(cfg, device="cuda", with_grads=False)
    store.init_weights(seed, std=0.05)
    store.p["lm_head"].mul_(4)                  # (a random head is nearly indifferent)
    return cfg, store, InferenceEngine(cfg, store)


def log_probs(store, cfg, ids, x=None, pos3=None):
    """Log probabilities of every next token, fp32, by the oracle's layers."""
    from sensenova_u1_b200.models import oracle
    from sensenova_u1_b200.ops.attention import make_meta
    p32 = {k: v.float() for k, v in store.p.items()}
    n = ids.numel()
    x = p32["embed_tokens"][ids.cuda()] if x is None else x
    t = torch.arange(n, device="cuda") if pos3 is None else pos3[0].cuda().long()
    pos3 = torch.stack([t, torch.zeros_like(t), torch.zeros_like(t)]) if pos3 is None else pos3.cuda()
    same = (torch.roll(t, 1) == t) | (torch.roll(t, -1) == t)
    meta = make_meta(torch.zeros(n, device="cuda"), t, same.int() * (t + 1).int())
    mask, isg = oracle.dense_mask(meta, meta), torch.zeros(n, dtype=torch.bool, device="cuda")
    for l in range(cfg.num_layers):
        x = oracle.decoder_layer(p32, l, x, isg, pos3, mask, cfg)
    return torch.log_softmax((oracle.rmsnorm(x, p32["final_norm"][0], cfg.rms_eps) @ p32["lm_head"].t()).double(), -1)


def score(store, cfg, prompt, tokens, penalty):
    lp = log_probs(store, cfg, torch.cat([prompt, torch.tensor(tokens)]))
    at = torch.arange(len(prompt) - 1, len(prompt) + len(tokens) - 1)
    return float(lp[at, tokens].sum()) / len(tokens) ** penalty


def prompts(cfg, lens, seed=2):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(8, cfg.vocab_size, (n,), generator=g) for n in lens]


# A hidden state is off by up to 3e-2 of its norm (the bound of the engine's other tests), and so are the logits: those of a token by up to
# 3e-2 of the norm of head row times hidden state, about 3e-2 * |w| * sqrt(hidden) = 3e-2 * (0.2 * 16) * 16 = 1.5 at the very most; over random signs
# a tenth of that.  e4m3 adds 2^-4 to the 3e-2.
ROOM = {BF16: 0.15, E4M3: 0.45}


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("beams,penalty,always", [(2, 1.0, True), (4, 0.0, False), (8, 1.0, True)])
def test_scores_are_those_of_the_sequences(beams, penalty, always, dtype, monkeypatch):
    from sensenova_u1_b200.ops import _lib, paged
    if always:                                  # prompts are read together however short they are
        monkeypatch.setattr(paged, "SHARE_TOKENS", (0, 0))
    cfg, store, eng = model()
    docs = prompts(cfg, [290, 37, 131])
    out = eng.beam_search(docs, beams, 12, stop_ids=(5,), length_penalty=penalty, best=beams, page=16, dtype=dtype)
    _lib.check_status()
    assert eng.last_decode_graph and len(out) == 3
    for doc, found in zip(docs, out):
        assert len(found) == beams and len({tuple(t) for t, _ in found}) == beams
        assert [s for _, s in found] == sorted((s for _, s in found), reverse=True)
        for tokens, s in found:
            assert 1 <= len(tokens) <= 12 and (len(tokens) == 12 or tokens[-1] == 5) and 5 not in tokens[:-1]
            want = score(store, cfg, doc, tokens, penalty)
            assert abs(s - want) <= ROOM[dtype] * len(tokens) ** (1 - penalty)


def test_captured_or_not_and_pages_of_any_size():
    cfg, store, eng = model(5)
    docs = prompts(cfg, [150, 129], 4)
    want = eng.beam_search(docs, 4, 10, best=4, use_graph=False)
    assert not eng.last_decode_graph
    assert eng.beam_search(docs, 4, 10, best=4) == want
    for page in (16, 128):
        got = eng.beam_search(docs, 4, 10, best=4, page=page)
        assert [[t for t, _ in d] for d in got] == [[t for t, _ in d] for d in want]


def test_it_is_a_search():
    """With as many beams as there are paths worth following, the best is at least as good as the greedy one, and one step with all tokens is exact."""
    cfg, store, eng = model(7)
    docs = prompts(cfg, [200], 6)
    best = eng.beam_search(docs, 16, 8, best=1)[0][0]
    lay, h = eng.prefill(docs, reserve_image_tokens=8)
    greedy = eng.decode_greedy(lay, h, 8)[0]
    assert best[1] >= score(store, cfg, docs[0], greedy, 1.0) - ROOM[BF16]
    one = eng.beam_search(docs, 8, 1, best=8)[0]
    lp = log_probs(store, cfg, docs[0])[-1]
    assert abs(one[0][1] - float(lp.max())) <= ROOM[BF16]
    assert all(abs(s - float(lp[t[0]])) <= ROOM[BF16] for t, s in one)


def test_stops_early():
    cfg, store, eng = model(9)
    docs = prompts(cfg, [140, 60], 8)
    first = [t for d in eng.beam_search(docs, 4, 1, best=4) for (t,), _ in d]
    out = eng.beam_search(docs, 4, 40, stop_ids=first[:8], early_stopping=True, best=4, check_every=2)
    for found in out:
        assert all(t[-1] in first[:8] for t, _ in found)
        assert found[0][0][-1] in first


def test_mixture_of_experts():
    cfg, store, eng = model(4, num_experts=8, num_experts_per_tok=2, gen_num_experts=4, gen_num_experts_per_tok=2, moe_intermediate_size=256)
    out = eng.beam_search(prompts(cfg, [140, 33], 8), 3, 6, best=3)
    assert all(len(d) == 3 and all(len(t) == 6 for t, _ in d) for d in out)


def test_pictures():
    """A prompt with a picture, whose tokens see one another; new tokens go on behind its t index."""
    cfg, store, eng = model(6)
    (ids,) = prompts(cfg, [180], 5)
    t, h, w = list(range(40)), [0] * 40, [0] * 40
    t += [40] * 96
    h += [i // 12 for i in range(96)]
    w += [i % 12 for i in range(96)]
    t += list(range(41, 41 + 44))
    h += [0] * 44
    w += [0] * 44
    pos3 = torch.tensor([t, h, w], dtype=torch.int32)
    x = store.p["embed_tokens"][ids.cuda()]
    out = eng.beam_search([ids], 4, 6, best=4, docs_embeds=[x], docs_pos3=[pos3], page=32)[0]
    p32 = store.p["embed_tokens"].float()
    for tokens, s in out:
        more = torch.arange(85, 85 + len(tokens))
        full = torch.cat([pos3, torch.stack([more, torch.zeros_like(more), torch.zeros_like(more)])], 1)
        lp = log_probs(store, cfg, torch.cat([ids, torch.tensor(tokens)]), torch.cat([x.float(), p32[torch.tensor(tokens).cuda()]]), full)
        want = float(lp[torch.arange(179, 179 + len(tokens)), tokens].sum()) / len(tokens)
        assert abs(s - want) <= ROOM[BF16]


def test_refusals():
    cfg, store, eng = model()
    docs = prompts(cfg, [20, 30])
    for kw in [dict(beams=65), dict(beams=0), dict(max_new_tokens=0), dict(best=5), dict(page=20), dict(stop_ids=range(9)), dict(early_stopping="maybe")]:
        with pytest.raises(ValueError):
            eng.beam_search(docs, **{**dict(beams=4, max_new_tokens=5), **kw})
    with pytest.raises(ValueError):
        eng.beam_search([], 4, 5)
    with pytest.raises(ValueError):
        eng.beam_search([docs[0][:0]], 4, 5)
    with pytest.raises(ValueError):
        eng.beam_search(docs * 9, 64, 5)


def test_chat_and_generate():
    from sensenova_u1_b200.inference.api import ByteTokenizer, NEOChatModel
    cfg, store, _ = model(8)
    m, tok = NEOChatModel(cfg, store), ByteTokenizer(cfg.vocab_size)
    text = m.chat(tok, None, "hello", generation_config={"num_beams": 4, "max_new_tokens": 6, "length_penalty": 0.5})
    assert isinstance(text, str)
    ids = torch.tensor([tok.encode("what is shown in this picture?")])
    one = m.generate(input_ids=ids, max_new_tokens=6, num_beams=4)
    many = m.generate(input_ids=ids, max_new_tokens=6, num_beams=4, num_return_sequences=3, eos_token_id=[7, 9], pad_token_id=1)
    assert one.shape == (1, 6) and many.shape[0] == 3 and many.dtype == torch.long
    assert m.generate(input_ids=ids, max_new_tokens=6).shape == (1, 6)
    with pytest.raises(ValueError):
        m.generate(input_ids=ids, max_new_tokens=6, num_beams=2, num_return_sequences=3)
    # what a beam search does not do goes without, as before there was one
    for kw, plain in [(dict(num_beams=4, do_sample=True, seed=3), dict(do_sample=True, seed=3)),
                      (dict(num_beams=4, repetition_penalty=1.2), dict(repetition_penalty=1.2)), (dict(num_return_sequences=2), {})]:
        with pytest.warns(UserWarning, match="left out"):
            got = m.generate(input_ids=ids, max_new_tokens=6, **kw)
        assert torch.equal(got, m.generate(input_ids=ids, max_new_tokens=6, **plain))
    assert isinstance(m.chat(tok, None, "hello", generation_config={"num_beams": 4, "num_return_sequences": 2, "max_new_tokens": 4}), str)


def test_layers_that_are_not_on_the_device():
    from sensenova_u1_b200.inference.api import NEOChatModel
    from sensenova_u1_b200.models.params import ParamStore
    cfg, store, eng = model(5)
    host = ParamStore(cfg, device="cpu", with_grads=False)
    for name in host.p:
        host.p[name].copy_(store.p[name])
    docs = prompts(cfg, [70, 33])
    kw = dict(beams=3, max_new_tokens=7, stop_ids=(5,), best=2)
    assert NEOChatModel(cfg, host, vram_mode="low", device="cuda").engine.beam_search(docs, **kw) == eng.beam_search(docs, **kw)
