"""Paged key/value cache (csrc/paged_cache.cu, attn_paged.cu, attn_paged_sm100.cu) against plain arithmetic in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
SCALE = D ** -0.5
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def tables_for(kv_lens, page, spare=3, seed=0):
    """Pages of every sequence in an order that no address computation gets right by chance, and how many there are."""
    need = [-(-k // page) for k in kv_lens]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    out = []
    for n in need:
        out.append(order[:n])
        order = order[n:]
    return out, sum(need) + spare


def quantised(x):
    """The definition in fp32: codes and scales of rows of 128.  (A number divided by a tensor would be the product with its reciprocal.)"""
    a = x.float().abs().amax(-1).clamp_min(2.0 ** -110)
    return (x.float() * (torch.full_like(a, 448.0) / a)[..., None]).to(E4M3), a / torch.full_like(a, 448.0)


def make(kv_lens, page, hk, dtype, seed=0, spare=3):
    """A cache full of random values, and per sequence what it holds, in 64 bits: [2, heads, keys, 128]."""
    from sensenova_u1_b200.ops import paged
    tables, pages = tables_for(kv_lens, page, spare, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(pages, 2, hk, page, D, device="cuda", generator=g).to(BF16)
    if dtype == E4M3:
        x = x * torch.exp2(torch.randint(-3, 4, x.shape[:4] + (1,), device="cuda", generator=g)).to(BF16)
        codes, scales = quantised(x)
        cache, held = paged.PagedCache(codes, scales), codes.double() * scales.double()[..., None]
    else:
        cache, held = paged.PagedCache(x), x.double()
    rows = [torch.cat([held[p] for p in t], 2)[:, :, :k] if k else held[0, :, :, :0] for t, k in zip(tables, kv_lens)]
    return cache, tables, rows


def exact(q, q_lens, rows, limits, dtype=BF16):
    """Attention in 64 bits, and how much of rounded factors an output element may show: the mean of |v| under the same
    probabilities, times 2^-8 + 2^-11 plus what widened keys add (see near)."""
    from sensenova_u1_b200.ops import paged
    out, room, r = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device), 0
    for n, kv in zip(q_lens, rows):
        if n and kv.shape[2]:
            g = q.shape[1] // kv.shape[1]
            k, v = kv[0].repeat_interleave(g, 0), kv[1].repeat_interleave(g, 0)
            x = q[r:r + n].double()
            hidden = torch.arange(kv.shape[2], device=q.device)[None] >= limits[r:r + n, None]
            s = torch.einsum("rhd,hkd->hrk", x, k) * SCALE
            p = torch.nan_to_num(torch.softmax(s.masked_fill(hidden, float("-inf")), -1), nan=0.0)
            out[r:r + n] = torch.einsum("hrk,hkd->rhd", p, v)
            room[r:r + n] = torch.einsum("hrk,hkd->rhd", p, v.abs()) * (2.0 ** -8 + 2.0 ** -11)
            if dtype == E4M3 and n * g > paged.CHUNK_FROM:
                most = (torch.einsum("rhd,hkd->hrk", x.abs(), k.abs()) * SCALE).masked_fill(hidden, 0.0).amax(-1)       # [heads, rows]
                room[r:r + n] *= 1 + 2 * 2.0 ** -11 * most.T[..., None] / (2.0 ** -8 + 2.0 ** -11)
        r += n
    return out, room


def causal(q_lens, kv_lens):
    return torch.tensor([k - n + i + 1 for n, k in zip(q_lens, kv_lens) for i in range(n)], device="cuda")


def near(got, ref, room):
    """One rounding of every probability (2^-8 of it, so 2^-8 of the mean of |v|) and one of the result (2^-8 of it).  Sums, the
    approximate exponentials (2^-22) and the fp32 scores add less than 2^-11 of the mean of |v|: scores below 2^6 have an
    error below 2^6 * 128 * 2^-24.  e4m3: probabilities are rounded to fp16 (2^-11), and chunks round code times scale to fp16:
    values 2^-11 of themselves; keys move a score by d <= 2^-11 of the sum of |q k|, probabilities by exp(+-d) before and after
    their sum is divided by, the result by 2 d of the mean of |v|.  All these signs are random, so the whole is far nearer: the
    2-norm of the differences stays below 2^-8 of the result's and half of the room's."""
    err = (got.double() - ref).abs()
    return bool((err <= room + 2.0 ** -8 * ref.abs()).all()) and float(err.norm()) <= 2.0 ** -8 * float(ref.norm()) + 0.5 * float(room.norm())


def attend(q_lens, kv_lens, hq, hk, page, dtype, limits=None, seed=0):
    from sensenova_u1_b200.ops import paged
    cache, tables, rows = make(kv_lens, page, hk, dtype, seed)
    n = sum(q_lens)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn(n + 2, hq + 3, D, device="cuda", generator=g).to(BF16)[:, 1:hq + 1]         # rows of a wider buffer
    out = torch.full((n + 2, hq, D), 7.0, device="cuda", dtype=BF16)
    plan = paged.build_plan(cache, hq, q_lens, kv_lens, tables, limits=limits)
    paged.paged_attention(q, cache, plan, SCALE, out=out)
    lim = causal(q_lens, kv_lens) if limits is None else torch.as_tensor(limits, device="cuda")
    ref, room = exact(q[:n], q_lens, rows, lim, dtype)
    assert near(out[:n], ref, room)
    assert (out[n:] == 7).all()                           # rows behind the last sequence
    assert (out[:n][lim == 0] == 0).all()                 # rows without keys
    again = paged.paged_attention(q, cache, plan, SCALE)
    assert torch.equal(again, out[:n])                    # the same bits, whatever order the CTAs ran in


# ------------------------------------------------------------------ writing and reading
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("hk", [1, 4, 7])
def test_write_then_read(page, hk, dtype):
    from sensenova_u1_b200.ops import paged
    q_lens, kv_lens = [1, 0, 130, 17, 5], [1, 3, 130, 200, 16]
    tables, pages = tables_for(kv_lens, page)
    cache = paged.PagedCache.empty(pages, page, hk, dtype)
    cache.data.view(torch.uint8).fill_(0x3c)
    if dtype == E4M3:
        cache.scales.fill_(0.25)
    before = cache.data.clone()
    n = sum(q_lens)
    g = torch.Generator(device="cuda").manual_seed(page + hk)
    x = (torch.randn(n + 3, 2 * hk + 2, D, device="cuda", generator=g) * torch.exp2(torch.randint(
        -40, 40, (n + 3, 2 * hk + 2, 1), device="cuda", generator=g))).to(BF16)
    k, v = x[:, 1:1 + hk], x[:, 2 + hk:]
    plan = paged.build_plan(cache, hk, q_lens, kv_lens, tables)
    paged.paged_write(cache, k, v, plan)
    want, touched = before.clone(), torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    scales = None if dtype == BF16 else torch.full((pages, 2, hk, page), 0.25, device="cuda")
    r = 0
    for n_, kv, t in zip(q_lens, kv_lens, tables):
        for i in range(n_):
            pos = kv - n_ + i
            pg, off = t[pos // page], pos % page
            row = torch.stack([k[r], v[r]])
            if dtype == BF16:
                want[pg, :, :, off] = row
            else:
                c, s = quantised(row)
                want.view(torch.uint8)[pg, :, :, off] = c.view(torch.uint8)
                scales[pg, :, :, off] = s
            touched[pg, off] = True
            r += 1
    assert torch.equal(cache.data.view(torch.uint8), want.view(torch.uint8))         # and nothing else was written
    if dtype == E4M3:
        assert torch.equal(cache.scales, scales)
    kr, vr = paged.paged_read(cache, plan)
    assert kr.shape == (sum(kv_lens), hk, D)
    at = 0
    for i, (kv, t) in enumerate(zip(kv_lens, tables)):
        for which, got in ((0, kr), (1, vr)):
            held = torch.cat([cache.data.view(torch.uint8)[p, which].view(dtype).float() for p in t], 1)[:, :kv] if kv else None
            if dtype == E4M3 and kv:
                held = held * torch.cat([cache.scales[p, which] for p in t], 1)[:, :kv, None]
            if kv:
                assert torch.equal(got[at:at + kv].transpose(0, 1), held.to(BF16))
        at += kv


def test_quantised_rows_are_within_half_a_step():
    """e4m3 has four significant bits: half a step is 2^-4 of the value, or 2^-10 of the row's scale below its smallest normal value
    (2^-6, steps of 2^-9); the product with the scale is rounded once more to bf16 (2^-8); fp32 steps before add 2^-22."""
    from sensenova_u1_b200.ops import paged
    cache = paged.PagedCache.empty(4, 128, 2, E4M3)
    plan = paged.build_plan(cache, 2, [512], [512], [[2, 0, 3, 1]])
    x = torch.randn(2, 512, 2, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(BF16)
    paged.paged_write(cache, x[0], x[1], plan)
    got = torch.stack(paged.paged_read(cache, plan)).double()
    scale = x.double().abs().amax(-1, keepdim=True) / 448
    step = torch.maximum(x.double().abs() * 2.0 ** -4, scale * 2.0 ** -10)
    assert ((got - x.double()).abs() <= step * (1 + 2.0 ** -8) + (2.0 ** -8 + 2.0 ** -20) * x.double().abs()).all()


def test_rows_at_the_ends_of_the_range():
    from sensenova_u1_b200.ops import paged
    cache = paged.PagedCache.empty(1, 16, 1, E4M3)
    big = torch.finfo(BF16).max
    x = torch.zeros(8, 1, D, device="cuda", dtype=BF16)
    x[1, 0, 5] = 2.0 ** -130                             # subnormal: below what a scale is made of
    x[2, 0, :2] = torch.tensor([big, -big])
    x[3, 0, 7], x[4, 0, 9], x[5, 0, 1] = float("inf"), float("nan"), float("-inf")
    x[6, 0] = 2.0 ** -100
    x[7, 0] = -1.0
    plan = paged.build_plan(cache, 1, [8], [8], [[0]])
    paged.paged_write(cache, x, x, plan)
    k, v = paged.paged_read(cache, plan)
    assert torch.equal(k.view(torch.int16), v.view(torch.int16))
    assert (k[0] == 0).all() and (k[1].abs() <= 2.0 ** -113).all() and torch.isnan(k[3:6]).all()
    assert torch.equal(k[2], x[2]) and torch.equal(k[6:], x[6:])


def test_every_code_is_widened_exactly():
    """Scores of one-hot queries with a key row of all 256 codes (in two rows) show how attention widens them; read does the same."""
    from sensenova_u1_b200.ops import paged
    cache = paged.PagedCache.empty(1, 16, 1, E4M3)
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    codes[127], codes[255] = 0, 0                         # the NaN codes never stand in a cache
    cache.data.view(torch.uint8).zero_()
    cache.data.view(torch.uint8)[0, :, 0, :2] = codes.view(2, D)
    cache.scales.fill_(1.0)
    plan = paged.build_plan(cache, 1, [2], [2], [[0]], limits=[1, 2])
    q = torch.zeros(2, 1, D, device="cuda", dtype=BF16)
    value = codes.view(torch.uint8).view(E4M3).double().view(2, D)
    out = paged.paged_attention(q, cache, plan, 1.0)      # one key: its value; two keys of equal scores: their mean
    assert torch.equal(out[0, 0].double(), value[0])
    assert ((out[1, 0].double() - value.mean(0)).abs() <= 2.0 ** -8 * value.mean(0).abs()).all()
    k, _ = paged.paged_read(cache, plan)
    assert torch.equal(k[:, 0].double(), value)
    # keys: query e_d gives the score k_d of row 0 and k'_d of row 1; v = (1, 0, ...), (0, 1, ...) shows both probabilities
    cache.data.view(torch.uint8)[0, 1].zero_()
    cache.data[0, 1, 0, 0, 0] = 1.0
    cache.data[0, 1, 0, 1, 1] = 1.0
    eye = torch.eye(D, device="cuda").to(BF16).view(D, 1, D)
    for a in range(0, D, 16):
        plan = paged.build_plan(cache, 1, [16], [16], [[0]], limits=[2] * 16)
        out = paged.paged_attention(eye[a:a + 16], cache, plan, 2.0 ** -6)[:, 0, :2].double()
        p = torch.softmax(value[:, a:a + 16].T * 2.0 ** -6, -1)
        assert ((out - p).abs() <= (2 * 2.0 ** -8 + 2.0 ** -12) * p).all()


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("hq,hk", [(4, 4), (4, 2), (12, 4), (8, 1), (20, 1)])
def test_one_token(hq, hk, page, dtype):
    attend([1] * 6, [1, 63, 64, 65, 700, 129], hq, hk, page, dtype)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("q_lens,kv_lens", [([5, 0, 3, 1], [5, 9, 300, 1000]), ([8, 7], [8, 71]), ([16], [2000]), ([33, 2], [33, 200])])
def test_a_few_tokens(q_lens, kv_lens, page, dtype):
    attend(q_lens, kv_lens, 8, 2, page, dtype)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("q_lens,kv_lens,hq,hk,page", [
    ([130, 1, 257], [130, 500, 1000], 8, 2, 16), ([64], [64], 4, 1, 64), ([300], [301], 3, 3, 32), ([97, 1, 1], [5000, 3, 129], 12, 4, 128),
    ([1, 200, 31, 0, 90], [64, 200, 95, 7, 128], 20, 2, 16), ([70], [70], 100, 1, 16)])
def test_chunks(q_lens, kv_lens, hq, hk, page, dtype):
    attend(q_lens, kv_lens, hq, hk, page, dtype)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("hq,hk", [(4, 1), (6, 2), (32, 8)])
def test_limits(hq, hk, dtype):
    """Pictures, rows without any key, rows that read a prefix only."""
    q_lens, kv_lens = [40, 3, 150], [90, 3, 700]
    lim = causal(q_lens, kv_lens).tolist()
    for i in range(10, 30):
        lim[i] = 50 + 30                                  # rows 10 .. 29 of the first sequence are a picture
    lim[0] = lim[41] = 0
    lim[40] = 3
    for i in range(60, 90):
        lim[i] = 700
    for i in range(90, 120):
        lim[i] = (i * 37) % 650                           # in any order
    lim[130:193] = [0] * 63
    attend(q_lens, kv_lens, hq, hk, 32, dtype, limits=lim)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_all_rows_without_keys(dtype):
    attend([3, 40], [64, 40], 8, 2, 16, dtype, limits=[0] * 43)


@pytest.mark.parametrize("q_len", [1, 6, 60])
def test_one_long_sequence_in_many_parts(q_len):
    attend([q_len], [20000 + q_len], 8, 2, 16, E4M3)
    attend([q_len], [9001], 4, 4, 64, BF16)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("q_lens", [[5], [6], [5, 1, 0, 6]])
def test_seventeen_to_twenty_four_rows(q_lens, dtype):
    attend(q_lens, [38100 - 9300 * i for i in range(len(q_lens))], 32, 8, 64, dtype, seed=4)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [50, 64]), ([5], [70]), ([100, 1], [300, 10])])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_no_row_may_read_does_not_matter(q_lens, kv_lens, bad, dtype):
    """Places behind a sequence's last token, pages of nobody, and keys beyond every limit hold NaN or infinities."""
    from sensenova_u1_b200.ops import paged
    page = 16
    cache, tables, _ = make(kv_lens, page, 2, dtype)
    lim = [max(0, x - 3) for x in causal(q_lens, kv_lens).tolist()]
    plan = paged.build_plan(cache, 8, q_lens, kv_lens, tables, limits=lim)
    q = torch.randn(sum(q_lens), 8, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(BF16)
    clean = paged.paged_attention(q, cache, plan, SCALE).clone()
    own = torch.zeros(cache.pages, page, dtype=torch.bool, device="cuda")
    r = 0
    for n, t in zip(q_lens, tables):
        for pos in range(max(lim[r:r + n])):
            own[t[pos // page], pos % page] = True
        r += n
    hide = ~own[:, None, None, :].expand(cache.pages, 2, 2, page)
    if dtype == E4M3:
        cache.scales[hide] = bad
        cache.data.view(torch.uint8)[hide] = 0x7e
    else:
        cache.data[hide] = bad
    assert torch.equal(paged.paged_attention(q, cache, plan, SCALE), clean)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("q_len,kv_len,at", [(5, 70, 67), (5, 70, 65), (100, 300, 250), (100, 300, 201), (300, 600, 511), (40, 2000, 1990)])
def test_a_value_that_is_not_finite_reaches_the_rows_that_read_it(q_len, kv_len, at, which, dtype):
    from sensenova_u1_b200.ops import paged
    cache, tables, _ = make([kv_len], 32, 2, dtype)
    plan = paged.build_plan(cache, 8, [q_len], [kv_len], tables)
    q = torch.randn(q_len, 8, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(BF16)
    clean = paged.paged_attention(q, cache, plan, SCALE).clone()
    pg, off = tables[0][at // 32], at % 32
    if dtype == E4M3:
        cache.scales[pg, which, 1, off] = float("nan")
    else:
        cache.data[pg, which, 1, off, 77] = float("nan")
    out = paged.paged_attention(q, cache, plan, SCALE)
    reads = torch.arange(kv_len - q_len, kv_len, device="cuda") >= at
    assert torch.equal(out[~reads], clean[~reads]) and torch.equal(out[:, :4], clean[:, :4])
    assert torch.isnan(out[reads][:, 4:]).any(-1).all()


def test_large_scores():
    """The running maximum moves by hundreds, and some keys' probabilities are 0 in fp32."""
    from sensenova_u1_b200.ops import paged
    kv, q_lens = [900, 400], [70, 1]
    cache, tables, rows = make(kv, 16, 2, BF16)
    q = (40 * torch.randn(71, 4, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))).to(BF16)
    plan = paged.build_plan(cache, 4, q_lens, kv, tables)
    out = paged.paged_attention(q, cache, plan, SCALE)
    ref, room = exact(q, q_lens, rows, causal(q_lens, kv))
    # scores up to 2^9: products of 2^9 sqrt(128) summed in fp32 are off by at most 2^12.5 * 128 / 2 * 2^-24 = 2^-5.5 in the worst
    # case of all terms of one sign; terms of random sign stay below 2^12.5 * 2^-24 * sqrt(128) = 2^-8: four times the usual room
    assert ((out.double() - ref).abs() <= 4 * room + 2.0 ** -8 * ref.abs()).all()


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_a_prompt_in_chunks_then_tokens(dtype):
    """Two sequences: one prompt in three chunks while the other decodes, then both decode in a captured step."""
    from sensenova_u1_b200.ops import paged
    hq, hk, page = 8, 2, 16
    steps = [[200, 40], [90, 1], [31, 1]] + [[1, 1]] * 9
    total = [sum(s[i] for s in steps) for i in range(2)]
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(2, max(total), h, D, device="cuda", generator=g).to(BF16) for h in (hq, hk, hk))
    tables, pages = tables_for(total, page)
    cache = paged.PagedCache.empty(pages, page, hk, dtype)
    cache.data.view(torch.uint8).fill_(0x7f)
    out, at = torch.zeros(2, max(total), hq, D, device="cuda", dtype=BF16), [0, 0]
    pick = lambda t, n: torch.cat([t[i, at[i]:at[i] + n[i]] for i in range(2)])
    for s in steps[:4]:
        plan = paged.build_plan(cache, hq, s, [a + n for a, n in zip(at, s)], tables)
        paged.paged_write(cache, pick(k, s), pick(v, s), plan)
        o = paged.paged_attention(pick(q, s), cache, plan, SCALE)
        for i in range(2):
            out[i, at[i]:at[i] + s[i]] = o[sum(s[:i]):sum(s[:i + 1])]
            at[i] += s[i]
    # a captured step that moves itself on
    left = len(steps) - 4
    plan = paged.build_plan(cache, hq, [1, 1], at, tables, grow=left)
    bufs = [torch.empty(2, h, D, device="cuda", dtype=BF16) for h in (hq, hk, hk)]
    o = torch.empty(2, hq, D, device="cuda", dtype=BF16)

    def step():
        plan.advance()
        paged.paged_write(cache, bufs[1], bufs[2], plan)
        paged.paged_attention(bufs[0], cache, plan, SCALE, out=o)

    def feed():
        for b, t in zip(bufs, (q, k, v)):
            b.copy_(pick(t, [1, 1]))

    feed()
    step()
    graph = torch.cuda.CUDAGraph()
    plan.advance(-1)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for _ in range(left):
        feed()
        graph.replay()
        for i in range(2):
            out[i, at[i]] = o[i]
            at[i] += 1
    assert at == total
    held = torch.stack([k, v], 1).transpose(2, 3)                       # [2, k v, heads, tokens, 128]
    if dtype == E4M3:
        codes, scales = quantised(held)
        held = codes.double() * scales.double()[..., None]
    for i in range(2):
        lim = torch.arange(1, total[i] + 1, device="cuda")
        ref, room = exact(q[i, :total[i]], [total[i]], [held[i, :, :, :total[i]].double()], lim, dtype)
        assert near(out[i, :total[i]], ref, room)


def test_the_whole_prompt_as_the_packed_kernel_sees_it():
    """Chunks over pages against the contiguous kernel on the same prompt with a picture in it."""
    from sensenova_u1_b200.ops import attention as A, paged
    n, hq, hk, a, b = 333, 8, 2, 100, 260
    g = torch.Generator(device="cuda").manual_seed(9)
    q, k, v = (torch.randn(n, h, D, device="cuda", generator=g).to(BF16) for h in (hq, hk, hk))
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    pos[a:b], pos[b:] = a, torch.arange(a + 1, a + 1 + n - b, device="cuda")
    img = torch.zeros_like(pos)
    img[a:b] = 1
    meta = A.make_meta(torch.zeros_like(pos), pos, img)
    ref, _ = A.attention_fwd(q, k, v, A.build_plan(meta), SCALE, want_lse=False)
    lim = [b if a <= i < b else i + 1 for i in range(n)]
    cache = paged.PagedCache.empty(6, 64, hk)
    tables, out = [[3, 0, 5, 1, 4, 2]], []
    for lo, hi in ((0, 90), (90, 261), (261, n)):
        plan = paged.build_plan(cache, hq, [hi - lo], [hi], tables, limits=lim[lo:hi])
        paged.paged_write(cache, k[lo:hi], v[lo:hi], plan)
        out.append(paged.paged_attention(q[lo:hi], cache, plan, SCALE))
    dense, room = exact(q, [n], [torch.stack([k, v]).transpose(1, 2).double()], torch.tensor(lim, device="cuda"))
    assert near(torch.cat(out), dense, room) and near(ref, dense, room)


def test_two_streams_and_a_shared_prompt():
    """Two batches at once on two streams; their sequences read the same first pages."""
    from sensenova_u1_b200.ops import paged
    kv, page = [700, 650], 16
    cache, tables, _ = make(kv, page, 2, E4M3)
    tables[1] = tables[0][:20] + tables[1][20:]
    g = torch.Generator(device="cuda").manual_seed(4)
    jobs = []
    for s, q_lens in ((torch.cuda.Stream(), [1, 1]), (torch.cuda.Stream(), [60, 3])):
        q = torch.randn(sum(q_lens), 8, D, device="cuda", generator=g).to(BF16)
        plan = paged.build_plan(cache, 8, q_lens, kv, tables)
        jobs.append((s, q, plan, paged.paged_attention(q, cache, plan, SCALE)))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (s, q, plan, _) in enumerate(jobs):
            with torch.cuda.stream(s):
                outs[i].append(paged.paged_attention(q, cache, plan, SCALE))
    torch.cuda.synchronize()
    for (_, _, _, ref), got in zip(jobs, outs):
        assert all(torch.equal(o, ref) for o in got)


def test_offsets_beyond_32_bits():
    """Pages behind the first four gigabytes of a cache."""
    from sensenova_u1_b200.ops import paged
    page, hk = 128, 8
    pages = (5 << 30) // (2 * hk * page * D)
    cache = paged.PagedCache.empty(pages, page, hk, E4M3)
    last = list(range(pages - 3, pages))
    q_lens, kv = [300], [300]
    k, v, q = (torch.randn(300, h, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(h)).to(BF16) for h in (hk, hk, 16))
    plan = paged.build_plan(cache, 16, q_lens, kv, [last])
    paged.paged_write(cache, k, v, plan)
    held = []
    for x in (k, v):
        c, s = quantised(x)
        held.append((c.double() * s.double()[..., None]).transpose(0, 1))
    got = paged.paged_read(cache, plan)
    for x, h in zip(got, held):
        assert torch.equal(x.transpose(0, 1), h.float().to(BF16))
    ref, room = exact(q, q_lens, [torch.stack(held)], causal(q_lens, kv), E4M3)
    assert near(paged.paged_attention(q, cache, plan, SCALE), ref, room)


def test_two_graphs_of_one_plan_at_once():
    """Scratch belongs to a call: two captured graphs of the same plan run on two streams at the same time."""
    from sensenova_u1_b200.ops import paged
    kv = [3000, 900, 5000, 17]
    cache, tables, _ = make(kv, 16, 8, E4M3)
    q = torch.randn(2, 4, 32, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)).to(BF16)
    plan = paged.build_plan(cache, 32, [1] * 4, kv, tables)
    assert plan.scratch > 0                               # parts meet in scratch
    want = [paged.paged_attention(x, cache, plan, SCALE).clone() for x in q]
    graphs, outs = [], [torch.empty(4, 32, D, device="cuda", dtype=BF16) for _ in q]
    torch.cuda.synchronize()
    for x, o in zip(q, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(8):
                paged.paged_attention(x, cache, plan, SCALE, out=o)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in q]
    for _ in range(10):
        for s, g, o in zip(streams, graphs, outs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                o.fill_(7.0)
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("q_lens,kv_lens", [([3, 1], [200, 90]), ([40, 100], [500, 100]), ([200], [200])])
def test_a_query_that_is_not_finite_is_its_own_matter(q_lens, kv_lens, dtype):
    from sensenova_u1_b200.ops import paged
    cache, tables, _ = make(kv_lens, 16, 2, dtype)
    plan = paged.build_plan(cache, 8, q_lens, kv_lens, tables)
    q = torch.randn(sum(q_lens), 8, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(BF16)
    clean = paged.paged_attention(q, cache, plan, SCALE)
    bad = q.clone()
    bad[1, 3, 5], bad[2, 6, 100], bad[0, 0, 0] = float("nan"), float("inf"), -float("inf")
    out = paged.paged_attention(bad, cache, plan, SCALE)
    hit = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    hit[1, 3] = hit[2, 6] = hit[0, 0] = True
    assert torch.equal(out[~hit], clean[~hit]) and not torch.isfinite(out[hit]).all(-1).any()


def test_many_short_sequences():
    attend([1] * 300, [1 + (7 * i) % 40 for i in range(300)], 8, 2, 16, E4M3)
    attend([2] * 300, [2 + (7 * i) % 40 for i in range(300)], 8, 2, 16, BF16)
    attend([9 + i % 8 for i in range(100)], [60 + (7 * i) % 90 for i in range(100)], 8, 2, 16, E4M3)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_more_heads_in_a_group_than_rows_in_a_tile(dtype):
    attend([1, 3], [40, 200], 130, 1, 16, dtype)


def test_values_of_very_different_sizes():
    """Scales from 2^-40 to 2^40 in one sequence: a token's probabilities are kept relative to the largest product, not the largest value."""
    from sensenova_u1_b200.ops import paged
    kv, page = [300, 700], 32
    tables, pages = tables_for(kv, page)
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(pages, 2, 2, page, D, device="cuda", generator=g).to(BF16)
    x[:, 1] *= torch.exp2(torch.randint(-40, 41, (pages, 2, page, 1), device="cuda", generator=g)).to(BF16)
    codes, scales = quantised(x)
    cache, held = paged.PagedCache(codes, scales), codes.double() * scales.double()[..., None]
    rows = [torch.cat([held[p] for p in t], 2)[:, :, :k] for t, k in zip(tables, kv)]
    q = (3 * torch.randn(3, 8, D, device="cuda", generator=g)).to(BF16)
    plan = paged.build_plan(cache, 8, [1, 2], kv, tables)
    ref, room = exact(q, [1, 2], rows, causal([1, 2], kv), E4M3)
    assert near(paged.paged_attention(q, cache, plan, SCALE), ref, room)


def test_growing_past_the_plan_is_reported():
    from sensenova_u1_b200.ops import _lib, paged
    cache = paged.PagedCache.empty(2, 16, 1)
    cache.data.zero_()
    plan = paged.build_plan(cache, 1, [1], [3], [[1, 0]], grow=2)
    one = torch.ones(1, 1, D, device="cuda", dtype=BF16)
    for n in range(3):
        paged.paged_write(cache, one, one, plan)
        _lib.check_status()
        plan.advance()
    paged.paged_write(cache, one, one, plan)             # a sixth token
    with pytest.raises(_lib.NativeLibraryError, match="limit"):
        _lib.check_status()
    assert cache.data[1, 0, 0, :, 0].tolist() == [0, 0, 1, 1, 1] + [0] * 11 and (cache.data[0] == 0).all()


# ------------------------------------------------------------------ refusals
def test_refusals():
    from sensenova_u1_b200.ops import paged
    cache, tables, _ = make([40], 16, 2, BF16)
    plan = paged.build_plan(cache, 8, [3], [40], tables)
    q, k = torch.zeros(3, 8, D, device="cuda", dtype=BF16), torch.zeros(3, 2, D, device="cuda", dtype=BF16)
    with pytest.raises(ValueError):
        paged.build_plan(cache, 7, [3], [40], tables)                    # heads
    for bad in (q[:2], q[:, :4], q.float(), q.cpu(), q[..., :64], q.transpose(0, 1)):
        with pytest.raises(ValueError):
            paged.paged_attention(bad, cache, plan, SCALE)
        with pytest.raises(ValueError):
            paged.paged_attention(q, cache, plan, SCALE, out=bad)
    for bad in (k[:2], k[:, :1], k.float(), k.cpu()):
        with pytest.raises(ValueError):
            paged.paged_write(cache, bad, k, plan)
        with pytest.raises(ValueError):
            paged.paged_write(cache, k, bad, plan)
    other = paged.PagedCache.empty(cache.pages, 32, 2)
    for call in (lambda: paged.paged_attention(q, other, plan, SCALE), lambda: paged.paged_write(other, k, k, plan),
                 lambda: paged.paged_read(other, plan)):
        with pytest.raises(ValueError):
            call()
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="scale"):
            paged.paged_attention(q, cache, plan, bad)
    shifted = torch.zeros(3 * 8 * D + 1, device="cuda", dtype=BF16)[1:].view(3, 8, D)      # rows of 16 bytes, off by two
    with pytest.raises(RuntimeError, match="aligned"):
        paged.paged_attention(shifted, cache, plan, SCALE)


def test_empty_calls():
    from sensenova_u1_b200.ops import paged
    cache, tables, _ = make([40], 16, 2, BF16)
    plan = paged.build_plan(cache, 8, [0], [40], tables)
    e = lambda h: torch.empty(0, h, D, device="cuda", dtype=BF16)
    assert paged.paged_attention(e(8), cache, plan, SCALE).shape == (0, 8, D)
    paged.paged_write(cache, e(2), e(2), plan)
    plan = paged.build_plan(cache, 8, [], [], [])
    assert paged.paged_read(cache, plan)[0].shape == (0, 2, D)


def test_a_page_that_does_not_exist_is_reported():
    """The table was changed on the device behind the plan's back: the launch ends, touches nothing outside, and says so."""
    from sensenova_u1_b200.ops import _lib, paged
    cache, tables, _ = make([40, 20], 16, 2, BF16)
    plan = paged.build_plan(cache, 8, [1, 1], [40, 20], tables)
    q, k = torch.zeros(2, 8, D, device="cuda", dtype=BF16), torch.zeros(2, 2, D, device="cuda", dtype=BF16)
    at = (plan._args.table - plan._store.data_ptr()) // 4
    for page in (cache.pages, -1):
        plan._store[at + 2] = page                       # third page of the first sequence, its new token's
        before = cache.data.clone()
        for call in (lambda: paged.paged_write(cache, k, k, plan), lambda: paged.paged_read(cache, plan),
                     lambda: paged.paged_attention(q, cache, plan, SCALE)):
            _lib.check_status()
            call()
            with pytest.raises(_lib.NativeLibraryError, match="page"):
                _lib.check_status()
        same = cache.data == before
        same[tables[1][1], :, :, 3] = True               # the second sequence's new token
        assert same.all()


@pytest.mark.parametrize("q_len,dtype", [(5, E4M3), (40, BF16), (40, E4M3), (300, E4M3)])      # every kernel that looks up pages
def test_a_bad_page_under_a_chunk_is_reported(q_len, dtype):
    from sensenova_u1_b200.ops import _lib, paged
    cache, tables, rows = make([600], 32, 2, dtype)
    plan = paged.build_plan(cache, 8, [q_len], [600], tables)
    q = torch.randn(q_len, 8, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(BF16)
    want = paged.paged_attention(q, cache, plan, SCALE)
    at = (plan._args.table - plan._store.data_ptr()) // 4 + 7
    good = plan._store[at].clone()
    for page in (cache.pages, -1):
        plan._store[at] = page
        _lib.check_status()
        paged.paged_attention(q, cache, plan, SCALE)
        with pytest.raises(_lib.NativeLibraryError, match="page"):
            _lib.check_status()
    plan._store[at] = good
    assert torch.equal(paged.paged_attention(q, cache, plan, SCALE), want)
    _lib.check_status()


def test_rows_that_overlap_are_refused():
    from sensenova_u1_b200.ops import paged
    cache, tables, _ = make([40], 16, 2, BF16)
    plan = paged.build_plan(cache, 8, [3], [40], tables)
    q, k = torch.zeros(3, 8, D, device="cuda", dtype=BF16), torch.zeros(3, 2, D, device="cuda", dtype=BF16)
    for call in (lambda: paged.paged_attention(q, cache, plan, SCALE, out=q[:1].expand(3, 8, D)),
                 lambda: paged.paged_attention(q[:1].expand(3, 8, D), cache, plan, SCALE),
                 lambda: paged.paged_write(cache, k[:1].expand(3, 2, D), k, plan)):
        with pytest.raises(ValueError, match="overlap"):
            call()


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_the_stride_of_one_row_or_one_head_says_nothing(dtype):
    from sensenova_u1_b200.ops import paged
    cache, tables, _ = make([40], 16, 1, dtype)
    one = lambda x: torch.as_strided(x, x.shape, (1, 8 if x.shape[1] == 1 else D, 1), x.storage_offset())
    plan = paged.build_plan(cache, 4, [1], [40], tables)
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(1, h, D, device="cuda", generator=g).to(BF16) for h in (4, 1, 1))
    paged.paged_write(cache, k, v, plan)
    want, held = paged.paged_attention(q, cache, plan, SCALE), cache.data.view(torch.uint8).clone()
    paged.paged_write(cache, one(k), one(v), plan)
    assert torch.equal(cache.data.view(torch.uint8), held)
    out = torch.empty(1, 4, D, device="cuda", dtype=BF16)
    paged.paged_attention(one(q), cache, plan, SCALE, out=one(out))
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [3000]), ([1] * 9, [70 * i + 1 for i in range(9)]), ([6, 300, 1, 40], [800, 5000, 9, 40])])
def test_the_output_may_be_the_queries(q_lens, kv_lens, dtype):
    from sensenova_u1_b200.ops import paged
    cache, tables, _ = make(kv_lens, 32, 2, dtype)
    plan = paged.build_plan(cache, 8, q_lens, kv_lens, tables)
    g = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn(sum(q_lens), 8, D, device="cuda", generator=g).to(BF16)
    want = paged.paged_attention(q, cache, plan, SCALE)
    assert paged.paged_attention(q, cache, plan, SCALE, out=q) is q
    assert torch.equal(q, want)


def test_a_plan_is_not_made_in_a_capture():
    from sensenova_u1_b200.ops import paged
    cache, tables, _ = make([40], 16, 2, BF16)
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="captured"):
            paged.build_plan(cache, 8, [3], [40], tables)


# ------------------------------------------------------------------ the engine over pages
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_engine_in_chunks_and_captured_tokens(dtype):
    """Two documents through ``InferenceEngine.paged_step``: prompts in chunks while the other decodes, then fixed tokens in a captured
    step, against the layers of the oracle in fp32."""
    from sensenova_u1_b200.config import tiny_mot
    from sensenova_u1_b200.inference.engine import InferenceEngine
    from sensenova_u1_b200.models import oracle
    from sensenova_u1_b200.models.params import ParamStore
    from sensenova_u1_b200.ops import paged
    from sensenova_u1_b200.ops.attention import make_meta
    cfg = tiny_mot(head_dim=128, patch_size=16, num_layers=2)
    store = ParamStore(cfg, device="cuda", with_grads=False)
    store.init_weights(3, std=0.05)
    eng = InferenceEngine(cfg, store)
    steps = [[150, 30], [61, 1], [1, 1], [1, 1], [1, 1], [1, 1]]
    total = [sum(s[i] for s in steps) for i in range(2)]
    g = torch.Generator().manual_seed(2)
    ids = [torch.randint(8, cfg.vocab_size, (n,), generator=g) for n in total]
    tables, pages = tables_for(total, 32)
    caches = eng.paged_caches(pages, 32, dtype)
    got, at = [[], []], [0, 0]

    def take(h, s):
        for i in range(2):
            got[i].append(h[sum(s[:i]):sum(s[:i + 1])].clone())
            at[i] += s[i]

    for s in steps[:3]:
        plan = paged.build_plan(caches[0], cfg.num_heads, s, [a + n for a, n in zip(at, s)], tables)
        take(eng.paged_step(plan, caches, ids=torch.cat([ids[i][at[i]:at[i] + s[i]] for i in range(2)])), s)
    left = len(steps) - 3
    plan = paged.build_plan(caches[0], cfg.num_heads, [1, 1], at, tables, grow=left)
    tok = torch.zeros(2, dtype=torch.long, device="cuda")
    out = torch.zeros(2, cfg.hidden_size, device="cuda", dtype=BF16)

    def step():
        plan.advance()
        out.copy_(eng.paged_step(plan, caches, ids=tok))

    tok.copy_(torch.tensor([ids[i][at[i]] for i in range(2)]))
    step()                                                # warm
    plan.advance(-1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for _ in range(left):
        tok.copy_(torch.tensor([ids[i][at[i]] for i in range(2)]))
        graph.replay()
        take(out, [1, 1])
    assert at == total
    p32 = {k: v.float() for k, v in store.p.items()}
    for i, n in enumerate(total):
        x = p32["embed_tokens"][ids[i].cuda()]
        pos = torch.arange(n, device="cuda")
        meta = make_meta(torch.zeros(n, device="cuda"), pos)
        mask, isg = oracle.dense_mask(meta, meta), torch.zeros(n, dtype=torch.bool, device="cuda")
        pos3 = torch.stack([pos, torch.zeros_like(pos), torch.zeros_like(pos)])
        for l in range(cfg.num_layers):
            x = oracle.decoder_layer(p32, l, x, isg, pos3, mask, cfg)
        h = torch.cat(got[i]).float()
        # bf16 activations: the bound of the engine's other tests.  e4m3: half a step of every cached value, 2^-4, besides.
        assert ((h - x).norm() / x.norm()).item() < 3e-2 + (0 if dtype == BF16 else 2.0 ** -4)


def test_engine_refusals():
    from sensenova_u1_b200.config import tiny_mot
    from sensenova_u1_b200.inference.engine import InferenceEngine
    from sensenova_u1_b200.models.params import ParamStore
    from sensenova_u1_b200.ops import paged
    cfg = tiny_mot(head_dim=128, patch_size=16, num_layers=2)
    store = ParamStore(cfg, device="cuda", with_grads=False)
    store.init_weights(0)
    eng = InferenceEngine(cfg, store)
    caches = eng.paged_caches(4, 16)
    plan = paged.build_plan(caches[0], cfg.num_heads, [3], [3], [[1]])
    ids = torch.tensor([5, 6, 7])
    with pytest.raises(ValueError):
        eng.paged_step(plan, caches[:1], ids=ids)
    with pytest.raises(ValueError):
        eng.paged_step(plan, caches, ids=ids[:2])
    with pytest.raises(ValueError):
        eng.paged_step(plan, caches)
    assert eng.paged_step(plan, caches, ids=ids).shape == (3, cfg.hidden_size)
    empty = paged.build_plan(caches[0], cfg.num_heads, [0], [3], [[1]])
    assert eng.paged_step(empty, caches, ids=ids[:0]).shape == (0, cfg.hidden_size)
    x = torch.zeros(3, cfg.hidden_size, device="cuda", dtype=BF16)
    assert eng.paged_step(plan, caches, embeds=x).shape == x.shape
    for bad in (x.float(), x[:, :-8], x[:2], x.cpu()):
        with pytest.raises(ValueError):
            eng.paged_step(plan, caches, embeds=bad)
    for bad in (torch.zeros(3, 2), torch.zeros(2, 3), torch.zeros(3)):
        with pytest.raises(ValueError):
            eng.paged_step(plan, caches, ids=ids, pos3=bad.int())


# ------------------------------------------------------------------ keys, values and queries of very different sizes
def filled(kv, page, seed=0):
    """An e4m3 cache that holds, per sequence, the given keys and values ([2, heads, keys, 128]), and what it then holds in 64 bits."""
    from sensenova_u1_b200.ops import paged
    lens, hk = [x.shape[2] for x in kv], kv[0].shape[1]
    tables, pages = tables_for(lens, page, seed=seed)
    data, scales = torch.zeros(pages, 2, hk, page, D, device="cuda", dtype=E4M3), torch.ones(pages, 2, hk, page, device="cuda")
    rows = []
    for x, t in zip(kv, tables):
        codes, s = quantised(x.to(BF16))
        rows.append(codes.double() * s.double()[..., None])
        pos = torch.arange(x.shape[2])
        pg, off = torch.tensor(t)[pos // page].cuda(), (pos % page).cuda()
        data.view(torch.uint8)[pg, :, :, off] = codes.view(torch.uint8).permute(2, 0, 1, 3)
        scales[pg, :, :, off] = s.permute(2, 0, 1)
    return paged.PagedCache(data, scales), tables, rows


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("q_len", [3, 40, 300])
@pytest.mark.parametrize("q_size,k_size", [(2.0 ** -34, 0.0), (2.0 ** -64, 2.0 ** -64), (2.0 ** -100, 1.0), (2.0 ** -64, 2.0 ** 64)])
def test_tiny_queries_and_keys(q_len, q_size, k_size):
    """The factors of queries and keys together may be smaller than fp32 holds: hidden keys stay hidden."""
    from sensenova_u1_b200.ops import paged
    x = torch.randn(2, 2, q_len + 150, D, device="cuda", generator=gen(q_len))
    x[0] *= k_size
    cache, tables, rows = filled([x], 32)
    q = (torch.randn(q_len, 8, D, device="cuda", generator=gen(1)) * q_size).to(BF16)
    plan = paged.build_plan(cache, 8, [q_len], [q_len + 150], tables)
    ref, room = exact(q, [q_len], rows, causal([q_len], [q_len + 150]), E4M3)
    assert near(paged.paged_attention(q, cache, plan, SCALE), ref, room)


def scores_of_any_size(q_len, size, dtype):
    """One channel of every query is ``size``, and one key that all rows read has 8 there, the others 3 at most: the result is that key's
    value, rounded once as a product (2^-8, fp16 2^-11) and once as a result."""
    from sensenova_u1_b200.ops import paged
    n = q_len + 170
    x = torch.randn(2, 2, n, D, device="cuda", generator=gen(q_len))
    x[0].clamp_(-3, 3)
    at = torch.randint(170, (2, D), device="cuda", generator=gen(2))
    x[0].scatter_(1, at[:, None], 8.0)
    if dtype == E4M3:
        x[1] *= torch.exp2(torch.randint(-3, 4, (2, n, 1), device="cuda", generator=gen(3)).float())
        cache, tables, rows = filled([x], 32)
    else:
        tables, pages = tables_for([n], 32)
        cache = paged.PagedCache.empty(pages, 32, 2)
        fill = paged.build_plan(cache, 8, [n], [n], tables)
        kv = x.to(BF16).transpose(1, 2).contiguous()
        paged.paged_write(cache, kv[0], kv[1], fill)
        rows = [x.to(BF16).double()]
    d = torch.arange(q_len * 8, device="cuda").view(q_len, 8) * 5 % D
    q = torch.zeros(q_len, 8, D, device="cuda", dtype=BF16).scatter_(2, d[..., None], size)
    plan = paged.build_plan(cache, 8, [q_len], [n], tables)
    head = torch.arange(8, device="cuda") // 4
    want = rows[0][1][head, at[head, d]]
    out = paged.paged_attention(q, cache, plan, SCALE).double()
    assert ((out - want).abs() <= (2 * 2.0 ** -8 + 2.0 ** -11) * want.abs()).all()


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("q_len", [40, 300])
@pytest.mark.parametrize("size", [2.0 ** e for e in (12, 17, 20, 22, 24, 26, 28, 30, 33, 60, 100)])
def test_scores_of_any_size_in_chunks(q_len, size, dtype):
    scores_of_any_size(q_len, size, dtype)


@pytest.mark.parametrize("q_len,kv_len", [(2, 150), (40, 300), (70, 1000), (300, 700)])
def test_a_large_query_is_its_own_matter(q_len, kv_len):
    """Rows side by side whose sizes are 2^60 and 2^-60: every other row is as near as without them."""
    from sensenova_u1_b200.ops import paged
    cache, tables, rows = make([kv_len], 32, 2, E4M3)
    q = torch.randn(q_len, 8, D, device="cuda", generator=gen(q_len)).to(BF16)
    large = torch.zeros(q_len, 8, dtype=torch.bool, device="cuda")
    large[1::7, 3] = large[0::9, 6] = True
    q[large] *= 2.0 ** 60
    q[1::5, 1] *= 2.0 ** -60
    plan = paged.build_plan(cache, 8, [q_len], [kv_len], tables)
    ref, room = exact(q, [q_len], rows, causal([q_len], [kv_len]), E4M3)
    out = paged.paged_attention(q, cache, plan, SCALE)
    assert near(out[~large], ref[~large], room[~large])
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("q_len,split", [(3, False), (40, False), (40, True), (300, False), (300, True)])
def test_many_keys_without_values(q_len, split, monkeypatch):
    """Thousands of keys whose values are zero count in the sums that the others are divided by: values in the last 100 keys only, and
    all scores but those of the first tile nearly 2^8 times the first tile's (the running maximum is left behind)."""
    from sensenova_u1_b200.ops import paged
    if not split:
        monkeypatch.setattr(paged, "_waves", lambda tiles, heads, slots: tiles * 0 + 1)
    n = 9000 + q_len
    x = torch.zeros(2, 2, n, D, device="cuda")
    x[0, :, 128:, 0] = 5.4
    x[1, :, 8900:] = torch.randn(2, n - 8900, D, device="cuda", generator=gen(3)) + 0.5
    cache, tables, rows = filled([x], 64)
    q = torch.zeros(q_len, 8, D, device="cuda", dtype=BF16)
    q[..., 0] = 11.25                                     # scores of 5.37 = 7.74 in log2 units
    plan = paged.build_plan(cache, 8, [q_len], [n], tables)
    ref, room = exact(q, [q_len], rows, causal([q_len], [n]), E4M3)
    assert near(paged.paged_attention(q, cache, plan, SCALE), ref, room)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("q_len", [1, 4, 6, 8])
@pytest.mark.parametrize("size", [2.0 ** e for e in (12, 17, 20, 22, 24, 26, 28, 30, 33, 60, 100)])
def test_scores_of_any_size_in_few_rows(q_len, size, dtype):
    scores_of_any_size(q_len, size, dtype)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("q_len", [1, 4, 6, 8, 40, 300])
@pytest.mark.parametrize("size", [2.0 ** e for e in (12, 20, 24, 27, 30, 33, 60, 100)])
def test_equal_scores_of_any_size(q_len, size, dtype):
    """The largest score occurs in several tiles (the mean of equal values is that value), behind tiles of ordinary and negative ones."""
    from sensenova_u1_b200.ops import paged
    n = q_len + 900
    x = torch.zeros(2, 2, n, D, device="cuda")
    x[0] = -2.0 * torch.rand(2, n, D, device="cuda", generator=gen(q_len))
    x[0, :, :140, :64] = 2.0 ** -14                       # channels whose first scores are ordinary
    x[0, :, 300:900:75] = 7.0
    x[1] = torch.randn(2, 1, D, device="cuda", generator=gen(3))
    x[1, :, :300] *= -1
    if dtype == E4M3:
        cache, tables, rows = filled([x], 32)
    else:
        tables, pages = tables_for([n], 32)
        cache = paged.PagedCache.empty(pages, 32, 2)
        kv = x.to(BF16).transpose(1, 2).contiguous()
        paged.paged_write(cache, kv[0], kv[1], paged.build_plan(cache, 8, [n], [n], tables))
        rows = [x.to(BF16).double()]
    d = torch.arange(q_len * 8, device="cuda").view(q_len, 8) * 5 % D
    q = torch.zeros(q_len, 8, D, device="cuda", dtype=BF16).scatter_(2, d[..., None], size)
    plan = paged.build_plan(cache, 8, [q_len], [n], tables)
    want = rows[0][1][torch.arange(8, device="cuda") // 4, 300].expand(q_len, 8, D)
    out = paged.paged_attention(q, cache, plan, SCALE).double()
    assert ((out - want).abs() <= (2 * 2.0 ** -8 + 2.0 ** -11) * want.abs()).all()


def test_a_captured_engine_step_outlives_larger_ones():
    """Two captured decode steps; then a chunk larger than anything before, whose buffers replace the engine's, and tensors in whatever
    memory that left free; then both graphs at once on two streams: they write nothing of that, and give what eager steps give."""
    from sensenova_u1_b200.config import tiny_mot
    from sensenova_u1_b200.inference.engine import InferenceEngine
    from sensenova_u1_b200.models.params import ParamStore
    from sensenova_u1_b200.ops import paged
    for moe in ({}, dict(num_experts=8, num_experts_per_tok=2, gen_num_experts=8, gen_num_experts_per_tok=2, moe_intermediate_size=128)):
        cfg = tiny_mot(head_dim=128, patch_size=16, num_layers=2, **moe)
        store = ParamStore(cfg, device="cuda", with_grads=False)
        store.init_weights(3, std=0.05)
        eng = InferenceEngine(cfg, store)
        sets = [eng.paged_caches(24, 32) for _ in range(2)]
        g = torch.Generator().manual_seed(2)
        jobs = []
        for caches, n in zip(sets, (2, 5)):
            tables, kv = [list(range(4 * i, 4 * i + 4)) for i in range(n)], [40 + 7 * i for i in range(n)]
            prompt = paged.build_plan(caches[0], cfg.num_heads, kv, kv, tables)
            eng.paged_step(prompt, caches, ids=torch.randint(8, cfg.vocab_size, (sum(kv),), generator=g))
            plan = paged.build_plan(caches[0], cfg.num_heads, [1] * n, kv, tables, grow=3)
            tok = torch.randint(8, cfg.vocab_size, (n,), generator=g).cuda()
            out = torch.zeros(n, cfg.hidden_size, device="cuda", dtype=BF16)
            plan.advance()
            want = [eng.paged_step(plan, caches, ids=tok)]
            plan.advance()
            want.append(eng.paged_step(plan, caches, ids=tok))
            plan.advance(-2)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                plan.advance()
                out.copy_(eng.paged_step(plan, caches, ids=tok))
            jobs.append((graph, plan, tok, out, want, torch.cuda.Stream()))
        large = eng.paged_caches(40, 32)
        chunk = paged.build_plan(large[0], cfg.num_heads, [1200], [1200], [list(range(38))])
        before = sum(t.numel() for t in eng.ws.bufs.values())
        eng.paged_step(chunk, large, ids=torch.randint(8, cfg.vocab_size, (1200,), generator=g))
        assert sum(t.numel() for t in eng.ws.bufs.values()) > before
        torch.cuda.synchronize()
        held = [torch.full((1 << s,), 77, dtype=torch.uint8, device="cuda") for s in range(9, 22) for _ in range(8)]
        torch.cuda.synchronize()
        for i in range(2):
            for graph, _, _, _, _, stream in jobs:
                with torch.cuda.stream(stream):
                    graph.replay()
            torch.cuda.synchronize()
            for _, _, _, out, want, _ in jobs:
                assert torch.equal(out, want[i])
        assert all((x == 77).all() for x in held)


@pytest.mark.parametrize("q_len,dtype", [(1, BF16), (1, E4M3), (6, E4M3), (40, BF16), (40, E4M3), (300, E4M3)])      # every kernel
def test_attention_past_the_plan_is_reported(q_len, dtype):
    from sensenova_u1_b200.ops import _lib, paged
    cache, tables, _ = make([400, 20], 32, 2, dtype)
    q = torch.randn(q_len, 8, D, device="cuda", generator=gen(3)).to(BF16)
    plan = paged.build_plan(cache, 8, [q_len, 0], [398, 20], tables, grow=2)       # a sequence without new rows does not grow
    for n in range(3):
        paged.paged_attention(q, cache, plan, SCALE)
        _lib.check_status()
        plan.advance()
    paged.paged_attention(q, cache, plan, SCALE)
    with pytest.raises(_lib.NativeLibraryError, match="limit"):
        _lib.check_status()


SIZES = [0.0, 2.0 ** -40, 1.0, 2.0 ** 8, 2.0 ** -40, 0.0, 1.0, 2.0 ** -20]


@pytest.mark.parametrize("q_len,split", [(3, True), (40, True), (40, False), (300, True), (300, False)])
@pytest.mark.parametrize("order", ["as they are", "backwards"])
@pytest.mark.parametrize("k_sizes", [[1.0], [2.0 ** -30, 2.0, 0.0, 1.0, 0.25]])
def test_tiles_of_very_different_sizes(q_len, split, order, k_sizes, monkeypatch):
    """Tiles of 128 keys with values from 2^-40 to 2^8 or zeros, and keys that differ by tile; rows that read only the first of them."""
    from sensenova_u1_b200.ops import paged
    if not split:
        monkeypatch.setattr(paged, "_waves", lambda tiles, heads, slots: tiles * 0 + 1)
    kv, sizes = [300 + 128 * 8 - 50, 128 * 7 + 3], SIZES if order == "as they are" else SIZES[::-1]
    q_lens, xs = [q_len, 2], []
    for i, n in enumerate(kv):
        tile = (torch.arange(n) // 128)
        x = torch.randn(2, 2, n, D, device="cuda", generator=gen(i))
        x[1] *= torch.tensor(sizes * 2)[tile].cuda()[:, None]
        x[0] *= torch.tensor(k_sizes * 16)[tile].cuda()[:, None]
        xs.append(x)
    cache, tables, rows = filled(xs, 32)
    lim = [1 + (i * 389) % n for n, k in zip(kv, q_lens) for i in range(k)]
    lim[0], lim[1] = kv[0], 128
    q = torch.randn(sum(q_lens), 8, D, device="cuda", generator=gen(7)).to(BF16)
    for limits in (lim, None):
        plan = paged.build_plan(cache, 8, q_lens, kv, tables, limits=limits)
        ref, room = exact(q, q_lens, rows, causal(q_lens, kv) if limits is None else torch.tensor(lim, device="cuda"), E4M3)
        out = paged.paged_attention(q, cache, plan, SCALE)
        assert near(out, ref, room)


@pytest.mark.parametrize("rows", [4, 8, 12, 16, 20, 24, 28, 32])
def test_probabilities_of_few_bf16_rows_keep_sixteen_bits(rows):
    """One-hot queries make scores exact, values of +1 and -1 make the result a difference of probabilities: each is off by 2^-16 of
    itself (two bf16 numbers) and by 2^-20 (exponential and fp32 sums; scores below 2^3), and the result is rounded once."""
    from sensenova_u1_b200.ops import paged
    n = 37
    g = gen(rows)
    x = torch.zeros(3, 2, 1, 16, D, device="cuda", dtype=BF16)
    k = torch.randn(n, D, device="cuda", generator=g).to(BF16)
    v = torch.ones(n, D, device="cuda", dtype=BF16)
    v[torch.rand(n, D, device="cuda", generator=g) < 0.5] = -1
    table = [2, 0, 1]
    for i in range(n):
        x[table[i // 16], 0, 0, i % 16], x[table[i // 16], 1, 0, i % 16] = k[i], v[i]
    cache = paged.PagedCache(x)
    q = torch.zeros(rows // 4, 4, D, device="cuda", dtype=BF16)
    q.view(rows, D)[torch.arange(rows), torch.arange(rows) * 3] = 1.0
    plan = paged.build_plan(cache, 4, [rows // 4], [n], [table], limits=[n] * (rows // 4))
    out = paged.paged_attention(q, cache, plan, 1.0).view(rows, D).double()
    p = torch.softmax(k[:, torch.arange(rows) * 3].double().T, -1)
    ref = p @ v.double()
    assert ((out - ref).abs() <= 2.0 ** -16 + 2.0 ** -20 + 2.0 ** -8 * ref.abs()).all()


def engine_and_oracle(dtype, **kw):
    """A prompt with a picture through ``InferenceEngine.paged_step`` in three chunks (the picture whole in one) beside a decoding text,
    and the oracle's layers in fp32 over the whole of both: hidden rows of both, and the routers' logits."""
    from sensenova_u1_b200.config import tiny_mot
    from sensenova_u1_b200.inference.engine import InferenceEngine
    from sensenova_u1_b200.models import oracle
    from sensenova_u1_b200.models.params import ParamStore
    from sensenova_u1_b200.ops import paged
    from sensenova_u1_b200.ops.attention import make_meta
    cfg = tiny_mot(head_dim=128, patch_size=16, num_layers=2, **kw)
    store = ParamStore(cfg, device="cuda", with_grads=False)
    store.init_weights(5, std=0.05)
    eng = InferenceEngine(cfg, store)
    total, a, b, wide = [190, 33], 60, 60 + 8 * 9, 9          # the first: 60 tokens of text, a picture of 8 x 9, text again
    g = gen(3)
    embeds = [(torch.randn(n, cfg.hidden_size, device="cuda", generator=g) * 0.05).to(BF16) for n in total]
    t = torch.arange(total[0])
    t[a:b], t[b:] = a, a + 1 + torch.arange(total[0] - b)
    h, w, img = torch.zeros_like(t), torch.zeros_like(t), torch.zeros_like(t)
    h[a:b], w[a:b], img[a:b] = torch.arange(b - a) // wide, torch.arange(b - a) % wide, 1
    pos3 = [torch.stack([t, h, w]), torch.stack([torch.arange(total[1]), torch.zeros(total[1]), torch.zeros(total[1])]).long()]
    limits = [[b if a <= i < b else i + 1 for i in range(total[0])], list(range(1, total[1] + 1))]
    tables, pages = tables_for(total, 32)
    caches = eng.paged_caches(pages, 32, dtype)
    got, at = [[], []], [0, 0]
    for s in ([40, 31], [100, 1], [50, 1]):
        pick = lambda x, d=0: torch.cat([x[i].narrow(d, at[i], s[i]) for i in range(2)], d)
        plan = paged.build_plan(caches[0], cfg.num_heads, s, [x + n for x, n in zip(at, s)], tables,
                                limits=[x for i in range(2) for x in limits[i][at[i]:at[i] + s[i]]])
        out = eng.paged_step(plan, caches, embeds=pick(embeds), pos3=pick(pos3, 1))
        for i in range(2):
            got[i].append(out[sum(s[:i]):sum(s[:i + 1])].clone())
            at[i] += s[i]
    assert at == total
    p32, want, logits = {k: v.float() for k, v in store.p.items()}, [], []
    for i, n in enumerate(total):
        x, pos = embeds[i].float(), pos3[i].cuda()
        meta = make_meta(torch.zeros(n, device="cuda"), pos[0], img.cuda() if i == 0 else None)
        aux = []
        for l in range(cfg.num_layers):
            x = oracle.decoder_layer(p32, l, x, torch.zeros(n, dtype=torch.bool, device="cuda"), pos, oracle.dense_mask(meta, meta), cfg, aux=aux)
        want.append(x)
        logits.append([u for u, _ in aux])
    return [torch.cat(x).float() for x in got], want, logits


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_engine_with_a_picture(dtype):
    got, want, _ = engine_and_oracle(dtype)
    for h, x in zip(got, want):
        # the bounds of test_engine_in_chunks_and_captured_tokens
        assert ((h - x).norm() / x.norm()).item() < 3e-2 + (0 if dtype == BF16 else 2.0 ** -4)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_engine_of_a_mixture_with_a_picture(dtype):
    got, want, logits = engine_and_oracle(dtype, num_experts=8, num_experts_per_tok=2, gen_num_experts=8, gen_num_experts_per_tok=2,
                                          moe_intermediate_size=128)
    room = 5e-2 + (0 if dtype == BF16 else 2.0 ** -4)          # 5e-2: the bound of the engine's other test of a mixture
    clears = 0
    for h, x, layers in zip(got, want, logits):
        # rows whose choice of experts is not near to another one: logits are off by the rows' error, room of their size, random in sign
        clear = torch.ones(len(h), dtype=torch.bool, device="cuda")
        for u in layers:
            top = u.sort(-1, descending=True).values
            clear &= top[:, 1] - top[:, 2] > 2 * room * u.std()
        clears += int(clear.sum())
        assert ((h - x)[clear].norm() / x[clear].norm()).item() < room
    assert clears > sum(map(len, got)) // 5                     # (of normal logits half are that clear per layer, a quarter in both)
