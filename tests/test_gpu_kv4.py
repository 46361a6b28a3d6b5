"""The paged 4-bit cache on the GPU: the step's plan, append and read-back, and attention over it, against the float64
restatement (oracle/attention.py).

What is stored is exact: power-of-two scales and roundings to a short list of values, so append and read-back are compared
for equality.  The attention's bars are per element, from its arithmetic (S: the largest sum of |q| |k| scale of the row, A:
the sum of p |v|, n: the keys):
  scores   float32 sums of D exact products: 2 D 2^-24 S, and what two bf16 terms leave of a float16 or float32 q, 2^-18 S;
           a score's error is a relative error of p, in the numerator and in the sum: twice;
  P        rounded to bf16, 2^-9, or to two bf16 terms, 2^-18; exp2 a few 2^-24;
  sums     n 2^-24 twice; the output's rounding 2^-9 (bf16), 2^-11 (f16).
All of them times A, which is at least |o|.  A bf16 value's rounding can be twice that, 2^-8: with a single term of P a row
of few keys would reach past these bars (such rows' P are two terms), one of many averages its roundings far below them."""
import random

import pytest
import torch

from macai.layer import kv4_append, kv4_attention, kv4_cache, kv4_plan, kv4_read, rotary, rotary_table
from oracle import attention as A

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I32 = dict(dtype=torch.int32, device="cuda")


def _bar(dtype, D, n, most, mag):
    one = dtype == BF16
    score = 2 * D * 2.0 ** -24 * most + (0 if one else 2.0 ** -18 * most)
    p = (2.0 ** -9 if one else 2.0 ** -18) + 8 * 2.0 ** -24
    out = {BF16: 2.0 ** -9, F16: 2.0 ** -11, F32: 2.0 ** -24}[dtype]
    return (2 * score[..., None] + p + 2 * n * 2.0 ** -24 + out) * mag * 1.02


def _setup(lens, Hk, D, page, dtype, seed, spare=3, junk=True):
    """A cache with random keys and values for requests of these lengths, in pages in a random order; every byte that no
    token wrote is 0xFF (a NaN's scale), table entries past a request's tokens are far out of range."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    cache = kv4_cache(pages, Hk, D, page)
    if junk:
        cache.fill_(255)
    order = torch.randperm(pages, generator=gen).tolist()
    blocks = torch.full((len(lens), max(max(need), 1) + 1), 2 ** 30, dtype=torch.int32)
    slots, at = [], 0
    for r, n in enumerate(lens):
        ids = order[at:at + need[r]]
        at += need[r]
        blocks[r, :need[r]] = torch.tensor(ids, dtype=torch.int32)
        slots += [ids[t // page] * page + t % page for t in range(n)]
    T = sum(lens)
    k, v = torch.randn(T, Hk, D, generator=gen).to(dtype), torch.randn(T, Hk, D, generator=gen).to(dtype)
    if T:
        kv4_append(None, k.cuda(), v.cuda(), cache, torch.tensor(slots, device="cuda"))
    return cache, blocks.cuda(), slots, A.stored(k), A.stored(v), gen


def _against_oracle(o, q, ks, vs, lens, qlens, dtype, scale=None):
    """Every row of every request within its bar; returns the worst error over its bar."""
    D, worst, tq, tk = q.shape[-1], 0.0, 0, 0
    o = o.double().cpu()
    assert torch.isfinite(o).all()
    for n, m in zip(lens, qlens):
        ref, mag, most = A.attention(q[tq:tq + m], ks[tk:tk + n], vs[tk:tk + n], D ** -0.5 if scale is None else scale)
        bar = _bar(dtype, D, n, most, mag) + 1e-37
        worst = max(worst, float(((o[tq:tq + m] - ref).abs() / bar).max()) if m else 0.0)
        tq, tk = tq + m, tk + n
    print(f"worst error over its bar {worst:.3f}", flush=True)
    assert worst <= 1.0
    return worst


# ---- append and read ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,page,T,Hk,Hq,width,interleaved", [(64, 16, 1, 1, 1, 64, False), (128, 32, 37, 2, 6, 32, True),
                                                              (256, 64, 70, 1, 8, 64, False), (64, 256, 50, 3, 3, 16, True),
                                                              (128, 16, 19, 8, 8, 128, False), (256, 128, 5, 2, 4, 48, False)])
def test_append_then_read(D, page, T, Hk, Hq, width, interleaved, dtype):
    gen = torch.Generator().manual_seed(5)
    qkv = torch.randn(T, Hq + 2 * Hk, D, generator=gen) * 2.0 ** torch.randint(-12, 12, (T, Hq + 2 * Hk, 1), generator=gen)
    qkv = qkv.to(dtype)
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=gen)[:T]
    slots[T // 2:T // 2 + 1] = -1 if T > 1 else slots[0]
    cache, table = kv4_cache(pages, Hk, D, page), rotary_table(width, 900, device="cuda")
    before = cache.clone()
    pos = torch.randint(0, 900, (T,), generator=gen, dtype=torch.int32)
    q, k, v = qkv.cuda().split([Hq, Hk, Hk], 1)
    qo = kv4_append(q, k, v, cache, slots.cuda(), table, pos.cuda(), interleaved)
    rq, rk = rotary(q, k, table, pos.cuda(), interleaved)
    assert torch.equal(qo, rq)
    gk, gv = kv4_read(cache, slots.cuda(), D, dtype=F32)
    there = slots >= 0
    assert torch.equal(gk[there.cuda()].double().cpu(), A.stored(rk.cpu())[there])
    assert torch.equal(gv[there.cuda()].double().cpu(), A.stored(v.cpu())[there])
    assert (gk[~there.cuda()] == 0).all() and (gv[~there.cuda()] == 0).all()
    # nothing but the tokens' own bytes was written
    others = [s for s in range(pages * page) if s not in set(slots.tolist())]
    if others:
        ok, ov = kv4_read(cache, torch.tensor(others, device="cuda"), D, dtype=F32)
        assert (ok == 0).all() and (ov == 0).all()
    assert int((cache != before).sum()) <= int(there.sum()) * 2 * Hk * 17 * D // 32
    assert torch.equal(kv4_read(cache, slots.cuda(), D, dtype=BF16)[0].float(), gk)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_page_bytes_are_the_documented_ones(D):
    """A page read byte by byte, from the format's description alone."""
    page, gen = 32, torch.Generator().manual_seed(6)
    k, v = torch.randn(page, 1, D, generator=gen), torch.randn(page, 1, D, generator=gen)
    cache = kv4_cache(1, 1, D, page)
    kv4_append(None, k.cuda(), v.cuda(), cache, torch.arange(page, device="cuda"))
    raw = cache.cpu()[0, :, 0].tolist()
    W = min(D, 128)
    run = W // 16
    for which, x in ((0, A.stored(k)), (1, A.stored(v))):
        for t in range(page):
            b, o = t // 16 * (17 * D // 2), t % 16
            for c in range(D):
                if which == 0:
                    code, sc = c // 32 * 256 + o * 16 + c % 32 // 2, 8 * D + c // 32 * 16 + o
                else:
                    code = c // W * 8 * W + o // 4 * 2 * W + c % W // run * 2 * run + o % 4 * (run // 2) + c % run // 2
                    sc = 8 * D + o // 4 * (D // 8) + c // 32 * 4 + o % 4
                byte = raw[which][b + code] >> (4 * (c % 2)) & 15
                value = A.MAGNITUDES[byte & 7] * (-1 if byte & 8 else 1) * 2.0 ** (raw[which][b + sc] - 127)
                assert value == float(x[t, 0, c]), (which, t, c)


@pytest.mark.parametrize("T", [4095, 4096, 5001, 9000])
def test_reading_many_rows(T):
    """Rows in any number come out as they do in calls of a few; slots outside of the cache among them."""
    gen = torch.Generator().manual_seed(22)
    cache = torch.randint(0, 128, (200, 2, 1, 32 * 17 * 64 // 32), generator=gen, dtype=torch.uint8).cuda()
    slots = torch.randint(-2, 200 * 32 + 2, (T,), generator=gen).cuda()
    k, v = kv4_read(cache, slots, 64)
    for a in range(0, T, 1000):
        few = kv4_read(cache, slots[a:a + 1000], 64)
        assert torch.equal(k[a:a + 1000], few[0]) and torch.equal(v[a:a + 1000], few[1]), a


def test_append_extremes():
    """Ties, the smallest and largest scales, zeros, and groups that hold an infinity or a NaN (they alone read as NaN)."""
    x = torch.zeros(8, 1, 64)
    x[0, 0, :8] = torch.tensor([7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    x[1, 0, :3] = torch.tensor([7.001, -0.5, 0.49])
    x[2, 0, 3], x[2, 0, 40] = float("inf"), 1.0
    x[3, 0, 33], x[3, 0, 2] = float("nan"), -3.0
    x[4, 0, :2] = torch.tensor([3.4e38, -1e38])
    x[5, 0, :2] = torch.tensor([1e-38, -1e-40])
    x[6, 0, :2] = torch.tensor([-float("inf"), float("nan")])
    cache, slots = kv4_cache(1, 1, 64, 16), torch.arange(8, device="cuda")
    kv4_append(None, x.cuda(), x.flip(0).contiguous().cuda(), cache, slots)
    k, v = kv4_read(cache, slots, 64, dtype=F32)
    want = A.stored(x)
    for got, ref in ((k, want), (v, want.flip(0))):
        got = got.double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(ref))


# ---- the plan ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,ctx,most,page,W,F,pad,seed", [(1, 0, 1, 16, 4, 4, 0, 1), (5, 40, 9, 16, 6, 60, 3, 2),
                                                          (64, 300, 1, 64, 8, 70, 0, 3), (300, 50, 700, 32, 30, 9000, 700, 4),
                                                          (1024, 9, 3, 16, 3, 500, 0, 5), (3000, 20, 4, 16, 2, 2500, 10, 6),
                                                          (2, 10, 0, 16, 2, 0, 0, 7), (3, 100, 900, 128, 20, 3, 5, 8)])
def test_plan(B, ctx, most, page, W, F, pad, seed):
    """Against the walk over requests: padding rows, pages that run out (small F), tables that are too narrow (small W),
    requests without new tokens, more requests than a workgroup takes at once; planned twice from the same inputs."""
    rng = random.Random(seed)
    lens = [min(rng.randint(0, ctx), W * page) for _ in range(B)]
    new = [rng.choice([0, most, rng.randint(0, most)]) for _ in range(B)]
    have = sum(-(-n // page) for n in lens)
    pool = list(range(have + F))
    rng.shuffle(pool)
    blocks = [[pool.pop() if c < -(-n // page) else -7 for c in range(W)] for n in lens]
    head, tokens = rng.choice([0, 2]), sum(new) + pad
    want = A.plan(lens, new, blocks, pool, head, tokens, page)
    table = torch.tensor(blocks, **I32)
    args = (torch.tensor(lens, **I32), torch.tensor(new, **I32), table, torch.tensor(pool, **I32), torch.tensor([head], **I32))
    for _ in range(2):
        pos, slots, starts, total, nxt = kv4_plan(*args, tokens, page)
        assert pos.tolist() == want[0] and slots.tolist() == want[1]
        assert starts.tolist() == want[2] and total.tolist() == want[3] and nxt.tolist() == [want[4]]
        # entries of pages that no token begins on (past the rows given) are the walk's all the same
        assert table.tolist() == want[5]


def test_plan_takes_negative_lengths_as_zero_and_too_few_rows():
    t = torch.full((2, 3), -1, **I32)
    i = lambda *x: torch.tensor(x, **I32)  # noqa: E731
    pos, slots, starts, total, nxt = kv4_plan(i(-5, 4), i(3, -2), t, i(9, 8, 7), i(0), 2, 16)
    assert pos.tolist() == [0, 1] and slots.tolist() == [144, 145]          # the third token has no row
    assert starts.tolist() == [0, 3, 3] and total.tolist() == [3, 4] and nxt.tolist() == [1]


# ---- attention --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,Hk,G,page", [(64, 2, 1, 16), (64, 1, 5, 32), (128, 2, 4, 64), (128, 1, 16, 16), (256, 2, 8, 64),
                                         (256, 1, 3, 256), (128, 1, 24, 128)])
def test_one_token_each(D, Hk, G, page, dtype):
    """Generation: lengths around the ends of blocks, tiles and pages, an empty request, many requests at once."""
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 517, 1000]
    cache, blocks, _, ks, vs, gen = _setup(lens, Hk, D, page, dtype, 11)
    q = torch.randn(len(lens), Hk * G, D, generator=gen).to(dtype)
    lens_d = torch.tensor(lens, **I32)
    o = kv4_attention(q.cuda(), cache, blocks, lens_d)
    assert (o[0] == 0).all() and o.dtype == dtype
    _against_oracle(o, q, ks, vs, lens, [1] * len(lens), dtype)
    starts = torch.arange(len(lens) + 1, **I32)
    assert torch.equal(kv4_attention(q.cuda(), cache, blocks, lens_d, starts), o)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,Hk,G,page,lens,qlens", [
    (128, 2, 4, 16, [5, 40, 0, 200, 33], [2, 4, 0, 3, 0]),                 # drafts; requests with none, and with no tokens
    (256, 1, 8, 64, [70, 300], [3, 4]),                                    # 32 rows to a group
    (64, 1, 2, 32, [130, 1, 77], [130, 1, 30]),                            # prompts from their first token on
    (128, 1, 3, 16, [400, 90], [100, 90]),                                 # groups of heads that 128 is no multiple of
    (256, 2, 8, 64, [260, 5], [40, 5]),                                    # several row groups a request
    (64, 2, 16, 16, [2, 50], [5, 20]),                                     # more queries than tokens: the first see nothing
    (128, 4, 1, 128, [700, 3, 129, 64], [300, 1, 129, 2])])
def test_several_tokens_each(D, Hk, G, page, lens, qlens, dtype):
    cache, blocks, _, ks, vs, gen = _setup(lens, Hk, D, page, dtype, 12)
    T = sum(qlens)
    q = torch.randn(T + 2, Hk * G, D, generator=gen).to(dtype)             # two rows past the last request's
    starts = torch.tensor([0] + qlens).cumsum(0).to(torch.int32).cuda()
    o = kv4_attention(q.cuda(), cache, blocks, torch.tensor(lens, **I32), starts)
    assert (o[T:] == 0).all()
    _against_oracle(o[:T], q[:T], ks, vs, lens, qlens, dtype)


@pytest.mark.parametrize("B,lens,qlen,G,D,Hk", [(1, [9000], 1, 8, 256, 2), (1, [5001], 1, 4, 128, 1), (3, [7000, 20, 3100], 1, 8, 64, 2),
                                               (2, [2500, 1800], 3, 8, 128, 1), (1, [2600], 33, 4, 64, 1)])
def test_long_contexts_split_over_the_chip(B, lens, qlen, G, D, Hk):
    """Contexts cut into many pieces and joined, uneven requests among them."""
    cache, blocks, _, ks, vs, gen = _setup(lens, Hk, D, 32, BF16, 13)
    q = torch.randn(B * qlen, Hk * G, D, generator=gen).to(BF16) * 2
    starts = torch.arange(0, B * qlen + 1, qlen, **I32)
    args = (q.cuda(), cache, blocks, torch.tensor(lens, **I32), starts)
    o = kv4_attention(*args)
    _against_oracle(o, q, ks, vs, lens, [qlen] * B, BF16)
    for _ in range(3):
        assert torch.equal(kv4_attention(*args), o)                       # the same bits every time


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B,Hk,G,D,ctx,most", [(12, 3, 8, 128, 300, 60), (10, 2, 8, 256, 200, 70), (9, 4, 10, 64, 260, 50)])
def test_many_row_groups_of_prompts(B, Hk, G, D, ctx, most, dtype):
    """More row groups than an eighth of the workgroups: few parts to a row group, most of them whole."""
    rng = random.Random(B)
    qlens = [most] + [rng.randint(most // 2, most) for _ in range(B - 1)]
    lens = [n + rng.randint(0, ctx) for n in qlens]
    cache, blocks, _, ks, vs, gen = _setup(lens, Hk, D, 32, dtype, 23)
    q = torch.randn(sum(qlens), Hk * G, D, generator=gen).to(dtype)
    starts = torch.tensor([0] + qlens).cumsum(0).to(torch.int32).cuda()
    o = kv4_attention(q.cuda(), cache, blocks, torch.tensor(lens, **I32), starts)
    _against_oracle(o, q, ks, vs, lens, qlens, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B,Hk,G,D,ctx,most", [(3, 2, 8, 128, 700, 7), (60, 8, 6, 256, 40, 5), (70, 1, 8, 64, 200, 6),
                                               (64, 2, 8, 128, 90, 4), (6, 1, 16, 256, 1500, 4), (130, 2, 4, 64, 30, 1)])
def test_requests_of_several_row_groups(B, Hk, G, D, ctx, most, dtype):
    """Few requests, whose row groups are cut apart from each other, and many, whose row groups share workgroups: with and
    without queries, with fewer tokens than queries, and with none."""
    rng = random.Random(B)
    lens = [0, 1, ctx] + [rng.randint(0, ctx) for _ in range(B - 3)]
    qlens = [most, most, most] + [rng.randint(0, most) for _ in range(B - 3)]
    cache, blocks, _, ks, vs, gen = _setup(lens, Hk, D, 16, dtype, 21)
    q = torch.randn(sum(qlens), Hk * G, D, generator=gen).to(dtype)
    starts = torch.tensor([0] + qlens).cumsum(0).to(torch.int32).cuda()
    o = kv4_attention(q.cuda(), cache, blocks, torch.tensor(lens, **I32), starts)
    _against_oracle(o, q, ks, vs, lens, qlens, dtype)


def test_scores_that_grow_along_the_keys():
    """The running maximum moves at every step, and large scores neither overflow nor lose the others."""
    lens = [900]
    cache, blocks, slots, ks, vs, gen = _setup(lens, 1, 64, 16, F32, 14)
    ramp = torch.linspace(-400, 400, 900)[:, None, None] * torch.ones(1, 1, 64) / 8
    vals = torch.randn(900, 1, 64, generator=gen)
    kv4_append(None, ramp.cuda(), vals.cuda(), cache, torch.tensor(slots, device="cuda"))
    q = torch.ones(1, 2, 64)
    q[:, 1] = -1
    o = kv4_attention(q.cuda(), cache, blocks, torch.tensor(lens, **I32))
    _against_oracle(o, q, A.stored(ramp), A.stored(vals), lens, [1], F32)


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F32), (256, BF16)])
def test_hidden_nan_and_infinity_stay_hidden(D, dtype):
    """A NaN or an infinity in a key or value that a query does not see leaves its row as it is; rows that see a value's
    show NaN in that group of channels alone, rows that see a key's are NaN."""
    lens, qlens, G, Hk = [50, 45], [12, 45], 2, 1
    cache, blocks, slots, ks, vs, gen = _setup(lens, Hk, D, 16, dtype, 15)
    q = torch.randn(sum(qlens), Hk * G, D, generator=gen).to(dtype)
    starts = torch.tensor([0, 12, 57], **I32)
    lens_d = torch.tensor(lens, **I32)
    clean = kv4_attention(q.cuda(), cache, blocks, lens_d, starts)
    bad_v = torch.randn(1, Hk, D, generator=gen)
    bad_v[0, 0, 37] = float("nan")
    at = 44                                             # the first request's queries are its tokens 38 .. 49
    one = torch.tensor([slots[at]], device="cuda")
    kv4_append(None, ks[at:at + 1].float().cuda(), bad_v.cuda(), cache, one)
    o = kv4_attention(q.cuda(), cache, blocks, lens_d, starts)
    see = torch.arange(12) >= at - 38
    hit = torch.zeros(D, dtype=torch.bool)
    hit[32:64] = True
    nan = torch.isnan(o[:12]).cpu()
    assert torch.equal(nan, (see[:, None, None] & hit[None, None]).expand(12, G, D))
    a, b = o[:12][~see.cuda()].float(), clean[:12][~see.cuda()].float()
    assert torch.allclose(a, b, rtol=2.0 ** -7, atol=2.0 ** -7)            # rounded in another order
    assert torch.equal(o[12:], clean[12:])
    bad_k = torch.full((1, Hk, D), float("inf"))
    kv4_append(None, bad_k.cuda(), vs[at:at + 1].float().cuda(), cache, one)
    o = kv4_attention(q.cuda(), cache, blocks, lens_d, starts)
    assert torch.isnan(o[:12][see.cuda()]).all() and torch.equal(o[:12][~see.cuda()], clean[:12][~see.cuda()])


def test_a_page_outside_of_the_cache_is_loud():
    lens = [100, 40, 30]
    cache, blocks, _, ks, vs, gen = _setup(lens, 2, 128, 16, BF16, 16)
    q = torch.randn(3, 8, 128, generator=gen).to(BF16).cuda()
    lens_d = torch.tensor(lens, **I32)
    clean = kv4_attention(q, cache, blocks, lens_d)
    for wrong in (-1, cache.shape[0], 2 ** 31 - 1):
        blocks[1, 1] = wrong
        o = kv4_attention(q, cache, blocks, lens_d)
        assert torch.isnan(o[1]).all() and torch.equal(o[0::2], clean[0::2])
    wide = torch.tensor([100, 40, 10 ** 9], **I32)        # more tokens than the table has room for: cut to the table
    assert torch.isnan(kv4_attention(q, cache, blocks, wide)[2]).all()


def test_strided_queries_scale_and_streams():
    lens = [80, 300, 1]
    cache, blocks, _, ks, vs, gen = _setup(lens, 2, 128, 32, BF16, 17)
    qkv = torch.randn(3, 12, 128, generator=gen).to(BF16)
    lens_d, q = torch.tensor(lens, **I32), qkv.cuda()[:, :8]
    assert not q.is_contiguous()
    o = kv4_attention(q, cache, blocks, lens_d, scale=0.2)
    _against_oracle(o, qkv[:, :8], ks, vs, lens, [1] * 3, BF16, scale=0.2)
    t = qkv.cuda().transpose(0, 1).contiguous().transpose(0, 1)[:, :8]
    assert torch.equal(kv4_attention(t, cache, blocks, lens_d, scale=0.2), o)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = kv4_attention(q, cache, blocks, lens_d, scale=0.2)
    s.synchronize()
    assert torch.equal(got, o)


def test_a_cache_past_32_bits():
    """Pages whose bytes begin beyond 2^32: slots, reads and attention address them."""
    D, Hk, page = 256, 8, 256
    per = 2 * Hk * page * 17 * D // 32
    pages = 2 ** 32 // per + 40
    cache = kv4_cache(pages, Hk, D, page)
    lens = [page + 30]
    ids = [pages - 1, pages - 7]
    gen = torch.Generator().manual_seed(18)
    slots = torch.tensor([ids[t // page] * page + t % page for t in range(lens[0])], device="cuda")
    k, v = torch.randn(lens[0], Hk, D, generator=gen).to(BF16), torch.randn(lens[0], Hk, D, generator=gen).to(BF16)
    kv4_append(None, k.cuda(), v.cuda(), cache, slots)
    gk, gv = kv4_read(cache, slots, D, dtype=F32)
    assert torch.equal(gk.double().cpu(), A.stored(k)) and torch.equal(gv.double().cpu(), A.stored(v))
    assert int(cache[:ids[1]].count_nonzero()) == 0
    q = torch.randn(1, 2 * Hk, D, generator=gen).to(BF16)
    o = kv4_attention(q.cuda(), cache, torch.tensor([ids], **I32), torch.tensor(lens, **I32))
    _against_oracle(o, q, A.stored(k), A.stored(v), lens, [1], BF16)


def _serve(steps, check_graph=False):
    """Requests served from their prompts on: plan, append and attend at every step, all lengths on the device."""
    gen = torch.Generator().manual_seed(19)
    B, Hq, Hk, D, page, W = 3, 8, 2, 64, 16, 12
    table = rotary_table(32, 400, device="cuda")
    cache = kv4_cache(40, Hk, D, page)
    blocks, free, head = torch.full((B, W), -1, **I32), torch.randperm(40, generator=gen).to(torch.int32).cuda(), torch.zeros(1, **I32)
    lens = torch.zeros(B, **I32)
    past = [[] for _ in range(B)]
    for new in steps:
        T = sum(new)
        qkv = torch.randn(T, Hq + 2 * Hk, D, generator=gen).to(BF16)
        q, k, v = qkv.cuda().split([Hq, Hk, Hk], 1)
        pos, slots, starts, lens, head = kv4_plan(lens, torch.tensor(new, **I32), blocks, free, head, T, page)
        qo = kv4_append(q, k, v, cache, slots, table, pos)
        o = kv4_attention(qo, cache, blocks, lens, starts)
        rq, rk = rotary(q, k, table, pos)
        at = 0
        for r, n in enumerate(new):
            past[r] += [(A.stored(rk[at + i:at + i + 1].cpu()), A.stored(v[at + i:at + i + 1].cpu())) for i in range(n)]
            at += n
        ks, vs = torch.cat([p[0] for x in past for p in x]), torch.cat([p[1] for x in past for p in x])
        _against_oracle(o, rq.cpu(), ks, vs, [len(x) for x in past], new, BF16)
    return head


def test_serving_from_prompts_on():
    head = _serve([[20, 1, 37], [1, 1, 1], [1, 0, 1], [4, 2, 1], [30, 1, 1]] + [[1, 1, 1]] * 6)
    assert 0 < int(head) <= 40


def test_a_captured_step():
    """A decode step in a HIP graph, replayed with other lengths, queries and slots in the same buffers: each replay equals
    the same step run eagerly."""
    gen = torch.Generator().manual_seed(20)
    B, Hq, Hk, D, page, W = 4, 8, 2, 128, 16, 40
    table = rotary_table(64, 700, device="cuda")
    qkv = torch.randn(B, Hq + 2 * Hk, D, generator=gen).to(BF16).cuda()
    free = torch.randperm(B * W, generator=gen).to(torch.int32).cuda()
    base = torch.randint(0, 256, (B * W, 2, Hk, page * 17 * D // 32), generator=gen, dtype=torch.uint8)
    base.clamp_(max=127)                                                   # finite values
    lens, blocks = torch.zeros(B, **I32), torch.zeros(B, W, **I32)
    cache, head, one = base.cuda(), torch.zeros(1, **I32), torch.ones(B, **I32)

    def step():
        pos, slots, starts, total, nxt = kv4_plan(lens, one, blocks, free, head, B, page)
        q = kv4_append(qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], cache, slots, table, pos)
        return kv4_attention(q, cache, blocks, total, starts), total, nxt

    def state(i):
        g = torch.Generator().manual_seed(100 + i)
        held = torch.randint(0, (W - 1) * page, (B,), generator=g).to(torch.int32)
        lens.copy_(held)
        blocks.copy_(torch.arange(B * W, dtype=torch.int32).view(B, W))
        cache.copy_(base)
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(BF16))

    state(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        state(i)
        graph.replay()
        got = [x.clone() for x in outs] + [cache.clone(), blocks.clone()]
        state(i)
        want = list(step()) + [cache, blocks]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
