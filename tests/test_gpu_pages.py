"""A prompt's own attention and a drafted tree's on the GPU against their float64 restatements.

Tolerances, from the formats. Index queries are formed in f64 on both sides: they are equal,
and so are selected pages. A page's score: the FP4 products of a head are multiples of a
quarter of the smallest pair of scales, at most 36 of the largest; where the scales of a query
and a key lie within 2^7 of each other their 128 products need 2 + 13 + 7 bits and f32 holds
their sum exactly. A head's max(0, x) w is summed as x w / 2 and |x| w / 2, so that what is
rounded has the magnitude of all |x w|, of heads below zero too. A lane's 32 heads go through
eight FMAs, two additions and one of the two tiles, a half's and the other's through one more:
12 roundings at most, each 2^-24 of the magnitudes' sum; a maximum moves no more than its
arguments.

An attention output is rounded to bf16, off by 2^-8 of it at most. Each probability is rounded
to bf16 too, 2^-8 of it. A logit's 576 exact products are added with as many roundings at most,
each 2^-24 of the terms' magnitudes (the FP8 matrix instruction lines its products up with the
largest and cuts what is below: 2^-16 of the magnitudes was seen, 578 2^-24 is 2^-14.8), and two
for the scale and the exponent. q comes as two E4M3 pieces. Four significant bits each hold
bf16's eight; only what is small beside its head's largest loses bits: with the first piece's
unit u the largest lies in (224 u, 448 u], the second piece's steps are 2^-9 u / 16 at least, half
of one is 2^-14 u, 2^-21.8 of the largest; in the last 64 dims 2^-9 u, so 2^-17.8. With L for
both, a probability and their sum move by L and the exponential's 2^-22 each, a part's scale by
2^-22 and its sum by as much; the sums of the values add 2^-24 of the magnitudes for each key.
Together an output moves by (2^-8 + 2 (L + 2^-21) + n 2^-24) sum p |v|. The roundings are at
random: over a whole tensor their root of squares stays within 2^-8 for each of the two kinds,
2^-7 of the norm together.
"""

import pytest
import torch

import pages_ref as ref
from sgl_amd_mono_amd import prompt, workloads
from sgl_amd_mono_amd.attn import SOFTMAX_SCALE, AttnCaches, AttnRuntime, AttnStep

pytestmark = pytest.mark.gpu
PAGE = 64


def _near(got, want, mag, top, keys, norm=True):
    got = got.cpu().double()
    bad = want.isnan()
    assert bool((got.isnan() == bad).all())
    tol = 2.0**-8 * want.abs() + (2.0**-8 + 2 * (top + 2.0**-21) + keys * 2.0**-24) * mag
    over = ((got - want).abs() / tol.clamp_min(1e-30))[~bad]
    assert float(over.max() if over.numel() else 0.0) <= 1.0, float(over.max())
    if norm and over.numel():
        off = float((got - want)[~bad].norm() / want[~bad].norm().clamp_min(1e-30))
        assert off <= 2.0**-7, off


# --------------------------------------------------------------------- queries
@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("tokens,wide,start", [(1, 0, 900), (3, 0, 0), (70, 64, 17), (129, 0, 5)])
def test_index_query(gpu_device, tokens, wide, start, f32):
    g = torch.Generator(device=gpu_device).manual_seed(tokens)
    cos, sin = workloads.rope_tables(start + tokens, gpu_device)
    x = (2.0 * torch.randn(tokens, wide + 8192, generator=g, device=gpu_device)).to(torch.float32 if f32 else torch.bfloat16)[:, wide:]
    pos = torch.arange(start, start + tokens, dtype=torch.int32, device=gpu_device)
    got = prompt.index_query(x, pos, cos, sin)
    want = ref.index_query(x.cpu(), pos.cpu(), cos.cpu(), sin.cpu())
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_index_query_pads_and_extreme_rows(gpu_device):
    g = torch.Generator(device=gpu_device).manual_seed(3)
    cos, sin = workloads.rope_tables(40, gpu_device)
    x = torch.randn(8, 8192, generator=g, device=gpu_device)
    x[1] = 0.0
    x[2] *= 1e30
    x[3] *= 1e-30
    x[4, 128 * 5 + 77] = torch.nan
    x[5, 128 * 63] = torch.inf
    pos = torch.tensor([0, 1, 2, 3, 4, 39, 40, -1], dtype=torch.int32, device=gpu_device)
    iq, iqs = (v.cpu() for v in prompt.index_query(x, pos, cos, sin))
    keep = torch.ones(8, 64, dtype=torch.bool)
    keep[4, 5] = keep[5, 63] = False
    clean = x.cpu().nan_to_num(0.0, posinf=0.0)
    want = ref.index_query(clean, pos.cpu(), cos.cpu(), sin.cpu())
    assert torch.equal(iq[keep], want[0][keep]) and torch.equal(iqs[keep], want[1][keep])
    assert bool((iqs[~keep] == 255).all()) and bool((iq[~keep] == 0).all())
    assert bool((iq[6:] == 0).all()) and bool((iqs[6:] == 0).all())


def test_index_query_of_no_tokens(gpu_device):
    cos, sin = workloads.rope_tables(4, gpu_device)
    iq, iqs = prompt.index_query(torch.empty(0, 8192, device=gpu_device), torch.empty(0, dtype=torch.int32, device=gpu_device), cos, sin)
    assert iq.shape == (0, 64, 64) and iqs.shape == (0, 64, 4)


# ---------------------------------------------------------------------- scores
def _requests(dev, spans, pads=0, spare=0, seed=7, pool=3):
    """Packed tokens of `spans` (first position, tokens), page tables with `spare` more columns."""
    need = [max(1, -(-(a + n) // PAGE)) for a, n in spans]
    table = torch.full((len(spans), max(need) + spare), -1, dtype=torch.int32)
    order = torch.randperm(sum(need) + pool, generator=torch.Generator().manual_seed(seed))
    at = 0
    for r, u in enumerate(need):
        table[r, :u] = order[at:at + u]
        at += u
    req = torch.cat([torch.full((n,), r) for r, (_, n) in enumerate(spans)] + [torch.full((pads,), -1)]).int()
    pos = torch.cat([torch.arange(a, a + n) for a, n in spans] + [torch.zeros(pads)]).int()
    return req.to(dev), pos.to(dev), table.to(dev), sum(need) + pool


def _index(dev, tokens, pages, seed=5):
    g = torch.Generator(device=dev).manual_seed(seed)
    u8 = dict(generator=g, device=dev, dtype=torch.uint8)
    return (torch.randint(0, 256, (tokens, 64, 64), **u8), torch.randint(124, 128, (tokens, 64, 4), **u8),
            torch.randn(tokens, 64, generator=g, device=dev).to(torch.bfloat16),
            AttnCaches(ikv=torch.randint(0, 256, (pages, 4, 64, 16), **u8), iks=torch.randint(125, 130, (pages, 4, 64), **u8), kv=None, kv_scale=None))


def _scores_near(got, iq, iqs, iw, req, pos, table, caches):
    want, mag = ref.page_scores(iq.cpu(), iqs.cpu(), iw.cpu(), req.cpu(), pos.cpu(), table.cpu(), caches.ikv.cpu(),
                                caches.iks.cpu(), got.shape[1])
    got = got.cpu().double()
    assert bool((got.isnan() == want.isnan()).all())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    assert bool(((got - want).abs() <= 12 * 2.0**-24 * mag)[fine].all())


@pytest.mark.parametrize("spans,pads,columns", [
    ([(0, 1)], 0, None), ([(63, 1)], 0, None), ([(64, 1)], 0, 9), ([(700, 9)], 0, None), ([(0, 131)], 0, 1),
    ([(5, 2), (200, 3), (0, 1), (64, 70)], 3, None), ([(3, 1)] * 9, 0, None), ([(1500, 6), (0, 0), (31, 5)], 1, 20),
])  # fmt: skip
def test_page_scores(gpu_device, spans, pads, columns):
    req, pos, table, pages = _requests(gpu_device, spans, pads, spare=1)
    iq, iqs, iw, caches = _index(gpu_device, len(pos), pages)
    got = prompt.page_scores(iq, iqs, iw, req, pos, table, caches, columns)
    assert got.shape == (len(pos), table.shape[1] if columns is None else columns)
    _scores_near(got, iq, iqs, iw, req, pos, table, caches)


def test_page_scores_of_tokens_in_any_order(gpu_device):
    req, pos, table, pages = _requests(gpu_device, [(90, 10), (0, 7), (300, 13)])
    iq, iqs, iw, caches = _index(gpu_device, len(pos), pages)
    order = torch.randperm(len(pos), generator=torch.Generator().manual_seed(1)).to(gpu_device)
    whole = prompt.page_scores(iq, iqs, iw, req, pos, table, caches)
    got = prompt.page_scores(iq[order], iqs[order], iw[order], req[order], pos[order], table, caches)
    assert torch.equal(got, whole[order])  # a token's bits do not depend on its company
    for n in (0, 12, 29):
        one = prompt.page_scores(iq[n:n + 1], iqs[n:n + 1], iw[n:n + 1], req[n:n + 1], pos[n:n + 1], table, caches)
        assert torch.equal(one[0], whole[n])


def test_page_scores_bad_pages_requests_and_values(gpu_device):
    req, pos, table, pages = _requests(gpu_device, [(200, 12), (100, 9)])
    iq, iqs, iw, caches = _index(gpu_device, len(pos), pages)
    req[3], req[4], pos[5], pos[6] = 2, -5, -1, 1 << 30  # (a position far behind the table sees all of it)
    table[0, 1], table[0, 2] = pages, -7
    caches.iks[int(table[1, 0]), 2, 9] = 255  # key 9 % 16 ...: one key of the page is no number
    iqs[11, 40, 1] = 255  # a query that is none
    iw[10, 3] = float("nan")
    iw[9] = -iw[9].abs()  # scores below zero
    got = prompt.page_scores(iq, iqs, iw, req, pos, table, caches)
    _scores_near(got, iq, iqs, iw, req, pos, table, caches)
    assert bool(got[12:, 0].isnan().all()) and bool(got[11, 0].isnan()) and bool(got[10, 0].isnan())
    # a key behind a token's position may be no number
    caches.iks[int(table[1, 1]), 0] = 255
    got = prompt.page_scores(iq, iqs, iw, req, pos.clamp_max(PAGE - 1), table, caches)
    assert bool((got[12:, 1:] == -torch.inf).all())


@pytest.mark.parametrize("tokens", [1, 5, 300])
def test_page_scores_of_heads_below_f32_s_range(gpu_device, tokens):
    """A head whose product, or weight times product, is below zero adds nothing however far below it is:
    minus infinity, too. A sum of the other heads' in f32: 16 FMAs a lane, a sum of two tiles' and one of
    two lanes', 18 roundings of what is not cut off."""
    req, pos, table, pages = _requests(gpu_device, [(140, tokens)])
    iq, iqs, iw, caches = _index(gpu_device, tokens, pages)
    caches.ikv[int(table[0, 1])] = 0xAA  # a page's keys: every dim -1 x 2^127
    caches.iks[int(table[0, 1])] = 254
    iqs[:] = 2  # the heads beside: 2^-125 of their codes
    iqs[:, 3] = iqs[:, 40] = 254  # 128 x -2^254
    iqs[:, 8:11] = 120  # 128 x -2^120 = -2^127, which a weight of 16 takes out of the range
    iq[:, [3, 40, 8, 9, 10]] = 0x22
    iw[:, 8], iw[:, 9], iw[:, 10] = 16.0, -16.0, 1.5
    got = prompt.page_scores(iq, iqs, iw, req, pos, table, caches).cpu().double()
    keep = sorted({0, tokens // 2, tokens - 1})
    cpu = (v[keep].cpu() for v in (iq, iqs, iw, req, pos))
    want, _ = ref.page_scores(*cpu, table.cpu(), caches.ikv.cpu(), caches.iks.cpu(), table.shape[1])
    for n, at in enumerate(keep):
        dot = -ref.oatt.index_query(iq[at].cpu(), iqs[at].cpu()).double().sum(-1) * 2.0**127
        mag = float((iw[at].cpu().double().abs() * dot.clamp_min(0)).sum())
        assert abs(float(got[at, 1] - want[n, 1])) <= 18 * 2.0**-24 * mag and mag > 0
    # upwards: infinite, of the weight's sign; and with both a NaN
    caches.ikv[int(table[0, 1])] = 0x22
    for weights, what in (((1.0, 2.0), torch.inf), ((-1.0, -2.0), -torch.inf), ((1.0, -2.0), torch.nan)):
        iw[:, 3], iw[:, 40] = weights
        iw[:, 8:11] = 1e-3
        got = prompt.page_scores(iq, iqs, iw, req, pos, table, caches)[:, 1].cpu()
        assert torch.equal(got, torch.full((tokens,), what)) or (what != what and bool(got.isnan().all()))


def test_page_scores_are_the_decode_launch_s(gpu_device):
    """The largest in each page of the index scores that the attention launch computes: the same
    products, 64 heads' sums in another order at most."""
    step, caches = workloads.attn_case([3000, 2500], gpu_device, seed=9, max_ctx=4096)
    rt = AttnRuntime(2, 4096, device=gpu_device)
    _, dbg = rt.forward(step, caches, debug=True)
    torch.cuda.synchronize()
    rt.check_errors()
    pos = step.seq_lens - 1
    req = torch.arange(2, dtype=torch.int32, device=gpu_device)
    got = prompt.page_scores(step.iq, step.iqs, step.iw, req, pos, step.page_table, caches)
    live = torch.arange(4096, device=gpu_device) <= pos[:, None]
    want = torch.where(live, dbg["scores"], -torch.inf).view(2, -1, PAGE).amax(-1)
    _, mag = ref.page_scores(step.iq.cpu(), step.iqs.cpu(), step.iw.cpu(), req.cpu(), pos.cpu(), step.page_table.cpu(),
                             caches.ikv.cpu(), caches.iks.cpu(), got.shape[1])
    fine = want.isfinite()
    assert torch.equal(got.isfinite(), fine)
    assert bool(((got - want).abs()[fine].cpu() <= (12 + 18) * 2.0**-24 * mag[fine.cpu()]).all())
    rt.close()


# ---------------------------------------------------------------------- select
@pytest.mark.parametrize("columns", [1, 2, 64, 65, 128, 129, 256, 300, 512, 513, 2048, 2049, 8192])
def test_select_pages(gpu_device, columns):
    g = torch.Generator().manual_seed(columns)
    t = 13
    pos = torch.randint(0, columns * PAGE + 100, (t,), generator=g).int()
    pos[0], pos[1], pos[2], pos[3] = 0, 63, columns * PAGE - 1, -1
    for values in ("spread", "ties", "odd"):
        scores = torch.randn(t, columns + 3, generator=g)
        if values == "ties":
            scores = (3 * scores).round() / 4
        if values == "odd":
            pick = torch.randint(0, 9, scores.shape, generator=g)
            for i, v in enumerate((torch.inf, -torch.inf, torch.nan, -torch.nan, 0.0, -0.0, 1e-45)):
                scores[pick == i] = v
        for picks, first, last in ((1, 0, 1), (1, 0, 0), (7, 2, 3), (32, 0, 1), (64, 64, 0), (min(columns, 1000), 1, 0), (columns, 0, 1)):
            if first + last > picks:
                continue
            got = prompt.select_pages(scores.to(gpu_device)[:, 3:], pos.to(gpu_device), picks, first, last)
            assert torch.equal(got.cpu(), ref.select_pages(scores[:, 3:], pos, picks, first, last)), (values, picks, first, last)


@pytest.mark.parametrize("columns", [2, 40, 64, 100, 128, 300, 1000, 2048, 2049, 8192])
def test_select_pages_scores_of_any_bits(gpu_device, columns):
    """NaNs of the largest and the smallest bits of either sign among scores, and rows of them alone:
    where the search begins, at either end of 32 bits."""
    g = torch.Generator().manual_seed(columns)
    t = 9
    pos = torch.randint(0, columns * PAGE, (t,), generator=g).int()
    pos[0], pos[1] = columns * PAGE - 1, columns * PAGE // 2
    scores = torch.randn(t, columns, generator=g)
    bits = scores.view(torch.int32)
    odd = torch.tensor([0x7FFFFFFF, 0x7F800001, -1, -0x7FFFFF, 0x7FFFFFFE, -2, 0x7F7FFFFF, -0x800001], dtype=torch.int32)
    place = torch.rand(t, columns, generator=g)
    bits[2:] = torch.where(place < 0.5, odd[torch.randint(0, len(odd), (t, columns), generator=g)], bits)[2:]
    bits[0, columns // 3] = bits[1, 0] = 0x7FFFFFFF  # one alone
    bits[2], bits[3] = 0x7FFFFFFF, -1  # a row of each
    for picks, first, last in ((1, 0, 0), (2, 0, 1), (31, 0, 1), (64, 0, 1), (70, 1, 2), (columns, 0, 0), (max(columns - 1, 1), 0, 1)):
        got = prompt.select_pages(scores.to(gpu_device), pos.to(gpu_device), picks, first, last)
        assert torch.equal(got.cpu(), ref.select_pages(scores, pos, picks, first, last)), (picks, first, last)


def test_a_table_of_no_pages_from_its_scores_to_its_attention(gpu_device):
    req, pos, table, pages = _requests(gpu_device, [(70, 5)])
    iq, iqs, iw, caches = _index(gpu_device, 5, pages)
    table = table[:, :0].contiguous()
    scores = prompt.page_scores(iq, iqs, iw, req, pos, table, caches)
    ids = prompt.select_pages(scores, pos)
    assert scores.shape == (5, 0) and torch.equal(ids.cpu(), torch.full((5, 32), -1, dtype=torch.int32))
    assert bool((prompt.attention(_q(gpu_device, 5, 32), req, pos, ids, table, _pool(gpu_device, pages, False)) == 0).all())


def test_select_pages_default_takes_all_of_2048_keys(gpu_device):
    pos = torch.tensor([0, 64, 2047, 2048], dtype=torch.int32, device=gpu_device)
    got = prompt.select_pages(torch.randn(4, 40, device=gpu_device), pos).cpu()
    for n, seen in enumerate((1, 2, 32)):
        assert got[n].tolist() == list(range(seen)) + [-1] * (32 - seen)
    assert int(got[3, -1]) == 32 and len(set(got[3].tolist())) == 32


# ------------------------------------------------------------------- attention
def _pool(dev, pages, raw, seed=3):
    g = torch.Generator(device=dev).manual_seed(seed)
    kv = torch.randn(pages * PAGE, 576, generator=g, device=dev).to(torch.float8_e4m3fn).view(torch.uint8)
    scale = None if raw else torch.rand(pages * PAGE, generator=g, device=dev) * 1.5 + 0.5
    return AttnCaches(ikv=None, iks=None, kv=kv, kv_scale=scale)


def _q(dev, tokens, heads, seed=4):
    return torch.randn(tokens, heads, 576, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(torch.bfloat16)


def _lists(dev, pos, columns, picks, seed=6):
    g = torch.Generator(device=dev).manual_seed(seed)
    scores = torch.randn(len(pos), columns, generator=g, device=dev)
    return prompt.select_pages(scores, pos, picks)


def _attend_near(q, req, pos, pages, table, c, scale=SOFTMAX_SCALE, **kw):
    got = prompt.attention(q, req, pos, pages, table, c, softmax_scale=scale, **kw)
    want, mag, top = ref.attention(q.cpu(), req.cpu(), pos.cpu(), pages.cpu(), table.cpu(), c.kv.cpu(),
                                   None if c.kv_scale is None else c.kv_scale.cpu(), scale)
    _near(got, want, mag, top, pages.shape[1] * PAGE)
    return got


@pytest.mark.parametrize("raw", [False, True], ids=["scaled", "raw"])
@pytest.mark.parametrize("heads", [1, 8, 16, 17, 32, 33, 64, 128])
def test_attention_heads(gpu_device, heads, raw):
    req, pos, table, pages = _requests(gpu_device, [(300, 3), (0, 2)], pads=1)
    _attend_near(_q(gpu_device, 6, heads), req, pos, _lists(gpu_device, pos, table.shape[1], 4), table, _pool(gpu_device, pages, raw))


@pytest.mark.parametrize("spans,pads,picks", [
    ([(0, 1)], 0, 1), ([(0, 1)], 0, 32), ([(5000, 1)], 0, 32), ([(63, 2)], 0, 2), ([(0, 70)], 0, 32), ([(1000, 9)], 0, 1),
    ([(900, 20), (0, 31), (64, 1), (4000, 3)], 4, 7), ([(5000, 2)], 0, 70), ([(4300, 600)], 0, 3), ([(8500, 1)], 0, 131),
])  # fmt: skip
def test_attention(gpu_device, spans, pads, picks):
    req, pos, table, pages = _requests(gpu_device, spans, pads, spare=1)
    _attend_near(_q(gpu_device, len(pos), 32), req, pos, _lists(gpu_device, pos, table.shape[1], picks), table,
                 _pool(gpu_device, pages, False))


def test_attention_to_each_key_once(gpu_device):
    """A query of zeros weighs every key alike, and a key has a one in its own dim: a dim of the
    output says how often that key was seen, exactly but for the division and its rounding."""
    req, pos, table, pages = _requests(gpu_device, [(440, 40)])
    kv = torch.zeros(pages * PAGE, 576, device=gpu_device)
    for c in range(table.shape[1]):
        for j in range(PAGE):
            kv[int(table[0, c]) * PAGE + j, (c * PAGE + j) % 512] = 1.0
    caches = AttnCaches(None, None, kv.to(torch.float8_e4m3fn), None)
    q = torch.zeros(40, 32, 576, dtype=torch.bfloat16, device=gpu_device)
    for lists in ([7, 6, 5, 4, 3, 2, 1, 0], [0, 3, 7], [5, -1, 2], [4, 4, 1, 4]):  # in any order, with gaps, twice
        ids = torch.tensor([lists] * 40, dtype=torch.int32, device=gpu_device)
        got = prompt.attention(q, req, pos, ids, table, caches).cpu().double()
        for n, p in enumerate(range(440, 480)):
            count = torch.zeros(512, dtype=torch.float64)
            for c in lists:
                for j in range(PAGE):
                    if c >= 0 and c * PAGE + j <= p:
                        count[c * PAGE + j] += 1
            want = count / count.sum()
            assert bool(((got[n] - want).abs() <= (2.0**-8 + 2.0**-22) * want).all())


def test_attention_rows_that_see_nothing_are_zeros(gpu_device):
    req, pos, table, pages = _requests(gpu_device, [(100, 8)])
    c = _pool(gpu_device, pages, False)
    req[0], req[1], pos[2] = -1, 1, -1
    ids = torch.tensor([[0, 1]] * 8, dtype=torch.int32, device=gpu_device)
    ids[3], ids[4], ids[5] = -1, 99, 1 << 30  # no page, none of the table's, none by far
    table[0, 0] = pages  # not of the pool
    ids[6] = 0
    pos[7] = 63  # page 1 lies behind it
    for rows in (slice(0, 8), slice(3, 4)):  # whole and split
        got = prompt.attention(_q(gpu_device, 8, 32)[rows], req[rows], pos[rows], ids[rows], table, c)
        assert bool((got == 0).all())


@pytest.mark.parametrize("tokens", [1, 40, 700])
def test_attention_does_not_look_at_what_is_not_seen(gpu_device, tokens):
    """Keys behind a token's position and pages that it does not list may hold anything."""
    req, pos, table, pages = _requests(gpu_device, [(130, tokens)], spare=1)
    c = _pool(gpu_device, pages, False)
    ids = torch.tensor([[0, 2]], dtype=torch.int32, device=gpu_device).repeat(tokens, 1)
    q = _q(gpu_device, tokens, 20)
    want = prompt.attention(q, req, pos, ids, table, c)
    for n in range(min(tokens, 3)):
        p = int(pos[n])
        d = AttnCaches(None, None, c.kv.clone(), c.kv_scale.clone())
        behind = int(table[0, 2]) * PAGE + p % PAGE + 1 if p < 191 else None
        lost = [s for s in range(int(table[0, 1]) * PAGE, int(table[0, 1]) * PAGE + PAGE)]
        if behind is not None:
            lost += list(range(behind, int(table[0, 2]) * PAGE + PAGE))
        d.kv[lost] = 0x7F
        d.kv_scale[lost] = float("nan")
        got = prompt.attention(q, req, pos, ids, table, d)
        assert torch.equal(got[:n + 1], want[:n + 1])
        d.kv_scale[lost] = float("inf")
        assert torch.equal(prompt.attention(q, req, pos, ids, table, d)[:n + 1], want[:n + 1])


@pytest.mark.parametrize("tokens", [2, 600])
def test_attention_values_that_are_not_finite_stay_visible(gpu_device, tokens):
    req, pos, table, pages = _requests(gpu_device, [(200, tokens)])
    c = _pool(gpu_device, pages, False)
    ids = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=gpu_device).repeat(tokens, 1)
    q = _q(gpu_device, tokens, 32)
    want = prompt.attention(q, req, pos, ids, table, c)
    q[0, 5, 100] = float("nan")
    q[1, 9, 575] = float("inf")
    got = prompt.attention(q, req, pos, ids, table, c)
    assert bool(got[0, 5].isnan().all()) and bool(got[1, 9].isnan().all())
    keep = torch.ones(tokens, 32, dtype=torch.bool, device=gpu_device)
    keep[0, 5] = keep[1, 9] = False
    assert torch.equal(got[keep], want[keep])
    c.kv[int(table[0, 1]) * PAGE + 3, 17] = 0xFF
    assert bool(prompt.attention(q, req, pos, ids, table, c).isnan().all())


@pytest.mark.parametrize("tokens,picks", [(1, 12), (600, 12)])
def test_attention_logits_that_grow_and_fall(gpu_device, tokens, picks):
    """Each page's logits far above, or below, those of the pages before it."""
    req, pos, table, pages = _requests(gpu_device, [(picks * PAGE - 1, tokens)])
    c = _pool(gpu_device, pages, False)
    for up in (True, False):
        for i in range(picks):
            c.kv_scale[int(table[0, i]) * PAGE:int(table[0, i]) * PAGE + PAGE] = 2.0 ** (i if up else picks - i) / 16
        ids = torch.arange(picks, dtype=torch.int32, device=gpu_device).repeat(tokens, 1)
        keep = min(tokens, 4)
        q = _q(gpu_device, tokens, 32)
        got = prompt.attention(q, req, pos, ids, table, c)
        want, mag, top = ref.attention(q[:keep].cpu(), req[:keep].cpu(), pos[:keep].cpu(), ids[:keep].cpu(), table.cpu(),
                                       c.kv.cpu(), c.kv_scale.cpu(), SOFTMAX_SCALE)
        _near(got[:keep], want, mag, top, picks * PAGE)


def test_attention_scales(gpu_device):
    req, pos, table, pages = _requests(gpu_device, [(150, 5)])
    c, ids = _pool(gpu_device, pages, True), torch.tensor([[0, 1, 2]] * 5, dtype=torch.int32, device=gpu_device)
    for scale in (0.0, 1e-3, 0.5, -0.1):
        _attend_near(_q(gpu_device, 5, 32), req, pos, ids, table, c, scale=scale)


def test_attention_split_or_whole(gpu_device):
    """A token alone has its pages shared out over workgroups, in a wide call it has not: the
    same but for f32's order of sums, which moves an output by a rounding of bf16 at most."""
    req, pos, table, pages = _requests(gpu_device, [(2100, 600)])
    c = _pool(gpu_device, pages, False)
    ids, q = _lists(gpu_device, pos, table.shape[1], 32), _q(gpu_device, 600, 32)
    whole = prompt.attention(q, req, pos, ids, table, c)
    for n in (0, 333, 599):
        one = prompt.attention(q[n:n + 1], req[n:n + 1], pos[n:n + 1], ids[n:n + 1], table, c)
        assert float((one - whole[n:n + 1]).float().norm() / one.float().norm()) <= 2.0**-7
    assert torch.equal(prompt.attention(q, req, pos, ids, table, c), whole)  # the same bits from call to call


def test_attention_pages_far_in_the_pool(gpu_device):
    """Byte offsets past 32 bits."""
    torch.cuda.empty_cache()
    pages = 240_000  # 8.8 GB
    req, pos, table, _ = _requests(gpu_device, [(200, 3)])
    near = _pool(gpu_device, 6, False)
    table = torch.arange(4, dtype=torch.int32, device=gpu_device)[None]
    ids = torch.tensor([[0, 1, 2, 3]] * 3, dtype=torch.int32, device=gpu_device)
    q = _q(gpu_device, 3, 32)
    want = prompt.attention(q, req, pos, ids, table, near)
    kv = torch.empty(pages * PAGE, 576, dtype=torch.uint8, device=gpu_device)
    kv_scale = torch.empty(pages * PAGE, device=gpu_device)
    kv[-6 * PAGE:], kv_scale[-6 * PAGE:] = near.kv, near.kv_scale
    far = AttnCaches(None, None, kv, kv_scale)
    assert torch.equal(prompt.attention(q, req, pos, ids, table + pages - 6, far), want)
    mask = torch.tensor([0, 1, 5], device=gpu_device)
    tree = (torch.tensor([0, 3], dtype=torch.int32, device=gpu_device), torch.tensor([200], dtype=torch.int32, device=gpu_device), mask)
    assert torch.equal(prompt.tree_attention(q, *tree, table + pages - 6, far), prompt.tree_attention(q, *tree, table, near))
    del kv, kv_scale, far
    torch.cuda.empty_cache()


def test_attention_out_and_no_rows(gpu_device):
    req, pos, table, pages = _requests(gpu_device, [(100, 4)])
    c, q = _pool(gpu_device, pages, False), _q(gpu_device, 4, 32)
    ids = torch.tensor([[0, 1]] * 4, dtype=torch.int32, device=gpu_device)
    out = torch.full((6, 32, 512), 3.0, dtype=torch.bfloat16, device=gpu_device)
    got = prompt.attention(q, req, pos, ids, table, c, out=out[1:5])
    assert got.data_ptr() == out[1:5].data_ptr() and torch.equal(got, prompt.attention(q, req, pos, ids, table, c))
    assert bool((out[0] == 3).all()) and bool((out[5] == 3).all())
    none = torch.empty(0, 32, 576, dtype=torch.bfloat16, device=gpu_device)
    assert prompt.attention(none, req[:0], pos[:0], ids[:0], table, c).shape == (0, 32, 512)
    assert bool((prompt.attention(q, req, pos, ids[:, :0].contiguous(), table, c) == 0).all())  # no pages at all
    assert bool((prompt.attention(q, req, pos, ids, table[:, :0].contiguous(), c) == 0).all())  # no tables
    buf = torch.zeros(4 * 32 * 1100, dtype=torch.bfloat16, device=gpu_device)
    with pytest.raises(ValueError, match="shares memory with q"):
        prompt.attention(buf[:4 * 32 * 576].view(4, 32, 576), req, pos, ids, table, c,
                         out=buf[4 * 32 * 576 - 8:4 * 32 * 1088 - 8].view(4, 32, 512))
    with pytest.raises(ValueError, match="shares memory with kv"):
        prompt.attention(q, req, pos, ids, table, AttnCaches(None, None, buf.view(torch.uint8)[:64 * 576].view(64, 576), None),
                         out=buf[:4 * 32 * 512].view(4, 32, 512))


@pytest.mark.parametrize("tokens,heads", [(8, 32), (9, 32), (51, 32), (52, 32), (12, 128), (13, 128), (31, 16), (32, 16), (33, 16), (256, 16), (257, 16), (512, 4), (513, 4), (65, 128)])
def test_attention_shared_out_or_not(gpu_device, tokens, heads):
    """Around the token counts at which pages are shared out, or joined, in another way."""
    req, pos, table, pages = _requests(gpu_device, [(400, tokens)])
    _attend_near(_q(gpu_device, tokens, heads), req, pos, _lists(gpu_device, pos, table.shape[1], 5), table, _pool(gpu_device, pages, False))


@pytest.mark.parametrize("tokens", [3, 600])
def test_attention_queries_of_unlike_elements(gpu_device, tokens):
    """Heads whose elements differ by factors of up to 2^20, and heads far apart in size."""
    req, pos, table, pages = _requests(gpu_device, [(200, tokens)])
    ids = torch.tensor([[0, 1, 2, 3]] * tokens, dtype=torch.int32, device=gpu_device)
    q = _q(gpu_device, tokens, 32).float()
    q[:, :8] *= torch.logspace(-6, 0, 576, device=gpu_device)
    q[:, 8:16] *= torch.logspace(0, -6, 576, device=gpu_device)
    q[:, 16, 3], q[:, 17, 570] = 300.0, -300.0
    q[:, 18:24] *= torch.tensor([1e-30, 1e-10, 1e-3, 3.0, 1e-38, 0.0], device=gpu_device)[:, None]
    q[:, 24] = 0.0
    q[:, 24, 511], q[:, 25, :] = 100.0, 448.0 / 256
    keep = min(tokens, 5)
    q, c = q.to(torch.bfloat16), _pool(gpu_device, pages, True)
    got = prompt.attention(q, req, pos, ids, table, c)[:keep]
    for h in range(32):  # (each head with its own bound)
        want, mag, top = ref.attention(q[:keep, h:h + 1].cpu(), req[:keep].cpu(), pos[:keep].cpu(), ids[:keep].cpu(), table.cpu(),
                                       c.kv.cpu(), None, SOFTMAX_SCALE)
        _near(got[:, h:h + 1], want, mag, top, 4 * PAGE, norm=False)


@pytest.mark.parametrize("power,sign,scale", [(10, 1, 0.07), (24, -1, 0.07), (31, 1, 0.07), (40, -1, 0.07), (70, 1, 1.3), (118, 1, 0.6), (121, -1, 0.6)])
@pytest.mark.parametrize("tokens", [1, 600])
def test_attention_logits_of_any_size(gpu_device, tokens, power, sign, scale):
    """Logits of thousands to 2.6e38, of either sign: one key's is the largest by far more than an
    exponential's range, so its row is the output, exactly."""
    req, pos, table, pages = _requests(gpu_device, [(640, tokens)])
    c, best = _pool(gpu_device, pages, False), [3, 200, 500, 639]
    pe = torch.tensor([1.0, 1.25, 1.5] if sign > 0 else [2.0, 2.5, 3.0], device=gpu_device)
    rows = c.kv.view(torch.float8_e4m3fn)
    rows[:, 512:] = pe[torch.arange(len(rows), device=gpu_device) % 3, None].to(torch.float8_e4m3fn)
    c.kv_scale.fill_(1.0)
    q = torch.zeros(tokens, 32, 576, dtype=torch.bfloat16, device=gpu_device)
    q[:, :, 512:] = sign * 2.0**power
    ids = torch.arange(10, dtype=torch.int32, device=gpu_device).repeat(tokens, 1)
    starts, prefix = (torch.tensor(v, dtype=torch.int32, device=gpu_device) for v in ([0, tokens], [640]))
    mask = torch.zeros(tokens, dtype=torch.int64, device=gpu_device)
    for p in best:
        d = AttnCaches(None, None, c.kv.clone(), c.kv_scale)
        slot = int(table[0, p // PAGE]) * PAGE + p % PAGE
        d.kv.view(torch.float8_e4m3fn)[slot, 512:] = torch.tensor(1.75, device=gpu_device).to(torch.float8_e4m3fn)
        want = d.kv.view(torch.float8_e4m3fn)[slot, :512].to(torch.bfloat16).expand(tokens, 32, 512)
        assert torch.equal(prompt.attention(q, req, pos, ids, table, d, softmax_scale=scale), want), p
        assert torch.equal(prompt.tree_attention(q, starts, prefix, mask, table, d, softmax_scale=scale), want), p


# ------------------------------------------------------------------------ tree
def _tree(dev, trees, seed=2, spare=0):
    """(starts, prefix, mask, table, pages) of trees (prefix, nodes): a node hangs from one of
    the three before it."""
    _, _, table, pages = _requests(dev, trees, spare=spare, seed=seed)
    g = torch.Generator().manual_seed(seed)
    mask = []
    for _, n in trees:
        seen = []
        for i in range(n):
            up = int(torch.randint(1, 4, (1,), generator=g))
            m = (seen[i - up] if i >= up else 0) | (1 << i if i < 64 else 0)
            seen.append(m)
            mask.append(m - (1 << 64) if m >> 63 else m)
    starts = torch.tensor([0] + [n for _, n in trees]).cumsum(0).int()
    return (starts.to(dev), torch.tensor([p for p, _ in trees]).int().to(dev), torch.tensor(mask, dtype=torch.int64).to(dev),
            table, pages)


def _tree_near(q, starts, prefix, mask, table, c, scale=SOFTMAX_SCALE):
    got = prompt.tree_attention(q, starts, prefix, mask, table, c, softmax_scale=scale)
    want, mag, top = ref.tree_attention(q.cpu(), starts.cpu(), prefix.cpu(), mask.cpu(), table.cpu(), c.kv.cpu(),
                                        None if c.kv_scale is None else c.kv_scale.cpu(), scale)
    _near(got, want, mag, top, table.shape[1] * PAGE)
    return got


@pytest.mark.parametrize("raw", [False, True], ids=["scaled", "raw"])
@pytest.mark.parametrize("trees", [[(0, 1)], [(1, 1)], [(63, 1)], [(64, 3)], [(60, 9)], [(0, 64)], [(1, 64)], [(130, 64)], [(700, 5)],
                                   [(200, 7), (0, 3), (64, 1), (900, 33)], [(33, 2)] * 70, [(2000, 2), (0, 0), (5, 0), (128, 4)],
                                   [(100, 90)]])
def test_tree_attention(gpu_device, trees, raw):
    starts, prefix, mask, table, pages = _tree(gpu_device, trees)
    _tree_near(_q(gpu_device, len(mask), 32), starts, prefix, mask, table, _pool(gpu_device, pages, raw))


@pytest.mark.parametrize("heads", [1, 8, 16, 17, 48, 64, 128])
def test_tree_attention_heads(gpu_device, heads):
    starts, prefix, mask, table, pages = _tree(gpu_device, [(150, 5), (64, 9)])
    _tree_near(_q(gpu_device, 14, heads), starts, prefix, mask, table, _pool(gpu_device, pages, False))


def test_tree_attention_wide(gpu_device):
    """More nodes than are split."""
    starts, prefix, mask, table, pages = _tree(gpu_device, [(70 + i, 64 - i) for i in range(12)])
    _tree_near(_q(gpu_device, len(mask), 16), starts, prefix, mask, table, _pool(gpu_device, pages, False))


@pytest.mark.parametrize("trees,heads", [
    ([(100 + i, 32) for i in range(8)], 16), ([(100 + i, 32) for i in range(8)] + [(500, 1)], 16),  # 256 nodes, 257
    ([(90, 30), (300, 34)], 128), ([(90, 30), (300, 35)], 128),  # 256 nodes' tiles of heads, 260
    ([(30 * PAGE, 8)], 32), ([(31 * PAGE, 8)], 32), ([(7, 3)], 100), ([(300, 9)], 33),  # 512 nodes' pages and tiles, 528
    ([(255 * PAGE, 8)], 16), ([(255 * PAGE + 1, 8)], 16),  # 2048 nodes' pages, 2056
    ([(50 * PAGE, 16)], 16), ([(50 * PAGE, 17)], 16),  # 256 heads, 272
    ([(9, 64), (700, 64)], 16), ([(9, 64), (700, 65)], 16),  # 128 nodes, 129
    ([(3000, 2)] + [(10, 30)] * 20, 8), ([(10, 64)] * 5 + [(2000, 5), (0, 0), (64, 63)], 64),  # long nodes among 602, 388 x 2 tiles
    ([(0, 64)] * 15 + [(1200, 64)], 4), ([(0, 64)] * 15 + [(1200, 65)], 4),  # 1024 nodes, 1025
    ([(30, 1)] * 255 + [(1500, 1)], 4), ([(30, 1)] * 256 + [(1500, 1)], 4), ([(30, 2)] * 200 + [(0, 0)] * 55 + [(2500, 1)], 4),  # requests: 256, 257
    ([(140_000, 1)], 4), ([(40_000, 1)], 33), ([(5, 1)] * 64 + [(3000, 2)] * 3 + [(0, 0)] * 70 + [(64, 1)], 16),
])  # fmt: skip
def test_tree_attention_shared_out_or_not(gpu_device, trees, heads):
    """Around the sizes at which pages are shared out, or joined, in another way."""
    starts, prefix, mask, table, pages = _tree(gpu_device, trees)
    _tree_near(_q(gpu_device, len(mask), heads), starts, prefix, mask, table, _pool(gpu_device, pages, True))


@pytest.mark.parametrize("trees,heads", [
    ([(1, 1)], 32), ([(4000, 1)], 32), ([(4000, 1)], 16), ([(4027, 5)], 32), ([(19990, 10)], 32), ([(2500, 3), (0, 2), (900, 33)], 32),
    ([(12000, 1)], 32), ([(6000, 2)], 32), ([(3000, 1), (2400, 2)], 64), ([(16383, 1)], 16), ([(16383, 1)], 4),
    ([(1275, 5), (640, 64)], 64), ([(60, 4)], 32), ([(64, 1)], 128), ([(8000, 2), (7990, 10)], 17), ([(300, 60)] * 20, 32),
])  # fmt: skip
def test_tree_attention_does_not_hang_on_the_table_s_width(gpu_device, trees, heads):
    """The same bits from a table that just holds the keys as from one with room for more."""
    starts, prefix, mask, table, pages = _tree(gpu_device, trees)
    c, q = _pool(gpu_device, pages, False), _q(gpu_device, len(mask), heads)
    want = _tree_near(q, starts, prefix, mask, table, c) if heads * len(mask) < 400 else prompt.tree_attention(q, starts, prefix, mask, table, c)
    for more in (1, 2, 700):
        wide = torch.cat([table, torch.full((len(table), more), -1, dtype=torch.int32, device=gpu_device)], 1)
        assert torch.equal(prompt.tree_attention(q, starts, prefix, mask, wide, c), want), more


def test_tree_attention_sees_each_key_once(gpu_device):
    starts, prefix, mask, table, pages = _tree(gpu_device, [(100, 60), (37, 64)])
    mask[3], mask[70], mask[71] = 0, -1, -(1 << 63)  # the prefix alone; every drafted key; the last alone
    kv = torch.zeros(pages * PAGE, 576, device=gpu_device)
    for r in range(2):
        for p in range(table.shape[1] * PAGE):
            if int(table[r, p // PAGE]) >= 0:
                kv[int(table[r, p // PAGE]) * PAGE + p % PAGE, p] = 1.0
    got = prompt.tree_attention(torch.zeros(124, 32, 576, dtype=torch.bfloat16, device=gpu_device), starts, prefix, mask, table,
                                AttnCaches(None, None, kv.to(torch.float8_e4m3fn), None)).cpu().double()
    for n in range(124):
        r = int(n >= 60)
        seen = torch.zeros(512, dtype=torch.float64)
        seen[:(100, 37)[r]] = 1
        for j in range(64):
            if int(mask[n]) >> j & 1:
                seen[(100, 37)[r] + j] = 1
        want = seen / seen.sum()
        assert bool(((got[n] - want).abs() <= (2.0**-8 + 2.0**-22) * want).all()), n


def test_tree_attention_nodes_that_see_nothing_are_zeros(gpu_device):
    starts, prefix, mask, table, pages = _tree(gpu_device, [(0, 4), (70, 3), (30, 2)])
    c, q = _pool(gpu_device, pages, False), _q(gpu_device, 12, 32)
    mask = torch.cat([mask, torch.full((3,), -1, device=gpu_device)])
    mask[1] = 0  # no prefix, no mask
    prefix[0] = -5  # (no keys: 0)
    table[1, :] = pages  # no page of the pool
    got = prompt.tree_attention(q, starts, prefix, mask, table, c)
    assert bool((got[1] == 0).all()) and bool((got[4:7] == 0).all())
    assert bool((got[9:] == 0).all())  # behind the last tree
    assert bool((got[[0, 2, 3, 7, 8]] != 0).any(-1).all())
    starts = starts + 2  # (the last tree ends behind the nodes)
    assert bool((prompt.tree_attention(q[:9], starts, prefix, mask[:9], table, c)[:2] == 0).all())  # before the first
    none = torch.empty(0, 32, 576, dtype=torch.bfloat16, device=gpu_device)
    assert prompt.tree_attention(none, starts, prefix, mask[:0], table, c).shape == (0, 32, 512)
    assert bool((prompt.tree_attention(q, starts[:1], prefix[:0], mask, table[:0], c) == 0).all())  # no requests


def test_tree_attention_does_not_look_at_siblings(gpu_device):
    starts, prefix, mask, table, pages = _tree(gpu_device, [(90, 40), (64, 20)])
    c, q = _pool(gpu_device, pages, False), _q(gpu_device, 60, 32)
    want = prompt.tree_attention(q, starts, prefix, mask, table, c)
    for n in (0, 7, 39, 40, 55):
        r = int(n >= 40)
        d = AttnCaches(None, None, c.kv.clone(), c.kv_scale.clone())
        lost = [p for p in range(int(prefix[r]), table.shape[1] * PAGE) if int(table[r, p // PAGE]) >= 0
                and not (p - int(prefix[r]) < 64 and int(mask[n]) >> (p - int(prefix[r])) & 1)]
        slots = [int(table[r, p // PAGE]) * PAGE + p % PAGE for p in lost]
        d.kv[slots], d.kv_scale[slots] = 0x7F, float("nan")
        assert torch.equal(prompt.tree_attention(q, starts, prefix, mask, table, d)[n], want[n])


def test_tree_attention_of_a_chain_is_causal_attention(gpu_device):
    """A chain of drafted tokens is a prompt's tail that reads every page."""
    req, pos, table, pages = _requests(gpu_device, [(250, 30)])
    c, q = _pool(gpu_device, pages, False), _q(gpu_device, 30, 32)
    ids = torch.arange(table.shape[1], dtype=torch.int32, device=gpu_device).repeat(30, 1)
    chain = torch.tensor([(1 << i + 1) - 1 for i in range(30)], device=gpu_device)
    starts, prefix = torch.tensor([0, 30], dtype=torch.int32, device=gpu_device), torch.tensor([250], dtype=torch.int32, device=gpu_device)
    a = prompt.attention(q, req, pos, ids, table, c).float()
    b = _tree_near(q, starts, prefix, chain, table, c).float()
    assert float((a - b).norm() / a.norm()) <= 2.0**-7


# -------------------------------------------------------------------- together
def _appended(dev, spans, seed=11):
    g = torch.Generator(device=dev).manual_seed(seed)
    req, pos, table, pages = _requests(dev, spans)
    u8 = dict(generator=g, device=dev, dtype=torch.uint8)
    caches = AttnCaches(ikv=torch.randint(0, 256, (pages, 4, 64, 16), **u8), iks=torch.full((pages, 4, 64), 255, dtype=torch.uint8, device=dev),
                        kv=torch.full((pages * 64, 576), 0x7F, dtype=torch.uint8, device=dev),
                        kv_scale=torch.full((pages * 64,), float("nan"), device=dev))
    w = dict(g_kv=(1 + 0.1 * torch.randn(512, generator=g, device=dev)).to(torch.bfloat16),
             g_ik=1 + 0.1 * torch.randn(128, generator=g, device=dev), b_ik=0.1 * torch.randn(128, generator=g, device=dev))
    cos, sin = workloads.rope_tables(table.shape[1] * PAGE, dev)
    return g, req, pos, table, caches, w, cos, sin


def test_a_prompt_from_its_projections_to_its_attention(gpu_device):
    """Appended keys, scored, selected and attended to; what no token wrote is no number."""
    dev = gpu_device
    g, req, pos, table, caches, w, cos, sin = _appended(dev, [(0, 450), (0, 90)])
    t = len(pos)
    kv_a, ik = torch.randn(t, 576, generator=g, device=dev), torch.randn(t, 128, generator=g, device=dev)
    prompt.append(kv_a, ik, req, pos, table, caches, **w, rope_cos=cos, rope_sin=sin)
    x = torch.randn(t, 8192, generator=g, device=dev).to(torch.bfloat16)
    iw = (0.1 * torch.randn(t, 64, generator=g, device=dev)).to(torch.bfloat16)
    q = _q(dev, t, 32)

    def run():
        iq, iqs = prompt.index_query(x, pos, cos, sin)
        scores = prompt.page_scores(iq, iqs, iw, req, pos, table, caches)
        pages = prompt.select_pages(scores, pos, 4)
        return iq, iqs, scores, pages, prompt.attention(q, req, pos, pages, table, caches)

    iq, iqs, scores, pages, out = run()
    keep = [0, 63, 64, 200, 300, 449, 450, 539]
    _scores_near(scores[keep], iq[keep], iqs[keep], iw[keep], req[keep], pos[keep], table, caches)
    assert torch.equal(pages.cpu(), ref.select_pages(scores.cpu(), pos.cpu(), 4, 0, 1))
    want, mag, top = ref.attention(q[keep].cpu(), req[keep].cpu(), pos[keep].cpu(), pages[keep].cpu(), table.cpu(),
                                   caches.kv.cpu(), caches.kv_scale.cpu(), SOFTMAX_SCALE)
    _near(out[keep], want, mag, top, 4 * PAGE)
    # on another stream, and captured: the same bits at every replay
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        again = run()
    other.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, (iq, iqs, scores, pages, out)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for i in range(3):
        q.copy_(_q(dev, t, 32, seed=20 + i))
        x.copy_(torch.randn(t, 8192, generator=g, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        eager = run()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))


def test_a_short_prompt_s_attention_is_the_decode_launch_s(gpu_device):
    """Up to 2048 keys both read every key."""
    lens = [1500, 700]
    step, caches = workloads.attn_case(lens, gpu_device, seed=31, max_ctx=2048)
    rt = AttnRuntime(2, 2048, device=gpu_device)
    want = rt.forward(step, caches)
    torch.cuda.synchronize()
    rt.check_errors()
    pos, req = step.seq_lens - 1, torch.arange(2, dtype=torch.int32, device=gpu_device)
    scores = prompt.page_scores(step.iq, step.iqs, step.iw, req, pos, step.page_table, caches)
    got = prompt.attention(step.q, req, pos, prompt.select_pages(scores, pos), step.page_table, caches)
    # (the launch rounds its parts to bf16 once more)
    assert float((got - want).float().norm() / want.float().norm()) <= 2.0**-7 + 2.0**-8
    rt.close()


def test_a_drafted_tree_from_its_keys_to_its_attention(gpu_device):
    """Siblings share a position and have a slot each; the accepted path is appended again where
    it belongs."""
    dev = gpu_device
    prefix, up = 70, [-1, 0, 0, 1, 1, 2]  # the nodes' parents
    depth = [0, 1, 1, 2, 2, 2]
    g, req, pos, table, caches, w, cos, sin = _appended(dev, [(0, prefix + len(up))])
    kv_a, ik = torch.randn(prefix + 6, 576, generator=g, device=dev), torch.randn(prefix + 6, 128, generator=g, device=dev)
    at = torch.cat([torch.arange(prefix), prefix + torch.tensor(depth)]).int().to(dev)
    prompt.append(kv_a, ik, req, at, table, caches, **w, rope_cos=cos, rope_sin=sin, slot_pos=pos)
    mask = []
    for i, u in enumerate(up):
        mask.append((mask[u] if u >= 0 else 0) | 1 << i)
    mask = torch.tensor(mask, device=dev)
    q = _q(dev, 6, 32)
    starts, pre = torch.tensor([0, 6], dtype=torch.int32, device=dev), torch.tensor([prefix], dtype=torch.int32, device=dev)
    got = _tree_near(q, starts, pre, mask, table, caches)
    # each path by itself, appended as the chain that it is
    for leaf in (3, 4, 5):
        path = [i for i in range(6) if int(mask[leaf]) >> i & 1]
        rows = torch.tensor(list(range(prefix)) + [prefix + i for i in path], device=dev)
        alone = _appended(dev, [(0, prefix + 6)])[4]
        n = len(rows)
        prompt.append(kv_a[rows], ik[rows], req[:n], pos[:n], table, alone, **w, rope_cos=cos, rope_sin=sin)
        for k, node in enumerate(path):
            one = torch.tensor([node], device=dev)
            chain = torch.tensor([(1 << k + 1) - 1], device=dev)
            want = prompt.tree_attention(q[one], torch.tensor([0, 1], dtype=torch.int32, device=dev), pre, chain, table, alone)
            assert float((got[one] - want).float().norm() / want.float().norm()) <= 2.0**-7
    # slots outside the table write nothing
    before = caches.kv.clone()
    prompt.append(kv_a[:2], ik[:2], req[:2], pos[:2], table, caches, **w, rope_cos=cos, rope_sin=sin,
                  slot_pos=torch.tensor([-1, table.shape[1] * PAGE], dtype=torch.int32, device=dev))
    assert torch.equal(caches.kv, before)


def test_two_captured_graphs_and_an_eager_call_keep_apart(gpu_device):
    """Calls whose pages are shared out hold scratch: each its own."""
    req, pos, table, pages = _requests(gpu_device, [(3000, 3)])
    c = _pool(gpu_device, pages, False)
    ids = _lists(gpu_device, pos, table.shape[1], 32)
    qs = [_q(gpu_device, 3, 32, seed=s) for s in (1, 2, 3)]
    want = [prompt.attention(q, req, pos, ids, table, c) for q in qs]
    graphs, outs = [], []
    for q in qs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(prompt.attention(q, req, pos, ids, table, c))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = prompt.attention(qs[2], req, pos, ids, table, c)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([*outs, eager], want))


def test_captured_trees_follow_their_lengths(gpu_device):
    """Which workgroup takes what is settled on the device: a replay with other trees in the same
    buffers, on two graphs at once."""
    dev = gpu_device
    _, _, table, pages = _requests(dev, [(2000, 40), (3000, 40), (500, 40)])
    c = _pool(dev, pages, False)
    trees = [([0, 20, 21, 40], [1900, 2950, 3]), ([0, 0, 37, 40], [0, 64, 500]), ([0, 1, 2, 30], [2000, 0, 130]), ([0, 13, 26, 40], [700, 3000, 499])]
    held = []
    for i in range(2):
        s = dict(q=_q(dev, 40, 32, seed=i), starts=torch.tensor(trees[0][0], dtype=torch.int32, device=dev),
                 prefix=torch.tensor(trees[0][1], dtype=torch.int32, device=dev), mask=torch.arange(1, 41, device=dev))
        prompt.tree_attention(**s, page_table=table, caches=c)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = prompt.tree_attention(**s, page_table=table, caches=c)
        held.append((s, graph, out, torch.cuda.Stream()))
    for k in range(4):
        for i, (s, _, out, _) in enumerate(held):
            starts, prefix = trees[(k + i) % 4]
            s["starts"].copy_(torch.tensor(starts, dtype=torch.int32))
            s["prefix"].copy_(torch.tensor(prefix, dtype=torch.int32))
            out.fill_(9)
        torch.cuda.synchronize()
        for _, graph, _, stream in held:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for s, _, out, _ in held:
            assert torch.equal(out, prompt.tree_attention(**s, page_table=table, caches=c))
    s = held[0][0]
    _tree_near(s["q"], s["starts"], s["prefix"], s["mask"], table, c)


def test_rows_far_into_their_tensors(gpu_device):
    """Offsets past 2^31 elements: the last rows of wide calls are those of small ones."""
    dev = gpu_device
    torch.cuda.empty_cache()
    tokens, last = 270_000, 5
    req, pos, table, pages = _requests(dev, [(300, last)])
    iq, iqs, iw, caches = _index(dev, last, pages)
    cos, sin = workloads.rope_tables(400, dev)

    def behind(t, fill=0):  # the rows of t behind so many others
        wide = torch.empty(tokens, *t.shape[1:], dtype=t.dtype, device=dev)
        wide[:-last] = fill
        wide[-last:] = t
        return wide

    x = torch.randn(last, 8192, device=dev).to(torch.bfloat16)
    for got, want in zip(prompt.index_query(behind(x), behind(pos, -1), cos, sin), prompt.index_query(x, pos, cos, sin)):
        assert torch.equal(got[-last:], want)
        del got
    want = prompt.page_scores(iq, iqs, iw, req, pos, table, caches, 8192)
    scores = prompt.page_scores(behind(iq), behind(iqs), behind(iw), behind(req, -1), behind(pos), table, caches, 8192)
    assert torch.equal(scores[-last:], want) and bool((scores[-last - 1] == -torch.inf).all())
    picked = prompt.select_pages(scores, behind(pos, -1), 8000)
    assert torch.equal(picked[-last:], prompt.select_pages(want, pos, 8000)) and bool((picked[-last - 1] == -1).all())
    del scores, picked
    torch.cuda.empty_cache()
    tokens = 70_000
    c, q = _pool(dev, pages, False), _q(dev, last, 64)
    ids = torch.tensor([[0, 3, 4]] * last, dtype=torch.int32, device=dev)
    want = prompt.attention(q, req, pos, ids, table, c)
    wide = behind(q)
    got = prompt.attention(wide, behind(req, -1), behind(pos), behind(ids), table, c)
    assert float((got[-last:] - want).float().norm() / want.float().norm()) <= 2.0**-7 and bool((got[-last - 1] == 0).all())
    del got
    tree = (torch.tensor([300], dtype=torch.int32, device=dev), torch.arange(1, last + 1, device=dev))
    want = prompt.tree_attention(q, torch.tensor([0, last], dtype=torch.int32, device=dev), *tree, table, c)
    got = prompt.tree_attention(wide, torch.tensor([tokens - last, tokens], dtype=torch.int32, device=dev), tree[0], behind(tree[1]), table, c)
    assert float((got[-last:] - want).float().norm() / want.float().norm()) <= 2.0**-7 and bool((got[-last - 1] == 0).all())
    del got, wide
    torch.cuda.empty_cache()
