"""GPU: the paged-cache operators against plain 64-bit forms.

Error bounds.  A product of 128 terms summed in FP32 in any order is off by at most 128 half steps of
the sum of magnitudes, so a score is off by `136 * 2^-24 * spread * scale` (eight more for the
scaling and the exponent's argument), a probability relatively by twice that (numerator and
denominator).  Probabilities enter the second product rounded to the activations' type (half a step
each, so at most half a step of sum_p |v|), its FP32 sum over n keys is off by n more FP32 half
steps, and the result is rounded once.
"""
import math
import threading

import pytest
import torch

from cudnn_vsa_b200 import vsa_cache
from cudnn_vsa_b200.vsa import vsa_attention, vsa_decode
from cudnn_vsa_b200.vsa_layout import Segment, build_vsa_layout
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
SCALE = 128 ** -0.5


def make_cache(pages, heads, dtype, gen, poison=True):
    """A cache of normal values; pages are filled, what no request holds can be poisoned later."""
    scales = (None, None)
    if dtype == E4M3:
        scales = tuple((torch.rand(heads, generator=gen) + 0.5).cuda() * (4.0 / 448) for _ in range(2))
    cache = vsa_cache.build_paged_cache(pages, heads, dtype=dtype, k_scale=scales[0], v_scale=scales[1])
    for x, scale in ((cache.k, scales[0]), (cache.v, scales[1])):
        value = torch.randn(x.shape, generator=gen).cuda()
        x.copy_(value if scale is None else (value / scale[:, None, None]).clamp(-448, 448))
    return cache


def poison_unused(cache, tables, lengths):
    """NaN in every row that no request has filled, in the sums of every page that no request holds."""
    live = torch.zeros(cache.pages, 64, dtype=torch.bool)
    for s, n in enumerate(lengths):
        for i in range(ref.pages_of(max(0, n))):
            live[int(tables[s, i]), :min(64, n - 64 * i)] = True
    dead = ~live.cuda()
    for x in (cache.k, cache.v):
        x.view(torch.uint8).copy_(torch.where(dead[:, None, :, None], 0xFF, x.view(torch.uint8)))
    unheld = dead.all(1)
    cache.k_sum[unheld] = math.nan
    cache.v_sum[unheld] = math.nan


def fill_sums(cache, tables, lengths):
    for page, (k, v, _, _) in ref.page_sums(cache, tables, lengths).items():
        cache.k_sum[page], cache.v_sum[page] = k.float().cuda(), v.float().cuda()


def check_attention(out, lse, want, cache, dtype, keys, extra=0.0):
    o, l, size, spread = want
    assert out.dtype == dtype and out.shape == o.shape
    p_half = ref.HALF_STEP[FP16 if cache.k.dtype == E4M3 else dtype]
    score = 136 * ref.FP32 * spread * SCALE
    bound = ref.HALF_STEP[dtype] * (o.abs() + size * p_half) + size * (p_half + 2 * score[..., None] + (keys + 16) * ref.FP32) + extra
    err = (out.cpu().double() - o).abs()
    assert (err <= bound).all(), f"off by {(err / bound.clamp_min(1e-300)).max():.3g} of the bound"
    if lse is not None:
        empty = l == -math.inf
        assert torch.equal(lse.cpu() == -math.inf, empty)
        off = (lse.cpu().double() - l)[~empty].abs()
        assert (off <= (score + (keys + 16) * ref.FP32 + 4 * ref.FP32 * l.abs())[~empty].clamp_min(1e-7)).all()


# ------------------------------------------------------------------------------------------- plan

def run_plan(lengths, new, width, pool, tokens, rows=None, inplace=False, spare=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    order = torch.randperm(pool, generator=gen).tolist()
    tables = [[-7] * width for _ in lengths]
    for s, n in enumerate(lengths):
        for i in range(ref.pages_of(n)):
            tables[s][i] = order.pop()
    free = order + [-9] * (pool - len(order))
    count = len(order) if spare is None else min(spare, len(order))

    def dev(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    d = {"lengths": dev(lengths), "new": dev(new), "tables": dev(tables), "free_pages": dev(free), "free_count": dev([count])}
    out = None
    if inplace:
        first = vsa_cache.plan_paged_step(d["lengths"], torch.zeros_like(d["new"]), d["tables"], d["free_pages"], d["free_count"],
                                          tokens=tokens, rows_per_request=rows)
        out = vsa_cache.PagedStep(d["lengths"], d["free_count"], first.admitted, first.row_slot, first.runs, d["tables"])
    step = vsa_cache.plan_paged_step(d["lengths"], d["new"], d["tables"], d["free_pages"], d["free_count"], tokens=tokens,
                                     rows_per_request=rows, out=out)
    want = ref.plan(lengths, new, tables, free, count, tokens, rows)
    for name, value in want.items():
        got = d["free_pages"] if name == "free_pages" else getattr(step, name)
        assert got.tolist() == value, name
    if inplace:
        assert step.lengths is d["lengths"] and d["lengths"].tolist() == want["lengths"]
    return d, step, want


@pytest.mark.parametrize("requests,longest,most,ended,tokens", [
    (1, 0, 1, 0, 1), (1, 64, 64, 0, 64), (1, 63, 1, 0, 1), (3, 200, 130, 1, 300), (64, 4000, 1, 5, 64), (64, 4000, 1, 5, 70),
    (300, 700, 90, 40, 14000), (1025, 100, 3, 100, 2100), (8192, 10, 2, 9, 9000), (5, 130, 5000, 0, 15000)])
def test_plan_matches_the_plain_form(requests, longest, most, ended, tokens):
    gen = torch.Generator().manual_seed(requests + longest)
    lengths = torch.randint(0, longest + 1, (requests,), generator=gen).tolist()
    new = torch.randint(0, most + 1, (requests,), generator=gen).tolist()
    lengths[0], new[0] = longest, most
    for i in range(ended):
        new[(7 * i + 1) % requests] = -1 - i % 3
    width = max(ref.pages_of(a + max(0, b)) for a, b in zip(lengths, new)) + 1
    pool = sum(ref.pages_of(a + max(0, b)) for a, b in zip(lengths, new)) + 2
    run_plan(lengths, new, width, pool, tokens)


def test_plan_refuses_what_does_not_fit():
    # Row 1 wants more pages than its table row has, row 3 more than the stack holds; rows behind it
    # that need a page are refused with it, one that needs none is served.
    d, step, want = run_plan([64, 100, 10, 0, 5, 60], [1, 60, 54, 640, 70, 4], 2, 20, 900, spare=3)
    assert want["admitted"] == [True, False, True, False, True, True]
    d, step, want = run_plan([64, 100, 10, 0, 5, 60], [1, 20, 54, 640, 70, 4], 20, 40, 900, spare=3)
    assert want["admitted"] == [True, True, True, False, False, True]
    # Pages that a request gives back in the same step serve another one.
    d, step, want = run_plan([640, 0], [-1, 640], 10, 10, 640)
    assert want["admitted"] == [False, True] and want["free_count"] == [0]
    # Rows that do not fit the step.
    d, step, want = run_plan([0, 0, 0], [5, 10, 0], 2, 9, 9)
    assert want["admitted"] == [True, False, True]


@pytest.mark.parametrize("requests", [20, 200])  # one CTA, a cluster of them
@pytest.mark.parametrize("most,ended,spare,short,rows,inplace", [
    (5, 0, 3, 0, None, False), (90, 4, 10, 50, None, True), (300, 15, 0, 0, None, False), (7, 3, 2, 0, 7, True), (130, 5, 40, 300, 130, False)])
def test_plan_of_more_than_fits(requests, most, ended, spare, short, rows, inplace):
    """Steps that may be short of pages, of rows, or of table columns: who is served, and with which pages."""
    gen = torch.Generator().manual_seed(requests + most)
    lengths = torch.randint(0, 400, (requests,), generator=gen).tolist()
    new = torch.randint(0, most + 1, (requests,), generator=gen).tolist()
    for i in range(ended):
        new[(7 * i + 1) % requests] = -1
    width = 7  # 448 tokens
    pool = sum(ref.pages_of(n) for n in lengths) + spare
    tokens = max(1, (requests * rows if rows else sum(max(0, n) for n in new)) - short)
    d, step, want = run_plan(lengths, new, width, pool, tokens, rows=rows, inplace=inplace, spare=spare)
    assert any(want["admitted"])


def test_plan_with_one_row_block_per_request_and_in_place():
    run_plan([0, 64, 65, 3], [1, 0, -1, 1], 4, 12, 4, rows=1)
    run_plan([0, 64, 65, 3, 9], [3, 2, 4, 0, 3], 4, 12, 14, rows=3)
    run_plan([10, 127, 64, 300], [1, 2, -1, 1], 8, 30, 8, inplace=True)


def test_plan_can_be_repeated():
    d, step, want = run_plan([100, 50, 640], [30, 20, -1], 12, 30, 64)
    again = vsa_cache.plan_paged_step(d["lengths"], d["new"], d["tables"], d["free_pages"], d["free_count"], tokens=64)
    for name in ("lengths", "free_count", "admitted", "row_slot", "runs", "tables"):
        assert torch.equal(getattr(again, name), getattr(step, name)), name


def test_plan_replays_as_a_graph_that_advances_its_own_state():
    requests, width, pool = 3, 4, 12
    lengths = torch.tensor([62, 0, 64], dtype=torch.int32, device="cuda")
    new = torch.ones(requests, dtype=torch.int32, device="cuda")
    tables = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    tables[0, 0], tables[2, 0] = 5, 7
    free = torch.tensor([0, 1, 2, 3, 4, 6, 8, 9, 10, 11, -1, -1], dtype=torch.int32, device="cuda")
    count = torch.tensor([10], dtype=torch.int32, device="cuda")
    state = [lengths.tolist(), tables.tolist(), free.tolist(), count.item()]
    step = vsa_cache.plan_paged_step(lengths.clone(), new * 0, tables, free, count.clone(), tokens=3)
    step = vsa_cache.PagedStep(lengths, count, step.admitted, step.row_slot, step.runs, tables)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        vsa_cache.plan_paged_step(lengths, new, tables, free, count, tokens=3, out=step)
    for _ in range(130):
        graph.replay()
        want = ref.plan(state[0], [1] * requests, state[1], state[2], state[3], 3)
        state = [want["lengths"], want["tables"], want["free_pages"], want["free_count"][0]]
        assert step.row_slot.tolist() == want["row_slot"]
    torch.cuda.synchronize()
    assert lengths.tolist() == state[0] and tables.tolist() == state[1] and count.item() == state[3]


# ----------------------------------------------------------------------------------------- append

def step_for(lengths, new, tables, tokens=None, rows=None):
    """A step whose pages are all in the tables already (none is taken from the stack)."""
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    tokens = tokens or max(1, sum(new))
    total = [a + b for a, b in zip(lengths, new)]
    # Hand the pages out through the plan itself: the stack holds them in the order they are popped.
    order, known = [], tables.cpu()
    for s, (a, b) in enumerate(zip(lengths, total)):
        order += known[s, ref.pages_of(a):ref.pages_of(b)].tolist()
    free = torch.tensor(order[::-1] or [0], dtype=torch.int32, device="cuda")
    step = vsa_cache.plan_paged_step(torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                                     torch.tensor(new, dtype=torch.int32, device="cuda"), tables, free,
                                     none + len(order), tokens=tokens, rows_per_request=rows)
    assert step.lengths.tolist() == total and step.admitted.all()
    return step


def append_case(dtype, store, heads, lengths, new, seed, padded=0, view=False):
    gen = torch.Generator().manual_seed(seed)
    total = [a + b for a, b in zip(lengths, new)]
    pages = sum(ref.pages_of(n) for n in total) + 3
    cache = make_cache(pages, heads, store, gen)
    tables = ref.make_tables(total, pages, gen)
    poison_unused(cache, tables, lengths)
    tokens = sum(new) + padded
    step = step_for(lengths, new, tables, tokens)
    if view:  # two fields of a fused projection
        mixed = torch.randn(tokens, heads, 4, 128, generator=gen).to(dtype).cuda()
        k, v = mixed[:, :, 1], mixed[:, :, 2]
    else:
        k, v = (torch.randn(tokens, heads, 128, generator=gen).to(dtype).cuda() for _ in range(2))
    return cache, tables, step, k, v, sum(new)


@pytest.mark.parametrize("dtype,store", [(BF16, BF16), (FP16, FP16), (BF16, E4M3), (FP16, E4M3)])
@pytest.mark.parametrize("heads,lengths,new,padded,view", [
    (1, [0], [1], 0, False), (1, [63], [2], 0, False), (2, [64], [64], 1, False), (3, [5, 0, 127, 64, 300], [1, 0, 1, 1, 1], 2, True),
    (2, [10, 0, 63, 64, 1], [200, 65, 1, 128, 63], 7, False), (5, [0], [1000], 0, True)])
def test_append_matches_the_plain_form(dtype, store, heads, lengths, new, padded, view):
    cache, tables, step, k, v, used = append_case(dtype, store, heads, lengths, new, 3, padded, view)
    before = {n: getattr(cache, n).clone() for n in ("k", "v", "k_sum", "v_sum")}
    vsa_cache.append_tokens(cache, k, v, step)
    slot = step.row_slot
    assert (slot[used:] == -1).all()
    page, row = slot[:used] // 64, slot[:used] % 64
    for x, new_rows, scale, old in ((cache.k, k, cache.k_scale, before["k"]), (cache.v, v, cache.v_scale, before["v"])):
        want = old.view(torch.uint8).clone()
        rows = ref.stored(new_rows[:used], scale, store).contiguous()
        want[page, :, row] = rows.view(torch.uint8).view(used, heads, -1)
        assert torch.equal(x.view(torch.uint8), want)  # new rows exact, every other byte untouched
    touched = {int(p) for p in page.tolist()}
    sums = ref.page_sums(cache, tables, step.lengths)
    for name, a, b in (("k_sum", 0, 2), ("v_sum", 1, 3)):
        got = getattr(cache, name)
        for p in range(cache.pages):
            if p in touched:
                bound = 66 * ref.FP32 * sums[p][b]  # 64 additions, and the scale's product
                assert ((got[p].cpu().double() - sums[p][a]).abs() <= bound).all()
            else:
                assert torch.equal(got[p].view(torch.int32), before[name][p].view(torch.int32))
    after = {n: getattr(cache, n).clone() for n in before}
    vsa_cache.append_tokens(cache, k, v, step)  # again: nothing changes
    for n, x in after.items():
        assert torch.equal(getattr(cache, n).view(torch.uint8), x.view(torch.uint8))
    vsa_cache.check_cache_status(cache)


def test_append_with_one_row_block_per_request():
    gen = torch.Generator().manual_seed(4)
    lengths, new = [63, 0, 64, 10], [2, 0, 1, 3]
    cache = make_cache(12, 2, FP16, gen)
    tables = ref.make_tables([65, 0, 65, 13], 12, gen)
    step = step_for(lengths, new, tables, tokens=12, rows=3)
    k, v = (torch.randn(12, 2, 128, generator=gen).to(FP16).cuda() for _ in range(2))
    vsa_cache.append_tokens(cache, k, v, step)
    for s, (a, b) in enumerate(zip(lengths, new)):
        for i in range(b):
            page = int(tables[s, (a + i) // 64])
            assert torch.equal(cache.k[page, :, (a + i) % 64], k[3 * s + i]) and torch.equal(cache.v[page, :, (a + i) % 64], v[3 * s + i])
    fill_sums(cache, tables, step.lengths)


def test_append_after_a_request_was_cut_back():
    cache, tables, step, k, v, _ = append_case(BF16, BF16, 2, [0, 30], [100, 30], 5)
    vsa_cache.append_tokens(cache, k, v, step)
    cut = step_for([70, 31], [3, 1], tables)  # 27 and 28 tokens of the last step are dropped
    rows = torch.randn(4, 2, 128, generator=torch.Generator().manual_seed(6)).to(BF16).cuda()
    vsa_cache.append_tokens(cache, rows, rows, cut)
    sums = ref.page_sums(cache, tables, cut.lengths)
    for page, (a, b, c, d) in sums.items():
        assert ((cache.k_sum[page].cpu().double() - a).abs() <= 66 * ref.FP32 * c).all()
        assert ((cache.v_sum[page].cpu().double() - b).abs() <= 66 * ref.FP32 * d).all()


def test_append_saturates_and_keeps_nan_in_an_e4m3_cache():
    one = torch.ones(1, device="cuda")
    cache = vsa_cache.build_paged_cache(2, 1, dtype=E4M3, k_scale=one, v_scale=one * 0.5)
    step = step_for([0], [2], torch.tensor([[1]], dtype=torch.int32, device="cuda"))
    k = torch.zeros(2, 1, 128, dtype=BF16, device="cuda")
    k[0, 0, :6] = torch.tensor([1e6, -1e6, math.inf, -math.inf, 440.0, 2.0 ** -10], dtype=BF16)
    k[1, 0, 0] = math.nan
    vsa_cache.append_tokens(cache, k, k, step)
    assert cache.k[1, 0, 0, :6].float().tolist() == [448.0, -448.0, 448.0, -448.0, 448.0, 0.0]
    assert cache.k[1, 0, 1, 0].float().isnan() and cache.k_sum[1, 0, 0].isnan()
    assert cache.k_sum[1, 0, 1].item() == -448.0 and cache.v_sum[1, 0, 1].item() == -224.0


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -7, 0.011, 1 / 448, 3.3e4, 1e-30, 1.5e-38, 1e38])
def test_append_rounds_every_number_as_its_quotient(dtype, scale):
    """All 65,536 numbers of the type, zeros, infinities and borders between two e4m3 numbers among them."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).view(512, 1, 128).cuda()
    scales = torch.full((1,), scale, device="cuda")
    cache = vsa_cache.build_paged_cache(8, 1, dtype=E4M3, k_scale=scales, v_scale=scales * 0.7)
    tables = torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8)
    vsa_cache.append_tokens(cache, x, x, step_for([0], [512], tables))
    for got, by in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        want = (x.float() / by).clamp(-448, 448).to(E4M3).view(torch.uint8).view(-1)
        got, nan = got.view(torch.uint8).view(-1), x.isnan().view(-1)
        assert torch.equal(got[~nan], want[~nan]) and ((got[nan] & 0x7F) == 0x7F).all()


def test_append_leaves_out_pages_the_cache_does_not_have():
    cache, tables, step, k, v, used = append_case(BF16, BF16, 2, [0, 0], [70, 5], 9)
    bad = step.runs.clone()
    lost = int(bad[1, 2])
    bad[1, 2] = cache.pages
    before = cache.k[lost].clone()
    vsa_cache.append_tokens(cache, k, v, vsa_cache.PagedStep(step.lengths, step.free_count, step.admitted, step.row_slot, bad, tables))
    assert torch.equal(cache.k[lost].view(torch.int16), before.view(torch.int16))
    with pytest.raises(RuntimeError, match="outside the cache"):
        vsa_cache.check_cache_status(cache)


# ----------------------------------------------------------------------------------------- select

def select_case(dtype, heads, group, lengths, seed, extra=1, view=False):
    gen = torch.Generator().manual_seed(seed)
    pages = sum(ref.pages_of(n) for n in lengths) + 2
    cache = vsa_cache.build_paged_cache(pages, heads, dtype=dtype)
    cache.k_sum.copy_(torch.randn(cache.k_sum.shape, generator=gen) * 20)
    cache.v_sum.copy_(torch.randn(cache.v_sum.shape, generator=gen) * 20)
    tables = ref.make_tables(lengths, pages, gen, extra)
    requests = len(lengths)
    if view:
        q = torch.randn(requests, heads * group, 3, 128, generator=gen).to(dtype).cuda()[:, :, 1]
    else:
        q = torch.randn(requests, heads * group, 128, generator=gen).to(dtype).cuda()
    return cache, q, tables, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def check_coarse(got, q, cache, tables, lengths, heads, pages):
    o, size, spread = ref.coarse(q, cache.k_sum, cache.v_sum, tables, lengths, heads)
    score = 136 * ref.FP32 * spread * SCALE
    bound = size * (2 * score[..., None] + (pages + 24) * ref.FP32)
    assert ((got.cpu().double() - o).abs() <= bound).all()


@pytest.mark.parametrize("dtype,wide", [(BF16, 0), (FP16, 0), (BF16, 150)])  # short tables have a kernel of their own
@pytest.mark.parametrize("heads,group,lengths,keep,first,last,extra,view", [
    (1, 1, [1], 2, 1, 1, 0, False), (2, 4, [0, 64, 65, 128, 129, 700], 2, 1, 1, 1, True), (3, 2, [1000, 2000, 640], 10, 0, 0, 3, False),
    (1, 3, [4000, 0, 9], 7, 2, 1, 1, False), (2, 7, [64 * 12, 64 * 13], 12, 3, 2, 1, False), (1, 16, [20000], 100, 1, 1, 0, True),
    (5, 1, [9000, 8000], 130, 0, 1, 0, False), (1, 1, [64 * 3000 + 1], 300, 4, 4, 0, False), (2, 5, [3000] * 40, 20, 1, 2, 700, False),
    (1, 2, [640], 700, 1, 1, 0, False), (2, 9, [800, 0, 5000], 6, 1, 1, 1, False), (1, 20, [70, 1300], 4, 1, 2, 0, True),
    (1, 1, [0] * 200 + [1000] + [0] * 60 + [65], 5, 1, 1, 0, False), (1, 2, [150] * 1000, 2, 1, 1, 1, False),
    (2, 9, [150, 900, 0, 6400] * 50, 5, 1, 1, 1, False), (2, 3, [2000, 64, 0] * 110, 7, 1, 1, 1, True)])
def test_select_matches_the_plain_form(dtype, wide, heads, group, lengths, keep, first, last, extra, view):
    cache, q, tables, n = select_case(dtype, heads, group, lengths, heads * 100 + keep, extra + wide, view)
    want = ref.select(q, cache.k_sum, tables, n, heads, keep, first, last)
    got = vsa_cache.select_pages(q, cache, tables, n, keep=keep, first=first, last=last)
    assert torch.equal(got.cpu(), want)
    both, mean = vsa_cache.select_pages(q, cache, tables, n, keep=keep, first=first, last=last, coarse=True)
    assert torch.equal(both, got)
    check_coarse(mean, q, cache, tables, n, heads, max(1, max(lengths)) // 64 + 1)
    none, alone = vsa_cache.select_pages(q, cache, tables, n, coarse=True)
    assert none is None and torch.equal(alone, mean)
    vsa_cache.check_cache_status(cache)


def test_select_ties_go_to_the_lowest_page():
    cache, q, tables, n = select_case(BF16, 2, 2, [64 * 40, 64 * 700], 1)
    cache.k_sum.copy_(cache.k_sum[:1].expand_as(cache.k_sum))  # every page scores alike
    got = vsa_cache.select_pages(q, cache, tables, n, keep=9, first=1, last=2).cpu()
    for s, pages in enumerate((40, 700)):
        assert got[s].tolist() == [[0, 1, 2, 3, 4, 5, 6, pages - 2, pages - 1]] * 2
    # A few values only: the interval that holds the border has many equal scores on both sides.
    gen = torch.Generator().manual_seed(2)
    level = torch.randint(0, 3, (cache.pages, 1, 1), generator=gen).float().cuda()
    cache.k_sum.copy_(level.expand_as(cache.k_sum))
    want = ref.select(q, cache.k_sum, tables, n, 2, 11)
    assert torch.equal(vsa_cache.select_pages(q, cache, tables, n, keep=11).cpu(), want)


def test_select_with_scores_of_all_sizes_infinities_and_nan():
    cache, q, tables, n = select_case(BF16, 1, 1, [64 * 500], 4)
    gen = torch.Generator().manual_seed(5)
    size = 10.0 ** (torch.rand(cache.pages, 1, 1, generator=gen) * 60 - 30)  # sixty orders of magnitude
    cache.k_sum.mul_(size.float().cuda())
    for keep in (2, 3, 40, 499):
        want = ref.select(q, cache.k_sum, tables, n, 1, keep)
        assert torch.equal(vsa_cache.select_pages(q, cache, tables, n, keep=keep).cpu(), want), keep
    q[0, 0, 5] = 1.0
    at = tables[0, [7, 100, 200, 300]].long()
    for page, value in zip(at.tolist(), (math.inf, -math.inf, math.nan, 3e38)):
        cache.k_sum[page, 0, 5] = value
    for keep in (2, 3, 4, 5, 60):
        want = ref.select(q, cache.k_sum, tables, n, 1, keep)
        assert torch.equal(vsa_cache.select_pages(q, cache, tables, n, keep=keep).cpu(), want), keep


def test_select_with_most_scores_next_to_one_another():
    """One score far above the others puts them all into one bin; their own spread decides."""
    cache, q, tables, n = select_case(BF16, 2, 1, [64 * 1500, 64 * 1400 + 5], 6)
    cache.k_sum[int(tables[0, 700])] *= 1e30
    cache.k_sum[int(tables[1, 10])] *= -1e30
    for keep in (2, 3, 4, 700, 1399):
        want = ref.select(q, cache.k_sum, tables, n, 2, keep)
        assert torch.equal(vsa_cache.select_pages(q, cache, tables, n, keep=keep).cpu(), want), keep
    # Many equal scores between higher and lower ones.
    level = (torch.arange(cache.pages) % 5 == 0).float() + (torch.arange(cache.pages) % 97 == 0).float()
    cache.k_sum.copy_(level[:, None, None].cuda().expand_as(cache.k_sum))
    for keep in (30, 200, 900):
        want = ref.select(q, cache.k_sum, tables, n, 2, keep)
        assert torch.equal(vsa_cache.select_pages(q, cache, tables, n, keep=keep).cpu(), want), keep


@pytest.mark.parametrize("requests", [1, 200, 400])  # tables of up to 128 pages: CTAs of 256, 128 and 64 threads
def test_select_with_ties_and_neighbours_in_short_tables(requests):
    cache, q, tables, n = select_case(BF16, 2, 2, [64 * 120] * requests, 7)
    cache.k_sum.mul_(1e-3).add_(1.0)  # most scores share a bin ...
    cache.k_sum[tables[:, 50].long()] *= 1e20
    for keep in (3, 40, 119):
        want = ref.select(q, cache.k_sum, tables, n, 2, keep)
        assert torch.equal(vsa_cache.select_pages(q, cache, tables, n, keep=keep).cpu(), want), keep
    cache.k_sum.copy_((torch.arange(cache.pages) % 3).float()[:, None, None].cuda().expand_as(cache.k_sum))  # ... or tie
    for keep in (3, 40, 119):
        want = ref.select(q, cache.k_sum, tables, n, 2, keep)
        assert torch.equal(vsa_cache.select_pages(q, cache, tables, n, keep=keep).cpu(), want), keep


@pytest.mark.parametrize("extra", [1, 150])
def test_select_leaves_out_pages_the_cache_does_not_have(extra):
    cache, q, tables, n = select_case(BF16, 1, 2, [640, 640], 8, extra)
    tables[0, 4] = cache.pages
    pages, mean = vsa_cache.select_pages(q, cache, tables, n, keep=20, coarse=True)
    assert pages[:, :, :10].tolist() == [[list(range(10))]] * 2
    # The attention over the means leaves the page out.
    rest = torch.stack([torch.cat([tables[0, :4], tables[0, 5:10], tables[0, :1]]), tables[1, :10]])
    check_coarse(mean, q, cache, rest, torch.tensor([64 * 9, 64 * 10], dtype=torch.int32), 1, 10)
    with pytest.raises(RuntimeError, match="outside the cache"):
        vsa_cache.check_cache_status(cache)


# -------------------------------------------------------------------------------------- attention

ATTENTION = [  # heads, group, lengths
    (1, 1, [1]), (1, 8, [100]), (2, 4, [0, 1, 63, 64, 65, 0]), (3, 3, [128, 129, 7, 500]), (1, 16, [1000, 1]), (2, 17, [300, 64]),
    (4, 7, [5, 1500, 20]), (1, 33, [65]), (8, 1, [400, 100, 90, 17]), (12, 1, [5000]), (1, 2, [20000, 1, 0, 64]), (2, 5, [90] * 70),
    (1, 3, [0] * 200 + [1000] + [0] * 60 + [65]), (2, 1, [30, 70] * 500), (2, 12, [700] * 30), (1, 40, [900, 0, 100]),
    (2, 2, [1000, 200] * 50)]


def attention_case(dtype, store, heads, group, lengths, seed, extra=1):
    gen = torch.Generator().manual_seed(seed)
    pages = sum(ref.pages_of(n) for n in lengths) + 2
    cache = make_cache(pages, heads, store, gen)
    tables = ref.make_tables(lengths, pages, gen, extra)
    poison_unused(cache, tables, lengths)
    q = torch.randn(len(lengths), heads * group, 128, generator=gen).to(dtype).cuda()
    return cache, q, tables, torch.tensor(lengths, dtype=torch.int32, device="cuda")


TABLES = [1, 70]  # columns of the tables behind the longest request: tables of few pages have a kernel of their own


@pytest.mark.parametrize("extra", TABLES)
@pytest.mark.parametrize("dtype,store", [(BF16, BF16), (FP16, FP16), (BF16, E4M3), (FP16, E4M3)])
@pytest.mark.parametrize("heads,group,lengths", ATTENTION)
def test_attention_matches_the_plain_form(dtype, store, heads, group, lengths, extra):
    cache, q, tables, n = attention_case(dtype, store, heads, group, lengths, heads * group + len(lengths), extra)
    out, lse = vsa_cache.paged_attention(q, cache, tables, n, return_lse=True)
    check_attention(out, lse, ref.attention(q, cache, tables, n), cache, dtype, max(lengths))
    again, lse2 = vsa_cache.paged_attention(q, cache, tables, n, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert torch.equal(vsa_cache.paged_attention(q, cache, tables, n), out)
    vsa_cache.check_cache_status(cache)


@pytest.mark.parametrize("dtype,store", [(BF16, BF16), (FP16, FP16), (BF16, E4M3)])
@pytest.mark.parametrize("heads,group,lengths,keep", [
    (1, 1, [700], 3), (2, 4, [0, 64, 65, 3000, 640], 5), (3, 2, [129, 40], 9), (1, 9, [6400, 6399], 70), (8, 1, [1000] * 9, 4)])
def test_attention_over_chosen_pages(dtype, store, heads, group, lengths, keep):
    cache, q, tables, n = attention_case(dtype, store, heads, group, lengths, keep)
    gen = torch.Generator().manual_seed(keep + 1)
    chosen = torch.full((len(lengths), heads, keep), -1, dtype=torch.int32)
    for s, length in enumerate(lengths):
        for h in range(heads):
            n_pages = ref.pages_of(length)
            some = torch.randperm(n_pages, generator=gen)[:keep - (h + s) % 2].sort().values.int()
            at = torch.randperm(min(keep, n_pages), generator=gen)[:len(some)].sort().values  # holes among the first
            chosen[s, h, at] = some
    out, lse = vsa_cache.paged_attention(q, cache, tables, n, pages=chosen.cuda(), return_lse=True)
    check_attention(out, lse, ref.attention(q, cache, tables, n, chosen), cache, dtype, keep * 64)
    none = torch.full_like(chosen, -1).cuda()
    out, lse = vsa_cache.paged_attention(q, cache, tables, n, pages=none, return_lse=True)
    assert not out.count_nonzero() and (lse == -math.inf).all()


def test_attention_with_strided_queries_gate_and_scale():
    heads, group, lengths = 2, 3, [300, 0, 65]
    cache, q, tables, n = attention_case(BF16, BF16, heads, group, lengths, 11)
    gen = torch.Generator().manual_seed(12)
    mixed = torch.randn(3, heads * group, 2, 128, generator=gen).to(BF16).cuda()
    q, gate = mixed[:, :, 0], mixed[:, :, 1]
    coarse = torch.randn(3, heads * group, 128, generator=gen).cuda()
    wide = torch.cat([tables, tables], 1)[:, :tables.shape[1]]  # a view whose rows are further apart
    out = vsa_cache.paged_attention(q, cache, wide, n, gate=gate, coarse=coarse)
    o, l, size, spread = ref.attention(q, cache, tables, n)
    merged = gate.cpu().double() * coarse.cpu().double()
    # The merge adds one FP32 product and sum.
    check_attention(out, None, (o + merged, l, size, spread), cache, BF16, 300, extra=2 * ref.FP32 * (merged.abs() + o.abs()))
    plain = vsa_cache.paged_attention(q.contiguous(), cache, tables, n)
    assert torch.equal(plain, vsa_cache.paged_attention(q, cache, wide, n))
    zero, lse = vsa_cache.paged_attention(q, cache, tables, n, scale=0.0, return_lse=True)
    want = ref.attention(q, cache, tables, n, scale=0.0)
    check_attention(zero, lse, (*want[:3], want[3] * 0), cache, BF16, 300)


@pytest.mark.parametrize("extra", TABLES)
def test_attention_with_infinities_and_nan_in_seen_and_unseen_rows(extra):
    cache, q, tables, n = attention_case(BF16, BF16, 1, 2, [100, 100, 100], 13, extra)
    cache.v[int(tables[0, 1]), 0, 35, 7] = math.inf   # row 99: seen
    cache.v[int(tables[1, 1]), 0, 36, 7] = math.inf   # row 100: not seen
    cache.k[int(tables[1, 1]), 0, 36] = math.inf
    cache.k[int(tables[2, 0]), 0, 5, 9] = math.nan
    out, lse = vsa_cache.paged_attention(q, cache, tables, n, return_lse=True)
    assert (out[0, :, 7] == math.inf).all() and out[0, :, :7].isfinite().all()
    assert out[1].isfinite().all() and lse[1].isfinite().all()
    assert out[2].isnan().all() and lse[2].isnan().all()
    # A first page whose scores are all -infinity leaves the weight to the second.
    cache, q, tables, n = attention_case(BF16, BF16, 1, 1, [100], 14, extra)
    cache.k[int(tables[0, 0]), 0, :, 3] = -math.inf
    q[0, 0, 3] = 1.0
    part = vsa_cache.paged_attention(q, cache, tables, n, pages=torch.tensor([[[1]]], dtype=torch.int32, device="cuda"))
    whole = vsa_cache.paged_attention(q, cache, tables, n)
    assert whole.isfinite().all()
    assert (whole - part).abs().max() <= 2 * 2.0 ** -8 * 4.0  # values of at most 4, rounded twice


@pytest.mark.parametrize("extra", TABLES)
def test_attention_scores_of_large_magnitude(extra):
    cache, q, tables, n = attention_case(BF16, BF16, 2, 2, [700, 3], 15, extra)
    q.mul_(30.0)  # scores in the hundreds: the softmax has one or two winners, far apart in the cache
    out, lse = vsa_cache.paged_attention(q, cache, tables, n, return_lse=True)
    check_attention(out, lse, ref.attention(q, cache, tables, n), cache, BF16, 700)


@pytest.mark.parametrize("extra", TABLES)
def test_attention_with_large_queries_and_shared_heads(extra):
    """Queries near the ends of BF16's range over an 8-bit cache, and one query row for all heads."""
    for size in (1e30, 1e-30):
        cache, q, tables, n = attention_case(BF16, E4M3, 2, 2, [700, 65], 18, extra)
        q.mul_(size)
        scale = SCALE / size if size > 1 else SCALE
        out, lse = vsa_cache.paged_attention(q, cache, tables, n, scale=scale, return_lse=True)
        o, l, mag, spread = ref.attention(q, cache, tables, n, scale=scale)
        check_attention(out, lse, (o, l, mag, spread * scale / SCALE), cache, BF16, 700)
    cache, q, tables, n = attention_case(BF16, BF16, 2, 3, [300, 64], 19, extra)
    one = q[:, :1].expand(-1, 6, -1)
    out = vsa_cache.paged_attention(one, cache, tables, n)
    assert torch.equal(out, vsa_cache.paged_attention(one.contiguous(), cache, tables, n))
    pages, mean = vsa_cache.select_pages(one, cache, tables, n, keep=3, coarse=True)
    again = vsa_cache.select_pages(one.contiguous(), cache, tables, n, keep=3, coarse=True)
    assert torch.equal(pages, again[0]) and torch.equal(mean, again[1])


@pytest.mark.parametrize("extra", TABLES)
def test_attention_leaves_out_pages_the_cache_does_not_have(extra):
    cache, q, tables, n = attention_case(BF16, BF16, 2, 2, [300, 64], 16, extra)
    tables[0, 2], tables[1, 0] = cache.pages, -1
    out, lse = vsa_cache.paged_attention(q, cache, tables, n, return_lse=True)
    check_attention(out, lse, ref.attention(q, cache, tables, n), cache, BF16, 300)
    assert not out[1].count_nonzero()
    with pytest.raises(RuntimeError, match="outside the cache"):
        vsa_cache.check_cache_status(cache)


def test_lengths_outside_the_table_are_clamped():
    cache, q, tables, n = attention_case(BF16, BF16, 1, 2, [128, 30], 17, extra=0)
    want = vsa_cache.paged_attention(q, cache, tables, n)
    big = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device="cuda")
    got = vsa_cache.paged_attention(q, cache, tables, big)
    assert torch.equal(got[0], want[0]) and not got[1].count_nonzero()
    pages, mean = vsa_cache.select_pages(q, cache, tables, big, keep=2, coarse=True)
    assert pages.tolist() == [[[0, 1]], [[-1, -1]]] and not mean[1].count_nonzero()


def test_offsets_beyond_32_bits():
    heads, pages = 8, 70000  # 4.6e9 elements
    k, v = (torch.empty(pages, heads, 64, 128, dtype=BF16, device="cuda") for _ in range(2))
    sums = [torch.zeros(pages, heads, 128, device="cuda") for _ in range(2)]
    cache = vsa_cache.PagedKVCache(k, v, *sums)
    lengths, new = [100, 0], [30, 200]
    total = [130, 200]
    tables = torch.stack([torch.tensor([pages - 1, pages - 5, 3, 0]), torch.tensor([2, pages - 2, pages - 3, pages - 4])]).int().cuda()
    gen = torch.Generator().manual_seed(1)
    held = tables.unique().long()
    for x in (k, v):
        x[held] = torch.randn(len(held), heads, 64, 128, generator=gen).to(BF16).cuda()
    step = step_for(lengths, new, tables)
    rows = torch.randn(230, heads, 128, generator=gen).to(BF16).cuda()
    vsa_cache.append_tokens(cache, rows, rows, step)
    q = torch.randn(2, heads, 128, generator=gen).to(BF16).cuda()
    # The same calls on a small cache that holds only these pages.
    small = vsa_cache.PagedKVCache(*(x[held].contiguous() for x in (k, v, *sums)))
    where = torch.searchsorted(held, tables.long()).int()
    vsa_cache.append_tokens(small, rows, rows, step_for(lengths, new, where.clone()))
    assert torch.equal(cache.k[held].view(torch.int16), small.k.view(torch.int16)) and torch.equal(cache.k_sum[held], small.k_sum)
    for wide in (0, 150):  # the kernels of short tables and of long ones
        more = torch.zeros(2, wide, dtype=torch.int32, device="cuda")
        got, lse = vsa_cache.paged_attention(q, cache, torch.cat([tables, more], 1), step.lengths, return_lse=True)
        want, lse2 = vsa_cache.paged_attention(q, small, torch.cat([where, more], 1), step.lengths, return_lse=True)
        assert torch.equal(got, want) and torch.equal(lse, lse2)
        check_attention(got, lse, ref.attention(q, small, where, step.lengths), small, BF16, 200)
        one = vsa_cache.select_pages(q, cache, torch.cat([tables, more], 1), step.lengths, keep=2, coarse=True)
        two = vsa_cache.select_pages(q, small, torch.cat([where, more], 1), step.lengths, keep=2, coarse=True)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


# ---------------------------------------------------------------------------------- run of them all

def test_decode_steps_across_pages_match_the_plain_form():
    """A hundred steps of three requests over e4m3 and BF16 caches: plan, append, select, attend, merge."""
    heads, group, keep = 2, 3, 3
    for store in (BF16, E4M3):
        gen = torch.Generator().manual_seed(21)
        cache = make_cache(24, heads, store, gen)
        lengths = torch.tensor([0, 60, 200], dtype=torch.int32, device="cuda")
        tables = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
        tables[1, :1] = 20
        tables[2, :4] = torch.tensor([23, 1, 9, 4], dtype=torch.int32)
        free = torch.tensor([i for i in range(24) if i not in (20, 23, 1, 9, 4)] + [-1] * 5, dtype=torch.int32, device="cuda")
        count = torch.tensor([19], dtype=torch.int32, device="cuda")
        fill_sums(cache, tables, lengths)
        new = torch.ones(3, dtype=torch.int32, device="cuda")
        for i in range(100):
            step = vsa_cache.plan_paged_step(lengths, new, tables, free, count, tokens=3)
            lengths, count = step.lengths, step.free_count
            k, v = (torch.randn(3, heads, 128, generator=gen).to(BF16).cuda() for _ in range(2))
            q, gate = (torch.randn(3, heads * group, 128, generator=gen).to(BF16).cuda() for _ in range(2))
            out = vsa_decode(q, k, v, gate, cache, step, keep=keep)
            if i % 9 == 0 or i > 96:
                chosen = ref.select(q, cache.k_sum, tables, lengths, heads, keep)
                o, l, size, spread = ref.attention(q, cache, tables, lengths, chosen)
                mean, msize, mspread = ref.coarse(q, cache.k_sum, cache.v_sum, tables, lengths, heads)
                g = gate.cpu().double()
                off = g.abs() * msize * (2 * 136 * ref.FP32 * mspread[..., None] * SCALE + 40 * ref.FP32)
                off = off + 2 * ref.FP32 * ((g * mean).abs() + o.abs())
                check_attention(out, None, (o + g * mean, l, size, spread), cache, BF16, 300, extra=off)
        vsa_cache.check_cache_status(cache)


def test_decode_answers_as_the_packed_attention_does():
    """The last token of a packed sample, as ``vsa_attention`` computes it and as a decode step does: two
    text chunks that are always visible, 24 video tiles of which a quarter is kept, and the token
    itself.  Two BF16 paths of the same function: each is within 2e-2 / 1e-2 of the FP32 oracle."""
    heads, text, video = 3, 129, (8, 16, 12)
    layout = build_vsa_layout([[Segment("text", text), Segment("video", video, .75)]], head_num=heads, device="cuda", input_order="block")
    tiles = 8 * 16 * 12 // 64
    gen = torch.Generator().manual_seed(31)
    q, k, v, gate = (torch.randn(layout.tokens, heads, 128, generator=gen).to(BF16).cuda() for _ in range(4))
    want = vsa_attention(q, k, v, gate, layout)[128]  # block order: 128 text rows, the single token, the tiles
    order = torch.cat([torch.arange(128), torch.arange(129, layout.tokens), torch.tensor([128])]).cuda()
    total = layout.tokens
    cache = vsa_cache.build_paged_cache(40, heads)
    tables = ref.make_tables([total], 40, gen)
    prompt = step_for([0], [total - 1], tables)
    vsa_cache.append_tokens(cache, k[order][:-1], v[order][:-1], prompt)
    step = step_for([total - 1], [1], tables)
    kept = math.ceil(0.25 * tiles)
    got = vsa_decode(q[128:129], k[128:129], v[128:129], gate[128:129], cache, step, keep=2 + kept + 1, first=2, last=1)[0]
    err = (got.double() - want.double())
    assert err.abs().max() <= 4e-2 and (err.norm() / want.double().norm()) <= 2e-2


def test_decode_without_gate_or_selection():
    cache, q, tables, n = attention_case(BF16, BF16, 2, 2, [130, 20], 41)
    fill_sums(cache, tables, n)
    step = step_for([129, 19], [1, 1], tables)
    k, v = (torch.randn(2, 2, 128, generator=torch.Generator().manual_seed(i)).to(BF16).cuda() for i in range(2))
    out = vsa_decode(q, k, v, None, cache, step)
    check_attention(out, None, ref.attention(q, cache, tables, step.lengths), cache, BF16, 130)
    out = vsa_decode(q, k, v, None, cache, step, keep=2)
    chosen = ref.select(q, cache.k_sum, tables, step.lengths, 2, 2)
    check_attention(out, None, ref.attention(q, cache, tables, step.lengths, chosen), cache, BF16, 130)
    gated = vsa_decode(q, k, v, q, cache, step)
    mean = vsa_cache.select_pages(q, cache, tables, step.lengths, coarse=True)[1]
    assert torch.equal(gated, vsa_cache.paged_attention(q, cache, tables, step.lengths, gate=q, coarse=mean))


def test_decode_keeping_more_pages_than_a_table_names():
    """A budget beyond the table's width is the whole request, whatever its size."""
    cache, q, tables, n = attention_case(BF16, BF16, 2, 2, [700, 20], 43)
    fill_sums(cache, tables, n)
    step = step_for([699, 19], [1, 1], tables)
    k, v = (torch.randn(2, 2, 128, generator=torch.Generator().manual_seed(i)).to(BF16).cuda() for i in range(2))
    for gate in (None, q):
        want = vsa_decode(q, k, v, gate, cache, step)
        for keep in (tables.shape[1], tables.shape[1] + 1, 2 ** 31 - 1):
            assert torch.equal(vsa_decode(q, k, v, gate, cache, step, keep=keep), want)


def test_cache_tensors_that_move_are_followed():
    """Storage of a cache that was moved (an offloaded cache that came back) is read and written where it is."""
    cache, q, tables, n = attention_case(BF16, BF16, 2, 2, [300, 20], 44)
    fill_sums(cache, tables, n)
    step = step_for([299, 19], [1, 1], tables)
    k, v = (torch.randn(2, 2, 128, generator=torch.Generator().manual_seed(i)).to(BF16).cuda() for i in range(2))
    want = vsa_decode(q, k, v, q, cache, step, keep=3)
    old = [x.data for x in (cache.k, cache.v, cache.k_sum, cache.v_sum)]
    for x in (cache.k, cache.v, cache.k_sum, cache.v_sum):
        x.data = x.data.clone()
    for x in old:
        x.view(torch.uint8).fill_(0xFF)
    assert torch.equal(vsa_decode(q, k, v, q, cache, step, keep=3), want)
    vsa_cache.append_tokens(cache, k, v, step)
    pages, mean = vsa_cache.select_pages(q, cache, tables, step.lengths, keep=3, coarse=True)
    assert torch.equal(vsa_cache.paged_attention(q, cache, tables, step.lengths, pages=pages, gate=q, coarse=mean), want)


def test_captured_behind_copies_fills_and_a_joined_stream():
    """Graph nodes of every kind before and between the operators: copies, fills, and work of another stream."""
    cache, q, tables, n = attention_case(BF16, BF16, 2, 2, [300, 20], 45)
    fill_sums(cache, tables, n)
    step = step_for([299, 19], [1, 1], tables)
    k, v, gate = (torch.randn(2, heads, 128, generator=torch.Generator().manual_seed(i)).to(BF16).cuda() for i, heads in enumerate((2, 2, 4)))
    want = vsa_decode(q, k, v, gate, cache, step, keep=3)
    alone = vsa_cache.paged_attention(q, cache, tables, step.lengths)
    held = [torch.zeros_like(x) for x in (q, k, v, gate)]
    lengths = step.lengths.clone()
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for x, y in zip(held, (q, k, v, gate)):
            x.copy_(y)
        start = torch.cuda.Event()
        start.record()
        with torch.cuda.stream(side):
            start.wait()
            now = vsa_cache.PagedStep(lengths.clone(), step.free_count, step.admitted, step.row_slot, step.runs, tables)
            other = vsa_cache.paged_attention(held[0], cache, tables, now.lengths)
            done.record()
        cache.status.zero_()
        done.wait()
        out = vsa_decode(*held, cache, now, keep=3)
        cache.status.zero_()
        again = vsa_cache.paged_attention(held[0], cache, tables, now.lengths)
    for _ in range(5):
        for x in (*held, out, other, again):
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(other, alone) and torch.equal(again, alone)


def test_captured_decode_steps_on_two_streams():
    """Two caches, each with a captured step (plan in place, then a layer), replayed side by side on two
    streams with inputs that change between replays."""
    heads, group = 2, 2
    worlds = []
    for seed in (51, 52):
        gen = torch.Generator().manual_seed(seed)
        cache = make_cache(16, heads, BF16, gen)
        tables = torch.arange(16, dtype=torch.int32, device="cuda").view(2, 8).contiguous()
        w = {"cache": cache, "tables": tables, "lengths": torch.tensor([60, 200], dtype=torch.int32, device="cuda"),
             "new": torch.ones(2, dtype=torch.int32, device="cuda"), "count": torch.tensor([10], dtype=torch.int32, device="cuda"),
             "free": torch.tensor([2, 3, 4, 5, 6, 7, 1, 13, 14, 15, 0, 0, 0, 0, 0, 0], dtype=torch.int32, device="cuda"), "gen": gen}
        fill_sums(cache, tables, w["lengths"])
        for name, n in (("q", heads * group), ("gate", heads * group), ("k", heads), ("v", heads)):
            w[name] = torch.randn(2, n, 128, generator=gen).to(BF16).cuda()
        blank = vsa_cache.plan_paged_step(w["lengths"].clone(), w["new"] * 0, tables, w["free"], w["count"].clone(), tokens=2)
        step = vsa_cache.PagedStep(w["lengths"], w["count"], blank.admitted, blank.row_slot, blank.runs, tables)
        w["stream"] = torch.cuda.Stream()
        w["graph"] = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(w["graph"], stream=w["stream"]):
            now = vsa_cache.plan_paged_step(w["lengths"], w["new"], tables, w["free"], w["count"], tokens=2, out=step)
            w["out"] = vsa_decode(w["q"], w["k"], w["v"], w["gate"], cache, now, keep=3)
        worlds.append(w)
    for _ in range(12):
        for w in worlds:
            for name in ("q", "gate", "k", "v"):
                w[name].copy_(torch.randn(w[name].shape, generator=w["gen"]).to(BF16))
        torch.cuda.synchronize()
        for w in worlds:
            with torch.cuda.stream(w["stream"]):
                w["graph"].replay()
        torch.cuda.synchronize()
        for w in worlds:
            chosen, mean = vsa_cache.select_pages(w["q"], w["cache"], w["tables"], w["lengths"], keep=3, coarse=True)
            want = vsa_cache.paged_attention(w["q"], w["cache"], w["tables"], w["lengths"], pages=chosen, gate=w["gate"], coarse=mean)
            assert torch.equal(w["out"], want)
    for w in worlds:
        assert w["lengths"].tolist() == [72, 212]
        o, l, size, spread = ref.attention(w["q"], w["cache"], w["tables"], w["lengths"])
        got = vsa_cache.paged_attention(w["q"], w["cache"], w["tables"], w["lengths"])
        check_attention(got, None, (o, l, size, spread), w["cache"], BF16, 212)


@pytest.mark.parametrize("requests", [5, 100])  # a plan of one CTA lets its successor start early; a cluster's does not
@pytest.mark.parametrize("width", [30, 200])  # the kernels of short tables and of long ones
@pytest.mark.parametrize("captured", [False, True])
def test_attention_and_selection_right_behind_a_plan(requests, width, captured):
    """A plan that advances lengths and tables, and the operators that read them, with nothing in between."""
    heads, group, pool = 2, 2, 25 * requests
    gen = torch.Generator().manual_seed(requests + width)
    cache = make_cache(pool, heads, BF16, gen)
    for x, of in ((cache.k_sum, cache.k), (cache.v_sum, cache.v)):
        x.copy_(of.float().sum(2))
    q = torch.randn(requests, heads * group, 128, generator=gen).to(BF16).cuda()
    ints = dict(dtype=torch.int32, device="cuda")
    tables = torch.full((requests, width), -1, **ints)
    free, count = torch.randperm(pool, generator=gen).int().cuda(), torch.tensor([pool], **ints)
    lengths, between = torch.zeros(requests, **ints), torch.zeros(requests, **ints)
    new = [torch.randint(0, 90, (requests,), generator=gen).int().cuda() for _ in range(2)]
    rows = 90 * requests
    blank = [vsa_cache.plan_paged_step(lengths, new[0] * 0, tables, free, count, tokens=rows) for _ in range(2)]
    steps = [vsa_cache.PagedStep(to, count, b.admitted, b.row_slot, b.runs, tables) for to, b in zip((between, lengths), blank)]
    calls = [lambda n: vsa_cache.paged_attention(q, cache, tables, n, return_lse=True),
             lambda n: vsa_cache.select_pages(q, cache, tables, n, keep=5, coarse=True)]

    def run():
        first = vsa_cache.plan_paged_step(lengths, new[0], tables, free, count, tokens=rows, out=steps[0])
        out = calls[0](first.lengths)
        second = vsa_cache.plan_paged_step(first.lengths, new[1], tables, free, count, tokens=rows, out=steps[1])
        return out, calls[1](second.lengths)
    graph = None
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = run()
    seen = []
    for i in range(14):
        if i == 9:  # some requests end and start again
            new[1][::3] = -1
        if captured:
            graph.replay()
        else:
            results = run()
        seen.append(([x.clone() for pair in results for x in pair], between.clone(), lengths.clone(), tables.clone()))
        if i == 9:
            new[1][::3] = 40
    assert lengths.max() > 640
    for got, n, n2, table in seen:
        torch.cuda.synchronize()
        want = vsa_cache.paged_attention(q, cache, table, n, return_lse=True) + vsa_cache.select_pages(q, cache, table, n2, keep=5, coarse=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    vsa_cache.check_cache_status(cache)


def test_plans_of_unequal_sizes_from_two_threads():
    """Steps of 8,192 and of 2,000 requests planned at the same time: their kernels need unequal shared memory."""
    failed = []

    def plan(requests, stream):
        ints = dict(dtype=torch.int32, device="cuda")
        with torch.cuda.stream(stream):
            n, tables, free = torch.zeros(requests, **ints), torch.zeros(requests, 1, **ints), torch.arange(requests, **ints)
            count = torch.tensor([requests], **ints)
            try:
                for _ in range(3000):
                    step = vsa_cache.plan_paged_step(n, n + 1, tables, free, count, tokens=requests)
                if step.lengths.sum().item() != requests:
                    failed.append("lengths")
            except RuntimeError as error:
                failed.append(str(error))
    threads = [threading.Thread(target=plan, args=(n, torch.cuda.Stream())) for n in (8192, 2000, 5000)]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
