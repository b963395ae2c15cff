"""GPU: how exactly paged attention holds its probabilities, and that no key is lost or counted twice.

An output in 16 bits hides an error below its own half step.  So the attention is called with a gate of
ones and `coarse = -o`, where `o` is the 64-bit result rounded to FP32: the merge forms `fine - o` in
FP32, which is exact for numbers this close, and what comes back is the error itself, off by a half
step of its own and of `o`.

Where an error is bounded by the scores, a query has one value that is not zero: its products are
exact, a score is off by the eight half steps of scaling, subtracting the maximum and the argument of
the exponential, whose own error is below 2^-22.

Sums: a warp adds 16 keys at a time to its running sum (once for every term of the probabilities, at
most three, cut instead of rounded: two half steps each), every page a split of the work can give it at most;
then the results of up to 16 warps and of the workers that share the request are added.
"""
import math

import pytest
import torch

from cudnn_vsa_b200 import vsa_cache
from tests import paged_reference as ref
from tests.test_gpu_paged import BF16, E4M3, FP16, SCALE, TABLES, attention_case

pytestmark = pytest.mark.gpu

KINDS = [(BF16, BF16), (FP16, FP16), (BF16, E4M3), (FP16, E4M3)]
# What the terms of a probability leave: two of FP16 (cut, then rounded); three of BF16 hold all 24 bits.
TERMS = {FP16: 2.0 ** -21, E4M3: 2.0 ** -21, BF16: 0.0}


def additions(cache, lengths, group):
    """FP32 half steps of the sums over a request's keys: see the top."""
    pages = [ref.pages_of(n) for n in lengths]
    share = -(-sum(pages) * cache.kv_heads * -(-group // 32) // 148) + 1  # pages of a worker
    # Requests of few pages are not split over workers: 16 keys of every page in turn, at least four warps.
    steps = max(share, min(max(pages), 32))
    return 2 * 3 * steps + 16 + min(max(pages), 160) + 8


def residual(q, cache, tables, n, o, scale=None):
    """`fine - o`, and what the rounding of the residual and of `o` add to it."""
    one = torch.ones_like(q)
    got = vsa_cache.paged_attention(q, cache, tables, n, gate=one, coarse=-o.float().cuda(), scale=scale).cpu().double()
    return got, ref.HALF_STEP[q.dtype] * got.abs() + ref.FP32 * o.abs() + (2.0 ** -25 if q.dtype == FP16 else 0.0)


@pytest.mark.parametrize("extra", TABLES)
@pytest.mark.parametrize("dtype,store", KINDS)
@pytest.mark.parametrize("heads,group,lengths", [
    (2, 8, [1, 2, 3, 5, 17]), (3, 3, [64, 65, 7, 100]), (1, 16, [2, 200, 3]), (1, 33, [3, 90]), (4, 7, [2, 3, 4, 5, 6, 7, 8, 9]), (1, 2, [1500, 4])])
def test_probabilities_keep_their_bits(dtype, store, heads, group, lengths, extra):
    cache, q, tables, n = attention_case(dtype, store, heads, group, lengths, 70 + heads * group, extra)
    at = torch.arange(q.shape[0] * q.shape[1], device="cuda").view(q.shape[:2]) * 5 % 128
    q = torch.zeros_like(q).scatter_(2, at[..., None], (q[..., :1] * 8).clamp(-20, 20))
    # Values of one sign: an error of the probabilities does not cancel in the sums.
    cache.v.copy_(cache.v.float().abs().to(store).view_as(cache.v))
    o, lse, size, spread = ref.attention(q, cache, tables, n)
    got, rounding = residual(q, cache, tables, n, o)
    exponent = 8 * ref.FP32 * spread[..., None] * SCALE + 2.0 ** -22
    floor = 2.0 ** -34 * max(lengths) * 8 if store == FP16 else 0.0  # the least FP16 number stands in for less
    bound = size * (TERMS[store] + 2 * exponent + 2 * additions(cache, lengths, group) * ref.FP32) + floor + rounding
    assert (got.abs() <= bound).all(), f"off by {(got.abs() / bound).max():.3g} of the bound"


@pytest.mark.parametrize("extra", TABLES)
@pytest.mark.parametrize("dtype,store", KINDS)
@pytest.mark.parametrize("heads,group,lengths", [
    (1, 1, [20000]), (12, 1, [5000]), (2, 4, [1, 63, 64, 65, 900, 8191]), (1, 9, [3000, 17, 4099]), (1, 20, [2500, 1111]),
    (3, 2, [700, 0, 320, 65, 6000, 1] * 8), (2, 1, [30, 70, 130, 1000] * 100)])
def test_every_key_counts_once(dtype, store, heads, group, lengths, extra):
    """All scores alike: the output is the mean of the values, whole numbers whose sums are exact.  Every
    group of 16 keys has a value of its own, and so has every key of a group, each as bits over the dims."""
    pages = sum(ref.pages_of(x) for x in lengths) + 2
    gen = torch.Generator().manual_seed(len(lengths) + heads)
    one = torch.ones(heads, device="cuda")
    cache = vsa_cache.build_paged_cache(pages, heads, dtype=store, **({"k_scale": one, "v_scale": one} if store == E4M3 else {}))
    row = torch.arange(pages * heads * 64)
    code = torch.cat([(row[:, None] // 16 >> torch.arange(32)) & 1, (row[:, None] % 16 == torch.arange(16)).long()], 1)
    code = torch.cat([code, 1 - code, code[:, :32]], 1).float().view(pages, heads, 64, 128)  # every row counts in half the dims
    cache.v.copy_(code.cuda())
    cache.k.copy_(torch.randn(cache.k.shape, generator=gen).cuda().clamp(-4, 4))
    tables = ref.make_tables(lengths, pages, gen, extra)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn(len(lengths), heads * group, 128, generator=gen).to(dtype).cuda()
    want = torch.zeros(len(lengths), heads, 128, dtype=torch.float64)
    for s, length in enumerate(lengths):
        rows = code[tables[s, :ref.pages_of(length)].cpu().long()].double().transpose(1, 2).reshape(-1, heads, 128)[:length]
        want[s] = rows.sum(0) / max(1, length)
    o = want.repeat_interleave(group, 1)
    got, rounding = residual(q, cache, tables, n, o, scale=0.0)
    # A warp's sums are exact.  Up to 16 warps' are then added, each with its factor 1 / sum (one rounding) in a
    # product and sum of one half step: 17 half steps, 3 for the merge and, of a split request, the second quotient.
    # A lost key changes the output by 1 / length of it, 800 half steps of 20,000 keys.  And FP16's least number.
    bound = o.abs() * (20 * ref.FP32) + rounding + (2.0 ** -33 if store == FP16 else 0.0)
    assert (got.abs() <= bound).all(), f"off by {(got.abs() / bound.clamp_min(1e-30)).max():.3g} of the bound"
    lse = vsa_cache.paged_attention(q, cache, tables, n, scale=0.0, return_lse=True)[1].cpu().double()
    for s, length in enumerate(lengths):
        if length == 0:
            assert (lse[s] == -math.inf).all()
        else:  # four half steps of a base-2 logarithm of at most log2(length) + 11, and of its parts
            assert ((lse[s] - math.log(length)).abs() <= 4 * ref.FP32 * (math.log2(length) + 22)).all(), length


@pytest.mark.parametrize("extra", TABLES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("least", [-math.inf, -30000.0])
@pytest.mark.parametrize("length", [3, 100, 64 * 40 + 36])
@pytest.mark.parametrize("which", ["odd rows", "first pages", "last pages"])
def test_keys_without_weight_do_not_count(dtype, least, length, which, extra):
    """Scores of -infinity, or so low that exp gives zero, leave their values out, the largest ones too: they might as well be zero."""
    cache, q, tables, n = attention_case(dtype, dtype, 1, 4, [length], 90, extra)
    pages = tables[0, :ref.pages_of(length)].long()
    some = {"odd rows": slice(1, None, 2), "first pages": slice(None), "last pages": slice(None)}[which]
    pages = {"odd rows": pages, "first pages": pages[:-1], "last pages": pages[1:]}[which]
    rows = torch.arange(64, device="cuda")[some]
    cache.k[pages[:, None], 0, rows[None], 3] = least
    q[0, :, 3] = 1.0
    results = []
    for value in (0.0, torch.finfo(dtype).max):
        cache.v[pages[:, None], 0, rows[None]] = value
        results.append(vsa_cache.paged_attention(q, cache, tables, n, return_lse=True))
    (want, lse), (got, lse2) = results
    assert want.isfinite().all() and torch.equal(got, want) and torch.equal(lse, lse2)


@pytest.mark.parametrize("extra", TABLES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("length", [100, 3000, 20000])
def test_the_largest_values_do_not_overflow(dtype, length, extra):
    """All values at most the type's largest: so is their weighted mean, though their sum is not an FP32 number."""
    cache, q, tables, n = attention_case(dtype, dtype, 1, 4, [length], 91, extra)
    most = torch.finfo(dtype).max
    cache.v.copy_(torch.where(cache.v > 0, most, most / 2))
    q[:, 2:] *= 8
    o, lse, size, spread = ref.attention(q, cache, tables, n)
    out = vsa_cache.paged_attention(q, cache, tables, n).cpu().double()
    # 136 FP32 half steps a score, twice; the sums, to which hardly any of these keys adds a rounding beyond its own.
    bound = ref.HALF_STEP[dtype] * o.abs() + size * (2 * 136 * ref.FP32 * spread[..., None] * SCALE + 2 * additions(cache, [length], 4) * ref.FP32 + 2.0 ** -21)
    assert ((out - o).abs() <= bound).all()


@pytest.mark.parametrize("extra", TABLES)
@pytest.mark.parametrize("length", [3, 100, 64 * 40 + 36])
def test_keys_of_next_to_no_weight_in_an_fp16_cache(length, extra):
    """Weights of exp(-40) and less, far below FP16's smallest number, do not count as that number: their values of up to
    65,504 add less than 2^-57 * 2^16 * 1,300 keys, nothing that a result of FP16 could show."""
    cache, q, tables, n = attention_case(FP16, FP16, 1, 4, [length], 92, extra)
    pages, rows = tables[0, :ref.pages_of(length)].long(), torch.arange(1, 64, 2, device="cuda")
    q[0, :, 3] = 1.0
    cache.k[pages, :, :, 3] = 0.0
    cache.k[pages[:, None], 0, rows[None], 3] = -60.0 / SCALE  # less the spread of the other scores, at most 20
    results = []
    for value in (0.0, torch.finfo(FP16).max):
        cache.v[pages[:, None], 0, rows[None]] = value
        results.append(vsa_cache.paged_attention(q, cache, tables, n))
    assert results[0].isfinite().all() and torch.equal(*results)
