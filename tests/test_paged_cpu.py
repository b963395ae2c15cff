"""CPU: what the paged-cache operators refuse, and what their C entry points refuse before a launch."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from cudnn_vsa_b200 import _cabi, vsa_cache
from cudnn_vsa_b200.vsa import vsa_decode
from tests import paged_reference as ref

BF16 = torch.bfloat16


def cache(pages=4, heads=2, dtype=BF16, **kw):
    return vsa_cache.build_paged_cache(pages, heads, dtype=dtype, device="cpu", **kw)


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def step(tokens=3, requests=3):
    return vsa_cache.PagedStep(i32(*[1] * requests), i32(1), torch.ones(requests, dtype=torch.bool), torch.zeros(tokens, dtype=torch.int64),
                               torch.zeros(tokens, 4, dtype=torch.int32), torch.zeros(requests, 2, dtype=torch.int32))


def test_cache_refusals():
    with pytest.raises(ValueError, match="bfloat16, float16 or float8"):
        cache(dtype=torch.float32)
    with pytest.raises(ValueError, match="positive integer"):
        cache(pages=0)
    with pytest.raises(ValueError, match="positive integer"):
        cache(heads=True)
    with pytest.raises(ValueError, match="needs k_scale and v_scale"):
        cache(dtype=torch.float8_e4m3fn)
    one = torch.ones(2)
    assert cache(dtype=torch.float8_e4m3fn, k_scale=one, v_scale=one).kv_heads == 2
    with pytest.raises(ValueError, match="belong to an e4m3"):
        cache(k_scale=one, v_scale=one)
    with pytest.raises(ValueError, match="needs k_scale"):
        cache(dtype=torch.float8_e4m3fn, k_scale=one, v_scale=torch.ones(3))
    c = cache()
    with pytest.raises(ValueError, match=r"\[pages, kv_heads, 64, 128\]"):
        vsa_cache.PagedKVCache(c.k[..., :64], c.v[..., :64], c.k_sum, c.v_sum)
    with pytest.raises(ValueError, match="identical"):
        vsa_cache.PagedKVCache(c.k, c.v[:3], c.k_sum, c.v_sum)
    with pytest.raises(ValueError, match="k_sum"):
        vsa_cache.PagedKVCache(c.k, c.v, c.k_sum.double(), c.v_sum)
    with pytest.raises(ValueError, match="contiguous"):
        vsa_cache.PagedKVCache(c.k.transpose(0, 1).contiguous().transpose(0, 1), c.v, c.k_sum, c.v_sum)
    vsa_cache.check_cache_status(c)
    c.status.fill_(200)
    with pytest.raises(RuntimeError, match="outside the cache"):
        vsa_cache.check_cache_status(c)


def test_plan_refusals():
    good = dict(lengths=i32(1, 2), new=i32(1, 1), tables=torch.zeros(2, 3, dtype=torch.int32), free_pages=i32(0, 1), free_count=i32(2))

    def plan(tokens=2, rows_per_request=None, out=None, **change):
        g = good | change
        return vsa_cache.plan_paged_step(g["lengths"], g["new"], g["tables"], g["free_pages"], g["free_count"], tokens=tokens,
                                         rows_per_request=rows_per_request, out=out)
    for change in ({"lengths": i32()}, {"lengths": torch.tensor([1, 2])}, {"new": i32(1)}, {"tables": torch.zeros(3, 3, dtype=torch.int32)},
                   {"tables": torch.zeros(2, 3, dtype=torch.int32).T.contiguous().T}, {"tables": torch.zeros(2, 0, dtype=torch.int32)},
                   {"free_pages": i32()}, {"free_count": i32(1, 2)}, {"tokens": 0}, {"tokens": 2.0}, {"tokens": True}, {"tokens": 2 ** 31},
                   {"rows_per_request": 0}, {"out": 3}):
        with pytest.raises(ValueError):
            plan(**change)
    many = torch.zeros(8193, dtype=torch.int32)
    with pytest.raises(ValueError, match="at most 8192"):
        plan(lengths=many, new=many, tables=torch.zeros(8193, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="out.row_slot"):
        plan(out=vsa_cache.PagedStep(i32(0, 0), i32(0), torch.ones(2, dtype=torch.bool), torch.zeros(3, dtype=torch.int64),
                                     torch.zeros(2, 4, dtype=torch.int32), good["tables"]))
    with pytest.raises(ValueError, match="CUDA"):
        plan()


def test_append_refusals():
    c, s = cache(), step()
    x = torch.zeros(3, 2, 128, dtype=BF16)
    for k, v, match in ((x[:2], x, "k must have shape"), (x, x[:, :1], "v must have shape"), (x.float(), x, "bfloat16"), (x, x.half(), "v must be bfloat16"),
                        (x[..., :64], x, "k must have shape"), (torch.zeros(3, 2, 256, dtype=BF16)[..., ::2], x, "contiguous heads"),
                        (torch.zeros(3, 2, 132, dtype=BF16)[..., :128], x, "multiples of 8"), (torch.zeros(3, 2, 136, dtype=BF16)[..., 1:129], x, "aligned")):
        with pytest.raises(ValueError, match=match):
            vsa_cache.append_tokens(c, k, v, s)
    with pytest.raises(ValueError, match="PagedStep"):
        vsa_cache.append_tokens(c, x, x, None)
    with pytest.raises(ValueError, match="PagedKVCache"):
        vsa_cache.append_tokens(c.k, x, x, s)
    with pytest.raises(ValueError, match="no backward"):
        vsa_cache.append_tokens(c, x.clone().requires_grad_(), x, s)
    with pytest.raises(ValueError, match="CUDA"):
        vsa_cache.append_tokens(c, x, x, s)


def test_select_and_attention_refusals():
    c = cache()
    q, tables, lengths = torch.zeros(3, 4, 128, dtype=BF16), torch.zeros(3, 2, dtype=torch.int32), i32(1, 2, 3)
    select, attend = vsa_cache.select_pages, vsa_cache.paged_attention
    for kw in ({}, {"keep": 0}, {"keep": 1}, {"keep": 5, "first": 3, "last": 3}, {"keep": 3, "first": -1}, {"keep": 2.0}, {"keep": True},
               {"keep": 3, "scale": float("nan")}, {"keep": 3, "scale": -1.0}):
        with pytest.raises(ValueError):
            select(q, c, tables, lengths, **kw)
    with pytest.raises(ValueError, match="at most 24576"):
        select(q, c, torch.zeros(3, 24577, dtype=torch.int32), lengths, keep=3)
    for call in (lambda *a: select(*a, keep=3), attend):
        with pytest.raises(ValueError, match="multiple"):
            call(q[:, :3], c, tables, lengths)
        with pytest.raises(ValueError, match="cache's dtype"):
            call(q.half(), c, tables, lengths)
        with pytest.raises(ValueError, match="one row for each"):
            call(q, c, tables[:2], lengths)
        with pytest.raises(ValueError, match="lengths"):
            call(q, c, tables, lengths.long())
        with pytest.raises(ValueError, match="rows, heads, 128"):
            call(q[0], c, tables, lengths)
        with pytest.raises(ValueError, match="no backward"):
            call(q.clone().requires_grad_(), c, tables, lengths)
        with pytest.raises(ValueError, match="CUDA"):
            call(q, c, tables, lengths)
    for kw in ({"pages": torch.zeros(3, 2, 0, dtype=torch.int32)}, {"pages": torch.zeros(3, 4, 2, dtype=torch.int32)}, {"pages": torch.zeros(3, 2, 2)},
               {"gate": q}, {"coarse": q.float()}, {"gate": q, "coarse": q}, {"gate": q[:2], "coarse": q.float()}, {"scale": float("inf")}):
        with pytest.raises(ValueError):
            attend(q, c, tables, lengths, **kw)
    with pytest.raises(ValueError, match="no backward"):
        attend(q, c, tables, lengths, gate=q, coarse=q.float().requires_grad_())
    with pytest.raises(ValueError, match="at most 8192"):
        attend(torch.zeros(8193, 2, 128, dtype=BF16), c, torch.zeros(8193, 1, dtype=torch.int32), torch.zeros(8193, dtype=torch.int32))
    x = torch.zeros(3, 2, 128, dtype=BF16)
    with pytest.raises(ValueError, match="CUDA"):
        vsa_decode(q, x, x, q, c, step(), keep=3)


def test_entry_points_refuse_bad_arguments_on_the_host():
    lib = _cabi.load()
    block = (ctypes.c_char * 64)()
    p = (ctypes.addressof(block) + 15) // 16 * 16  # any aligned host address: nothing is launched

    def call(name, args, **change):
        """The entry point on the packed arguments, with argument `at` replaced by `bad`."""
        args = [change["bad"] if i in change.get("at", ()) else x for i, x in enumerate(args)]
        return getattr(lib, name)(vsa_cache._PACK[name](*(0 if x is None else x for x in args)))
    plan = [p, p, p, 4, 4, 2, p, 8, p, 16, 0, p, p, p, p, p, 6, None]
    for i, bad in ((0, None), (3, 3), (4, 0), (5, 0), (7, 0), (9, 0), (10, -1), (15, p + 4), (16, 0)):
        assert call("vsa_paged_plan", plan, at=(i,), bad=bad) == 1, i
    assert call("vsa_paged_plan", plan, at=(5,), bad=8193) == 5
    assert call("vsa_paged_plan", plan, at=(9,), bad=2 ** 40) == 1
    for name in vsa_cache._PACK:
        assert getattr(lib, name)(None) == 1, name
    append = [p, p, 256, 128, 256, 128, 0, 3, p, p, 0, p, p, None, None, p, 3, 4, 2, None, None]
    for i, bad in ((0, None), (0, p + 8), (2, 12), (3, -8), (6, 2), (10, 1), (10, 2), (16, 0), (17, 0), (18, 0)):
        assert call("vsa_paged_append", append, at=(i,), bad=bad) == 1, (i, bad)
    size = lib.vsa_paged_select_workspace_bytes(3, 2, 2, 200, 1, 1)
    assert size > lib.vsa_paged_select_workspace_bytes(3, 2, 2, 200, 1, 0) > 0
    assert lib.vsa_paged_select_workspace_bytes(3, 2, 2, 2, 1, 1) == 0  # short requests are scored where pages are chosen
    select = [p, 512, 128, 0, p, p, p, 200, 200, p, 3, 2, 2, 4, 3, 1, 1, 0.1, p, p, p, size, None, None]
    for i, bad in ((20, None), (20, p + 8), (21, size - 1), (0, None), (1, 4), (3, 3), (7, 1), (8, 0), (10, 0), (12, 0), (14, 1), (15, -1)):
        assert call("vsa_paged_select", select, at=(i,), bad=bad) == 1, (i, bad)
    assert call("vsa_paged_select", select, at=(7, 8), bad=30000) == 5
    size = lib.vsa_paged_workspace_bytes(3, 2, 2, 20, 0)
    assert size > 0 and lib.vsa_paged_workspace_bytes(3, 2, 2, 2, 0) == 0  # short tables are not split
    attend = [p, 512, 128, 0, p, p, 0, None, None, 4, p, 20, 20, p, 3, 2, 2, None, 0, None, 0, 0, None, 0.1, p, None, p, size, None, None]
    for i, bad in ((0, None), (2, 4), (3, 2), (6, 1), (6, 2), (9, 0), (12, 0), (14, 0), (16, 0), (19, p), (24, None), (26, None), (27, size - 1)):
        assert call("vsa_paged_attention", attend, at=(i,), bad=bad) == 1, (i, bad)
    assert call("vsa_paged_attention", attend, at=(9,), bad=2 ** 25) == 5
    size = lib.vsa_paged_decode_workspace_bytes(3, 2, 2, 2, 3, 1, 0)
    assert size > lib.vsa_paged_decode_workspace_bytes(3, 2, 2, 2, 0, 0, 0) > 0
    decode = [p, 512, 128, p, p, 256, 128, 256, 128, 0, 3, p, p, 0, p, p, None, None, 4, 2, 2, p, 3, p, 2, 2, p, 3, 3, 1, 1, p, 512, 128,
              0.1, p, p, size, None, None]
    for i, bad in ((3, None), (9, 2), (19, 0), (20, 0), (25, 0), (27, 0), (28, -1), (36, None), (37, size - 1)):
        assert call("vsa_paged_decode", decode, at=(i,), bad=bad) == 1, (i, bad)


@pytest.mark.parametrize("scale", [1e39, 2.0 ** 127 * 1.0001, -1e-9, float("inf"), float("nan")])
def test_scales_that_are_no_fp32_numbers_are_refused(scale):
    q, x, tables, lengths = torch.zeros(3, 4, 128, dtype=BF16), torch.zeros(3, 2, 128, dtype=BF16), torch.zeros(3, 2, dtype=torch.int32), i32(1, 2, 3)
    for call in (lambda s: vsa_cache.paged_attention(q, cache(), tables, lengths, scale=s), lambda s: vsa_decode(q, x, x, q, cache(), step(), scale=s),
                 lambda s: vsa_cache.select_pages(q, cache(), tables, lengths, coarse=True, scale=s)):
        with pytest.raises(ValueError, match="scale must be"):
            call(scale)
        with pytest.raises(ValueError, match="CUDA"):
            call(2.0 ** 127)


def test_gradients_and_tangents_are_refused():
    """Of every floating-point tensor of a call: the operators have no backward and no forward-mode derivative."""
    one = torch.ones(2)
    tables, lengths, s = torch.zeros(3, 2, dtype=torch.int32), i32(1, 2, 3), step()

    def inputs():
        q, x = torch.zeros(3, 4, 128, dtype=BF16), torch.zeros(3, 2, 128, dtype=BF16)
        c = cache(dtype=torch.float8_e4m3fn, k_scale=one.clone(), v_scale=one.clone())
        return {"q": q, "k": x, "v": x.clone(), "gate": q.clone(), "coarse": q.float(), "k_sum": c.k_sum, "v_sum": c.v_sum, "k_scale": c.k_scale,
                "v_scale": c.v_scale, "k_cache": c.k, "v_cache": c.v}

    def calls(t):
        c = vsa_cache.PagedKVCache(t["k_cache"], t["v_cache"], t["k_sum"], t["v_sum"], t["k_scale"], t["v_scale"])
        return {"append": lambda: vsa_cache.append_tokens(c, t["k"], t["v"], s),
                "select": lambda: vsa_cache.select_pages(t["q"], c, tables, lengths, keep=3),
                "attend": lambda: vsa_cache.paged_attention(t["q"], c, tables, lengths, gate=t["gate"], coarse=t["coarse"]),
                "decode": lambda: vsa_decode(t["q"], t["k"], t["v"], t["gate"], c, s, keep=3)}
    takes = {"append": {"k", "v"}, "select": {"q"}, "attend": {"q", "gate", "coarse"}, "decode": {"q", "k", "v", "gate"}}
    held = ["k_sum", "v_sum", "k_scale", "v_scale"]
    for name in ("q", "k", "v", "gate", "coarse", *held):
        for op, used in takes.items():
            match = "no backward" if name in used or name in held else "CUDA"
            t = inputs()
            t[name].requires_grad_()
            with pytest.raises(ValueError, match=match):
                calls(t)[op]()
            with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
                calls(t)[op]()
            t = inputs()
            with forward_ad.dual_level():
                t[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
                with pytest.raises(ValueError, match=match):
                    calls(t)[op]()


def test_sizes_that_are_taken_and_refused():
    """2,048 requests with tables of 16,384 columns and eight by eight heads are taken; the limits are refused by name."""
    c = cache(heads=8)
    big = torch.empty(1, 1, 128, dtype=BF16)

    def call(which, requests, heads, width):
        q, tables, lengths = big.expand(requests, heads, 128), torch.empty(requests, width, dtype=torch.int32), torch.empty(requests, dtype=torch.int32)
        with pytest.raises(ValueError) as error:
            which(q, c, tables, lengths)
        return str(error.value)
    for which in (vsa_cache.paged_attention, lambda *a: vsa_cache.select_pages(*a, coarse=True)):
        assert "CUDA" in call(which, 2048, 64, 16384)  # all that is wrong is the device
        assert "below 2**31" in call(which, 8192, 72, 16384)
        assert "2**25 - 1 columns" in call(which, 1, 8, 2 ** 25)
    with pytest.raises(ValueError, match="at most 65535"):
        vsa_cache.append_tokens(cache(1, 65536), torch.zeros(3, 65536, 128, dtype=BF16), torch.zeros(3, 65536, 128, dtype=BF16), step())
    with pytest.raises(ValueError, match="2\\*\\*25 - 1 columns"):
        vsa_cache.plan_paged_step(i32(1), i32(1), torch.empty(1, 2 ** 25, dtype=torch.int32), i32(0), i32(1), tokens=1)
    # The entry points: 5 = too large; a workspace that is a byte short keeps the rest from a launch.
    lib = _cabi.load()
    block = (ctypes.c_char * 64)()
    p = (ctypes.addressof(block) + 15) // 16 * 16
    size = lib.vsa_paged_workspace_bytes(2048, 8, 8, 16384, 0)
    attend = [p, 8192, 128, 0, p, p, 0, 0, 0, 4, p, 16384, 16384, p, 2048, 8, 8, 0, 0, 0, 0, 0, 0, 0.1, p, 0, p, size - 1, 0, 0]
    assert lib.vsa_paged_attention(vsa_cache._PACK["vsa_paged_attention"](*attend)) == 1
    attend[14:17] = 8192, 8, 9
    assert lib.vsa_paged_attention(vsa_cache._PACK["vsa_paged_attention"](*attend)) == 5
    size = lib.vsa_paged_select_workspace_bytes(2048, 8, 8, 16384, 1, 1)
    select = [p, 8192, 128, 0, p, p, p, 16384, 16384, p, 2048, 8, 8, 4, 3, 1, 1, 0.1, p, p, p, size - 1, 0, 0]
    assert lib.vsa_paged_select(vsa_cache._PACK["vsa_paged_select"](*select)) == 1
    select[10:13] = 8192, 8, 9
    assert lib.vsa_paged_select(vsa_cache._PACK["vsa_paged_select"](*select)) == 5


def test_plan_entry_point_refuses_a_list_of_runs_that_may_be_too_short():
    """A step that drops runs would leave slots unwritten: min(tokens, tokens / 64 + 2 * requests) entries, or a refusal."""
    lib = _cabi.load()
    block = (ctypes.c_char * 64)()
    p = (ctypes.addressof(block) + 15) // 16 * 16
    for tokens, requests in ((16, 2), (3, 2), (1, 1), (6400, 30), (2 ** 31 - 1, 8192)):
        most = min(tokens, tokens // 64 + 2 * requests)
        for runs in (1, most - 1):
            if 0 < runs < most:
                args = (p, p, p, 4, 4, requests, p, 8, p, tokens, 0, p, p, p, p, p, runs, 0)
                assert lib.vsa_paged_plan(vsa_cache._PACK["vsa_paged_plan"](*args)) == 1, (tokens, requests, runs)


def test_plain_plan_of_a_small_step():
    """The plain form that the GPU tests compare with, on a step worked out by hand."""
    got = ref.plan([64, 10, 70], [1, 60, -1], [[5, -1], [6, -1], [1, 2]], [3, 4, 0, 0, 0, 0, 0], 2, 62)
    assert got["lengths"] == [65, 70, 0] and got["free_count"] == [2] and got["admitted"] == [True, True, False]
    assert got["tables"] == [[5, 2], [6, 1], [1, 2]] and got["free_pages"][:4] == [3, 4, 1, 2]
    assert got["row_slot"][0] == 2 * 64 and got["row_slot"][1] == 6 * 64 + 10 and got["row_slot"][55] == 64 and got["row_slot"][61] == -1
    assert got["runs"][:4] == [[0, 1, 2, 0], [1, 54, 6, 10], [55, 6, 1, 0], [0, 0, 0, 0]]
