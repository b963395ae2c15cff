"""Operators that answer one new token per request over a paged key/value cache: their cases, plain
forms and 64-bit results.

  plan       block tables and slot maps of a step, built on the GPU from the request lengths
  append     new key/value rows into their pages, and the pages' running sums
  select     pages that a cheap score (query . mean key of the page) selects, and the attention over the page means
  attention  one new token per request over its pages, or over the selected ones
  decode     append, select and attention with the gated merge, as a layer of a model calls them

A page holds 64 tokens of every key/value head; `tables[s, i]` is the physical page of logical page `i`
of request `s`.  Where `own` is false everything is elementary torch arithmetic; where it is true the
framework's kernels are called.
"""
import math
import random

import torch

own = False

PAGE, DIM = 64, 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
#: Key/value elements of the largest listed cache: a drawn case stays below it.
MOST_ELEMENTS = 1 << 30


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One decode step of a batch: every request gets one token, a few cross into a new page.
        {"name": "plan decode step", "op": "plan", "requests": 64, "shortest": 1, "longest": 16384, "new": 1, "ended": 3},
        # A batch of prompts enters, ragged, while old requests leave.
        {"name": "plan prompts", "op": "plan", "requests": 301, "shortest": 1, "longest": 9000, "new": 700, "ended": 40},
        # One token for each of a batch: latency.
        {"name": "append decode step", "op": "append", "requests": 64, "shortest": 1, "longest": 4096, "new": 1, "kv_heads": 8, "dtype": "bf16", "cache": "bf16"},
        # The keys and values of a 720p video of 31 x 45 x 80 latents with 2048 text tokens enter the cache.
        {"name": "append 720p context", "op": "append", "requests": 1, "shortest": 0, "longest": 0, "new": 113648, "kv_heads": 12, "dtype": "bf16", "cache": "bf16"},
        # Ragged prompts behind cached prefixes, into an 8-bit cache.
        {"name": "append prompts e4m3", "op": "append", "requests": 37, "shortest": 0, "longest": 1000, "new": 611, "kv_heads": 4, "dtype": "bf16", "cache": "e4m3"},
        # Page choice of a small batch over middling contexts.
        {"name": "select small batch", "op": "select", "requests": 4, "shortest": 500, "longest": 8000, "kv_heads": 2, "group": 4, "keep": 16, "coarse": False, "dtype": "bf16"},
        # Page choice and attention over the page means for requests that each hold a 720p video.
        {"name": "select 720p contexts", "op": "select", "requests": 16, "shortest": 111600, "longest": 113648, "kv_heads": 12, "group": 1, "keep": 178, "coarse": True, "dtype": "bf16"},
        # One short request of a model with one key/value head: nothing but latency.
        {"name": "attention one request", "op": "attention", "requests": 1, "shortest": 100, "longest": 100, "kv_heads": 1, "group": 8, "keep": 0, "dtype": "bf16", "cache": "bf16"},
        # An ordinary serving batch in half precision, lengths spread over a factor of sixty.
        {"name": "attention batch fp16", "op": "attention", "requests": 32, "shortest": 129, "longest": 8192, "kv_heads": 8, "group": 4, "keep": 0, "dtype": "fp16", "cache": "fp16"},
        # A question about one 720p video: a single long request, every head with its own keys.
        {"name": "attention 720p context", "op": "attention", "requests": 1, "shortest": 113648, "longest": 113648, "kv_heads": 12, "group": 1, "keep": 0, "dtype": "bf16", "cache": "bf16"},
        # The largest: many long requests in an 8-bit cache, seven query heads to a key/value head.
        {"name": "attention large e4m3", "op": "attention", "requests": 48, "shortest": 2000, "longest": 32768, "kv_heads": 8, "group": 7, "keep": 0, "dtype": "bf16", "cache": "e4m3"},
        # A layer of the sparse decode over 720p contexts: a tenth of the pages is kept.
        {"name": "decode 720p contexts", "op": "decode", "requests": 8, "shortest": 111600, "longest": 113648, "kv_heads": 4, "group": 3, "keep": 178, "new": 1, "dtype": "bf16", "cache": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["plan", "append", "select", "attention", "attention", "decode"])
    case = {"op": op, "requests": _log(rng, 1, 300)}
    if op == "plan":
        case |= {"shortest": rng.choice([0, 1, 63]), "longest": _log(rng, 64, 20000), "new": _log(rng, 1, 800)}
        case["ended"] = rng.randrange(0, case["requests"] // 4 + 1)
        return case
    case["kv_heads"] = rng.choice([1, 2, 3, 4, 5, 8, 12])
    case["dtype"] = rng.choice(["bf16", "fp16"])
    longest = _log(rng, 1, 120000)
    room = MOST_ELEMENTS // (case["kv_heads"] * DIM)
    if op == "append":
        case |= {"shortest": 0, "longest": min(longest, 2000), "new": _log(rng, 1, 4000), "cache": rng.choice([case["dtype"], "e4m3"])}
        most = max(1, min(case["requests"], room // (case["longest"] + case["new"] + PAGE)))
        case["requests"] = most
        return case
    case["requests"] = max(1, min(case["requests"], room // (longest + PAGE)))
    case |= {"shortest": rng.randint(max(1, longest // 50), longest), "longest": longest, "group": rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 16])}
    if op == "select":
        case |= {"keep": _log(rng, 2, 200), "coarse": rng.random() < 0.5}
    else:
        case["cache"] = rng.choice([case["dtype"], "e4m3"])
        case["keep"] = _log(rng, 2, 200) if op == "decode" or rng.random() < 0.3 else 0
    if op == "decode":
        case["new"] = 1
    return case


def _sizes(case):
    """Tokens in the cache and new tokens of every request: they go by the case alone, so that `work` knows them."""
    rng = random.Random("%(requests)d %(shortest)d %(longest)d" % case)
    low, high = case["shortest"], case["longest"]
    cached = [high] + [_log(rng, low + 1, high + 1) - 1 for _ in range(case["requests"] - 1)]
    cached = [min(max(n, low), high) for n in cached]
    new = case.get("new", 0)
    if new > 1:  # prompts: ragged
        new = [new] + [_log(rng, max(1, new // 20), new) for _ in range(case["requests"] - 1)]
    else:
        new = [new] * case["requests"]
    for i in range(case.get("ended", 0)):
        new[(i * 7 + 1) % case["requests"]] = -1
    return cached, new


def _rows(new):
    return sum(max(0, n) for n in new) + len(new) // 16


def _pages(tokens):
    return -(-tokens // PAGE)


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    cached, new = _sizes(case)
    total = [c + max(0, n) for c, n in zip(cached, new)]
    count = len(cached)
    width = max(_pages(n) for n in total) + 2

    def i32(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    # Physical pages in random order: the cached tokens' first, the rest is the free stack.
    held = [_pages(n) for n in (cached if case["op"] in ("plan", "append") else total)]
    pages = sum(_pages(n) + 1 for n in total) + 3
    order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
    before = i32([sum(held[:i]) for i in range(count)])
    col = torch.arange(width, device="cuda", dtype=torch.int32)
    mine = col[None] < i32(held)[:, None]
    tables = torch.where(mine, order[(before[:, None] + col[None]).clamp(max=pages - 1).long()], -1).contiguous()
    state = {"case": dict(case), "tables": tables, "lengths": i32(cached), "pages": pages}
    if case["op"] in ("plan", "append", "decode"):
        used = sum(held)
        # The batch is padded: the last rows belong to no request.
        state |= {"new": i32(new), "tokens": _rows(new)}
        state["free_pages"] = torch.cat([order[used:], order[:used]])  # the stack's own room is the whole pool
        state["free_count"] = i32([pages - used])
    if case["op"] == "plan":
        return state
    heads, dtype = case["kv_heads"], DTYPES[case["dtype"]]
    store = DTYPES[case.get("cache", case["dtype"])]

    def normal(*shape, dtype=dtype):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16 if dtype == torch.float8_e4m3fn else dtype)

    scales = None
    if store == torch.float8_e4m3fn:  # the largest value of a head sits near the top of the range
        scales = (torch.rand(2, heads, generator=gen, device="cuda") + 0.5) * (5.0 / 448.0)
    state["scales"] = scales
    if case["op"] == "select":
        # The sums of 64 keys and values whose mean differs from page to page.
        state["k_sum"] = torch.randn(pages, heads, DIM, generator=gen, device="cuda") * 12
        state["v_sum"] = torch.randn(pages, heads, DIM, generator=gen, device="cuda") * 12
    else:
        kv = [normal(pages, heads, PAGE, DIM, dtype=store) for _ in range(2)]
        if scales is not None:
            kv = [(x.float() / scales[i][None, :, None, None]).clamp(-448, 448).to(store) for i, x in enumerate(kv)]
        state["k"], state["v"] = kv
        state["k_sum"], state["v_sum"] = (torch.zeros(pages, heads, DIM, device="cuda") for _ in range(2))
        if case["op"] == "decode":
            for name in ("k", "v"):
                torch.sum(state[name], 2, dtype=torch.float32, out=state[name + "_sum"])
    if case["op"] != "append":
        group = case["group"]
        state["q"] = normal(count, heads * group, DIM)
        state["scale"] = DIM ** -0.5
    if case["op"] == "attention" and case["keep"]:
        # Ascending logical pages, chosen at random, for every request and key/value head.
        n = i32(held)[:, None, None]
        rank = torch.rand(count, heads, width, generator=gen, device="cuda").masked_fill(col >= n, 2.0)
        chosen = rank.argsort(-1)[..., :case["keep"]].sort(-1).values.int()
        chosen = torch.where(chosen < n, chosen, width).sort(-1).values
        chosen = torch.nn.functional.pad(chosen, (0, case["keep"] - chosen.shape[-1]), value=width)
        state["chosen"] = torch.where(chosen < width, chosen, -1).int().contiguous()
    if case["op"] in ("append", "decode"):
        state["new_k"], state["new_v"] = (normal(state["tokens"], heads, DIM) for _ in range(2))
    if case["op"] == "decode":
        state["gate"] = normal(count, heads * case["group"], DIM)
    # What a program holds through its whole life, and the plan that a step makes once for all layers.
    if case["op"] in ("append", "decode"):
        state["plan"] = _plan(state)
        state["tables"] = state["plan"]["tables"]
    if own:
        from cudnn_vsa_b200 import vsa_cache
        if case["op"] == "select":
            k = v = torch.empty(pages, heads, PAGE, DIM, dtype=dtype, device="cuda")
            state["cache"] = vsa_cache.PagedKVCache(k, v, state["k_sum"], state["v_sum"])
        else:
            pair = (None, None) if scales is None else (scales[0], scales[1])
            state["cache"] = vsa_cache.PagedKVCache(state["k"], state["v"], state["k_sum"], state["v_sum"], *pair)
        if "plan" in state:
            p = state["plan"]
            state["step"] = vsa_cache.PagedStep(p["lengths"], p["free_count"], p["admitted"], p["row_slot"], p["runs"], p["tables"])
    return state


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    op, case = state["case"]["op"], state["case"]
    if not own:
        return {"plan": _plan, "append": _append, "select": _select, "attention": _attention, "decode": _decode}[op](state)
    from cudnn_vsa_b200 import vsa, vsa_cache
    if op == "plan":
        step = vsa_cache.plan_paged_step(state["lengths"], state["new"], state["tables"], state["free_pages"], state["free_count"], tokens=state["tokens"])
        return {"lengths": step.lengths, "free_count": step.free_count, "admitted": step.admitted, "row_slot": step.row_slot,
                "runs": step.runs, "tables": step.tables, "free_pages": state["free_pages"]}
    if op == "append":
        cache = state["cache"]
        vsa_cache.append_tokens(cache, state["new_k"], state["new_v"], state["step"])
        return {"k": cache.k, "v": cache.v, "k_sum": cache.k_sum, "v_sum": cache.v_sum}
    if op == "select":
        got = vsa_cache.select_pages(state["q"], state["cache"], state["tables"], state["lengths"], keep=case["keep"], coarse=case["coarse"])
        return {"pages": got[0], "coarse": got[1]} if case["coarse"] else {"pages": got}
    if op == "attention":
        out, lse = vsa_cache.paged_attention(state["q"], state["cache"], state["tables"], state["lengths"], pages=state.get("chosen"), return_lse=True)
        return {"out": out, "lse": lse}
    cache = state["cache"]
    out = vsa.vsa_decode(state["q"], state["new_k"], state["new_v"], state["gate"], cache, state["step"], keep=case["keep"])
    return {"out": out, "k": cache.k, "v": cache.v, "k_sum": cache.k_sum, "v_sum": cache.v_sum}


# ------------------------------------------------------------------------------------------ plain forms
def _plan(state):
    """Ended requests (new < 0) give their pages back, then requests in order take pages from the stack's
    top until it is empty; a request that cannot be served keeps its length."""
    length, new, tables = state["lengths"].long(), state["new"].long(), state["tables"]
    free, count, tokens = state["free_pages"], state["free_count"].long(), state["tokens"]
    width, room, requests = tables.shape[1], free.shape[0], length.shape[0]
    col = torch.arange(width, device=length.device)
    ends, add = new < 0, new.clamp(min=0)
    total, held = length + add, (length + PAGE - 1) // PAGE
    want, after = (total + PAGE - 1) // PAGE, add.cumsum(0)
    start = after - add
    fits = ~ends & (want <= width) & ((add == 0) | (after <= tokens))
    need, back = torch.where(fits, want - held, 0), torch.where(ends, held, 0)
    place = (count + back.cumsum(0) - back)[:, None] + col
    place = torch.where(col < back[:, None], place, room)
    free = torch.cat([free, free[:1]]).scatter(0, place.flatten(), tables.flatten())[:room]
    top, taken = count + back.sum(), need.cumsum(0)
    admitted = fits & ((need == 0) | (taken <= top))
    pick = (top - 1 - (taken - need))[:, None] - (col - held[:, None])
    fresh = admitted[:, None] & (col >= held[:, None]) & (col < want[:, None])
    tables = torch.where(fresh, free[pick.clamp(0, room - 1)], tables)
    lengths = torch.where(ends, 0, torch.where(admitted, total, length))

    row = torch.arange(tokens, device=length.device)
    s = torch.searchsorted(after, row, right=True).clamp(max=requests - 1)
    at = length[s] + row - start[s]
    page = tables[s, (at // PAGE).clamp(max=width - 1)].long()
    row_slot = torch.where(admitted[s] & (row < after[s]), page * PAGE + at % PAGE, -1)

    number = torch.where(admitted & (add > 0), (total - 1) // PAGE - length // PAGE + 1, 0)
    runs_after = number.cumsum(0)
    run = torch.arange(min(tokens, tokens // PAGE + 2 * requests), device=length.device)
    s = torch.searchsorted(runs_after, run, right=True).clamp(max=requests - 1)
    logical = length[s] // PAGE + run - (runs_after - number)[s]
    first, last = torch.maximum(length[s], logical * PAGE), torch.minimum(total[s], (logical + 1) * PAGE)
    page = tables[s, logical.clamp(0, width - 1)].long()
    runs = torch.stack([start[s] + first - length[s], last - first, page, first - logical * PAGE], 1)
    runs = torch.where((run < runs_after[-1])[:, None], runs, 0)
    return {"lengths": lengths.int(), "free_count": (top - torch.where(admitted, need, 0).sum()).int().reshape(1), "admitted": admitted,
            "row_slot": row_slot, "runs": runs.int(), "tables": tables, "free_pages": free}


def _stored(x, scale, dtype):
    """A row as the cache holds it: rounded once; 8 bits hold x / scale, saturated."""
    return x if scale is None else (x.float() / scale[None, :, None]).clamp(-448.0, 448.0).to(dtype)


def _append(state):
    plan, out = state["plan"], {}
    runs = plan["runs"].long()
    slot = plan["row_slot"]
    row = torch.arange(PAGE, device=slot.device)
    touched = runs[:, 2]
    filled = torch.where(runs[:, 1] > 0, runs[:, 1] + runs[:, 3], 0)
    for i, name in enumerate(("k", "v")):
        cache, total = state[name], state[name + "_sum"]
        scale = None if state["scales"] is None else state["scales"][i]
        # Rows without a slot go to the row of the first one again, with its value.
        keep = torch.where(slot >= 0, torch.arange(slot.shape[0], device=slot.device), (slot >= 0).int().argmax())
        at = slot[keep]
        raw = cache.view(torch.uint8) if scale is not None else cache
        rows = _stored(state["new_" + name][keep], scale, cache.dtype)
        raw[at // PAGE, :, at % PAGE] = rows.view(torch.uint8) if scale is not None else rows
        values = cache[touched].float() if scale is None else raw[touched].view(cache.dtype).float() * scale[None, :, None, None]
        live = (row < filled[:, None])[:, None, :, None]
        fresh = torch.where(live, values, 0.0).sum(2)
        # Unused entries of the list name page 0: they give the first entry's page its value again.
        used = torch.where(runs[:, 1] > 0, torch.arange(runs.shape[0], device=slot.device), 0)
        total[touched[used]] = fresh[used]
        out |= {name: cache, name + "_sum": total}
    return out


def _page_scores(state, dtype):
    """Mean keys of every request's logical pages, which of them it has, and where its last pages are."""
    tables, lengths = state["tables"], state["lengths"].long()
    col = torch.arange(tables.shape[1], device=tables.device)
    held = ((lengths + PAGE - 1) // PAGE)[:, None]
    live = col < held
    size = (lengths[:, None] - col * PAGE).clamp(1, PAGE).to(dtype)
    return tables.clamp(min=0).long(), live, size, held, col


def _select(state):
    case = state["case"]
    heads, group, keep = case["kv_heads"], case["group"], case["keep"]
    q = state["q"].view(state["q"].shape[0], heads, group, DIM)
    tables, live, size, held, col = _page_scores(state, torch.float64)
    # The order of scores next to the last one kept is decided in 64 bits.
    mean = state["k_sum"][tables].double() / size[..., None, None]
    score = (mean * q.double().sum(2)[:, None]).sum(-1).transpose(1, 2)
    score = torch.where(score.isnan(), math.inf, score)
    always = ((col < 1) | (col >= held - 1)) & live
    score = torch.where(live[:, None], score, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices
    rank = (always.int() + live.int())[:, None].expand_as(score).gather(-1, order).sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, rank)[..., :keep]
    none = tables.shape[1]
    chosen = torch.where(torch.arange(order.shape[-1], device=q.device) < held[..., None], order, none).sort(-1).values
    chosen = torch.nn.functional.pad(chosen, (0, keep - chosen.shape[-1]), value=none)
    pages = torch.where(chosen < none, chosen, -1).int()
    if not case.get("coarse", True):
        return {"pages": pages}
    size = size.float()
    s = torch.einsum("shgd,sphd->shgp", q.float(), state["k_sum"][tables] / size[..., None, None]) * state["scale"]
    p, _ = _softmax(torch.where(live[:, None, None], s, -math.inf))
    coarse = torch.einsum("shgp,sphd->shgd", p, state["v_sum"][tables] / size[..., None, None])
    return {"pages": pages, "coarse": coarse.reshape(q.shape[0], heads * group, DIM)}


def _softmax(s):
    """Softmax and its log sum; a row without any entry gives zeros."""
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total), (total.log() + top).squeeze(-1)


def _attend(state, lengths, chosen):
    case = state["case"]
    heads, group = case["kv_heads"], case["group"]
    q = state["q"].view(state["q"].shape[0], heads, group, DIM).float()
    tables = state["tables"]
    if chosen is None:
        chosen = torch.arange(tables.shape[1], device=q.device, dtype=torch.int32).expand(q.shape[0], 1, -1)
    at = chosen.long() * PAGE
    at = at[..., None] + torch.arange(PAGE, device=q.device)
    live = (chosen >= 0)[..., None] & (at < lengths.long()[:, None, None, None])
    request = torch.arange(q.shape[0], device=q.device)[:, None, None]
    page = tables[request, chosen.clamp(min=0).long()].clamp(min=0).long()
    head = torch.arange(heads, device=q.device)[:, None]

    def rows(name, i):
        x = state[name]
        if state["scales"] is None:
            return x[page, head].float()
        x = x.view(torch.uint8)[page, head].view(x.dtype).float()
        return x * state["scales"][i][:, None, None, None]
    s = torch.einsum("shgd,shptd->shgpt", q, rows("k", 0)) * state["scale"]
    s = torch.where(live[:, :, None], s, -math.inf).flatten(3)
    p, lse = _softmax(s)
    out = torch.einsum("shgn,shnd->shgd", p, rows("v", 1).flatten(2, 3))
    return out.reshape(q.shape[0], heads * group, DIM), lse.reshape(q.shape[0], heads * group)


def _attention(state):
    out, lse = _attend(state, state["lengths"], state.get("chosen"))
    return {"out": out.to(state["q"].dtype), "lse": lse}


def _decode(state):
    appended = _append(state)
    now = state | {"lengths": state["plan"]["lengths"]}
    picked = _select(now)
    out, _ = _attend(now, now["lengths"], picked["pages"])
    return {"out": (out + state["gate"].float() * picked["coarse"]).to(state["q"].dtype)} | appended


# ------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The operators' definitions in 64 bits, request by request."""
    global own
    if case["op"] == "plan":
        return None
    kept, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = kept
    heads, scales = case["kv_heads"], state["scales"]
    cached, new = _sizes(case)
    decode = case["op"] == "decode"
    total = [c + n for c, n in zip(cached, new)] if decode or case["op"] == "append" else cached
    tables = state["tables"].cpu()
    result = {}
    sums = {name: state[name + "_sum"].double() for name in ("k", "v")}
    value = {}
    if case["op"] != "select":
        for i, name in enumerate(("k", "v")):
            value[name] = state[name]
            if scales is not None:
                value[name] = state[name].to(torch.float32).to(torch.float16)  # every 8-bit value has a 16-bit one
        if decode or case["op"] == "append":
            row = 0
            for s, (c, n) in enumerate(zip(cached, new)):
                if n == 0:
                    continue
                at = torch.arange(c, c + n)
                page, slot = tables[s, at // PAGE].long().cuda(), (at % PAGE).cuda()
                for i, name in enumerate(("k", "v")):
                    x = state["new_" + name][row:row + n].double()
                    if scales is not None:
                        x = (x / scales[i].double()[None, :, None]).clamp(-448, 448).to(torch.float32).to(torch.float8_e4m3fn).float()
                    value[name][page, :, slot] = x.to(value[name].dtype)
                    for logical in range(c // PAGE, _pages(c + n)):
                        p, filled = int(tables[s, logical]), min(PAGE, c + n - logical * PAGE)
                        v = value[name][p, :, :filled].double().sum(1)
                        sums[name][p] = v if scales is None else v * scales[i].double()[:, None]
                row += n
            result = {name: value[name] for name in value} | {name + "_sum": sums[name] for name in sums}
            if case["op"] == "append":
                return result
    group, scale = case["group"], DIM ** -0.5
    q = state["q"].double().view(-1, heads, group, DIM)
    outs, lses, coarses = [], [], []
    want = decode or case["op"] == "select"
    chosen = _select(state | {"lengths": torch.tensor(total, device="cuda")} | {"k_sum": sums["k"].float(), "v_sum": sums["v"].float()})["pages"].cpu() if want else state.get("chosen")
    if case["op"] == "select" and not case["coarse"]:
        return None
    for s, n in enumerate(total):
        if want:
            page = tables[s, :_pages(n)].long().cuda()
            size = torch.full((len(page),), float(PAGE), dtype=torch.float64, device="cuda")
            size[-1] = n - PAGE * (len(page) - 1)
            k, v = (sums[name][page] / size[:, None, None] for name in ("k", "v"))
            p = torch.softmax(torch.einsum("hgd,nhd->hgn", q[s], k) * scale, -1)
            coarses.append(torch.einsum("hgn,nhd->hgd", p, v).reshape(heads * group, DIM))
        if case["op"] == "select":
            continue
        for h in range(heads):
            logical = torch.arange(_pages(n)) if chosen is None else chosen[s, h].cpu()
            logical = logical[logical >= 0].long()
            at = (logical[:, None] * PAGE + torch.arange(PAGE)).flatten()
            at = at[at < n]
            page, slot = tables[s, at // PAGE].long().cuda(), (at % PAGE).cuda()
            k, v = (value[name][page, h, slot].double() for name in ("k", "v"))
            if scales is not None:
                k, v = k * scales[0, h].double(), v * scales[1, h].double()
            x = q[s, h] @ k.T * scale
            outs.append(torch.softmax(x, -1) @ v)
            lses.append(torch.logsumexp(x, -1))
    if case["op"] == "select":
        return {"pages": None, "coarse": torch.stack(coarses)}
    out = torch.stack(outs).reshape(len(total), heads * group, DIM)
    if decode:
        return {"out": out + state["gate"].double() * torch.stack(coarses)} | result
    return {"out": out, "lse": torch.stack(lses).reshape(len(total), heads * group)}


# ------------------------------------------------------------------------------------------ what it takes
def work(case):
    cached, new = _sizes(case)
    op, count = case["op"], len(cached)
    add = [max(0, n) for n in new]
    tokens = _rows(new) if op == "plan" else sum(add)
    total = [c + a for c, a in zip(cached, add)]
    if op == "plan":
        moved = sum(_pages(t) - _pages(c) if n >= 0 else _pages(c) for c, t, n in zip(cached, total, new))
        runs = min(tokens, tokens // PAGE + 2 * count)
        # lengths and new in, lengths and admitted out; a slot for every row; the list of runs; pages that change hands.
        return {"bytes": 13 * count + 8 * tokens + 16 * runs + 8 * moved, "flops": 0}
    heads = case["kv_heads"]
    each = 1 if case.get("cache") == "e4m3" else 2
    bytes_, flops = 0, 0
    if op in ("append", "decode"):
        # A new row is read and written; rows that a touched page already holds are read for its sum.
        old = sum(c % PAGE for c, a in zip(cached, add) if a)
        touched = sum((t - 1) // PAGE - c // PAGE + 1 for c, t, a in zip(cached, total, add) if a)
        bytes_ += 2 * heads * DIM * (tokens * (2 + each) + old * each + 4 * touched)
        flops += 2 * heads * DIM * (tokens + old)
    if op == "append":
        return {"bytes": bytes_ + 16 * touched, "flops": flops}
    group = case["group"]
    rows = count * heads * group
    keep = case["keep"]
    pages = sum(_pages(t) for t in total)
    if op in ("select", "decode"):
        coarse = case.get("coarse", True)
        bytes_ += pages * heads * DIM * 4 * (2 if coarse else 1) + 4 * pages + 2 * rows * DIM
        bytes_ += (4 * rows * DIM if coarse else 0) + 4 * count * heads * keep if op == "select" else 0
        flops += 2 * pages * heads * DIM * (1 + (2 * group if coarse else 0))
    if op in ("attention", "decode"):
        held = [min(t, keep * PAGE) if keep else t for t in total]
        bytes_ += 2 * sum(held) * heads * DIM * each + 2 * 2 * rows * DIM + 4 * sum(_pages(h) for h in held)
        bytes_ += 2 * rows * DIM if op == "decode" else 4 * rows
        flops += 4 * sum(held) * heads * group * DIM
    return {"bytes": bytes_, "flops": flops}
