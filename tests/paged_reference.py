"""Plain 64-bit forms of the paged-cache operators, request by request, and seeded inputs for them."""
import math

import torch

PAGE, DIM = 64, 128
# Half a step of each type, relative to the value.
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4}
FP32 = 2.0 ** -24


def pages_of(tokens):
    return -(-tokens // PAGE)


def plan(lengths, new, tables, free, count, tokens, rows_per_request=None):
    """Lists in, dict of lists out: the step, one request after the other."""
    requests, width = len(lengths), len(tables[0])
    tables, free = [list(t) for t in tables], list(free)
    out_lengths, admitted = list(lengths), [False] * requests
    for s in range(requests):
        if new[s] < 0:
            for i in range(pages_of(lengths[s])):
                free[count] = tables[s][i]
                count += 1
            out_lengths[s] = 0
    row_slot, runs = [-1] * tokens, []
    row, asked, top = 0, 0, count
    for s in range(requests):
        if new[s] < 0:
            continue
        start = row if rows_per_request is None else s * rows_per_request
        row += new[s]
        total, held = lengths[s] + new[s], pages_of(lengths[s])
        if pages_of(total) > width or (new[s] and start + new[s] > tokens) or (rows_per_request is not None and new[s] > rows_per_request):
            continue
        need = pages_of(total) - held
        if need:
            asked += need
            if asked > top:
                continue
        admitted[s] = True
        out_lengths[s] = total
        for i in range(held, held + need):
            count -= 1
            tables[s][i] = free[count]
        for t in range(new[s]):
            at = lengths[s] + t
            row_slot[start + t] = tables[s][at // PAGE] * PAGE + at % PAGE
            if t == 0 or at % PAGE == 0:
                runs.append([start + t, 0, tables[s][at // PAGE], at % PAGE])
            runs[-1][1] += 1
    most = min(tokens, tokens // PAGE + 2 * requests)
    assert len(runs) <= most
    return {"lengths": out_lengths, "free_count": [count], "admitted": admitted, "row_slot": row_slot, "tables": tables,
            "free_pages": free, "runs": runs + [[0, 0, 0, 0]] * (most - len(runs))}


def values(x, scale):
    """Cached ``[.., kv_heads, rows, 128]`` values in 64 bits."""
    x = x.float().double() if x.dtype == torch.float8_e4m3fn else x.double()
    return x if scale is None else x * scale.double()[:, None, None]


def stored(x, scale, dtype):
    """Rows ``[tokens, kv_heads, 128]`` as the cache holds them."""
    return x if scale is None else (x.float() / scale[None, :, None]).clamp(-448, 448).to(dtype)


def attention(q, cache, tables, lengths, pages=None, scale=DIM ** -0.5):
    """``(out, lse, size, spread)`` in 64 bits on the CPU: ``size`` is sum_p |v| per output element and
    ``spread`` the largest sum_d |q_d k_d| of a query row, the magnitudes that rounding errors go by."""
    k, v = (values(x.cpu(), None if s is None else s.cpu()) for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    q, tables, lengths = q.cpu().double(), tables.cpu().tolist(), lengths.cpu().tolist()
    requests, heads = q.shape[0], k.shape[1]
    group = q.shape[1] // heads
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    spread = torch.zeros(q.shape[:2], dtype=torch.float64)
    for s in range(requests):
        n = max(0, lengths[s])
        for h in range(heads):
            logical = list(range(pages_of(n))) if pages is None else [int(i) for i in pages[s, h] if 0 <= int(i) < pages_of(n)]
            logical = [i for i in logical if 0 <= tables[s][i] < k.shape[0]]
            if not logical:
                continue
            ks = torch.cat([k[tables[s][i], h, :min(PAGE, n - i * PAGE)] for i in logical])
            vs = torch.cat([v[tables[s][i], h, :min(PAGE, n - i * PAGE)] for i in logical])
            rows = q[s, h * group:(h + 1) * group]
            x = rows @ ks.T * scale
            p = torch.softmax(x, -1)
            at = slice(h * group, (h + 1) * group)
            out[s, at], lse[s, at] = p @ vs, torch.logsumexp(x, -1)
            size[s, at] = p @ vs.abs()
            spread[s, at] = (rows.abs() @ ks.abs().T).amax(-1)
    return out, lse, size, spread


def scores(q, k_sum, table, length, heads):
    """64-bit page scores of one request, ``[kv_heads, pages]``; NaN counts as +inf."""
    n = pages_of(length)
    page = torch.tensor(table[:n], dtype=torch.long)
    tokens = torch.tensor([min(PAGE, length - i * PAGE) for i in range(n)], dtype=torch.float64)
    group = q.shape[0] // heads
    summed = q.double().view(heads, group, DIM).sum(1)
    s = (k_sum[page].double() * summed[None]).sum(-1).T / tokens
    return torch.where(s.isnan(), math.inf, s)


def select(q, k_sum, tables, lengths, heads, keep, first=1, last=1):
    q, k_sum, tables, lengths = q.cpu(), k_sum.cpu(), tables.cpu().tolist(), lengths.cpu().tolist()
    result = torch.full((q.shape[0], heads, keep), -1, dtype=torch.int32)
    for s, length in enumerate(lengths):
        n = pages_of(length)
        if n == 0:
            continue
        table = scores(q[s], k_sum, tables[s], length, heads)
        for h in range(heads):
            def rank(i):
                always = i < first or i >= n - last
                return (not always, -table[h, i].item() if not always else 0, i)
            chosen = sorted(sorted(range(n), key=rank)[:keep])
            result[s, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return result


def coarse(q, k_sum, v_sum, tables, lengths, heads, scale=DIM ** -0.5):
    """``(out, size, spread)`` as for :func:`attention`."""
    q, tables, lengths = q.cpu().double(), tables.cpu().tolist(), lengths.cpu().tolist()
    k_sum, v_sum = k_sum.cpu().double(), v_sum.cpu().double()
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    spread = torch.zeros(q.shape[:2], dtype=torch.float64)
    group = q.shape[1] // heads
    for s, length in enumerate(lengths):
        n = pages_of(length)
        if n == 0:
            continue
        page = torch.tensor(tables[s][:n], dtype=torch.long)
        tokens = torch.tensor([min(PAGE, length - i * PAGE) for i in range(n)], dtype=torch.float64)
        for h in range(heads):
            ks, vs = k_sum[page, h] / tokens[:, None], v_sum[page, h] / tokens[:, None]
            at = slice(h * group, (h + 1) * group)
            p = torch.softmax(q[s, at] @ ks.T * scale, -1)
            out[s, at], size[s, at] = p @ vs, p @ vs.abs()
            spread[s, at] = (q[s, at].abs() @ ks.abs().T).amax(-1)
    return out, size, spread


def page_sums(cache, tables, lengths):
    """64-bit sums of the filled rows of all requests' pages, ``{page: (k, v, sum |k|, sum |v|)}``."""
    k, v = (values(x.cpu(), None if s is None else s.cpu()) for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    tables, result = tables.cpu().tolist(), {}
    for s, length in enumerate(lengths.cpu().tolist()):
        for i in range(pages_of(length)):
            a, b = (x[tables[s][i], :, :min(PAGE, length - i * PAGE)] for x in (k, v))
            result[tables[s][i]] = (a.sum(1), b.sum(1), a.abs().sum(1), b.abs().sum(1))
    return result


def make_tables(lengths, pages, gen, extra=1, device="cuda"):
    """Scattered physical pages; entries behind a request's own name a page that does not exist."""
    held = [pages_of(max(0, n)) for n in lengths]
    assert sum(held) <= pages
    order = torch.randperm(pages, generator=gen).tolist()
    tables = torch.full((len(lengths), max(held) + extra), 2 ** 31 - 1, dtype=torch.int32)
    for s, n in enumerate(held):
        tables[s, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return tables.to(device)
