"""Paged key/value cache and the operators that answer one new token per request over it.

The training form of the path is :func:`cudnn_vsa_b200.vsa.vsa_attention` over whole packed samples.
To answer, a model keeps the keys and values of every request in pages of 64 tokens - the blocks of
that path - and each new token sees the pages that its own scores select, plus the gated attention
over the page means:

1. :func:`plan_paged_step`  block tables and slot maps of a step, built on the GPU (once per step)
2. :func:`append_tokens`    new rows into their pages, and the pages' FP32 sums (per layer)
3. :func:`select_pages`     ``keep`` pages per request and key/value head, and the coarse attention
4. :func:`paged_attention`  one new token per request over all its pages or the selected ones

:func:`cudnn_vsa_b200.vsa.vsa_decode` runs 2 to 4 as a layer of a model does.  All of them launch on
the current stream of their tensors' device, never synchronise, allocate only what they return and
a workspace of their own per call, and can be captured into CUDA graphs.  They have no
backward and no forward-mode derivative, and refuse tensors that need one.

Sizes: at most 8192 requests a call; pages * kv_heads * 64, table columns * 64, requests * heads and
requests * table columns * kv_heads * ceil(heads / kv_heads / 8) below 2**31; pages are selected from
at most 24,576 of a request, rows added to at most 65,535 key/value heads.
"""
from __future__ import annotations

import functools
import struct
from dataclasses import dataclass, field

import torch
from torch.autograd import forward_ad

from . import _cabi
from .vsa_layout import BLOCK

HEAD_DIM = 128
MAX_REQUESTS = 8192        # of one step
MAX_SELECT_PAGES = 24576   # of one request, when pages are selected (1.5 million tokens)
MAX_WIDTH = 2 ** 25 - 1    # columns of the tables: a request's tokens are numbered by 32-bit integers
MAX_APPEND_HEADS = 65535   # key/value heads, when rows are added

_ACTIVATIONS = {torch.bfloat16: 0, torch.float16: 1}
_STORES = {torch.bfloat16: 0, torch.float16: 1, torch.float8_e4m3fn: 2}


@dataclass(frozen=True, eq=False)
class PagedKVCache:
    """Keys and values of one attention layer.

    ``k``, ``v`` are ``[pages, kv_heads, 64, 128]`` in BF16, FP16 or e4m3; ``k_sum``, ``v_sum``
    ``[pages, kv_heads, 128]`` FP32 hold the sums of every page's filled rows.  An e4m3 cache holds
    ``x / scale`` rounded and saturated, with one FP32 scale per key/value head in ``k_scale`` and
    ``v_scale``.  ``status`` is a device word that kernels set when a table names a page that does
    not exist (:func:`check_cache_status`).
    """
    k: torch.Tensor
    v: torch.Tensor
    k_sum: torch.Tensor
    v_sum: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None
    status: torch.Tensor = field(init=False, repr=False)
    pages: int = field(init=False)
    kv_heads: int = field(init=False)
    store: int = field(init=False, repr=False)  # the C entry points' number of the cache's dtype

    def __post_init__(self):
        k, v = self.k, self.v
        if k.dtype not in _STORES:
            raise ValueError("A paged cache holds bfloat16, float16 or float8_e4m3fn")
        if k.ndim != 4 or k.shape[2] != BLOCK or k.shape[3] != HEAD_DIM or any(n <= 0 for n in k.shape):
            raise ValueError("Cache keys and values must have shape [pages, kv_heads, 64, 128] with positive dimensions")
        if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
            raise ValueError("Cache keys and values must have identical shape, dtype and device")
        sums = (k.shape[0], k.shape[1], HEAD_DIM)
        for x in (self.k_sum, self.v_sum):
            if x.shape != sums or x.dtype != torch.float32 or x.device != k.device:
                raise ValueError("k_sum and v_sum must be float32 [pages, kv_heads, 128] on the cache's device")
        if k.shape[0] * k.shape[1] * BLOCK > 2 ** 31 - 1:
            raise ValueError("A paged cache has fewer than 2**31 rows (pages * kv_heads * 64)")
        scales = (self.k_scale, self.v_scale)
        if k.dtype == torch.float8_e4m3fn:
            for x in scales:
                if x is None or x.shape != (k.shape[1],) or x.dtype != torch.float32 or x.device != k.device:
                    raise ValueError("An e4m3 cache needs k_scale and v_scale, float32 [kv_heads] on its device")
        elif any(x is not None for x in scales):
            raise ValueError("k_scale and v_scale belong to an e4m3 cache")
        for x in (k, v, self.k_sum, self.v_sum, *scales):
            if x is not None and not x.is_contiguous():
                raise ValueError("Cache tensors must be contiguous")
        for name, value in (("status", torch.zeros(1, dtype=torch.int32, device=k.device)), ("pages", k.shape[0]),
                            ("kv_heads", k.shape[1]), ("store", _STORES[k.dtype])):
            object.__setattr__(self, name, value)


def build_paged_cache(pages, kv_heads, *, dtype=torch.bfloat16, k_scale=None, v_scale=None, device="cuda"):
    """An empty :class:`PagedKVCache`; its keys and values are unwritten until they are appended."""
    for n, what in ((pages, "pages"), (kv_heads, "kv_heads")):
        if isinstance(n, bool) or not isinstance(n, int) or n <= 0:
            raise ValueError(f"{what} must be a positive integer")
    shape = (pages, kv_heads, BLOCK, HEAD_DIM)
    k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
    k_sum, v_sum = (torch.zeros(pages, kv_heads, HEAD_DIM, device=device) for _ in range(2))
    return PagedKVCache(k, v, k_sum, v_sum, k_scale, v_scale)


def check_cache_status(cache):
    """Raise if a kernel met a page id outside the cache or gave up a bounded wait (synchronises)."""
    code = int(cache.status.item())
    if code == 200:
        raise RuntimeError("A block table named a page outside the cache; its tokens were left out")
    if code:
        raise RuntimeError(f"Paged cache kernel reported device error {code} (a bounded wait timed out)")


@dataclass(eq=False)
class PagedStep:
    """What a step's layers share: made by :func:`plan_paged_step`.

    ``lengths`` int32 ``[requests]`` and ``free_count`` int32 ``[1]`` are the state after the step,
    ``admitted`` bool ``[requests]``, ``row_slot`` int64 ``[tokens]`` the cache slot
    (``page * 64 + row``) of every row or -1, ``runs`` int32 ``[n, 4]`` the list ``(first row, rows,
    page, first row in the page)`` of touched pages, zero behind its end, and ``tables`` the block
    tables the plan completed in place.
    """
    lengths: torch.Tensor
    free_count: torch.Tensor
    admitted: torch.Tensor
    row_slot: torch.Tensor
    runs: torch.Tensor
    tables: torch.Tensor


# The argument structs of the C entry points (include/vsa_b200.h): 64-bit integers and addresses, and
# the scale as a double where there is one.
_PACK = {name: struct.Struct(fields).pack for name, fields in (
    ("vsa_paged_plan", "18q"), ("vsa_paged_append", "21q"), ("vsa_paged_select", "17qd6q"),
    ("vsa_paged_attention", "23qd6q"), ("vsa_paged_decode", "34qd5q"))}


def _address(t):
    return 0 if t is None else t.data_ptr()


def _integers(x, shape, what, dtype=torch.int32):
    if not isinstance(x, torch.Tensor) or x.dtype != dtype or x.shape != shape:
        raise ValueError(f"{what} must be {str(dtype)[6:]} with shape {list(shape)}")
    if not x.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def _entries(x, what, of):
    """Checks a nonempty int32 vector; returns its length."""
    if not isinstance(x, torch.Tensor) or x.dtype != torch.int32 or x.ndim != 1 or x.shape[0] == 0:
        raise ValueError(f"{what} must be int32 with shape [{of}], at least one")
    if not x.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    return x.shape[0]


def _tables(tables, requests):
    """Checks block tables; returns their row stride and width."""
    if not isinstance(tables, torch.Tensor) or tables.dtype != torch.int32 or tables.ndim != 2 or 0 in tables.shape:
        raise ValueError("tables must be int32 [requests, pages per request]")
    rows, width = tables.shape
    stride, one = tables.stride()
    if rows != requests:
        raise ValueError(f"tables must have one row for each of the {requests} requests")
    if width > MAX_WIDTH:
        raise ValueError("tables must have at most 2**25 - 1 columns")
    if rows == 1:
        stride = width
    if (one != 1 and width > 1) or stride < width:
        raise ValueError("tables must have contiguous rows that do not overlap")
    return stride, width


def _same_device(index, *tensors):
    """Checks that `index` is a CUDA device and the one of all tensors."""
    if index < 0:
        raise ValueError("The paged cache operators require CUDA tensors; this build has no CPU path")
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError("All tensors of a paged cache call must be on the same CUDA device")


def _launch(index, launches, name, *args):
    """Launch on the tensors' device and its current stream, whatever the current device is."""
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return _launch(index, launches, name, *args)
    _cabi.call(name, _PACK[name](*args, torch._C._cuda_getCurrentRawStream(index)), launches=launches)


def _no_gradient(*tensors):
    """Refuses tensors whose gradient, or whose forward-mode derivative, a call would lose."""
    grad, dual = torch.is_grad_enabled(), forward_ad._current_level >= 0
    if not grad and not dual:
        return
    for x in tensors:
        if x is not None and (grad and x.requires_grad or dual and forward_ad.unpack_dual(x).tangent is not None):
            raise ValueError("The paged cache operators have no backward and no forward-mode derivative; call them under "
                             "torch.no_grad(), on tensors without tangents")


def _rows(x, rows, heads, dtype, what):
    """Checks ``[rows, heads, 128]`` activations; returns their row and head stride in elements."""
    if not isinstance(x, torch.Tensor) or x.ndim != 3:
        raise ValueError(f"{what} must have shape [rows, heads, 128]")
    m, n, d = x.shape
    if d != HEAD_DIM or (rows is not None and m != rows) or (heads is not None and n != heads) or m == 0 or n == 0:
        raise ValueError(f"{what} must have shape [{'rows' if rows is None else rows}, "
                         f"{'heads' if heads is None else heads}, 128] with positive dimensions")
    if x.dtype not in _ACTIVATIONS or (dtype is not None and x.dtype != dtype):
        raise ValueError(f"{what} must be {'bfloat16 or float16' if dtype is None else str(dtype)[6:]}")
    row, head, one = x.stride()
    if m == 1:
        row = 0
    if n == 1:
        head = 0
    if one != 1 or row % 8 or head % 8 or x.data_ptr() % 16:
        raise ValueError(f"{what} needs contiguous heads of 128, strides in multiples of 8 elements and a 16-byte "
                         "aligned start")
    if x.requires_grad or forward_ad._current_level >= 0:
        _no_gradient(x)
    return row, head


def _cache(cache):
    if not isinstance(cache, PagedKVCache):
        raise ValueError("Expected a PagedKVCache from build_paged_cache")
    if (forward_ad._current_level >= 0 or cache.k.requires_grad or cache.v.requires_grad
            or cache.k_sum.requires_grad or cache.v_sum.requires_grad
            or cache.store == 2 and (cache.k_scale.requires_grad or cache.v_scale.requires_grad)):
        _no_gradient(cache.k, cache.v, cache.k_sum, cache.v_sum, cache.k_scale, cache.v_scale)


def _query(q, cache, tables, lengths):
    """Checks the arguments that selection and attention share; returns the numbers that a launch takes."""
    _cache(cache)
    row, head = _rows(q, None, None, None, "q")
    requests, heads, _ = q.shape
    if heads % cache.kv_heads:
        raise ValueError("The query heads must be a multiple of the cache's key/value heads")
    if cache.store != 2 and cache.store != _ACTIVATIONS[q.dtype]:
        raise ValueError("q must have the cache's dtype (or the cache be e4m3)")
    if requests > MAX_REQUESTS:
        raise ValueError(f"A call takes at most {MAX_REQUESTS} requests")
    stride, width = _tables(tables, requests)
    _integers(lengths, (requests,), "lengths")
    group = heads // cache.kv_heads
    if max(width * cache.kv_heads * -(-group // 8), heads) * requests > 2 ** 31 - 1:
        raise ValueError("requests * table columns * kv_heads * ceil(group / 8) and requests * heads must be below 2**31")
    return row, head, requests, group, stride, width


def _budget(keep, first, last, width):
    """Checks a page budget (None = all pages)."""
    for n, what in ((keep, "keep"), (first, "first"), (last, "last")):
        if type(n) is not int or not 0 <= n <= 2 ** 31 - 1:
            if n is not None or what != "keep":
                raise ValueError(f"{what} must be a nonnegative integer below 2**31")
    if keep is not None:
        if keep < 1 or keep < first + last:
            raise ValueError("keep must be positive and at least first + last")
        if width > MAX_SELECT_PAGES:
            raise ValueError(f"Pages are selected from at most {MAX_SELECT_PAGES} per request")


@functools.lru_cache(maxsize=64)
def _select_workspace_bytes(requests, kv_heads, group, width, choose, coarse):
    return _cabi.load().vsa_paged_select_workspace_bytes(requests, kv_heads, group, width, choose, coarse)


@functools.lru_cache(maxsize=64)
def _decode_plan(requests, kv_heads, group, width, keep, gated, store):
    """Workspace bytes and kernels of a decode step."""
    kernels = 2 + bool(_workspace_bytes(requests, kv_heads, group, width, keep, store))
    if keep or gated:
        kernels += 1 + bool(_select_workspace_bytes(requests, kv_heads, group, width, keep > 0, gated))
    return _cabi.load().vsa_paged_decode_workspace_bytes(requests, kv_heads, group, width, keep, gated, store), kernels


@functools.lru_cache(maxsize=64)
def _workspace_bytes(requests, kv_heads, group, width, keep, store):
    return _cabi.load().vsa_paged_workspace_bytes(requests, kv_heads, group, min(width, keep) if keep else width, store)


def _scale(scale):
    scale = HEAD_DIM ** -0.5 if scale is None else float(scale)
    if not 0.0 <= scale <= 2.0 ** 127:  # the kernels take scale * log2(e) in FP32
        raise ValueError("scale must be a nonnegative number of at most 2**127")
    return scale


def plan_paged_step(lengths, new, tables, free_pages, free_count, *, tokens, rows_per_request=None, out=None):
    """Block tables and slot maps of one step, built on the GPU from the requests' lengths.

    ``lengths`` int32 ``[requests]``: tokens in the cache.  ``new`` int32 ``[requests]``: tokens that
    the step adds; a negative value ends the request, its pages return to the stack and its length
    becomes 0.  ``tables`` int32 ``[requests, width]`` names the physical page of every logical page
    and is completed in place; a page belongs to one request, and entries behind a request's pages keep
    what they held.  ``free_pages`` int32 ``[pages]`` is the stack of free pages with ``free_count`` int32
    ``[1]`` valid entries: ended requests push, then the others pop from its top, all in request order.

    A request is admitted if its rows fit ``tokens``, its pages fit ``width``, and the stack holds
    what it and the requests before it ask for; otherwise ``admitted`` is false, its rows get slot
    -1 and its length stays.  The step has ``tokens`` rows (a host integer, so that nothing
    synchronises): packed in request order, or request ``s`` at row ``s * rows_per_request``.

    ``lengths``, ``free_count``, ``admitted``, ``row_slot`` and ``runs`` of the returned
    :class:`PagedStep` are new tensors, or those of ``out``, a step of an earlier call with the same
    sizes.  ``out.lengths`` may be ``lengths`` itself and ``out.free_count`` ``free_count``, so that a
    captured step advances its own state.
    """
    requests = _entries(lengths, "lengths", "requests")
    _integers(new, (requests,), "new")
    stride, width = _tables(tables, requests)
    pool = _entries(free_pages, "free_pages", "pages")
    _integers(free_count, (1,), "free_count")
    if requests * width > 2 ** 31 - 1:
        raise ValueError("requests * table columns must be below 2**31")
    if requests > MAX_REQUESTS:
        raise ValueError(f"A step has at most {MAX_REQUESTS} requests")
    if type(tokens) is not int or not 1 <= tokens <= 2 ** 31 - 1:
        raise ValueError("tokens must be a positive integer below 2**31")
    if rows_per_request is not None and (type(rows_per_request) is not int or not 1 <= rows_per_request <= 2 ** 31 - 1):
        raise ValueError("rows_per_request must be a positive integer below 2**31")
    max_runs = min(tokens, tokens // BLOCK + 2 * requests)
    if out is not None:
        if not isinstance(out, PagedStep):
            raise ValueError("out must be a PagedStep")
        _integers(out.lengths, (requests,), "out.lengths")
        _integers(out.free_count, (1,), "out.free_count")
        _integers(out.admitted, (requests,), "out.admitted", torch.bool)
        _integers(out.row_slot, (tokens,), "out.row_slot", torch.int64)
        _integers(out.runs, (max_runs, 4), "out.runs")
    index = lengths.get_device()
    _same_device(index, new, tables, free_pages, free_count,
                 *(() if out is None else (out.lengths, out.free_count, out.admitted, out.row_slot, out.runs)))
    if out is None:
        out = PagedStep(torch.empty_like(lengths), torch.empty_like(free_count), torch.empty_like(lengths, dtype=torch.bool),
                        torch.empty_strided((tokens,), (1,), dtype=torch.int64, device=lengths.device),
                        lengths.new_empty(max_runs, 4), tables)
    else:
        out = PagedStep(out.lengths, out.free_count, out.admitted, out.row_slot, out.runs, tables)
    _launch(index, 1, "vsa_paged_plan", lengths.data_ptr(), new.data_ptr(), tables.data_ptr(), stride, width, requests, free_pages.data_ptr(), pool,
            free_count.data_ptr(), tokens, rows_per_request or 0, out.lengths.data_ptr(), out.free_count.data_ptr(),
            out.admitted.data_ptr(), out.row_slot.data_ptr(), out.runs.data_ptr(), max_runs)
    return out


def append_tokens(cache, k, v, step):
    """Write the step's rows ``k``, ``v`` ``[tokens, kv_heads, 128]`` into their pages of ``cache`` and
    form the sums of the pages they touch.

    Rows may be strided views (two fields of a fused projection); rows without a slot are skipped,
    and rows of a page behind its filled ones stay as they are.  A touched page's sum is formed from
    all its rows, so a repeated call changes nothing, and a request that was cut back to a shorter
    length is right again after its next append.
    """
    tokens, k_strides, v_strides = _new_rows(cache, k, v, step)
    index = cache.k.get_device()
    _same_device(index, k, v, step.runs)
    _launch(index, 1, "vsa_paged_append", k.data_ptr(), v.data_ptr(), *k_strides, *v_strides, _ACTIVATIONS[k.dtype], tokens,
            cache.k.data_ptr(), cache.v.data_ptr(), cache.store, cache.k_sum.data_ptr(), cache.v_sum.data_ptr(),
            _address(cache.k_scale), _address(cache.v_scale), step.runs.data_ptr(), step.runs.shape[0], cache.pages,
            cache.kv_heads, cache.status.data_ptr())


def _new_rows(cache, k, v, step):
    """Checks the rows that a step adds; returns their count and strides."""
    _cache(cache)
    if not isinstance(step, PagedStep):
        raise ValueError("Expected a PagedStep from plan_paged_step")
    if cache.kv_heads > MAX_APPEND_HEADS:
        raise ValueError(f"Rows are added to at most {MAX_APPEND_HEADS} key/value heads")
    tokens = step.row_slot.shape[0]
    k_strides = _rows(k, tokens, cache.kv_heads, None if cache.store == 2 else cache.k.dtype, "k")
    v_strides = _rows(v, tokens, cache.kv_heads, k.dtype, "v")
    runs = step.runs
    if runs.ndim != 2 or runs.shape[0] == 0:
        raise ValueError("step.runs must be int32 [n, 4]")
    _integers(runs, (runs.shape[0], 4), "step.runs")
    return tokens, k_strides, v_strides


def select_pages(q, cache, tables, lengths, *, keep=None, first=1, last=1, coarse=False, scale=None):
    """Pages that each request's new token sees, and the attention over the page means.

    ``q`` is ``[requests, heads, 128]``, one token per request, ``heads`` a multiple of the cache's
    key/value heads.  Per key/value head a page scores the product of the group's summed queries
    with its mean key, formed in 64 bits.  Returns int32 ``[requests, kv_heads, keep]``: the first
    ``first`` and last ``last`` logical pages and the highest-scoring others (ties to the lowest),
    ascending, -1 behind the last.  A request with at most ``keep`` pages gets all of them.

    With ``coarse=True`` the result is ``(pages, coarse)``: ``coarse`` FP32 ``[requests, heads, 128]``
    is ``softmax(scale * q . mean keys) @ mean values`` over all pages of the request, the second
    branch of the path; ``keep=None`` computes it alone (``pages`` is ``None``).  Requests of length 0
    get no pages and zeros.
    """
    row, head, requests, group, stride, width = _query(q, cache, tables, lengths)
    _budget(keep, first, last, width)
    if keep is None and not coarse:
        raise ValueError("select_pages needs keep, coarse=True or both")
    scale = _scale(scale)
    index = cache.k.get_device()
    _same_device(index, q, tables, lengths)
    pages = None if keep is None else lengths.new_empty(requests, cache.kv_heads, keep)
    mean = torch.empty_like(q, dtype=torch.float32, memory_format=torch.contiguous_format) if coarse else None
    size = _select_workspace_bytes(requests, cache.kv_heads, group, width, keep is not None, coarse)
    workspace = lengths.new_empty(size // 4) if size else None
    _launch(index, 2 if size else 1, "vsa_paged_select", q.data_ptr(), row, head, _ACTIVATIONS[q.dtype],
            cache.k_sum.data_ptr(), cache.v_sum.data_ptr(), tables.data_ptr(), stride, width, lengths.data_ptr(), requests,
            cache.kv_heads, group, cache.pages, keep or 0, first, last, scale, _address(pages), _address(mean),
            _address(workspace), size, cache.status.data_ptr())
    return (pages, mean) if coarse else pages


def paged_attention(q, cache, tables, lengths, *, pages=None, gate=None, coarse=None, scale=None, return_lse=False):
    """Attention of one new token per request over its cached tokens.

    ``q`` is ``[requests, heads, 128]``; query head ``h`` reads key/value head ``h // group``.  The token
    sees the first ``lengths[s]`` tokens of request ``s``, or those of them that lie in the logical
    pages ``pages`` ``[requests, kv_heads, keep]`` (each page once; -1 = none; of a request with fewer
    than ``keep`` pages only that many entries are read).  With ``gate`` (same
    shape and dtype as ``q``) and ``coarse`` (FP32, from :func:`select_pages`) the result is
    ``fine + gate * coarse``.  Returns ``[requests, heads, 128]`` in ``q``'s dtype, and with
    ``return_lse`` also the FP32 log sum of the softmax ``[requests, heads]``; a request without
    tokens gives zeros and ``-inf``.  The cache is read in one pass whose work is split over its
    length as well; partial results are joined in a fixed order, so equal calls give equal bits.
    """
    row, head, requests, group, stride, width = _query(q, cache, tables, lengths)
    keep = 0
    if pages is not None:
        if not isinstance(pages, torch.Tensor) or pages.ndim != 3 or pages.shape[2] == 0:
            raise ValueError("pages must be int32 [requests, kv_heads, keep]")
        keep = pages.shape[2]
        _integers(pages, (requests, cache.kv_heads, keep), "pages")
    if (gate is None) != (coarse is None):
        raise ValueError("gate and coarse are given together")
    gate_row = gate_head = 0
    if gate is not None:
        gate_row, gate_head = _rows(gate, requests, q.shape[1], q.dtype, "gate")
        if coarse.shape != q.shape or coarse.dtype != torch.float32 or not coarse.is_contiguous():
            raise ValueError("coarse must be contiguous float32 [requests, heads, 128]")
        _no_gradient(coarse)
    scale = _scale(scale)
    index = cache.k.get_device()
    _same_device(index, q, tables, lengths, pages, gate, coarse)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    heads = group * cache.kv_heads
    lse = torch.empty_strided((requests, heads), (heads, 1), dtype=torch.float32, device=q.device) if return_lse else None
    size = _workspace_bytes(requests, cache.kv_heads, group, width, keep, cache.store)
    workspace = lengths.new_empty(size // 4) if size else None
    _launch(index, 2 if size else 1, "vsa_paged_attention", q.data_ptr(), row, head, _ACTIVATIONS[q.dtype],
            cache.k.data_ptr(), cache.v.data_ptr(), cache.store, _address(cache.k_scale), _address(cache.v_scale), cache.pages,
            tables.data_ptr(), stride, width, lengths.data_ptr(), requests, cache.kv_heads, group, _address(pages), keep,
            _address(gate), gate_row, gate_head, _address(coarse), scale, out.data_ptr(), _address(lse), _address(workspace),
            size, cache.status.data_ptr())
    return (out, lse) if return_lse else out


def decode_layer(q, k, v, gate, cache, step, *, keep=None, first=1, last=1, scale=None):
    """Append, select and attend in one call; see :func:`cudnn_vsa_b200.vsa.vsa_decode`."""
    tokens, k_strides, v_strides = _new_rows(cache, k, v, step)
    tables, lengths, runs = step.tables, step.lengths, step.runs
    row, head, requests, group, stride, width = _query(q, cache, tables, lengths)
    if k.dtype != q.dtype:
        raise ValueError("q, k and v must have the same dtype")
    _budget(keep, first, last, width)
    gate_row = gate_head = 0
    if gate is not None:
        gate_row, gate_head = _rows(gate, requests, q.shape[1], q.dtype, "gate")
    scale = _scale(scale)
    if keep is not None and keep >= width:  # every page: the choice would list them all
        keep = None
    index = cache.k.get_device()
    _same_device(index, q, k, v, gate, tables, lengths, runs)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    size, kernels = _decode_plan(requests, cache.kv_heads, group, width, keep or 0, gate is not None, cache.store)
    workspace = lengths.new_empty(size // 4)
    _launch(index, kernels, "vsa_paged_decode", q.data_ptr(), row, head, k.data_ptr(), v.data_ptr(), *k_strides, *v_strides,
            _ACTIVATIONS[q.dtype], tokens, cache.k.data_ptr(), cache.v.data_ptr(), cache.store, cache.k_sum.data_ptr(),
            cache.v_sum.data_ptr(), _address(cache.k_scale), _address(cache.v_scale), cache.pages, cache.kv_heads, group,
            runs.data_ptr(), runs.shape[0], tables.data_ptr(), stride, width, lengths.data_ptr(), requests, keep or 0, first, last, _address(gate), gate_row, gate_head, scale, out.data_ptr(),
            workspace.data_ptr(), size, cache.status.data_ptr())
    return out
