"""Public entry points: ``vsa_attention`` and the two boundary reorder helpers.

Same names, arguments, validation order and error texts as the reference's ``vsa.py`` (:9-121),
so a caller can switch ``from vsa import ...`` to ``from cudnn_vsa_b200.vsa import ...``.
"""
from __future__ import annotations

import torch

from . import vsa_cache, vsa_core, vsa_kernels
from .vsa_layout import VSALayout

_REORDER_DTYPES = (torch.float16, torch.bfloat16, torch.float32, torch.float64, torch.int8, torch.uint8,
                   torch.int16, torch.int32, torch.int64, torch.bool)


def _reorder_tokens(x, layout, inverse):
    """Checks of reference ``vsa.py:9-24`` in the same order, then the row kernel."""
    if not isinstance(layout, VSALayout) or layout.input_order != "block":
        raise ValueError('Token reordering requires a VSALayout with input_order="block"')
    if inverse and layout.ring is not None:
        raise ValueError("block_wo_padding_to_raster requires a full VSALayout; gather Ring outputs explicitly")
    tokens = layout.tokens if layout.ring is None else layout.ring.global_tokens
    if not isinstance(x, torch.Tensor) or x.ndim < 1 or x.shape[0] != tokens:
        raise ValueError(f"Expected one tensor with shape [{tokens}, ...]")
    if any(size == 0 for size in x.shape[1:]) or not x.is_contiguous():
        raise ValueError("Token-reorder input must be contiguous with nonempty row dimensions")
    if x.dtype not in _REORDER_DTYPES:
        raise ValueError("Unsupported token-reorder dtype")
    if not x.is_cuda or x.device != layout.input_rows.device:
        raise ValueError("Token-reorder input and layout must be on the same CUDA device")
    return vsa_kernels.reorder_tokens(x, layout.input_rows, inverse=inverse)


def raster_to_block_wo_padding(x, *, vsa_layout):
    """Reorder one global raster tensor ``[T_global, ...]`` into compact block order.

    With a full block layout all rows come back reordered; with a ring layout only the rows
    this rank owns, ``[layout.tokens, ...]``, in one gather.  Dtype and trailing dimensions
    are preserved.  Differentiable to any order; the backward scatters to the original rows
    and leaves unowned rows zero.  Call once before the stack of VSA layers, separately for
    tokens, position ids and any other row-aligned field.
    """
    return _reorder_tokens(x, vsa_layout, inverse=False)


def block_wo_padding_to_raster(x, *, vsa_layout):
    """Inverse of :func:`raster_to_block_wo_padding` for a full (non-ring) block layout."""
    return _reorder_tokens(x, vsa_layout, inverse=True)


def _validate(q, k, v, gate):
    if q is None or k is None or v is None:
        raise ValueError("Q, K and V are required separate tensors")
    if gate is None:
        raise ValueError("VSA requires a gate tensor; use FA4 full attention without a gate")
    if q.ndim != 3 or any(n <= 0 for n in q.shape):
        raise ValueError("Q/K/V must have shape [tokens, heads, head_dim] with positive dimensions")
    for x in (q, k, v, gate):
        if x.shape != q.shape or x.dtype != q.dtype or x.device != q.device:
            raise ValueError("Q/K/V/gate must have identical shape, dtype and device")
        if not x.is_contiguous():
            raise ValueError("Q/K/V/gate must be contiguous; materialize projections before calling attention")


def vsa_attention(q, k, v, gate, vsa_layout, *, scale=None):
    """Packed video-sparse attention: ``[T, H, 128]`` BF16 Q/K/V/gate -> O in the same row order.

    ``vsa_layout`` comes from :func:`build_vsa_layout` for the current batch geometry and is
    reused across layers.  Inputs follow ``layout.input_order`` (raster, or compact block order
    without padding) and the output uses the same order.  Per (query block, head) the KV blocks
    of every sparse video region are chosen from the current Q/K with the budgets fixed in the
    layout; dense regions are always visible; ``layout.dense_query_full`` lets dense queries see
    everything.  Samples made only of dense segments run fine attention alone and never read
    ``gate``.  ``scale`` defaults to ``head_dim ** -0.5``.  A ring layout (``layout.ring``) runs
    the context-parallel path with the process group bound at layout construction.
    """
    layout = vsa_layout
    if not isinstance(layout, VSALayout):
        raise ValueError("Expected a VSALayout from build_vsa_layout")
    _validate(q, k, v, gate)
    if q.shape[0] != layout.tokens:
        raise ValueError("Expected [layout.tokens, heads, head_dim] inputs")
    if q.shape[1] != layout.head_num:
        raise ValueError("Q/K/V head count must match VSALayout.head_num")
    if layout.block_sizes.device != q.device:
        raise ValueError("VSALayout and activations must be on the same device")
    if not q.is_cuda or q.dtype != torch.bfloat16 or q.shape[-1] != 128:
        raise ValueError("The B200 VSA kernels require CUDA BF16 and head_dim=128")
    if layout.ring is not None:
        return vsa_core.ring_attention(q, k, v, gate, layout, scale=scale)
    return vsa_core.attention(q, k, v, gate, layout, scale=scale)


def vsa_attention_fused(mixed, vsa_layout, *, scale=None):
    """``vsa_attention`` on the caller's fused projection output.

    ``mixed`` is one contiguous ``[T, H, 4, 128]`` BF16 tensor holding q, k, v and gate of every
    head side by side (a ``Linear(C, 4 * C)`` output viewed as ``[T, H, 4, D]``, as in the
    reference's context-parallel demo, ``README.md:477``).  Equivalent to
    ``vsa_attention(*(t.contiguous() for t in mixed.unbind(2)), vsa_layout)`` - bit for bit - but
    the four ``.contiguous()`` copies never happen and the backward pass writes one
    ``[T, H, 4, 128]`` gradient instead of four tensors that autograd would have to stack.
    Single-device layouts only; rows follow ``layout.input_order``.
    """
    layout = vsa_layout
    if not isinstance(layout, VSALayout):
        raise ValueError("Expected a VSALayout from build_vsa_layout")
    if mixed is None or mixed.ndim != 4 or mixed.shape[2] != 4 or any(n <= 0 for n in mixed.shape):
        raise ValueError("Expected one [tokens, heads, 4, head_dim] tensor with positive dimensions")
    if not mixed.is_contiguous():
        raise ValueError("The fused Q/K/V/gate tensor must be contiguous")
    if mixed.shape[0] != layout.tokens:
        raise ValueError("Expected [layout.tokens, heads, 4, head_dim] inputs")
    if mixed.shape[1] != layout.head_num:
        raise ValueError("Q/K/V head count must match VSALayout.head_num")
    if layout.block_sizes.device != mixed.device:
        raise ValueError("VSALayout and activations must be on the same device")
    if not mixed.is_cuda or mixed.dtype != torch.bfloat16 or mixed.shape[-1] != 128:
        raise ValueError("The B200 VSA kernels require CUDA BF16 and head_dim=128")
    if layout.ring is not None:
        raise ValueError("vsa_attention_fused runs single-device layouts; pass separate tensors to a ring layout")
    return vsa_core.attention_fused(mixed, layout, scale=scale)


def vsa_decode(q, k, v, gate, cache, step, *, keep=None, first=1, last=1, scale=None):
    """One layer's answer to one new token per request, over its paged key/value cache.

    The decode form of :func:`vsa_attention`: ``k``, ``v`` ``[tokens, kv_heads, 128]`` are the rows that
    the step adds (see :func:`cudnn_vsa_b200.vsa_cache.plan_paged_step`), and row ``s`` of ``q``
    ``[requests, heads, 128]`` then answers over all ``step.lengths[s]`` tokens of its request:
    ``out = fine + gate * coarse``, with fine attention over the ``keep`` pages that ``q`` selects
    (``None``: over all pages) and coarse attention over the page means.  With ``gate=None`` the
    result is the fine attention alone.  Returns ``[requests, heads, 128]``.
    """
    return vsa_cache.decode_layer(q, k, v, gate, cache, step, keep=keep, first=first, last=last, scale=scale)
