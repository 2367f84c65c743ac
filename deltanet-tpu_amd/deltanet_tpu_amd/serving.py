"""What a server calls around the softmax-attention layers of ``attention.py``: pages
from a pool as the sequences grow, slots and positions of a step's tokens, queries,
keys and values normed, rotated and stored in one launch, attention of drafted trees,
and the accepted tokens moved to the front.  A step that verifies drafts:

    short = paged_reserve(pool, page_table, held, lens, page_size=P)
    positions, slots, visible = paged_slots(page_table, lens, N, page_size=P, cu_seqlens=cu, held=held, parents=parents, nodes=T)
    # in every softmax-attention layer:
    q = paged_qkv_append(q, k, v, k_cache, v_cache, slots, positions, q_weight=wq, k_weight=wk, table=table)
    out = paged_tree_attention(q, k_cache, v_cache, page_table, lens, visible, cu_seqlens=cu)
    # the drafts that the model agrees with, ``kept``:
    lens = paged_kv_keep(k_caches, v_caches, page_table, starts, kept, held=held)
    paged_reserve(pool, page_table, held, lens, page_size=P)

Nothing here reads a device tensor on the host; all of it can be captured in a graph.  A
step goes on where the pool runs short: with ``held``, tokens behind the pages that their
sequence has get no slot, are not stored and not kept, whatever ``kept`` says, and what
attention returns for them means nothing; the others' results are right (for chains by
``paged_attention`` only as long as no length passes the page table).  (Behind them
the page table holds numbers of pages that may be another sequence's by now: leave
``held`` out only where no sequence is ever short.)
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .attention import (
    _INT, _attention_common, _forward_ad, _grad_enabled, _bump, _call, _calls, _check_caches, _check_norm, _check_pages, _check_table, _check_weights,
    _dense_channels, _differentiated, _on_gpu, _rows16, _window)
from .gdn2 import _DT

__all__ = ["page_pool", "paged_reserve", "paged_slots", "paged_qkv_append", "paged_tree_attention", "paged_kv_keep"]

_NODES = 1024   # new tokens of a tree
_SCALE = {D: 1.0 / math.sqrt(D) for D in (64, 128, 256)}
_CONTIGUOUS, _I32, _I64 = torch.contiguous_format, torch.int32, torch.int64

# A step calls these once or once per layer, a token or two per sequence at a time, and
# what it costs on the host is most of such a call.  So each asks in one expression
# whether everything is as it mostly is, and goes through the checks with their messages
# (the functions _check_..., which decide) only if it is not.


def _check_page_size(page_size):
    if isinstance(page_size, bool) or not isinstance(page_size, int) or page_size < 1 or page_size & (page_size - 1) or page_size > 1 << 30:
        raise ValueError(f"page_size must be a power of two, got {page_size!r}.")


def _check_table_rows(page_table):
    if page_table.ndim != 2 or page_table.dtype is not torch.int32 or (page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError(f"page_table must be int32 (B, max_pages) with contiguous rows, got {page_table.dtype} {tuple(page_table.shape)}.")
    if page_table.shape[1] < 1:
        raise ValueError("page_table must have a column.")
    return page_table.shape[0]


def _check_int32(name, t, shape):
    if t.dtype is not torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor {shape}, got {t.dtype} {tuple(t.shape)}.")


def page_pool(pages, *, device=None):
    """A pool of the cache's pages 0 .. pages - 1, all of them free: an int32 tensor
    (2 + pages) with the number of free pages, a word that the kernels use and that is
    0 between calls, and the free pages as a stack, page 0 on top.  For ``paged_reserve``."""
    if isinstance(pages, bool) or not isinstance(pages, int) or not 0 <= pages <= 0x7ffffff0:
        raise ValueError(f"pages must be an integer from 0 on, got {pages!r}.")
    device = torch.device("cuda" if device is None else device)
    pool = torch.zeros(2 + pages, dtype=torch.int32, device=device)
    pool[0] = pages
    pool[2:] = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
    return pool


def paged_reserve(pool, page_table, held, lens, *, page_size: int):
    """Pages taken from ``pool`` and given back, so that each sequence has exactly the
    pages that its ``lens`` tokens need: for the new tokens of a step, to trim a
    sequence whose drafts were rejected, and with length 0 to release one.

    pool: from ``page_pool``.  page_table: int32 (B, max_pages), the first ``held[b]``
    entries of row b are its pages.  held, lens: int32 (B,).  pool, page_table and held
    are updated in place; a page belongs to one sequence, and calls on one pool follow
    one another on a stream.  Pages that are no longer needed go back first; then
    sequences take theirs in the order of the batch.  From the first for which the pool
    does not hold enough on, those that need more get nothing, and neither does one
    that needs more than max_pages.  Returns int32 (B,): the pages that a sequence is
    short of, 0 where it has what it needs.  What is given back comes out again in the
    order in which it was taken, so that growing and trimming leave the pool as it was.
    B is at most 4096.
    """
    B, most = page_table.shape if page_table.ndim == 2 else (-1, 0)
    if not (type(page_size) is int and 0 < page_size <= 1 << 30 and not page_size & (page_size - 1) and 0 <= B <= _lib.MAX_SEQUENCES and most > 0
            and page_table.dtype is _I32 and pool.dtype is _I32 and held.dtype is _I32 and lens.dtype is _I32
            and page_table.stride(1) == 1 and page_table.stride(0) >= most and pool.ndim == 1 and pool.is_contiguous() and held.shape == lens.shape == (B,) and held.is_contiguous()
            and lens.is_contiguous() and 2 <= pool.shape[0] <= 0x7fffffff - B * most):
        _check_reserve(pool, page_table, held, lens, page_size)
    dev = pool.get_device()
    if not page_table.get_device() == held.get_device() == lens.get_device() == dev >= 0:
        _on_gpu(pool, page_table, held, lens)
    short = torch.empty_like(lens)
    if B:
        _call("dn_paged_reserve", dev, _lib.PAGED_RESERVE_PACK(
            _lib.DN_ABI_VERSION, pool.shape[0] - 2, B, page_size, most, pool.data_ptr(), page_table.data_ptr(), held.data_ptr(),
            lens.data_ptr(), short.data_ptr(), page_table.stride(0)))
        _bump((pool, page_table, held))   # autograd sees the stores
    return short


def _check_reserve(pool, page_table, held, lens, page_size):
    _check_page_size(page_size)
    B = _check_table_rows(page_table)
    if pool.dtype is not torch.int32 or pool.ndim != 1 or pool.shape[0] < 2 or not pool.is_contiguous():
        raise ValueError(f"pool must be a tensor of page_pool, got {pool.dtype} {tuple(pool.shape)}.")
    _check_int32("held", held, (B,))
    _check_int32("lens", lens, (B,))
    if B > _lib.MAX_SEQUENCES:
        raise ValueError(f"paged_reserve takes at most {_lib.MAX_SEQUENCES} sequences, got {B}.")
    if B > 1 and page_table.stride(0) < page_table.shape[1]:
        raise ValueError(f"the rows of page_table overlap, got strides {page_table.stride()} of {tuple(page_table.shape)}.")
    if B * page_table.shape[1] + pool.shape[0] > 0x7fffffff:
        raise ValueError("page_table and pool have too many pages.")


def paged_slots(page_table, seq_lens, tokens: int, *, page_size: int, cu_seqlens=None, held=None, parents=None, nodes=None):
    """Where the new tokens of a step go: their positions and their slots in the cache,
    once for all layers; of drafted trees also what each token sees.

    page_table: int32 (B, max_pages).  seq_lens: int32 (B,), the new tokens included.
    tokens: new tokens in all; ``cu_seqlens`` int32 (B + 1,) says where each sequence's
    start, and without it every sequence has tokens / B.  held: int32 (B,), the pages
    that each sequence has (``paged_reserve``); tokens behind them get no slot.
    parents: int32 (tokens,), the place of each drafted token's parent among its
    sequence's new tokens, a negative number for the children of the cached text; a
    parent must come before its children (one that does not counts as none).  nodes:
    the most new tokens of a sequence then, at most 1024 (rounded up to 64; those past
    it are no tokens).

    Returns (positions int32, slots int64), each (tokens,), or with parents (positions,
    slots, visible).  New token i of n has slot page * page_size + place in the page of
    token seq_lens - n + i, which is its position too; in a tree the position is
    seq_lens - n plus the number of its ancestors.  Slot -1: no place in the cache.
    visible: int64 (tokens, ceil(nodes / 64)), bit j % 64 of word j // 64 says that the
    token sees new token j of its sequence: itself and its ancestors.  Tokens that
    cu_seqlens gives to no sequence have position and slot -1 and see nothing.
    """
    B, most = page_table.shape if page_table.ndim == 2 else (-1, 0)
    if not (type(page_size) is int and 0 < page_size <= 1 << 30 and not page_size & (page_size - 1) and B > 0 and most > 0
            and type(tokens) is int and 0 <= tokens <= 0x7fffffff and page_table.dtype is _I32 and page_table.stride(1) == 1
            and seq_lens.dtype is _I32 and seq_lens.shape == (B,) and seq_lens.is_contiguous()
            and (tokens % B == 0 if cu_seqlens is None else cu_seqlens.dtype is _I32 and cu_seqlens.shape == (B + 1,) and cu_seqlens.is_contiguous())
            and (held is None or held.dtype is _I32 and held.shape == (B,) and held.is_contiguous())
            and (nodes is None if parents is None else type(nodes) is int and 1 <= nodes <= _NODES and parents.dtype is _I32
                 and parents.shape == (tokens,) and parents.is_contiguous())):
        _check_slots(page_table, seq_lens, tokens, page_size, cu_seqlens, held, parents, nodes)
    dev = page_table.get_device()
    if not (seq_lens.get_device() == dev >= 0 and (cu_seqlens is None or cu_seqlens.get_device() == dev) and (held is None or held.get_device() == dev)
            and (parents is None or parents.get_device() == dev)):
        _on_gpu(page_table, seq_lens, cu_seqlens, held, parents)
    words = 0 if parents is None else (nodes + 63) >> 6
    positions, slots = seq_lens.new_empty(tokens), seq_lens.new_empty(tokens, dtype=_I64)
    visible = slots.new_empty((tokens, words)) if words else None
    if tokens:
        _call("dn_paged_slots", dev, _lib.PAGED_SLOTS_PACK(
            _lib.DN_ABI_VERSION, tokens, B, page_size, most, words, page_table.data_ptr(), seq_lens.data_ptr(),
            0 if cu_seqlens is None else cu_seqlens.data_ptr(), 0 if held is None else held.data_ptr(), 0 if parents is None else parents.data_ptr(),
            positions.data_ptr(), slots.data_ptr(), 0 if visible is None else visible.data_ptr(), page_table.stride(0)))
    return (positions, slots, visible) if words else (positions, slots)


def _check_slots(page_table, seq_lens, tokens, page_size, cu_seqlens, held, parents, nodes):
    _check_page_size(page_size)
    B = _check_table_rows(page_table)
    if isinstance(tokens, bool) or not isinstance(tokens, int) or not 0 <= tokens <= 0x7fffffff:
        raise ValueError(f"tokens must be an integer from 0 on, got {tokens!r}.")
    _check_int32("seq_lens", seq_lens, (B,))
    if cu_seqlens is not None:
        _check_int32("cu_seqlens", cu_seqlens, (B + 1,))
    if held is not None:
        _check_int32("held", held, (B,))
    if tokens and not B or cu_seqlens is None and B and tokens % B:
        raise ValueError(f"without cu_seqlens every sequence has tokens / B of them, got {tokens} for {B}.")
    if (parents is None) != (nodes is None):
        raise ValueError("parents goes with nodes.")
    if parents is not None:
        _check_int32("parents", parents, (tokens,))
        if isinstance(nodes, bool) or not isinstance(nodes, int) or not 1 <= nodes <= _NODES:
            raise ValueError(f"nodes must be an integer from 1 to {_NODES}, got {nodes!r}.")


def paged_qkv_append(q, k, v, k_cache, v_cache, slots, positions, *, q_weight=None, k_weight=None, eps: float = 1e-6,
                     weight_offset: float = 0.0, table=None, interleaved: bool = False):
    """Queries, keys and values of new tokens on their way from the projection to
    ``paged_attention`` or ``paged_tree_attention``, in one launch: queries and keys
    normed by their weights (as in ``norm_rotary``; without weights not) and rotated
    by their positions (without table not), keys and values stored in the cache.

    q: (N, Hq, D) or (B, T, Hq, D); k, v: the same with the cache's heads; one of
    float32, bfloat16 and float16, channels contiguous.  k_cache, v_cache: (pages,
    page_size, Hkv, D) as in ``paged_kv_append``, written in place (rounded to the
    cache's type).  slots: int64, positions: int32 or int64, contiguous, one per token
    (``paged_slots``).  A token whose slot is outside the cache is not stored; a token
    at a negative position is none: it is not stored and its queries are zeros; a
    position past the table gives NaN in the rotated channels.  Slots must differ.
    Products in float32, one rounding.  Returns the queries, contiguous in q's shape and type.
    """
    cs, qs, ks = k_cache.shape, q.shape, k.shape
    dt, ct, lead = q.dtype, k_cache.dtype, slots.shape
    kcs, vcs = k_cache.stride(), v_cache.stride()
    wt = dt if q_weight is None else q_weight.dtype
    if not (len(cs) == 4 and v_cache.shape == cs and v_cache.dtype is ct and ct in _DT and dt in _DT and k.dtype is dt and v.dtype is dt
            and kcs[3] == vcs[3] == 1 and cs[1] > 0 and not cs[1] & (cs[1] - 1) and len(qs) in (3, 4) and qs[:-2] == lead and v.shape == ks
            and ks[:-2] == lead and ks[-2:] == cs[2:] and qs[-1] == cs[3] and slots.dtype is _I64 and slots.is_contiguous()
            and positions.dtype in _INT and positions.shape == lead and positions.is_contiguous()
            and type(eps) is float and 0.0 <= eps <= 3e38 and type(weight_offset) is float and -3e38 <= weight_offset <= 3e38
            and (k_weight is None if q_weight is None else k_weight is not None and k_weight.dtype is wt and wt in _DT
                 and q_weight.shape == k_weight.shape == cs[3:] and q_weight.is_contiguous() and k_weight.is_contiguous())):
        eps, weight_offset = _check_qkv_append(q, k, v, k_cache, v_cache, slots, positions, q_weight, k_weight, eps, weight_offset)
    pages, page, Hkv, D = cs
    rows = R = 0
    if table is not None:
        _check_table(table, D)
        rows, R = table.shape
    dev = q.get_device()
    if not (k.get_device() == v.get_device() == k_cache.get_device() == v_cache.get_device() == slots.get_device() == positions.get_device() == dev >= 0
            and (q_weight is None or q_weight.get_device() == k_weight.get_device() == dev) and (table is None or table.get_device() == dev)):
        _on_gpu(q, k, v, k_cache, v_cache, slots, positions, q_weight, k_weight, table)
    if (_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or k_cache.requires_grad or v_cache.requires_grad
                             or q_weight is not None and (q_weight.requires_grad or k_weight.requires_grad))) \
            or _forward_ad._current_level >= 0 and _differentiated(q, k, v, k_cache, v_cache, q_weight, k_weight):
        raise ValueError("paged_qkv_append is not differentiable; call it under torch.no_grad() (norm_rotary is its form for training).")
    qt, kt, vt = q.stride(), k.stride(), v.stride()
    if not qt[-1] == kt[-1] == vt[-1] == 1:
        q, k, v = _dense_channels(q), _dense_channels(k), _dense_channels(v)
        qt, kt, vt = q.stride(), k.stride(), v.stride()
    out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    if len(qs) == 3:   # (strides of the batch: there is one)
        B, T, qb, kb, vb = 1, qs[0], 0, 0, 0
    else:
        B, T, qb, kb, vb = qs[0], qs[1], qt[0], kt[0], vt[0]
    if B and T:
        _call("dn_qkv_append", dev, _lib.QKV_APPEND_PACK(
            _lib.DN_ABI_VERSION, B, T, qs[-2], Hkv, D, R, _DT[dt], _DT[ct], _DT[wt],
            _INT[positions.dtype], 1 if interleaved else 0, rows, pages, page, eps, weight_offset,
            q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(),
            out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr(), positions.data_ptr(), table.data_ptr() if R else 0,
            qb, qt[-3], qt[-2], kb, kt[-3], kt[-2], vb, vt[-3], vt[-2], kcs[0], kcs[1], kcs[2], vcs[0], vcs[1], vcs[2]))
        _bump((k_cache, v_cache))   # autograd sees the stores
    return out


def _check_qkv_append(q, k, v, k_cache, v_cache, slots, positions, q_weight, k_weight, eps, weight_offset):
    pages, page, Hkv, D = _check_caches(k_cache, v_cache)
    if page < 1 or page & (page - 1):
        raise ValueError(f"page_size must be a power of two, got {page}.")
    if q.ndim not in (3, 4) or q.dtype not in _DT or q.shape[-1] != D:
        raise ValueError(f"q must be (N, Hq, D) or (B, T, Hq, D), float32, bfloat16 or float16, with the cache's channels ({D}), got {q.dtype} {tuple(q.shape)}.")
    lead = q.shape[:-2]
    for name, t in (("k", k), ("v", v)):
        if t.dtype is not q.dtype or t.shape != (*lead, Hkv, D):
            raise ValueError(f"{name} must match q's tokens and type and the cache's heads {(*lead, Hkv, D)}, got {t.dtype} {tuple(t.shape)}.")
    if slots.dtype is not torch.int64 or slots.shape != lead or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 tensor {tuple(lead)}, got {slots.dtype} {tuple(slots.shape)}.")
    if positions.dtype not in _INT or positions.shape != lead or not positions.is_contiguous():
        raise ValueError(f"positions must be a contiguous int32 or int64 tensor {tuple(lead)}, got {positions.dtype} {tuple(positions.shape)}.")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight goes with k_weight.")
    if q_weight is not None:
        _check_weights(D, q_weight, k_weight)
    return _check_norm(eps, weight_offset)


def paged_tree_attention(q, k_cache, v_cache, page_table, seq_lens, visible, *, cu_seqlens=None, scale=None, window=None,
                         return_lse: bool = False):
    """Attention of drafted trees over a paged cache that holds their keys and values
    already (``paged_qkv_append``): every new token sees all tokens of its sequence in
    front of the new ones, and of those the ones that its row of ``visible`` names.

    q, caches, page_table, seq_lens, cu_seqlens, scale: as in ``paged_attention``.
    visible: int64 (tokens, words), contiguous, words from 1 to 16, from ``paged_slots``
    or any others: bit j % 64 of word j // 64 says that the token sees new token j of
    its sequence (new tokens that have no bit are seen by none; bits past a sequence's
    new tokens mean nothing).  window: at least 64 words; the last ``window`` of the
    tokens that a token sees.  A token that sees nothing gets zeros (lse -inf).  Tokens
    that the page table has no place for (seq_lens past it) are seen by none; the others
    keep their positions.  As there, bfloat16 and float16 probabilities are rounded to the
    type once before their product with the values (their sum is not).  Returns as
    ``paged_attention`` does.
    """
    cs, qs, ct = k_cache.shape, q.shape, k_cache.dtype
    kcs, vcs, qt = k_cache.stride(), v_cache.stride(), q.stride()
    N, words = visible.shape if visible.ndim == 2 else (-1, 0)
    B, most = page_table.shape if page_table.ndim == 2 else (-1, 0)
    nd, e = len(qs), 4 if ct is torch.float32 else 2
    if not (len(cs) == 4 and v_cache.shape == cs and v_cache.dtype is ct and q.dtype is ct and ct in _DT and kcs[3] == vcs[3] == 1
            and cs[0] > 0 and cs[1] > 0 and not cs[1] & (cs[1] - 1) and 3 <= nd <= 4 and qs[-1] == cs[3] and cs[3] in _SCALE
            and cs[2] > 0 and qs[-2] > 0 and qs[-2] % cs[2] == 0 and B >= 0 and most > 0 and page_table.dtype is _I32 and page_table.stride(1) == 1
            and seq_lens.dtype is _I32 and seq_lens.shape == (B,) and seq_lens.is_contiguous()
            and (qs[0] == B and N == (B if nd == 3 else B * qs[1]) if cu_seqlens is None else nd == 3 and qs[0] == N and cu_seqlens.dtype is _I32
                 and cu_seqlens.shape == (B + 1,) and cu_seqlens.is_contiguous())
            and visible.dtype is _I64 and visible.is_contiguous() and 1 <= words <= _NODES >> 6 and scale is None
            and (window is None or type(window) is int and window >= 64 * words)
            and not ((kcs[0] | kcs[1] | kcs[2] | vcs[0] | vcs[1] | vcs[2]) * e | k_cache.data_ptr() | v_cache.data_ptr()) & 15):
        scale = _check_tree_attention(q, k_cache, v_cache, page_table, seq_lens, visible, cu_seqlens, scale, window)
    else:
        scale = _SCALE[cs[3]]
    pages, page, Hkv, D = cs
    dev = q.get_device()
    if not (k_cache.get_device() == v_cache.get_device() == page_table.get_device() == seq_lens.get_device() == visible.get_device() == dev >= 0
            and (cu_seqlens is None or cu_seqlens.get_device() == dev)):
        _on_gpu(q, k_cache, v_cache, page_table, seq_lens, visible, cu_seqlens)
    if _grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad) \
            or _forward_ad._current_level >= 0 and _differentiated(q, k_cache, v_cache):
        raise ValueError("paged_tree_attention is not differentiable; call it under torch.no_grad().")
    if qt[-1] != 1 or (q.data_ptr() | (qt[0] | qt[-3] | qt[-2]) * e) & 15:
        q = _rows16(q)
        qt = q.stride()
    out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    lse = torch.empty(qs[:-1], dtype=torch.float32, device=q.device) if return_lse else None
    if N:
        block = _lib.PAGED_ATTENTION_PACK(
            _lib.DN_ABI_VERSION, N, B, qs[-2], Hkv, D, _DT[ct], _window(window), pages, page, most, scale,
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
            page_table.data_ptr(), seq_lens.data_ptr(), 0 if cu_seqlens is None else cu_seqlens.data_ptr(),
            qt[0], qt[0] if nd == 3 else qt[1], qt[-2], kcs[0], kcs[1], kcs[2], vcs[0], vcs[1], vcs[2], page_table.stride(0))
        size = _calls.get("dn_paged_tree_attention_workspace_size") or _lib.packed_call("dn_paged_tree_attention_workspace_size")
        need = size(block, words)
        ws = q.new_empty(-(-need // e))
        _call("dn_paged_tree_attention", dev, block, visible.data_ptr(), words, ws.data_ptr(), need)
    return (out, lse) if return_lse else out


def _check_tree_attention(q, k_cache, v_cache, page_table, seq_lens, visible, cu_seqlens, scale, window):
    """The checks; the scale as a number."""
    pages, page, Hkv, D = _check_caches(k_cache, v_cache)
    if page < 1 or page & (page - 1) or pages < 1:
        raise ValueError(f"page_size must be a power of two and the cache have a page, got {tuple(k_cache.shape)}.")
    if q.dtype is not k_cache.dtype or q.shape[-1] != D:
        raise ValueError(f"q {tuple(q.shape)} {q.dtype} must have the cache's channels and type ({D}, {k_cache.dtype}).")
    _check_table_rows(page_table)
    _, N, _, _ = _check_pages(page_table, seq_lens, cu_seqlens, q, "q")
    scale = _attention_common(D, q.shape[-2], Hkv, q.dtype, scale, window)
    if visible.dtype is not torch.int64 or visible.ndim != 2 or visible.shape[0] != N or not 1 <= visible.shape[1] <= _NODES // 64 \
            or not visible.is_contiguous():
        raise ValueError(f"visible must be a contiguous int64 tensor ({N}, words) of 1 to {_NODES // 64} words, got {visible.dtype} {tuple(visible.shape)}.")
    words = visible.shape[1]
    if window is not None and window < 64 * words:
        raise ValueError(f"the window of a tree must take in the {64 * words} new tokens that visible has bits for, got {window}.")
    _on_gpu(q, k_cache, v_cache, page_table, seq_lens, visible, cu_seqlens)
    kcs, vcs = k_cache.stride(), v_cache.stride()
    if (k_cache.data_ptr() | v_cache.data_ptr() | (kcs[0] | kcs[1] | kcs[2] | vcs[0] | vcs[1] | vcs[2]) * q.element_size()) & 15:
        raise ValueError(f"cache rows must start on 16 bytes, got strides {kcs} and {vcs}.")
    return scale


def paged_kv_keep(k_cache, v_cache, page_table, starts, kept, *, held=None):
    """The keys and values of accepted drafts moved to the front of their sequence's
    new tokens, in all layers: token starts + kept[i] goes to starts + i.

    k_cache, v_cache: (pages, page_size, Hkv, D), or (layers, pages, page_size, Hkv, D)
    for the caches of all layers, any strides, written in place.  page_table: int32
    (B, max_pages).  starts: int32 (B,), each sequence's tokens in front of the new
    ones.  kept: int32 (B, most), the places of the accepted ones among the new,
    rising, with negative numbers behind the last; what comes after an entry that is
    negative, not above the one before it, past the page table or past the pages that its
    sequence has is not kept; held: int32 (B,), those pages (``paged_reserve``).  Pages
    that are written must not be shared.  Returns int32 (B,): the sequences' lengths
    then, starts plus the number of tokens kept, for ``paged_reserve``.
    """
    cs, ct = k_cache.shape, k_cache.dtype
    ks, vs = k_cache.stride(), v_cache.stride()
    B, most = kept.shape if kept.ndim == 2 else (-1, 0)
    if not (4 <= len(cs) <= 5 and v_cache.shape == cs and v_cache.dtype is ct and ct in _DT and ks[-1] == vs[-1] == 1 and cs[-3] > 0
            and not cs[-3] & (cs[-3] - 1) and page_table.ndim == 2 and page_table.dtype is _I32 and page_table.shape[0] == B <= 65535
            and page_table.shape[1] > 0 and page_table.stride(1) == 1 and starts.dtype is _I32 and starts.shape == (B,) and starts.is_contiguous()
            and kept.dtype is _I32 and kept.is_contiguous()
            and (held is None or held.dtype is _I32 and held.shape == (B,) and held.is_contiguous())):
        _check_keep(k_cache, v_cache, page_table, starts, kept, held)
    dev = k_cache.get_device()
    if not (v_cache.get_device() == page_table.get_device() == starts.get_device() == kept.get_device() == dev >= 0
            and (held is None or held.get_device() == dev)):
        _on_gpu(k_cache, v_cache, page_table, starts, kept, held)
    if _grad_enabled() and (k_cache.requires_grad or v_cache.requires_grad) or _forward_ad._current_level >= 0 and _differentiated(k_cache, v_cache):
        raise ValueError("paged_kv_keep is not differentiable; call it under torch.no_grad().")
    lens = torch.empty_like(starts)
    if B:
        many = len(cs) == 5
        _call("dn_kv_keep", dev, _lib.KV_KEEP_PACK(
            _lib.DN_ABI_VERSION, cs[0] if many else 1, B, cs[-2], cs[-1], most, _DT[ct], cs[-4], cs[-3], page_table.shape[1],
            k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(), starts.data_ptr(), kept.data_ptr(), lens.data_ptr(),
            ks[0] if many else 0, ks[-4], ks[-3], ks[-2], vs[0] if many else 0, vs[-4], vs[-3], vs[-2], page_table.stride(0),
            0 if held is None else held.data_ptr()))
        _bump((k_cache, v_cache))   # autograd sees the stores
    return lens


def _check_keep(k_cache, v_cache, page_table, starts, kept, held):
    many = k_cache.ndim == 5 and v_cache.ndim == 5
    if many and k_cache.shape[0] != v_cache.shape[0]:
        raise ValueError(f"v_cache {tuple(v_cache.shape)} must have the layers of k_cache {tuple(k_cache.shape)}.")
    one = (lambda c: c[0] if c.shape[0] else c.new_empty(c.shape[1:])) if many else (lambda c: c)
    _, page, _, _ = _check_caches(one(k_cache), one(v_cache))
    if page < 1 or page & (page - 1):
        raise ValueError(f"page_size must be a power of two, got {page}.")
    B = _check_table_rows(page_table)
    _check_int32("starts", starts, (B,))
    if kept.ndim != 2:
        raise ValueError(f"kept must be int32 (B, most), got {kept.dtype} {tuple(kept.shape)}.")
    _check_int32("kept", kept, (B, kept.shape[1]))
    if held is not None:
        _check_int32("held", held, (B,))
    if B > 65535:
        raise ValueError(f"paged_kv_keep takes at most 65535 sequences, got {B}.")
