"""The softmax-attention layers that a hybrid model has between its delta-rule
layers: rotary positions, a paged key/value cache and attention over it for
serving, causal attention for training.  The reference has the delta-rule layers
alone; these entry points follow its conventions (token-major tensors, grouped
heads, documents by ``segment_ids`` or ``cu_seqlens``, ``ValueError`` for a bad
argument) and this package's: HIP kernels on the tensors' GPU and the current
stream, no CPU path.

Nothing here reads a device tensor on the host, except ``causal_attention`` a
``cu_seqlens`` tensor, as ``chunk_gdn2`` does.
"""

from __future__ import annotations

import math

import numpy as np
import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib
from .gdn2 import _DT, _is_integer_dtype, _raw_stream, _require_gpu

__all__ = ["rotary_table", "apply_rotary", "norm_rotary", "paged_kv_append", "paged_attention", "causal_attention"]

_INT = {torch.int32: _lib.DN_I32, torch.int64: _lib.DN_I64}


_current = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_calls = _lib._packed_calls
_grad_enabled = torch.is_grad_enabled
_bump = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)


def _call(name, dev, block, *args):
    """An entry point on the current stream of GPU `dev`."""
    f = _calls.get(name) or _lib.packed_call(name)
    if dev == _current():
        rc = f(block, *args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = f(block, *args, _raw_stream(dev))
    if rc:
        _lib.check(rc, name)


def _on_gpu(*ts):
    """The index of the GPU that all of them (None aside) are on; the message of
    ``_require_gpu`` otherwise."""
    try:
        dev = ts[0].get_device()
        for t in ts:
            if t is not None and t.get_device() != dev:
                dev = -1
        if dev >= 0:
            return dev
    except AttributeError:
        pass
    return _require_gpu(*ts).index


def _differentiated(*ts):
    """Whether a derivative goes through one of them (None aside): backwards, or as a
    forward-mode tangent, which no ``requires_grad`` shows."""
    if _grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return _forward_ad._current_level >= 0 and any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in ts)


def _dense_channels(t):
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

def rotary_table(max_position, rotary_dim, *, base: float = 10000.0, scaling=None, device=None):
    """The angles of positions 0 .. max_position - 1: a float32 tensor
    (max_position, rotary_dim) with row p = [cos(p f_i) | sin(p f_i)] and
    f_i = base^(-2i / rotary_dim), computed in float64.

    ``scaling`` stretches the table for contexts longer than the trained one.  A
    dict with ``type`` and ``factor`` >= 1:

    - ``"linear"``: positions divided by the factor;
    - ``"ntk"``: base multiplied by factor^(R / (R - 2)), so that the slowest
      frequency is divided by the factor and the fastest is kept;
    - ``"yarn"``: frequencies that turn more than ``beta_fast`` (32) times within
      ``original_max_position`` are kept, those that turn less than ``beta_slow``
      (1) times are divided by the factor, with a linear ramp over i in between;
      cos and sin are multiplied by ``attention_factor`` (0.1 ln(factor) + 1).
    """
    P, R = int(max_position), int(rotary_dim)
    if P < 1:
        raise ValueError(f"max_position must be at least 1, got {max_position}.")
    if R < 2 or R % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}.")
    if not base > 0:
        raise ValueError(f"base must be positive, got {base}.")
    i = torch.arange(0, R, 2, dtype=torch.float64)
    freq, gain = float(base) ** (-i / R), 1.0
    if scaling is not None:
        kind, factor = scaling.get("type"), float(scaling.get("factor", 0.0))
        if not factor >= 1.0:
            raise ValueError(f"scaling factor must be at least 1, got {scaling.get('factor')!r}.")
        if kind == "linear":
            freq = freq / factor
        elif kind == "ntk":
            if R < 4:
                raise ValueError("scaling 'ntk' needs rotary_dim of at least 4.")
            freq = (float(base) * factor ** (R / (R - 2.0))) ** (-i / R)
        elif kind == "yarn":
            trained = scaling.get("original_max_position")
            if not trained or not trained > 0:
                raise ValueError("scaling 'yarn' needs original_max_position.")
            fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
            if not (fast > slow > 0) or not base > 1:
                raise ValueError("scaling 'yarn' needs beta_fast > beta_slow > 0 and base > 1.")
            # the index (in units of i / 2) whose frequency turns `n` times within the trained length
            at = lambda n: R * math.log(trained / (n * 2.0 * math.pi)) / (2.0 * math.log(base))
            lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), R - 1)
            keep = 1.0 - ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
            freq = freq / factor * (1.0 - keep) + freq * keep
            gain = scaling.get("attention_factor")
            gain = 0.1 * math.log(factor) + 1.0 if gain is None else float(gain)
        else:
            raise ValueError(f"scaling type must be 'linear', 'ntk' or 'yarn', got {kind!r}.")
    device = torch.device("cuda" if device is None else device)
    angle = torch.arange(P, dtype=torch.float64, device=device)[:, None] * freq.to(device)
    return torch.cat([torch.cos(angle), torch.sin(angle)], dim=1).mul_(gain).to(torch.float32)


def _check_table(table, D):
    if table.ndim != 2 or table.dtype is not torch.float32 or not table.is_contiguous():
        raise ValueError(f"table must be a contiguous float32 tensor (positions, rotary_dim), got {table.dtype} {tuple(table.shape)}.")
    R = table.shape[1]
    if R < 2 or R % 2 or R > D:
        raise ValueError(f"rotary_dim ({R}) must be even, positive and at most the head dimension ({D}).")
    if table.shape[0] < 1:
        raise ValueError("table must have a row for position 0.")
    return R


def _rotary_launch(q, k, pos, ps, table, interleaved, inverse):
    B, L, Hq, D = q.shape
    q_out = q.new_empty(q.shape)
    sq = q.stride()
    if k is None:
        Hk, sk, kp, ko, k_out = 0, (0, 0, 0), 0, 0, None
    else:
        k_out = k.new_empty(k.shape)
        Hk, sk, kp, ko = k.shape[2], k.stride(), k.data_ptr(), k_out.data_ptr()
    block = _lib.ROTARY_PACK(_lib.DN_ABI_VERSION, B, L, Hq, Hk, D, table.shape[1], _DT[q.dtype], _INT[pos.dtype],
                             1 if interleaved else 0, 1 if inverse else 0, table.shape[0], q.data_ptr(), kp, q_out.data_ptr(),
                             ko, pos.data_ptr(), table.data_ptr(), sq[0], sq[1], sq[2], sk[0], sk[1], sk[2], ps[0], ps[1])
    _call("dn_rotary", q.get_device(), block)
    return q_out, k_out


class _RotaryFn(torch.autograd.Function):
    """The rotation is orthogonal up to the table's gain: its gradient is the same
    rotation with the sines negated."""

    @staticmethod
    def forward(ctx, q, k, pos, ps, table, interleaved, inverse):
        ctx.save_for_backward(pos, table)
        ctx.meta = ps, interleaved, inverse
        ctx.set_materialize_grads(False)
        q_out, k_out = _rotary_launch(q, k, pos, ps, table, interleaved, inverse)
        return (q_out, k_out) if k is not None else q_out

    @staticmethod
    def backward(ctx, dq, dk=None):
        pos, table = ctx.saved_tensors
        ps, interleaved, inverse = ctx.meta
        given = [_dense_channels(g) for g in (dq, dk) if g is not None]
        if not given:
            return (None,) * 7
        a, b = given[0], given[1] if len(given) > 1 else None
        if torch.is_grad_enabled() or _differentiated(a, b):   # create_graph: the rotation of the gradients is differentiable in turn
            turned = _RotaryFn.apply(a, b, pos, ps, table, interleaved, not inverse)
            turned = turned if b is not None else (turned, None)
        else:
            turned = _rotary_launch(a, b, pos, ps, table, interleaved, not inverse)
        if dq is None:
            turned = None, turned[0]
        return turned[0], turned[1], None, None, None, None, None


def apply_rotary(q, k, positions, table, *, interleaved: bool = False):
    """Queries and keys with the first ``table.shape[1]`` channels of every head
    rotated by the angles of their positions.

    q: (B, L, Hq, D) or (N, Hq, D); k: the same with Hk heads, or None; both
    float32, bfloat16 or float16, channels contiguous, any other strides (slices
    of a fused projection are read in place).  positions: int32 or int64, (B, L)
    or (L,) for every row alike, (N,) for rank 3.  table: from ``rotary_table``.
    Pairs are (i, i + R/2), or (2i, 2i + 1) with ``interleaved``.  A position
    outside the table gives NaN in the rotated channels.  Products in float32,
    one rounding.  Differentiable in q and k, any number of times (backwards; tangents
    are refused).  Returns (q', k') with k' None if k is None; the results are contiguous.
    """
    if q.ndim not in (3, 4):
        raise ValueError(f"q must have rank 3 (N, Hq, D) or rank 4 (B, L, Hq, D), got shape {tuple(q.shape)}.")
    if q.dtype not in _DT:
        raise ValueError(f"q must be float32, bfloat16 or float16, got {q.dtype}.")
    if k is not None and (k.ndim != q.ndim or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1] or k.dtype != q.dtype):
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} must match q {tuple(q.shape)} {q.dtype} in all but the heads.")
    _check_table(table, q.shape[-1])
    if positions.dtype not in _INT:
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}.")
    _on_gpu(q, k, positions, table)
    lead = q.shape[:-2]
    if positions.shape == lead:
        ps = positions.stride()
    elif positions.ndim == 1 and positions.shape[0] == lead[-1]:
        ps = (0, positions.stride(0))
    else:
        raise ValueError(f"positions {tuple(positions.shape)} must have the token dimensions of q {tuple(lead)}, or the last of them.")
    flat = q.ndim == 3
    if flat:
        q, k, ps = q[None], None if k is None else k[None], (0, ps[-1])
    q, k = _dense_channels(q), None if k is None else _dense_channels(k)
    if _differentiated(q, k):
        r = _RotaryFn.apply(q, k, positions, ps, table, bool(interleaved), False)
        q_out, k_out = r if k is not None else (r, None)
    else:
        q_out, k_out = _rotary_launch(q, k, positions, ps, table, interleaved, False)
    if flat:
        q_out, k_out = q_out[0], None if k_out is None else k_out[0]
    return q_out, k_out


# ---------------------------------------------------------------------------
# norms of heads
# ---------------------------------------------------------------------------

def _finite(name, x):
    try:
        x = float(x)
    except (TypeError, ValueError) as e:
        raise ValueError(f"{name} must be convertible to a concrete float, got {type(x)}: {e}")
    if not abs(x) <= 3e38:
        raise ValueError(f"{name} must be finite in float32, got {x}.")
    return x


def _check_norm(eps, offset):
    eps, offset = _finite("eps", eps), _finite("weight_offset", offset)
    if eps < 0.0:
        raise ValueError(f"eps must not be negative, got {eps}.")
    return eps, offset


def _check_weights(D, *ws):
    for w in ws:
        if w.dtype not in _DT or w.dtype is not ws[0].dtype or w.shape != (D,) or (D > 1 and w.stride(0) != 1):
            raise ValueError(f"norm weights must be contiguous ({D},) tensors of one type, float32, bfloat16 or float16, got {w.dtype} {tuple(w.shape)}.")


def _norm_block(q, k, qw, kw, q_out, k_out, pos, table, meta):
    """The argument block; one of q and k may be None, with its weights."""
    ps0, ps1, eps, offset, inter = meta
    one, w = (k, kw) if q is None else (q, qw)
    B, L, Hq, D = one.shape
    q0, q1, q2, _ = k0, k1, k2, _ = one.stride()
    if q is None:
        Hq, Hk = 0, Hq
    elif k is None:
        Hk = 0
    else:
        Hk = k.shape[2]
        k0, k1, k2, _ = k.stride()
    rows, R = (0, 0) if table is None else table.shape
    return _lib.NORM_ROTARY_PACK(
        _lib.DN_ABI_VERSION, B, L, Hq, Hk, D, R, _DT[one.dtype], _DT[w.dtype], _lib.DN_I32 if pos is None else _INT[pos.dtype], inter, rows,
        eps, offset, 0 if q is None else q.data_ptr(), 0 if k is None else k.data_ptr(), 0 if qw is None else qw.data_ptr(),
        0 if kw is None else kw.data_ptr(), 0 if q_out is None else q_out.data_ptr(), 0 if k_out is None else k_out.data_ptr(),
        0 if pos is None else pos.data_ptr(), 0 if table is None else table.data_ptr(), q0, q1, q2, k0, k1, k2, ps0, ps1)


def _norm_launch(q, k, qw, kw, pos, table, meta):
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    _call("dn_norm_rotary", q.get_device(), _norm_block(q, k, qw, kw, q_out, k_out, pos, table, meta))
    return q_out, k_out


class _NormRotaryFn(torch.autograd.Function):
    """Keeps the inputs; the backward computes the heads' norms again."""

    @staticmethod
    def forward(ctx, q, k, qw, kw, pos, table, meta):
        ctx.save_for_backward(q, k, qw, kw, pos, table)
        ctx.meta = meta
        ctx.set_materialize_grads(False)
        q_out, k_out = _norm_launch(q, k, qw, kw, pos, table, meta)
        return (q_out, k_out) if k is not None else q_out

    @staticmethod
    def backward(ctx, d_q, d_k=None):
        q, k, qw, kw, pos, table = ctx.saved_tensors
        want_q, want_k, want_qw, want_kw = ctx.needs_input_grad[:4]
        gq = gk = gqw = gkw = None
        q0 = q1 = q2 = k0 = k1 = k2 = 0
        # a side whose result nobody used, or whose gradients nobody wants, has none
        if d_q is None or not (want_q or want_qw):
            q = qw = d_q = None
        else:
            if d_q.stride(-1) != 1:
                d_q = _dense_channels(d_q)
            if want_q:
                gq = torch.empty_like(q, memory_format=torch.contiguous_format)
            if want_qw:
                gqw = torch.empty_like(qw)
            q0, q1, q2, _ = d_q.stride()
        if d_k is None or not (want_k or want_kw):
            k = kw = d_k = None
        else:
            if d_k.stride(-1) != 1:
                d_k = _dense_channels(d_k)
            if want_k:
                gk = torch.empty_like(k, memory_format=torch.contiguous_format)
            if want_kw:
                gkw = torch.empty_like(kw)
            k0, k1, k2, _ = d_k.stride()
        if q is None and k is None:
            return None, None, None, None, None, None, None
        block = _norm_block(q, k, qw, kw, None, None, pos, table, ctx.meta)
        need = (_calls.get("dn_norm_rotary_bwd_workspace_size") or _lib.packed_call("dn_norm_rotary_bwd_workspace_size"))(block)
        if need:
            ws = (k if q is None else q).new_empty(need, dtype=torch.uint8)
            grads = _lib.NORM_ROTARY_GRADS_PACK(
                0 if d_q is None else d_q.data_ptr(), 0 if d_k is None else d_k.data_ptr(), 0 if gq is None else gq.data_ptr(),
                0 if gk is None else gk.data_ptr(), 0 if gqw is None else gqw.data_ptr(), 0 if gkw is None else gkw.data_ptr(), q0, q1, q2, k0, k1, k2)
            _call("dn_norm_rotary_bwd", ws.get_device(), block, grads, ws.data_ptr(), need)
        else:   # no token, or no head
            for g in (gqw, gkw):
                if g is not None:
                    g.zero_()
        if _grad_enabled() or _forward_ad._current_level >= 0 and _differentiated(d_q, d_k):   # create_graph
            gq, gk, gqw, gkw = _NoSecondNorm.apply(gq, gk, gqw, gkw, d_q, d_k, q, k, qw, kw)
        return gq, gk, gqw, gkw, None, None, None


class _NoSecondNorm(torch.autograd.Function):
    """Gradients that depend on the cotangents and the inputs, whose own gradient is refused."""

    @staticmethod
    def forward(ctx, gq, gk, gqw, gkw, *_):
        return gq, gk, gqw, gkw

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("norm_rotary is once_differentiable: the gradient of its gradient is not implemented.")


def norm_rotary(q, k, q_weight, k_weight, positions=None, table=None, *, eps: float = 1e-6, weight_offset: float = 0.0,
                interleaved: bool = False):
    """Queries and keys normed head by head, y = x / sqrt(mean(x^2) + eps) *
    (weight_offset + weight), and then rotated as by ``apply_rotary``, in one pass.

    q: (B, L, Hq, D) or (N, Hq, D); k: the same with Hk heads, or None (with k_weight
    None); both float32, bfloat16 or float16, channels contiguous, any other strides.
    q_weight, k_weight: (D,), both of one of these types.  weight_offset: 1 for
    weights kept as differences from 1.  positions, table, interleaved: as in
    ``apply_rotary``; neither positions nor table: no rotation.  Statistics and
    products in float32, one rounding at the end.  Differentiable in q, k and the
    weights (backwards and once; tangents are refused), of which those that want no
    gradient cost none; the weights' gradients are summed in float32 over the tokens of a
    thread and in 64 bits over threads and blocks (rounded to float32 in between), and are
    the same bits every time.  Returns (q', k') with k' None if k is None; the results are
    contiguous.
    """
    qs = q.shape
    if not (3 <= len(qs) <= 4 and q.dtype in _DT and qs[-1] > 0 and type(eps) is float and 0.0 <= eps <= 3e38 and type(weight_offset) is float
            and -3e38 <= weight_offset <= 3e38 and q_weight.dtype in _DT and q_weight.shape == qs[-1:] and q_weight.is_contiguous()
            and (k_weight is None if k is None else k_weight is not None and k.dtype is q.dtype and k.ndim == len(qs) and k.shape[:-2] == qs[:-2]
                 and k.shape[-1] == qs[-1] and k_weight.dtype is q_weight.dtype and k_weight.shape == q_weight.shape and k_weight.is_contiguous())
            and (table is None if positions is None else table is not None)):
        eps, weight_offset = _check_norm_rotary(q, k, q_weight, k_weight, positions, table, eps, weight_offset)
    ps0 = ps1 = 0
    dev = q.get_device()
    if table is not None:
        rows, R = table.shape if table.ndim == 2 else (0, 0)
        if not (table.dtype is torch.float32 and rows > 0 and 2 <= R <= qs[-1] and not R & 1 and table.is_contiguous()):
            _check_table(table, qs[-1])
        if positions.dtype not in _INT:
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}.")
        at, st = positions.shape, positions.stride()
        if at == qs[:-2]:
            ps0, ps1 = st if len(at) == 2 else (0, st[0])
        elif len(at) == 1 and at[0] == qs[-3]:
            ps1 = st[0]
        else:
            raise ValueError(f"positions {tuple(at)} must have the token dimensions of q {tuple(qs[:-2])}, or the last of them.")
    if not (q_weight.get_device() == dev >= 0 and (k is None or k.get_device() == k_weight.get_device() == dev)
            and (table is None or positions.get_device() == table.get_device() == dev)):
        _on_gpu(q, k, q_weight, k_weight, positions, table)
    flat = len(qs) == 3
    if flat:
        q, k = q[None], None if k is None else k[None]
    if q.stride(-1) != 1 or k is not None and k.stride(-1) != 1:
        q, k = _dense_channels(q), None if k is None else _dense_channels(k)
    meta = ps0, ps1, eps, weight_offset, 1 if interleaved else 0
    if _grad_enabled() and (q.requires_grad or q_weight.requires_grad or k is not None and (k.requires_grad or k_weight.requires_grad)) \
            or _forward_ad._current_level >= 0 and _differentiated(q, k, q_weight, k_weight):
        r = _NormRotaryFn.apply(q, k, q_weight, k_weight, positions, table, meta)
        q_out, k_out = r if k is not None else (r, None)
    else:
        q_out, k_out = _norm_launch(q, k, q_weight, k_weight, positions, table, meta)
    if flat:
        q_out, k_out = q_out[0], None if k_out is None else k_out[0]
    return q_out, k_out


def _check_norm_rotary(q, k, q_weight, k_weight, positions, table, eps, weight_offset):
    if q.ndim not in (3, 4):
        raise ValueError(f"q must have rank 3 (N, Hq, D) or rank 4 (B, L, Hq, D), got shape {tuple(q.shape)}.")
    if q.dtype not in _DT:
        raise ValueError(f"q must be float32, bfloat16 or float16, got {q.dtype}.")
    if k is not None and (k.ndim != q.ndim or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1] or k.dtype != q.dtype):
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} must match q {tuple(q.shape)} {q.dtype} in all but the heads.")
    if (k is None) != (k_weight is None) or (positions is None) != (table is None):
        raise ValueError("k goes with k_weight, and positions with table.")
    D = q.shape[-1]
    if D < 1:
        raise ValueError("q must have a channel.")
    _check_weights(D, *([q_weight] if k is None else [q_weight, k_weight]))
    return _check_norm(eps, weight_offset)


# ---------------------------------------------------------------------------
# paged cache
# ---------------------------------------------------------------------------

def _check_caches(k_cache, v_cache):
    shape = k_cache.shape
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.ndim != 4 or c.dtype not in _DT:
            raise ValueError(f"{name} must be a float32, bfloat16 or float16 tensor (pages, page_size, Hkv, D), got {c.dtype} {tuple(c.shape)}.")
        if c.stride(-1) != 1:
            raise ValueError(f"{name} must have contiguous channels, got strides {c.stride()}.")
    if v_cache.shape != shape or v_cache.dtype is not k_cache.dtype:
        raise ValueError(f"v_cache {tuple(v_cache.shape)} {v_cache.dtype} must match k_cache {tuple(shape)} {k_cache.dtype}.")
    return shape


def _check_pages(page_table, seq_lens, cu_seqlens, x, name):
    """Sequences, new tokens and the strides (batch, token) of new tokens `x`
    (N, H, D) or (B, T, H, D); device int32 arrays are checked by shape alone."""
    if page_table.ndim != 2 or page_table.dtype is not torch.int32 or (page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError(f"page_table must be int32 (B, max_pages) with contiguous rows, got {page_table.dtype} {tuple(page_table.shape)}.")
    B = page_table.shape[0]
    if seq_lens.shape != (B,) or seq_lens.dtype is not torch.int32 or not seq_lens.is_contiguous():
        raise ValueError(f"seq_lens must be a contiguous int32 tensor ({B},), got {seq_lens.dtype} {tuple(seq_lens.shape)}.")
    if x.ndim == 4:
        if cu_seqlens is not None:
            raise ValueError(f"cu_seqlens goes with {name} of rank 3 (N, H, D), got shape {tuple(x.shape)}.")
        if x.shape[0] != B:
            raise ValueError(f"{name} batch dimension ({x.shape[0]}) must match page_table ({B}).")
        return B, B * x.shape[1], x.stride(0), x.stride(1)
    if x.ndim != 3:
        raise ValueError(f"{name} must have rank 3 (N, H, D) or rank 4 (B, T, H, D), got shape {tuple(x.shape)}.")
    if cu_seqlens is None:
        if x.shape[0] != B:
            raise ValueError(f"{name} of rank 3 without cu_seqlens has one token per sequence ({B}), got {x.shape[0]}.")
    elif cu_seqlens.shape != (B + 1,) or cu_seqlens.dtype is not torch.int32 or not cu_seqlens.is_contiguous():
        raise ValueError(f"cu_seqlens must be a contiguous int32 tensor ({B + 1},), got {cu_seqlens.dtype} {tuple(cu_seqlens.shape)}.")
    return B, x.shape[0], x.stride(0), x.stride(0)


def paged_kv_append(k, v, k_cache, v_cache, page_table, seq_lens, *, cu_seqlens=None, table=None, interleaved: bool = False):
    """Stores the keys and values of new tokens in a paged cache, the keys rotated
    by their positions when ``table`` (``rotary_table``) is given.

    k, v: (N, Hkv, D) with ``cu_seqlens`` (B + 1) int32 (where each sequence's new
    tokens start), (B, Hkv, D) for one token per sequence, or (B, T, Hkv, D).
    k_cache, v_cache: (pages, page_size, Hkv, D), page_size a power of two, any
    strides of the first three axes, written in place (rounded to the cache's
    type).  page_table: int32 (B, max_pages), the pages of each sequence in order.
    seq_lens: int32 (B,), each sequence's tokens, the new ones included: new token
    i of n has position seq_lens - n + i.  A token whose position is negative or
    past the page table, or whose page is outside the cache, is not stored; a
    position outside ``table`` stores NaN in the rotated channels.  Pages that are
    written must not be shared.  Returns (k_cache, v_cache).
    """
    pages, page, H, D = _check_caches(k_cache, v_cache)
    if page < 1 or page & (page - 1):
        raise ValueError(f"page_size must be a power of two, got {page}.")
    if k.dtype not in _DT or v.dtype is not k.dtype or v.shape != k.shape:
        raise ValueError(f"k and v must be of one shape and float32, bfloat16 or float16, got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}.")
    if k.shape[-2:] != (H, D):
        raise ValueError(f"k {tuple(k.shape)} must have the cache's heads and channels ({H}, {D}).")
    dev = _on_gpu(k, v, k_cache, v_cache, page_table, seq_lens, cu_seqlens, table)
    k, v = _dense_channels(k), _dense_channels(v)
    B, N, ksb, kst = _check_pages(page_table, seq_lens, cu_seqlens, k, "k")
    R = _check_table(table, D) if table is not None else 0
    vs, kcs, vcs = v.stride(), k_cache.stride(), v_cache.stride()
    if _differentiated(k, v, k_cache, v_cache):
        raise ValueError("paged_kv_append is not differentiable; call it under torch.no_grad().")
    if N and pages:
        block = _lib.KV_APPEND_PACK(
            _lib.DN_ABI_VERSION, N, B, H, D, R, _DT[k.dtype], _DT[k_cache.dtype], 1 if interleaved else 0, table.shape[0] if R else 0,
            pages, page, page_table.shape[1], k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            page_table.data_ptr(), seq_lens.data_ptr(), 0 if cu_seqlens is None else cu_seqlens.data_ptr(),
            table.data_ptr() if R else 0, ksb, kst, k.stride(-2), vs[0], vs[0] if v.ndim == 3 else vs[1], vs[-2],
            kcs[0], kcs[1], kcs[2], vcs[0], vcs[1], vcs[2], page_table.stride(0))
        _call("dn_kv_append", dev, block)
        # autograd sees the store (inference tensors have no version)
        _bump([c for c in (k_cache, v_cache) if not c.is_inference()])
    return k_cache, v_cache


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _rows16(t):
    """A tensor whose rows of channels start on 16 bytes, as the kernels read them."""
    s, per = t.stride(), 16 // t.element_size()
    if s[-1] == 1 and t.data_ptr() % 16 == 0 and not any(x % per for x in s[:-1]):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _attention_common(D, Hq, Hkv, dtype, scale, window):
    if D not in (64, 128, 256):
        raise ValueError(f"Unsupported head dimension {D}; attention takes 64, 128 or 256.")
    if dtype not in _DT:
        raise ValueError(f"attention takes float32, bfloat16 or float16, got {dtype}.")
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"Query heads ({Hq}) must be divisible by key heads ({Hkv}).")
    if window is not None and (isinstance(window, bool) or not isinstance(window, int) or window < 1):
        raise ValueError(f"window must be a positive integer or None, got {window!r}.")
    if scale is None:
        return 1.0 / math.sqrt(D)
    try:
        scale = float(scale)
    except (TypeError, ValueError) as e:
        raise ValueError(f"scale must be convertible to a concrete float, got {type(scale)}: {e}")
    if not abs(scale) <= 2.0 ** 127:   # (its product with log2(e) is a float32)
        raise ValueError(f"scale must be finite in float32, got {scale}.")
    return scale


def _window(window):
    return min(window or 0, 0x7fffffff)   # (rows are shorter)


def paged_attention(q, k_cache, v_cache, page_table, seq_lens, *, cu_seqlens=None, scale=None, window=None,
                    return_lse: bool = False):
    """Causal attention of new tokens over a paged cache that holds their keys and
    values already (``paged_kv_append``): single tokens, drafts, prompts in chunks,
    and any mixture of them in one call.

    q: (N, Hq, D) with ``cu_seqlens`` (B + 1) int32, (B, Hq, D) for one token per
    sequence, or (B, T, Hq, D); D 64, 128 or 256; the cache's type.  Caches,
    page_table and seq_lens as in ``paged_kv_append``; query head h reads key head
    h // (Hq // Hkv).  A query at position p sees positions 0 .. p, or the last
    ``window`` of them; a length past the page table counts as the table's end.  scale: any finite number, 1 / sqrt(D) unless given.  Sums and
    softmax statistics in float32 (which the sums stay within as long as the largest value
    times the tokens that a query sees is below 2^120); probabilities of 16-bit types are
    rounded to the type once before their product with the values.  A query without a key gets zeros (lse -inf), and
    so do tokens in front of cu_seqlens[0] and from cu_seqlens[-1] on (a batch of fixed
    size that is not full); in between cu_seqlens must not fall.  Returns the output in
    q's shape and type, and with ``return_lse`` also the log of the sum of exponentials
    (float32, q's shape without D).
    """
    pages, page, Hkv, D = _check_caches(k_cache, v_cache)
    if page < 1 or page & (page - 1) or pages < 1:
        raise ValueError(f"page_size must be a power of two and the cache have a page, got {tuple(k_cache.shape)}.")
    if q.dtype is not k_cache.dtype or q.shape[-1] != D:
        raise ValueError(f"q {tuple(q.shape)} {q.dtype} must have the cache's channels and type ({D}, {k_cache.dtype}).")
    dev = _on_gpu(q, k_cache, v_cache, page_table, seq_lens, cu_seqlens)
    if _differentiated(q, k_cache, v_cache):
        raise ValueError("paged_attention is not differentiable; use causal_attention for training.")
    q = _rows16(q)
    B, N, qsb, qst = _check_pages(page_table, seq_lens, cu_seqlens, q, "q")
    Hq = q.shape[-2]
    scale = _attention_common(D, Hq, Hkv, q.dtype, scale, window)
    kcs, vcs = k_cache.stride(), v_cache.stride()
    if (k_cache.data_ptr() | v_cache.data_ptr() | (kcs[0] | kcs[1] | kcs[2] | vcs[0] | vcs[1] | vcs[2]) * q.element_size()) & 15:
        raise ValueError(f"cache rows must start on 16 bytes, got strides {kcs} and {vcs}.")
    if page_table.shape[1] < 1:
        raise ValueError("page_table must have a column.")
    out = q.new_empty(q.shape)
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device) if return_lse else None
    block = _lib.PAGED_ATTENTION_PACK(
        _lib.DN_ABI_VERSION, N, B, Hq, Hkv, D, _DT[q.dtype], _window(window), pages, page, page_table.shape[1], scale,
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
        page_table.data_ptr(), seq_lens.data_ptr(), 0 if cu_seqlens is None else cu_seqlens.data_ptr(),
        qsb, qst, q.stride(-2), kcs[0], kcs[1], kcs[2], vcs[0], vcs[1], vcs[2], page_table.stride(0))
    if N:
        need = (_calls.get("dn_paged_attention_workspace_size") or _lib.packed_call("dn_paged_attention_workspace_size"))(block)
        ws = q.new_empty(-(-need // q.element_size())) if need else None
        _call("dn_paged_attention", dev, block, 0 if ws is None else ws.data_ptr(), need)
    return (out, lse) if return_lse else out


def _document_starts(segment_ids, cu_seqlens, B, L, dev):
    """(B, L) int32 first token of each token's document (checks and messages as in
    ``chunk_gdn2``)."""
    if segment_ids is not None and cu_seqlens is not None:
        raise ValueError("Cannot pass both segment_ids and cu_seqlens; specify at most one.")
    if segment_ids is not None:
        seg = segment_ids if isinstance(segment_ids, torch.Tensor) else torch.as_tensor(np.asarray(segment_ids))
        if not _is_integer_dtype(seg.dtype):
            raise ValueError(f"segment_ids must have integer dtype, got {seg.dtype}.")
        if seg.ndim == 1:
            if seg.shape[0] != L:
                raise ValueError(f"1D segment_ids length ({seg.shape[0]}) must match sequence length ({L}).")
        elif seg.ndim == 2:
            if tuple(seg.shape) != (B, L):
                raise ValueError(f"2D segment_ids shape {tuple(seg.shape)} must match (B={B}, L={L}).")
        else:
            raise ValueError(f"segment_ids must be 1D (L,) or 2D (B, L), got rank {seg.ndim} with shape {tuple(seg.shape)}.")
        if seg.dtype not in _INT:
            seg = seg.to(torch.int64)
    else:
        cu = cu_seqlens.detach().cpu().numpy() if isinstance(cu_seqlens, torch.Tensor) else np.asarray(cu_seqlens)
        if len(cu) == 0 or int(cu[0]) != 0:
            raise ValueError(f"cu_seqlens[0] must be 0, got {cu[0] if len(cu) else 'empty'}.")
        if int(cu[-1]) != L:
            raise ValueError(f"cu_seqlens[-1] ({int(cu[-1])}) must equal sequence length ({L}).")
        lens = np.diff(cu.astype(np.int64))
        if len(lens) > 0 and np.any(lens <= 0):
            raise ValueError(f"cu_seqlens must be strictly monotonically increasing, got {cu_seqlens}.")
        seg = torch.from_numpy(np.repeat(np.arange(len(lens), dtype=np.int32), lens))
    seg = seg.to(dev).contiguous()
    starts = torch.empty((B, L), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.load_library().dn_document_starts(seg.data_ptr(), _INT[seg.dtype], int(seg.ndim == 2), B, L,
                                                          starts.data_ptr(), _raw_stream(dev.index)), "dn_document_starts")
    return starts


def _attention_block(q, k, v, out, low, lse, starts, scale, window):
    B, L, Hq, D = q.shape
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    return _lib.ATTENTION_PACK(
        _lib.DN_ABI_VERSION, B, L, Hq, k.shape[2], D, _DT[q.dtype], _window(window), scale, q.data_ptr(), k.data_ptr(),
        v.data_ptr(), out.data_ptr(), 0 if low is None else low.data_ptr(), 0 if lse is None else lse.data_ptr(), 0 if starts is None else starts.data_ptr(),
        qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2])


def _attention_forward(q, k, v, starts, scale, window, want_lse, want_low=False):
    out = q.new_empty(q.shape)
    low = q.new_empty(q.shape) if want_low else None
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device) if want_lse else None
    if q.numel():
        _call("dn_attention_fwd", q.get_device(), _attention_block(q, k, v, out, low, lse, starts, scale, window))
    return out, low, lse


class _NoSecond(torch.autograd.Function):
    """Gradients that depend on d_out, q, k and v, whose own gradient is refused."""

    @staticmethod
    def forward(ctx, dq, dk, dv, d_out, q, k, v):
        return dq, dk, dv

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("causal_attention is once_differentiable: the gradient of its gradient is not implemented.")


class _AttentionFn(torch.autograd.Function):
    """Causal attention under autograd: the forward keeps the log of each row's sum
    of exponentials, from which the backward recomputes the probabilities, and what
    rounding cut off the output, which the backward's row sums read with it."""

    @staticmethod
    def forward(ctx, q, k, v, starts, scale, window):
        out, low, lse = _attention_forward(q, k, v, starts, scale, window, True, q.dtype is not torch.float32)
        ctx.save_for_backward(q, k, v, out, low, lse, starts)
        ctx.meta = scale, window
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    def backward(ctx, d_out, _):
        q, k, v, out, low, lse, starts = ctx.saved_tensors
        scale, window = ctx.meta
        if d_out is None:
            return (None,) * 6
        d_out = _rows16(d_out.contiguous())   # (a concatenation hands out slices that start anywhere)
        dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        if q.numel():
            block = _attention_block(q, k, v, out, low, lse, starts, scale, window)
            need = _lib.packed_call("dn_attention_bwd_workspace_size")(block)
            ws = q.new_empty(-(-need // q.element_size()))
            _call("dn_attention_bwd", q.get_device(), block, d_out.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                  ws.data_ptr(), need)
        if torch.is_grad_enabled() or _differentiated(d_out):   # create_graph
            dq, dk, dv = _NoSecond.apply(dq, dk, dv, d_out, q, k, v)
        return dq, dk, dv, None, None, None


def causal_attention(q, k, v, *, segment_ids=None, cu_seqlens=None, scale=None, window=None, return_lse: bool = False):
    """Causal softmax attention of whole rows.

    q: (B, L, Hq, D); k, v: (B, L, Hkv, D) with Hkv dividing Hq; one of float32,
    bfloat16 and float16; D 64, 128 or 256.  Documents by ``segment_ids`` or
    ``cu_seqlens`` as in ``chunk_gdn2``: token i sees the tokens of its document up
    to itself, or the last ``window`` of them.  scale: any finite number,
    1 / sqrt(D) unless given.  Sums and softmax statistics in float32.  Returns the
    output in q's shape and type, and with ``return_lse`` also the log of the sum of
    exponentials (B, L, Hq) in float32.  Differentiable in q, k and v (backwards and
    once, not through the lse); gradients come in the inputs' type, those of k and v summed over the heads
    that share them, and are the same bits every time.
    """
    if q.ndim != 4:
        raise ValueError(f"Query tensor q must be 4D (B, L, Hq, D), got shape {tuple(q.shape)}.")
    B, L, Hq, D = q.shape
    if k.ndim != 4 or k.shape[:2] != (B, L) or k.shape[3] != D:
        raise ValueError(f"Key tensor k {tuple(k.shape)} must match query q {tuple(q.shape)} in all but the heads.")
    if v.shape != k.shape:
        raise ValueError(f"Value tensor v shape {tuple(v.shape)} must match key k shape {tuple(k.shape)}.")
    if k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise ValueError(f"q, k and v must be of one type, got {q.dtype}, {k.dtype} and {v.dtype}.")
    scale = _attention_common(D, Hq, k.shape[2], q.dtype, scale, window)
    _on_gpu(q, k, v, segment_ids if isinstance(segment_ids, torch.Tensor) else None)
    starts = None
    if segment_ids is not None or cu_seqlens is not None:
        starts = _document_starts(segment_ids, cu_seqlens, B, L, q.device)
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    if _differentiated(q, k, v):
        out, lse = _AttentionFn.apply(q, k, v, starts, scale, window)
    else:
        out, _, lse = _attention_forward(q, k, v, starts, scale, window, return_lse)
    return (out, lse) if return_lse else out
