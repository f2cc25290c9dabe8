"""Norms of queries and keys for each head with the position rotation.

An extension: the reference's entry points take q and k as they are.  The rows come out laid
out as the attention entry points read them, in one pass over q and k, and the call is
differentiable in q, k and the gains (fmlm_norm_rope / fmlm_norm_rope_bwd,
include/flash_mlm_hip.h).
"""

from __future__ import annotations

import math

import torch

from flash_mlm import _lib
from flash_mlm.host.cache import PackMetadata
from flash_mlm.host.host import _wants_grad, rows16
from flash_mlm.host.host_utils import _device_scope, require_cuda_tensors, validate_head_dim_supported

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_INTS = (torch.int32, torch.int64)


def aligned16(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and 16-byte aligned (a copy where it is not)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _Call:
    """The checked arguments of one call, and its parameter blocks."""

    __slots__ = ("shapes", "heads", "layout", "B", "N", "D", "rows", "flags", "eps", "cu", "tokens", "table_rows", "R")

    def params(self, xs, ws, cos, sin, positions, context_lens):
        p = _lib.NormRopeParams()
        p.dtype = _lib.dtype_code(xs[0].dtype)
        w = ws[0] if ws[0] is not None else ws[1]
        p.w_dtype = _lib.DTYPE_F32 if w is None else _lib.dtype_code(w.dtype)
        p.flags, p.layout = self.flags, self.layout
        p.B, p.N, p.D, p.rotary_dim = self.B, self.N, self.D, self.R
        p.rows, p.table_rows, p.eps = self.rows, self.table_rows, self.eps
        p.cos, p.sin = _lib.ptr(cos), _lib.ptr(sin)
        p.cu_seqlens, p.token_indices = _lib.ptr(self.cu), _lib.ptr(self.tokens)
        p.positions, p.offsets = _lib.ptr(positions), _lib.ptr(context_lens)
        return p

    def strides(self, x: torch.Tensor):
        if self.layout == _lib.LAYOUT_PACKED:
            return 0, self.rows * self.D, self.D
        return x.stride(0), x.stride(1), x.stride(2)

    def tensor(self, t, i: int, x, y, w, dy=None, dw=None) -> None:
        t.heads = self.heads[i]
        t.x, (t.x_sb, t.x_sh, t.x_sn) = x.data_ptr(), self.strides(x)
        t.y, (t.y_sb, t.y_sh, t.y_sn) = y.data_ptr(), self.strides(y)
        if dy is not None:
            t.dy, (t.dy_sb, t.dy_sh, t.dy_sn) = dy.data_ptr(), self.strides(dy)
        if w is not None:
            t.weight = w.data_ptr()
            t.w_sh = self.D if w.ndim == 2 else 0
        t.dweight = _lib.ptr(dw)


def _forward(call: _Call, q, k, wq, wk, cos, sin, positions, context_lens):
    outs = [torch.empty(s, dtype=q.dtype, device=q.device) for s in call.shapes]
    if call.rows:
        p = call.params((q, k), (wq, wk), cos, sin, positions, context_lens)
        call.tensor(p.q, 0, q, outs[0], wq)
        call.tensor(p.k, 1, k, outs[1], wk)
        with _device_scope(q.device):
            rc = _lib.load().fmlm_norm_rope(p, _lib.stream_of(q.device))
        _lib.check(rc, "fmlm_norm_rope")
    return tuple(outs)


def _backward(call: _Call, xs, ws, angles, dys, needs):
    """Gradients (dq, dk, dwq, dwk); ``needs`` says which are wanted, None in ``dys`` is zero."""
    lib = _lib.load()
    dev = xs[0].device
    p = call.params(xs, ws, *angles)
    dxs, dws, keep = [None, None], [None, None], []
    for i, t in enumerate((p.q, p.k)):
        if dys[i] is None or not (needs[i] or needs[2 + i]):
            continue
        dy = rows16(dys[i])
        dxs[i] = torch.empty(call.shapes[i], dtype=xs[i].dtype, device=dev)
        if ws[i] is not None and needs[2 + i]:
            dws[i] = torch.empty(ws[i].shape, dtype=ws[i].dtype, device=dev)
        call.tensor(t, i, xs[i], dxs[i], ws[i], dy, dws[i])
        keep.append(dy)
    if keep:
        nbytes = int(lib.fmlm_norm_rope_bwd_workspace_bytes(p))
        _lib.check(nbytes if nbytes < 0 else 0, "fmlm_norm_rope_bwd_workspace_bytes")
        ws_buf = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        p.workspace, p.workspace_bytes = ws_buf.data_ptr(), nbytes
        with _device_scope(dev):
            rc = lib.fmlm_norm_rope_bwd(p, _lib.stream_of(dev))
        _lib.check(rc, "fmlm_norm_rope_bwd")
    return (*dxs, *dws)


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, call, q, k, wq, wk, cos, sin, positions, context_lens):
        ctx.call = call
        ctx.set_materialize_grads(False)
        # saved so that autograd rejects a backward after any of them changed in place
        ctx.save_for_backward(q, k, wq, wk, cos, sin, positions, context_lens)
        return _forward(call, q, k, wq, wk, cos, sin, positions, context_lens)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        q, k, wq, wk, *angles = ctx.saved_tensors
        grads = _backward(ctx.call, (q, k), (wq, wk), angles, (dq, dk), ctx.needs_input_grad[1:5])
        return (None, *grads, None, None, None, None)


def _accumulator(leaf: torch.Tensor):
    """The node that autograd delivers the leaf's gradient to: one for all live graphs."""
    return leaf.view_as(leaf).grad_fn.next_functions[0][0]


def _capture_leaves(*tensors) -> list[torch.Tensor]:
    """The leaves among ``tensors`` when the current stream is being captured (else none), checked.

    Autograd runs a leaf's accumulator on the stream of the graph that made it.  When that is an
    eager graph on the default stream, a captured backward drags the default stream into the
    capture, which ends the process when the capture ends.  An accumulator outlives its
    last reference here exactly when another live graph holds it.
    """
    if not torch.cuda.is_current_stream_capturing():
        return []
    leaves = [t for t in tensors if t is not None and t.requires_grad and t.is_leaf]
    for t in leaves:
        token = object()
        _accumulator(t).metadata["fmlm_probe"] = token
        node = _accumulator(t)
        if node.metadata.get("fmlm_probe") is token and "fmlm_captured" not in node.metadata:
            raise ValueError(
                "qk_norm_rope is being captured into a graph while another autograd graph of one of its leaves "
                "lives: drop the outputs of the earlier calls on it first"
            )
    return leaves


def _check_gain(w, what: str, heads: int, d: int, device):
    if w is None:
        return None
    if tuple(w.shape) not in ((d,), (heads, d)):
        raise ValueError(f"{what} must be [head_dim] or [heads, head_dim]")
    if w.dtype not in _FLOATS or w.device != device:
        raise ValueError(f"{what} must be bf16, fp16 or fp32 on the device of q and k")
    return aligned16(w)


def _check_index(t, what: str, shape, device, lo_hi=None):
    """An int32 / int64 tensor on ``device``; one on the CPU is range-checked and copied."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype not in _INTS or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must be an int32 or int64 tensor of shape {tuple(shape)}")
    if not t.is_cuda and lo_hi is not None and t.numel():
        if int(t.min()) < lo_hi[0] or int(t.max()) >= lo_hi[1]:
            raise ValueError(f"{what} values must lie in [{lo_hi[0]}, {lo_hi[1]})")
    return t.to(device).contiguous()


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    *,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    norm: bool = True,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    context_lens: torch.Tensor | None = None,
    interleaved: bool = False,
    q_meta: PackMetadata | None = None,
    num_heads: int | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head's queries and keys, then the rotation of their positions.

    q [B, H, N, D] and k [B, H_k, N, D], or packed [H*T, D] and [H_k*T, D] (head-major; T =
    ``q_meta.total_tokens``, or without ``q_meta`` one sequence of T = rows / ``num_heads``
    tokens).  Returns contiguous tensors of the same shapes.  A row x of D elements becomes, in
    fp32 and rounded once,

      n = x * (mean(x^2) + eps)^-1/2 * gain              (``norm=False``: n = x)
      pairs (a, b) of n's first R elements -> (a cos - b sin, a sin + b cos)

    ``q_weight`` / ``k_weight``: gains [D] or for each head [H, D] (None: 1), of one dtype.
    ``cos`` / ``sin``: fp32 tables [positions, R/2], R <= D a multiple of 16 (None: no
    rotation).  Pair i is elements (i, i + R/2), with ``interleaved`` (2i, 2i + 1).  A token's
    row of the tables is its entry of ``positions`` ([B, N]; [T] with ``q_meta`` or packed
    rows), or its place p in its sequence plus ``context_lens[b]`` (tokens that precede the
    sequence in its context).  Positions on the CPU are range-checked; on the GPU they are
    not read back, and the kernel clamps them to the tables.

    With ``q_meta``, rows of padding tokens come out as zeros, whatever they held.
    Differentiable in q, k and the gains; gradients of padding rows are zero.  A call captured
    into a graph together with its backward raises ValueError while outputs of earlier calls
    on the same leaves are alive (autograd would run part of the backward on their stream).
    """
    for t in (q, k):
        if t.ndim not in (2, 4) or t.ndim != q.ndim:
            raise ValueError("q and k must both be rank-4 [B, H, N, D] or packed rank-2 [H*T, D]")
    d = int(q.shape[-1])
    if int(k.shape[-1]) != d:
        raise ValueError("q and k must have the same head_dim")
    validate_head_dim_supported(d, is_mla=True)
    if q.dtype not in _FLOATS or k.dtype != q.dtype:
        raise ValueError("q and k must be of one dtype: bf16, fp16 or fp32")
    if k.device != q.device:
        raise ValueError("q and k must be on one device")
    require_cuda_tensors(q, k, q_weight, k_weight, cos, sin)
    dev = q.device
    if q_meta is not None and q_meta.cu_seqlens.device != dev:
        raise ValueError("q_meta must be on the device of q and k")

    c = _Call()
    c.D, c.cu, c.tokens = d, None, None
    if q.ndim == 4:
        b, _, n, _ = (int(x) for x in q.shape)
        if (int(k.shape[0]), int(k.shape[2])) != (b, n):
            raise ValueError("q and k must have the same batch and length")
        if q_meta is not None:
            if q_meta.B != b or q_meta.N != n:
                raise ValueError("q_meta shape metadata does not match q/k padded shape")
            c.cu = q_meta.cu_seqlens
        if num_heads is not None and num_heads != int(q.shape[1]):
            raise ValueError("q head dimension must match num_heads")
        c.layout, c.B, c.N, c.rows = _lib.LAYOUT_PADDED, b, n, b * n
        c.heads = (int(q.shape[1]), int(k.shape[1]))
        pos_shape = (b, n) if q_meta is None else (int(q_meta.total_tokens),)
    else:
        if q_meta is not None:
            b, n, t = q_meta.B, q_meta.N, int(q_meta.total_tokens)
            c.cu, c.tokens = q_meta.cu_seqlens, q_meta.token_indices
        else:
            if num_heads is None or num_heads < 1 or int(q.shape[0]) % num_heads:
                raise ValueError("packed q needs q_meta, or num_heads that divides its rows")
            b, t = 1, int(q.shape[0]) // num_heads
            n = t
        c.heads = tuple(int(x.shape[0]) // t if t else 0 for x in (q, k))
        if any(int(x.shape[0]) != h * t for x, h in zip((q, k), c.heads)):
            raise ValueError("packed q and k rows must be a multiple of the token count")
        if num_heads is not None and t and num_heads != c.heads[0]:
            raise ValueError("q first dim must equal num_heads * tokens")
        c.layout, c.B, c.N, c.rows = _lib.LAYOUT_PACKED, b, n, t
        pos_shape = (t,)
    c.shapes = (tuple(q.shape), tuple(k.shape))
    if c.B * c.N > 0x7FFFFFFF:
        raise ValueError("q and k must have fewer than 2**31 tokens")

    if not norm and (q_weight is not None or k_weight is not None):
        raise ValueError("gains need norm=True")
    if not norm and cos is None:
        raise ValueError("nothing to do: norm=False and no cos/sin tables")
    if norm and not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and >= 0")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight must have the same dtype")
    wq = _check_gain(q_weight, "q_weight", c.heads[0], d, dev)
    wk = _check_gain(k_weight, "k_weight", c.heads[1], d, dev)

    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    c.R, c.table_rows = 0, 0
    if cos is not None:
        if cos.ndim != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32 \
                or cos.device != dev or sin.device != dev:
            raise ValueError("cos and sin must be fp32 tables [positions, rotary_dim / 2] on the device of q and k")
        c.table_rows, c.R = int(cos.shape[0]), 2 * int(cos.shape[1])
        if c.R < 16 or c.R % 16 or c.R > d or c.table_rows < 1:
            raise ValueError("rotary_dim must be a multiple of 16 and at most head_dim, with at least one position")
        cos, sin = aligned16(cos), aligned16(sin)
    elif positions is not None or context_lens is not None:
        raise ValueError("positions and context_lens need cos and sin")
    if positions is not None and context_lens is not None:
        raise ValueError("positions and context_lens are mutually exclusive")
    positions = _check_index(positions, "positions", pos_shape, dev, (0, c.table_rows))
    context_lens = _check_index(context_lens, "context_lens", (c.B,), dev, (0, c.table_rows))

    c.eps = float(eps)
    c.flags = (_lib.NR_NORM if norm else 0) | (_lib.NR_INTERLEAVED if interleaved else 0)
    if positions is not None and positions.dtype == torch.int64:
        c.flags |= _lib.NR_POSITIONS_I64
    if context_lens is not None and context_lens.dtype == torch.int64:
        c.flags |= _lib.NR_OFFSETS_I64
    args = (c, rows16(q), rows16(k), wq, wk, cos, sin, positions, context_lens)
    if _wants_grad(q, k, q_weight, k_weight):
        leaves = _capture_leaves(q, k, q_weight, k_weight)
        out = _NormRope.apply(*args)
        for t in leaves:  # this capture's own graph: later calls of it may share the leaf
            _accumulator(t).metadata["fmlm_captured"] = True
        return out
    return _forward(*args)
