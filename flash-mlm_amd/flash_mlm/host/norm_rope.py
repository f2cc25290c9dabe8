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
from flash_mlm.host.host_utils import (
    aligned16,
    capture_leaves,
    keep_leaves,
    pack_indices,
    refuse_tangents,
    require_cuda_tensors,
    rows16,
    validate_head_dim_supported,
)

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_INTS = (torch.int32, torch.int64)
_HEAD_DIMS = (16, 32, 64, 128, 256, 512)


class _Call:
    """The checked arguments of one call as a parameter block without the rows' addresses."""

    __slots__ = ("block", "packed", "keep", "sizes")

    def put(self, t, x, y) -> None:
        """Rows in and out of tensor ``t`` of a block (packed rows: strides are the block's)."""
        t.x, t.y = x.data_ptr(), y.data_ptr()
        if not self.packed:
            t.x_sb, t.x_sh, t.x_sn, _ = x.stride()


# ---------------------------------------------------------------------------
# Launch memo, as of the attention entry points (host.py): kept on the PackMetadata, in a
# module-level table for calls without one.  A key holds everything that the checks and the parameter
# block depend on but addresses; an entry the block and the metadata's index tensors.
# ---------------------------------------------------------------------------
_MEMO_MAX = 16
_MEMO: dict = {}


def _layout(t):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):  # refused below
        return type(t)
    return t.shape, t.stride(), t.dtype, t.device, t.data_ptr() & 15


class _Memo:
    __slots__ = ("block", "packed", "keep", "sizes", "meta")

    def __init__(self, call: _Call, q_meta):
        self.block = _lib.NormRopeParams.from_buffer_copy(call.block)
        self.packed, self.keep, self.sizes = call.packed, call.keep, call.sizes
        self.meta = None
        if q_meta is not None:
            self.meta = (q_meta.cu_seqlens, q_meta.token_indices, q_meta.total_tokens, q_meta.B, q_meta.N)

    def fits(self, q_meta) -> bool:
        """Whether ``q_meta`` still is what the entry was made for (its fields can be replaced)."""
        m = self.meta
        return m is None or (m[0] is q_meta.cu_seqlens and m[1] is q_meta.token_indices
                             and m[2:] == (q_meta.total_tokens, q_meta.B, q_meta.N))

    def call_for(self, wq, wk, cos, sin, idx, offsets: bool) -> _Call:
        call = _Call()
        p = call.block = _lib.NormRopeParams.from_buffer_copy(self.block)
        call.packed, call.keep, call.sizes = self.packed, self.keep, self.sizes
        if wq is not None:
            p.q.weight = wq.data_ptr()
        if wk is not None:
            p.k.weight = wk.data_ptr()
        if cos is not None:
            p.cos, p.sin = cos.data_ptr(), sin.data_ptr()
        if idx is not None:
            if offsets:
                p.offsets = idx.data_ptr()
            else:
                p.positions = idx.data_ptr()
        return call


def _out(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _run(entry, name: str, p, device) -> None:
    if device.index == torch.cuda.current_device():
        rc = entry(p, _lib.stream_of(device))
    else:
        with torch.cuda.device(device):
            rc = entry(p, _lib.stream_of(device))
    if rc:
        _lib.check(rc, name)


def _forward(call: _Call, q, k):
    outs = _out(q), _out(k)
    p = call.block
    if p.rows:
        call.put(p.q, q, outs[0])
        call.put(p.k, k, outs[1])
        _run(_lib.load().fmlm_norm_rope, "fmlm_norm_rope", p, q.device)
    return outs


def _saved(t: torch.Tensor, size: int, dtype, device: int, layout) -> torch.Tensor:
    """``t`` of the saved tensors as the kernel reads it (``layout`` of it where it is not)."""
    if t.numel() != size or t.dtype is not dtype or t.get_device() != device:
        raise RuntimeError("qk_norm_rope: a saved tensor came back with another size or type, or on another device")
    return t if t.is_contiguous() and not t.data_ptr() & 15 else layout(t)


def _rebind(call: _Call, p, saved) -> tuple:
    """Rows and gains of the saved tensors, and the block's other addresses from them.  They need not be where
    the forward's were: a checkpoint recomputes them and a saved-tensor hook brings copies, laid out
    as it likes.  The last of the tuple is held until the launch."""
    q, k, wq, wk, cos, sin, positions, context_lens = saved
    nq, nk, dtype, nwq, nwk, w_dtype, table, indices, i_dtype, dev = call.sizes
    layout = aligned16 if call.packed else rows16
    q, k = _saved(q, nq, dtype, dev, layout), _saved(k, nk, dtype, dev, layout)
    if wq is not None:
        wq = _saved(wq, nwq, w_dtype, dev, aligned16)
        p.q.weight = wq.data_ptr()
    if wk is not None:
        wk = _saved(wk, nwk, w_dtype, dev, aligned16)
        p.k.weight = wk.data_ptr()
    index = positions if positions is not None else context_lens
    if cos is not None:
        cos = _saved(cos, table, torch.float32, dev, aligned16)
        sin = _saved(sin, table, torch.float32, dev, aligned16)
        p.cos, p.sin = cos.data_ptr(), sin.data_ptr()
        if index is not None:
            index = _saved(index, indices, i_dtype, dev, aligned16)
            if positions is not None:
                p.positions = index.data_ptr()
            else:
                p.offsets = index.data_ptr()
    return (q, k), (wq, wk), (cos, sin, index)


def _backward(call: _Call, saved, dys, needs):
    """Gradients (dq, dk, dwq, dwk); ``needs`` says which are wanted, None in ``dys`` is zero."""
    lib = _lib.load()
    dev = saved[0].device
    p = _lib.NormRopeParams.from_buffer_copy(call.block)  # (a graph can be walked more than once)
    if p.rows == 0:
        return tuple(torch.zeros_like(t) if n else None for t, n in zip(saved, needs))
    xs, ws, _tables = _rebind(call, p, saved)
    dxs, dws, keep = [None, None], [None, None], []
    for i, t in enumerate((p.q, p.k)):
        if dys[i] is None or not (needs[i] or needs[2 + i]):
            t.heads = 0
            continue
        dy = aligned16(dys[i]) if call.packed else rows16(dys[i])
        dx = dxs[i] = _out(xs[i])
        call.put(t, xs[i], dx)
        t.dy = dy.data_ptr()
        if call.packed:
            t.dy_sh, t.dy_sn = t.y_sh, t.y_sn
        else:
            t.dy_sb, t.dy_sh, t.dy_sn, _ = dy.stride()
        if needs[2 + i]:
            dw = dws[i] = torch.empty_like(ws[i])
            t.dweight = dw.data_ptr()
        keep.append(dy)
    if keep:
        nbytes = lib.fmlm_norm_rope_bwd_workspace_bytes(p)
        _lib.check(nbytes if nbytes < 0 else 0, "fmlm_norm_rope_bwd_workspace_bytes")
        buf = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        p.workspace, p.workspace_bytes = buf.data_ptr(), nbytes
        _run(lib.fmlm_norm_rope_bwd, "fmlm_norm_rope_bwd", p, dev)
    return (*dxs, *dws)


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, call, q, k, wq, wk, cos, sin, positions, context_lens):
        ctx.call = call
        ctx.set_materialize_grads(False)
        # saved so that autograd rejects a backward after any of them changed in place, and read
        # from there: autograd may free these and bring others (_rebind)
        ctx.save_for_backward(q, k, wq, wk, cos, sin, positions, context_lens)
        return _forward(call, q, k)

    @staticmethod
    def backward(ctx, dq, dk):
        # grad mode: create_graph, where the gradients must refuse to be differentiated.  (Without
        # it the wrapper's grad-mode switches alone took 5 us of a 117 us training call.)
        return (_backward_once if torch.is_grad_enabled() else _backward_node)(ctx, dq, dk)


def _backward_node(ctx, dq, dk):
    grads = _backward(ctx.call, ctx.saved_tensors, (dq, dk), ctx.needs_input_grad[1:5])
    return (None, *grads, None, None, None, None)


_backward_once = torch.autograd.function.once_differentiable(_backward_node)


def _capture_leaves(*tensors) -> list[torch.Tensor]:
    return capture_leaves("qk_norm_rope", *tensors)


def _check_gain(w, what: str, heads: int, d: int, device):
    ws = w.shape
    if ws[-1:] != (d,) or not (len(ws) == 1 or (len(ws) == 2 and ws[0] == heads)):
        raise ValueError(f"{what} must be [head_dim] or [heads, head_dim]")
    if w.dtype not in _FLOATS or w.device != device:
        raise ValueError(f"{what} must be bf16, fp16 or fp32 on the device of q and k")
    return aligned16(w)


def _check_index(t, what: str, shape, device, lo_hi):
    """An int32 / int64 tensor on ``device``; one on the CPU is range-checked and copied."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _INTS or t.shape != shape:
        raise ValueError(f"{what} must be an int32 or int64 tensor of shape {shape}")
    if not t.is_cuda and t.numel():
        if int(t.min()) < lo_hi[0] or int(t.max()) >= lo_hi[1]:
            raise ValueError(f"{what} values must lie in [{lo_hi[0]}, {lo_hi[1]})")
    return (t if t.device == device else t.to(device)).contiguous()


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
    Differentiable in q, k and the gains; gradients of padding rows are zero.  No forward-mode
    derivative: inputs with a tangent raise ValueError.  A call that is
    captured into a graph and takes leaves that require grad raises ValueError while
    outputs of earlier calls on them are alive (autograd would run part of a captured backward
    on their stream); capture a forward alone under ``torch.no_grad()``.
    """
    # a call laid out like an earlier one takes its parameter block with its own addresses
    idx = idx_ = context_lens if positions is None else positions
    cos_, sin_ = cos, sin
    memo = _MEMO if q_meta is None else q_meta.launch_memo
    key = ("norm_rope", _layout(q), _layout(k), _layout(q_weight), _layout(k_weight), _layout(cos), _layout(sin),
           _layout(idx), positions is None, positions is None or context_lens is None, eps, norm, interleaved, num_heads)
    m = memo.get(key)
    if m is not None and m.fits(q_meta):
        call = m.call_for(q_weight, k_weight, cos, sin, idx, positions is None)
        return _apply(call, q, k, q_weight, k_weight, cos, sin, positions, context_lens)

    qs, ks, dtype, dev = q.shape, k.shape, q.dtype, q.device
    rank = len(qs)
    if rank not in (2, 4) or len(ks) != rank:
        raise ValueError("q and k must both be rank-4 [B, H, N, D] or packed rank-2 [H*T, D]")
    d = qs[-1]
    if ks[-1] != d:
        raise ValueError("q and k must have the same head_dim")
    if d not in _HEAD_DIMS:
        validate_head_dim_supported(d, is_mla=True)
    if dtype not in _FLOATS or k.dtype != dtype:
        raise ValueError("q and k must be of one dtype: bf16, fp16 or fp32")
    if k.device != dev:
        raise ValueError("q and k must be on one device")
    if not q.is_cuda:
        require_cuda_tensors(q)
    cu = tokens = None
    if q_meta is not None:
        cu, tokens = pack_indices(q_meta, dev)

    call = _Call()
    p = call.block = _lib.NormRopeParams()
    packed = call.packed = rank == 2
    if not packed:
        b, hq, n, _ = qs
        hk = ks[1]
        if ks[0] != b or ks[2] != n:
            raise ValueError("q and k must have the same batch and length")
        if q_meta is not None:
            if q_meta.B != b or q_meta.N != n:
                raise ValueError("q_meta shape metadata does not match q/k padded shape")
            tokens = None
        if num_heads is not None and num_heads != hq:
            raise ValueError("q head dimension must match num_heads")
        rows = b * n
        for t, h in ((p.q, hq), (p.k, hk)):
            t.y_sb, t.y_sh, t.y_sn = h * n * d, n * d, d
    else:
        if q_meta is not None:
            b, n, rows = q_meta.B, q_meta.N, q_meta.total_tokens
        else:
            if num_heads is None or num_heads < 1 or qs[0] % num_heads:
                raise ValueError("packed q needs q_meta, or num_heads that divides its rows")
            b, n = 1, qs[0] // num_heads
            rows = n
        hq, hk = (qs[0] // rows, ks[0] // rows) if rows else (0, 0)
        if qs[0] != hq * rows or ks[0] != hk * rows:
            raise ValueError("packed q and k rows must be a multiple of the token count")
        if num_heads is not None and rows and num_heads != hq:
            raise ValueError("q first dim must equal num_heads * tokens")
        p.layout = _lib.LAYOUT_PACKED
        for t in (p.q, p.k):
            t.x_sh = t.y_sh = rows * d
            t.x_sn = t.y_sn = d
    if b * n > 0x7FFFFFFF:
        raise ValueError("q and k must have fewer than 2**31 tokens")
    p.dtype = _lib.dtype_code(dtype)
    p.B, p.N, p.D, p.rows = b, n, d, rows
    p.q.heads, p.k.heads = hq, hk
    if cu is not None:
        p.cu_seqlens = cu.data_ptr()
    if tokens is not None:
        p.token_indices = tokens.data_ptr()

    # before the copies below, which would hide a leaf and hold its accumulator themselves
    leaves = _capture_leaves(q, k, q_weight, k_weight) if torch.is_grad_enabled() else []
    flags = 0
    p.w_dtype = _lib.DTYPE_F32
    wq, wk = q_weight, k_weight
    if norm:
        if not (math.isfinite(eps) and eps >= 0):
            raise ValueError("eps must be finite and >= 0")
        p.eps = eps
        flags = _lib.NR_NORM
        if wq is not None:
            wq = _check_gain(wq, "q_weight", hq, d, dev)
            p.w_dtype = _lib.dtype_code(wq.dtype)
            p.q.weight, p.q.w_sh = wq.data_ptr(), d if wq.ndim == 2 else 0
        if wk is not None:
            wk = _check_gain(wk, "k_weight", hk, d, dev)
            if wq is not None and wq.dtype != wk.dtype:
                raise ValueError("q_weight and k_weight must have the same dtype")
            p.w_dtype = _lib.dtype_code(wk.dtype)
            p.k.weight, p.k.w_sh = wk.data_ptr(), d if wk.ndim == 2 else 0
    elif wq is not None or wk is not None:
        raise ValueError("gains need norm=True")
    elif cos is None:
        raise ValueError("nothing to do: norm=False and no cos/sin tables")

    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        cs = cos.shape
        if len(cs) != 2 or cs != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32 \
                or cos.device != dev or sin.device != dev:
            raise ValueError("cos and sin must be fp32 tables [positions, rotary_dim / 2] on the device of q and k")
        table, r = cs[0], 2 * cs[1]
        if r < 16 or r % 16 or r > d or table < 1:
            raise ValueError("rotary_dim must be a multiple of 16 and at most head_dim, with at least one position")
        cos, sin = aligned16(cos), aligned16(sin)
        p.cos, p.sin, p.table_rows, p.rotary_dim = cos.data_ptr(), sin.data_ptr(), table, r
        if interleaved:
            flags |= _lib.NR_INTERLEAVED
        if positions is not None:
            if context_lens is not None:
                raise ValueError("positions and context_lens are mutually exclusive")
            shape = (b, n) if not packed and q_meta is None else (q_meta.total_tokens if q_meta is not None else rows,)
            idx = positions = _check_index(positions, "positions", shape, dev, (0, table))
            p.positions, p.n_positions = positions.data_ptr(), positions.numel()
            if positions.dtype == torch.int64:
                flags |= _lib.NR_POSITIONS_I64
        elif context_lens is not None:
            idx = context_lens = _check_index(context_lens, "context_lens", (b,), dev, (0, table))
            p.offsets = context_lens.data_ptr()
            if context_lens.dtype == torch.int64:
                flags |= _lib.NR_OFFSETS_I64
    elif positions is not None or context_lens is not None:
        raise ValueError("positions and context_lens need cos and sin")
    p.flags = flags
    q_, k_ = (aligned16(q), aligned16(k)) if packed else (rows16(q), rows16(k))
    call.keep = (cu, tokens)
    # elements, types and device of what the backward reads (_rebind)
    call.sizes = (q.numel(), k.numel(), dtype, *((None if w is None else w.numel()) for w in (wq, wk)),
                  next((w.dtype for w in (wq, wk) if w is not None), None), None if cos is None else cos.numel(),
                  *((None, None) if idx is None else (idx.numel(), idx.dtype)), q.get_device())
    own = q_meta is None or ((cu is None or cu is q_meta.cu_seqlens) and (tokens is None or tokens is q_meta.token_indices))
    if q_ is q and k_ is k and wq is q_weight and wk is k_weight and cos is cos_ and sin is sin_ and idx is idx_ and own:
        if len(memo) >= _MEMO_MAX:
            memo.clear()
        memo[key] = _Memo(call, q_meta)
    return _apply(call, q_, k_, wq, wk, cos, sin, positions, context_lens, leaves)


def _apply(call: _Call, q, k, wq, wk, cos, sin, positions, context_lens, leaves=None):
    refuse_tangents("qk_norm_rope", q, k, wq, wk, cos, sin)
    if torch.is_grad_enabled():
        if cos is not None and (cos.requires_grad or sin.requires_grad):
            raise ValueError("cos and sin are constants: qk_norm_rope has no gradient of them")
        if q.requires_grad or k.requires_grad or (wq is not None and wq.requires_grad) \
                or (wk is not None and wk.requires_grad):
            if leaves is None:
                leaves = _capture_leaves(q, k, wq, wk)
            out = _NormRope.apply(call, q, k, wq, wk, cos, sin, positions, context_lens)
            keep_leaves(leaves)
            return out
    return _forward(call, q, k)
