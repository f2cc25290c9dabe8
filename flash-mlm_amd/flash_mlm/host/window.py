"""Window attention with sinks: attention of a sequence's tokens to a window of recent keys and a
few first ones, over cached contexts in 16 or 4 bits and for training.  An extension: the
reference's queries see all keys."""

from __future__ import annotations

import math
import weakref

import torch

from flash_mlm import _lib
from flash_mlm.host.cache import PAGE_ROWS, InferenceCache, PackMetadata
from flash_mlm.host.host import _context_index, _entry_of, _tkey, _wants_grad, rows16
from flash_mlm.host.host_utils import (
    _device_scope,
    aligned16,
    capture_leaves,
    keep_leaves,
    pack_indices,
    refuse_tangents,
    require_cuda_tensors,
    validate_cache_request,
)

_HEAD_DIMS = (32, 64, 128, 256)
_MAX = (1 << 30) - 2
_MEMO_MAX = 16


def _limit(x, what: str) -> int:
    if x is None:
        return -1
    if isinstance(x, bool) or not isinstance(x, int) or x < 0:
        raise ValueError(f"{what} must be an integer >= 0 (window sides: or None, no limit)")
    return min(x, _MAX)


class _Call:
    """The checked arguments of a call as parameter blocks without the addresses of its own rows."""

    __slots__ = ("params", "window", "nbytes", "out_shape", "entry_ref", "keep", "cu", "shape", "strides", "grads")

    def run(self, q, k, v, lse=None, low=None):
        """One launch on rows laid out as the call's; returns the output.  ``lse`` and ``low`` take what
        the backward reads: the rows' statistics, and what the output's rounding took away."""
        p = _lib.AttnParams.from_buffer_copy(self.params)
        dev = q.device
        out = torch.empty(self.out_shape, dtype=q.dtype, device=dev)
        p.q, p.o = q.data_ptr(), out.data_ptr()
        if k is not None:
            p.k, p.v = k.data_ptr(), v.data_ptr()
        lib = _lib.load()
        ws, nbytes, w = None, self.nbytes, self.window
        if lse is not None:
            p.lse = lse.data_ptr()
            w = _lib.Window.from_buffer_copy(w)
            w.o_low = low.data_ptr()
        elif nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
        with _device_scope(dev):
            rc = lib.fmlm_window_fwd(p, w, _lib.stream_of(dev))
        del ws  # held until here
        _lib.check(rc, "fmlm_window_fwd")
        return out


_MAX_PITCH = 1 << 22  # elements from row to row: a tile's byte offsets are 32 bits in the kernels


def _rows(t: torch.Tensor) -> torch.Tensor:
    if t.ndim != 4:
        return aligned16(t)
    if t.stride(2) >= _MAX_PITCH and t.shape[2] > 1:
        return t.clone(memory_format=torch.contiguous_format)
    return rows16(t)


def _strides(t: torch.Tensor, tokens: int):
    """Element strides (batch, head, position) of padded rows [B, H, N, D] or packed ones [H * T, D]."""
    if t.ndim == 4:
        sb, sh, sn, _ = t.stride()
        return sb, sh, sn if t.shape[2] > 1 else t.shape[3]  # (of a single row: any)
    return 0, tokens * int(t.shape[1]), int(t.shape[1])


def _context(entry, p, w, *, b: int, context_index, appended: bool, device):
    """The fields of the cached context ``entry``; returns the tensors they point to."""
    cu_kv = entry.cu_seqlens_kv
    if cu_kv is None:
        raise ValueError("window attention needs a packed or paged context (with cu_seqlens_kv)")
    if cu_kv.device != device:  # (stored as given: a host address would reach the kernel)
        raise ValueError("cu_seqlens_kv of the cached context must be on the device of q")
    cbs, total, d = entry.context_batch_size, int(entry.total_context_len), entry.head_dim
    index = _context_index(context_index, b=b, cbs=cbs, prefill=False, context_batch_size=None, device=device)
    if index is None and 1 < cbs < b:
        raise ValueError("context_batch_size must be 1 or at least the batch size")
    if index is None and appended and cbs < b:
        raise ValueError("tokens in the context need a context batch for each sequence")
    cu_kv = cu_kv.to(torch.int32).contiguous()
    p.cu_seqlens_kv, p.ctx_batch, p.ctx_index = cu_kv.data_ptr(), cbs, _lib.ptr(index)
    p.ctx_rows, p.c_sh, p.c_sn = total, total * d, d
    k, v = entry.k_cache, entry.v_cache
    table = entry.block_table
    if table is not None and (total == 0 or table.shape[1] == 0):
        p.ctx_rows = 0  # no page to read, and no address of a table without columns
    elif table is not None:
        p.ctx_block_table, p.ctx_pages_per_batch = table.data_ptr(), int(table.shape[1])
        p.ctx_page_stride, p.ctx_rows = PAGE_ROWS * d, total // PAGE_ROWS
    elif k.numel():
        k, v = aligned16(k), aligned16(v)
    if k.numel():
        p.k_ctx, p.v_ctx = k.data_ptr(), v.data_ptr()
    if entry.k_scales is not None:
        w.flags |= _lib.WINDOW_FP4
        w.k_scales, w.v_scales = entry.k_scales.data_ptr(), entry.v_scales.data_ptr()
    return k, v, cu_kv, index


def _build(q, k, v, num_heads: int, q_meta: PackMetadata, scale, left, right, sinks, entry, context_index) -> _Call:
    """The checks of a call, and its parameter blocks."""
    if q.ndim not in (2, 4):
        raise ValueError("q must be padded [B, H, N, D] or packed [H * T, D]")
    if (k is None) != (v is None):
        raise ValueError("k and v come together")
    if k is not None and (k.shape != q.shape or v.shape != q.shape):
        raise ValueError("q, k, v must have the same shape")
    t, d, dev = int(q_meta.total_tokens), int(q.shape[-1]), q.device
    if num_heads < 1:
        raise ValueError("num_heads must be >= 1")
    if q.ndim == 4:
        if q.shape[1] != num_heads:
            raise ValueError("q/k/v head dimension must match num_heads")
        if q.shape[0] != q_meta.B or q.shape[2] != q_meta.N:
            raise ValueError("q_meta shape metadata does not match q/k/v padded shape")
    elif q.shape[0] != num_heads * t:
        raise ValueError("q first dim must equal num_heads * q_meta.total_tokens")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("window attention needs bf16 or fp16 inputs")
    if d not in _HEAD_DIMS:
        raise ValueError("window attention needs head_dim 32, 64, 128 or 256")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if k is not None and (k.dtype != q.dtype or v.dtype != q.dtype):
        raise ValueError("q, k and v must have the same dtype")
    if k is not None and (k.device != dev or v.device != dev):
        raise ValueError("q, k and v must be on one device")
    if t >= _MAX or int(q_meta.B) * int(q_meta.N) > 0x7FFFFFFF:
        raise ValueError("the call must have fewer than 2**30 tokens")
    require_cuda_tensors(q, k, v)
    cu = pack_indices(q_meta, dev)[0]

    call = _Call()
    p, w = call.params, call.window = _lib.AttnParams(), _lib.Window()
    p.dtype = _lib.dtype_code(q.dtype)
    p.B, p.H, p.D, p.N, p.total_q = int(q_meta.B), num_heads, d, int(q_meta.N), t
    p.scale, p.cu_seqlens_q = float(scale), cu.data_ptr()
    w.left, w.right, w.sinks = left, right, sinks
    context = None
    if k is None:
        w.flags = _lib.WINDOW_APPENDED
        if entry is None:
            raise ValueError("without k and v the tokens must be in the layer's cached context")
    if entry is not None:
        if (entry.is_mla, entry.num_heads, entry.head_dim) != (False, num_heads, d):
            raise ValueError("the layer's cached context has another mode (MLA), num_heads or head_dim")
        if entry.dtype != q.dtype or entry.device != dev:
            raise ValueError("cached context dtype/device must match q")
        context = _context(entry, p, w, b=p.B, context_index=context_index, appended=k is None, device=dev)
    elif context_index is not None:
        raise ValueError("context_index needs a cached context")
    # layouts, from rows as the kernel reads them
    q_, k_, v_ = _rows(q), None if k is None else _rows(k), None if v is None else _rows(v)
    layout = _lib.LAYOUT_PADDED if q.ndim == 4 else _lib.LAYOUT_PACKED
    p.q_layout, p.kv_layout, p.o_layout = layout, layout, _lib.LAYOUT_PACKED
    p.q_sb, p.q_sh, p.q_sn = _strides(q_, t)
    p.o_sh, p.o_sn = t * d, d
    if k is not None:
        p.k_sb, p.k_sh, p.k_sn = _strides(k_, t)
        p.v_sb, p.v_sh, p.v_sn = _strides(v_, t)
    call.out_shape = (num_heads * t, d)
    if k is not None:  # of the backward: rows laid out like these, and contiguous gradients
        call.shape, call.strides = q.shape, (q_.stride(), k_.stride(), v_.stride())
        g = call.grads = _lib.AttnGrads()
        g.do_sh, g.do_sn, g.workspace_bytes = p.o_sh, p.o_sn, 4 * num_heads * t
        n = p.N * d
        s3 = (num_heads * n, n, d) if q.ndim == 4 else (0, t * d, d)
        g.dq_sb, g.dq_sh, g.dq_sn = s3
        g.dk_sb, g.dk_sh, g.dk_sn = s3
        g.dv_sb, g.dv_sh, g.dv_sn = s3
    call.entry_ref = None if entry is None else weakref.ref(entry)
    call.cu = cu
    call.keep = (cu, context)
    # sizes of the split's records: the addresses that the checks ask for come with each run
    p.q = p.o = 256
    if k is not None:
        p.k = p.v = 256
    nbytes = _lib.load().fmlm_window_workspace_bytes(p, w) if t else 0
    _lib.check(nbytes if nbytes < 0 else 0, "fmlm_window_workspace_bytes")
    call.nbytes = nbytes
    return call, (q_, k_, v_)


class _Window(torch.autograd.Function):
    @staticmethod
    def forward(ctx, call, q, k, v):
        p = call.params
        lse = torch.empty(call.out_shape[:1], dtype=torch.float32, device=q.device)
        low = torch.empty(call.out_shape, dtype=q.dtype, device=q.device)
        out = call.run(_rows(q), _rows(k), _rows(v), lse, low)
        ctx.call, ctx.cu_version = call, _version(call)
        # read from there in the backward: autograd may free these and bring others
        ctx.save_for_backward(q, k, v, out, lse, low)
        return out

    @staticmethod
    def backward(ctx, dout):
        # grad mode: create_graph, where the gradients must refuse to be differentiated (the wrapper's
        # grad-mode switches cost 4 us)
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, dout)


def _version(call):
    """How often the call's offsets have been changed in place (a copy of the metadata's never is)."""
    cu = call.cu
    return None if cu.is_inference() else cu._version


def _check_saved(call, saved, dtype, device) -> None:
    """A saved-tensor hook may bring any tensors: the kernels read these addresses with the call's sizes."""
    rows, out = call.shape, call.out_shape
    for t, shape, kind in zip(saved, (rows, rows, rows, out, out[:1], out), (dtype, dtype, dtype, dtype, torch.float32, dtype)):
        if t.shape != shape or t.dtype is not kind or t.device != device:
            raise RuntimeError(
                "flash_attn_mlm_window: a saved tensor came back with another shape or type, or on another device")


def _backward(ctx, dout):
    call = ctx.call
    q, k, v, out, lse, low = saved = ctx.saved_tensors
    _check_saved(call, saved, dout.dtype, dout.device)
    if _version(call) != ctx.cu_version:
        raise RuntimeError("flash_attn_mlm_window: q_meta.cu_seqlens has been modified by an inplace operation since the forward")
    if dout.shape != out.shape:
        raise ValueError("gradient of the attention output has the wrong shape")
    if call.params.total_q == 0:  # no token: padding rows alone
        return None, torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    p = _lib.AttnParams.from_buffer_copy(call.params)
    p.q, p.k, p.v = ptrs = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if (q.stride(), k.stride(), v.stride()) != call.strides or (ptrs[0] | ptrs[1] | ptrs[2]) & 15:
        q, k, v = _rows(q), _rows(k), _rows(v)  # (brought back by a hook, or copied by the forward too)
        t = p.total_q
        p.q, p.k, p.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
        p.q_sb, p.q_sh, p.q_sn = _strides(q, t)
        p.k_sb, p.k_sh, p.k_sn = _strides(k, t)
        p.v_sb, p.v_sh, p.v_sn = _strides(v, t)
    out, lse, low, dout = aligned16(out), aligned16(lse), aligned16(low), aligned16(dout)
    shape, dtype, dev = q.shape, q.dtype, q.device
    dq = torch.empty(shape, dtype=dtype, device=dev)
    dk = torch.empty(shape, dtype=dtype, device=dev)
    dv = torch.empty(shape, dtype=dtype, device=dev)
    ws = torch.empty_like(lse)
    p.o, p.lse = out.data_ptr(), lse.data_ptr()
    g = _lib.AttnGrads.from_buffer_copy(call.grads)
    g.dout, g.dq, g.dk, g.dv, g.workspace = dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr()
    w = _lib.Window.from_buffer_copy(call.window)
    w.o_low = low.data_ptr()
    with _device_scope(dev):
        rc = _lib.load().fmlm_window_bwd(p, w, g, _lib.stream_of(dev))
    if rc:
        _lib.check(rc, "fmlm_window_bwd")
    return None, dq, dk, dv


_backward_once = torch.autograd.function.once_differentiable(_backward)


def flash_attn_mlm_window(
    q: torch.Tensor,
    k: torch.Tensor | None,
    v: torch.Tensor | None,
    num_heads: int,
    q_meta: PackMetadata,
    scale: float,
    *,
    window: tuple[int | None, int | None] = (None, None),
    sinks: int = 0,
    inference_cache: InferenceCache | None = None,
    layer_id: int | str | None = None,
    context_index: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention within a window of positions, with a few first tokens that stay visible.

    q, k, v: padded [B, H, N, D] or packed [H * T, D], the tokens that ``q_meta`` describes.  Returns
    the packed output [H * T, D] (head-major).  Keys are numbered from the first row of the sequence's
    cached context, the new tokens after them, and token i of a sequence with n context rows is at
    position s = n + i.  With ``window`` = (left, right) it sees the keys j with

      j <= s + right  and  (j >= s - left  or  j < sinks)

    None is no limit: (255, 0) is causal over 256 tokens, (64, 64) local both ways, (None, None)
    what :func:`flash_attn_mlm_compressed` computes.  A row that sees no key is zero.

    ``k`` and ``v`` None: the new tokens have been appended already
    (:meth:`InferenceCache.append_paged_kv_cache`) and are the last L_b rows of their sequence's
    context; s = n - L_b + i.

    The context is the layer's packed, paged or 4-bit entry (none: no context), with
    ``context_index`` as in :func:`flash_attn_mlm_compressed`.  bf16 and fp16, D = 32, 64, 128 or 256,
    a finite scale, no MLA.  Differentiable in q, k and v without a cached context, for finite inputs (in
    fp16 gradients are finite while |P (dO V^T - rowsum(dO O))| stays below 65504); gradients are
    the same bits every time, those of padding rows zero.  With a context, inputs or cached rows that
    require grad raise ValueError (use ``torch.no_grad()``); with a forward-mode tangent always.  A
    call that is captured into a graph and takes leaves that require grad raises ValueError while
    outputs of earlier calls on them are alive.
    """
    entry = _entry_of(inference_cache, layer_id)
    context = () if entry is None else (entry.k_cache, entry.v_cache)
    refuse_tangents("flash_attn_mlm_window", q, k, v, *context)
    if _wants_grad(*context):
        raise ValueError("flash_attn_mlm_window has no gradient of a cached context; call it under torch.no_grad()")
    grad = torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)
                                        or (v is not None and v.requires_grad))
    # (before the kept calls are asked: 1.0 and True equal 1 there)
    if not isinstance(window, (tuple, list)) or len(window) != 2:
        raise ValueError("window must be a pair (left, right)")
    left, right = _limit(window[0], "window"), _limit(window[1], "window")
    if sinks is None:
        raise ValueError("sinks must be an integer >= 0")
    sinks = _limit(sinks, "sinks")
    call = key = None
    if context_index is None and type(num_heads) is int:
        # all that the checks depend on
        key = ("window", _tkey(q), None if k is None else _tkey(k), None if v is None else _tkey(v), num_heads,
               q_meta.B, q_meta.N, q_meta.total_tokens, float(scale), left, right, sinks,
               None if entry is None else id(entry), inference_cache is None, layer_id is None)
        call = q_meta.launch_memo.get(key)
        if call is not None and (call.cu is not q_meta.cu_seqlens or
                                 (None if call.entry_ref is None else call.entry_ref()) is not entry):
            call = None
    rows = (q, k, v)
    if call is None:
        validate_cache_request(prefill=False, inference_cache=inference_cache, layer_id=layer_id)
        call, rows = _build(q, k, v, num_heads, q_meta, scale, left, right, sinks, entry, context_index)
        cu, kept = call.keep
        if (key is not None and rows[0] is q and rows[1] is k and rows[2] is v and cu is q_meta.cu_seqlens
                and (kept is None or (kept[0] is entry.k_cache and kept[1] is entry.v_cache
                                      and kept[2] is entry.cu_seqlens_kv))):
            if len(q_meta.launch_memo) >= _MEMO_MAX:
                q_meta.launch_memo.clear()
            # the entry's tensors are held by the entry alone, as in the other memos
            stored = _Call()
            for name in _Call.__slots__:
                setattr(stored, name, getattr(call, name, None))
            stored.keep = None
            q_meta.launch_memo[key] = stored
    if grad:
        if entry is not None:
            raise ValueError("flash_attn_mlm_window has no backward over a cached context; call it under torch.no_grad()")
        leaves = capture_leaves("flash_attn_mlm_window", q, k, v)
        out = _Window.apply(call, q, k, v)
        keep_leaves(leaves)
        return out
    return call.run(*rows)
