"""Trees of drafted tokens: their ancestor masks, and attention over a cached context in which
a token sees only its own branch.  An extension: the reference's new tokens all see each
other."""

from __future__ import annotations

from dataclasses import dataclass

import torch

from flash_mlm import _lib
from flash_mlm.host.cache import InferenceCache, PackMetadata
from flash_mlm.host.host import (
    _check_cache_dtype,
    _context_index,
    _ctx_rows,
    _entry_of,
    _memo_lookup,
    _memo_run,
    _memo_store,
    _Memo,
    _packed_context,
    _page_stride,
    _prepare,
    _refuse_fp4,
    _tkey,
    _wants_grad,
    AttnLaunch,
    rows16,
    tile_config_value,
)
from flash_mlm.host.host_utils import (
    _device_scope,
    _maybe_get_cache_context,
    _require_device,
    make_contiguous,
    pack_indices,
    refuse_tangents,
    require_cuda_tensors,
    validate_cache_request,
    validate_cu_seqlens_rank1_min2,
    validate_head_dim_supported,
    validate_packed_cache_shapes,
    validate_qkv_same_shape_rank4,
)

MAX_TREE_TOKENS = _lib.MAX_TREE  # drafted tokens of a sequence
_INTS = (torch.int32, torch.int64)


@dataclass
class TreeMetadata:
    """Ancestors and positions of a batch of drafted trees (:func:`build_tree_metadata`).

    mask       [T, words] int64  bit j % 64 of word j // 64: packed token t sees token j of its
                                 sequence (itself and its ancestors)
    positions  [T] int32         context length + number of ancestors
    """

    mask: torch.Tensor
    positions: torch.Tensor


def build_tree_metadata(
    parents: torch.Tensor,
    q_meta: PackMetadata,
    *,
    context_lens: torch.Tensor | None = None,
    check: bool = True,
) -> TreeMetadata:
    """Ancestor masks and positions of drafted trees, on the GPU.

    ``parents`` [T] (int32 or int64, packed like ``q_meta``): for every drafted token the index,
    within its sequence, of the token it follows, -1 for a token that follows the context.  A
    parent comes before its children.  ``context_lens`` [B] are added to the positions.  At most
    256 tokens a sequence.

    With ``check`` one integer is read back, and a parent that is neither -1 nor before its
    child raises ValueError; without, such a token counts as a root.
    """
    dev = q_meta.cu_seqlens.device
    b, n, t = int(q_meta.B), int(q_meta.N), int(q_meta.total_tokens)
    if n > MAX_TREE_TOKENS:
        raise ValueError(f"a drafted tree has at most {MAX_TREE_TOKENS} tokens (q_meta.N)")
    if not isinstance(parents, torch.Tensor) or parents.dtype not in _INTS or tuple(parents.shape) != (t,):
        raise ValueError("parents must be an int32 or int64 tensor with one entry per packed token")
    if context_lens is not None and (
            not isinstance(context_lens, torch.Tensor) or context_lens.dtype not in _INTS
            or tuple(context_lens.shape) != (b,)):
        raise ValueError("context_lens must be an int32 or int64 tensor with one entry per sequence")
    _require_device(parents, context_lens, what="build_tree_metadata")
    if parents.device != dev or (context_lens is not None and context_lens.device != dev):
        raise ValueError("parents and context_lens must be on the device of q_meta")
    parents = parents.contiguous()
    context_lens = None if context_lens is None else context_lens.contiguous()
    cu = pack_indices(q_meta, dev)[0]
    words = max(1, -(-n // 64))
    mask = torch.empty((t, words), dtype=torch.int64, device=dev)
    positions = torch.empty(t, dtype=torch.int32, device=dev)
    bad = torch.zeros(1, dtype=torch.int32, device=dev) if check else None
    with _device_scope(dev):
        rc = _lib.load().fmlm_tree_mask(
            parents.data_ptr(), int(parents.dtype == torch.int64), cu.data_ptr(), b, n, t, words,
            _lib.ptr(context_lens), int(context_lens is not None and context_lens.dtype == torch.int64),
            mask.data_ptr(), positions.data_ptr(), _lib.ptr(bad), _lib.stream_of(dev),
        )
    _lib.check(rc, "fmlm_tree_mask")
    if check and int(bad):
        raise ValueError("parents must be -1 or come before their children")
    return TreeMetadata(mask=mask, positions=positions)


class TreeLaunch(AttnLaunch):
    """A prepared fmlm_attn_tree_fwd call."""

    __slots__ = ("mask",)

    def __call__(self) -> None:
        records = self.own_buffers(row_stats=False)
        nbytes = self.lib.fmlm_attn_tree_workspace_bytes(self.params)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes > 0 else None
        with _device_scope(self.device):
            rc = self.lib.fmlm_attn_tree_fwd(self.params, self.mask.data_ptr(), int(self.mask.shape[1]), _lib.ptr(ws),
                                             nbytes, self.stream)
        del records  # held until here
        _lib.check(rc, "fmlm_attn_tree_fwd")

    @classmethod
    def of(cls, plan: AttnLaunch, mask: torch.Tensor) -> TreeLaunch:
        tree = cls(plan.lib, plan.params, plan.stream, plan.device, plan.keep)
        tree.records, tree.mask = plan.records, mask
        return tree


def flash_attn_mlm_tree(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    num_heads: int,
    q_meta: PackMetadata,
    tree: TreeMetadata,
    scale: float,
    inference_cache: InferenceCache | None = None,
    layer_id: int | str | None = None,
    is_mla: bool = False,
    context_batch_size: int | None = None,
    context_index: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of drafted trees: like :func:`flash_attn_mlm_compressed` over padded q/k/v
    [B, H, N, D], but token i of a sequence attends to [its cached context || itself and its
    ancestors in ``tree``] instead of all tokens of its sequence.

    Returns the packed output [H * T, D] (head-major).  A chain (``parents = i - 1``) is ordinary
    causal decoding of several tokens; ``tree.mask`` may also be set bit by bit, to what no tree
    is, and a row that sees no key at all is zero.  Context, ``is_mla`` and ``context_index`` are as in
    :func:`flash_attn_mlm_compressed`; at most 256 tokens a sequence.  The context is not
    changed: store the accepted tokens with :meth:`InferenceCache.append_paged_kv_cache`.
    No gradients: inputs that require grad raise ValueError (use ``torch.no_grad()``), those with
    a forward-mode tangent too.
    """
    memo, entry, mask = q_meta.launch_memo, _entry_of(inference_cache, layer_id), tree.mask
    _refuse_fp4(inference_cache, layer_id)
    context = (entry.k_cache, entry.v_cache) if entry is not None else ()
    refuse_tangents("flash_attn_mlm_tree", q, k, v, *context)
    if _wants_grad(q, k, v, *context):
        raise ValueError("flash_attn_mlm_tree has no backward; call it under torch.no_grad()")
    key = None
    if context_index is None and all(isinstance(t, torch.Tensor) for t in (q, k, v, mask)):
        # all that the checks below depend on
        key = ("tree", _tkey(q), _tkey(k), _tkey(v), _tkey(mask), num_heads, q_meta.B, q_meta.N, q_meta.total_tokens,
               float(scale), is_mla, context_batch_size, tile_config_value(), None if entry is None else id(entry),
               inference_cache is None, layer_id is None)
        m = _memo_lookup(memo, key, entry, q_meta.cu_seqlens)
        if m is not None:
            return _memo_run(m, q, k, v, entry, wrap=lambda plan: TreeLaunch.of(plan, mask))[0]
    b, h, n, d = validate_qkv_same_shape_rank4(q, k, v, error_prefix="q/k/v")
    if h != num_heads:
        raise ValueError("q/k/v head dimension must match num_heads")
    if q_meta.B != b or q_meta.N != n:
        raise ValueError("q_meta shape metadata does not match q/k/v padded shape")
    if n > MAX_TREE_TOKENS:
        raise ValueError(f"a drafted tree has at most {MAX_TREE_TOKENS} tokens (q_meta.N)")
    T = int(q_meta.total_tokens)
    if mask.ndim != 2 or mask.dtype != torch.int64 or int(mask.shape[0]) != T or int(mask.shape[1]) * 64 < n:
        raise ValueError("tree.mask must be [tokens, words] int64, built for this q_meta")
    validate_cache_request(prefill=False, inference_cache=inference_cache, layer_id=layer_id)
    ctx = _maybe_get_cache_context(
        inference_cache=inference_cache,
        layer_id=layer_id,
        batch_size=b,
        is_mla=is_mla,
        num_heads=num_heads,
        head_dim=d,
        context_batch_size=context_batch_size,
        dtype=q.dtype,
        device=q.device,
        compressed=True,
    )
    require_cuda_tensors(q, k, v, mask, q_meta.cu_seqlens, ctx.k_cache, ctx.v_cache, ctx.cu_seqlens_kv)
    if mask.device != q.device or q_meta.cu_seqlens.device != q.device:
        raise ValueError("tree and q_meta must be on the device of q/k/v")
    if num_heads < 1:
        raise ValueError("num_heads must be >= 1")
    validate_packed_cache_shapes(
        ctx.k_cache, ctx.v_cache, num_heads=num_heads, total_context_len=int(ctx.total_context_len), head_dim=d,
        is_mla=is_mla,
    )
    validate_head_dim_supported(d, is_mla=is_mla)
    validate_cu_seqlens_rank1_min2(q_meta.cu_seqlens, ctx.cu_seqlens_kv)
    cbs, c_strides = _packed_context(
        ctx, num_heads=num_heads, d=d, is_mla=is_mla, b=b, prefill=False, indexed=context_index is not None
    )
    ctx_index = _context_index(
        context_index, b=b, cbs=cbs, prefill=False, context_batch_size=context_batch_size, device=q.device
    )
    _check_cache_dtype(ctx.k_cache, q)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must have the same dtype")

    out = torch.empty((num_heads * T, d), dtype=q.dtype, device=q.device)
    if T == 0:
        return out
    q_, k_, v_ = rows16(q), rows16(k), rows16(v)
    k_cache, v_cache = make_contiguous(ctx.k_cache, ctx.v_cache)
    cu_q = pack_indices(q_meta, q.device)[0]
    cu_kv = ctx.cu_seqlens_kv.to(torch.int32).contiguous()
    k_strides = (k_.stride(0), 0 if is_mla else k_.stride(1), k_.stride(2))
    v_strides = k_strides if is_mla else (v_.stride(0), v_.stride(1), v_.stride(2))
    # a schedule or parameter block made during a capture lives in the graph's memory and is filled
    # by its replays: it stays this call's own
    capturing = torch.cuda.is_current_stream_capturing()
    plan = _prepare(
        q=q_,
        out=out,
        k=k_,
        v=None if is_mla else v_,
        B=b,
        H=num_heads,
        D=d,
        N=n,
        total_q=T,
        cu_seqlens_q=cu_q,
        q_strides=(q_.stride(0), q_.stride(1), q_.stride(2)),
        q_layout=_lib.LAYOUT_PADDED,
        o_strides=(0, T * d, d),
        o_layout=_lib.LAYOUT_PACKED,
        k_strides=k_strides,
        v_strides=v_strides,
        kv_layout=_lib.LAYOUT_PADDED,
        k_ctx=k_cache,
        v_ctx=None if is_mla else v_cache,
        c_strides=c_strides,
        cu_seqlens_kv=cu_kv,
        ctx_len=0,
        ctx_batch=cbs,
        ctx_rows=_ctx_rows(ctx),
        scale=scale,
        flags=_lib.FLAG_TREE | (_lib.FLAG_MLA if is_mla else 0),
        inference_cache=inference_cache,
        schedule_cache=dict(q_meta.kernel_schedules) if capturing else q_meta.kernel_schedules,
        schedule_of=q_meta.cu_seqlens,
        ctx_index=ctx_index,
        block_table=ctx.block_table,
        page_stride=_page_stride(ctx, num_heads, d, is_mla),
    )
    TreeLaunch.of(plan, mask.contiguous())()
    if (key is not None and not capturing and q_ is q and k_ is k and v_ is v and k_cache is ctx.k_cache and v_cache is ctx.v_cache
            and plan.keep[10] is None and mask.is_contiguous()):
        extra = (cu_q, cu_kv, k_cache if entry is None else None, v_cache if entry is None else None)
        _memo_store(memo, key, _Memo(plan, entry, extra, tuple(out.shape), cu=q_meta.cu_seqlens))
    return out
