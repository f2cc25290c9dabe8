"""Filling paged KV contexts: block tables and slots of a step's new tokens, and the copy of
their rows into the pages.  Extensions: the reference's roadmap lists paged KV
(README.md:41)."""

from __future__ import annotations

from dataclasses import dataclass

import torch

from flash_mlm import _lib
from flash_mlm.host.cache import PAGE_ROWS, PackMetadata
from flash_mlm.host.host_utils import _device_scope, _require_device, pack_indices

_INTS = (torch.int32, torch.int64)


@dataclass
class PagedMetadata:
    """Where a step's new tokens go in a paged context (:func:`build_block_table`).

    block_table    [B, max_pages] int32  pages of each request, its new ones included; -1 past them
    slot_mapping   [T] int64   row of the pool (page * 64 + row) of each packed new token, -1: not stored
    positions      [T] int32   old context length + place in the sequence
    context_lens   [B] int32   context lengths once the tokens are stored
    cu_seqlens_kv  [B+1] int32 their prefix sums
    summary        [4] int32   pages taken from the free list, pages it lacked, requests that were
                               out of range, tokens stored
    pages_taken    the first of these on the host (None when the call did not read them back)
    """

    block_table: torch.Tensor
    slot_mapping: torch.Tensor
    positions: torch.Tensor | None
    context_lens: torch.Tensor
    cu_seqlens_kv: torch.Tensor
    summary: torch.Tensor | None = None
    pages_taken: int | None = None


def _ints(t: torch.Tensor, what: str, ndim: int, device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.ndim != ndim or t.dtype not in _INTS:
        raise ValueError(f"{what} must be a rank-{ndim} int32 or int64 tensor")
    if t.device != device:
        _require_device(t, what="build_block_table")
        raise ValueError(f"{what} must be on the device of q_meta")
    return t.contiguous()


def build_block_table(
    q_meta: PackMetadata,
    context_lens: torch.Tensor,
    *,
    free_pages: torch.Tensor,
    block_table: torch.Tensor | None = None,
    max_pages: int | None = None,
    keep: torch.Tensor | None = None,
    check: bool = True,
) -> PagedMetadata:
    """Give the new tokens of every request their pages and slots, on the GPU.

    ``q_meta`` describes the new tokens (L_b of request b), ``context_lens`` [B] the tokens
    that request b already has in the pages ``block_table[b]`` ([B, pages], None: no request has
    any).  A request that needs more pages takes them from ``free_pages`` [F], in request
    order from the front; the next step's list starts ``pages_taken`` entries later.  ``keep``
    ([T] bool, e.g. the accepted tokens of a verified draft) stores only some of the new
    tokens, in their order.  ``max_pages`` is the width of the new table (default: that of
    ``block_table``; without one, enough for ``q_meta.N`` tokens).  ``block_table`` itself is
    left as it is.

    With ``check`` the call reads four integers back (one synchronisation, as
    :func:`build_pack_metadata`) and raises ValueError when the free list is too short, an old
    length is negative or exceeds its table row, or a request outgrows ``max_pages``.  Without,
    nothing is read back: such a request keeps the tokens that fit, the others' slots are -1, and
    ``summary`` tells.
    """
    dev = q_meta.cu_seqlens.device
    b, t = int(q_meta.B), int(q_meta.total_tokens)
    _require_device(q_meta.cu_seqlens, what="build_block_table")
    context_lens = _ints(context_lens, "context_lens", 1, dev)
    free_pages = _ints(free_pages, "free_pages", 1, dev)
    if int(context_lens.numel()) != b:
        raise ValueError("context_lens must have one entry per sequence")
    if block_table is not None:
        block_table = _ints(block_table, "block_table", 2, dev)
        if int(block_table.shape[0]) != b:
            raise ValueError("block_table must have one row per sequence")
    if max_pages is None:
        max_pages = int(block_table.shape[1]) if block_table is not None else -(-int(q_meta.N) // PAGE_ROWS)
    if max_pages < 0 or max_pages > 0x7FFFFFFF // PAGE_ROWS:
        raise ValueError(f"max_pages must lie in [0, {0x7FFFFFFF // PAGE_ROWS}]")
    if keep is not None:
        if not isinstance(keep, torch.Tensor) or keep.dtype != torch.bool or tuple(keep.shape) != (t,):
            raise ValueError("keep must be a bool tensor with one entry per packed token")
        _require_device(keep, what="build_block_table")
        if keep.device != dev:
            raise ValueError("keep must be on the device of q_meta")
        keep = keep.contiguous()
    if b * int(q_meta.N) > 0x7FFFFFFF or int(free_pages.numel()) > 0x7FFFFFFF:
        raise ValueError("the call must have fewer than 2**31 tokens and free pages")

    lib = _lib.load()
    p = _lib.BlockTableParams()
    p.flags = (
        (_lib.BT_OLD_I64 if context_lens.dtype == torch.int64 else 0)
        | (_lib.BT_TABLE_I64 if block_table is not None and block_table.dtype == torch.int64 else 0)
        | (_lib.BT_FREE_I64 if free_pages.dtype == torch.int64 else 0)
    )
    p.B, p.N, p.T = b, int(q_meta.N), t
    p.max_pages, p.in_pages = max_pages, 0 if block_table is None else int(block_table.shape[1])
    p.n_free = int(free_pages.numel())
    p.keep = _lib.ptr(keep)
    nbytes = lib.fmlm_block_table_workspace_bytes(p)
    _lib.check(nbytes if nbytes < 0 else 0, "fmlm_block_table_workspace_bytes")
    slots = torch.empty(t, dtype=torch.int64, device=dev)
    # the 32-bit results share one allocation with the workspace
    ws, table, positions, new_lens, cu, summary = torch.empty(
        b * max_pages + t + 2 * b + 5 + nbytes // 4, dtype=torch.int32, device=dev
    ).split_with_sizes((nbytes // 4, b * max_pages, t, b, b + 1, 4))
    table = table.view(b, max_pages)
    cu_q, tokens = pack_indices(q_meta, dev)
    p.old_lens, p.cu_seqlens, p.token_indices = context_lens.data_ptr(), cu_q.data_ptr(), tokens.data_ptr()
    p.table_in, p.free_pages = _lib.ptr(block_table), free_pages.data_ptr()
    p.block_table, p.slot_mapping, p.positions = table.data_ptr(), slots.data_ptr(), positions.data_ptr()
    p.new_lens, p.cu_kv, p.summary = new_lens.data_ptr(), cu.data_ptr(), summary.data_ptr()
    p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    with _device_scope(dev):
        rc = lib.fmlm_block_table(p, _lib.stream_of(dev))
    _lib.check(rc, "fmlm_block_table")
    plan = PagedMetadata(table, slots, positions, new_lens, cu, summary)
    if check:
        taken, lacking, bad, _ = summary.tolist()
        if bad:
            raise ValueError("context_lens must fit block_table, and every request max_pages pages")
        if lacking:
            raise ValueError(f"free_pages is too short: {lacking} more pages are needed")
        plan.pages_taken = taken
    return plan


_ONE, _PAIR = _lib.PagedTensor * 1, _lib.PagedTensor * 2


def paged_append(pairs, *, heads: int, d: int, q_meta: PackMetadata, slots: torch.Tensor, pool_rows: int) -> None:
    """Rows of each (source, pool) pair to their slots in one HIP launch (fmlm_paged_append);
    the kernel of :meth:`InferenceCache.append_paged_kv_cache`."""
    arr = _PAIR() if len(pairs) == 2 else _ONE()
    packed = pairs[0][0].ndim == 2
    t = int(q_meta.total_tokens)
    keep = []
    for a, (src, pool) in zip(arr, pairs):
        if packed or src.stride(-1) != 1:
            src = src.contiguous()
        keep.append(src)
        a.src, a.pool = src.data_ptr(), pool.data_ptr()
        if packed:
            a.s_sh, a.s_sn = t * d, d
        else:
            a.s_sb, a.s_sh, a.s_sn, _ = src.stride()
            a.batch = src.shape[0]
    dev = slots.device
    tokens = pack_indices(q_meta, dev)[1]
    with _device_scope(dev):
        rc = _lib.load().fmlm_paged_append(
            arr, len(pairs), pairs[0][0].element_size(), heads, d, t, int(q_meta.N),
            _lib.LAYOUT_PACKED if packed else _lib.LAYOUT_PADDED, tokens.data_ptr(), slots.data_ptr(),
            pool_rows, _lib.stream_of(dev),
        )
    _lib.check(rc, "fmlm_paged_append")
