"""build_block_table and InferenceCache.append_paged_kv_cache: refusals (CPU), and on the GPU
block tables and slots against a request-by-request restatement (oracle/paged_step_ref.py),
appended rows bit for bit, and the attention that reads them."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from flash_mlm import (
    InferenceCache,
    PackMetadata,
    PagedMetadata,
    _lib,
    build_block_table,
    build_pack_metadata,
    flash_attn_mlm_compressed,
)
from oracle import paged_step_ref as ref

PAGE = 64


def _cpu_meta(lens, N):
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    tok = torch.tensor([b * N + p for b, n in enumerate(lens) for p in range(n)], dtype=torch.int64)
    return PackMetadata(B=len(lens), N=N, lengths=torch.tensor(lens, dtype=torch.int32), cu_seqlens=cu, token_indices=tok,
                        total_tokens=sum(lens), batch_ids_block_n=32, batch_ids_q=cu, q_tile_starts_q=cu)


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------
def test_table_refusals_on_the_cpu():
    meta = _cpu_meta([2, 1], 2)
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU compute path"):
        build_block_table(meta, i32, free_pages=i32)


def test_append_refusals_on_the_cpu():
    meta = _cpu_meta([2, 1], 2)
    cache = InferenceCache()
    plan = PagedMetadata(torch.zeros((2, 1), dtype=torch.int32), torch.zeros(3, dtype=torch.int64), None,
                         torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    k = torch.zeros((2, 2, 2, 16), dtype=torch.float16)
    with pytest.raises(ValueError, match="no cached KV entry"):
        cache.append_paged_kv_cache(0, k=k, v=k, q_meta=meta, plan=plan)
    cache.prefill_kv_cache(0, k_cache=torch.zeros((4, 16)), v_cache=torch.zeros((4, 16)), total_context_len=2,
                           context_batch_size=1, is_mla=False, num_heads=2, head_dim=16)
    with pytest.raises(ValueError, match="requires a paged entry"):
        cache.append_paged_kv_cache(0, k=k, v=k, q_meta=meta, plan=plan)
    pages = torch.zeros((2, 3, PAGE, 16), dtype=torch.float16)
    cache.prefill_paged_kv_cache(0, k_pages=pages, v_pages=pages.clone(), block_table=plan.block_table,
                                 context_lens=torch.zeros(2, dtype=torch.int32), is_mla=False, num_heads=2, head_dim=16)
    for match, kw in [
        ("requires v", dict(v=None)),
        ("k must be padded", dict(k=k[:1])),
        ("v must be padded", dict(v=k.view(-1, 16))),
        ("dtype/device", dict(k=k.float())),
        ("slot_mapping", dict(plan=PagedMetadata(plan.block_table, plan.slot_mapping[:2], None, None, plan.cu_seqlens_kv))),
        ("slot_mapping", dict(plan=PagedMetadata(plan.block_table, plan.slot_mapping.int(), None, None, plan.cu_seqlens_kv))),
        ("block_table", dict(plan=PagedMetadata(plan.block_table, plan.slot_mapping, None, None, plan.cu_seqlens_kv[:2]))),
    ]:
        with pytest.raises(ValueError, match=match):
            cache.append_paged_kv_cache(0, **{**dict(k=k, v=k, q_meta=meta, plan=plan), **kw})
    cache.prefill_paged_kv_cache(1, k_pages=pages.clone().requires_grad_(), v_pages=pages, block_table=plan.block_table,
                                 context_lens=torch.zeros(2, dtype=torch.int32), is_mla=False, num_heads=2, head_dim=16)
    with pytest.raises(ValueError, match="requires grad"):
        cache.append_paged_kv_cache(1, k=k, v=k, q_meta=meta, plan=plan)


def test_abi_refuses():
    lib = _lib.load()
    assert lib.fmlm_block_table(None, None) == -1
    p = _lib.BlockTableParams()
    assert lib.fmlm_block_table(p, None) == -1  # no outputs
    p.B, p.N, p.T = 2, 3, 7
    assert lib.fmlm_block_table_workspace_bytes(p) == -1  # more tokens than the batch holds
    p.T = 5
    assert lib.fmlm_block_table_workspace_bytes(p) == 4 * 8
    p.keep = 256
    assert lib.fmlm_block_table_workspace_bytes(p) == 4 * (8 + 6)
    p.max_pages = 1 << 26
    assert lib.fmlm_block_table_workspace_bytes(p) == -1  # lengths past 32 bits
    p.max_pages = 4
    for f in ("old_lens", "cu_seqlens", "token_indices", "block_table", "slot_mapping", "positions", "new_lens",
              "cu_kv"):
        setattr(p, f, 256)
    assert lib.fmlm_block_table(p, None) == -1  # no summary
    p.summary = 256
    assert lib.fmlm_block_table(p, None) == -5  # no workspace
    p.n_free = 3
    assert lib.fmlm_block_table(p, None) == -1  # no free list
    a = lib.fmlm_paged_append
    t = (_lib.PagedTensor * 1)()
    assert a(t, 1, 3, 1, 16, 1, 1, 1, None, 256, 64, None) == -2
    assert a(None, 1, 2, 1, 16, 1, 1, 1, None, 256, 64, None) == -1
    assert a(t, 1, 2, 1, 16, 1, 1, 1, None, 256, 64, None) == -1  # no source
    assert a(t, 1, 2, 1, 16, 0, 1, 1, None, None, 64, None) == 0
    t[0].src, t[0].pool = 256, 512
    assert a(t, 1, 2, 1, 16, 1, 1, 0, None, 256, 64, None) == -1  # padded without token indices
    t[0].src = 257
    assert a(t, 1, 2, 1, 16, 1, 1, 1, None, 256, 64, None) == -4


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------
def _table_case(seed, B, N, ctx, *, short=0, outgrow=0, fresh=False, keep=False, wide=False, lo=0):
    r = random.Random(seed)
    lens = [r.randint(lo, N) for _ in range(B)]
    old = [0 if fresh else r.randint(0, ctx) for _ in range(B)]
    width = -(-max(o + n for o, n in zip(old, lens)) // PAGE) - outgrow + (3 if wide else 0)
    pages = -(-ctx // PAGE)
    ids = list(range(B * (pages + -(-N // PAGE) + 1) + 5))
    r.shuffle(ids)
    table, at = [], 0
    for o in old:
        have = -(-o // PAGE)
        table.append(ids[at : at + have] + [-7] * (pages - have))
        at += have
    k = [r.random() < 0.5 for _ in range(sum(lens))] if keep else None
    need = sum(-(-(o + n) // PAGE) - -(-o // PAGE) for o, n in zip(old, lens))
    free = ids[at:][: max(0, need - short)] if short else ids[at:]
    return lens, old, None if fresh else table, free, max(width, 0), k


def _run_table(case, N, device, *, i64=False, check=False, max_pages=True):
    lens, old, table, free, width, keep = case
    dt = torch.int64 if i64 else torch.int32
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    plan = build_block_table(
        meta, torch.tensor(old, dtype=dt, device=device), free_pages=torch.tensor(free, dtype=dt, device=device),
        block_table=None if table is None else torch.tensor(table, dtype=dt, device=device).view(len(lens), -1),
        max_pages=width if max_pages else None,
        keep=None if keep is None else torch.tensor(keep, dtype=torch.bool, device=device), check=check)
    return meta, plan


def _expect(case, plan):
    lens, old, table, free, width, keep = case
    t, slots, pos, new, taken, lacking, bad = ref.block_table(old, lens, free, table, width, keep)
    assert plan.summary.tolist() == [taken, lacking, bad, sum(n - min(max(o, 0), n) for n, o in zip(new, old))]
    assert plan.block_table.tolist() == t
    assert plan.slot_mapping.tolist() == slots
    assert plan.positions.tolist() == pos
    assert plan.context_lens.tolist() == new
    assert plan.cu_seqlens_kv.tolist() == [sum(new[:i]) for i in range(len(new) + 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("B, N, ctx, lo", [
    (1, 1, 0, 1), (1, 1, 64, 1), (1, 200, 300, 200), (7, 5, 200, 0), (64, 1, 6000, 1), (64, 1, 1000, 0),
    (33, 130, 64, 0), (1500, 2, 130, 0), (2, 9000, 64, 0), (90, 700, 300, 0), (300, 40, 5000, 0), (5, 5000, 700, 0),
])
def test_table(B, N, ctx, lo, keep, device):
    """one workgroup (small) and three kernels (the last lines), with and without `keep`"""
    for seed, wide in ((B + N, False), (B + N + 1, True)):
        case = _table_case(seed, B, N, ctx, keep=keep, wide=wide, lo=lo)
        _expect(case, _run_table(case, N, device)[1])
        _expect(case, _run_table(case, N, device, i64=True)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("B, N, ctx", [(6, 150, 300), (700, 70, 2000)])
def test_table_that_does_not_fit(B, N, ctx, keep, device):
    """a short free list, requests that outgrow the table, old lengths out of range"""
    case = _table_case(1, B, N, ctx, short=B // 2 + 1, keep=keep)
    _expect(case, _run_table(case, N, device)[1])
    case = _table_case(2, B, N, ctx, outgrow=1, keep=keep)
    _expect(case, _run_table(case, N, device)[1])
    lens, old, table, free, width, k = _table_case(3, B, N, ctx, keep=keep)
    old[1], old[2] = -5, ctx + 1000
    case = (lens, old, table, free, width, k)
    t, slots, pos, new, *_ = ref.block_table(old, lens, free, table, width, k)
    plan = _run_table(case, N, device)[1]
    assert plan.block_table.tolist() == t and plan.slot_mapping.tolist() == slots
    assert plan.context_lens.tolist() == new and int(plan.summary[2]) == 2
    # no free pages at all, and an empty table
    case = _table_case(4, B, N, ctx, keep=keep)
    case = (*case[:3], [], *case[4:])
    _expect(case, _run_table(case, N, device)[1])
    case = _table_case(5, B, N, 0, fresh=True, keep=keep)
    case = (*case[:4], 0, case[5])
    _expect(case, _run_table(case, N, device)[1])


@pytest.mark.gpu
def test_table_of_new_requests_and_checks(device):
    case = _table_case(9, 5, 130, 0, fresh=True)
    meta, plan = _run_table(case, 130, device, check=True)
    _expect(case, plan)
    assert plan.pages_taken == int(plan.summary[0])
    lens, old, _, free, _, _ = case
    assert build_block_table(meta, torch.tensor(old, device=device), free_pages=torch.tensor(free, device=device),
                             ).block_table.shape == (5, 3)  # wide enough for N tokens
    z, f = torch.zeros(5, dtype=torch.int32, device=device), torch.arange(40, dtype=torch.int32, device=device)
    with pytest.raises(ValueError, match="more pages are needed"):
        build_block_table(meta, z, free_pages=f[:2])
    with pytest.raises(ValueError, match="must fit"):
        build_block_table(meta, z + 1, free_pages=f)
    with pytest.raises(ValueError, match="must fit"):
        build_block_table(meta, z, free_pages=f, max_pages=1)
    for match, kw in [("one row per", dict(block_table=f.view(4, 10))), ("max_pages", dict(max_pages=-1)),
                      ("keep must", dict(keep=f)), ("keep must", dict(keep=f[:5].bool())),
                      ("rank-2", dict(block_table=f))]:
        with pytest.raises(ValueError, match=match):
            build_block_table(meta, z, free_pages=f, **kw)
    with pytest.raises(ValueError, match="one entry per sequence"):
        build_block_table(meta, z[:4], free_pages=f)
    for bad in (z.float(), z[None], z.tolist()):
        with pytest.raises(ValueError, match="rank-1"):
            build_block_table(meta, bad, free_pages=f)
    for kw in (dict(free_pages=f.cpu()), dict(free_pages=f, block_table=f.cpu().view(5, 8))):
        with pytest.raises(ValueError, match="no CPU compute path"):
            build_block_table(meta, z, **kw)


@pytest.mark.gpu
def test_table_in_a_graph(device):
    case = _table_case(11, 40, 20, 900, keep=True)
    lens, old, table, free, width, keep = case
    meta = build_pack_metadata(torch.tensor(lens, device=device), 20, 32)
    o, k = torch.tensor(old, dtype=torch.int32, device=device), torch.tensor(keep, device=device)
    f = torch.tensor(free, dtype=torch.int32, device=device)
    t = torch.tensor(table, dtype=torch.int32, device=device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = build_block_table(meta, o, free_pages=f, block_table=t, max_pages=width, keep=k, check=False)
    for s in range(3):
        r = random.Random(s)
        old = [r.randint(0, x) for x in old]
        keep = [r.random() < 0.7 for _ in keep]
        o.copy_(torch.tensor(old))
        k.copy_(torch.tensor(keep))
        graph.replay()
        torch.cuda.synchronize()
        _expect((lens, old, table, free, width, keep), plan)


def _pool(h, P, D, dtype, device, seed):
    return torch.randn((h, P, PAGE, D), generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def _append_case(device, dtype, H, D, mla, lens, N, packed, keep, seed=0):
    r = random.Random(seed)
    B, T, hk = len(lens), sum(lens), 1 if mla else H
    g = torch.Generator().manual_seed(seed)
    shape = (hk * T, D) if packed else (B, H, N, D)
    k, v = (torch.randn(shape, generator=g).to(dtype).to(device) for _ in range(2))
    old = [r.randint(0, 100) for _ in lens]
    width = -(-(max(old) + N) // PAGE)
    P = B * width + 4
    ids = list(range(P))
    r.shuffle(ids)
    table = [ids[b * width : b * width + -(-o // PAGE)] + [-1] * (width - -(-o // PAGE)) for b, o in enumerate(old)]
    free = [i for i in ids if all(i not in row for row in table)]
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    kept = torch.tensor([r.random() < 0.6 for _ in range(T)], dtype=torch.bool, device=device) if keep else None
    bt = torch.tensor(table, dtype=torch.int32, device=device)
    oldt = torch.tensor(old, dtype=torch.int32, device=device)
    kp, vp = _pool(hk, P, D, dtype, device, 1), None if mla else _pool(hk, P, D, dtype, device, 2)
    cache = InferenceCache()
    cache.prefill_paged_kv_cache(0, k_pages=kp, v_pages=vp, block_table=bt, context_lens=oldt, is_mla=mla, num_heads=H,
                                 head_dim=D)
    plan = build_block_table(meta, oldt, free_pages=torch.tensor(free, dtype=torch.int32, device=device), block_table=bt,
                             keep=kept)
    return k, v, meta, plan, kp, vp, cache


def _expected_pool(pool, x, meta, slots, hk):
    want = pool.clone()
    T = int(meta.total_tokens)
    rows = x.view(hk, T, -1) if x.ndim == 2 else x.transpose(1, 2).reshape(meta.B * meta.N, x.shape[1], -1)[
        meta.token_indices][:, :hk].transpose(0, 1)
    ok = (slots >= 0) & (slots < pool.shape[1] * PAGE)
    want.view(hk, -1, x.shape[-1])[:, slots[ok]] = rows[:, ok]
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H, D, mla", [(3, 16, False), (1, 64, False), (9, 128, False), (4, 256, False), (4, 512, True)])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("keep", [False, True])
def test_append(dtype, H, D, mla, packed, keep, device):
    k, v, meta, plan, kp, vp, cache = _append_case(device, dtype, H, D, mla, [1, 0, 70, 33], 70, packed, keep, D)
    hk = 1 if mla else H
    want = [_expected_pool(p, x, meta, plan.slot_mapping, hk) for p, x in ((kp, k), (vp, v)) if p is not None]
    cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan)
    for p, w in zip((kp, vp), want):
        assert torch.equal(p, w)
    entry = cache.layer_entry(0)
    assert torch.equal(entry.block_table, plan.block_table) and torch.equal(entry.cu_seqlens_kv, plan.cu_seqlens_kv)
    assert entry.k_cache.data_ptr() == kp.data_ptr() and entry.context_batch_size == 4


@pytest.mark.gpu
def test_append_of_views_and_bad_slots(device):
    """q/k/v of one projection, an odd start, slots outside the pool and a sequence of no tokens"""
    H, D, N = 2, 64, 40
    k, v, meta, plan, kp, vp, cache = _append_case(device, torch.float16, H, D, False, [40, 3, 0], N, False, False, 3)
    qkv = torch.randn((3, N, 3, H, D), device=device).half()
    kk = qkv[:, :, 1].transpose(1, 2)
    buf = torch.empty(3 * H * N * D + 1, dtype=torch.float16, device=device)
    vv = buf[1:].view(3, H, N, D).copy_(v)
    plan.slot_mapping[5] = kp.shape[1] * PAGE
    plan.slot_mapping[6] = 2**40
    plan.slot_mapping[7] = -2**40
    want = [_expected_pool(p, x, meta, plan.slot_mapping, H) for p, x in ((kp, kk), (vp, vv))]
    cache.append_paged_kv_cache(0, k=kk, v=vv, q_meta=meta, plan=plan)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    # a layout whose last dim is not contiguous
    kt = k.transpose(2, 3).contiguous().transpose(2, 3)
    cache.append_paged_kv_cache(0, k=kt, v=v, q_meta=meta, plan=plan)
    assert torch.equal(kp, _expected_pool(kp, k, meta, plan.slot_mapping, H))


@pytest.mark.gpu
def test_append_on_another_stream_and_in_a_graph(device):
    """A step's table and append, captured: replays with new lengths, rows and kept tokens."""
    H, D, N, lens = 3, 64, 20, [20, 1, 0, 13]
    k, v, meta, plan, kp, vp, cache = _append_case(device, torch.bfloat16, H, D, False, lens, N, False, False, 5)
    want = [_expected_pool(p, x, meta, plan.slot_mapping, H) for p, x in ((kp, k), (vp, v))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan)
    side.synchronize()
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    old = torch.tensor([3, 60, 0, 64], dtype=torch.int32, device=device)
    table = torch.tensor([[0, -1], [1, -1], [-1, -1], [2, -1]], dtype=torch.int32, device=device)
    free = torch.arange(3, 8, dtype=torch.int32, device=device)
    kept = torch.ones(sum(lens), dtype=torch.bool, device=device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = build_block_table(meta, old, free_pages=free, block_table=table, keep=kept, check=False)
        cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=step)
    g = torch.Generator().manual_seed(1)
    for ctx in ([3, 60, 0, 64], [64, 0, 0, 50], [44, 64, 0, 1]):
        old.copy_(torch.tensor(ctx))
        kept.copy_(torch.rand(sum(lens), generator=g) < 0.7)
        k.copy_(torch.randn(k.shape, generator=g))
        v.copy_(torch.randn(v.shape, generator=g))
        eager = build_block_table(meta, old, free_pages=free, block_table=table, keep=kept)
        want = [_expected_pool(p, x, meta, eager.slot_mapping, H) for p, x in ((kp, k), (vp, v))]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(step.slot_mapping, eager.slot_mapping)
        assert torch.equal(step.block_table, eager.block_table)
        assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


@pytest.mark.gpu
def test_append_past_32_bits(device):
    """A pool of more than 2^32 elements: rows of its first and last pages."""
    D, N, lens, P = 512, 70, [70, 5], 131100
    pool = torch.empty((1, P, PAGE, D), dtype=torch.bfloat16, device=device)
    ends = [0, 1, P - 3, P - 2, P - 1]
    pool[:, ends] = 0
    cache = InferenceCache()
    table = torch.tensor([[P - 1, -1], [0, -1]], dtype=torch.int32, device=device)
    old = torch.tensor([60, 63], dtype=torch.int32, device=device)
    cache.prefill_paged_kv_cache(0, k_pages=pool, block_table=table, context_lens=old, is_mla=True, num_heads=2, head_dim=D)
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    free = torch.tensor([P - 3, 1, P - 2], dtype=torch.int32, device=device)
    plan = build_block_table(meta, old, free_pages=free, block_table=table, max_pages=3)
    assert plan.pages_taken == 3 and int(plan.slot_mapping.max()) * D > 2**32
    k = torch.randn((2, 2, N, D), device=device).bfloat16()
    cache.append_paged_kv_cache(0, k=k, q_meta=meta, plan=plan)
    rows = torch.cat([k[0, 0, :70], k[1, 0, :5]])
    flat = pool.view(-1, D)
    assert torch.equal(flat[plan.slot_mapping], rows)
    left = pool[:, ends]
    assert int((left != 0).any(-1).sum()) == sum(lens)


@pytest.mark.gpu
def test_appended_context_is_what_attention_reads(device):
    """Attend, append, attend: the second call over the pages equals one over the same rows
    stored contiguously, bit for bit; rows of the pool that hold no token may be NaN."""
    torch.manual_seed(4)
    H, D, N, lens = 4, 128, 90, [90, 1, 50]
    B = len(lens)
    P, width = 12, 3
    kp, vp = (torch.full((H, P, PAGE, D), float("nan"), dtype=torch.bfloat16, device=device) for _ in range(2))
    free = torch.randperm(P, device=device).int()
    cache = InferenceCache()
    zero = torch.zeros(B, dtype=torch.int32, device=device)
    cache.prefill_paged_kv_cache(0, k_pages=kp, v_pages=vp, block_table=torch.full((B, width), -1, dtype=torch.int32,
                                 device=device), context_lens=zero, is_mla=False, num_heads=H, head_dim=D)
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    plan = build_block_table(meta, zero, free_pages=free, max_pages=width)
    k, v = (torch.randn((B, H, N, D), device=device).bfloat16() for _ in range(2))
    cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan)
    flat = InferenceCache()
    rows = [torch.cat([x[b, :, :n] for b, n in enumerate(lens)], 1).reshape(-1, D).contiguous() for x in (k, v)]
    flat.prefill_kv_cache(0, k_cache=rows[0], v_cache=rows[1], total_context_len=sum(lens),
                          cu_seqlens_kv=meta.cu_seqlens, context_batch_size=B, is_mla=False, num_heads=H, head_dim=D)
    meta1 = build_pack_metadata(torch.tensor([1, 2, 1], device=device), 2, 32)
    q1, k1, v1 = (torch.randn((B, H, 2, D), device=device).bfloat16() for _ in range(3))
    a = flash_attn_mlm_compressed(q1, k1, v1, H, meta1, 0.1, cache, 0)
    b = flash_attn_mlm_compressed(q1, k1, v1, H, meta1, 0.1, flat, 0)
    assert torch.equal(a, b) and bool(a.isfinite().all())
    plan2 = build_block_table(meta1, plan.context_lens, free_pages=free[plan.pages_taken :], block_table=plan.block_table)
    cache.append_paged_kv_cache(0, k=k1, v=v1, q_meta=meta1, plan=plan2)
    assert np.diff(plan2.cu_seqlens_kv.tolist()).tolist() == [91, 3, 51]
    c = flash_attn_mlm_compressed(q1, k1, v1, H, meta1, 0.1, cache, 0)
    assert not torch.equal(a, c) and bool(c.isfinite().all())


def test_append_is_a_change_in_place_to_autograd(monkeypatch):
    """What was saved of the pools before an append is refused in a backward after it."""
    from flash_mlm.host import paged

    calls = []
    monkeypatch.setattr(paged, "paged_append", lambda pairs, **kw: calls.append(len(pairs)))
    for mla in (False, True):
        for inference in (False, True):
            with torch.inference_mode(inference):
                pages = torch.zeros((1 if mla else 2, 3, PAGE, 16), dtype=torch.float16)
                vpages = None if mla else pages.clone()
                k = torch.zeros((2, 2, 2, 16), dtype=torch.float16)
            table, zero = torch.zeros((2, 1), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
            cache = InferenceCache()
            cache.prefill_paged_kv_cache(0, k_pages=pages, v_pages=vpages, block_table=table, context_lens=zero, is_mla=mla,
                                         num_heads=2, head_dim=16)

            def append(lens):
                plan = PagedMetadata(table, torch.zeros(sum(lens), dtype=torch.int64), None, zero,
                                     torch.zeros(3, dtype=torch.int32))
                cache.append_paged_kv_cache(0, k=k, v=k, q_meta=_cpu_meta(lens, 2), plan=plan)

            if inference:  # these count no versions
                append([2, 1])
                continue
            saved = [torch.ones(t.shape, requires_grad=True) * t for t in (pages, vpages) if t is not None]
            before = pages._version
            append([0, 0])  # nothing is written
            assert pages._version == before
            append([2, 1])
            assert pages._version > before and (mla or vpages._version > 0)
            for x in saved:
                with pytest.raises(RuntimeError, match="modified by an inplace"):
                    x.sum().backward()
    assert calls == [2, 2, 1, 1]


@pytest.mark.gpu
def test_backward_after_an_append_is_refused(device):
    """Attention's backward reads the pool again: after an append it raises, as after any change in
    place, instead of differentiating the new rows."""
    H, D, N = 3, 64, 20
    k, v, meta, plan, kp, vp, cache = _append_case(device, torch.bfloat16, H, D, False, [20, 1, 0, 13], N, False, False, 6)
    q = torch.randn((4, H, N, D), device=device).bfloat16().requires_grad_()

    def attend():
        return flash_attn_mlm_compressed(q, k, v, H, meta, 0.125, cache, 0)

    want = torch.autograd.grad(attend().sum(), q)[0]
    out, other = attend(), attend()
    assert torch.equal(torch.autograd.grad(other.sum(), q)[0], want)
    cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()
    assert torch.autograd.grad(attend().sum(), q)[0].isfinite().all()


@pytest.mark.parametrize("b", [1, 3, 5])
def test_append_refuses_the_plan_of_another_step(b):
    """A plan for another number of requests than q_meta has"""
    pages = torch.zeros((2, 3, PAGE, 16), dtype=torch.float16)
    k, zero = torch.zeros((2, 2, 2, 16), dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    cache = InferenceCache()
    cache.prefill_paged_kv_cache(0, k_pages=pages, v_pages=pages.clone(), block_table=zero.view(2, 1), context_lens=zero,
                                 is_mla=False, num_heads=2, head_dim=16)
    entry = cache.layer_entry(0)
    plan = PagedMetadata(torch.zeros((b, 1), dtype=torch.int32), torch.zeros(3, dtype=torch.int64), None,
                         torch.zeros(b, dtype=torch.int32), torch.zeros(b + 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="requests"):
        cache.append_paged_kv_cache(0, k=k, v=k, q_meta=_cpu_meta([2, 1], 2), plan=plan)
    assert cache.layer_entry(0) is entry


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("B, n, width", [(64, 1, 128), (64, 1, 129), (2048, 1, 4), (2049, 2, 3), (2731, 1, 3), (1, 4096, 70),
                                         (1, 4097, 70), (4, 1024, 2048), (8192, 0, 1), (4096, 1, 2), (4097, 1, 2)])
def test_table_around_the_sizes_of_one_workgroup(B, n, width, keep, device):
    """Two rounds of table entries, one of tokens, more requests than threads: and one more of each"""
    r = random.Random(B + n + width)
    lens = [n] * B
    old = [r.randint(0, min(min(width, 40) * PAGE, width * PAGE - n)) if r.random() < 0.9 else 0 for _ in lens]
    ids = r.sample(range(10 * B * 40 + 100), B * min(width, 40) + 2 * B + 70)
    table = [ids[b * min(width, 40) :][: min(width, 40)] + [-1] * (width - min(width, 40)) for b in range(B)]
    free = ids[B * min(width, 40) :]
    kept = [r.random() < 0.5 for _ in range(n * B)] if keep else None
    case = (lens, old, table, free, width, kept)
    _expect(case, _run_table(case, max(n, 1), device)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", ["offsets", "tokens"])
def test_inconsistent_metadata_stays_in_bounds(bad, device):
    """Metadata that was not made by build_pack_metadata: offsets and token indices far out of range.  What
    they say is clamped to the tensors; requests whose own are right get what is theirs."""
    import dataclasses

    from flash_mlm import build_tree_metadata, qk_norm_rope

    B, N, H, D, far = 4, 3000, 2, 64, 2**30
    for lens in ([3, 0, 7, 5], [3000, 10, 2900, 7]):  # one workgroup, and three kernels
        T = sum(lens)
        meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
        cu, tok = meta.cu_seqlens.clone(), meta.token_indices.clone()
        if bad == "offsets":
            cu[:] = torch.tensor([-far, far, 2, -7, far], device=device)
        else:
            tok[1:] = torch.randint(-(2**40), 2**40, (T - 1,), device=device)
            tok[1::2] = 2**32 - 1
        wrong = dataclasses.replace(meta, cu_seqlens=cu, token_indices=tok, launch_memo={}, kernel_schedules={})
        old = torch.tensor([5, 70, 0, 64], dtype=torch.int32, device=device)
        free = torch.arange(400, dtype=torch.int32, device=device)
        table = torch.full((B, 100), 399, dtype=torch.int32, device=device)
        for keep in (None, torch.rand(T, device=device) < 0.5):
            plan = build_block_table(wrong, old, free_pages=free, block_table=table, keep=keep, check=False)
            assert int(plan.slot_mapping.max()) < 400 * PAGE and int(plan.slot_mapping.min()) >= -1
        q, k = (torch.randn((B, H, N, D), device=device) for _ in range(2))
        cos, sin = torch.ones((50, 32), device=device), torch.zeros((50, 32), device=device)
        for where in (dict(positions=torch.zeros(T, dtype=torch.int32, device=device)),
                      dict(context_lens=torch.zeros(B, dtype=torch.int64, device=device))):
            a, b = qk_norm_rope(q, k, cos=cos, sin=sin, q_meta=wrong, **where)
            assert bool(a.isfinite().all()) and bool(b.isfinite().all())
            a, b = qk_norm_rope(torch.randn((H * T, D), device=device), torch.randn((H * T, D), device=device), cos=cos,
                                sin=sin, q_meta=wrong, **where)
            assert bool(a.isfinite().all())
        cache = InferenceCache()
        kp, vp = (torch.zeros((H, 400, PAGE, D), dtype=torch.bfloat16, device=device) for _ in range(2))
        cache.prefill_paged_kv_cache(0, k_pages=kp, v_pages=vp, block_table=table, context_lens=old, is_mla=False, num_heads=H,
                                     head_dim=D)
        good = build_block_table(meta, old, free_pages=free, block_table=table, check=False)
        cache.append_paged_kv_cache(0, k=q.bfloat16(), v=k.bfloat16(), q_meta=wrong, plan=good)
        assert torch.equal(kp.view(H, -1, D)[:, good.slot_mapping[0]], q[0, :, 0].bfloat16())
        small = dataclasses.replace(wrong, N=200)
        tree = build_tree_metadata(torch.full((T,), -1, device=device), small, check=False)
        assert tree.mask.shape == (T, 4)
        torch.cuda.synchronize()
