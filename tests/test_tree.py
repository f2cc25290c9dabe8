"""build_tree_metadata and flash_attn_mlm_tree: refusals (CPU), and on the GPU masks against sets
of ancestors, attention against its 64-bit restatement (oracle/paged_step_ref.py), and a
speculative decoding loop over a paged cache.

Tolerances.  With W = sum of w |v| of an output element, h half a step of the type and u =
2^-24: the context's part is rounded once (h of it) and the output once more (h |o|); the
probabilities of both parts are rounded (2 h W with their sums); a score's error e moves the
result by at most 2 e W, and e is (D + 16) u S in fp32, S = scale * sum |q k|; exponentials and
sums add (keys + 64) u W at most.
Fp16 probabilities below 2^-14 have an absolute error of 2^-25 each.
"""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from flash_mlm import (
    InferenceCache,
    PackMetadata,
    TreeMetadata,
    _lib,
    build_block_table,
    build_pack_metadata,
    build_tree_metadata,
    flash_attn_mlm_tree,
    qk_norm_rope,
    unpack_from_kernel,
)
from oracle import paged_step_ref as ref

PAGE, U = 64, 2.0**-24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _f(t):
    return t.detach().double().cpu().numpy()


def _random_parents(r, lens):
    return [-1 if i == 0 or r.random() < 0.1 else (i - 1 if r.random() < 0.5 else r.randrange(i))
            for n in lens for i in range(n)]


def _cpu_meta(lens, N):
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    tok = torch.tensor([b * N + p for b, n in enumerate(lens) for p in range(n)], dtype=torch.int64)
    return PackMetadata(B=len(lens), N=N, lengths=torch.tensor(lens, dtype=torch.int32), cu_seqlens=cu, token_indices=tok,
                        total_tokens=sum(lens), batch_ids_block_n=32, batch_ids_q=cu, q_tile_starts_q=cu)


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------
def test_refusals_on_the_cpu():
    meta = _cpu_meta([2, 1], 2)
    par = torch.tensor([-1, 0, -1])
    with pytest.raises(ValueError, match="no CPU compute path"):
        build_tree_metadata(par, meta)
    with pytest.raises(ValueError, match="parents must"):
        build_tree_metadata(par[:2], meta)
    with pytest.raises(ValueError, match="parents must"):
        build_tree_metadata(par.float(), meta)
    with pytest.raises(ValueError, match="context_lens must"):
        build_tree_metadata(par, meta, context_lens=par)
    with pytest.raises(ValueError, match="at most 256"):
        build_tree_metadata(par, _cpu_meta([2, 1], 257))
    tree = TreeMetadata(torch.zeros((3, 1), dtype=torch.int64), torch.zeros(3, dtype=torch.int32))
    q = torch.zeros((2, 2, 2, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA tensors"):
        flash_attn_mlm_tree(q, q, q, 2, meta, tree, 1.0)
    with pytest.raises(ValueError, match="num_heads"):
        flash_attn_mlm_tree(q, q, q, 3, meta, tree, 1.0)
    with pytest.raises(ValueError, match="q_meta"):
        flash_attn_mlm_tree(q[:1], q[:1], q[:1], 2, meta, tree, 1.0)
    with pytest.raises(ValueError, match="tree.mask"):
        flash_attn_mlm_tree(q, q, q, 2, meta, TreeMetadata(tree.mask[:2], None), 1.0)
    with pytest.raises(ValueError, match="no backward"):
        flash_attn_mlm_tree(q.clone().requires_grad_(), q, q, 2, meta, tree, 1.0)


def test_abi_refuses():
    lib = _lib.load()
    m = lib.fmlm_tree_mask
    assert m(None, 0, None, 1, 257, 1, 5, None, 0, None, None, None, None) == -1  # too long
    assert m(None, 0, None, 1, 65, 1, 1, None, 0, None, None, None, None) == -1  # too few words
    assert m(None, 0, None, 1, 4, 4, 1, None, 0, None, None, None, None) == -1  # no tensors
    assert m(None, 0, None, 0, 4, 0, 1, None, 0, None, None, None, None) == 0
    f = lib.fmlm_attn_tree_fwd

    def a(p, mask, words, ws=None, n=0):
        return f(p, mask, words, ws, n, None)

    assert a(None, None, 1) == -1
    p = _lib.AttnParams()
    p.dtype, p.B, p.H, p.D, p.N, p.total_q = _lib.DTYPE_BF16, 1, 1, 64, 4, 4
    p.q = p.k = p.v = p.o = p.cu_seqlens_q = 256
    assert a(p, 256, 1) == -1  # not a tree call
    p.flags = _lib.FLAG_TREE
    assert a(p, None, 1) == -1  # no mask
    p.N = p.total_q = 300
    assert a(p, 256, 8) == -1  # too long
    p.N, p.total_q = 0, 257
    assert a(p, 256, 8) == -1  # too long, for all that is known
    p.N, p.total_q = 4, 4
    assert a(p, 256, 0) == -1  # no words
    assert a(p, 256, 1) == -5  # the attention kernel's workspace
    assert lib.fmlm_attn_tree_workspace_bytes(p) == 0
    p.cu_seqlens_q = None
    assert a(p, 256, 1) == -1  # dense
    p.cu_seqlens_q = 256
    p.flags |= _lib.FLAG_PREFILL
    assert a(p, 256, 1) == -1
    p.flags = _lib.FLAG_TREE
    assert lib.fmlm_attn_fwd(p, None) == -1
    assert lib.fmlm_attn_fwd_noalloc(p, None) == -1
    g = _lib.AttnGrads()
    g.dout = g.dq = g.dk = g.dv = 256
    assert lib.fmlm_attn_bwd(p, g, None) == -1
    p.dtype = _lib.DTYPE_F32
    assert lib.fmlm_attn_tree_workspace_bytes(p) == 0 and a(p, 256, 1) == -5
    p.D, p.v = 512, 264  # the tree's part in a kernel of its own
    assert lib.fmlm_attn_tree_workspace_bytes(p) == 4 * 4 * 513
    assert a(p, 256, 1) == -5
    assert a(p, 256, 1, 256, 4 * 4 * 513) == -4
    p.dtype, p.D = _lib.DTYPE_BF16, 512  # only the latent
    assert lib.fmlm_attn_workspace_bytes(p) == -3
    assert a(p, 256, 1, 256, 4 * 4 * 513) == -4
    p.v = 256
    assert a(p, 256, 1, 256, 4 * 4 * 513) == -3


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("lens, N", [([1], 1), ([2, 0, 1], 2), ([64, 63, 65], 65), ([256, 1, 129], 256),
                                     ([7] * 300, 9)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_masks(lens, N, dtype, device):
    r = random.Random(N)
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    start = [r.randint(0, 100) for _ in lens]
    b = np.repeat(np.arange(len(lens)), lens)
    for parents in (_random_parents(r, lens), [i - 1 for n in lens for i in range(n)], [-1] * sum(lens)):
        seen = ref.ancestors(parents, lens)
        for ctx in (None, torch.tensor(start, dtype=dtype, device=device)):
            tree = build_tree_metadata(torch.tensor(parents, dtype=dtype, device=device), meta, context_lens=ctx)
            assert np.array_equal(tree.mask.cpu().numpy(), ref.mask_words(seen, tree.mask.shape[1]))
            want = [len(s) - 1 + (0 if ctx is None else start[x]) for s, x in zip(seen, b)]
            assert tree.positions.tolist() == want


@pytest.mark.gpu
def test_bad_parents(device):
    meta = build_pack_metadata(torch.tensor([4, 3], device=device), 4, 32)
    parents = [-1, 1, -2, 9, -1, 0, 2]
    t = torch.tensor(parents, device=device)
    with pytest.raises(ValueError, match="before their children"):
        build_tree_metadata(t, meta)
    tree = build_tree_metadata(t, meta, check=False)
    assert np.array_equal(tree.mask.cpu().numpy(), ref.mask_words(ref.ancestors(parents, [4, 3]), 1))


def _close(got, q, k, v, seen, scale, kc, vc, dtype):
    o, w, c, s = ref.tree_attention(_f(q), _f(k), _f(v), seen, scale, _f(kc), _f(vc))
    h = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    keys, D = kc.shape[0] + k.shape[0], q.shape[-1]
    e = (D + 16) * U * s[:, None]
    bound = h * (np.abs(o) + c) + (2 * h + 2 * e + (keys + 64) * U) * w
    if dtype == torch.float16:
        bound = bound + 2.0**-25 * (keys * np.abs(np.concatenate([_f(vc), _f(v)])).max() + 1)
    err = np.abs(_f(got) - o)
    assert np.all(err <= bound * 1.01 + 1e-30), f"worst {np.max(err / (bound + 1e-30)):.3f} of the bound"


def _context(kind, lens, H, D, mla, dtype, device, seed=0):
    """(cache, list of (k, v) [H_kv, C_b, D] of every sequence, extra arguments)"""
    g = torch.Generator().manual_seed(seed)
    hk, B = 1 if mla else H, len(lens)
    cache, kw = InferenceCache(), {}
    if kind == "none":
        e = torch.empty((hk, 0, D), dtype=dtype, device=device)
        return None, [(e, e)] * B, kw
    n = {"shared": [lens[0]], "index": lens[:2]}.get(kind, lens)
    rows = [[torch.randn((hk, c, D), generator=g).to(dtype).to(device) for _ in range(1 if mla else 2)] for c in n]
    if kind in ("paged", "index"):
        need = [-(-c // PAGE) for c in n]
        P = sum(need) + 2
        ids = torch.randperm(P, generator=g).tolist()
        pools = [torch.full((hk, P, PAGE, D), float("nan"), dtype=dtype, device=device) for _ in range(1 if mla else 2)]
        table = torch.full((len(n), max(need + [1])), -1, dtype=torch.int32)
        for b, c in enumerate(n):
            for i in range(need[b]):
                page = ids.pop()
                table[b, i] = page
                for pool, x in zip(pools, rows[b]):
                    part = x[:, i * PAGE : (i + 1) * PAGE]
                    pool[:, page, : part.shape[1]] = part
        cache.prefill_paged_kv_cache(0, k_pages=pools[0], v_pages=None if mla else pools[1], block_table=table.to(device),
                                     context_lens=torch.tensor(n), is_mla=mla, num_heads=H, head_dim=D)
    else:
        flat = [torch.cat([x[i] for x in rows], 1).reshape(-1, D).contiguous() for i in range(1 if mla else 2)]
        cu = torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32, device=device)
        cache.prefill_kv_cache(0, k_cache=flat[0], v_cache=None if mla else flat[1], total_context_len=sum(n),
                               cu_seqlens_kv=cu, context_batch_size=len(n), is_mla=mla, num_heads=H, head_dim=D)
    pick = list(range(B))
    if kind == "shared":
        pick = [0] * B
    if kind == "index":
        pick = [b % 2 for b in range(B)]
        kw["context_index"] = torch.tensor(pick, dtype=torch.int32, device=device)
    return cache, [(rows[i][0], rows[i][-1]) for i in pick], kw


def _run(device, dtype, *, lens, N, H, D, ctx, kind, mla=False, scale=None, seed=0, parents=None, spoil=None):
    r = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    scale = D**-0.5 if scale is None else scale
    q, k, v = (torch.randn((B, H, N, D), generator=g).to(dtype).to(device) for _ in range(3))
    if mla:
        v = k
    parents = _random_parents(r, lens) if parents is None else parents
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    tree = build_tree_metadata(torch.tensor(parents, device=device), meta)
    cache, rows, kw = _context(kind, ctx, H, D, mla, dtype, device, seed)
    if spoil is not None:
        spoil(k, v)
    out = flash_attn_mlm_tree(q, k, v, H, meta, tree, scale, cache, None if cache is None else 0, is_mla=mla, **kw)
    T, at, seen = sum(lens), 0, ref.ancestors(parents, lens)
    got = out.view(H, T, D)
    for b, n in enumerate(lens):
        for h in range(H if n else 0):
            j = 0 if mla else h
            _close(got[h, at : at + n], q[b, h, :n], k[b, j, :n], v[b, j, :n], seen[at : at + n], scale,
                   rows[b][0][j], rows[b][1][j], dtype)
        at += n
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("kind", ["none", "packed", "paged"])
def test_attention(dtype, D, kind, device):
    if dtype == "fp32" and kind == "paged":
        pytest.skip("paged contexts are bf16 / fp16")
    _run(device, DT[dtype], lens=[40, 1, 0, 17], N=41, H=3, D=D, ctx=[70, 0, 5, 129], kind=kind, seed=D)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("kind", ["none", "packed", "paged", "index"])
def test_mla(dtype, kind, device):
    if dtype == "fp32" and kind in ("paged", "index"):
        pytest.skip("paged contexts are bf16 / fp16")
    _run(device, DT[dtype], lens=[7, 40], N=40, H=2, D=128, ctx=[30, 100], kind=kind, mla=True, seed=2)
    _run(device, DT[dtype], lens=[5, 33, 1], N=33, H=4, D=512, ctx=[300, 65, 0], kind=kind, mla=True, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["packed", "paged"])
@pytest.mark.parametrize("lens, H, ctx", [([5, 33, 1, 0, 2], 16, [4000, 65, 900, 70, 0]), ([1], 32, [3800]),
                                          ([9, 12], 64, [600, 2000])])
def test_mla_split_contexts(kind, lens, H, ctx, device):
    """Long latent contexts of few rows are split; the tree's kernel merges the parts, beside
    sequences that are not split or have no context."""
    _run(device, torch.bfloat16, lens=lens, N=max(lens), H=H, D=512, ctx=ctx, kind=kind, mla=True, seed=5)


@pytest.mark.gpu
def test_buffers_of_a_launch_are_apart(device, monkeypatch):
    """The records of a split context and the rows that the tree's part reads live at once."""
    lib, seen = _lib.load(), []
    launch = lib.fmlm_attn_tree_fwd

    def spy(p, mask, words, ws, n, stream):
        seen.append((p.workspace, p.workspace_bytes, ws, n))
        return launch(p, mask, words, ws, n, stream)

    monkeypatch.setattr(lib, "fmlm_attn_tree_fwd", spy)
    lens = [9, 9, 9, 8, 9, 9, 9, 8, 9, 7, 8, 9, 8]
    ctx = [5858, 6266, 5193, 3825, 4380, 5922, 3749, 2784, 5662, 7539, 4647, 4385, 2065]
    _run(device, torch.float16, lens=lens, N=9, H=32, D=512, ctx=ctx, kind="paged", mla=True)
    assert seen
    for rec, rec_bytes, ws, n in seen:
        assert rec and rec_bytes > 0 and ws and n > 0
        assert rec + rec_bytes <= ws or ws + n <= rec


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, kind", [("bf16", "shared"), ("fp16", "index"), ("fp32", "shared"), ("bf16", "index")])
def test_shared_and_indexed_contexts(dtype, kind, device):
    _run(device, DT[dtype], lens=[9, 20, 3], N=20, H=2, D=64, ctx=[200, 77, 1], kind=kind, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("chain", [False, True])
def test_long_drafts_and_long_contexts(dtype, chain, device):
    lens = [256, 200, 1]
    parents = [i - 1 for n in lens for i in range(n)] if chain else None
    _run(device, DT[dtype], lens=lens, N=256, H=2, D=64, ctx=[5000, 1, 3], kind="packed", seed=5, parents=parents)


@pytest.mark.gpu
def test_wide_head_dim_tiles(device):
    """D = 256: 64- and 128-row workgroups, and the library's choice of the latter"""
    from flash_mlm.host.host import tile_config

    run = dict(lens=[200, 140, 3], N=200, H=2, D=256, ctx=[130, 64, 300], kind="packed", seed=2)
    with tile_config(1):
        a = _run(device, torch.bfloat16, **run)
    with tile_config(2):
        b = _run(device, torch.bfloat16, **run)
    assert a.shape == b.shape
    with tile_config(2), pytest.raises(RuntimeError, match="invalid argument"):
        _run(device, torch.bfloat16, lens=[9], N=9, H=2, D=64, ctx=[9], kind="packed")
    _run(device, torch.float16, lens=[70] * 8, N=70, H=8, D=256, ctx=[2300] * 8, kind="paged", seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_scales(dtype, scale, device):
    _run(device, DT[dtype], lens=[30, 2], N=30, H=2, D=64, ctx=[90, 0], kind="packed", scale=scale, seed=6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("D, mla", [(32, False), (64, False), (128, False), (256, False), (512, True)])
@pytest.mark.parametrize("ctx", [[0, 0, 0], [70, 0, 4000]])
def test_masks_of_any_kind(dtype, D, mla, ctx, device):
    """Masks that no tree has: rows that see nothing (they have the context alone, or are zero), rows
    that see later tokens or only another key tile's, bits past the sequence, a word too many."""
    r, H, lens, N = random.Random(D), 2, [90, 3, 150], 151
    g = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn((3, H, N, D), generator=g).to(DT[dtype]).to(device) for _ in range(3))
    v = k if mla else v
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    seen = []
    for n in lens:
        kinds = [set(), set(range(n)), {n - 1}, set(range(64, n)), set(range(min(64, n)))]
        seen += [kinds[i] if i < 5 else {j for j in range(n) if r.random() < 0.3} if i % 7 else set() for i in range(n)]
    words = np.zeros((sum(lens), 4), dtype=np.uint64)
    past = [n for n in lens for _ in range(n)]
    for t, (s, n) in enumerate(zip(seen, past)):
        for j in list(s) + [x for x in (n, n + 1, 200, 255) if r.random() < 0.5]:
            words[t, j // 64] |= np.uint64(1 << (j % 64))
    tree = TreeMetadata(torch.from_numpy(words.view(np.int64)).to(device), None)
    cache, rows, kw = _context("packed", ctx, H, D, mla, DT[dtype], device, 3)
    got = flash_attn_mlm_tree(q, k, v, H, meta, tree, D**-0.5, cache, 0, is_mla=mla, **kw).view(H, -1, D)
    at = 0
    for b, n in enumerate(lens):
        some = [i for i in range(n) if seen[at + i] or ctx[b]]
        none = [at + i for i in range(n) if not seen[at + i] and not ctx[b]]
        for h in range(H):
            j = 0 if mla else h
            _close(got[h, [at + i for i in some]], q[b, h, some], k[b, j, :n], v[b, j, :n], [seen[at + i] for i in some],
                   D**-0.5, rows[b][0][j], rows[b][1][j], DT[dtype])
        assert not got[:, none].any()
        at += n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_values_that_are_not_finite(dtype, value, device):
    """Token 3 holds NaN or an infinity in K or V: the rows that do not see it are as without it,
    those that see it are not finite.  So is padding behind a sequence."""
    lens, N, H, D = [40, 7], 44, 2, 64
    parents = [-1 if i < 4 else i - 4 for n in lens for i in range(n)]  # four chains

    def run(spoil):
        r = torch.Generator().manual_seed(8)
        q, k, v = (torch.randn((2, H, N, D), generator=r).to(DT[dtype]).to(device) for _ in range(3))
        spoil(k, v)
        meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
        tree = build_tree_metadata(torch.tensor(parents, device=device), meta)
        cache, _, _ = _context("packed", [30, 3], H, D, False, DT[dtype], device, 1)
        return unpack_from_kernel(flash_attn_mlm_tree(q, k, v, H, meta, tree, 0.125, cache, 0), meta, H)

    clean = run(lambda k, v: None)
    rows = torch.zeros((2, N), dtype=torch.bool, device=device)
    rows[0, 3:40:4] = rows[1, 3] = True

    def pad(k, v):
        for b, n in enumerate(lens):
            k[b, :, n:] = value
            v[b, :, n:] = value

    assert torch.equal(run(pad), clean)
    for what in ("k", "v"):
        def spoil(k, v):
            (k if what == "k" else v)[:, :, 3, 5] = value

        got = run(spoil)
        for h in range(H):
            assert torch.equal(got[:, h][~rows], clean[:, h][~rows])
            if what == "v":
                assert not got[:, h][rows][:, 5].isfinite().any()
                keep = [d for d in range(D) if d != 5]
                torch.testing.assert_close(got[:, h][rows][:, keep], clean[:, h][rows][:, keep], rtol=4 * torch.finfo(
                    DT[dtype]).eps, atol=4 * torch.finfo(DT[dtype]).eps)
            elif value != value:
                assert got[:, h][rows].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("D, mla, ctx", [(512, True, [300, 0]), (512, True, [0, 4000]), (128, True, [70, 3]),
                                         (256, False, [2100, 64])])
def test_wide_rows_that_are_not_finite(dtype, value, D, mla, ctx, device):
    """As above at the widths that other kernels or tiles take; MLA rows are key and value at once."""
    lens, N, H = [70, 7], 75, 2
    parents = [-1 if i < 4 else i - 4 for n in lens for i in range(n)]  # four chains

    def run(spoil):
        r = torch.Generator().manual_seed(9)
        q, k, v = (torch.randn((2, H, N, D), generator=r).to(DT[dtype]).to(device) for _ in range(3))
        v = k if mla else v
        spoil(k, v)
        meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
        tree = build_tree_metadata(torch.tensor(parents, device=device), meta)
        cache, _, _ = _context("packed", ctx, H, D, mla, DT[dtype], device, 1)
        return unpack_from_kernel(
            flash_attn_mlm_tree(q, k, v, H, meta, tree, D**-0.5, cache, 0, is_mla=mla), meta, H)

    clean = run(lambda k, v: None)
    assert clean.isfinite().all()

    def pad(k, v):
        for b, n in enumerate(lens):
            k[b, :, n:] = value
            v[b, :, n:] = value

    assert torch.equal(run(pad), clean)
    for token in (3, 66):  # of the first and of a later key tile
        rows = torch.zeros((2, N), dtype=torch.bool, device=device)
        rows[0, token:70:4] = True
        rows[1, token:7:4] = True

        def spoil(k, v):
            v[:, :, token, 5] = value

        got = run(spoil)
        for h in range(H):
            assert torch.equal(got[:, h][~rows], clean[:, h][~rows])
            assert not got[:, h][rows][:, 5].isfinite().any()


@pytest.mark.gpu
def test_chain_of_one_is_the_ordinary_call(device):
    """One token a sequence sees its context and itself, as in flash_attn_mlm_compressed."""
    _run(device, torch.bfloat16, lens=[1] * 9, N=1, H=4, D=128, ctx=[700] * 9, kind="paged", seed=9)


@pytest.mark.gpu
def test_refusals(device):
    q = torch.zeros((1, 2, 3, 64), dtype=torch.bfloat16, device=device)
    meta = build_pack_metadata(torch.tensor([3], device=device), 3, 32)
    tree = build_tree_metadata(torch.tensor([-1, 0, 0], device=device), meta)
    with pytest.raises(ValueError, match="same dtype"):
        flash_attn_mlm_tree(q, q.float(), q, 2, meta, tree, 1.0)
    with pytest.raises(ValueError, match="layer_id|inference_cache"):
        flash_attn_mlm_tree(q, q, q, 2, meta, tree, 1.0, InferenceCache())
    with pytest.raises(ValueError, match="HEAD_DIM"):
        x = torch.zeros((1, 2, 3, 48), device=device)
        flash_attn_mlm_tree(x, x, x, 2, meta, tree, 1.0)
    empty = build_pack_metadata(torch.tensor([0], device=device), 3, 32)
    none = build_tree_metadata(torch.zeros(0, dtype=torch.int32, device=device), empty)
    assert flash_attn_mlm_tree(q, q, q, 2, empty, none, 1.0).shape == (0, 64)


@pytest.mark.gpu
def test_repeated_calls_streams_and_graphs(device):
    """The memoised second call, another layout, another stream, two captured graphs replayed in
    turn with eager work between: all the bits of the first call."""
    H, D, N, lens = 4, 64, 24, [24, 5, 11]
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn((3, H, N, D), generator=g).bfloat16().to(device) for _ in range(3))
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    trees = [build_tree_metadata(torch.tensor(_random_parents(random.Random(s), lens), device=device), meta)
             for s in range(2)]
    cache, _, _ = _context("paged", [900, 2000, 64], H, D, False, torch.bfloat16, device, 2)

    def call(t, q=q):
        return flash_attn_mlm_tree(q, k, v, H, meta, t, 0.125, cache, 0)

    want = [call(t).clone() for t in trees]
    assert not torch.equal(*want)
    assert torch.equal(call(trees[0]), want[0])
    strided = torch.empty((3, N, H, D), dtype=q.dtype, device=device).transpose(1, 2).copy_(q)
    assert torch.equal(call(trees[0], strided), want[0])
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=device)[1:].view(q.shape).copy_(q)
    assert torch.equal(call(trees[0], odd), want[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(trees[1])
    side.synchronize()
    assert torch.equal(other, want[1])
    graphs, outs = [], []
    for t in trees:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(t))
        graphs.append(graph)
    for _ in range(3):
        for i in (0, 1):
            outs[i].fill_(7)
            graphs[i].replay()
            call(trees[1 - i])
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i])


@pytest.mark.gpu
@pytest.mark.parametrize("H, D, mla, P", [(2, 128, False, 262200), (4, 512, True, 131100)])
def test_contexts_past_32_bits(H, D, mla, P, device):
    """Pages at the ends of a pool of more than 2^32 elements: the bits of a small pool's."""
    hk, N, lens, ctx = 1 if mla else H, 6, [6, 2], [150, 64]
    g = torch.Generator().manual_seed(7)
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    tree = build_tree_metadata(torch.tensor([-1, 0, 0, 1, 1, 2, -1, 0], device=device), meta)
    q, k, v = (torch.randn((2, H, N, D), generator=g).bfloat16().to(device) for _ in range(3))
    small = [torch.randn((hk, 4, PAGE, D), generator=g).bfloat16().to(device) for _ in range(1 if mla else 2)]
    outs = []
    for far in (False, True):
        pages = [P - 1, 0, P - 2, P - 3] if far else [0, 1, 2, 3]
        pools = small
        if far:
            pools = [torch.empty((hk, P, PAGE, D), dtype=torch.bfloat16, device=device) for _ in small]
            assert pools[0].numel() > 2**32
            for big, x in zip(pools, small):
                big[:, pages] = x
        table = torch.tensor([pages[:3], [pages[3], -1, -1]], dtype=torch.int32, device=device)
        cache = InferenceCache()
        cache.prefill_paged_kv_cache(0, k_pages=pools[0], v_pages=None if mla else pools[1], block_table=table,
                                     context_lens=torch.tensor(ctx), is_mla=mla, num_heads=H, head_dim=D)
        outs.append(flash_attn_mlm_tree(q, k, v, H, meta, tree, D**-0.5, cache, 0, is_mla=mla))
    assert torch.isfinite(outs[0]).all() and torch.equal(*outs)


@pytest.mark.gpu
@pytest.mark.parametrize("D, mla", [(64, False), (512, True)])
def test_first_call_of_a_metadata_in_a_graph(D, mla, device):
    """A capture leaves nothing behind on the metadata that only its replays fill: an eager call
    before the first replay, and the replays, give what an eager call gives."""
    H, N, lens = 4, 20, [20, 3]
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn((2, H, N, D), generator=g).bfloat16().to(device) for _ in range(3))
    cache, _, _ = _context("paged", [1500, 70], H, D, mla, torch.bfloat16, device, 4)

    def call(meta, tree):
        return flash_attn_mlm_tree(q, k, v, H, meta, tree, 0.125, cache, 0, is_mla=mla)

    metas = []
    for _ in range(2):
        meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
        metas.append((meta, build_tree_metadata(torch.tensor([-1] + [0] * 19 + [-1, 0, 1], device=device), meta)))
    want = call(*metas[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(*metas[1])
    assert torch.equal(call(*metas[1]), want)
    for _ in range(3):
        out.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(call(*metas[1]), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_speculative_decoding_over_a_paged_cache(dtype, device):
    """The operators as a server uses them: prompts are stored, then drafted trees attend to the
    pages, one branch is accepted and stored.  At every step the accepted branch's rows are what
    attention over the whole accepted text gives them at 64 bits."""
    dt, H, D, B, N = DT[dtype], 4, 64, 3, 12
    r, g = random.Random(0), torch.Generator().manual_seed(0)
    P, width = 20, 4
    pools = [torch.full((H, P, PAGE, D), float("nan"), dtype=dt, device=device) for _ in range(2)]
    free = torch.randperm(P, generator=g).to(torch.int32).to(device)
    cos, sin = (f(torch.arange(300)[:, None] * 100.0 ** (-torch.arange(32) / 32)).float().to(device)
                for f in (torch.cos, torch.sin))
    lens = torch.zeros(B, dtype=torch.int32, device=device)
    table = torch.full((B, width), -1, dtype=torch.int32, device=device)
    cache = InferenceCache()
    cache.prefill_paged_kv_cache(0, k_pages=pools[0], v_pages=pools[1], block_table=table, context_lens=lens,
                                 is_mla=False, num_heads=H, head_dim=D)
    text = [[torch.zeros((H, 0, D), device=device, dtype=dt) for _ in range(2)] for _ in range(B)]  # stored k, v

    for step in range(6):
        n_new = [r.randint(40, 100) for _ in range(B)] if step == 0 else [r.randint(1, N) for _ in range(B)]
        n = max(n_new)
        meta = build_pack_metadata(torch.tensor(n_new, device=device), n, 32)
        q, k, v = (torch.randn((B, H, n, D), generator=g).to(dt).to(device) for _ in range(3))
        parents = [i - 1 for m in n_new for i in range(m)] if step == 0 else _random_parents(r, n_new)
        tree = build_tree_metadata(torch.tensor(parents, device=device), meta, context_lens=lens)
        q, k = qk_norm_rope(q, k, cos=cos, sin=sin, positions=tree.positions, q_meta=meta)
        out = flash_attn_mlm_tree(q, k, v, H, meta, tree, 0.125, cache, 0).view(H, -1, D)
        seen = ref.ancestors(parents, n_new)
        keep, at = [], 0
        for b, m in enumerate(n_new):  # accept the branch that ends in a token drawn at random
            branch = sorted(seen[at + (m - 1 if step == 0 else r.randrange(m))])
            keep += [i in branch for i in range(m)]
            idx = torch.tensor(branch, device=device)
            kb, vb = (torch.cat([old, x[b, :, idx]], 1) for old, x in zip(text[b], (k, v)))
            for h in range(H):
                c = text[b][0].shape[1]
                _close(out[h, at + idx], q[b, h, idx], kb[h, c:], vb[h, c:], [set(range(i + 1)) for i in range(len(branch))],
                       0.125, kb[h, :c], vb[h, :c], dt)
            text[b] = [kb, vb]
            at += m
        plan = build_block_table(meta, lens, free_pages=free, block_table=table,
                                 keep=torch.tensor(keep, device=device))
        cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan)
        lens, table, free = plan.context_lens, plan.block_table, free[plan.pages_taken :]
        assert lens.tolist() == [t[0].shape[1] for t in text]
        for b in range(B):  # the pages hold the text
            rows = torch.arange(int(lens[b]), device=device)
            slot = table[b].long()[rows // PAGE] * PAGE + rows % PAGE
            for pool, t in zip(pools, text[b]):
                assert torch.equal(pool.view(H, -1, D)[:, slot], t)


def test_schedules_do_not_depend_on_contexts():
    """A schedule serves calls over other contexts (one metadata, several layers): its size, so the
    rows a unit of it stands for, follows from what its key holds.  The context's share in the
    choice of a tile is advice, which the caller puts into tile_config."""
    lib = _lib.load()
    p = _lib.AttnParams()
    p.flags = _lib.FLAG_TREE | _lib.FLAG_NOSPLIT
    p.cu_seqlens_q = p.cu_seqlens_kv = p.q = p.k = p.v = p.o = p.k_ctx = p.v_ctx = 256
    for dtype in (_lib.DTYPE_BF16, _lib.DTYPE_F16, _lib.DTYPE_F32):
        for d in (16, 32, 64, 128, 256):
            for B, H, n in ((8, 8, 100), (1, 16, 256), (3, 2, 9)):
                p.dtype, p.D, p.B, p.H, p.N, p.total_q, p.tile_config = dtype, d, B, H, n, B * n, 0
                sizes, advice = set(), set()
                for paged in (False, True) if dtype != _lib.DTYPE_F32 else (False,):
                    for pages in (1, 20, 33, 500):
                        p.ctx_batch, p.ctx_rows, p.ctx_block_table, p.ctx_pages_per_batch = B, B * pages * PAGE, None, 0
                        if paged:
                            p.ctx_rows, p.ctx_block_table, p.ctx_pages_per_batch = B * pages, 256, pages
                            p.ctx_page_stride = PAGE * d
                        sizes.add(lib.fmlm_attn_workspace_bytes(p))
                        advice.add((pages >= 32, lib.fmlm_attn_tree_tile(p)))
                assert len(sizes) == 1, (dtype, d, B, H, n)
                wide = dtype != _lib.DTYPE_F32 and d == 256
                if (B, H, n) == (8, 8, 100) and wide:
                    assert advice == {(False, 1), (True, 2)}
                else:
                    assert {x for _, x in advice} == {1 if wide else 0}
    p.dtype, p.D, p.tile_config = _lib.DTYPE_BF16, 256, 2
    assert lib.fmlm_attn_tree_tile(p) == 2  # the caller's own
    p.flags = 0
    assert lib.fmlm_attn_tree_tile(p) == -1 and lib.fmlm_attn_tree_tile(None) == -1  # tree calls


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["paged", "packed"])
@pytest.mark.parametrize("order", [(33, 20), (20, 33), (33, 20, 33, 1)])
def test_layers_of_one_metadata_with_other_contexts(kind, order, device):
    """D = 256: layers whose contexts ask for 64- and for 128-row workgroups, one metadata"""
    H, D, lens, N = 8, 256, [100] * 8, 100
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    parents = _random_parents(random.Random(1), lens)
    tree = build_tree_metadata(torch.tensor(parents, device=device), meta)
    seen = ref.ancestors(parents, lens)
    layers = []
    for i, pages in enumerate(order):
        g = torch.Generator().manual_seed(i)
        q, k, v = (torch.randn((8, H, N, D), generator=g).bfloat16().to(device) for _ in range(3))
        layers.append((q, k, v, *_context(kind, [pages * PAGE - b for b in range(8)], H, D, False, torch.bfloat16, device, i)))
    for _ in range(2):  # the second time by the memos of the first
        for q, k, v, cache, rows, _ in layers:
            poison = torch.full((H * sum(lens), D), float("nan"), dtype=torch.bfloat16, device=device)
            del poison  # rows that no workgroup writes
            got = flash_attn_mlm_tree(q, k, v, H, meta, tree, D**-0.5, cache, 0).view(H, -1, D)
            for b in (0, 5):
                part = slice(100 * b, 100 * b + 100)
                for h in (0, 7):
                    _close(got[h, part], q[b, h], k[b, h], v[b, h], seen[part], D**-0.5, rows[b][0][h], rows[b][1][h],
                           torch.bfloat16)
            assert bool(got.isfinite().all())


@pytest.mark.gpu
def test_refusals_after_legal_calls(device):
    """A wrong call is refused whatever ran before it."""
    meta = build_pack_metadata(torch.tensor([3, 1], device=device), 3, 32)
    tree = build_tree_metadata(torch.tensor([-1, 0, 0, -1], device=device), meta)
    q = torch.randn((2, 2, 3, 64), device=device).bfloat16()
    cache, _, _ = _context("packed", [5, 70], 2, 64, False, torch.bfloat16, device)
    for _ in range(2):
        flash_attn_mlm_tree(q, q, q, 2, meta, tree, 1.0)
        flash_attn_mlm_tree(q, q, q, 2, meta, tree, 1.0, cache, "no such layer")
        flash_attn_mlm_tree(q, q, q, 2, meta, tree, 1.0, cache, 0)
        for args in ((None, 0), (cache, None)):
            with pytest.raises(ValueError, match="provided together"):
                flash_attn_mlm_tree(q, q, q, 2, meta, tree, 1.0, *args)
        with pytest.raises(ValueError, match="num_heads"):
            flash_attn_mlm_tree(q, q, q, 1, meta, tree, 1.0)
        with pytest.raises(ValueError, match="tree.mask"):
            flash_attn_mlm_tree(q, q, q, 2, meta, TreeMetadata(tree.mask[:3], None), 1.0)
        with pytest.raises(ValueError, match="no backward"):
            flash_attn_mlm_tree(q.clone().requires_grad_(), q, q, 2, meta, tree, 1.0)


def test_refuses_tangents():
    from torch.autograd import forward_ad as fw

    meta = _cpu_meta([2, 1], 2)
    tree = TreeMetadata(torch.zeros((3, 1), dtype=torch.int64), torch.zeros(3, dtype=torch.int32))
    with fw.dual_level():
        args = [torch.zeros((2, 2, 2, 64), dtype=torch.float16) for _ in range(3)]
        for i in range(3):
            some = list(args)
            some[i] = fw.make_dual(args[i], args[i])
            with pytest.raises(ValueError, match="forward-mode"):
                flash_attn_mlm_tree(*some, 2, meta, tree, 1.0)
        pool = torch.zeros((2, 1, PAGE, 64), dtype=torch.float16)
        cache = InferenceCache()
        cache.prefill_paged_kv_cache(0, k_pages=pool, v_pages=fw.make_dual(pool.clone(), pool), is_mla=False, num_heads=2,
                                     block_table=torch.zeros((2, 1), dtype=torch.int32), head_dim=64,
                                     context_lens=torch.zeros(2, dtype=torch.int32))
        with pytest.raises(ValueError, match="forward-mode"):
            flash_attn_mlm_tree(*args, 2, meta, tree, 1.0, cache, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, kind, D, mla", [("bf16", "paged", 64, False), ("fp16", "packed", 512, True),
                                                 ("fp32", "packed", 64, False)])
@pytest.mark.parametrize("first", [[40, 1, 23], [23, 40, 1]])
def test_metadata_whose_fields_were_replaced(first, dtype, kind, D, mla, device):
    """Parameter blocks and schedules kept on a metadata are those of its index tensors: other offsets
    (as many tokens), other integer types, and the first offsets again"""
    import dataclasses

    from flash_mlm import flash_attn_mlm_compressed

    H, N, ctx = 3, 40, [3000, 70, 200]
    second = first[1:] + first[:1]
    g = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn((3, H, N, D), generator=g).to(DT[dtype]).to(device) for _ in range(3))
    v = k if mla else v
    cache, _, _ = _context(kind, ctx, H, D, mla, DT[dtype], device, 2)

    def calls(meta, tree):
        return (flash_attn_mlm_tree(q, k, v, H, meta, tree, D**-0.5, cache, 0, is_mla=mla),
                flash_attn_mlm_compressed(q, k, v, H, meta, D**-0.5, cache, 0, is_mla=mla))

    fresh = [build_pack_metadata(torch.tensor(lens, device=device), N, 32) for lens in (first, second)]
    trees = [build_tree_metadata(torch.tensor([i - 1 for n in lens for i in range(n)], device=device), m)
             for lens, m in zip((first, second), fresh)]
    want = [[x.clone() for x in calls(m, t)] for m, t in zip(fresh, trees)]
    assert not torch.equal(want[0][0], want[1][0])
    meta = build_pack_metadata(torch.tensor(first, device=device), N, 32)
    shared = dataclasses.replace(meta, cu_seqlens=fresh[1].cu_seqlens, token_indices=fresh[1].token_indices)

    def put(i, cast=lambda t: t):
        for f in ("lengths", "cu_seqlens", "token_indices", "batch_ids_q", "q_tile_starts_q"):
            setattr(meta, f, cast(getattr(fresh[i], f)))

    for i in (0, 0, 1, 1, 0, 1):
        put(i)
        for a, b in zip(calls(meta, trees[i]), want[i]):
            assert torch.equal(a, b)
        for a, b in zip(calls(shared, trees[1]), want[1]):  # a copy that shares what is kept
            assert torch.equal(a, b)
    put(0, lambda t: t.long())
    for _ in range(2):
        for a, b in zip(calls(meta, trees[0]), want[0]):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("D, mla, kind", [(64, False, "paged"), (512, True, "packed"), (64, False, "none")])
@pytest.mark.parametrize("wide", [False, True])
def test_first_calls_of_a_metadata_on_two_streams(D, mla, kind, wide, device):
    """The schedule, and offsets that a call derives (``wide``: of int64 metadata), are made on the first
    call's stream; calls on other streams wait for them, by the memo (layer 0) or without (layer 1)."""
    from flash_mlm import flash_attn_mlm_compressed

    H, N, lens = 4, 20, [20, 3]
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn((2, H, N, D), generator=g).bfloat16().to(device) for _ in range(3))
    v = k if mla else v
    caches = [_context(kind, c, H, D, mla, torch.bfloat16, device, 4)[0] for c in ([1500, 70], [64, 3000])]
    cast = torch.Tensor.long if wide else lambda t: t
    parents = torch.tensor([-1] + [0] * 19 + [-1, 0, 1], device=device)

    def fresh():
        meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
        meta.cu_seqlens = cast(meta.cu_seqlens)
        return meta, build_tree_metadata(parents, meta)

    def calls(meta, tree, i):
        args = (caches[i], None if caches[i] is None else 0)
        return (flash_attn_mlm_tree(q, k, v, H, meta, tree, 0.125, *args, is_mla=mla),
                flash_attn_mlm_compressed(q, k, v, H, meta, 0.125, *args, is_mla=mla))

    meta, tree = fresh()  # (layer 0's contexts steer where both layers' key ranges are split)
    want = [calls(meta, tree, i) for i in range(2)]
    busy = torch.randn((8192, 8192), device=device)
    for _ in range(3):
        meta, tree = fresh()
        streams = [torch.cuda.Stream() for _ in range(3)]
        torch.cuda.synchronize()
        got, done = [], torch.cuda.Event()
        with torch.cuda.stream(streams[0]):
            for _ in range(4):
                torch.mm(busy, busy)
            done.record()
            got.append((0, calls(meta, tree, 0)))
        for s in streams[1:]:
            with torch.cuda.stream(s):
                got += [(i, calls(meta, tree, i)) for i in (0, 1, 0)]
        overlapped = not done.query()
        torch.cuda.synchronize()
        assert overlapped  # the first stream was still busy when the last call was made
        for i, outs in got:
            for a, b in zip(outs, want[i]):
                assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, D, kind", [("bf16", 64, "paged"), ("fp16", 128, "packed"), ("bf16", 256, "paged"),
                                            ("fp32", 64, "packed"), ("fp32", 128, "packed"), ("bf16", 512, "paged")])
def test_rows_that_see_nothing_in_a_split_call(dtype, D, kind, device):
    """A schedule cuts sequence 0 for one layer's long context; in the next layer that context is empty, and
    rows whose masks are empty too are zero, as unsplit rows are."""
    H, N, lens, mla = 2, 70, [70, 5], D == 512
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    r = random.Random(D)
    seen = [set() if i % 3 == 0 else {j for j in range(n) if r.random() < 0.2} - ({i} if i % 2 else set())
            for n in lens for i in range(n)]
    tree = TreeMetadata(torch.from_numpy(ref.mask_words(seen, 2)).to(device), None)
    g = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn((2, H, N, D), generator=g).to(DT[dtype]).to(device) for _ in range(3))
    v = k if mla else v
    for ctx in ([9000, 100], [0, 9000], [9000, 0]):
        cache, rows, _ = _context(kind, ctx, H, D, mla, DT[dtype], device, 3)
        for _ in range(2):
            got = flash_attn_mlm_tree(q, k, v, H, meta, tree, D**-0.5, cache, 0, is_mla=mla).view(H, -1, D)
            at = 0
            for b, n in enumerate(lens):
                some = [i for i in range(n) if seen[at + i] or ctx[b]]
                none = [at + i for i in range(n) if not seen[at + i] and not ctx[b]]
                for h in range(H):
                    j = 0 if mla else h
                    _close(got[h, [at + i for i in some]], q[b, h, some], k[b, j, :n], v[b, j, :n],
                           [seen[at + i] for i in some], D**-0.5, rows[b][0][j], rows[b][1][j], DT[dtype])
                assert not got[:, none].any()
                at += n
    # the first layer's schedule was a split one
    (sched,) = meta.kernel_schedules.values()
    assert int(sched[:8].view(torch.int32)[1]) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D, mla, ctx", [(64, False, [300, 3000]), (128, False, [65, 0]), (256, False, [900, 64]),
                                         (512, True, [300, 3000])])
def test_the_context_part_is_not_rounded(dtype, D, mla, ctx, device, monkeypatch):
    """As the tolerances above, without a rounding of the context's part (h of it): the parts of a row meet
    in fp32 in every kernel."""
    def close(got, q, k, v, seen, scale, kc, vc, dt):
        o, w, _, s = ref.tree_attention(_f(q), _f(k), _f(v), seen, scale, _f(kc), _f(vc))
        h, keys = torch.finfo(dt).eps / 2, kc.shape[0] + k.shape[0]
        bound = h * np.abs(o) + (2 * h + 2 * (D + 16) * U * s[:, None] + (keys + 64) * U) * w
        if dt == torch.float16:
            bound = bound + 2.0**-25 * (keys * np.abs(np.concatenate([_f(vc), _f(v)])).max() + 1)
        # (1.01: the products of the terms above with each other, each below 1 / 100 of them)
        assert np.all(np.abs(_f(got) - o) <= bound * 1.01)

    monkeypatch.setitem(_run.__globals__, "_close", close)
    _run(device, DT[dtype], lens=[30, 12], N=30, H=3, D=D, ctx=ctx, kind="packed", mla=mla, seed=D)
