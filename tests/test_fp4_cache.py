"""Paged contexts in 4 bits and appends that rotate: the oracle and refusals (CPU), and on the GPU
codes, scales and rotated rows bit for bit against the 64-bit restatement
(oracle/window_ref.py)."""

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
    build_tree_metadata,
    flash_attn_mlm,
    flash_attn_mlm_compressed,
    flash_attn_mlm_precompressed,
    flash_attn_mlm_tree,
    flash_attn_mlm_window,
)
from oracle import window_ref as ref

PAGE = 64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _meta(lens, N, device):
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=device)
    tok = torch.tensor([b * N + p for b, n in enumerate(lens) for p in range(n)], dtype=torch.int64, device=device)
    return PackMetadata(B=len(lens), N=N, lengths=torch.tensor(lens, dtype=torch.int32, device=device), cu_seqlens=cu,
                        token_indices=tok, total_tokens=sum(lens), batch_ids_block_n=32, batch_ids_q=cu, q_tile_starts_q=cu)


def _fp4_pools(H, P, D, device="cpu", fill=0):
    make = lambda cols: torch.full((H, P, PAGE, cols), fill, dtype=torch.uint8, device=device)  # noqa: E731
    return dict(k_pages=make(D // 2), k_scales=make(D // 32), v_pages=make(D // 2), v_scales=make(D // 32))


def _fp4_cache(H, P, D, dtype, B=1, width=1, device="cpu", fill=0):
    cache = InferenceCache()
    pools = _fp4_pools(H, P, D, device, fill)
    cache.prefill_paged_fp4_cache(0, **pools, block_table=torch.zeros((B, width), dtype=torch.int32),
                                  context_lens=torch.zeros(B, dtype=torch.int32), num_heads=H, head_dim=D, dtype=dtype)
    return cache, pools


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------
def test_oracle_codes_by_hand():
    x = np.zeros((1, 32))
    x[0, :10] = [6, -0.25, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -6.9]
    codes, scales = ref.fp4_encode(x, "bf16")
    assert scales.tolist() == [[127]]  # 6.9 < 7 * 2^0
    got = ref.fp4_values(codes, scales)[0, :10]
    # halfway goes to the even code: 0.25 -> 0, 0.75 -> 1, 1.25 -> 1, 1.75 -> 2, 2.5 -> 2, 3.5 -> 4, 5 -> 4
    assert got.tolist() == [6, 0, 0, 1, 1, 2, 2, 4, 4, -6]
    assert np.signbit(got[1])
    x[0, 0] = 7.0
    assert ref.fp4_encode(x, "bf16")[1].tolist() == [[128]]
    x[0, 0] = np.inf
    assert ref.fp4_encode(x, "fp16")[1].tolist() == [[127 + 13]]
    assert ref.fp4_encode(x, "bf16")[1].tolist() == [[127 + 125]]
    assert ref.fp4_encode(np.zeros((1, 32)), "fp16")[1].tolist() == [[127 - 23]]
    assert ref.fp4_values(*ref.fp4_encode(np.full((1, 32), np.nan), "bf16")).tolist() == [[0.0] * 32]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_oracle_codes_are_nearest(dtype):
    """No value is further from its code than half the gap around it, and the scale is the smallest
    that keeps the largest within the codes."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((200, 64)) * 2.0 ** rng.integers(-9, 9, (200, 1))
    codes, scales = ref.fp4_encode(x, dtype)
    y = ref.fp4_values(codes, scales)
    s = np.repeat(2.0 ** (scales.astype(float) - 127), 32, -1)
    gap = np.where(np.abs(x) / s < 2, 0.5, np.where(np.abs(x) / s < 4, 1.0, 2.0))
    assert (np.abs(x - y) <= s * gap / 2).all()
    top = np.abs(x).reshape(200, 2, 32).max(-1) / 2.0 ** (scales.astype(float) - 127)
    assert (top < 7).all() and (top >= 3.5).all()


def test_oracle_rotation_keeps_lengths_and_differences():
    rng = np.random.default_rng(5)
    for inter in (False, True):
        x, y = rng.standard_normal((2, 7, 32))
        ang = np.arange(7)[:, None] * 10.0 ** -np.arange(8)
        a = ref.rotate(x, np.cos(ang), np.sin(ang), inter)
        assert np.allclose((a**2).sum(-1), (x**2).sum(-1)) and (a[:, 16:] == x[:, 16:]).all()
        # products depend on differences of positions alone
        b = ref.rotate(y, np.cos(ang), np.sin(ang), inter)
        s = lambda u, d: ref.rotate(u, np.cos(ang + d), np.sin(ang + d), inter)  # noqa: E731
        d = 0.37 * 10.0 ** -np.arange(8)
        assert np.allclose((a * b).sum(-1), (s(x, d) * s(y, d)).sum(-1))


def test_pool_refusals():
    pools = _fp4_pools(2, 3, 64)
    args = dict(block_table=torch.zeros((1, 3), dtype=torch.int32), context_lens=torch.zeros(1, dtype=torch.int32),
                num_heads=2, head_dim=64, dtype=torch.bfloat16)
    InferenceCache().prefill_paged_fp4_cache(0, **pools, **args)
    for match, kw in [
        ("bf16 or fp16", dict(dtype=torch.float32)),
        ("head_dim 32, 64", dict(head_dim=16)),
        ("head_dim 32, 64", dict(head_dim=512)),
        ("k_pages must be uint8", dict(k_pages=pools["k_pages"].to(torch.int32))),
        ("k_pages must be uint8", dict(k_pages=pools["k_pages"][0])),
        ("v_pages must be uint8", dict(v_pages=pools["v_pages"][:, :2])),
        ("k_scales must be uint8", dict(k_scales=pools["v_pages"])),
        ("v_scales must be contiguous", dict(v_scales=torch.zeros((2, 3, PAGE, 4), dtype=torch.uint8)[..., :2])),
        ("block_table must be", dict(block_table=torch.zeros(3, dtype=torch.int32))),
        ("context_lens must lie", dict(context_lens=torch.tensor([193]))),
        ("context_lens must have", dict(context_lens=torch.zeros(2, dtype=torch.int32))),
        ("num_heads", dict(num_heads=0)),
    ]:
        with pytest.raises(ValueError, match=match):
            InferenceCache().prefill_paged_fp4_cache(0, **{**pools, **args, **kw})


def test_values_refusals():
    cache, _ = _fp4_cache(2, 3, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="no cached KV entry"):
        cache.paged_kv_values(1)
    with pytest.raises(ValueError, match="no CPU compute path"):
        cache.paged_kv_values(0)
    cache.prefill_kv_cache(1, k_cache=torch.zeros((4, 16)), v_cache=torch.zeros((4, 16)), total_context_len=2,
                           context_batch_size=1, is_mla=False, num_heads=2, head_dim=16)
    with pytest.raises(ValueError, match="requires a paged entry"):
        cache.paged_kv_values(1)


def test_other_entry_points_refuse_four_bits():
    cache, _ = _fp4_cache(2, 3, 64, torch.bfloat16)
    q = torch.zeros((1, 2, 4, 64), dtype=torch.bfloat16)
    meta = _meta([4], 4, "cpu")
    match = "a 4-bit context serves"
    with pytest.raises(ValueError, match=match):
        flash_attn_mlm(q, q, q, 1.0, cache, 0)
    flat = q.view(8, 64)
    with pytest.raises(ValueError, match=match):
        flash_attn_mlm_precompressed(flat, flat, flat, 2, 4, meta.cu_seqlens, meta.cu_seqlens, meta.cu_seqlens, 1.0, cache, 0)

    class Tree:
        mask = torch.zeros((4, 1), dtype=torch.int64)

    with pytest.raises(ValueError, match=match):
        flash_attn_mlm_tree(q, q, q, 2, meta, Tree(), 1.0, cache, 0)
    for kw in (dict(is_mla=True), dict(causal_query_seq_attn=True)):
        with pytest.raises(ValueError, match="neither MLA nor"):
            flash_attn_mlm_compressed(q, q, q, 2, meta, 1.0, cache, 0, **kw)
    with pytest.raises(ValueError, match="context_batch_size"):
        flash_attn_mlm_compressed(q, q, q, 2, meta, 1.0, cache, 0, context_batch_size=3)
    with pytest.raises(ValueError, match="different block_n"):
        flash_attn_mlm_compressed(q, q, q, 2, meta, 1.0, cache, 0, block_n=64)


def _append_args(D=64, H=2, fp4=False, dtype=torch.bfloat16):
    meta = _meta([2, 1], 2, "cpu")
    cache = InferenceCache()
    table = torch.zeros((2, 1), dtype=torch.int32)
    lens = torch.zeros(2, dtype=torch.int32)
    if fp4:
        cache, _ = _fp4_cache(H, 3, D, dtype, B=2)
    else:
        pages = torch.zeros((H, 3, PAGE, D), dtype=dtype)
        cache.prefill_paged_kv_cache(0, k_pages=pages, v_pages=pages.clone(), block_table=table, context_lens=lens,
                                     is_mla=False, num_heads=H, head_dim=D)
    plan = PagedMetadata(table, torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), lens,
                         torch.zeros(3, dtype=torch.int32))
    k = torch.zeros((2, H, 2, D), dtype=dtype)
    cos = torch.zeros((5, D // 2))
    return cache, dict(k=k, v=k, q_meta=meta, plan=plan), cos


@pytest.mark.parametrize("fp4", [False, True])
def test_append_refusals(fp4):
    cache, args, cos = _append_args(fp4=fp4)
    k, plan = args["k"], args["plan"]
    for match, kw in [
        ("need cos", dict(q=k)),
        ("need cos", dict(sin=cos)),
        ("need cos", dict(positions=plan.positions)),
        ("need cos", dict(interleaved=True)),
        ("dtype/device must match", dict(k=k.float())),
    ]:
        with pytest.raises(ValueError, match=match):
            cache.append_paged_kv_cache(0, **{**args, **kw})
    with pytest.raises(ValueError, match="no CPU compute path"):  # checked before anything else of the call
        cache.append_paged_kv_cache(0, **args, cos=cos, sin=cos)
    for kw in (dict(positions=[0, 1, 0]), dict(sin=cos.numpy()), dict(q=k.tolist())):
        with pytest.raises(ValueError, match="must be tensors"):
            cache.append_paged_kv_cache(0, **{**args, "cos": cos, "sin": cos, **kw})


@pytest.mark.parametrize("fp4", [False, True])
def test_gradients_and_tangents_of_the_rotated_q_are_refused(fp4):
    """Those of q and of the tables it is rotated by: the returned q would drop them without a word."""
    import torch.autograd.forward_ad as fwd

    cache, args, cos = _append_args(fp4=fp4)
    args.update(q=args["k"], cos=cos, sin=cos)
    for name in ("q", "cos", "sin"):
        with pytest.raises(ValueError, match="the rotated q has no gradient"):
            cache.append_paged_kv_cache(0, **{**args, name: args[name].clone().requires_grad_()})
        with torch.no_grad(), pytest.raises(ValueError, match="no CPU compute path"):
            cache.append_paged_kv_cache(0, **{**args, name: args[name].clone().requires_grad_()})
        with fwd.dual_level(), pytest.raises(ValueError, match="no forward-mode"):
            cache.append_paged_kv_cache(0, **{**args, name: fwd.make_dual(args[name], torch.ones_like(args[name]))})


def test_rotating_append_checks():
    """What paged._tables refuses, without a GPU."""
    from flash_mlm.host.paged import _tables

    cos, pos = torch.zeros((5, 32)), torch.zeros(3, dtype=torch.int32)
    dev = torch.device("cpu")
    ok = dict(d=64, t=3, dev=dev)
    _tables(cos, cos, pos, **ok)
    for match, a in [
        ("come together", (cos, None, pos)),
        ("fp32 tables", (cos.half(), cos.half(), pos)),
        ("fp32 tables", (cos, cos[:4], pos)),
        ("fp32 tables", (cos[0], cos[0], pos)),
        ("multiple of 16", (cos[:, :4], cos[:, :4], pos)),
        ("multiple of 16", (torch.zeros((5, 40)), torch.zeros((5, 40)), pos)),
        ("at least one position", (cos[:0], cos[:0], pos)),
        ("the plan has none", (cos, cos, None)),
        ("one entry per packed token", (cos, cos, pos[:2])),
        ("one entry per packed token", (cos, cos, pos.float())),
    ]:
        with pytest.raises(ValueError, match=match):
            _tables(*a, **ok)


def test_mla_latents_are_not_rotated():
    cache = InferenceCache()
    pages = torch.zeros((1, 3, PAGE, 64), dtype=torch.float16)
    cache.prefill_paged_kv_cache(0, k_pages=pages, block_table=torch.zeros((2, 1), dtype=torch.int32),
                                 context_lens=torch.zeros(2, dtype=torch.int32), is_mla=True, num_heads=2, head_dim=64)
    _, args, cos = _append_args()
    with pytest.raises(ValueError, match="MLA latents"):
        cache.append_paged_kv_cache(0, **args, cos=cos, sin=cos)


def test_argument_rejection_without_launch():
    lib = _lib.load()
    p = _lib.AppendParams()
    assert lib.fmlm_rotate_append(None, None) == -1
    p.dtype, p.D, p.H, p.B, p.N, p.T = _lib.DTYPE_F32, 64, 2, 1, 4, 4
    assert lib.fmlm_rotate_append(p, None) == -2
    p.dtype = _lib.DTYPE_BF16
    p.D = 512
    assert lib.fmlm_rotate_append(p, None) == -3
    p.D, p.flags = 16, _lib.AP_FP4
    assert lib.fmlm_rotate_append(p, None) == -3
    p.D, p.flags, p.rotary_dim = 64, 0, 24
    assert lib.fmlm_rotate_append(p, None) == -1
    p.rotary_dim = 32  # without tables
    assert lib.fmlm_rotate_append(p, None) == -1
    p.rotary_dim = 0
    assert lib.fmlm_rotate_append(p, None) == -1  # padded, without offsets
    p.cu_seqlens = 256
    p.k.dst = 256
    assert lib.fmlm_rotate_append(p, None) == -1  # a pool without slots
    p.slots = 256
    assert lib.fmlm_rotate_append(p, None) == -1  # ... without a source
    p.k.src = 264
    assert lib.fmlm_rotate_append(p, None) == -4
    p.k.src, p.flags = 256, _lib.AP_FP4
    assert lib.fmlm_rotate_append(p, None) == -1  # ... without scales
    p.B = p.N = 1 << 17
    p.flags = 0
    assert lib.fmlm_rotate_append(p, None) == -1  # too many rows
    r = (_lib.Fp4Rows * 2)()
    values = lambda dtype=0, n=1, rows=1, D=64: lib.fmlm_fp4_values(dtype, r, n, rows, D, None)  # noqa: E731
    assert values(dtype=2) == -2 and values(D=48) == -3 and values(rows=-1) == -1 and values(n=3) == -1
    assert values() == -1 and values(rows=0) == 0
    r[0].codes = r[0].scales = r[0].out = 256
    assert values(n=2) == -1
    r[0].out = 264
    assert values() == -4
    assert lib.fmlm_fp4_values(0, None, 1, 1, 64, None) == -1


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------
def _f64(t):
    return t.detach().double().cpu().numpy()


def _case(device, dtype, lens, N, H, D, fp4, packed, seed=0, spread=True):
    """New tokens, a pool of random rows and a plan with shuffled distinct slots."""
    g = torch.Generator(device=device).manual_seed(seed)
    dt, T, B = TYPES[dtype], sum(lens), len(lens)
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)

    def rows():
        x = torch.randn((H * T, D) if packed else (B, H, N, D), generator=g, device=device)
        if spread:  # blocks of very different sizes
            x = x * torch.exp2(torch.randint(-9, 9, x.shape[:-1] + (1,), generator=g, device=device).float())
        return x.to(dt)

    q, k, v = rows(), rows(), rows()
    P = (T + PAGE - 1) // PAGE + 2
    cache = InferenceCache()
    table = torch.zeros((B, 1), dtype=torch.int32, device=device)
    zero = torch.zeros(B, dtype=torch.int32, device=device)
    if fp4:
        pools = {n: torch.randint(0, 256, x.shape, generator=g, device=device, dtype=torch.uint8)
                 for n, x in _fp4_pools(H, P, D).items()}
        for n in ("k_scales", "v_scales"):
            pools[n] = pools[n] % 9 + 120
        cache.prefill_paged_fp4_cache(0, **pools, block_table=table, context_lens=zero, num_heads=H, head_dim=D, dtype=dt)
    else:
        pools = {n: torch.randn((H, P, PAGE, D), generator=g, device=device).to(dt) for n in ("k_pages", "v_pages")}
        cache.prefill_paged_kv_cache(0, **pools, block_table=table, context_lens=zero, is_mla=False, num_heads=H, head_dim=D)
    r = random.Random(seed)
    slots = r.sample(range(P * PAGE), T)
    for i in range(0, T, 5):
        slots[i] = [-1, P * PAGE, -7][i % 3]  # not stored
    plan = PagedMetadata(table, torch.tensor(slots, dtype=torch.int64, device=device),
                         torch.tensor([r.randrange(90) for _ in range(T)], dtype=torch.int32, device=device), zero,
                         torch.zeros(B + 1, dtype=torch.int32, device=device))
    return meta, q, k, v, cache, pools, plan, slots


def _tables(D, R, device, n=90):
    freq = 10000.0 ** (-torch.arange(0, R // 2, dtype=torch.float64) * 2 / R)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * freq
    return ang.cos().float().to(device), ang.sin().float().to(device)


def _tokens(x, lens, H, D):
    """[H, T, D] numpy of padded or packed rows"""
    x = _f64(x)
    if x.ndim == 2:
        return x.reshape(H, -1, D)
    return np.concatenate([x[b, :, :n] for b, n in enumerate(lens)], 1)


def _expect(pools, lens, H, D, k, v, slots, dtype, fp4, turn):
    """What the pools hold after the append"""
    out = {n: x.cpu().numpy().copy() if fp4 else _f64(x) for n, x in pools.items()}
    for name, x in (("k", turn(_tokens(k, lens, H, D))), ("v", _tokens(v, lens, H, D))):
        P = out[name + "_pages"].shape[1]
        if fp4:
            rows = dict(zip((name + "_pages", name + "_scales"), ref.fp4_encode(x, dtype)))
        else:
            # one rounding to the type, ties and all, by torch
            rows = {name + "_pages": _f64(torch.from_numpy(x).to(TYPES[dtype]))}
        for n, y in rows.items():
            flat = out[n].reshape(H, P * PAGE, -1)
            for t, slot in enumerate(slots):
                if 0 <= slot < P * PAGE:
                    flat[:, slot] = y[:, t]
    return out


SHAPES = [  # lens, N, H, D, R, packed
    ([1], 1, 1, 32, 32, False),
    ([0, 1, 3, 0], 3, 5, 64, 32, False),
    ([7, 0, 19], 19, 4, 128, 128, True),
    ([33, 65, 2], 65, 3, 256, 48, False),
    ([5, 6], 9, 7, 64, 64, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rotated_append_into_four_bits_is_exact(device, shape, dtype, interleaved):
    lens, N, H, D, R, packed = shape
    meta, q, k, v, cache, pools, plan, slots = _case(device, dtype, lens, N, H, D, True, packed)
    cos, sin = _tables(D, R, device)
    pos = plan.positions.cpu().numpy()
    turn = lambda x: ref.rotate(x, _f64(cos)[pos], _f64(sin)[pos], interleaved)  # noqa: E731
    want = _expect(pools, lens, H, D, k, v, slots, dtype, True, turn)
    got_q = cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan, q=q, cos=cos, sin=sin, interleaved=interleaved)
    for n, x in want.items():
        assert (pools[n].cpu().numpy() == x).all(), n
    _check_q(got_q, q, turn, lens, H, D, dtype)
    # the values that the codes stand for
    for name, x in zip("kv", cache.paged_kv_values(0)):
        assert (_f64(x) == ref.fp4_values(want[name + "_pages"], want[name + "_scales"])).all()


def _check_q(got, q, turn, lens, H, D, dtype):
    """Rotated in fp32 (two products, one sum: 2 * 2^-24 of the larger products) and rounded once"""
    assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
    want = turn(_tokens(q, lens, H, D))
    top = np.abs(_tokens(q, lens, H, D)).max(-1, keepdims=True)
    tol = np.abs(want) * torch.finfo(TYPES[dtype]).eps / 2 + top * 2.0**-21 + 2.0**-25  # (fp16 below 2^-14: its step)
    assert (np.abs(_tokens(got, lens, H, D) - want) <= tol).all()
    if got.ndim == 4:  # padding rows
        for b, n in enumerate(lens):
            assert not got[b, :, n:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES + [([3, 8], 8, 2, 16, 16, False)], ids=str)
def test_rotated_append_into_sixteen_bits(device, shape, dtype, interleaved):
    lens, N, H, D, R, packed = shape
    meta, q, k, v, cache, pools, plan, slots = _case(device, dtype, lens, N, H, D, False, packed)
    cos, sin = _tables(D, R, device)
    pos = plan.positions.cpu().numpy()
    turn = lambda x: ref.rotate(x, _f64(cos)[pos], _f64(sin)[pos], interleaved)  # noqa: E731
    want = _expect(pools, lens, H, D, k, v, slots, dtype, False, turn)
    got_q = cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan, q=q, cos=cos, sin=sin, interleaved=interleaved)
    assert (_f64(pools["v_pages"]) == want["v_pages"]).all()
    # k: rounded twice (fp32, then the type), so at most a step from the value rounded once
    top = float(np.abs(_tokens(k, lens, H, D)).max(initial=0.0))
    eps = torch.finfo(TYPES[dtype]).eps
    assert (np.abs(_f64(pools["k_pages"]) - want["k_pages"]) <= np.abs(want["k_pages"]) * eps + top * 2.0**-21 + 2.0**-24).all()
    # unstored rows and rows of other pages are untouched: equal to the last bit
    stored = {s for s in slots if s >= 0}
    P = pools["k_pages"].shape[1]
    rest = [i for i in range(P * PAGE) if i not in stored]
    assert (_f64(pools["k_pages"]).reshape(H, -1, D)[:, rest] == want["k_pages"].reshape(H, -1, D)[:, rest]).all()
    _check_q(got_q, q, turn, lens, H, D, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,packed,dtype", [(5, False, "bf16"), (17, False, "fp16"), (20, True, "bf16")])
def test_appends_of_many_rows(device, H, packed, dtype, interleaved, fp4):
    """Calls whose threads take 16 heads each: the bits of appends of a few hundred rows at a time, whose threads take
    four (the tests above are of those), and a sample of them against the oracle"""
    lens, N, D, R = [2900, 0, 2001, 700], 2900, 256, 96
    meta, q, k, v, cache, pools, plan, slots = _case(device, dtype, lens, N, H, D, fp4, packed, spread=False)
    T, B = sum(lens), len(lens)
    assert (T if packed else B * N) * D // 8 >= 256 * 2048 // 3 > 600 * D // 8
    cos, sin = _tables(D, R, device)
    start = {n: x.clone() for n, x in pools.items()}
    got_q = cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan, q=q, cos=cos, sin=sin, interleaved=interleaved)
    got = {n: x.clone() for n, x in pools.items()}
    for n, x in pools.items():
        x.copy_(start[n])
    flat = [x.view(H, T, D) if packed else torch.cat([x[b, :, :n] for b, n in enumerate(lens)], 1) for x in (q, k, v, got_q)]
    zero = torch.zeros(1, dtype=torch.int32, device=device)
    for at in range(0, T, 600):
        n = min(600, T - at)
        piece = PagedMetadata(plan.block_table[:1], plan.slot_mapping[at:at + n].contiguous(),
                              plan.positions[at:at + n].contiguous(), zero, torch.zeros(2, dtype=torch.int32, device=device))
        qq, kk, vv, want_q = (x[:, at:at + n].reshape(H * n, D) for x in flat)
        out = cache.append_paged_kv_cache(0, k=kk, v=vv, q_meta=build_pack_metadata(torch.tensor([n], device=device), n, 32),
                                          plan=piece, q=qq, cos=cos, sin=sin, interleaved=interleaved)
        assert torch.equal(out, want_q)
    assert all(torch.equal(x, got[n]) for n, x in pools.items())
    if not packed:
        for b, n in enumerate(lens):
            assert not got_q[b, :, n:].any()
    some = random.Random(1).sample([t for t in range(T) if 0 <= slots[t] < pools["k_pages"].shape[1] * PAGE], 200)
    pos = plan.positions.cpu().numpy()[some]
    kk = ref.rotate(_f64(flat[1][:, some]), _f64(cos)[pos], _f64(sin)[pos], interleaved)
    for name, x in (("k", kk), ("v", _f64(flat[2][:, some]))):
        rows = lambda n: got[name + n].view(H, -1, got[name + n].shape[-1])[:, [slots[t] for t in some]].cpu()  # noqa: B023,E731
        if fp4:
            codes, scales = ref.fp4_encode(x, dtype)
            assert (rows("_pages").numpy() == codes).all() and (rows("_scales").numpy() == scales).all()
        else:
            tol = np.abs(x) * torch.finfo(TYPES[dtype]).eps / 2 + (np.abs(x).max() * 2.0**-21 + 2.0**-25 if name == "k" else 0)
            assert (np.abs(_f64(rows("_pages")) - x) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_values_that_are_not_finite(device, dtype):
    """Infinities as the largest value, NaN as 0, zeros, the smallest and the largest values"""
    lens, H, D = [40], 2, 64
    meta, q, k, v, cache, pools, plan, _ = _case(device, dtype, lens, 40, H, D, True, False)
    plan.slot_mapping = torch.arange(40, device=device)
    fin = torch.finfo(TYPES[dtype])
    for x in (k, v):
        x[:, :, 0] = 0
        x[:, :, 1, 3] = float("inf")
        x[:, :, 2, 5] = float("-inf")
        x[:, :, 3, ::3] = float("nan")
        x[:, :, 4] = float("nan")
        x[:, :, 5] = fin.max
        x[:, :, 6] = fin.tiny
        x[:, :, 7] = fin.smallest_normal * 2.0**-3
        x[:, :, 8] = 7 * 2.0**-2
        x[:, :, 9] = fin.max
        x[:, :, 9, 1::2] = -fin.max / 2
    want = _expect(pools, lens, H, D, k, v, list(range(40)), dtype, True, lambda x: x)
    cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan)
    for n, x in want.items():
        assert (pools[n].cpu().numpy() == x).all(), n
    for x in cache.paged_kv_values(0):
        assert torch.isfinite(x).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_codes_next_to_borders(device, dtype):
    """Every value of a type's mantissas around every border of two codes and of two scales"""
    H, D, n = 1, 32, 4096
    meta = build_pack_metadata(torch.tensor([n], device=device), n, 32)
    dt = TYPES[dtype]
    g = torch.Generator(device=device).manual_seed(2)
    # a largest value in [3.5, 7) times a power of two, and 31 values of at most it
    bits = 7 if dtype == "bf16" else 10
    top = (1 + torch.randint(0, 2**bits, (n, 1), generator=g, device=device).double() / 2**bits) * 4
    rest = torch.randint(-(2**bits), 2**bits + 1, (n, 31), generator=g, device=device).double() / 2**bits
    x = (torch.cat((top, rest * top), 1) * torch.exp2(torch.randint(-6, 6, (n, 1), generator=g, device=device).double())).to(dt)
    P = n // PAGE
    pools = _fp4_pools(H, P, D, device, 1)
    cache = InferenceCache()
    table = torch.arange(P, dtype=torch.int32, device=device)[None]
    cache.prefill_paged_fp4_cache(0, **pools, block_table=table, context_lens=torch.zeros(1, dtype=torch.int32),
                                  num_heads=H, head_dim=D, dtype=dt)
    plan = PagedMetadata(table, torch.arange(n, device=device), None, torch.tensor([n], dtype=torch.int32, device=device),
                         torch.tensor([0, n], dtype=torch.int32, device=device))
    cache.append_paged_kv_cache(0, k=x, v=x, q_meta=meta, plan=plan)
    codes, scales = ref.fp4_encode(_f64(x), dtype)
    assert (pools["k_pages"].cpu().numpy().reshape(n, -1) == codes).all()
    assert (pools["v_scales"].cpu().numpy().reshape(n, -1) == scales).all()


@pytest.mark.gpu
def test_positions(device):
    """int64 and CPU positions, those out of range clamped on the GPU and refused on the CPU"""
    meta, q, k, v, cache, pools, plan, slots = _case(device, "bf16", [3, 2], 3, 2, 64, True, False)
    cos, sin = _tables(64, 64, device)
    run = lambda p: cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan, q=q, cos=cos, sin=sin, positions=p)  # noqa: E731
    want = run(None)
    assert torch.equal(run(plan.positions.long()), want) and torch.equal(run(plan.positions.cpu()), want)
    wild = torch.tensor([-5, 2**31 - 1, 0, 89, 90], dtype=torch.int32, device=device)
    assert torch.equal(run(wild), run(wild.clamp(0, 89)))
    wild = torch.tensor([-(2**40), 2**62, 0, 89, 90], dtype=torch.int64, device=device)
    assert torch.equal(run(wild), run(wild.clamp(0, 89)))
    with pytest.raises(ValueError, match="positions must lie"):
        run(wild.cpu())
    plan.positions = None
    with pytest.raises(ValueError, match="the plan has none"):
        run(None)


@pytest.mark.gpu
def test_append_q_refusals(device):
    meta, q, k, v, cache, pools, plan, slots = _case(device, "bf16", [3, 2], 3, 2, 64, True, False)
    cos, sin = _tables(64, 64, device)
    run = lambda **kw: cache.append_paged_kv_cache(0, **{**dict(k=k, v=v, q_meta=meta, plan=plan, q=q, cos=cos, sin=sin), **kw})  # noqa: E731
    before = {n: x.clone() for n, x in pools.items()}
    for match, kw in [("laid out like k", dict(q=q[:, :1])), ("q dtype/device", dict(q=q.half())),
                      ("no gradient", dict(q=q.clone().requires_grad_()))]:
        with pytest.raises(ValueError, match=match):
            run(**kw)
    assert all(torch.equal(before[n], x) for n, x in pools.items())
    with torch.no_grad():
        assert torch.equal(run(q=q.clone().requires_grad_()), run())


@pytest.mark.gpu
@pytest.mark.parametrize("fp4", [False, True])
def test_strided_rows(device, fp4):
    """Rows of other strides, unaligned ones, and broadcast heads"""
    lens, N, H, D = [4, 7], 7, 4, 64
    meta, q, k, v, cache, pools, plan, slots = _case(device, "fp16", lens, N, H, D, fp4, False)
    cos, sin = _tables(D, D, device)
    run = lambda q, k, v: cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan, q=q, cos=cos, sin=sin)  # noqa: E731
    want = run(q, k, v)
    after = {n: x.clone() for n, x in pools.items()}
    wide = torch.zeros((len(lens), N, 3, H, D + 8), dtype=q.dtype, device=device)
    parts = [wide[:, :, i, :, :D].transpose(1, 2) for i in range(3)]
    odd = [torch.zeros(q.numel() + 1, dtype=q.dtype, device=device)[1:].view(q.shape) for _ in range(3)]
    for dst in (parts, odd):
        for x, y in zip(dst, (q, k, v)):
            x.copy_(y)
        for x in pools.values():
            x.zero_()
        assert torch.equal(run(*dst), want)
        slot = [s for s in slots if 0 <= s < pools["k_pages"].shape[1] * PAGE]
        for n, x in pools.items():
            a, b = (y.view(H, -1, y.shape[-1])[:, slot] for y in (x, after[n]))
            assert torch.equal(a, b)
    one = q[:, :1].expand(-1, H, -1, -1)
    got = run(one, one, one)
    assert torch.equal(got, got[:, :1].expand(-1, H, -1, -1))


@pytest.mark.gpu
@pytest.mark.parametrize("fp4", [False, True])
def test_append_in_a_graph(device, fp4):
    """A captured append, replayed on other rows, slots and positions with eager work in between"""
    lens, N, H, D = [5, 3], 5, 3, 64
    meta, q, k, v, cache, pools, plan, slots = _case(device, "bf16", lens, N, H, D, fp4, False)
    cos, sin = _tables(D, D, device)
    run = lambda: cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan, q=q, cos=cos, sin=sin)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(4):
        for x in (q, k, v):
            x.normal_()
        plan.slot_mapping.copy_(torch.randperm(pools["k_pages"].shape[1] * PAGE, device=device)[: sum(lens)])
        plan.positions.random_(0, 90)
        for x in pools.values():
            x.fill_(i + 110 if fp4 else 1)
        graph.replay()
        got = out.clone(), {n: x.clone() for n, x in pools.items()}
        torch.cuda.synchronize()
        for x in pools.values():
            x.fill_(i + 110 if fp4 else 1)
        want = run()
        assert torch.equal(got[0], want) and all(torch.equal(got[1][n], x) for n, x in pools.items())


@pytest.mark.gpu
def test_append_counts_as_a_change_of_the_pools(device):
    meta, q, k, v, cache, pools, plan, slots = _case(device, "bf16", [5, 3], 5, 3, 64, True, False)
    before = {n: x._version for n, x in pools.items()}
    cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan)
    assert all(x._version > before[n] for n, x in pools.items())


@pytest.mark.gpu
def test_metadata_that_contradicts_itself_stays_in_bounds(device):
    """Offsets outside the call's tokens: such rows are no tokens (q's are zeros, nothing is stored)"""
    meta, q, k, v, cache, pools, plan, slots = _case(device, "bf16", [5, 3], 5, 3, 64, True, False)
    cos, sin = _tables(64, 64, device)
    meta.cu_seqlens = torch.tensor([-(2**30), 2**30, 2**31 - 1], dtype=torch.int32, device=device)
    before = {n: x.clone() for n, x in pools.items()}
    got = cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan, q=q, cos=cos, sin=sin)
    assert not got.any() and all(torch.equal(before[n], x) for n, x in pools.items())


@pytest.mark.gpu
@pytest.mark.parametrize("fp4", [False, True])
def test_more_threads_than_a_grid_has_in_x(device, fp4):
    """A padded batch of 2^27 positions and more with 256 dims a row: 2^32 threads.  (Rows of one address; the only
    tokens are the first and last ones.)"""
    N, B, H, D = (1 << 16) + 8, 1 << 11, 1, 256
    lens = [1] + [0] * (B - 2) + [N]
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    T, P = N + 1, (N + 1 + PAGE - 1) // PAGE
    g = torch.Generator(device=device).manual_seed(4)
    x = torch.randn((1, 1, 1, D), generator=g, device=device).bfloat16()
    k = x.expand(B, H, N, D)
    cache, table = InferenceCache(), torch.zeros((B, 1), dtype=torch.int32, device=device)
    index = dict(block_table=table, context_lens=torch.zeros(B, dtype=torch.int32), num_heads=H, head_dim=D)
    if fp4:
        pools = _fp4_pools(H, P, D, device)
        cache.prefill_paged_fp4_cache(0, **pools, dtype=x.dtype, **index)
    else:
        pools = {n: torch.zeros((H, P, PAGE, D), dtype=x.dtype, device=device) for n in ("k_pages", "v_pages")}
        cache.prefill_paged_kv_cache(0, **pools, is_mla=False, **index)
    plan = PagedMetadata(table, torch.arange(T, device=device), torch.zeros(T, dtype=torch.int32, device=device),
                         torch.zeros(B, dtype=torch.int32, device=device), torch.zeros(B + 1, dtype=torch.int32, device=device))
    cos = torch.ones((1, D // 2), device=device)  # (position 0: as they are)
    cache.append_paged_kv_cache(0, k=k, v=k, q_meta=meta, plan=plan, cos=cos, sin=torch.zeros_like(cos))
    want = torch.from_numpy(ref.fp4_values(*ref.fp4_encode(_f64(x), "bf16"))).to(device) if fp4 else x.double()
    for pages in cache.paged_kv_values(0):
        rows = pages.view(-1, D).double()
        assert torch.equal(rows[:T], want.view(1, D).expand(T, D)) and not rows[T:].any()


@pytest.mark.gpu
def test_pools_past_32_bits(device):
    """Rows behind element 2^32 of a pool: stored, read back and attended to"""
    H, D, P = 2, 256, 135000  # 2 * 135000 * 64 * 256 = 4.4e9 elements
    n = 70
    cache = InferenceCache()
    pools = _fp4_pools(H, P, D, device)
    table = torch.tensor([[P - 1, P - 3]], dtype=torch.int32, device=device)
    lens = torch.tensor([n], dtype=torch.int32, device=device)
    cache.prefill_paged_fp4_cache(0, **pools, block_table=table, context_lens=torch.zeros(1, dtype=torch.int32),
                                  num_heads=H, head_dim=D, dtype=torch.bfloat16)
    meta = build_pack_metadata(lens, n, 32)
    g = torch.Generator(device=device).manual_seed(1)
    q, k, v = (torch.randn((1, H, n, D), generator=g, device=device).bfloat16() for _ in range(3))
    slots = [(P - 1) * PAGE + i for i in range(64)] + [(P - 3) * PAGE + i for i in range(6)]
    plan = PagedMetadata(table, torch.tensor(slots, device=device), None, lens,
                         torch.tensor([0, n], dtype=torch.int32, device=device))
    cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan)
    codes, scales = ref.fp4_encode(_f64(k[0]), "bf16")
    for name, rows in (("k_pages", codes), ("k_scales", scales)):
        got = pools[name].view(H, P * PAGE, -1)[:, slots].cpu().numpy()
        assert (got == rows).all()
    out = flash_attn_mlm_window(q, None, None, H, meta, 0.0625, window=(20, 0), inference_cache=cache, layer_id=0)
    kd = ref.fp4_values(codes, scales)
    vd = ref.fp4_values(*ref.fp4_encode(_f64(v[0]), "bf16"))
    seen = ref.visible(0, n, n, 20, 0, 0)
    for h in range(H):
        o, P_ = ref.attend(_f64(q[0, h]), kd[h], vd[h], seen, 0.0625)
        # probabilities and the output are rounded, at most half a step each, the sum follows the former
        assert (np.abs(_f64(out.view(H, n, D)[h]) - o) <= 3.2 * 2.0**-8 * (P_ @ np.abs(vd[h])) + 1e-4).all()
