"""qk_norm_rope: refusals (CPU) and, on the GPU, rows and gradients against the 64-bit
restatement (oracle/paged_step_ref.py).

Tolerances, u = 2^-24: a row's sum of squares takes 8 fused steps and up to 6 additions
(14 u, half of it in its inverse root), the root and the products x r w and the rotation
8 u more: 16 u of the magnitudes a result is made of, and half a step of the output type.  A
gradient has two such factors and one more sum: 40 u.  dw sums at most `rows` terms.
"""

from __future__ import annotations

import itertools

import numpy as np
import pytest
import torch

from flash_mlm import _lib, build_pack_metadata, qk_norm_rope
from oracle import paged_step_ref as ref

U = 2.0**-24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _f(t):
    return t.detach().double().cpu().numpy()


def _tables(n, r, device):
    freq = 10000.0 ** (-torch.arange(0, r // 2, dtype=torch.float64) * 2 / r)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * freq
    return ang.cos().float().to(device), ang.sin().float().to(device)


def _half(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def _close(got, want, mag, dtype, steps):
    bound = _half(dtype) * np.abs(want) + steps * U * mag * (1 + _half(dtype)) + 1e-30
    if dtype == torch.float16:
        bound = bound + 2.0**-25  # half a step of its smallest values
    err = np.abs(got - want)
    assert np.all(err <= bound), f"worst {np.max(err / bound):.3f} of the bound"


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------
def test_needs_gpu_tensors():
    q = torch.zeros(1, 2, 3, 64)
    with pytest.raises(ValueError, match="CUDA tensors"):
        qk_norm_rope(q, q)


@pytest.mark.parametrize("q, k, kw, match", [
    ((1, 2, 64), (1, 2, 64), {}, "rank-4"),
    ((1, 2, 3, 64), (6, 64), {}, "rank-4"),
    ((1, 2, 3, 64), (1, 2, 3, 32), {}, "head_dim"),
    ((1, 2, 3, 80), (1, 2, 3, 80), {}, "HEAD_DIM"),
])
def test_refuses_shapes(q, k, kw, match):
    with pytest.raises(ValueError, match=match):
        qk_norm_rope(torch.zeros(q), torch.zeros(k), **kw)


def test_refuses_dtypes():
    q = torch.zeros(1, 2, 3, 64, dtype=torch.float64)
    with pytest.raises(ValueError, match="one dtype"):
        qk_norm_rope(q, q)
    with pytest.raises(ValueError, match="one dtype"):
        qk_norm_rope(q.float(), q.half())


def test_abi_refuses():
    lib = _lib.load()
    assert lib.fmlm_norm_rope(None, None) == -1
    p = _lib.NormRopeParams()
    p.dtype = 7
    assert lib.fmlm_norm_rope(p, None) == -2
    p.dtype, p.w_dtype, p.D = _lib.DTYPE_BF16, _lib.DTYPE_BF16, 48
    assert lib.fmlm_norm_rope(p, None) == -3
    p.D = 64
    assert lib.fmlm_norm_rope(p, None) == 0  # no rows
    p.B, p.N, p.rows = 1, 4, 5
    assert lib.fmlm_norm_rope(p, None) == -1  # rows are not B * N
    p.rows, p.q.heads = 4, 1
    assert lib.fmlm_norm_rope(p, None) == -1  # no tensor
    p.q.x, p.q.y = 256, 256 + 8
    assert lib.fmlm_norm_rope(p, None) == -4
    p.q.y, p.rotary_dim = 512, 24
    assert lib.fmlm_norm_rope(p, None) == -1  # rotary_dim
    p.rotary_dim = 32
    assert lib.fmlm_norm_rope(p, None) == -1  # no tables
    p.rotary_dim, p.layout, p.B, p.N, p.rows = 0, _lib.LAYOUT_PACKED, 2, 4, 4
    assert lib.fmlm_norm_rope(p, None) == -1  # packed rows of two sequences without token indices
    p.layout, p.rows, p.flags = _lib.LAYOUT_PADDED, 8, _lib.NR_NORM
    assert lib.fmlm_norm_rope_bwd_workspace_bytes(p) == -1  # no dy
    p.q.dy, p.q.weight, p.q.dweight = 1024, 2048, 4096
    need = lib.fmlm_norm_rope_bwd_workspace_bytes(p)
    assert need == 64 * 4  # one partial row
    assert lib.fmlm_norm_rope_bwd(p, None) == -5


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------
def _case(device, dtype, *, H, Hk, D, lens, N, R, gain, packed, inter, where, norm=True, seed=0, grad=False):
    g = torch.Generator().manual_seed(seed)
    B, T = len(lens), sum(lens)

    def rnd(*s):
        return torch.randn(s, generator=g)

    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    shape = (lambda h: (h * T, D)) if packed else (lambda h: (B, h, N, D))
    q, k, dq, dk = ((rnd(*shape(h)) * (1 + i)).to(dtype).to(device) for i, h in enumerate((H, Hk, H, Hk)))
    wq = wk = None
    if gain != "none":
        wq, wk = ((1 + 0.2 * rnd(*((h, D) if gain == "head" else (D,)))).to(dtype).to(device) for h in (H, Hk))
    kw = dict(q_weight=wq, k_weight=wk, norm=norm, interleaved=inter, q_meta=meta, eps=1e-5)
    b = np.repeat(np.arange(B), lens)
    p = np.concatenate([np.arange(n) for n in lens]) if T else np.zeros(0, int)
    cos = sin = None
    if R:
        kw["cos"], kw["sin"] = _tables(N + 40, R, device)
        if where == "context":
            start = torch.randint(0, 30, (B,), generator=g)
            kw["context_lens"], pos = start.to(device), start.numpy()[b] + p
        elif where == "positions":
            pos = torch.randint(0, N + 40, (T,), generator=g).numpy()
            kw["positions"] = torch.from_numpy(pos).to(torch.int32).to(device)
        else:
            pos = p
        cos, sin = _f(kw["cos"])[pos], _f(kw["sin"])[pos]
    if grad:
        for t in (q, k, wq, wk):
            if t is not None:
                t.requires_grad_()

    def tokens(x, h):  # [h, T, D]
        x = _f(x)
        return x.reshape(h, T, D) if packed else x[b, :, p].transpose(1, 0, 2)

    def whole(y, h):
        if packed:
            return y.reshape(h * T, D)
        out = np.zeros((B, h, N, D))
        out[b, :, p] = y.transpose(1, 0, 2)
        return out

    return q, k, dq, dk, kw, cos, sin, tokens, whole


def _check(device, dtype, *, grad=False, **c):
    H, Hk, gain, inter, norm = c["H"], c["Hk"], c["gain"], c["inter"], c.get("norm", True)
    q, k, dq, dk, kw, cos, sin, tokens, whole = _case(device, dtype, grad=grad, **c)
    outs = qk_norm_rope(q, k, **kw)
    opt = dict(eps=1e-5, norm=norm, interleaved=inter)
    gains = []
    for y, x, w, h in zip(outs, (q, k), (kw["q_weight"], kw["k_weight"]), (H, Hk)):
        wd = None if w is None else _f(w)[:, None, :] if gain == "head" else _f(w)
        gains.append(wd)
        want, mag = ref.norm_rope(tokens(x, h), wd, cos, sin, **opt)
        assert y.is_contiguous() and y.dtype == dtype and y.shape == x.shape
        _close(_f(y), whole(want, h), whole(mag, h), dtype, 16)
    if not grad:
        return
    leaves = [t for t in (q, k, kw["q_weight"], kw["k_weight"]) if t is not None]
    grads = torch.autograd.grad(outs, leaves, (dq, dk))
    for i, (x, dy, h) in enumerate(((q, dq, H), (k, dk, Hk))):
        dx, mag, dw, dwm = ref.norm_rope_grads(tokens(x, h), gains[i], cos, sin, tokens(dy, h), **opt)
        _close(_f(grads[i]), whole(dx, h), whole(mag, h), dtype, 40)
        if gains[i] is not None:
            axes = 1 if gain == "head" else (0, 1)
            rows = dw.shape[1] * (1 if gain == "head" else h)
            _close(_f(grads[2 + i]), dw.sum(axes), dwm.sum(axes), dtype, 40 + rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256, 512])
@pytest.mark.parametrize("inter", [False, True])
def test_rows_and_gradients(dtype, D, inter, device):
    _check(device, DT[dtype], H=5, Hk=3, D=D, lens=[37, 0, 1, 20], N=37, R=D, gain="shared", packed=False, inter=inter,
           where="context", seed=D, grad=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("packed, gain, where, R", [
    x for x in itertools.product([False, True], ["none", "shared", "head"], ["place", "positions"], [0, 16, 64])
    if not (x[3] == 0 and x[2] == "positions")
])
def test_layouts_gains_and_positions(dtype, packed, gain, where, R, device):
    _check(device, DT[dtype], H=4, Hk=1, D=128, lens=[3, 17, 9], N=19, R=R, gain=gain, packed=packed, inter=False,
           where=where, seed=7, grad=True)


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [False, True])
def test_rotation_alone(inter, device):
    _check(device, torch.float16, H=2, Hk=2, D=64, lens=[5, 8], N=8, R=32, gain="none", packed=False, inter=inter,
           where="place", norm=False, grad=True)


@pytest.mark.gpu
@pytest.mark.parametrize("lens, N", [([1], 1), ([1] * 70, 1), ([0, 0], 4), ([2000, 1500, 1999], 2000)])
@pytest.mark.parametrize("gain", ["shared", "head"])
def test_lengths(lens, N, gain, device):
    _check(device, torch.bfloat16, H=6, Hk=6, D=64, lens=lens, N=N, R=64, gain=gain, packed=False, inter=False,
           where="context", seed=N, grad=True)


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("shape", [(2, 0), (0, 3)])
def test_no_tokens(packed, shape, device):
    """Outputs and gradients of nothing are empty, the gains' gradients zero."""
    B, N = shape
    if packed:
        meta = build_pack_metadata(torch.zeros(2, dtype=torch.int32, device=device), 4, 32)
        q = torch.zeros((0, 64), device=device, requires_grad=True)
        kw = dict(q_meta=meta)
    else:
        q = torch.zeros((B, 3, N, 64), device=device, requires_grad=True)
        kw = {}
    w = torch.ones(64, device=device, requires_grad=True)
    cos, sin = _tables(4, 64, device)
    out = qk_norm_rope(q, q, q_weight=w, k_weight=w, cos=cos, sin=sin, **kw)
    assert out[0].shape == q.shape
    dq, dw = torch.autograd.grad(out, (q, w), tuple(torch.zeros_like(x) for x in out))
    assert dq.shape == q.shape and dw.shape == w.shape and not dw.any()


@pytest.mark.gpu
def test_mixed_gains(device):
    """Gains per head for q, shared for k: one launch, two layouts of dw."""
    q, k, dq, dk, kw, cos, sin, tokens, _ = _case(device, torch.float32, H=5, Hk=3, D=32, lens=[9, 30], N=30, R=32,
                                                  gain="head", packed=False, inter=False, where="place", grad=True)
    kw["k_weight"] = kw["k_weight"].detach()[0].clone().requires_grad_()
    outs = qk_norm_rope(q, k, **kw)
    gw = torch.autograd.grad(outs, (kw["q_weight"], kw["k_weight"]), (dq, dk))
    for g, x, dy, w, h, axes in ((gw[0], q, dq, _f(kw["q_weight"])[:, None], 5, 1),
                                 (gw[1], k, dk, _f(kw["k_weight"]), 3, (0, 1))):
        _, _, t, m = ref.norm_rope_grads(tokens(x, h), w, cos, sin, tokens(dy, h), eps=1e-5)
        _close(_f(g), t.sum(axes), m.sum(axes), torch.float32, 40 + 39 * 3)


@pytest.mark.gpu
def test_gradient_against_differences(device):
    """The gradient along a direction is what the (64-bit) loss does along it."""
    q, k, dq, dk, kw, cos, sin, tokens, _ = _case(device, torch.float32, H=2, Hk=2, D=64, lens=[6], N=6, R=64,
                                                  gain="shared", packed=False, inter=False, where="place", grad=True)
    grads = torch.autograd.grad(qk_norm_rope(q, k, **kw), (q, kw["q_weight"]), (dq, dk))
    rng = np.random.default_rng(0)
    x, w, dy = tokens(q, 2), _f(kw["q_weight"]), tokens(dq, 2)
    vx, vw = rng.standard_normal(x.shape), rng.standard_normal(w.shape)

    def loss(e):
        return (ref.norm_rope(x + e * vx, w + e * vw, cos, sin, eps=1e-5)[0] * dy).sum()

    h = 1e-5  # differences at 64 bits: error about h^2
    slope = (loss(h) - loss(-h)) / (2 * h)
    got = (tokens(grads[0], 2) * vx).sum() + (_f(grads[1]) * vw).sum()
    size = np.abs(tokens(grads[0], 2) * vx).sum() + np.abs(_f(grads[1]) * vw).sum()
    assert abs(got - slope) <= 60 * U * size + 1e-7 * size


@pytest.mark.gpu
def test_strides_padding_and_alignment(device):
    """q and k as views of one projection, NaN in padding rows, an unaligned view, a
    gradient of other strides."""
    B, N, H, D = 2, 13, 3, 64
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn((B, N, 3, H, D), generator=g).to(torch.bfloat16).to(device)
    meta = build_pack_metadata(torch.tensor([13, 4], device=device), N, 32)
    qkv[1, 4:] = float("nan")
    q, k = (qkv[:, :, i].transpose(1, 2) for i in range(2))
    cos, sin = _tables(N, D, device)
    kw = dict(cos=cos, sin=sin, q_meta=meta)
    got = qk_norm_rope(q, k, **kw)
    want = qk_norm_rope(q.contiguous(), k.contiguous(), **kw)
    for x, y in zip(got, want):
        assert torch.equal(x, y) and not x[1, :, 4:].any()
    flat = torch.empty(B * H * N * D + 1, dtype=torch.bfloat16, device=device)
    odd = flat[1:].view(B, H, N, D).copy_(q)
    assert odd.data_ptr() % 16
    assert torch.equal(qk_norm_rope(odd, k, **kw)[0], want[0])
    assert torch.equal(qk_norm_rope(q, k, cos=torch.cat([cos[:, :1], cos], 1)[:, 1:], sin=sin, q_meta=meta)[0], want[0])
    ql = q.detach().clone().requires_grad_()
    out = qk_norm_rope(ql, k, **kw)[0]
    dy = torch.randn((B, N, H, D), generator=g).to(torch.bfloat16).to(device)
    a = torch.autograd.grad(out, ql, dy.transpose(1, 2), retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(out, ql, dy.transpose(1, 2).contiguous())[0])
    assert not a[1, :, 4:].any()


@pytest.mark.gpu
def test_repeated_calls(device):
    """A call laid out like an earlier one takes its parameter block: with other tensors, after the
    metadata's fields were replaced, in another mode"""
    import dataclasses

    cos, sin = _tables(30, 64, device)
    meta = build_pack_metadata(torch.tensor([9, 4], device=device), 9, 32)

    def fresh(q, k, **kw):  # the same call on metadata that has seen none
        m = dataclasses.replace(meta, launch_memo={})
        return qk_norm_rope(q, k, cos=cos, sin=sin, q_meta=m, **kw)

    g = torch.Generator().manual_seed(0)
    for i in range(4):
        q, k = (torch.randn((2, 3, 9, 64), generator=g).to(device) for _ in range(2))
        w = torch.rand(64, generator=g).to(device)
        start = torch.randint(0, 20, (2,), generator=g).to(device)
        pos = torch.randint(0, 30, (13,), generator=g).to(device)
        for kw in (dict(), dict(q_weight=w), dict(q_weight=w, k_weight=w + 1, context_lens=start), dict(positions=pos),
                   dict(positions=pos, interleaved=True), dict(context_lens=start.int(), eps=0.5)):
            got, want = qk_norm_rope(q, k, cos=cos, sin=sin, q_meta=meta, **kw), fresh(q, k, **kw)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    other = build_pack_metadata(torch.tensor([2, 9], device=device), 9, 32)
    meta.cu_seqlens, meta.token_indices, meta.total_tokens = other.cu_seqlens, other.token_indices, other.total_tokens
    assert torch.equal(qk_norm_rope(q, k, cos=cos, sin=sin, q_meta=meta)[0],
                       qk_norm_rope(q, k, cos=cos, sin=sin, q_meta=other)[0])
    a = qk_norm_rope(q, k)
    assert torch.equal(qk_norm_rope(k, q)[0], a[1]) and torch.equal(qk_norm_rope(q, k)[0], a[0])


@pytest.mark.gpu
def test_packed_rows_of_other_strides_and_metadata(device):
    """Packed rows and gradients that are columns of a wider tensor; metadata of other integer
    types; metadata whose tables do not fit its counts"""
    import dataclasses

    lens, D = [5, 9], 64
    meta = build_pack_metadata(torch.tensor(lens, device=device), 9, 32)
    wide = torch.randn((2 * 14, 3 * D), device=device).half()
    q, k = wide[:, :D], wide[:, D : 2 * D]
    cos, sin = _tables(9, D, device)
    ql = q.contiguous().requires_grad_()
    want = qk_norm_rope(ql, k.contiguous(), cos=cos, sin=sin, q_meta=meta)
    dy = torch.randn((2 * 14, 2 * D), device=device).half()[:, D:]
    gw = torch.autograd.grad(want[0], ql, dy.contiguous(), retain_graph=True)[0]
    got = qk_norm_rope(q, k, cos=cos, sin=sin, q_meta=meta)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(torch.autograd.grad(want[0], ql, dy)[0], gw)
    other = dataclasses.replace(meta, cu_seqlens=meta.cu_seqlens.long(), token_indices=meta.token_indices.int())
    assert torch.equal(qk_norm_rope(q, k, cos=cos, sin=sin, q_meta=other)[0], want[0])
    for bad in (dict(token_indices=meta.token_indices[:-1]), dict(cu_seqlens=meta.cu_seqlens[:-1])):
        with pytest.raises(ValueError, match="do not match"):
            qk_norm_rope(q, k, q_meta=dataclasses.replace(meta, **bad))
    with pytest.raises(ValueError, match="device"):
        qk_norm_rope(q, k, q_meta=dataclasses.replace(meta, cu_seqlens=meta.cu_seqlens.cpu()))


@pytest.mark.gpu
@pytest.mark.parametrize("wt", ["fp16", "fp32"])
def test_gains_of_another_type(wt, device):
    """bf16 rows with gains of their own type: rows and gradients as at 64 bits"""
    q, k, dq, dk, kw, cos, sin, tokens, whole = _case(device, torch.bfloat16, H=3, Hk=2, D=64, lens=[7, 12], N=12, R=64,
                                                      gain="shared", packed=False, inter=False, where="place")
    w = kw["q_weight"] = kw["q_weight"].to(DT[wt]).requires_grad_()
    kw["k_weight"] = kw["k_weight"].to(DT[wt])
    out = qk_norm_rope(q, k, **kw)
    want, mag = ref.norm_rope(tokens(q, 3), _f(w), cos, sin, eps=1e-5)
    _close(_f(out[0]), whole(want, 3), whole(mag, 3), torch.bfloat16, 16)
    g = torch.autograd.grad(out[0], w, dq)[0]
    _, _, t, m = ref.norm_rope_grads(tokens(q, 3), _f(w), cos, sin, tokens(dq, 3), eps=1e-5)
    assert g.dtype == DT[wt]
    _close(_f(g), t.sum((0, 1)), m.sum((0, 1)), DT[wt], 40 + 57)


@pytest.mark.gpu
def test_positions_are_clamped_on_the_gpu_and_refused_on_the_cpu(device):
    q = torch.randn((1, 2, 4, 64), device=device)
    cos, sin = _tables(8, 64, device)
    far = torch.tensor([[-5, 3, 100, 7]], device=device)
    near = torch.tensor([[0, 3, 7, 7]])
    a = qk_norm_rope(q, q, cos=cos, sin=sin, positions=far)
    b = qk_norm_rope(q, q, cos=cos, sin=sin, positions=near)
    assert torch.equal(a[0], b[0])
    with pytest.raises(ValueError, match="positions values"):
        qk_norm_rope(q, q, cos=cos, sin=sin, positions=far.cpu())


@pytest.mark.gpu
def test_refusals(device):
    q = torch.zeros((2, 3, 5, 64), device=device)
    cos, sin = _tables(8, 64, device)
    meta = build_pack_metadata(torch.tensor([5, 2], device=device), 5, 32)
    w = torch.ones(64, device=device)
    for match, kw in [
        ("nothing to do", dict(norm=False)),
        ("gains need", dict(norm=False, cos=cos, sin=sin, q_weight=w)),
        ("same dtype", dict(q_weight=w, k_weight=w.half())),
        ("head_dim", dict(q_weight=w[:32])),
        ("come together", dict(cos=cos)),
        ("fp32 tables", dict(cos=cos.half(), sin=sin.half())),
        ("multiple of 16", dict(cos=cos[:, :4], sin=sin[:, :4])),
        ("multiple of 16", dict(cos=cos[:0], sin=sin[:0])),
        ("need cos", dict(context_lens=torch.zeros(2, dtype=torch.int32, device=device))),
        ("shape", dict(cos=cos, sin=sin, positions=[0, 1])),
        ("exclusive", dict(cos=cos, sin=sin, context_lens=torch.zeros(2, dtype=torch.int32, device=device),
                           positions=torch.zeros((2, 5), dtype=torch.int32, device=device))),
        ("shape", dict(cos=cos, sin=sin, positions=torch.zeros(7, dtype=torch.int32, device=device))),
        ("shape", dict(cos=cos, sin=sin, positions=torch.zeros((2, 5), device=device))),
        ("eps", dict(eps=float("nan"))),
        ("num_heads", dict(num_heads=4)),
    ]:
        with pytest.raises(ValueError, match=match):
            qk_norm_rope(q, q, **kw)
    with pytest.raises(ValueError, match="constants"):
        qk_norm_rope(q, q, cos=cos.clone().requires_grad_(), sin=sin)
    with pytest.raises(ValueError, match="q_meta"):
        qk_norm_rope(q[:1], q[:1], q_meta=meta)
    with pytest.raises(ValueError, match="packed q needs"):
        qk_norm_rope(q.view(-1, 64), q.view(-1, 64))
    with pytest.raises(ValueError, match="multiple of the token count"):
        qk_norm_rope(q.view(-1, 64), q.view(-1, 64), q_meta=meta)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        x = q.clone().requires_grad_()
        starts = torch.zeros(2, dtype=torch.int32, device=device)
        y = qk_norm_rope(x, q, cos=cos, sin=sin, context_lens=starts)[0]
        starts += 1
        y.sum().backward()


@pytest.mark.gpu
def test_unused_outputs_and_partial_gradients(device):
    q, k, dq, dk, kw, *_ = _case(device, torch.float32, H=2, Hk=2, D=64, lens=[6, 3], N=6, R=64, gain="shared",
                                 packed=False, inter=False, where="place", grad=True)
    wq, wk = kw["q_weight"], kw["k_weight"]
    all_ = torch.autograd.grad(qk_norm_rope(q, k, **kw), (q, k, wq, wk), (dq, dk))
    out = qk_norm_rope(q, k, **kw)
    a = torch.autograd.grad(out[0], (q, k, wq, wk), dq, allow_unused=True)
    assert torch.equal(a[0], all_[0]) and torch.equal(a[2], all_[2]) and a[1] is None and a[3] is None
    kw["q_weight"] = wq.detach()
    out = qk_norm_rope(q.detach(), k.detach(), **kw)
    assert not out[0].requires_grad or out[1].requires_grad
    assert torch.equal(torch.autograd.grad(out[1], wk, dk)[0], all_[3])


@pytest.mark.gpu
def test_same_bits_every_time_on_another_stream_and_in_a_graph(device):
    q, k, dq, dk, kw, *_ = _case(device, torch.bfloat16, H=8, Hk=8, D=128, lens=[300, 411, 5], N=411, R=128,
                                 gain="shared", packed=False, inter=False, where="context", grad=True)
    leaves = (q, k, kw["q_weight"], kw["k_weight"])

    def step():
        out = qk_norm_rope(q, k, **kw)
        return [*out, *torch.autograd.grad(out, leaves, (dq, dk))]

    first = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    for a, b in zip(first, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    # outputs of an eager call hold its autograd graph: the capture is refused until they are gone
    with pytest.raises(ValueError, match="being captured"):
        with torch.cuda.graph(graph):
            qk_norm_rope(q, k, **kw)
    del other, b
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
        twice = step()  # the same leaves again, in the same capture
    captured, twice = ([t.detach() for t in x] for x in (captured, twice))
    for seed in range(3):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)).to(q.dtype))
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(captured, step(), twice):
            assert torch.equal(a, b) and torch.equal(c, b)


@pytest.mark.gpu
def test_feeds_attention(device):
    """The rows go into the packed attention as they come out, and gradients flow through both."""
    from flash_mlm import flash_attn_mlm_compressed

    B, H, N, D = 2, 4, 24, 64
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn((B, H, N, D), generator=g).to(device).requires_grad_() for _ in range(3))
    meta = build_pack_metadata(torch.tensor([24, 9], device=device), N, 32)
    cos, sin = _tables(N, D, device)
    qn, kn = qk_norm_rope(q, k, cos=cos, sin=sin, q_meta=meta)
    out = flash_attn_mlm_compressed(qn, kn, v, H, meta, 0.125)
    dout = torch.randn(out.shape, generator=g).to(device)
    got = torch.autograd.grad(out, (q, k, v), dout)
    # the same in elementary operations at 64 bits
    x = [t.detach().double().requires_grad_() for t in (q, k, v)]

    def rot(t):
        t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6)
        a, b = t[..., :32], t[..., 32:]
        c, s = cos.double(), sin.double()
        return torch.cat((a * c - b * s, a * s + b * c), -1)

    parts = []
    for b, n in enumerate((24, 9)):
        w = torch.softmax(0.125 * rot(x[0])[b, :, :n] @ rot(x[1])[b, :, :n].transpose(1, 2), -1)
        parts.append(w @ x[2][b, :, :n])
    want = torch.autograd.grad(torch.cat(parts, 1).reshape(H * 33, D), x, dout.double())
    for a, b in zip(got, want):
        # fp32 throughout: sums of up to 64 products a score, 24 keys a row
        assert (a.double() - b).abs().max() <= 2000 * U * b.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("through", [False, True])  # whether the incoming gradients have one
def test_gradients_have_no_gradient(through, device):
    q, k = (torch.randn((1, 2, 5, 64), device=device, requires_grad=True) for _ in range(2))
    a, b = qk_norm_rope(q, k)
    plain = torch.autograd.grad((a, b), (q, k), (torch.ones_like(a), torch.ones_like(b)), retain_graph=True)
    ones = [torch.ones_like(a).requires_grad_(through), torch.ones_like(b).requires_grad_(through)]
    dq, dk = torch.autograd.grad((a, b), (q, k), ones, create_graph=True)
    assert torch.equal(dq, plain[0]) and torch.equal(dk, plain[1])
    with pytest.raises(RuntimeError, match="once_differentiable" if through else "does not require grad"):
        dq.sum().backward()


@pytest.mark.gpu
def test_rows_past_32_bits(device):
    """Rows at both ends of a tensor of more than 2^32 elements: the bits of the same rows alone."""
    H, N, D, n = 2, 4194400, 512, 3
    q = torch.empty((1, H, N, D), dtype=torch.bfloat16, device=device).normal_()
    k = torch.empty((1, 1, N, D), dtype=torch.bfloat16, device=device).normal_()
    assert q.numel() > 2**32
    angle = torch.arange(8, device=device)[:, None] * torch.linspace(1, 0.01, 128, device=device)
    cos, sin = angle.cos(), angle.sin()
    pos = (torch.arange(N, dtype=torch.int32, device=device) % 8)[None]
    q.requires_grad_(), k.requires_grad_()
    a, b = qk_norm_rope(q, k, cos=cos, sin=sin, positions=pos)
    dq, dk = torch.autograd.grad((a, b), (q, k), (q.detach(), k.detach()))
    for part in (slice(0, n), slice(N // 2, N // 2 + n), slice(N - n, N)):
        x, y = (t.detach()[:, :, part].contiguous().requires_grad_() for t in (q, k))
        c, d = qk_norm_rope(x, y, cos=cos, sin=sin, positions=pos[:, part])
        dx, dy = torch.autograd.grad((c, d), (x, y), (x.detach(), y.detach()))
        for big, small in ((a, c), (b, d), (dq, dx), (dk, dy)):
            assert torch.equal(big[:, :, part], small)


def _hooked_layer(device, dtype, seed=3):
    """A layer whose gains, tables and positions are temporaries: (leaves, function of them, gradients in)"""
    g = torch.Generator().manual_seed(seed)
    B, H, N, D, R = 2, 3, 20, 64, 32
    meta = build_pack_metadata(torch.tensor([20, 9], device=device), N, 32) if device.type == "cuda" else None
    q, k, dq, dk = (torch.randn((B, H, N, D), generator=g).to(dtype).to(device) for _ in range(4))
    w = (1 + 0.2 * torch.randn((2, H, D), generator=g)).to(device)

    def layer(q, k, w):
        cos, sin = _tables(N + 40, R, device)
        if meta is None:
            where = dict(positions=(torch.arange(B * N, device=device) % 50).view(B, N) + 3)
        else:
            where = dict(q_meta=meta, context_lens=torch.tensor([5, 30], device=device))
        wide = torch.stack([w, w], -1).to(dtype)[..., 0]  # a strided temporary: copied inside the call
        return qk_norm_rope(q, k, q_weight=wide[0], k_weight=wide[1], cos=cos, sin=sin, eps=1e-5, **where)

    for t in (q, k, w):
        t.requires_grad_()
    return (q, k, w), layer, (dq, dk)


def test_backward_reads_what_autograd_kept(monkeypatch):
    """Saved tensors may come back at other addresses (checkpoints, offload hooks): the gradient's block
    holds those, not the forward's."""
    import ctypes

    from flash_mlm.host import norm_rope as nr

    blocks = []

    def run(entry, name, p, device):
        def at(ptr, n, ctype):
            return list((ctype * n).from_address(ptr)) if ptr else None

        rows = p.rows * p.D
        blocks.append((name, [at(t.x, t.heads * rows, ctypes.c_float) for t in (p.q, p.k)],
                       [at(t.weight, t.heads * p.D, ctypes.c_float) for t in (p.q, p.k)],
                       [at(x, p.table_rows * p.rotary_dim // 2, ctypes.c_float) for x in (p.cos, p.sin)],
                       at(p.positions, p.rows, ctypes.c_int64)))

    monkeypatch.setattr(nr, "_run", run)
    monkeypatch.setattr(nr, "require_cuda_tensors", lambda *t: None)
    monkeypatch.setattr(nr, "_MEMO", {})  # (real calls must not find these)
    monkeypatch.setattr(nr, "_capture_leaves", lambda *t: [])
    originals = []

    def pack(t):
        originals.append(t)
        return t.detach().clone()

    for unpack in (lambda t: t, lambda t: torch.stack([t, t], -1)[..., 0]):  # as they were, and strided
        blocks.clear()
        originals.clear()
        leaves, layer, dys = _hooked_layer(torch.device("cpu"), torch.float32)
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            out = layer(*leaves)
        for t in originals:  # their memory belongs to something else by now
            t.data.fill_(7)
        torch.autograd.grad(out, leaves, dys)
        assert [b[0] for b in blocks] == ["fmlm_norm_rope", "fmlm_norm_rope_bwd"]
        assert blocks[0][1:] == blocks[1][1:]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.flatten()[:8]):
        out = layer(*_hooked_layer(torch.device("cpu"), torch.float32)[0])
    with pytest.raises(RuntimeError, match="saved tensor"):
        out[0].sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("way", ["checkpoint", "clone", "strided", "cpu"])
def test_gradients_of_checkpointed_and_hooked_calls(dtype, way, device):
    from torch.utils.checkpoint import checkpoint

    leaves, layer, dys = _hooked_layer(device, DT[dtype])
    want = torch.autograd.grad(layer(*leaves), leaves, dys)
    if way == "checkpoint":
        out = checkpoint(layer, *leaves, use_reentrant=False)
    else:
        pack, unpack = {"clone": (lambda t: t.clone(), lambda t: t), "cpu": (lambda t: t.cpu(), lambda t: t.to(device)),
                        "strided": (lambda t: torch.stack([t, t], -1), lambda t: t[..., 0])}[way]
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            out = layer(*leaves)
    spoil = [torch.full((n,), float("nan"), device=device) for n in (32, 96, 192, 480, 960, 1920, 7680) for _ in range(40)]
    got = torch.autograd.grad(out, leaves, dys)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    del spoil
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.cpu()):
        out = layer(*leaves)
    with pytest.raises(RuntimeError, match="another device"):
        torch.autograd.grad(out, leaves, dys)


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_refusals_after_a_legal_call(packed, device):
    """A wrong call is refused whatever ran before it: also when all but its fault is like an earlier call"""
    meta = build_pack_metadata(torch.tensor([5, 2], device=device), 5, 32)
    q = torch.randn((21, 64) if packed else (2, 3, 5, 64), device=device)
    cos, sin = _tables(8, 64, device)
    pos, starts = torch.zeros(7, dtype=torch.int32, device=device), torch.zeros(2, dtype=torch.int32, device=device)
    for q_meta in (meta, None):
        kw = dict(cos=cos, sin=sin, q_meta=q_meta)
        at = pos if q_meta is not None or packed else torch.zeros((2, 5), dtype=torch.int32, device=device)
        if q_meta is None and packed:
            kw["num_heads"] = 3
        for _ in range(2):
            qk_norm_rope(q, q, positions=at, **kw)
            for bad in (starts, torch.zeros(9, device=device), [1, 2]):
                with pytest.raises(ValueError, match="exclusive"):
                    qk_norm_rope(q, q, positions=at, context_lens=bad, **kw)
            with pytest.raises(ValueError, match="come together"):
                qk_norm_rope(q, q, positions=at, **{**kw, "sin": None})
            with pytest.raises(ValueError, match="shape"):
                qk_norm_rope(q, q, positions=at.float(), **kw)
            with pytest.raises(ValueError, match="gains need"):
                qk_norm_rope(q, q, positions=at, norm=False, q_weight=torch.ones(64, device=device), **kw)


@pytest.mark.parametrize("which", range(6))
def test_refuses_tangents(which, monkeypatch):
    """Forward-mode tangents are refused, not dropped, in a first call and in one like an earlier one"""
    from flash_mlm.host import norm_rope as nr
    from torch.autograd import forward_ad as fw

    monkeypatch.setattr(nr, "_run", lambda *a: None)
    monkeypatch.setattr(nr, "require_cuda_tensors", lambda *t: None)
    monkeypatch.setattr(nr, "_MEMO", {})  # (real calls must not find these)
    cos, sin = _tables(8, 32, "cpu")
    args = [torch.randn(1, 2, 3, 64), torch.randn(1, 2, 3, 64), torch.ones(64), torch.ones(64), cos, sin]

    def call(a):
        return qk_norm_rope(a[0], a[1], q_weight=a[2], k_weight=a[3], cos=a[4], sin=a[5], eps=1e-5 * (1 + which))

    for _ in range(2):
        with fw.dual_level():
            dual = list(args)
            dual[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
            with pytest.raises(ValueError, match="forward-mode"):
                call(dual)
            call(args)
        call(args)


@pytest.mark.gpu
def test_refuses_tangents_on_the_gpu(device):
    from torch.autograd import forward_ad as fw

    q = torch.randn((1, 2, 3, 64), device=device)
    want = qk_norm_rope(q, q)
    with fw.dual_level():
        dual = fw.make_dual(q, torch.ones_like(q))
        for x in (dual, dual.detach().requires_grad_(), dual.transpose(1, 2).contiguous().transpose(1, 2)):
            if x is dual or fw.unpack_dual(x).tangent is not None:
                with pytest.raises(ValueError, match="forward-mode"):
                    qk_norm_rope(x, q)
        assert torch.equal(qk_norm_rope(q, q)[0], want[0])
    with pytest.raises(Exception):
        torch.func.jvp(lambda x: qk_norm_rope(x, q)[0], (q,), (torch.ones_like(q),))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["q", "k", "gain", "packed"])
def test_captures_of_leaves_that_are_copied(which, device):
    """A leaf that the call copies for its kernel (an odd start, another stride) is checked as any other: no
    capture while an eager graph of it lives, and captured gradients replay."""
    g = torch.Generator().manual_seed(4)
    B, H, N, D = 2, 3, 9, 64

    def odd(*shape):
        n = int(np.prod(shape))
        t = torch.empty(n + 1, dtype=torch.bfloat16, device=device)[1:].view(shape)
        return t.copy_(torch.randn(shape, generator=g)).requires_grad_()

    shape = (H * B * N, D) if which == "packed" else (B, H, N, D)
    q, k = (odd(*shape) if which in (n, "packed") else
            torch.randn(shape, generator=g).bfloat16().to(device).requires_grad_() for n in "qk")
    w = torch.ones((D, 2), dtype=torch.bfloat16, device=device)[:, 0] if which == "gain" else torch.ones(D, device=device).bfloat16()
    w.requires_grad_()
    kw = dict(q_weight=w, k_weight=w, num_heads=H)
    dys = [torch.randn(shape, generator=g).bfloat16().to(device) for _ in range(2)]
    leaves = (q, k, w)
    assert all(t.is_leaf for t in leaves)

    def step():
        out = qk_norm_rope(q, k, **kw)
        return [*out, *torch.autograd.grad(out, leaves, dys)]

    alive = qk_norm_rope(q, k, **kw)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match="being captured") as refusal:
        with torch.cuda.graph(graph):
            qk_norm_rope(q, k, **kw)
    del alive  # (the refusal's traceback lives on)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
        twice = step()
    captured, twice = ([t.detach() for t in x] for x in (captured, twice))
    for seed in range(3):
        with torch.no_grad():
            q.copy_(torch.randn(shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(captured, step(), twice):
            assert torch.equal(a, b) and torch.equal(c, b)
