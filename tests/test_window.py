"""flash_attn_mlm_window: the oracle and refusals (CPU); on the GPU outputs over every kind of
context and gradients against the 64-bit restatement (oracle/window_ref.py), masks that leave
rows empty, values that are not finite where nobody looks, graphs, and a server's steps with the
appends that fill the context."""

from __future__ import annotations

import gc
import random

import numpy as np
import pytest
import torch

import flash_mlm as fm
from flash_mlm import InferenceCache, PackMetadata, _lib, build_block_table, build_pack_metadata, flash_attn_mlm_window
from oracle import window_ref as ref

PAGE = 64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _half(dtype):
    return torch.finfo(TYPES[dtype]).eps / 2  # a rounding is off by at most this, relative to the value


def _cpu_meta(lens, N):
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    tok = torch.tensor([b * N + p for b, n in enumerate(lens) for p in range(n)], dtype=torch.int64)
    return PackMetadata(B=len(lens), N=N, lengths=torch.tensor(lens, dtype=torch.int32), cu_seqlens=cu, token_indices=tok,
                        total_tokens=sum(lens), batch_ids_block_n=32, batch_ids_q=cu, q_tile_starts_q=cu)


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------
def test_oracle_sets_by_hand():
    see = lambda **kw: ref.visible(**{**dict(first=2, n=3, total=6, left=None, right=None, sinks=0), **kw}).astype(int).tolist()  # noqa: E731
    assert see() == [[1] * 6] * 3
    assert see(right=0) == [[1, 1, 1, 0, 0, 0], [1, 1, 1, 1, 0, 0], [1, 1, 1, 1, 1, 0]]
    assert see(left=1, right=0) == [[0, 1, 1, 0, 0, 0], [0, 0, 1, 1, 0, 0], [0, 0, 0, 1, 1, 0]]
    assert see(left=0, right=1, sinks=2) == [[1, 1, 1, 1, 0, 0], [1, 1, 0, 1, 1, 0], [1, 1, 0, 0, 1, 1]]
    assert see(first=-2, left=0, right=1, sinks=4) == [[0] * 6, [1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0]]


def test_oracle_attention_and_gradients():
    rng = np.random.default_rng(0)
    n, m, D = 5, 7, 4
    q, k, v, do = (rng.standard_normal((x, D)) for x in (n, m, m, n))
    seen = ref.visible(2, n, m, 2, 1, 1)
    o, P = ref.attend(q, k, v, seen, 0.7)
    z = np.where(seen, q @ k.T * 0.7, -np.inf)
    w = np.exp(z) / np.exp(z).sum(1, keepdims=True)
    assert np.allclose(o, w @ v) and np.allclose(P, w)
    assert not ref.attend(q, k, v, np.zeros((n, m), bool), 0.7)[0].any()
    grads = ref.attend_backward(q, k, v, seen, 0.7, do)
    f = lambda a, b, c: (ref.attend(a, b, c, seen, 0.7)[0] * do).sum()  # noqa: E731
    for i, x in enumerate((q, k, v)):
        for _ in range(6):
            d = rng.standard_normal(x.shape)
            args = lambda h: [y + h * d if j == i else y for j, y in enumerate((q, k, v))]  # noqa: E731
            diff = (f(*args(1e-5)) - f(*args(-1e-5))) / 2e-5
            assert abs(diff - (grads[i] * d).sum()) <= 1e-7 * (1 + abs(diff))


def test_refusals():
    meta = _cpu_meta([2, 1], 2)
    q = torch.zeros((2, 2, 2, 64), dtype=torch.bfloat16)
    cache = InferenceCache()
    call = dict(q=q, k=q, v=q, num_heads=2, q_meta=meta, scale=1.0)
    for match, kw in [
        ("window must be a pair", dict(window=5)),
        ("window must be a pair", dict(window=(1, 2, 3))),
        ("window must be an integer", dict(window=(-1, 0))),
        ("window must be an integer", dict(window=(1.5, 0))),
        ("window must be an integer", dict(window=[0, True])),
        ("sinks must be an integer", dict(sinks=-1)),
        ("sinks must be an integer", dict(sinks=None)),
        ("together or both omitted", dict(inference_cache=cache)),
        ("together or both omitted", dict(layer_id=0)),
        ("k and v come together", dict(v=None)),
        ("same shape", dict(k=q[:1])),
        ("q must be padded", dict(q=q[0], k=q[0], v=q[0])),
        ("must match num_heads", dict(num_heads=3)),
        ("num_heads must be", dict(num_heads=0)),
        ("does not match q/k/v padded shape", dict(q=q[:1], k=q[:1], v=q[:1])),
        ("num_heads \\* q_meta.total_tokens", dict(q=q.view(-1, 64), k=q.view(-1, 64), v=q.view(-1, 64))),
        ("bf16 or fp16", dict(q=q.float(), k=q.float(), v=q.float())),
        ("head_dim 32, 64", dict(q=q[..., :16], k=q[..., :16], v=q[..., :16])),
        ("the same dtype", dict(k=q.half())),
        ("must be CUDA tensors", dict()),
        ("must be CUDA tensors", dict(q=q.view(-1, 64)[:6], k=q.view(-1, 64)[:6], v=q.view(-1, 64)[:6])),
    ]:
        with pytest.raises(ValueError, match=match):
            flash_attn_mlm_window(**{**call, **kw})


def test_context_refusals():
    """What the context's part of the checks refuses, without a GPU."""
    from flash_mlm.host.window import _context

    cache = InferenceCache()
    rows = torch.zeros((2 * 6, 64), dtype=torch.bfloat16)
    store = lambda n, cu: cache.prefill_kv_cache(  # noqa: E731
        n, k_cache=rows, v_cache=rows, total_context_len=6, cu_seqlens_kv=cu, context_batch_size=2, is_mla=False,
        num_heads=2, head_dim=64)
    store("dense", None)
    store("packed", torch.tensor([0, 2, 6], dtype=torch.int32))
    run = lambda n, b, index=None, appended=False: _context(  # noqa: E731
        cache.layer_entry(n), _lib.AttnParams(), _lib.Window(), b=b, context_index=index, appended=appended,
        device=torch.device("cpu"))
    run("packed", 2)
    run("packed", 2, appended=True)
    run("packed", 3, torch.tensor([0, 1, 1]))
    for match, a in [
        ("packed or paged context", ("dense", 2)),
        ("1 or at least the batch size", ("packed", 3)),
        ("one entry per sequence", ("packed", 3, torch.tensor([0, 1]))),
        ("must lie in", ("packed", 2, torch.tensor([0, 2]))),
    ]:
        with pytest.raises(ValueError, match=match):
            run(*a)
    cache.layer_entry("packed").context_batch_size = 1
    with pytest.raises(ValueError, match="a context batch for each sequence"):
        run("packed", 2, appended=True)


@pytest.mark.parametrize("kind", ["paged", "fp4"])
@pytest.mark.parametrize("pages,width", [(3, 0), (0, 2), (0, 0)])
def test_contexts_without_a_page_to_read(kind, pages, width):
    """A block table without columns (torch gives it no address) or a pool without pages: no context rows."""
    from flash_mlm.host.window import _context

    H, D, cache = 2, 64, InferenceCache()
    index = dict(block_table=torch.zeros((2, width), dtype=torch.int32), context_lens=torch.zeros(2, dtype=torch.int32),
                 num_heads=H, head_dim=D)
    pool = lambda cols, dt: torch.zeros((H, pages, PAGE, cols), dtype=dt)  # noqa: E731
    if kind == "fp4":
        codes, scales = pool(D // 2, torch.uint8), pool(D // 32, torch.uint8)
        cache.prefill_paged_fp4_cache(0, k_pages=codes, v_pages=codes, k_scales=scales, v_scales=scales,
                                      dtype=torch.bfloat16, **index)
    else:
        rows = pool(D, torch.bfloat16)
        cache.prefill_paged_kv_cache(0, k_pages=rows, v_pages=rows, is_mla=False, **index)
    p, w = _lib.AttnParams(), _lib.Window()
    p.dtype, p.B, p.H, p.D, p.N, p.total_q, p.cu_seqlens_q, p.q, p.o = 0, 2, H, D, 4, 8, 256, 256, 256
    keep = _context(cache.layer_entry(0), p, w, b=2, context_index=None, appended=True, device=torch.device("cpu"))  # noqa: F841
    w.flags |= _lib.WINDOW_APPENDED
    assert p.ctx_rows == 0 and p.ctx_pages_per_batch == 0
    assert _lib.load().fmlm_window_workspace_bytes(p, w) == 0


def test_rows_far_apart_are_copied():
    """Positions 2^22 elements apart and more are outside the kernels' tile offsets; a single row has no pitch."""
    from flash_mlm.host.window import _rows, _strides

    make = lambda n, pitch: torch.empty_strided((2, 3, n, 64), (192, 64, pitch, 1), dtype=torch.bfloat16, device="meta")  # noqa: E731
    near, far, one = make(5, (1 << 22) - 8), make(5, 1 << 22), make(1, 1 << 40)
    assert _rows(near) is near and _strides(near, 0) == (192, 64, (1 << 22) - 8)
    assert _rows(far).is_contiguous() and _strides(_rows(far), 0) == (3 * 5 * 64, 5 * 64, 64)
    assert _rows(one) is one and _strides(one, 0) == (192, 64, 64)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_scales_that_are_not_finite_are_refused(scale):
    """Masked scores are -inf times the scale."""
    q = torch.zeros((2, 2, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="scale must be finite"):
        flash_attn_mlm_window(q, q, q, 2, _cpu_meta([2, 1], 2), scale)
    p, w = _lib.AttnParams(), _lib.Window()
    p.dtype, p.B, p.H, p.D, p.N, p.total_q, p.cu_seqlens_q = _lib.DTYPE_BF16, 1, 1, 64, 4, 4, 256
    p.q = p.o = p.k = p.v = 256
    assert _lib.load().fmlm_window_workspace_bytes(p, w) == 0
    p.scale = scale
    assert _lib.load().fmlm_window_workspace_bytes(p, w) == -1 and _lib.load().fmlm_window_fwd(p, w, None) == -1


@pytest.mark.parametrize("which", [0, 1])
def test_gradients_and_tangents_of_a_context_are_refused(which):
    """Of keys or of values: the call would drop them without a word."""
    import torch.autograd.forward_ad as fwd

    q, meta = torch.zeros((2, 2, 2, 64), dtype=torch.bfloat16), _cpu_meta([2, 1], 2)
    rows = [torch.zeros((2 * 6, 64), dtype=torch.bfloat16) for _ in range(2)]
    cache = InferenceCache()

    def run():
        cache.prefill_kv_cache(0, k_cache=rows[0], v_cache=rows[1], total_context_len=6,
                               cu_seqlens_kv=torch.tensor([0, 2, 6], dtype=torch.int32), context_batch_size=2,
                               is_mla=False, num_heads=2, head_dim=64)
        flash_attn_mlm_window(q, q, q, 2, meta, 1.0, inference_cache=cache, layer_id=0)

    plain, rows[which] = rows[which], rows[which].clone().requires_grad_()
    with pytest.raises(ValueError, match="no gradient of a cached context"):
        run()
    with torch.no_grad(), pytest.raises(ValueError, match="must be CUDA tensors"):
        run()
    with fwd.dual_level():
        rows[which] = fwd.make_dual(plain, torch.ones_like(plain))
        with pytest.raises(ValueError, match="no forward-mode"):
            run()


def test_offsets_of_a_context_on_another_device_are_refused():
    """A packed entry keeps the offsets that it was given: their host address must not reach the kernel."""
    from flash_mlm.host.window import _context

    cache, rows = InferenceCache(), torch.zeros((2 * 6, 64), dtype=torch.bfloat16)
    cache.prefill_kv_cache(0, k_cache=rows, v_cache=rows, total_context_len=6,
                           cu_seqlens_kv=torch.tensor([0, 2, 6], dtype=torch.int32), context_batch_size=2, is_mla=False,
                           num_heads=2, head_dim=64)
    with pytest.raises(ValueError, match="cu_seqlens_kv of the cached context must be on the device"):
        _context(cache.layer_entry(0), _lib.AttnParams(), _lib.Window(), b=2, context_index=None, appended=False,
                 device=torch.device("meta"))


def test_saved_tensors_that_do_not_fit_are_refused():
    """What a saved-tensor hook brings back is checked before its address is used."""
    from flash_mlm.host.window import _Call, _check_saved

    call, dev, dt = _Call(), torch.device("cpu"), torch.bfloat16
    call.shape, call.out_shape = torch.Size((2, 3, 5, 32)), (3 * 7, 32)
    rows, out = [torch.zeros(call.shape, dtype=dt) for _ in range(3)], torch.zeros(call.out_shape, dtype=dt)
    saved = [*rows, out, torch.zeros(21), out.clone()]
    _check_saved(call, saved, dt, dev)
    _check_saved(call, [rows[0].transpose(0, 1).contiguous().transpose(0, 1), *saved[1:]], dt, dev)
    for i, x in enumerate(saved):
        for y in (x[:1], x.view(-1), x[None], x.half(), x.to(torch.float8_e4m3fn), x.to("meta")):
            if y.shape == x.shape and y.dtype == x.dtype and y.device == x.device:
                continue  # (the statistics have one dimension)
            with pytest.raises(RuntimeError, match="saved tensor came back"):
                _check_saved(call, [*saved[:i], y, *saved[i + 1:]], dt, dev)


def test_offsets_changed_since_the_forward_are_refused():
    """The row statistics belong to the offsets that the forward read."""
    from types import SimpleNamespace

    from flash_mlm.host.window import _backward, _Call, _version

    call, dt = _Call(), torch.bfloat16
    call.shape, call.out_shape, call.cu = torch.Size((21, 32)), (21, 32), torch.tensor([0, 3, 7])
    x = torch.zeros((21, 32), dtype=dt)
    ctx = SimpleNamespace(call=call, cu_version=_version(call), saved_tensors=(x, x, x, x, torch.zeros(21), x))
    call.cu.copy_(torch.tensor([0, 5, 7]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        _backward(ctx, x)
    with torch.inference_mode():
        call.cu = call.cu.clone()
    assert _version(call) is None  # (such a tensor counts no changes)


def test_argument_rejection_without_launch():
    lib = _lib.load()
    p, w = _lib.AttnParams(), _lib.Window()
    assert lib.fmlm_window_fwd(None, w, None) == -1 and lib.fmlm_window_fwd(p, None, None) == -1
    fwd = lambda: lib.fmlm_window_fwd(p, w, None)  # noqa: E731
    p.dtype, p.B, p.H, p.D, p.N, p.total_q = _lib.DTYPE_F32, 1, 1, 64, 4, 4
    assert fwd() == -2
    p.dtype, p.D = _lib.DTYPE_BF16, 16
    assert fwd() == -3
    p.D = 64
    for flag in (_lib.FLAG_MLA, _lib.FLAG_PREFILL, _lib.FLAG_CAUSAL_SEQ, _lib.FLAG_TREE):
        p.flags = flag
        assert fwd() == -1
    p.flags = 0
    assert fwd() == -1  # no offsets
    p.cu_seqlens_q = 256
    assert fwd() == -4  # no rows
    p.q = p.o = p.k = p.v = 256
    p.q_sn = 4
    assert fwd() == -4
    p.q_sn = 64
    w.flags = _lib.WINDOW_APPENDED  # without a context
    assert fwd() == -1
    w.flags = 4
    assert fwd() == -1
    w.flags = 0
    p.total_q = 1 << 30
    assert fwd() == -1
    p.total_q = 4
    p.ctx_len = 5  # without offsets
    assert fwd() == -1
    p.ctx_len, p.cu_seqlens_kv, p.ctx_rows, p.ctx_batch = 0, 256, 70, 0
    assert fwd() == -1
    p.ctx_batch, p.B = 2, 3  # fewer context batches than sequences
    assert fwd() == -1
    p.ctx_batch, p.B = 1, 1
    assert fwd() == -4  # no context rows
    p.k_ctx = p.v_ctx = 256
    w.flags = _lib.WINDOW_FP4  # 4 bits without pages
    assert fwd() == -1
    w.flags = 0
    # records of a call that is split
    p.ctx_rows, p.c_sn, p.c_sh, w.left = 1 << 20, 64, 1 << 26, -1
    assert lib.fmlm_window_workspace_bytes(p, w) > 0
    assert fwd() == -5
    p.flags = _lib.FLAG_NOSPLIT
    assert lib.fmlm_window_workspace_bytes(p, w) == 0
    p.flags, p.lse = 0, 256
    assert lib.fmlm_window_workspace_bytes(p, w) == 0
    g = _lib.AttnGrads()
    assert lib.fmlm_window_bwd(p, w, g, None) == -1  # a context
    p.cu_seqlens_kv, p.lse = None, None
    assert lib.fmlm_window_bwd(p, w, g, None) == -1  # no statistics
    p.lse = 256
    assert lib.fmlm_window_bwd(p, w, g, None) == -4
    g.dout = g.dq = g.dk = g.dv = 256
    assert lib.fmlm_window_bwd(p, w, g, None) == -5
    assert lib.fmlm_window_bwd(p, w, None, None) == -1


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------
def _f64(t):
    return t.detach().double().cpu().numpy()


def _rand(g, shape, dt):
    return torch.randn(shape, generator=g, device=g.device).to(dt)


class _Layer:
    """A cached context of each kind with its rows as 64-bit values: k[b], v[b] [H, rows, D]"""

    def __init__(self, kind, dtype, H, D, ctx, device, g, spare=2):
        dt, B = TYPES[dtype], len(ctx)
        self.cache, self.k, self.v = InferenceCache(), [], []
        lens = torch.tensor(ctx, dtype=torch.int32, device=device)
        if kind == "packed":
            T = sum(ctx) + spare
            self.rows = [_rand(g, (H, T, D), dt) for _ in range(2)]
            cu = [sum(ctx[:b]) for b in range(B + 1)]
            self.cache.prefill_kv_cache(0, k_cache=self.rows[0].view(-1, D), v_cache=self.rows[1].view(-1, D),
                                        total_context_len=T, cu_seqlens_kv=torch.tensor(cu, dtype=torch.int32, device=device),
                                        context_batch_size=B, is_mla=False, num_heads=H, head_dim=D)
            self.at = [list(range(cu[b], cu[b + 1])) for b in range(B)]
        else:
            need = [(n + PAGE - 1) // PAGE for n in ctx]
            P = sum(need) + spare
            ids = random.Random(sum(ctx)).sample(range(P), P)
            width = max(need) + 1
            table, self.at, i = [], [], 0
            for n, m in zip(ctx, need):
                mine = ids[i:i + m]
                i += m
                table.append(mine + [-1, 10**6][: width - m] + [-5] * (width - m - 2))
                self.at.append([mine[j // PAGE] * PAGE + j % PAGE for j in range(n)])
            table = torch.tensor([t[:width] for t in table], dtype=torch.int32, device=device)
            if kind == "fp4":
                self.pools = {}
                for name in "kv":
                    codes, scales = ref.fp4_encode(_f64(_rand(g, (H, P, PAGE, D), dt)), dtype)
                    for n, x in (("_pages", codes), ("_scales", scales)):
                        self.pools[name + n] = torch.from_numpy(x).to(device)
                self.cache.prefill_paged_fp4_cache(0, **self.pools, block_table=table, context_lens=lens, num_heads=H,
                                                   head_dim=D, dtype=dt)
                self.rows = [torch.from_numpy(ref.fp4_values(self.pools[n + "_pages"].cpu().numpy(),
                                                             self.pools[n + "_scales"].cpu().numpy())) for n in "kv"]
            else:
                self.rows = [_rand(g, (H, P, PAGE, D), dt) for _ in range(2)]
                self.cache.prefill_paged_kv_cache(0, k_pages=self.rows[0], v_pages=self.rows[1], block_table=table,
                                                  context_lens=lens, is_mla=False, num_heads=H, head_dim=D)
            self.rows = [x.view(H, P * PAGE, D) for x in self.rows]
        self.read()

    def read(self):
        k, v = (_f64(x) for x in self.rows)
        self.k, self.v = ([x[:, at] for at in self.at] for x in (k, v))


def _check(out, q, k, v, lens, ctx, layer, window, sinks, scale, dtype, appended=False, batch=None):
    """Every row against the oracle: probabilities are rounded (at most half a step, the sum is that of
    the rounded ones) and the output: h (P |v| + |o|) + h |o| <= 3 h P |v|; 1e-4 of it for fp32 scores
    (to 20, 2^-24 a product) and exponentials, and fp16's probabilities below 2^-14."""
    B, H, D = len(lens), q.shape[1], q.shape[-1]
    got = _f64(out).reshape(H, sum(lens), D)
    at = 0
    for b, n in enumerate(lens):
        cb = b if batch is None else batch[b]
        m = ctx[cb] if layer is not None else 0
        for h in range(H):
            kk = np.zeros((0, D)) if layer is None else layer.k[cb][h]
            vv = np.zeros((0, D)) if layer is None else layer.v[cb][h]
            if not appended:
                kk, vv = (np.concatenate((x, _f64(y[b, h, :n]))) for x, y in ((kk, k), (vv, v)))
            seen = ref.visible(m - n if appended else m, n, len(kk), *window, sinks)
            o, P = ref.attend(_f64(q[b, h, :n]), kk, vv, seen, scale)
            with np.errstate(invalid="ignore"):
                size = np.where(P > 0, P, 0) @ np.abs(np.where(np.isfinite(vv), vv, 0))
            tol = (3 * _half(dtype) + 1e-4) * size + 2.0**-24 * len(kk)
            err = np.abs(got[h, at:at + n] - o)
            assert (err <= tol).all(), (b, h, (err / np.maximum(tol, 1e-30)).max())
            assert not got[h, at:at + n][~seen.any(1)].any()
        at += n


def _inputs(device, dtype, lens, N, H, D, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    q, k, v = (_rand(g, (len(lens), H, N, D), TYPES[dtype]) for _ in range(3))
    meta = build_pack_metadata(torch.tensor(lens, device=device), N, 32)
    return g, q, k, v, meta


WINDOWS = [((None, None), 0), ((None, 0), 0), ((0, 0), 0), ((7, 0), 2), ((63, 64), 1), ((100, None), 70), ((1, 3), 130)]


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS, ids=str)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_without_a_context(device, dtype, D, window, sinks):
    lens, N, H = [1, 0, 130, 64, 37], 131, 2
    _, q, k, v, meta = _inputs(device, dtype, lens, N, H, D, 1)
    out = flash_attn_mlm_window(q, k, v, H, meta, 0.2, window=window, sinks=sinks)
    _check(out, q, k, v, lens, None, None, window, sinks, 0.2, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS, ids=str)
@pytest.mark.parametrize("appended", [False, True])
@pytest.mark.parametrize("kind,dtype,D", [("packed", "fp16", 64), ("paged", "bf16", 128), ("fp4", "bf16", 32), ("fp4", "fp16", 64),
                                          ("fp4", "bf16", 128), ("fp4", "fp16", 256), ("paged", "fp16", 256), ("packed", "bf16", 32)])
def test_contexts(device, kind, dtype, D, appended, window, sinks):
    """Few rows (key ranges are split) over contexts of no rows, one, whole and partial pages"""
    lens, N, H, ctx = [3, 1, 0, 5, 2, 1], 5, 2, [0, 1, 64, 700, 65, 129]
    g, q, k, v, meta = _inputs(device, dtype, lens, N, H, D, 2)
    layer = _Layer(kind, dtype, H, D, ctx, device, g)
    kv = (None, None) if appended else (k, v)
    out = flash_attn_mlm_window(q, *kv, H, meta, -0.15, window=window, sinks=sinks, inference_cache=layer.cache, layer_id=0)
    _check(out, q, k, v, lens, ctx, layer, window, sinks, -0.15, dtype, appended)


def _kept_bytes(meta):
    """Bytes of the split's records of the one kept call of ``meta``"""
    call, = meta.launch_memo.values()
    return call.nbytes


@pytest.mark.gpu
@pytest.mark.parametrize("appended", [False, True])
@pytest.mark.parametrize("window,sinks", [((None, None), 0), ((1500, 0), 4)], ids=str)
@pytest.mark.parametrize("N", [1, 4, 5, 16])
@pytest.mark.parametrize("kind,dtype,D", [("fp4", "bf16", 32), ("fp4", "fp16", 64), ("fp4", "bf16", 128), ("fp4", "fp16", 256),
                                          ("paged", "fp16", 64), ("packed", "bf16", 128), ("paged", "bf16", 256)])
def test_few_rows_whose_key_ranges_are_split(device, kind, dtype, D, N, window, sinks, appended):
    """Long contexts with partial last pages beside a short one, which stays whole in the same call"""
    lens, H, ctx = [N, 1, max(N - 2, 1)], 2, [2500, 130, 2111]
    g, q, k, v, meta = _inputs(device, dtype, lens, N, H, D, 41)
    layer = _Layer(kind, dtype, H, D, ctx, device, g)
    kv = (None, None) if appended else (k, v)
    out = flash_attn_mlm_window(q, *kv, H, meta, 0.15, window=window, sinks=sinks, inference_cache=layer.cache, layer_id=0)
    assert _kept_bytes(meta) > 0
    _check(out, q, k, v, lens, ctx, layer, window, sinks, 0.15, dtype, appended)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp4", "paged"])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("N", [1, 6])
def test_the_most_parts(device, kind, D, N):
    """One sequence over 20 thousand keys: 32 parts, joined by one and by several rows a workgroup"""
    lens, H, ctx = [N], 1, [20001]
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 42)
    layer = _Layer(kind, "bf16", H, D, ctx, device, g)
    out = flash_attn_mlm_window(q, k, v, H, meta, 0.15, inference_cache=layer.cache, layer_id=0)
    assert _kept_bytes(meta) == 32 * 8 * N * (D + 4) * 4  # (8: pairs are counted in eights)
    _check(out, q, k, v, lens, ctx, layer, (None, None), 0, 0.15, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 16])
def test_few_rows_whose_key_ranges_stay_whole(device, N):
    lens, H, D, ctx = [N, 1], 2, 64, [400, 3]
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 43)
    layer = _Layer("fp4", "bf16", H, D, ctx, device, g)
    out = flash_attn_mlm_window(q, k, v, H, meta, 0.15, inference_cache=layer.cache, layer_id=0)
    assert _kept_bytes(meta) == 0
    _check(out, q, k, v, lens, ctx, layer, (None, None), 0, 0.15, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("appended", [False, True])
@pytest.mark.parametrize("kind", ["packed", "paged", "fp4"])
@pytest.mark.parametrize("lens", [[3, 1, 0, 5], [16, 2, 9, 16], [200, 40, 0, 1]], ids=str)
@pytest.mark.parametrize("D", [64, 128])
def test_layouts_beside_a_context(device, kind, lens, appended, D):
    """Packed rows, rows of other strides and unaligned ones: the same bits as contiguous padded ones"""
    N, H, ctx = max(lens), 3, [300, 64, 7, 129]
    g, q, k, v, meta = _inputs(device, "fp16", lens, N, H, D, 44)
    layer = _Layer(kind, "fp16", H, D, ctx, device, g)
    run = lambda q, k, v: flash_attn_mlm_window(q, *((None, None) if appended else (k, v)), H, meta, 0.1, window=(120, 3),  # noqa: E731
                                                sinks=5, inference_cache=layer.cache, layer_id=0)
    want = run(q, k, v)
    _check(want, q, k, v, lens, ctx, layer, (120, 3), 5, 0.1, "fp16", appended)
    flat = [torch.cat([x[b, :, :n] for b, n in enumerate(lens)], 1).reshape(-1, D) for x in (q, k, v)]
    assert torch.equal(run(*flat), want)
    wide = torch.zeros((len(lens), N, 3, H, D + 8), dtype=q.dtype, device=device)
    parts = [wide[:, :, i, :, :D].transpose(1, 2) for i in range(3)]
    odd = [torch.zeros(q.numel() + 1, dtype=q.dtype, device=device)[1:].view(q.shape) for _ in range(3)]
    for dst in (parts, odd):
        for x, y in zip(dst, (q, k, v)):
            x.copy_(y)
        assert torch.equal(run(*dst), want)
    one = [x[:, :1].expand(-1, H, -1, -1) for x in (q, k, v)]
    assert torch.equal(run(*one), run(*(x.contiguous() for x in one)))


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS[1:5], ids=str)
@pytest.mark.parametrize("kind", ["packed", "paged", "fp4"])
def test_long_rows_over_contexts(device, kind, window, sinks):
    lens, N, H, D, ctx = [200, 129, 0, 1], 200, 2, 64, [100, 0, 5, 300]
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 3)
    layer = _Layer(kind, "bf16", H, D, ctx, device, g)
    out = flash_attn_mlm_window(q, k, v, H, meta, 0.125, window=window, sinks=sinks, inference_cache=layer.cache, layer_id=0)
    _check(out, q, k, v, lens, ctx, layer, window, sinks, 0.125, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS, ids=str)
@pytest.mark.parametrize("kind,dtype", [("packed", "fp16"), ("paged", "bf16")])
def test_tall_tiles_over_contexts(device, kind, dtype, window, sinks):
    """Enough heads for 128-row tiles in 16 bits; the first ones are checked"""
    lens, N, H, D, ctx = [200, 129, 0, 1], 200, 64, 128, [100, 0, 5, 300]
    g, q, k, v, meta = _inputs(device, dtype, lens, N, H, D, 31)
    layer = _Layer(kind, dtype, H, D, ctx, device, g)
    out = flash_attn_mlm_window(q, k, v, H, meta, 0.1, window=window, sinks=sinks, inference_cache=layer.cache, layer_id=0)
    _check(out[: 2 * sum(lens)], q[:, :2], k[:, :2], v[:, :2], lens, ctx, layer, window, sinks, 0.1, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS + [((150, 20), 3)], ids=str)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_tall_tiles_and_their_gradients(device, dtype, window, sinks):
    """Enough heads for 128-row tiles; the first two are checked, the others repeat them"""
    lens, N, H, D = [200, 129, 0, 300], 301, 64, 128
    g, q, k, v, meta = _inputs(device, dtype, lens, N, 2, D, 32)
    leaves = [x.repeat(1, H // 2, 1, 1).requires_grad_() for x in (q, k, v)]
    out = flash_attn_mlm_window(*leaves, H, meta, 0.15, window=window, sinks=sinks)
    two = 2 * sum(lens)
    assert torch.equal(out, out[:two].repeat(H // 2, 1))
    _check(out[:two], q, k, v, lens, None, None, window, sinks, 0.15, dtype)
    do = _rand(g, (two, D), out.dtype)
    grads = torch.autograd.grad(out, leaves, do.repeat(H // 2, 1))
    assert all(torch.equal(x, x[:, :2].repeat(1, H // 2, 1, 1)) for x in grads)
    got = [_by_sequence(x[:, :2], lens, 2, D) for x in grads]
    _grad_check(got, q, k, v, _f64(do).reshape(2, -1, D), lens, window, sinks, 0.15, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["packed", "paged", "fp4"])
def test_context_index_and_shared_contexts(device, kind):
    lens, N, H, D = [2, 1, 3], 3, 2, 64
    g, q, k, v, meta = _inputs(device, "fp16", lens, N, H, D, 4)
    layer = _Layer(kind, "fp16", H, D, [70, 5], device, g)
    index = torch.tensor([1, 0, 1], device=device)
    run = lambda **kw: flash_attn_mlm_window(q, k, v, H, meta, 0.125, window=(40, 1), sinks=3, inference_cache=layer.cache,  # noqa: E731
                                             layer_id=0, **kw)
    _check(run(context_index=index), q, k, v, lens, [70, 5], layer, (40, 1), 3, 0.125, "fp16", batch=[1, 0, 1])
    assert torch.equal(run(context_index=index), run(context_index=index.cpu()))
    wild = torch.tensor([2**31 - 1, -9, 1], device=device)  # clamped
    assert torch.equal(run(context_index=wild), run(context_index=index))
    with pytest.raises(ValueError, match="at least the batch size"):
        run()
    one = _Layer(kind, "fp16", H, D, [90], device, g)  # shared by all
    out = flash_attn_mlm_window(q, k, v, H, meta, 0.125, window=(40, 1), sinks=3, inference_cache=one.cache, layer_id=0)
    _check(out, q, k, v, lens, [90], one, (40, 1), 3, 0.125, "fp16", batch=[0, 0, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_compressed_calls_over_four_bits(device, dtype, D):
    """flash_attn_mlm_compressed: all of the context and all of the sequence's tokens"""
    lens, N, H, ctx = [3, 1, 0, 70], 70, 3, [200, 64, 3, 0]
    g, q, k, v, meta = _inputs(device, dtype, lens, N, H, D, 5)
    layer = _Layer("fp4", dtype, H, D, ctx, device, g)
    out = fm.flash_attn_mlm_compressed(q, k, v, H, meta, 0.1, layer.cache, 0)
    _check(out, q, k, v, lens, ctx, layer, (None, None), 0, 0.1, dtype)
    assert torch.equal(out, fm.flash_attn_mlm_compressed(q, k, v, H, meta, 0.1, layer.cache, 0, context_batch_size=4))


@pytest.mark.gpu
def test_it_agrees_with_compressed_calls(device):
    """Without a limit: what flash_attn_mlm_compressed computes over the same pages"""
    lens, N, H, D, ctx = [9, 30], 30, 2, 128, [500, 77]
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 6)
    layer = _Layer("paged", "bf16", H, D, ctx, device, g)
    a = flash_attn_mlm_window(q, k, v, H, meta, 0.09, inference_cache=layer.cache, layer_id=0)
    b = fm.flash_attn_mlm_compressed(q, k, v, H, meta, 0.09, layer.cache, 0)
    assert (a.float() - b.float()).abs().max() <= 8 * 2.0**-8 * b.float().abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -1e-30, 3.0])
def test_scales(device, scale):
    lens, N, H, D = [40, 3], 40, 2, 64
    _, q, k, v, meta = _inputs(device, "fp16", lens, N, H, D, 7)
    out = flash_attn_mlm_window(q, k, v, H, meta, scale, window=(9, 2), sinks=1)
    _check(out, q, k, v, lens, None, None, (9, 2), 1, scale, "fp16")


@pytest.mark.gpu
def test_strides_and_packed_rows(device):
    lens, N, H, D = [40, 3, 0, 17], 40, 3, 64
    _, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 8)
    run = lambda q, k, v: flash_attn_mlm_window(q, k, v, H, meta, 0.125, window=(9, 2), sinks=1)  # noqa: E731
    want = run(q, k, v)
    wide = torch.zeros((len(lens), N, 3, H, D + 8), dtype=q.dtype, device=device)
    parts = [wide[:, :, i, :, :D].transpose(1, 2) for i in range(3)]
    odd = [torch.zeros(q.numel() + 1, dtype=q.dtype, device=device)[1:].view(q.shape) for _ in range(3)]
    rev = [torch.zeros((H, len(lens), N, D), dtype=q.dtype, device=device).transpose(0, 1) for _ in range(3)]
    for dst in (parts, odd, rev):
        for x, y in zip(dst, (q, k, v)):
            x.copy_(y)
        assert torch.equal(run(*dst), want)
    flat = [torch.cat([x[b, :, :n] for b, n in enumerate(lens)], 1).reshape(-1, D) for x in (q, k, v)]
    assert torch.equal(run(*flat), want)
    one = [x[:, :1].expand(-1, H, -1, -1) for x in (q, k, v)]
    assert torch.equal(run(*one), run(*(x.contiguous() for x in one)))


@pytest.mark.gpu
@pytest.mark.parametrize("fp4", [False, True])
def test_more_workgroups_than_a_grid_has_in_x(device, fp4):
    """2^24 and more (sequence, head) pairs: 2^32 threads.  A single token sees itself alone: its output is its
    value and dv the output's gradient, bit for bit."""
    B, H, D = 65537, 256, 32
    g = torch.Generator(device=device).manual_seed(19)
    meta = build_pack_metadata(torch.ones(B, dtype=torch.int32, device=device), 1, 32)
    q, k, v = (torch.randn((B, H, 1, D), generator=g, device=device, dtype=torch.bfloat16) for _ in range(3))
    heads_first = lambda x: x[:, :, 0].transpose(0, 1).reshape(H * B, D)  # noqa: E731
    if fp4:  # over an empty context
        pool = lambda cols: torch.zeros((H, 1, PAGE, cols), dtype=torch.uint8, device=device)  # noqa: E731
        cache = InferenceCache()
        cache.prefill_paged_fp4_cache(0, k_pages=pool(16), v_pages=pool(16), k_scales=pool(1), v_scales=pool(1),
                                      block_table=torch.zeros((1, 1), dtype=torch.int32), context_lens=torch.zeros(1, dtype=torch.int32),
                                      num_heads=H, head_dim=D, dtype=q.dtype)
        out = fm.flash_attn_mlm_compressed(q, k, v, H, meta, 0.3, cache, 0)
        assert torch.equal(out, heads_first(v))
        return
    v.requires_grad_()
    out = flash_attn_mlm_window(q, k, v, H, meta, 0.3, window=(3, 0))
    assert torch.equal(out, heads_first(v))
    do = torch.randn(out.shape, generator=g, device=device, dtype=out.dtype)
    dv, = torch.autograd.grad(out, v, do)
    assert torch.equal(heads_first(dv), do)


@pytest.mark.gpu
def test_calls_past_32_bits(device):
    """Packed rows behind element 2^32 of q, k, v, the output and the gradients: the bits of the last sequence alone"""
    H, D, n = 2, 256, 90
    long = (1 << 32) // (H * D) + 1000
    T = long + n
    meta, alone = (build_pack_metadata(torch.tensor(x, device=device), max(x), 32) for x in ([long, n], [n]))
    g = torch.Generator(device=device).manual_seed(20)
    xs = [torch.randn((H * T, D), generator=g, device=device, dtype=torch.bfloat16).requires_grad_() for _ in range(3)]
    do = torch.randn((H * T, D), generator=g, device=device, dtype=torch.bfloat16)
    tail = lambda x: x.view(H, T, D)[:, long:].reshape(H * n, D).detach()  # noqa: E731
    ys = [tail(x).requires_grad_() for x in xs]
    a = flash_attn_mlm_window(*xs, H, meta, 0.07, window=(50, 3), sinks=2)
    b = flash_attn_mlm_window(*ys, H, alone, 0.07, window=(50, 3), sinks=2)
    assert torch.equal(tail(a), b)
    want = torch.autograd.grad(b, ys, tail(do))
    del b
    assert all(torch.equal(tail(x), y) for x, y in zip(torch.autograd.grad(a, xs, do), want))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 90])
@pytest.mark.parametrize("kind", ["paged", "packed"])
def test_contexts_past_32_bits(device, kind, n):
    """Context rows behind element 2^32: the bits of the same rows in a small context"""
    H, D, P = 2, 256, 135000  # 2 * 135000 * 64 * 256 = 4.4e9 elements
    lens, ctx = [n], [300]
    g, q, k, v, meta = _inputs(device, "fp16", lens, n, H, D, 21)
    small = _Layer(kind, "fp16", H, D, ctx, device, g)
    run = lambda cache: flash_attn_mlm_window(q, k, v, H, meta, 0.07, window=(200, 3), sinks=2, inference_cache=cache, layer_id=0)  # noqa: E731
    want = run(small.cache)
    rows = [torch.zeros((H, P * PAGE, D), dtype=q.dtype, device=device) for _ in range(2)]
    cache = InferenceCache()
    if kind == "packed":
        first = P * PAGE - 300
        cache.prefill_kv_cache(0, k_cache=rows[0].view(-1, D), v_cache=rows[1].view(-1, D), total_context_len=P * PAGE,
                               cu_seqlens_kv=torch.tensor([0, first, first + 300], dtype=torch.int32, device=device),
                               context_batch_size=2, is_mla=False, num_heads=H, head_dim=D)
        at = list(range(first, first + 300))
        index = dict(context_index=torch.tensor([1], device=device))
        run = lambda cache: flash_attn_mlm_window(q, k, v, H, meta, 0.07, window=(200, 3), sinks=2, inference_cache=cache,  # noqa: E731
                                                  layer_id=0, **index)
    else:
        pages = [P - 1, P - 7, P - 2, P - 3, P - 5]
        cache.prefill_paged_kv_cache(0, k_pages=rows[0].view(H, P, PAGE, D), v_pages=rows[1].view(H, P, PAGE, D),
                                     block_table=torch.tensor([pages], device=device), context_lens=torch.tensor([300]),
                                     is_mla=False, num_heads=H, head_dim=D)
        at = [pages[j // PAGE] * PAGE + j % PAGE for j in range(300)]
    for x, y in zip(rows, small.rows):
        x[:, at] = y[:, small.at[0]]
    # (key ranges may be cut otherwise: the larger context's rule knows its rows only)
    got = run(cache)
    _check(got, q, k, v, lens, ctx, small, (200, 3), 2, 0.07, "fp16")
    assert (got.float() - want.float()).abs().max() <= 4 * 2.0**-11 * want.float().abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_padding_rows_stay_out_of_gradients(device, D):
    """Rows of a padded batch behind its sequences that are not finite"""
    lens, N, H = [70, 0, 129, 1], 140, 2
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 22)
    do = _rand(g, (H * sum(lens), D), q.dtype)
    run = lambda xs: torch.autograd.grad(flash_attn_mlm_window(*xs, H, meta, 0.1, window=(40, 9), sinks=3), xs, do)  # noqa: E731
    want = run([x.clone().requires_grad_() for x in (q, k, v)])
    for x in (q, k, v):
        for b, n in enumerate(lens):
            x[b, :, n:] = float("nan")
    assert all(torch.equal(a, b) for a, b in zip(run([x.requires_grad_() for x in (q, k, v)]), want))


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 3])
def test_positions_far_apart(device, N):
    """Rows whose positions are 2^22 elements apart, as in a [N, B, H, D] batch of many sequences"""
    lens, H, D = [N, 1], 2, 64
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 18)
    far = [torch.empty_strided(q.shape, (H * D, D, 1 << 22, 1), dtype=q.dtype, device=device).copy_(x) for x in (q, k, v)]
    run = lambda a: flash_attn_mlm_window(*a, H, meta, 0.125, window=(9, 2), sinks=1)  # noqa: E731
    assert torch.equal(run(far), run((q, k, v)))
    do = _rand(g, (H * sum(lens), D), q.dtype)
    grads = []
    for xs in (far, (q, k, v)):
        xs = [x.detach().requires_grad_() for x in xs]
        grads.append(torch.autograd.grad(run(xs), xs, do))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.gpu
def test_rows_behind_the_sequences_stay_out(device):
    """Padding rows that are not finite, and pages and rows behind a context's end"""
    lens, N, H, D, ctx = [3, 70], 90, 2, 64, [70, 3]
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 9)
    layers = [_Layer(kind, "bf16", H, D, ctx, device, g) for kind in ("packed", "paged", "fp4")]
    want = [flash_attn_mlm_window(q, k, v, H, meta, 0.1, window=(50, 2), sinks=2, inference_cache=x.cache, layer_id=0)
            for x in layers]
    for x in (q, k, v):
        for b, n in enumerate(lens):
            x[b, :, n:] = float("nan")
    for layer in layers:
        used = {i for at in layer.at for i in at}
        rest = [i for i in range(layer.rows[0].shape[1]) if i not in used]
        if hasattr(layer, "pools"):
            for n, x in layer.pools.items():
                x.view(H, -1, x.shape[-1])[:, rest] = 255
        else:
            for x in layer.rows:
                x[:, rest] = float("inf")
    for a, layer in zip(want, layers):
        assert torch.equal(a, flash_attn_mlm_window(q, k, v, H, meta, 0.1, window=(50, 2), sinks=2,
                                                    inference_cache=layer.cache, layer_id=0))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 128, 256])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("kind", ["packed", "paged", None])
def test_values_that_are_not_finite_where_a_row_does_not_look(device, kind, bad, D):
    """Keys and values of the rows that no window of the checked rows reaches"""
    lens, N, H = [100], 100, 2
    ctx = [150] if kind else None
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 10)
    layer = _Layer(kind, "bf16", H, D, ctx, device, g) if kind else None
    first = ctx[0] if kind else 0
    run = lambda: flash_attn_mlm_window(q, k, v, H, meta, 0.1, window=(11, 4), sinks=3,  # noqa: E731
                                        inference_cache=layer.cache if kind else None, layer_id=0 if kind else None)
    spots = [first + 40, first + 41, first + 77] + ([90, 149] if kind else [])
    for s in spots:
        for rows, main in zip(layer.rows if kind else (None, None), (k, v)):
            if s >= first:
                main[0, :, s - first] = bad
            else:
                rows[:, layer.at[0][s]] = bad
    got = _f64(run()).reshape(H, 100, D)
    if kind:
        layer.read()
    clean = [i for i in range(100) if not any(first + i - 11 <= s <= first + i + 4 for s in spots)]
    dirty = [i for i in range(100) if i not in clean]
    assert len(clean) > 50 and np.isnan(got[:, dirty]).any(2).all()
    for h in range(H):
        kk, vv = _f64(k[0, h]), _f64(v[0, h])
        if kind:
            kk, vv = np.concatenate((layer.k[0][h], kk)), np.concatenate((layer.v[0][h], vv))
        seen = ref.visible(first, 100, len(kk), 11, 4, 3)[clean]
        o, P = ref.attend(_f64(q[0, h])[clean], kk, vv, seen, 0.1)
        size = P @ np.abs(np.where(np.isfinite(vv), vv, 0))
        assert (np.abs(got[h, clean] - o) <= (3 * _half("bf16") + 1e-4) * size).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["packed", "paged", "fp4", None])
@pytest.mark.parametrize("D", [64, 128])
def test_values_that_are_not_finite_under_long_windows(device, kind, D):
    """The same where tiles of rows are tall and waves pass tiles that their own rows do not see"""
    # (heads: calls of fewer workgroups take 64-row tiles in 16 bits)
    n, H, window, sinks = (150 if kind else 850), (2 if kind == "fp4" or D < 128 else 128 if kind else 74), (600, 4), 3
    g, q, k, v, meta = _inputs(device, "bf16", [n], n, H, D, 13)
    layer = _Layer(kind, "bf16", H, D, [700], device, g) if kind else None
    first = 700 if kind else 0
    run = lambda: flash_attn_mlm_window(q, k, v, H, meta, 0.1, window=window, sinks=sinks,  # noqa: E731
                                        inference_cache=layer.cache if kind else None, layer_id=0 if kind else None)
    out = run()
    _check(out[: 2 * n], q[:, :2], k[:, :2], v[:, :2], [n], [700], layer, window, sinks, 0.1, "bf16")
    spots = [first + 133] if kind else [40, 41, 845]
    if kind:
        behind = [layer.at[0][j] for j in (100, 101, 130)]
        if kind == "fp4":
            for name in ("k_scales", "v_scales"):
                layer.pools[name].view(H, -1, D // 32)[:, behind] = 255
        else:
            for x in layer.rows:
                x[:, behind] = float("inf")
        spots += [100, 101, 130]
    for s in spots:
        if s >= first:
            k[0, :, s - first] = v[0, :, s - first] = float("nan")
    clean = [i for i in range(n) if not any(first + i - 600 <= s <= first + i + 4 for s in spots)]
    assert len(clean) > 90
    got, was = (_f64(x).reshape(H, n, D) for x in (run(), out))
    for h in range(H):
        vv = _f64(v[0, h]) if layer is None else np.concatenate((layer.v[0][h], _f64(v[0, h])))
        # the same sums in another order at most: each is off by what _check allows
        size = np.abs(np.where(np.isfinite(vv), vv, 0)).max(0)
        assert (np.abs(got[h, clean] - was[h, clean]) <= 2 * (3 * _half("bf16") + 1e-4) * size).all()
    dirty = [i for i in range(n) if i not in clean]
    assert not np.isfinite(got[:, dirty]).all(2).any()


def _clean_rows(got, q, layer, k, v, first, clean, window, sinks, scale, dtype):
    """The rows ``clean`` of one sequence against the oracle, as _check does; k and v None: the context holds them"""
    for h in range(q.shape[1]):
        kk, vv = layer.k[0][h], layer.v[0][h]
        if k is not None:
            kk, vv = (np.concatenate((x, _f64(y[0, h]))) for x, y in ((kk, k), (vv, v)))
        seen = ref.visible(first, q.shape[2], len(kk), *window, sinks)[clean]
        o, P = ref.attend(_f64(q[0, h])[clean], kk, vv, seen, scale)
        size = P @ np.abs(np.where(np.isfinite(vv), vv, 0))
        assert (np.abs(got[h, clean] - o) <= (3 * _half(dtype) + 1e-4) * size + 2.0**-24 * len(kk)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("appended", [False, True])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("n", [1, 5, 16, 17])
def test_four_bit_values_that_are_not_finite_where_a_row_does_not_look(device, n, D, appended):
    """Rows of a 4-bit context whose scales are no numbers, in tiles that the window and the sinks cut, and new
    tokens that some rows do not see: calls of few rows (at most 16) and of more"""
    dtype, H, ctx, window, sinks = "bf16", 2, 700, (40, 2), 3
    g, q, k, v, meta = _inputs(device, dtype, [n], n, H, D, 15)
    layer = _Layer("fp4", dtype, H, D, [ctx], device, g)
    first = ctx - n if appended else ctx
    kv = (None, None) if appended else (k, v)
    run = lambda: flash_attn_mlm_window(q, *kv, H, meta, 0.1, window=window, sinks=sinks, inference_cache=layer.cache,  # noqa: E731
                                        layer_id=0)
    _check(run(), q, k, v, [n], [ctx], layer, window, sinks, 0.1, dtype, appended)
    for late in (False, True):
        # hidden from all rows: behind the sinks, in front of the band; then two that some rows see
        spots = [3, 40, first - 41, first - 60] + ([first - 38, first + 10] if late else [])
        for s in [s for s in spots if s < ctx]:
            for name in ("k_scales", "v_scales"):
                layer.pools[name].view(H, -1, D // 32)[:, layer.at[0][s]] = 255
        for s in [s for s in spots if ctx <= s < first + n]:
            k[0, :, s - first] = v[0, :, s - first] = float("nan")
        dirty = [i for i in range(n) if any(first + i - 40 <= s <= first + i + 2 and s < first + n for s in spots)]
        clean = [i for i in range(n) if i not in dirty]
        assert len(clean) == n if not late else len(dirty) > 0
        got = _f64(run()).reshape(H, n, D)
        assert not np.isfinite(got[:, dirty]).any()
        _clean_rows(got, q, layer, *kv, first, clean, window, sinks, 0.1, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("n", [5, 16])
def test_new_values_that_are_not_finite_beside_few_rows_over_four_bits(device, n, bad):
    """Only v of one new token, finite everywhere else: rows that see it get what it is"""
    dtype, H, D, ctx, window = "fp16", 2, 64, 130, (100, 0)
    g, q, k, v, meta = _inputs(device, dtype, [n], n, H, D, 16)
    layer = _Layer("fp4", dtype, H, D, [ctx], device, g)
    v[0, :, n - 2] = bad
    out = flash_attn_mlm_window(q, k, v, H, meta, 0.1, window=window, inference_cache=layer.cache, layer_id=0)
    got = _f64(out).reshape(H, n, D)
    _clean_rows(got, q, layer, k, v, ctx, list(range(n - 2)), window, 0, 0.1, dtype)
    assert (np.isnan(got[:, n - 2:]) if np.isnan(bad) else got[:, n - 2:] == bad).all()


@pytest.mark.gpu
def test_refusals_after_a_legal_call(device):
    """What equals a legal argument and is none is refused also when the legal one's call is kept"""
    _, q, k, v, meta = _inputs(device, "bf16", [3, 5], 5, 2, 64, 14)
    run = lambda H=2, **kw: flash_attn_mlm_window(q, k, v, H, meta, 0.1, **kw)  # noqa: E731
    run(window=(1, 0), sinks=1)
    for kw in (dict(window=(1.0, 0), sinks=1), dict(window=(1, False), sinks=1), dict(window=(1, 0), sinks=True),
               dict(window=(1, 0), sinks=1.0), dict(window=(1, 0), sinks=1, layer_id=0)):
        with pytest.raises(ValueError):
            run(**kw)
    with pytest.raises((TypeError, ValueError)):
        run(H=2.0, window=(1, 0), sinks=1)
    assert torch.equal(run(window=(1, 0), sinks=1), run(window=[1, 0], sinks=1))


@pytest.mark.gpu
def test_scores_of_infinite_size(device):
    """Scores far below the others, and the largest scores a type can make, in a row's last keys"""
    lens, N, H, D = [130], 130, 1, 64
    _, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 11)
    q[..., 0] = 3.0
    k[:, :, :, 0] = torch.linspace(-200, 200, N, device=device).bfloat16()
    out = flash_attn_mlm_window(q, k, v, H, meta, 1.0, window=(70, 1), sinks=1)
    kk, vv = _f64(k[0, 0]), _f64(v[0, 0])
    o, P = ref.attend(_f64(q[0, 0]), kk, vv, ref.visible(0, N, N, 70, 1, 1), 1.0)
    # scores to 620: fp32 sums are off by at most 64 2^-24 of the sum of the products' sizes, about 620
    size = P @ np.abs(vv)
    assert (np.abs(_f64(out) - o) <= (3 * _half("bf16") + 2 * 64 * 2.0**-24 * 650) * size).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["paged", "fp4", None])
def test_padded_outputs_and_whole_key_ranges(device, kind):
    """The C entry point with what the Python one does not ask for: a padded output, whose padding rows stay as they
    were, and key ranges that are not split"""
    from flash_mlm.host.window import _build

    lens, N, H, D = [3, 0, 5], 6, 2, 64
    ctx = [2500, 0, 300] if kind else None
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 45)
    layer = _Layer(kind, "bf16", H, D, ctx, device, g) if kind else None
    call, _rows = _build(q, k, v, H, meta, 0.15, 40, 2, 3, layer.cache.layer_entry(0) if kind else None, None)
    assert call.nbytes == 0  # a short window
    call, _rows = _build(q, k, v, H, meta, 0.15, -1, -1, 0, layer.cache.layer_entry(0) if kind else None, None)
    assert (call.nbytes > 0) == (kind is not None)
    p, lib = call.params, _lib.load()
    out = torch.full((len(lens), H, N, D), 7.0, dtype=q.dtype, device=device)
    p.q, p.k, p.v, p.o = (x.data_ptr() for x in (q, k, v, out))
    p.o_layout, p.o_sb, p.o_sh, p.o_sn = _lib.LAYOUT_PADDED, H * N * D, N * D, D
    ws = torch.empty(max(call.nbytes, 16), dtype=torch.uint8, device=device)
    p.workspace, p.workspace_bytes = ws.data_ptr(), call.nbytes
    for flags in (0, _lib.FLAG_NOSPLIT):
        p.flags = flags
        if flags:
            assert lib.fmlm_window_workspace_bytes(p, call.window) == 0
            p.workspace = None
        out.fill_(7)
        assert lib.fmlm_window_fwd(p, call.window, _lib.stream_of(device)) == 0
        _check(torch.cat([out[b, :, :n] for b, n in enumerate(lens)], 1).reshape(-1, D), q, k, v, lens, ctx, layer,
               (None, None), 0, 0.15, "bf16")
        for b, n in enumerate(lens):
            assert (out[b, :, n:] == 7).all()


@pytest.mark.gpu
def test_gradients_with_a_padded_output(device):
    """The C entry points of a training call with o, o_low and dout padded: the bits of the packed ones"""
    from flash_mlm.host.window import _build

    lens, N, H, D = [70, 0, 9], 71, 2, 64
    g, q, k, v, meta = _inputs(device, "fp16", lens, N, H, D, 46)
    xs = [x.requires_grad_() for x in (q, k, v)]
    packed = flash_attn_mlm_window(*xs, H, meta, 0.15, window=(20, 1), sinks=2)
    do = _rand(g, packed.shape, q.dtype)
    want = torch.autograd.grad(packed, xs, do)
    call, _rows = _build(*(x.detach() for x in xs), H, meta, 0.15, 20, 1, 2, None, None)
    p, w, gr, lib, stream = call.params, call.window, call.grads, _lib.load(), _lib.stream_of(device)
    out, low, dout = (torch.zeros_like(q) for _ in range(3))
    at = 0
    for b, n in enumerate(lens):
        dout[b, :, :n] = do.view(H, -1, D)[:, at:at + n]
        at += n
    lse, ws = torch.empty(H * at, device=device), torch.empty(H * at, device=device)
    p.q, p.k, p.v, p.o, p.lse, w.o_low = (x.data_ptr() for x in (q, k, v, out, lse, low))
    p.o_layout, p.o_sb, p.o_sh, p.o_sn = _lib.LAYOUT_PADDED, H * N * D, N * D, D
    assert lib.fmlm_window_fwd(p, w, stream) == 0
    assert torch.equal(torch.cat([out[b, :, :n] for b, n in enumerate(lens)], 1).reshape(-1, D), packed)
    grads = [torch.full_like(q, 7.0) for _ in range(3)]
    gr.dout, gr.workspace = dout.data_ptr(), ws.data_ptr()
    gr.dq, gr.dk, gr.dv = (x.data_ptr() for x in grads)
    gr.do_sb, gr.do_sh, gr.do_sn = H * N * D, N * D, D
    assert lib.fmlm_window_bwd(p, w, gr, stream) == 0
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


@pytest.mark.gpu
def test_calls_repeat_with_other_tensors(device):
    """A call laid out like an earlier one, other rows, another entry, other offsets"""
    lens, N, H, D, ctx = [3, 5], 6, 2, 64, [100, 200]
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 12)
    layer = _Layer("paged", "bf16", H, D, ctx, device, g)
    run = lambda a, b, c: flash_attn_mlm_window(a, b, c, H, meta, 0.125, window=(90, 0), sinks=4,  # noqa: E731
                                                inference_cache=layer.cache, layer_id=0)
    _check(run(q, k, v), q, k, v, lens, ctx, layer, (90, 0), 4, 0.125, "bf16")
    q2, k2, v2 = (_rand(g, q.shape, q.dtype) for _ in range(3))
    _check(run(q2, k2, v2), q2, k2, v2, lens, ctx, layer, (90, 0), 4, 0.125, "bf16")
    layer = _Layer("paged", "bf16", H, D, [64, 3], device, g)
    _check(run(q, k, v), q, k, v, lens, [64, 3], layer, (90, 0), 4, 0.125, "bf16")
    meta.cu_seqlens = torch.tensor([0, 5, 8], dtype=torch.int32, device=device)
    _check(run(q, k, v), q, k, v, [5, 3], [64, 3], layer, (90, 0), 4, 0.125, "bf16")
    index = torch.tensor([1, 0], device=device)
    out = flash_attn_mlm_window(q, k, v, H, meta, 0.125, window=(90, 0), sinks=4, inference_cache=layer.cache, layer_id=0,
                                context_index=index)
    _check(out, q, k, v, [5, 3], [64, 3], layer, (90, 0), 4, 0.125, "bf16", batch=[1, 0])


@pytest.mark.gpu
def test_entries_that_do_not_fit_are_refused(device):
    _, q, k, v, meta = _inputs(device, "bf16", [3], 3, 2, 64, 13)
    g = torch.Generator(device=device).manual_seed(0)
    for match, layer, a in [
        ("num_heads or head_dim", _Layer("paged", "bf16", 3, 64, [5], device, g), (q, k, v)),
        ("num_heads or head_dim", _Layer("fp4", "bf16", 2, 128, [5], device, g), (q, k, v)),
        ("dtype/device must match", _Layer("fp4", "fp16", 2, 64, [5], device, g), (q, k, v)),
        ("dtype/device must match", _Layer("packed", "fp16", 2, 64, [5], device, g), (q, k, v)),
    ]:
        with pytest.raises(ValueError, match=match):
            flash_attn_mlm_window(*a, 2, meta, 1.0, inference_cache=layer.cache, layer_id=0)
    for a in ((q, k, v), (q, None, None)):
        with pytest.raises(ValueError, match="context_index needs|must be in the layer"):
            flash_attn_mlm_window(*a, 2, meta, 1.0, inference_cache=InferenceCache(), layer_id=0,
                                  context_index=torch.zeros(1, dtype=torch.int32))
    # a layer without an entry has no context
    want = flash_attn_mlm_window(q, k, v, 2, meta, 1.0)
    assert torch.equal(want, flash_attn_mlm_window(q, k, v, 2, meta, 1.0, inference_cache=InferenceCache(), layer_id=0))


@pytest.mark.gpu
def test_no_tokens_and_empty_pools(device):
    _, q, k, v, meta = _inputs(device, "bf16", [0, 0], 4, 2, 64, 14)
    assert flash_attn_mlm_window(q, k, v, 2, meta, 1.0).shape == (0, 64)
    q.requires_grad_()
    assert flash_attn_mlm_window(q, k, v, 2, meta, 1.0).shape == (0, 64)
    g = torch.Generator(device=device).manual_seed(0)
    _, q, k, v, meta = _inputs(device, "bf16", [3, 1], 4, 2, 64, 14)
    for kind in ("packed", "paged", "fp4"):
        layer = _Layer(kind, "bf16", 2, 64, [0, 0], device, g, spare=0)
        out = flash_attn_mlm_window(q, k, v, 2, meta, 1.0, window=(1, 0), inference_cache=layer.cache, layer_id=0)
        assert torch.equal(out, flash_attn_mlm_window(q, k, v, 2, meta, 1.0, window=(1, 0)))
        assert not flash_attn_mlm_window(q, None, None, 2, meta, 1.0, inference_cache=layer.cache, layer_id=0).any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["paged", "fp4"])
def test_block_tables_without_columns(device, kind):
    """Contexts of no rows over a pool that has pages: before anyone's first token is stored"""
    g, q, k, v, meta = _inputs(device, "bf16", [3, 1], 4, 2, 64, 14)
    layer = _Layer(kind, "bf16", 2, 64, [70, 3], device, g)
    index = dict(block_table=torch.zeros((2, 0), dtype=torch.int32, device=device),
                 context_lens=torch.zeros(2, dtype=torch.int32, device=device), num_heads=2, head_dim=64)
    if kind == "fp4":
        layer.cache.prefill_paged_fp4_cache(0, **layer.pools, dtype=torch.bfloat16, **index)
    else:
        k_pages, v_pages = layer.cache.paged_kv_values(0)
        layer.cache.prefill_paged_kv_cache(0, k_pages=k_pages, v_pages=v_pages, is_mla=False, **index)
    run = lambda k, v, **kw: flash_attn_mlm_window(q, k, v, 2, meta, 1.0, window=(1, 0), **kw)  # noqa: E731
    assert torch.equal(run(k, v, inference_cache=layer.cache, layer_id=0), run(k, v))
    assert not run(None, None, inference_cache=layer.cache, layer_id=0).any()
    got = fm.flash_attn_mlm_compressed(q, k, v, 2, meta, 1.0, layer.cache, 0)
    want = flash_attn_mlm_window(q, k, v, 2, meta, 1.0)
    assert (got.float() - want.float()).abs().max() <= 8 * 2.0**-8 * want.float().abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_a_batch_without_tokens_has_gradients(device, packed):
    """Zeros, through the graph as those of any other batch"""
    _, q, k, v, meta = _inputs(device, "bf16", [0, 0], 4, 2, 64, 14)
    xs = [(x.view(-1, 64)[:0] if packed else x).clone().requires_grad_() for x in (q, k, v)]
    for leaves in ((0, 1, 2), (1,)):
        args = [x if i in leaves else x.detach() for i, x in enumerate(xs)]
        for _ in range(2):  # the second call is the kept one
            out = flash_attn_mlm_window(*args, 2, meta, 1.0, window=(3, 0), sinks=1)
            assert out.shape == (0, 64) and out.requires_grad
            grads = torch.autograd.grad(out.float().sum(), [xs[i] for i in leaves])
            assert all(g.shape == xs[0].shape and not g.any() for g in grads)
    with torch.no_grad():
        assert not flash_attn_mlm_window(*xs, 2, meta, 1.0).requires_grad


@pytest.mark.gpu
def test_metadata_that_contradicts_itself_stays_in_bounds(device):
    _, q, k, v, meta = _inputs(device, "bf16", [3, 1], 4, 2, 64, 15)
    g = torch.Generator(device=device).manual_seed(0)
    layer = _Layer("paged", "bf16", 2, 64, [90, 3], device, g)
    for cu in ([-(2**31), 2**31 - 1, 5], [5, 2, 9], [2**31 - 1, 3, 1]):
        meta.cu_seqlens = torch.tensor(cu, dtype=torch.int32, device=device)
        flash_attn_mlm_window(q, k, v, 2, meta, 1.0, window=(1, 0), inference_cache=layer.cache, layer_id=0)
        q.grad = None
        x = q.clone().requires_grad_()
        flash_attn_mlm_window(x, k, v, 2, meta, 1.0, window=(1, 0)).float().sum().backward()
    layer.cache.layer_entry(0).cu_seqlens_kv.copy_(torch.tensor([2**30, -5, 2**31 - 1], device=device))
    meta.cu_seqlens = torch.tensor([0, 3, 4], dtype=torch.int32, device=device)
    flash_attn_mlm_window(q, k, v, 2, meta, 1.0, window=(1, 0), inference_cache=layer.cache, layer_id=0)
    torch.cuda.synchronize()


# ---- gradients
def _grad_check(got, q, k, v, do, lens, window, sinks, scale, dtype):
    """Each gradient against the oracle's.  dS = P (dP - delta) scale is off by a rounding of its own and
    by delta's, which comes from a rounded output; dq and dk are rounded themselves, dv's P too:
      dq: h (2 |dS| |k| + delta's 1.5 h (|do| |o|) P |k| scale), dk alike, dv: h 2 P^T |do|,
    1e-4 of these for fp32's part, and fp16 below its normal range (2^-25 a value)."""
    h_, H, D = _half(dtype), q.shape[1], q.shape[-1]
    at = 0
    for b, n in enumerate(lens):
        for h in range(H):
            qq, kk, vv = (_f64(x[b, h, :n]) for x in (q, k, v))
            dd = do[h, at:at + n]
            seen = ref.visible(0, n, n, *window, sinks)
            o, P = ref.attend(qq, kk, vv, seen, scale)
            want = ref.attend_backward(qq, kk, vv, seen, scale, dd)
            dS = np.abs(P * (dd @ vv.T - (dd * o).sum(1)[:, None]) * scale)
            off = (1.5 * h_ * (np.abs(dd) * np.abs(o)).sum(1))[:, None] * P * abs(scale) + h_ * dS
            tiny = 2.0**-24 * abs(scale)
            tols = [off @ np.abs(kk) + h_ * np.abs(want[0]), off.T @ np.abs(qq) + h_ * np.abs(want[1]),
                    h_ * (P.T @ np.abs(dd) + np.abs(want[2]))]
            sizes = [dS @ np.abs(kk), dS.T @ np.abs(qq), P.T @ np.abs(dd)]
            more = [np.abs(kk).sum(0), np.abs(qq).sum(0), np.abs(dd).sum(0)]
            for name, x, y, tol, size, m in zip("qkv", got, want, tols, sizes, more):
                err = np.abs(x[b][h] - y)
                lim = tol + 2e-4 * size + tiny * m + 2.0**-25
                assert (err <= lim).all(), (name, b, h, (err / lim).max())
        at += n


def _by_sequence(x, lens, H, D):
    """64-bit gradients [b][h] of padded or packed rows; padding rows must be zero"""
    if x.ndim == 4:
        for b, n in enumerate(lens):
            assert not x[b, :, n:].any()
        return [_f64(x[b, :, :n]) for b, n in enumerate(lens)]
    x = _f64(x).reshape(H, -1, D)
    cu = np.cumsum([0] + list(lens))
    return [x[:, cu[b]:cu[b + 1]] for b in range(len(lens))]


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS, ids=str)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype,D", [("bf16", 32), ("fp16", 32), ("bf16", 64), ("fp16", 64), ("bf16", 128), ("fp16", 128),
                                     ("bf16", 256), ("fp16", 256)])
def test_gradients(device, dtype, D, packed, window, sinks):
    lens, N, H = [1, 0, 150, 64], 151, 2
    g, q, k, v, meta = _inputs(device, dtype, lens, N, H, D, 21)
    leaves = [q, k, v]
    if packed:
        leaves = [torch.cat([x[b, :, :n] for b, n in enumerate(lens)], 1).reshape(-1, D) for x in leaves]
    for x in leaves:
        x.requires_grad_()
    out = flash_attn_mlm_window(*leaves, H, meta, 0.15, window=window, sinks=sinks)
    do = _rand(g, out.shape, out.dtype)
    _check(out, q, k, v, lens, None, None, window, sinks, 0.15, dtype)
    grads = torch.autograd.grad(out, leaves, do, retain_graph=True)
    got = [_by_sequence(x, lens, H, D) for x in grads]
    _grad_check(got, q, k, v, _f64(do).reshape(H, -1, D), lens, window, sinks, 0.15, dtype)
    again = torch.autograd.grad(out, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("left,right", [(1, 0), (8, 0), (40, 0), (None, 0), (2, None)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_gradients_of_queries_that_see_few_keys(device, dtype, left, right, D):
    """dq's root mean square error is that of its own rounding and of the forward's rounded probabilities in delta,
    simulated here: dS brings no further one (rounded to the type it adds a third).  The roundings are of other
    mantissas than the simulation's and a quarter of the error comes from rows of few keys: 10%."""
    n, H, scale = 300, 16, D**-0.5
    g, q, k, v, meta = _inputs(device, dtype, [n], n, H, D, 36)
    q.requires_grad_()
    out = flash_attn_mlm_window(q, k, v, H, meta, scale, window=(left, right))
    do = _rand(g, out.shape, out.dtype)
    got = _f64(torch.autograd.grad(out, q, do)[0][0])
    low = lambda x: _f64(torch.from_numpy(x).to(TYPES[dtype]))  # noqa: E731
    seen, err, ideal = ref.visible(0, n, n, left, right, 0), 0.0, 0.0
    for h, dd in enumerate(_f64(do).reshape(H, n, D)):
        qq, kk, vv = (_f64(x[0, h]) for x in (q, k, v))
        want = ref.attend_backward(qq, kk, vv, seen, scale, dd)[0]
        z = np.where(seen, qq @ kk.T * scale, -np.inf)
        P = np.exp(z - z.max(1, keepdims=True))
        rounded = low(P)
        delta = (dd * (rounded @ vv / rounded.sum(1, keepdims=True))).sum(1, keepdims=True)
        dS = P / P.sum(1, keepdims=True) * (dd @ vv.T - delta) * scale
        err += ((got[h] - want) ** 2).sum()
        ideal += ((low(dS @ kk) - want) ** 2).sum()
    assert err <= 1.1**2 * ideal, (err / ideal) ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_gradients_of_keys_and_values_that_few_share(device, dtype, D):
    """dk's and dv's root mean square errors over windows of four keys are those of P and dS rounded to the type and
    of their own rounding: the row statistics bring no further one (that of the forward's rounded P adds 7%).  The
    roundings are the simulation's own but for fp32's part; 4% as for the keys above."""
    n, H, scale, window, sinks = 600, 16, D**-0.5, (2, 0), 1
    g, q, k, v, meta = _inputs(device, dtype, [n], n, H, D, 37)
    k.requires_grad_()
    v.requires_grad_()
    out = flash_attn_mlm_window(q, k, v, H, meta, scale, window=window, sinks=sinks)
    do = _rand(g, out.shape, out.dtype)
    got = [_f64(x)[0] for x in torch.autograd.grad(out, (k, v), do)]
    low = lambda x: _f64(torch.from_numpy(x).to(TYPES[dtype]))  # noqa: E731
    seen, err, ideal = ref.visible(0, n, n, *window, sinks), np.zeros(2), np.zeros(2)
    for h, dd in enumerate(_f64(do).reshape(H, n, D)):
        qq, kk, vv = (_f64(x[0, h]) for x in (q, k, v))
        _, dk, dv = ref.attend_backward(qq, kk, vv, seen, scale, dd)
        o, P = ref.attend(qq, kk, vv, seen, scale)
        dS = P * (dd @ vv.T - (dd * o).sum(1)[:, None])
        for i, (want, best) in enumerate(((dk, low(low(dS).T @ qq * scale)), (dv, low(low(P).T @ dd)))):
            err[i] += ((got[i][h] - want) ** 2).sum()
            ideal[i] += ((best - want) ** 2).sum()
    assert (err <= 1.04**2 * ideal).all(), (err / ideal) ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0**-10, 2.0**9])
@pytest.mark.parametrize("D", [32, 128])
def test_gradients_of_small_and_large_losses_in_fp16(device, D, size):
    """dS is an fp16 operand: its normal range holds losses scaled by hundreds either way"""
    lens, N, H = [90, 33], 90, 2
    g, q, k, v, meta = _inputs(device, "fp16", lens, N, H, D, 35)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = flash_attn_mlm_window(*leaves, H, meta, D**-0.5, window=(20, 3), sinks=2)
    do = _rand(g, out.shape, torch.float32).mul_(size).to(out.dtype)
    got = [_by_sequence(x, lens, H, D) for x in torch.autograd.grad(out, leaves, do)]
    _grad_check(got, q, k, v, _f64(do).reshape(H, -1, D), lens, (20, 3), 2, D**-0.5, "fp16")


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_gradients_with_other_scales(device, D, scale):
    """Negative scales turn the masks' infinities round, 0 leaves dv alone"""
    lens, N, H = [70, 0, 33], 70, 2
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 34)
    leaves = [(x if scale < 1 else x * 0.3).requires_grad_() for x in (q, k, v)]
    q, k, v = leaves
    out = flash_attn_mlm_window(*leaves, H, meta, scale, window=(20, 3), sinks=2)
    _check(out, q, k, v, lens, None, None, (20, 3), 2, scale, "bf16")
    do = _rand(g, out.shape, out.dtype)
    got = [_by_sequence(x, lens, H, D) for x in torch.autograd.grad(out, leaves, do)]
    _grad_check(got, q, k, v, _f64(do).reshape(H, -1, D), lens, (20, 3), 2, scale, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_gradients_of_keys_are_as_exact_as_their_operands(device, dtype):
    """dK's root mean square error is that of dS rounded to the type, and of its own rounding: delta brings no
    further one (that of the forward's rounded P adds 6%).  Over 100 thousand values a root mean square is
    within 1% of its expectation, the rounding of the same values by the same rule; 4% leave fp32's part room."""
    n, H, D, scale = 200, 16, 32, 32**-0.5
    g, q, k, v, meta = _inputs(device, dtype, [n], n, H, D, 33)
    k.requires_grad_()
    out = flash_attn_mlm_window(q, k, v, H, meta, scale, window=(103, 0))
    do = _rand(g, out.shape, out.dtype)
    got = _f64(torch.autograd.grad(out, k, do)[0][0])
    low = lambda x: _f64(torch.from_numpy(x).to(TYPES[dtype]))  # noqa: E731
    seen, err, ideal = ref.visible(0, n, n, 103, 0, 0), 0.0, 0.0
    for h, dd in enumerate(_f64(do).reshape(H, n, D)):
        qq, kk, vv = (_f64(x[0, h]) for x in (q, k, v))
        o, P = ref.attend(qq, kk, vv, seen, scale)
        dS = P * (dd @ vv.T - (dd * o).sum(1)[:, None])
        want = dS.T @ qq * scale
        err += ((got[h] - want) ** 2).sum()
        ideal += ((low(low(dS).T @ qq * scale) - want) ** 2).sum()
    assert err <= 1.04**2 * ideal, (err / ideal) ** 0.5


@pytest.mark.gpu
def test_gradients_against_differences(device):
    """Directional differences of the 64-bit forward at the very inputs, in fp16"""
    lens, N, H, D, window, sinks = [40, 9], 40, 2, 64, (6, 2), 3
    g, q, k, v, meta = _inputs(device, "fp16", lens, N, H, D, 22)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = flash_attn_mlm_window(*leaves, H, meta, 0.2, window=window, sinks=sinks)
    do = _rand(g, out.shape, out.dtype)
    grads = [_f64(x) for x in torch.autograd.grad(out, leaves, do)]
    dd, rng = _f64(do).reshape(H, -1, D), np.random.default_rng(1)
    base = [_f64(x) for x in leaves]

    def f(args):
        s, at = 0.0, 0
        for b, n in enumerate(lens):
            for h in range(H):
                o = ref.attend(*(x[b, h, :n] for x in args), ref.visible(0, n, n, *window, sinks), 0.2)[0]
                s += (o * dd[h, at:at + n]).sum()
            at += n
        return s

    for i in range(3):
        for _ in range(3):
            d = rng.standard_normal(base[i].shape)
            move = lambda e: [x + e * d if j == i else x for j, x in enumerate(base)]  # noqa: E731
            diff = (f(move(1e-4)) - f(move(-1e-4))) / 2e-4
            # each gradient entry is off by a few roundings of independent sign (2^-11 each)
            assert abs(diff - (grads[i] * d).sum()) <= 6 * 4 * 2.0**-11 * np.sqrt((grads[i] ** 2).sum()) + 1e-4


@pytest.mark.gpu
def test_gradients_of_strided_shared_and_repeated_leaves(device):
    lens, N, H, D = [30, 7], 30, 3, 64
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 23)
    run = lambda q, k, v: flash_attn_mlm_window(q, k, v, H, meta, 0.125, window=(9, 2), sinks=1)  # noqa: E731
    do = _rand(g, (H * sum(lens), D), q.dtype)
    leaf = lambda x: x.detach().clone().requires_grad_()  # noqa: E731
    # heads that share their rows: the gradient is the heads' sum
    one = leaf(k[:, :1])
    full = leaf(k[:, :1].expand(-1, H, -1, -1))
    a, = torch.autograd.grad(run(q, one.expand(-1, H, -1, -1), v), one, do)
    b, = torch.autograd.grad(run(q, full, v), full, do)
    assert (a.float() - b.float().sum(1, keepdim=True)).abs().max() <= 4 * 2.0**-8 * b.float().abs().sum(1).max()
    # one tensor as q, k and v
    x = leaf(q)
    a, = torch.autograd.grad(run(x, x, x), x, do)
    xs = [leaf(q) for _ in range(3)]
    parts = torch.autograd.grad(run(*xs), xs, do)
    assert (a.float() - sum(p.float() for p in parts)).abs().max() <= 4 * 2.0**-8 * sum(p.float().abs() for p in parts).max()
    # other strides, and a gradient that is no contiguous tensor
    t = [leaf(x.transpose(1, 2).contiguous()) for x in (q, k, v)]
    wide = torch.zeros((H * sum(lens), 2 * D), dtype=q.dtype, device=device)
    wide[:, :D] = do
    got = torch.autograd.grad(run(*(x.transpose(1, 2) for x in t)), t, wide[:, :D])
    xs = [leaf(x) for x in (q, k, v)]
    want = torch.autograd.grad(run(*xs), xs, do)
    assert all(torch.equal(x.transpose(1, 2), y) for x, y in zip(got, want))
    # a gradient for one of them only
    got, = torch.autograd.grad(run(q, xs[1], v), xs[1], do)
    assert torch.equal(got, want[1])


@pytest.mark.gpu
def test_gradient_refusals(device):
    g, q, k, v, meta = _inputs(device, "bf16", [5, 2], 5, 2, 64, 24)
    layer = _Layer("paged", "bf16", 2, 64, [9, 70], device, g)
    x = q.clone().requires_grad_()
    run = lambda q: flash_attn_mlm_window(q, k, v, 2, meta, 0.1, inference_cache=layer.cache, layer_id=0)  # noqa: E731
    want = run(q)
    with pytest.raises(ValueError, match="no backward over a cached context"):
        run(x)
    with torch.no_grad():
        assert torch.equal(run(x), want)
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level():
        with pytest.raises(ValueError, match="no forward-mode"):
            run(fwd.make_dual(q, torch.ones_like(q)))
    out = flash_attn_mlm_window(x, k, v, 2, meta, 0.1)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(out.float().sum(), x, create_graph=True)[0].float().sum(), x)
    out = flash_attn_mlm_window(x, k, v, 2, meta, 0.1)
    with torch.no_grad():
        k.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.float().sum().backward()
    layer.rows[0].requires_grad_()
    pages = layer.rows[0].view(2, -1, PAGE, 64)
    layer.cache.prefill_paged_kv_cache(0, k_pages=pages, v_pages=pages.detach(),
                                       block_table=torch.zeros((2, 2), dtype=torch.int32),
                                       context_lens=torch.tensor([9, 70]), is_mla=False, num_heads=2, head_dim=64)
    with pytest.raises(ValueError, match="no gradient of a cached context"):
        run(q)


@pytest.mark.gpu
def test_checkpoints_and_saved_tensor_hooks(device):
    from torch.utils.checkpoint import checkpoint

    g, q, k, v, meta = _inputs(device, "bf16", [33, 2], 33, 2, 64, 25)
    xs = [x.requires_grad_() for x in (q, k, v)]
    run = lambda *a: flash_attn_mlm_window(*a, 2, meta, 0.1, window=(5, 1), sinks=2)  # noqa: E731
    do = _rand(g, (70, 64), q.dtype)
    want = torch.autograd.grad(run(*xs), xs, do)
    got = torch.autograd.grad(checkpoint(run, *xs, use_reentrant=False), xs, do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    swap = lambda x: x.transpose(0, -1).contiguous() if x.ndim == 4 else x.clone()  # noqa: E731
    back = lambda x: x.transpose(0, -1) if x.ndim == 4 else x  # noqa: E731
    with torch.autograd.graph.saved_tensors_hooks(swap, back):
        out = run(*xs)
    got = torch.autograd.grad(out, xs, do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_offsets_changed_between_forward_and_backward(device):
    g, q, k, v, meta = _inputs(device, "bf16", [3, 2], 3, 2, 64, 25)
    q.requires_grad_()
    run = lambda: flash_attn_mlm_window(q, k, v, 2, meta, 0.1)  # noqa: E731
    run().float().sum().backward()
    out = run()
    meta.cu_seqlens.copy_(torch.tensor([0, 2, 5], device=device))
    with pytest.raises(RuntimeError, match="cu_seqlens has been modified"):
        out.float().sum().backward()
    run().float().sum().backward()  # a new forward has the new offsets


@pytest.mark.gpu
def test_hooks_that_bring_other_tensors_are_refused(device):
    g, q, k, v, meta = _inputs(device, "bf16", [33, 2], 33, 2, 64, 25)
    q.requires_grad_()
    for back in (lambda x: x.cpu(), lambda x: x.to(torch.float8_e4m3fn), lambda x: x[:1], lambda x: x.view(-1)):
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, back):
            out = flash_attn_mlm_window(q, k, v, 2, meta, 0.1)
        with pytest.raises(RuntimeError, match="saved tensor came back"):
            out.float().sum().backward()
    assert q.grad is None


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["paged", "fp4", None])
def test_calls_in_a_graph(device, kind):
    """Two captured calls, replayed on other rows and lengths with eager work in between"""
    lens, N, H, D = [4, 70], 70, 2, 64
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 26)
    layer = _Layer(kind, "bf16", H, D, [2000, 300], device, g) if kind else None
    run = lambda: [flash_attn_mlm_window(q, k, v, H, meta, 0.1, window=w, sinks=3, inference_cache=layer.cache if kind else None,  # noqa: E731
                                         layer_id=0 if kind else None) for w in ((None, None), (90, 0))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i in range(4):
        for x in (q, k, v):
            x.normal_()
        if kind:
            layer.cache.layer_entry(0).cu_seqlens_kv.copy_(torch.tensor([0, 500 * i, 500 * i + 60 * i], device=device))
        graph.replay()
        got = [x.clone() for x in outs]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run()))


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 7])
@pytest.mark.parametrize("kind", ["paged", "fp4"])
def test_split_calls_in_two_graphs(device, kind, N):
    """Two graphs of calls whose key ranges are split, replayed in turn on other rows and lengths: records of their own"""
    lens, H, D = [N, 1], 2, 128
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 27)
    layer = _Layer(kind, "bf16", H, D, [3000, 2000], device, g)
    q2 = _rand(g, q.shape, q.dtype)
    run = lambda x: flash_attn_mlm_window(x, k, v, H, meta, 0.1, inference_cache=layer.cache, layer_id=0)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(q)
    torch.cuda.current_stream().wait_stream(side)
    assert _kept_bytes(meta) > 0
    graphs, outs = [], []
    for x in (q, q2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(x))
        graphs.append(graph)
    for i in range(4):
        for x in (q, q2, k, v):
            x.normal_()
        layer.cache.layer_entry(0).cu_seqlens_kv.copy_(torch.tensor([0, 900 * i, 900 * i + 600 * i], device=device))
        for j in (i & 1, 1 - (i & 1)):
            graphs[j].replay()
        got = [x.clone() for x in outs]
        torch.cuda.synchronize()
        assert all(torch.equal(a, run(x)) for a, x in zip(got, (q, q2)))


@pytest.mark.gpu
def test_training_in_a_graph(device):
    lens, N, H, D = [4, 70], 70, 2, 64
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 27)
    xs = [x.requires_grad_() for x in (q, k, v)]
    do = _rand(g, (H * 74, D), q.dtype)
    run = lambda: torch.autograd.grad(flash_attn_mlm_window(*xs, H, meta, 0.1, window=(9, 3), sinks=2), xs, do)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = run()
    for _ in range(4):
        with torch.no_grad():
            for x in (*xs, do):
                x.normal_()
        graph.replay()
        got = [x.clone() for x in grads]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run()))


@pytest.mark.gpu
def test_a_capture_refuses_leaves_of_a_living_graph(device):
    g, q, k, v, meta = _inputs(device, "bf16", [4], 4, 2, 64, 28)
    q.requires_grad_()
    run = lambda: flash_attn_mlm_window(q, k, v, 2, meta, 0.1)  # noqa: E731
    alive = run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    refused = None
    with torch.cuda.graph(graph):
        try:
            run()
        except ValueError as e:
            refused = str(e)
        x = torch.zeros(1, device=device)  # (a capture of something)
    assert refused is not None and "flash_attn_mlm_window is being captured" in refused
    assert alive.requires_grad


@pytest.mark.gpu
def test_streams(device):
    """Calls at once on two streams, split ones with records of their own"""
    lens, N, H, D = [1, 2], 2, 4, 128
    g, q, k, v, meta = _inputs(device, "bf16", lens, N, H, D, 29)
    layer = _Layer("fp4", "bf16", H, D, [3000, 2500], device, g)
    qs = [_rand(g, q.shape, q.dtype) for _ in range(2)]
    run = lambda x: fm.flash_attn_mlm_compressed(x, k, v, H, meta, 0.1, layer.cache, 0)  # noqa: E731
    want = [run(x) for x in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for s, x, o in zip(streams, qs, outs):
            with torch.cuda.stream(s):
                o.append(run(x))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for o, w in zip(outs, want) for y in o)


# ---- as a server runs them
@pytest.mark.gpu
@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("window,sinks", [((None, 0), 0), ((40, 0), 3)])
def test_a_server_step_by_step(device, fp4, window, sinks):
    """Conversations of three requests: every step's new tokens (a prompt, then few) are given slots,
    rotated and stored, and attend causally over the pages"""
    H, D, dtype = 2, 64, "fp16"
    dt, B, scale = TYPES[dtype], 3, 0.125
    steps = [[70, 5, 0], [1, 1, 66], [1, 0, 1], [3, 62, 1], [1, 1, 1]]
    g = torch.Generator(device=device).manual_seed(31)
    P = 9
    cache = InferenceCache()
    lens = torch.zeros(B, dtype=torch.int32, device=device)
    table = torch.full((B, 3), -1, dtype=torch.int32, device=device)
    free = torch.randperm(P, generator=g, device=device).to(torch.int32)
    if fp4:
        pools = {n: torch.zeros((H, P, PAGE, c), dtype=torch.uint8, device=device)
                 for n, c in (("k_pages", D // 2), ("k_scales", D // 32), ("v_pages", D // 2), ("v_scales", D // 32))}
        cache.prefill_paged_fp4_cache(0, **pools, block_table=table, context_lens=lens, num_heads=H, head_dim=D, dtype=dt)
    else:
        cache.prefill_paged_kv_cache(0, k_pages=torch.zeros((H, P, PAGE, D), dtype=dt, device=device),
                                     v_pages=torch.zeros((H, P, PAGE, D), dtype=dt, device=device), block_table=table,
                                     context_lens=lens, is_mla=False, num_heads=H, head_dim=D)
    ang = torch.arange(200, dtype=torch.float64)[:, None] * 1000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    cos, sin = ang.cos().float().to(device), ang.sin().float().to(device)
    ks, vs, old = [np.zeros((H, 0, D)) for _ in range(B)], [np.zeros((H, 0, D)) for _ in range(B)], [0] * B
    for new in steps:
        N = max(new)
        meta = build_pack_metadata(torch.tensor(new, device=device), N, 32)
        q, k, v = (_rand(g, (B, H, N, D), dt) for _ in range(3))
        plan = build_block_table(meta, lens, free_pages=free, block_table=table)
        rq = cache.append_paged_kv_cache(0, k=k, v=v, q_meta=meta, plan=plan, q=q, cos=cos, sin=sin)
        out = flash_attn_mlm_window(rq, None, None, H, meta, scale, window=window, sinks=sinks, inference_cache=cache, layer_id=0)
        lens, table, free = plan.context_lens, plan.block_table, free[plan.pages_taken:]
        got, at = _f64(out).reshape(H, -1, D), 0
        for b, n in enumerate(new):
            pos = np.arange(old[b], old[b] + n)
            c, s = _f64(cos)[pos], _f64(sin)[pos]
            rk, rv = ref.rotate(_f64(k[b, :, :n]), c, s, False), _f64(v[b, :, :n])
            if fp4:
                rk, rv = (ref.fp4_values(*ref.fp4_encode(x, dtype)) for x in (rk, rv))
            ks[b], vs[b] = np.concatenate((ks[b], rk), 1), np.concatenate((vs[b], rv), 1)
            rq64 = ref.rotate(_f64(q[b, :, :n]), c, s, False)
            for h in range(H):
                seen = ref.visible(old[b], n, ks[b].shape[1], *window, sinks)
                o, P_ = ref.attend(rq64[h], ks[b][h], vs[b][h], seen, scale)
                # q's and (16 bits) k's roundings move a score by at most 2 h sum |q k| scale and
                # tilt the probabilities by e^(twice that) - 1; then as in _check
                hh = _half(dtype)
                move = 2 * hh * (np.abs(rq64[h]) @ np.abs(ks[b][h]).T).max(1, initial=0.0) * scale
                tol = (3 * hh + 1e-4 + 2.1 * move[:, None]) * (P_ @ np.abs(vs[b][h])) + 2.0**-24 * 200
                assert (np.abs(got[h, at:at + n] - o) <= tol).all()
            at += n
            old[b] += n
    assert lens.tolist() == old
