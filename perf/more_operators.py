"""A server of long conversations, and the training of its attention, as cases that can be
timed and checked.

A step of such a server rotates the new queries and keys while it stores keys and values in
the pages of a cache, in 16 or in 4 bits, and attends over the pages, to a window of recent
tokens and a few first ones (sinks) or to all of them.  Training runs the same window over
whole sequences.  A case is one pass through one of these operators.

Ways (``case["way"]``):
  append  new queries rotated, keys rotated and stored, values stored in a paged context
          (``fp4``: in 4 bits, and the pages read back as values)
  attn    attention of new tokens over a cached context (``kind``: pages in 16 bits, pages in
          4 bits, packed rows), within a window or over all of it
  train   window attention of whole sequences and its gradients

With ``own`` false, ``run`` computes a pass in plain torch; with ``own`` true it calls the
framework.  ``exact`` restates a case at 64 bits.

4-bit rows: E2M1 codes, two a byte (low half first), and for every 32 values of a row a scale
2^e as the byte e + 127.  e is the smallest integer with which the largest magnitude is below
7 * 2^e (it rounds to at most 6), within the range in which the row's type holds every value.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_PAGE = 64
_BLOCK = 32
_SCALES = {"bf16": (-125, 125), "fp16": (-23, 13)}  # exponents whose values the type holds
_FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _fm():
    pkg = str(Path(__file__).resolve().parent.parent / "flash-mlm_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import flash_mlm

    return flash_mlm


def _case(c, name):
    if name is not None:
        c["name"] = name
    return c


def _append(dtype, B, H, N, D, *, lo, R, fp4=False, ctx=0, packed=False, interleaved=False, lens=0, name=None):
    """lo: shortest sequence (the longest is N); R: rotated dims; ctx: positions start at up to ctx."""
    return _case(dict(way="append", dtype=dtype, B=B, H=H, N=N, D=D, lo=lo, R=R, fp4=fp4, ctx=ctx, packed=packed,
                      interleaved=interleaved, lens=lens), name)


def _attn(dtype, kind, B, H, N, D, *, lo, ctx_lo, ctx_hi, left=-1, right=-1, sinks=0, appended=False, lens=0,
          name=None):
    """left, right: the window (-1: no limit); appended: the new tokens are the context's last rows
    already."""
    return _case(dict(way="attn", dtype=dtype, kind=kind, B=B, H=H, N=N, D=D, lo=lo, ctx_lo=ctx_lo, ctx_hi=ctx_hi,
                      left=left, right=right, sinks=sinks, appended=appended, lens=lens), name)


def _train(dtype, B, H, N, D, *, lo, left, right, sinks=0, packed=False, lens=0, name=None):
    return _case(dict(way="train", dtype=dtype, B=B, H=H, N=N, D=D, lo=lo, left=left, right=right, sinks=sinks,
                      packed=packed, lens=lens), name)


def listed():
    return [
        # one new token of each of 64 users (the smallest): latency
        _append("bf16", 64, 16, 1, 128, lo=1, R=128, ctx=6000, name="append_bf16_decode"),
        # a ragged batch of prompts is stored
        _append("fp16", 32, 16, 1024, 128, lo=256, R=128, lens=3, name="append_fp16_prompts"),
        # a few new tokens of 24 users are stored in 4 bits
        _append("bf16", 24, 16, 16, 128, lo=1, R=128, fp4=True, ctx=6000, lens=5, name="append4_bf16_serving"),
        # a ragged batch of prompts is stored in 4 bits, half of the dims rotated
        _append("bf16", 32, 12, 1024, 64, lo=256, R=32, fp4=True, lens=3, name="append4_bf16_prompts"),
        # one user's next token over a long document in 4 bits: latency
        _attn("bf16", "fp4", 1, 16, 1, 128, lo=1, ctx_lo=8000, ctx_hi=8000, name="attn4_bf16_one"),
        # the next tokens of 64 users over long contexts in 4 bits
        _attn("bf16", "fp4", 64, 16, 1, 128, lo=1, ctx_lo=500, ctx_hi=8192, lens=5, name="attn4_bf16_serving"),
        # parts of four prompts over what is stored of them in 4 bits
        _attn("fp16", "fp4", 4, 16, 512, 128, lo=300, ctx_lo=2000, ctx_hi=4000, lens=7, name="attn4_fp16_chunks"),
        # the next tokens of 64 users, stored before, within a window of long contexts
        _attn("bf16", "paged", 64, 16, 1, 128, lo=1, ctx_lo=2000, ctx_hi=8192, left=1023, right=0, sinks=4,
              appended=True, lens=5, name="window_bf16_decode"),
        # parts of eight prompts, causal within a window
        _attn("fp16", "paged", 8, 16, 1024, 128, lo=400, ctx_lo=500, ctx_hi=4000, left=511, right=0, sinks=4, lens=7,
              name="window_fp16_chunks"),
        # masked-language-model training with local attention both ways, ragged batch
        _train("bf16", 32, 12, 512, 64, lo=64, left=64, right=64, sinks=1, lens=10, name="train_bf16_mlm"),
        # training on long packed documents, causal (the most arithmetic)
        _train("fp16", 4, 16, 4096, 128, lo=2000, left=1023, right=0, sinks=4, packed=True, lens=3,
               name="train_fp16_long"),
        # wide heads
        _train("bf16", 8, 8, 1024, 256, lo=300, left=255, right=255, lens=11, name="train_bf16_wide"),
    ]


def draw(rng: random.Random):
    def size(lo, hi):  # spread over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    way = rng.choice(["append", "append", "attn", "attn", "attn", "train", "train"])
    lens = rng.randrange(1 << 30)
    dtype = rng.choice(["bf16", "fp16"])
    H = rng.choice([4, 8, 12, 16])
    D = rng.choice([32, 64, 64, 128, 128, 256])
    if way == "append":
        N = size(1, 64) if rng.random() < 0.5 else size(16, 1024)
        B = min(size(1, 128), max(1, (32 * 1024 * 16 * 128 - 1) // (N * H * D)))
        return _append(dtype, B, H, N, D, lo=rng.randint(0, N), R=rng.choice([D, D, D // 2]), fp4=rng.random() < 0.5,
                       ctx=rng.choice([0, size(1, 8192)]), packed=rng.random() < 0.4, interleaved=rng.random() < 0.3,
                       lens=lens)
    left = rng.choice([-1, size(1, 2048), size(1, 2048)])
    right = rng.choice([-1, 0, 0, size(1, 512)])
    sinks = rng.choice([0, 1, 4, size(1, 128)])
    if way == "attn":
        kind = rng.choice(["fp4", "fp4", "paged", "packed"])
        N = rng.choice([1, size(1, 64), size(1, 1024)])
        B = min(size(1, 64), max(1, 4096 // N))
        c0 = min(size(32, 4096), max(32, 262144 // B))
        if D == 256:
            c0 = min(c0, 2048)
        return _attn(dtype, kind, B, H, N, D, lo=rng.randint(1, N), ctx_lo=c0, ctx_hi=rng.randint(c0, 2 * c0),
                     left=left, right=right, sinks=sinks, appended=rng.random() < 0.4, lens=lens)
    N = size(16, 2048)
    B = min(size(1, 32), max(1, 8192 * 128 // (N * max(D, 128))))
    return _train(dtype, B, H, N, D, lo=rng.randint(1, N), left=left, right=right, sinks=sinks,
                  packed=rng.random() < 0.4, lens=lens)


# ---------------------------------------------------------------------------
# sizes and inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    r = random.Random(case["lens"])
    lens = [r.randint(case["lo"], case["N"]) for _ in range(case["B"])]
    return [max(lens[0], 1)] + lens[1:]


def _contexts(case):
    """context rows of each sequence (with its new tokens where they are stored already)"""
    r = random.Random(case["lens"] + 1)
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["B"])]
    return [c + n for c, n in zip(ctx, _lengths(case))] if case["appended"] else ctx


def _pages(n):
    return (n + _PAGE - 1) // _PAGE


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rand(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _where(lens):
    """(sequence, position in it) of every packed token"""
    b = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    start = torch.cumsum(torch.tensor([0] + lens), 0)
    return b.cuda(), (torch.arange(sum(lens)) - start[b]).cuda()


def _encode(x, dtype):
    """(codes, scales) of rows x (32 or 64 bits, finite) in 4 bits"""
    lo, hi = _SCALES[dtype]
    blocks = x.unflatten(-1, (-1, _BLOCK))
    m, k = torch.frexp(blocks.abs().amax(-1))  # in [1/2, 1) and its exponent
    e = torch.where(m == 0, lo, torch.where(m < 0.875, k - 3, k - 2)).clamp(lo, hi)
    y = torch.ldexp(blocks.abs(), -e[..., None].to(torch.int32))
    # borders between the codes; halfway goes to the even code
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=x.dtype, device=x.device)
    down = torch.nextafter(mids, torch.zeros_like(mids))
    border = torch.where(torch.arange(7, device=x.device) % 2 == 1, down, mids)
    code = torch.bucketize(y, border).to(torch.uint8) | (torch.signbit(blocks).to(torch.uint8) << 3)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _decode(codes, scales, dtype):
    """the values of 4-bit rows, in dtype"""
    code = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    table = torch.tensor(_FP4 + tuple(-v for v in _FP4), dtype=torch.float32, device=codes.device)
    x = table[code.int()].unflatten(-1, (-1, _BLOCK))
    return torch.ldexp(x, scales[..., None].to(torch.int32) - 127).flatten(-2).to(dtype)


def prepare(case, seed):
    g, way = _gen(seed), case["way"]
    lens = _lengths(case)
    s = dict(case=case, lens=lens, T=sum(lens))
    s["b"], s["p"] = _where(lens)
    s["lengths"] = _ints(lens)
    if own:
        s["fm"] = _fm()
        s["meta"] = s["fm"].build_pack_metadata(s["lengths"], case["N"], 32)
    r = random.Random(seed)
    if way == "append":
        _prepare_append(s, case, g, r)
    elif way == "attn":
        _prepare_attn(s, case, g, r)
    else:
        _prepare_train(s, case, g)
    return s


def _prepare_append(s, case, g, r):
    B, H, N, D, R, T = case["B"], case["H"], case["N"], case["D"], case["R"], s["T"]
    dt = _DTYPES[case["dtype"]]
    shape = (H * T, D) if case["packed"] else (B, H, N, D)
    s["q"], s["k"], s["v"] = (_rand(g, shape, dt) for _ in range(3))
    # the new tokens follow up to two pages of rows, and the pool has room for just that; positions
    # go on from where a longer conversation is
    old = [r.randint(0, 2 * _PAGE) for _ in range(B)]
    need = [_pages(o + n) for o, n in zip(old, s["lens"])]
    P = sum(_pages(2 * _PAGE + n) for n in s["lens"]) + 3
    ids = list(range(P))
    r.shuffle(ids)
    slots, table, width, at = [], [], max(need + [1]), 0
    for o, n, m in zip(old, s["lens"], need):
        mine = ids[at:at + m]
        at += m
        table.append(mine + [-1] * (width - m))
        slots += [mine[(o + i) // _PAGE] * _PAGE + (o + i) % _PAGE for i in range(n)]
    s["slots"], s["table"], s["old"] = _ints(slots, torch.int64), _ints(table), _ints(old)
    first = _ints([r.randint(0, case["ctx"]) for _ in range(B)], torch.int64)
    s["positions"] = (first[s["b"]] + s["p"]).to(torch.int32)
    freq = 10000.0 ** (-torch.arange(0, R // 2, dtype=torch.float64, device="cuda") * 2 / R)
    ang = torch.arange(N + case["ctx"] + 1, dtype=torch.float64, device="cuda")[:, None] * freq
    s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    for name in ("k", "v"):
        rows = _rand(g, (H, P, _PAGE, D), dt)
        if case["fp4"]:
            s[name + "_pages"], s[name + "_scales"] = _encode(rows.float(), case["dtype"])
        else:
            s[name + "_pages"] = rows
    if own:
        fm = s["fm"]
        s["cache"] = fm.InferenceCache()
        if case["fp4"]:
            s["cache"].prefill_paged_fp4_cache(0, k_pages=s["k_pages"], k_scales=s["k_scales"], v_pages=s["v_pages"],
                                               v_scales=s["v_scales"], block_table=s["table"], context_lens=s["old"],
                                               num_heads=H, head_dim=D, dtype=dt)
        else:
            s["cache"].prefill_paged_kv_cache(0, k_pages=s["k_pages"], v_pages=s["v_pages"], block_table=s["table"],
                                              context_lens=s["old"], is_mla=False, num_heads=H, head_dim=D)
        new = s["old"] + s["lengths"]
        cu = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
        cu[1:] = torch.cumsum(new, 0)
        s["plan"] = fm.PagedMetadata(block_table=s["table"], slot_mapping=s["slots"], positions=s["positions"],
                                     context_lens=new, cu_seqlens_kv=cu)


def _prepare_attn(s, case, g, r):
    B, H, N, D, kind = case["B"], case["H"], case["N"], case["D"], case["kind"]
    dt = _DTYPES[case["dtype"]]
    ctx = s["ctx"] = _contexts(case)
    s["scale"] = 1.0 / math.sqrt(D)
    s["q"] = _rand(g, (B, H, N, D), dt)
    s["k"], s["v"] = (None, None) if case["appended"] else (_rand(g, (B, H, N, D), dt) for _ in range(2))
    if kind == "packed":
        C = sum(ctx)
        s["k_ctx"], s["v_ctx"] = (_rand(g, (H, C, D), dt) for _ in range(2))
        s["rows"] = [torch.arange(sum(ctx[:b]), sum(ctx[:b + 1]), device="cuda") for b in range(B)]
    else:
        P = sum(_pages(n) for n in ctx) + 3
        for name in ("k", "v"):
            rows = _rand(g, (H, P, _PAGE, D), dt)
            if kind == "fp4":
                codes, scales = zip(*(_encode(x.float(), case["dtype"]) for x in rows))  # a head at a time
                s[name + "_pages"], s[name + "_scales"] = torch.stack(codes), torch.stack(scales)
            else:
                s[name + "_pages"] = rows
                s[name + "_ctx"] = rows.view(H, P * _PAGE, D)
        ids = list(range(P))
        r.shuffle(ids)
        width, at, table, s["rows"] = max(_pages(n) for n in ctx), 0, [], []
        for n in ctx:
            mine = ids[at:at + _pages(n)]
            at += len(mine)
            table.append(mine + [-1] * (width - len(mine)))
            j = torch.arange(n, device="cuda")
            s["rows"].append(_ints(mine, torch.int64)[j // _PAGE] * _PAGE + j % _PAGE)
        s["table"] = _ints(table)
    if own:
        s["cache"] = s["fm"].InferenceCache()
        if kind == "packed":
            cu = [sum(ctx[:b]) for b in range(B + 1)]
            s["cache"].prefill_kv_cache(0, k_cache=s["k_ctx"].view(-1, D), v_cache=s["v_ctx"].view(-1, D),
                                        total_context_len=cu[-1], cu_seqlens_kv=_ints(cu), context_batch_size=B,
                                        is_mla=False, num_heads=H, head_dim=D)
        elif kind == "fp4":
            s["cache"].prefill_paged_fp4_cache(0, k_pages=s["k_pages"], k_scales=s["k_scales"], v_pages=s["v_pages"],
                                               v_scales=s["v_scales"], block_table=s["table"], context_lens=_ints(ctx),
                                               num_heads=H, head_dim=D, dtype=dt)
        else:
            s["cache"].prefill_paged_kv_cache(0, k_pages=s["k_pages"], v_pages=s["v_pages"], block_table=s["table"],
                                              context_lens=_ints(ctx), is_mla=False, num_heads=H, head_dim=D)


def _prepare_train(s, case, g):
    B, H, N, D, T = case["B"], case["H"], case["N"], case["D"], s["T"]
    dt = _DTYPES[case["dtype"]]
    shape = (H * T, D) if case["packed"] else (B, H, N, D)
    s["scale"] = 1.0 / math.sqrt(D)
    s["q"], s["k"], s["v"] = (_rand(g, shape, dt) for _ in range(3))
    s["dout"] = _rand(g, (H * T, D), dt)
    if own:
        for name in ("q", "k", "v"):
            s[name].requires_grad_()


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    way = s["case"]["way"]
    if way == "append":
        return _own_append(s) if own else _plain_append(s)
    if way == "attn":
        return _own_attn(s) if own else _plain_attn(s)
    return _own_train(s) if own else _plain_train(s)


def _window(c):
    return tuple(None if c[n] < 0 else c[n] for n in ("left", "right"))


def _own_append(s):
    c = s["case"]
    q = s["cache"].append_paged_kv_cache(0, k=s["k"], v=s["v"], q_meta=s["meta"], plan=s["plan"], q=s["q"],
                                         cos=s["cos"], sin=s["sin"], interleaved=c["interleaved"])
    if c["fp4"]:
        return [q, *s["cache"].paged_kv_values(0)]
    return [q, s["k_pages"], s["v_pages"]]


def _own_attn(s):
    c = s["case"]
    if c["kind"] == "fp4" and c["left"] < 0 and c["right"] < 0 and not c["appended"]:
        return s["fm"].flash_attn_mlm_compressed(s["q"], s["k"], s["v"], c["H"], s["meta"], s["scale"], s["cache"], 0)
    return s["fm"].flash_attn_mlm_window(s["q"], s["k"], s["v"], c["H"], s["meta"], s["scale"], window=_window(c),
                                         sinks=c["sinks"], inference_cache=s["cache"], layer_id=0)


def _own_train(s):
    c = s["case"]
    out = s["fm"].flash_attn_mlm_window(s["q"], s["k"], s["v"], c["H"], s["meta"], s["scale"], window=_window(c),
                                        sinks=c["sinks"])
    return [out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])]


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = rot[..., :half], rot[..., half:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((y, rest), dim=-1)


def _plain_append(s):
    """keys in 64 bits where they are stored in 4: a value next to a border of two codes"""
    c = s["case"]
    H, D, T = c["H"], c["D"], s["T"]

    def tokens(x):  # [H, T, D]
        return x.view(H, T, D) if c["packed"] else x[s["b"], :, s["p"]].transpose(0, 1)

    cos, sin = s["cos"][s["positions"].long()], s["sin"][s["positions"].long()]
    y = _plain_rotate(tokens(s["q"]).float(), cos, sin, c["interleaved"]).to(s["q"].dtype)
    if c["packed"]:
        q = y.reshape(H * T, D)
    else:
        q = torch.zeros_like(s["q"])
        q[s["b"], :, s["p"]] = y.transpose(0, 1)
    wide = torch.float64 if c["fp4"] else torch.float32
    k = _plain_rotate(tokens(s["k"]).to(wide), cos.to(wide), sin.to(wide), c["interleaved"])
    out = [q]
    for x, name in ((k, "k"), (tokens(s["v"]), "v")):
        pages = s[name + "_pages"]
        if c["fp4"]:
            scales = s[name + "_scales"]
            codes, sc = _encode(x if name == "k" else x.float(), c["dtype"])
            pages.view(H, -1, D // 2)[:, s["slots"]] = codes
            scales.view(H, -1, D // _BLOCK)[:, s["slots"]] = sc
            pages = _decode(pages, scales, s["q"].dtype)
        else:
            pages.view(H, -1, D)[:, s["slots"]] = x.to(pages.dtype)
        out.append(pages)
    return out


def _visible(c, first, n, total, device="cuda"):
    """[n, total]: which keys the queries at positions first .. first + n see"""
    p = torch.arange(first, first + n, device=device)[:, None]
    j = torch.arange(total, device=device)[None]
    seen = torch.ones(n, total, dtype=torch.bool, device=device)
    if c["right"] >= 0:
        seen &= j <= p + c["right"]
    if c["left"] >= 0:
        seen &= (j >= p - c["left"]) | (j < c["sinks"])
    return seen


def _context(s, name, b):
    """context rows of sequence b, [H, rows, D]"""
    rows, D = s["rows"][b], s["case"]["D"]
    if s["case"]["kind"] == "fp4":
        H = s["case"]["H"]
        codes = s[name + "_pages"].view(H, -1, D // 2)[:, rows]
        return _decode(codes, s[name + "_scales"].view(H, -1, D // _BLOCK)[:, rows], torch.float32)
    return s[name + "_ctx"][:, rows].float()


def _softmax_product(q, k, v, seen, scale):
    z = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
    z = z.masked_fill(~seen, -math.inf)
    e = torch.exp(z - z.amax(-1, keepdim=True))
    return torch.matmul(e / e.sum(-1, keepdim=True), v)


def _plain_attn(s):
    c = s["case"]
    H, D = c["H"], c["D"]
    out = torch.empty(H, s["T"], D, dtype=s["q"].dtype, device="cuda")
    at = 0
    for b, n in enumerate(s["lens"]):
        if n == 0:
            continue
        k, v = _context(s, "k", b), _context(s, "v", b)
        first = s["ctx"][b]
        if c["appended"]:
            first -= n
        else:
            k = torch.cat((k, s["k"][b, :, :n].float()), 1)
            v = torch.cat((v, s["v"][b, :, :n].float()), 1)
        seen = _visible(c, first, n, k.shape[1])
        out[:, at:at + n] = _softmax_product(s["q"][b, :, :n].float(), k, v, seen, s["scale"]).to(out.dtype)
        at += n
    return out.view(H * s["T"], D)


def _plain_train(s):
    c = s["case"]
    H, D, T = c["H"], c["D"], s["T"]
    dt = s["q"].dtype
    out = torch.empty(H, T, D, dtype=dt, device="cuda")
    grads = [torch.zeros_like(s[n]) for n in ("q", "k", "v")]
    at = 0
    for b, n in enumerate(s["lens"]):
        if n == 0:
            continue
        pick = (lambda x: x.view(H, T, D)[:, at:at + n]) if c["packed"] else (lambda x: x[b, :, :n])
        leaves = [pick(s[name]).float().requires_grad_() for name in ("q", "k", "v")]
        o = _softmax_product(*leaves, _visible(c, 0, n, n), s["scale"])
        out[:, at:at + n] = o.detach().to(dt)
        for whole, part in zip(grads, torch.autograd.grad(o, leaves, s["dout"].view(H, T, D)[:, at:at + n].float())):
            pick(whole).copy_(part.to(dt))
        at += n
    return [out.view(H * T, D), *grads]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _pairs(case, first, n, total):
    """(pairs that attend, keys that anyone sees)"""
    left, right, sinks = case["left"], case["right"], case["sinks"]
    pairs, low, high = 0, total, 0
    for p in range(first, first + n):
        hi = total if right < 0 else min(total, p + right + 1)
        lo = 0 if left < 0 else min(max(0, p - left), hi)
        pairs += hi - lo + min(sinks, lo)
        low, high = min(low, lo), max(high, hi)
    return pairs, high - low + min(sinks, low)


def work(case):
    lens = _lengths(case)
    T, way, H, D = sum(lens), case["way"], case["H"], case["D"]
    row4 = D // 2 + D // _BLOCK
    if way == "append":
        whole = H * (T if case["packed"] else case["B"] * case["N"]) * D * 2
        n = 3 * H * T * D * 2 + whole + 8 * T + 4 * T + 4 * T * case["R"]
        if case["fp4"]:  # rows stored, then the pages read and their values written
            P = sum(_pages(2 * _PAGE + m) for m in lens) + 3
            n += 2 * H * T * row4 + 2 * H * P * _PAGE * (row4 + 2 * D)
        else:
            n += 2 * H * T * D * 2
        return {"bytes": n, "flops": 3 * 2 * H * T * case["R"]}
    if way == "train":
        pairs = sum(_pairs(case, 0, n, n)[0] for n in lens)
        rows = 4 if case["packed"] else 3 * case["B"] * case["N"] / T + 1  # padded gradients are written whole
        return {"bytes": int((4 + rows) * H * T * D * 2), "flops": 14 * H * D * pairs}
    pairs = keys = 0
    for n, c in zip(lens, _contexts(case)):
        a, k = _pairs(case, c - n, n, c) if case["appended"] else _pairs(case, c, n, c + n)
        pairs, keys = pairs + a, keys + (k if case["appended"] else max(k - n, 0))
    n = 2 * H * keys * (row4 if case["kind"] == "fp4" else 2 * D) + (2 if case["appended"] else 4) * H * T * D * 2
    return {"bytes": n, "flops": 4 * H * D * pairs}


# ---------------------------------------------------------------------------
# the definitions at 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["way"] == "append":
        return _exact_append(s)
    return _exact_attn(s) if case["way"] == "attn" else _exact_train(s)


def _exact_code(x, dtype):
    """the nearest 4-bit values to x [..., 32 n], by distance to each of the eight magnitudes"""
    lo, hi = _SCALES[dtype]
    blocks = x.unflatten(-1, (-1, _BLOCK))
    top = blocks.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, lo)
    for k in range(lo, hi):  # the smallest exponent with top < 7 * 2^e
        e = torch.where(top >= 7 * 2.0**k, k + 1.0, e)
    y = blocks.abs() / torch.exp2(e)
    best, gap = torch.zeros_like(y), y.clone()
    for i, v in enumerate(_FP4[1:], 1):
        d = (y - v).abs()
        take = d <= gap if i % 2 == 0 else d < gap  # halfway: the even code
        best, gap = torch.where(take, v, best), torch.where(take, d, gap)
    return (torch.copysign(best, blocks) * torch.exp2(e)).flatten(-2)


def _exact_values(codes, scales):
    """64-bit values of 4-bit rows, half by half"""
    out = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=codes.device)
    mags = torch.tensor(_FP4, dtype=torch.float64, device=codes.device)
    for half, shift in ((0, 0), (1, 4)):
        c = (codes.int() >> shift) & 15
        out[..., half::2] = torch.where(c >= 8, -1.0, 1.0) * mags[c & 7]
    return out * torch.exp2(scales.double() - 127).repeat_interleave(_BLOCK, -1)


def _exact_append(s):
    """every token's rotation as a complex product, the pages a slot at a time"""
    c = s["case"]
    H, D, R, T = c["H"], c["D"], c["R"], s["T"]
    pos = s["positions"].long()
    cos, sin = s["cos"].double()[pos], s["sin"].double()[pos]

    def tokens(x):  # [T, H, D]
        x = x.double()
        return x.view(H, T, D).permute(1, 0, 2) if c["packed"] else x[s["b"], :, s["p"]]

    def rotate(y):
        y = y.clone()
        ia, ib = (slice(0, R, 2), slice(1, R, 2)) if c["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        a, b = y[..., ia].clone(), y[..., ib].clone()
        y[..., ia] = a * cos[:, None] - b * sin[:, None]
        y[..., ib] = a * sin[:, None] + b * cos[:, None]
        return y

    yq = rotate(tokens(s["q"]))
    if c["packed"]:
        q = yq.permute(1, 0, 2).reshape(H * T, D)
    else:
        q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        q[s["b"], :, s["p"]] = yq
    out = [q]
    for name, x in (("k", rotate(tokens(s["k"]))), ("v", tokens(s["v"]))):
        pages = s[name + "_pages"]
        if c["fp4"]:
            values = _exact_values(pages, s[name + "_scales"])
            x = torch.stack([_exact_code(x[:, h], c["dtype"]) for h in range(H)], 1)
        else:
            values = pages.double()
        for h in range(H):
            values[h].view(-1, D).index_copy_(0, s["slots"], x[:, h].contiguous())
        out.append(values)
    return out


def _exact_rows(q, k, v, c, first, scale):
    """(output, P) of one head's rows"""
    z = (q @ k.T) * scale
    z = torch.where(_visible(c, first, q.shape[0], k.shape[0]), z, torch.full_like(z, -math.inf))
    lse = torch.logsumexp(z, 1, keepdim=True)
    P = torch.exp(z - lse)
    return P @ v, P


def _exact_attn(s):
    c = s["case"]
    H, D = c["H"], c["D"]
    out = torch.empty(H, s["T"], D, dtype=torch.float64, device="cuda")
    at = 0
    for b, n in enumerate(s["lens"]):
        rows = s["rows"][b]
        for h in range(H):
            if c["kind"] == "fp4":
                k, v = (_exact_values(s[x + "_pages"][h].view(-1, D // 2)[rows],
                                      s[x + "_scales"][h].view(-1, D // _BLOCK)[rows]) for x in "kv")
            else:
                k, v = (s[x + "_ctx"][h].index_select(0, rows).double() for x in "kv")
            first = s["ctx"][b]
            if c["appended"]:
                first -= n
            else:
                k, v = (torch.cat((y, s[x][b, h, :n].double())) for x, y in (("k", k), ("v", v)))
            out[h, at:at + n] = _exact_rows(s["q"][b, h, :n].double(), k, v, c, first, s["scale"])[0]
        at += n
    return out.view(H * s["T"], D)


def _exact_train(s):
    c = s["case"]
    H, D, T = c["H"], c["D"], s["T"]
    out = torch.empty(H, T, D, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda") for _ in range(3)]
    at = 0
    for b, n in enumerate(s["lens"]):
        for h in range(H):
            def pick(x):
                return x.view(H, T, D)[h, at:at + n] if c["packed"] else x[b, h, :n]

            q, k, v = (pick(s[x]).double() for x in "qkv")
            do = s["dout"].view(H, T, D)[h, at:at + n].double()
            o, P = _exact_rows(q, k, v, c, 0, s["scale"])
            out[h, at:at + n] = o
            dS = P * (do @ v.T - (do * o).sum(1, keepdim=True)) * s["scale"]
            for whole, part in zip(grads, (dS @ k, dS.T @ q, P.T @ do)):
                pick(whole).copy_(part)
        at += n
    return [out.view(H * T, D), *grads]
