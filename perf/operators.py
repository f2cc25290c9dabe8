"""The operators around a paged context, as cases that can be timed and checked.

One serving step over a paged cache normalises and rotates the new queries and keys, gives
the new tokens their pages and slots, attends, and stores the new keys and values; its
first part is also what training runs in every layer.  A case is one pass through one of
these operators.

Ways (``case["way"]``):
  norm    RMS norms of queries and keys for each head, with the position rotation
  train   the same and its gradients (of q, k and both gains)
  table   block table, slots and positions of a step's new tokens, from request lengths
          (``tree``: the ancestor masks of its drafted tokens too)
  append  the new keys and values written to their slots of a paged pool
  tree    attention of a tree of drafted tokens over a paged (fp32: packed) context

With ``own`` false, ``run`` computes a pass in plain torch; with ``own`` true it calls the
framework.  ``exact`` restates a case at 64 bits.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_PAGE = 64
_EPS = 1e-6


def _fm():
    pkg = str(Path(__file__).resolve().parent.parent / "flash-mlm_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import flash_mlm

    return flash_mlm


def _norm(way, dtype, B, H, N, D, *, lo, R, Hk=0, packed=False, interleaved=False, gain="shared", ctx=0, lens=0,
          name=None):
    """lo: shortest sequence (the longest is N); R: rotated dims; Hk: key heads (0: H); packed:
    [H*T, D] rows instead of [B, H, N, D]; gain: "shared" [D] or "head" [H, D]; ctx: positions
    start at up to ctx."""
    c = dict(way=way, dtype=dtype, B=B, H=H, N=N, D=D, lo=lo, R=R, Hk=Hk or H, packed=packed,
             interleaved=interleaved, gain=gain, ctx=ctx, lens=lens)
    if name is not None:
        c["name"] = name
    return c


def _table(B, N, *, lo, ctx, keep=False, tree=False, lens=0, name=None):
    """ctx: longest context before the step; keep: only some of the new tokens are stored."""
    c = dict(way="table", B=B, N=N, lo=lo, ctx=ctx, keep=keep, tree=tree, lens=lens)
    if name is not None:
        c["name"] = name
    return c


def _append(dtype, B, H, N, D, *, lo, packed=False, mla=False, keep=False, lens=0, name=None):
    c = dict(way="append", dtype=dtype, B=B, H=H, N=N, D=D, lo=lo, packed=packed, mla=mla, keep=keep, lens=lens)
    if name is not None:
        c["name"] = name
    return c


def _tree(dtype, B, H, N, D, *, lo, ctx_lo, ctx_hi, mla=False, lens=0, name=None):
    c = dict(way="tree", dtype=dtype, B=B, H=H, N=N, D=D, lo=lo, ctx_lo=ctx_lo, ctx_hi=ctx_hi, mla=mla, lens=lens)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one new token for each of 64 users, between two matrix products: latency
        _norm("norm", "bf16", 64, 16, 1, 128, lo=1, R=128, ctx=6000, name="norm_bf16_decode"),
        # a ragged batch of prompts is taken in
        _norm("norm", "fp16", 32, 16, 1024, 128, lo=256, R=128, lens=3, name="norm_fp16_prompts"),
        # masked-language-model training, ragged batch; the largest pass over rows is below
        _norm("train", "bf16", 32, 12, 512, 64, lo=64, R=64, lens=10, name="train_bf16_mlm"),
        # training on packed rows, a gain for each head, half of the dims rotated
        _norm("train", "fp16", 32, 16, 1024, 128, lo=256, R=64, packed=True, gain="head", lens=3,
              name="train_fp16_packed"),
        # single-precision training with neighbouring pairs
        _norm("train", "fp32", 8, 12, 512, 64, lo=64, R=64, interleaved=True, lens=11, name="train_fp32"),
        # one new token for each of 64 users (the smallest)
        _table(64, 1, lo=1, ctx=6000, name="table_decode"),
        # many users verify drafted trees: accepted tokens get slots, the next trees their masks
        _table(512, 32, lo=1, ctx=8192, keep=True, tree=True, lens=5, name="table_drafts"),
        # a few new tokens of 24 users are stored
        _append("bf16", 24, 16, 16, 128, lo=1, lens=5, name="append_bf16_serving"),
        # a ragged batch of prompts is stored
        _append("fp16", 32, 16, 1024, 128, lo=256, lens=3, name="append_fp16_prompts"),
        # one user's drafts against a long document: latency
        _tree("bf16", 1, 16, 32, 128, lo=32, ctx_lo=8000, ctx_hi=8000, name="tree_bf16_one"),
        # drafts of 24 users with long contexts of their own
        _tree("bf16", 24, 16, 64, 128, lo=1, ctx_lo=500, ctx_hi=6000, lens=5, name="tree_bf16_serving"),
        # MLA: drafts of 16 users, 64 query heads over one cached latent (the most arithmetic)
        _tree("bf16", 16, 64, 16, 512, lo=1, ctx_lo=1000, ctx_hi=8192, mla=True, lens=7, name="tree_bf16_mla"),
    ]


def draw(rng: random.Random):
    def size(lo, hi):  # spread over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    way = rng.choice(["norm", "norm", "train", "train", "table", "table", "append", "append", "tree", "tree", "tree"])
    lens = rng.randrange(1 << 30)
    H = rng.choice([4, 8, 12, 16])
    if way in ("norm", "train"):
        D = rng.choice([32, 64, 64, 128, 128, 256])
        N = size(1, 64) if way == "norm" and rng.random() < 0.5 else size(16, 1024)
        B = min(size(1, 128), max(1, (32 * 1024 * 16 * 128 - 1) // (N * H * D)))
        return _norm(way, rng.choice(["bf16", "fp16", "fp32"] if way == "train" else ["bf16", "bf16", "fp16", "fp32"]),
                     B if D < 256 else min(B, 32), H, N, D, lo=rng.randint(1, N), R=rng.choice([D, D, D // 2]),
                     Hk=rng.choice([H, H, max(1, H // 4), 1]), packed=rng.random() < 0.4,
                     interleaved=rng.random() < 0.3, gain=rng.choice(["shared", "shared", "head"]),
                     ctx=rng.choice([0, size(1, 8192)]), lens=lens)
    if way == "table":
        N = size(1, 1024)
        B = min(size(1, 512), max(1, 32768 // N))
        return _table(B, N, lo=rng.randint(0, N), ctx=size(1, 8192), keep=rng.random() < 0.5,
                      tree=N <= 256 and rng.random() < 0.5, lens=lens)
    if way == "append":
        mla = rng.random() < 0.2
        D = 512 if mla else rng.choice([32, 64, 64, 128, 128, 256])
        N = size(1, 64) if rng.random() < 0.5 else size(16, 1024)
        B = min(size(1, 128), max(1, (32 * 1024 * 16 * 128 - 1) // (N * H * D)))
        return _append(rng.choice(["bf16", "fp16"]), B, H, N, D, lo=rng.randint(0, N), packed=rng.random() < 0.4,
                       mla=mla, keep=rng.random() < 0.3, lens=lens)
    mla = rng.random() < 0.25
    if mla:
        N = size(1, 16)
        lo = rng.randint(300, 4000)
        return _tree(rng.choice(["bf16", "fp16"]), rng.randint(1, 16), rng.choice([16, 32, 64]), N, 512,
                     lo=rng.randint(1, N), ctx_lo=lo, ctx_hi=rng.randint(lo, 8192), mla=True, lens=lens)
    N = size(1, 256)
    B = min(size(1, 32), max(1, 2048 // N))
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    D = rng.choice([32, 64, 128, 128, 256])
    c0 = size(32, 4096 if D < 256 else 2048)
    if dtype == "fp32":
        B, c0 = min(B, 8), min(c0, 1024)
    return _tree(dtype, B, H, N, D, lo=rng.randint(1, N), ctx_lo=c0, ctx_hi=rng.randint(c0, c0 + c0 // 2), lens=lens)


# ---------------------------------------------------------------------------
# sizes and inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    r = random.Random(case["lens"])
    lens = [r.randint(case["lo"], case["N"]) for _ in range(case["B"])]
    return [max(lens[0], 1)] + lens[1:]


def _contexts(case):
    r = random.Random(case["lens"] + 1)
    return [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["B"])]


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


def _parents(r, lens):
    """a random tree for each sequence: a chain with branches, roots -1"""
    out = []
    for n in lens:
        out += [-1 if i == 0 or r.random() < 0.05 else (i - 1 if r.random() < 0.5 else r.randrange(i)) for i in range(n)]
    return out


def prepare(case, seed):
    g, way = _gen(seed), case["way"]
    lens = _lengths(case)
    T = sum(lens)
    s = dict(case=case, lens=lens, T=T)
    s["b"], s["p"] = _where(lens)
    s["lengths"] = _ints(lens)
    if own:
        s["fm"] = _fm()
        s["meta"] = s["fm"].build_pack_metadata(s["lengths"], case["N"], 32)
    r = random.Random(seed)
    if way in ("norm", "train"):
        _prepare_norm(s, case, g, r)
    elif way == "table":
        _prepare_table(s, case, r)
    elif way == "append":
        _prepare_append(s, case, g, r)
    else:
        _prepare_tree(s, case, g, r)
    return s


def _prepare_norm(s, case, g, r):
    B, H, Hk, N, D, R = (case[k] for k in ("B", "H", "Hk", "N", "D", "R"))
    T = s["T"]
    dt = _DTYPES[case["dtype"]]
    rows = (lambda h: (h * T, D)) if case["packed"] else (lambda h: (B, h, N, D))
    s["q"], s["k"] = _rand(g, rows(H), dt), _rand(g, rows(Hk), dt) * 2
    gain = (lambda h: (h, D)) if case["gain"] == "head" else (lambda h: (D,))
    s["wq"], s["wk"] = ((1 + 0.1 * _rand(g, gain(h), torch.float32)).to(dt) for h in (H, Hk))
    starts = [r.randint(0, case["ctx"]) for _ in range(B)]
    s["start"] = _ints(starts)
    n = case["N"] + case["ctx"] + 1
    freq = 10000.0 ** (-torch.arange(0, R // 2, dtype=torch.float64, device="cuda") * 2 / R)
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * freq
    s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    if case["way"] == "train":
        s["dq"], s["dk"] = _rand(g, rows(H), dt), _rand(g, rows(Hk), dt)
        if own:
            for name in ("q", "k", "wq", "wk"):
                s[name].requires_grad_()


def _prepare_table(s, case, r):
    B, N, ctx, T = case["B"], case["N"], case["ctx"], s["T"]
    old = [r.randint(0, ctx) for _ in range(B)]
    width = _pages(ctx + N)
    ids = list(range(B * width + 7))
    r.shuffle(ids)
    table, at = [], 0
    for n in old:
        have = _pages(n)
        table.append(ids[at:at + have] + [-1] * (width - have))
        at += have
    s["old"], s["table"], s["free"] = _ints(old), _ints(table), _ints(ids[at:])
    s["width"] = width
    s["keep"] = torch.tensor([r.random() < 0.6 for _ in range(T)], dtype=torch.bool, device="cuda") if case["keep"] else None
    s["parents"] = _ints(_parents(r, s["lens"])) if case["tree"] else None


def _prepare_append(s, case, g, r):
    B, H, N, D, T, mla = case["B"], case["H"], case["N"], case["D"], s["T"], case["mla"]
    dt = _DTYPES[case["dtype"]]
    Hk = 1 if mla else H
    shape = (Hk * T, D) if case["packed"] else (B, H, N, D)
    s["k"] = _rand(g, shape, dt)
    s["v"] = None if mla else _rand(g, shape, dt)
    # the new tokens follow contexts of up to two pages, and the pool has room for just that
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
        keep = [not case["keep"] or r.random() < 0.6 for _ in range(n)]
        a = o
        for kept in keep:
            slots.append(mine[a // _PAGE] * _PAGE + a % _PAGE if kept else -1)
            a += kept
    s["slots"], s["table"], s["old"] = _ints(slots, torch.int64), _ints(table), _ints(old)
    s["k_pages"] = _rand(g, (Hk, P, _PAGE, D), dt)
    s["v_pages"] = None if mla else _rand(g, (Hk, P, _PAGE, D), dt)
    if own:
        fm = s["fm"]
        s["cache"] = fm.InferenceCache()
        s["cache"].prefill_paged_kv_cache(0, k_pages=s["k_pages"], v_pages=s["v_pages"], block_table=s["table"],
                                          context_lens=s["old"], is_mla=mla, num_heads=H, head_dim=D)
        cu = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
        new = s["old"] + s["lengths"]
        cu[1:] = torch.cumsum(new, 0)
        s["plan"] = fm.PagedMetadata(block_table=s["table"], slot_mapping=s["slots"], positions=None,
                                     context_lens=new, cu_seqlens_kv=cu)


def _prepare_tree(s, case, g, r):
    B, H, N, D, mla = case["B"], case["H"], case["N"], case["D"], case["mla"]
    dt = _DTYPES[case["dtype"]]
    Hk = 1 if mla else H
    ctx = _contexts(case)
    s["ctx"] = ctx
    s["scale"] = 1.0 / math.sqrt(D)
    s["q"] = _rand(g, (B, H, N, D), dt)
    s["k"] = _rand(g, (B, H, N, D), dt)
    s["v"] = s["k"] if mla else _rand(g, (B, H, N, D), dt)
    s["parents"] = _ints(_parents(r, s["lens"]))
    # which tokens of its own sequence each token sees
    seen = torch.zeros(B, N, N, dtype=torch.bool)
    at, host = 0, s["parents"].tolist()
    for b, n in enumerate(s["lens"]):
        for i in range(n):
            if host[at + i] >= 0:
                seen[b, i] = seen[b, host[at + i]]
            seen[b, i, i] = True
        at += n
    s["seen"] = seen.cuda()
    if case["dtype"] == "fp32":  # packed context, one run of rows for each head
        C = sum(ctx)
        s["k_ctx"], s["v_ctx"] = _rand(g, (Hk, C, D), dt), _rand(g, (Hk, C, D), dt)
        starts = [sum(ctx[:b]) for b in range(B)]
        s["rows"] = [torch.arange(a, a + n, device="cuda") for a, n in zip(starts, ctx)]
    else:
        P = sum(_pages(n) for n in ctx) + 3
        s["k_pages"] = _rand(g, (Hk, P, _PAGE, D), dt)
        s["v_pages"] = s["k_pages"] if mla else _rand(g, (Hk, P, _PAGE, D), dt)
        s["k_ctx"], s["v_ctx"] = (x.view(Hk, P * _PAGE, D) for x in (s["k_pages"], s["v_pages"]))
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
        fm = s["fm"]
        s["cache"] = fm.InferenceCache()
        if case["dtype"] == "fp32":
            cu = [sum(ctx[:b]) for b in range(B + 1)]
            s["cache"].prefill_kv_cache(0, k_cache=s["k_ctx"].view(-1, D), v_cache=s["v_ctx"].view(-1, D),
                                        total_context_len=cu[-1], cu_seqlens_kv=_ints(cu), context_batch_size=B,
                                        is_mla=mla, num_heads=H, head_dim=D)
        else:
            s["cache"].prefill_paged_kv_cache(0, k_pages=s["k_pages"], v_pages=None if mla else s["v_pages"],
                                              block_table=s["table"], context_lens=_ints(ctx), is_mla=mla,
                                              num_heads=H, head_dim=D)
        s["tree"] = fm.build_tree_metadata(s["parents"], s["meta"], context_lens=_ints(ctx), check=False)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    way = s["case"]["way"]
    if way == "norm":
        return _own_norm(s) if own else _plain_norm(s, s["q"], s["k"], s["wq"], s["wk"])
    if way == "train":
        return _own_train(s) if own else _plain_train(s)
    if way == "table":
        return _own_table(s) if own else _plain_table(s)
    if way == "append":
        return _own_append(s) if own else _plain_append(s)
    return _own_tree(s) if own else _plain_tree(s)


def _own_norm(s):
    c = s["case"]
    return s["fm"].qk_norm_rope(s["q"], s["k"], q_weight=s["wq"], k_weight=s["wk"], eps=_EPS, cos=s["cos"],
                                sin=s["sin"], context_lens=s["start"], interleaved=c["interleaved"],
                                q_meta=s["meta"])


def _own_train(s):
    q, k = _own_norm(s)
    grads = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["dq"], s["dk"]))
    return [q.detach(), k.detach(), *grads]


def _own_table(s):
    fm = s["fm"]
    plan = fm.build_block_table(s["meta"], s["old"], free_pages=s["free"], block_table=s["table"], keep=s["keep"],
                                check=False)
    out = [plan.block_table, plan.slot_mapping, plan.positions, plan.context_lens, plan.cu_seqlens_kv]
    if s["parents"] is not None:
        tree = fm.build_tree_metadata(s["parents"], s["meta"], context_lens=s["old"], check=False)
        out += [tree.mask, tree.positions]
    return out


def _own_append(s):
    s["cache"].append_paged_kv_cache(0, k=s["k"], v=s["v"], q_meta=s["meta"], plan=s["plan"])
    return [s["k_pages"]] if s["v_pages"] is None else [s["k_pages"], s["v_pages"]]


def _own_tree(s):
    c = s["case"]
    return s["fm"].flash_attn_mlm_tree(s["q"], s["k"], s["v"], c["H"], s["meta"], s["tree"], s["scale"], s["cache"], 0,
                                       is_mla=c["mla"])


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _per_row(s, per_token):
    """[T, ...] values of the packed tokens, laid out for broadcasting over the rows of q and
    k: [1, T, ...] of [heads, T, D], or padded to [B, 1, N, ...] with zeros"""
    c = s["case"]
    if c["packed"]:
        return per_token[None]
    out = per_token.new_zeros((c["B"], c["N"]) + per_token.shape[1:])
    out[s["b"], s["p"]] = per_token
    return out[:, None]


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


def _plain_norm(s, q, k, wq, wk, cast=True):
    c = s["case"]
    pos = s["start"].long()[s["b"]] + s["p"]
    cos, sin = _per_row(s, s["cos"][pos]), _per_row(s, s["sin"][pos])
    real = _per_row(s, torch.ones(s["T"], 1, dtype=torch.bool, device="cuda"))
    out = []
    for x, w, h in ((q, wq, c["H"]), (k, wk, c["Hk"])):
        y = (x.view(h, s["T"], c["D"]) if c["packed"] else x).float()
        w = w.float()
        if c["gain"] == "head":
            w = w[:, None, :]
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + _EPS) * w
        y = torch.where(real, _plain_rotate(y, cos, sin, c["interleaved"]), 0.0).view(x.shape)
        out.append(y.to(x.dtype) if cast else y)
    return out


def _plain_train(s):
    leaves = [s[n].float().requires_grad_() for n in ("q", "k", "wq", "wk")]
    q, k = _plain_norm(s, *leaves, cast=False)
    grads = torch.autograd.grad((q, k), leaves, (s["dq"].float(), s["dk"].float()))
    dt = s["q"].dtype
    return [x.detach().to(dt) for x in (q, k, *grads)]


def _plain_table(s):
    old, lens, b, p = s["old"].long(), s["lengths"].long(), s["b"], s["p"]
    start = torch.cumsum(lens, 0) - lens
    if s["keep"] is None:
        rank, count, keep = p, lens, None
    else:
        keep = s["keep"]
        run_ = torch.cumsum(keep.long(), 0)  # kept tokens up to and with each one
        before = torch.cat((run_.new_zeros(1), run_))
        first = before[start]
        rank, count = run_ - keep.long() - first[b], before[start + lens] - first
    new = old + count
    have, total = (old + _PAGE - 1) // _PAGE, (new + _PAGE - 1) // _PAGE
    need = total - have
    base = torch.cumsum(need, 0) - need
    i = torch.arange(s["width"], device="cuda")[None]
    fresh = s["free"].long()[(base[:, None] + i - have[:, None]).clamp(0, s["free"].numel() - 1)]
    table = torch.where(i < have[:, None], s["table"].long(), torch.where(i < total[:, None], fresh, -1))
    a = old[b] + rank
    slots = table[b, (a // _PAGE).clamp(max=s["width"] - 1)] * _PAGE + a % _PAGE
    if keep is not None:
        slots = torch.where(keep, slots, -1)
    cu = torch.cat((new.new_zeros(1), torch.cumsum(new, 0)))
    i32 = torch.int32
    out = [table.to(i32), slots, (old[b] + p).to(i32), new.to(i32), cu.to(i32)]
    if s["parents"] is not None:
        out += _plain_masks(s)
    return out


def _plain_masks(s):
    c, T, b, p = s["case"], s["T"], s["b"], s["p"]
    N = c["N"]
    words = max(1, (N + 63) // 64)
    step = torch.zeros(c["B"], N + 1, dtype=torch.long, device="cuda")  # parent of each token, N: none
    step.fill_(N)
    parent = s["parents"].long()
    step[b, p] = torch.where(parent < 0, N, parent)
    bits = torch.zeros(T, words, dtype=torch.long, device="cuda")
    depth = torch.full((T,), -1, dtype=torch.long, device="cuda")
    at, token = p.clone(), torch.arange(T, device="cuda")
    for _ in range(N):  # every token walks to its root, a step at a time
        live = at < N
        word = torch.where(live, at // 64, 0)
        bits[token, word] |= torch.where(live, 1 << (at % 64), 0)
        depth += live
        at = step[b, at]
    return [bits, (s["old"].long()[b] + depth).to(torch.int32)]


def _plain_append(s):
    c = s["case"]
    slots = s["slots"]
    kept = slots >= 0
    out = []
    for x, pages in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
        if x is None:
            continue
        hk = pages.shape[0]
        rows = x.view(hk, s["T"], c["D"]) if c["packed"] else x[s["b"], :hk, s["p"]].transpose(0, 1)
        pages.view(hk, -1, c["D"])[:, slots[kept]] = rows[:, kept]
        out.append(pages)
    return out


def _plain_tree(s):
    c = s["case"]
    H, D = c["H"], c["D"]
    out = torch.empty(H, s["T"], D, dtype=s["q"].dtype, device="cuda")
    at = 0
    for b, n in enumerate(s["lens"]):
        if n == 0:
            continue
        heads = 1 if c["mla"] else H
        rows = s["rows"][b]
        q = s["q"][b, :, :n].float()
        k = torch.cat((s["k_ctx"][:, rows], s["k"][b, :heads, :n]), 1).float()
        v = torch.cat((s["v_ctx"][:, rows], s["v"][b, :heads, :n]), 1).float()
        if c["mla"]:  # one latent head for all query heads
            z = (q.reshape(H * n, D) @ k[0].t()).view(H, n, -1) * s["scale"]
        else:
            z = torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"]
        z[:, :, rows.numel():].masked_fill_(~s["seen"][b, :n, :n], -math.inf)
        e = torch.exp(z - z.amax(-1, keepdim=True))
        w = e / e.sum(-1, keepdim=True)
        o = (w.view(H * n, -1) @ v[0]).view(H, n, D) if c["mla"] else torch.matmul(w, v)
        out[:, at:at + n] = o.to(out.dtype)
        at += n
    return out.view(H * s["T"], D)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    lens = _lengths(case)
    T, way, B = sum(lens), case["way"], case["B"]
    if way == "table":
        width = _pages(case["ctx"] + case["N"])
        n = 2 * 4 * B * width + 4 * 4 * B + 12 * T + (T if case["keep"] else 0)
        if case["tree"]:
            n += T * (4 + 4 + 8 * max(1, (case["N"] + 63) // 64))
        return {"bytes": n, "flops": 0}
    D, H = case["D"], case["H"]
    es = _DTYPES[case["dtype"]].itemsize
    if way in ("norm", "train"):
        heads = H + case["Hk"]
        real = heads * T * D * es
        whole = real if case["packed"] else heads * B * case["N"] * D * es
        n = real + whole + 4 * T * case["R"]  # rows in and out; the angles once
        flops = 9 * heads * T * D
        if way == "train":
            n += 2 * real + whole + 4 * T * case["R"]
            flops += 20 * heads * T * D
        return {"bytes": n, "flops": flops}
    if way == "append":
        rows = (1 if case["mla"] else 2 * H) * T
        return {"bytes": 2 * rows * D * es + 8 * T, "flops": 0}
    ctx = _contexts(case)
    Hk = 1 if case["mla"] else 2 * H
    n = (Hk * (sum(ctx) + T) + 2 * H * T) * D * es
    pairs = sum(m * (c + (m + 1) / 2) for m, c in zip(lens, ctx))
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
    way = case["way"]
    if way in ("norm", "train"):
        return _exact_norm(s, way == "train")
    if way == "table":
        return _exact_table(s)
    if way == "append":
        return _exact_append(s)
    return _exact_tree(s)


def _exact_norm(s, train):
    """every token by itself: rows [heads, D] of token t, whose rotation is a complex product"""
    c = s["case"]
    D, R, T = c["D"], c["R"], s["T"]
    pos = s["start"].long()[s["b"]] + s["p"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None, :]  # [T, 1, R/2]

    def tokens(x, h):  # [T, h, D]
        x = x.detach().double()
        return x.view(h, T, D).permute(1, 0, 2) if c["packed"] else x[s["b"], :, s["p"]]

    def back(y, like):
        if c["packed"]:
            return y.permute(1, 0, 2).reshape(like.shape)
        out = torch.zeros(like.shape, dtype=torch.float64, device="cuda")
        out[s["b"], :, s["p"]] = y
        return out

    def rotate(y, by):
        y = y.clone()
        if c["interleaved"]:
            z = torch.complex(y[..., 0:R:2], y[..., 1:R:2]) * by
            y[..., 0:R:2], y[..., 1:R:2] = z.real, z.imag
        else:
            z = torch.complex(y[..., :R // 2], y[..., R // 2:R]) * by
            y[..., :R // 2], y[..., R // 2:R] = z.real, z.imag
        return y

    outs, dxs, dws = [], [], []
    for x, w, dy, h in ((s["q"], s["wq"], s.get("dq"), c["H"]), (s["k"], s["wk"], s.get("dk"), c["Hk"])):
        xt, wd = tokens(x, h), w.detach().double()
        inv = 1.0 / torch.sqrt((xt * xt).sum(-1, keepdim=True) / D + _EPS)
        unit = xt * inv
        outs.append(back(rotate(unit * wd, turn), x))
        if train:
            gy = rotate(tokens(dy, h), turn.conj())
            u = gy * wd
            dxs.append(back(inv * (u - unit * ((u * unit).sum(-1, keepdim=True) / D)), x))
            dws.append((gy * unit).sum(0) if c["gain"] == "head" else (gy * unit).sum((0, 1)))
    return outs + dxs + dws


def _exact_table(s):
    """request by request, on the host"""
    c = s["case"]
    old, table, free = s["old"].tolist(), s["table"].tolist(), s["free"].tolist()
    keep = [True] * s["T"] if s["keep"] is None else s["keep"].tolist()
    slots, pos, new, at, taken = [], [], [], 0, 0
    for b, n in enumerate(s["lens"]):
        a = old[b]
        for p in range(n):
            pos.append(old[b] + p)
            if not keep[at + p]:
                slots.append(-1)
                continue
            if a % _PAGE == 0:
                table[b][a // _PAGE] = free[taken]
                taken += 1
            slots.append(table[b][a // _PAGE] * _PAGE + a % _PAGE)
            a += 1
        new.append(a)
        at += n
    out = [_ints(table), _ints(slots, torch.int64), _ints(pos), _ints(new),
           _ints([sum(new[:b]) for b in range(len(new) + 1)])]
    if s["parents"] is not None:
        words = max(1, (c["N"] + 63) // 64)
        parent, at, bits, where = s["parents"].tolist(), 0, [], []
        for b, n in enumerate(s["lens"]):
            mine = []
            for i in range(n):
                up = parent[at + i]
                mine.append((mine[up] if up >= 0 else 0) | (1 << i))
                where.append(old[b] + bin(mine[i]).count("1") - 1)
            at += n
            for m in mine:
                w = [(m >> (64 * j)) & (2**64 - 1) for j in range(words)]
                bits.append([x - 2**64 if x >= 2**63 else x for x in w])
        out += [_ints(bits, torch.int64).view(-1, words), _ints(where)]
    return out


def _exact_append(s):
    """the pools as they are after the rows have been stored, a page row at a time"""
    c, T = s["case"], s["T"]
    out = []
    for x, pages in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
        if x is None:
            continue
        hk, P = pages.shape[:2]
        src = torch.full((P * _PAGE,), -1, dtype=torch.long, device="cuda")  # token stored in each slot
        kept = (s["slots"] >= 0).nonzero()[:, 0]
        src[s["slots"][kept]] = kept
        src = src.view(P, _PAGE)
        y = pages.double()
        page, row = (src >= 0).nonzero(as_tuple=True)
        t = src[page, row]
        for h in range(hk):
            y[h, page, row] = (x.view(hk, T, c["D"])[h, t] if c["packed"] else x[s["b"][t], h, s["p"][t]]).double()
        out.append(y)
    return out


def _exact_tree(s):
    """head by head: the context's part and the ancestors' part, joined by their sums"""
    c = s["case"]
    H, D = c["H"], c["D"]
    out = torch.empty(H, s["T"], D, dtype=torch.float64, device="cuda")
    at = 0
    for b, n in enumerate(s["lens"]):
        for h in range(H):
            j = 0 if c["mla"] else h
            q = s["q"][b, h, :n].double() * s["scale"]
            kc, vc = (x[j].index_select(0, s["rows"][b]).double() for x in (s["k_ctx"], s["v_ctx"]))
            km, vm = s["k"][b, j, :n].double(), s["v"][b, j, :n].double()
            zc, zm = q @ kc.T, q @ km.T
            zm = torch.where(s["seen"][b, :n, :n], zm, torch.full_like(zm, -math.inf))
            top = torch.maximum(zc.amax(1), zm.amax(1))[:, None]
            ec, em = torch.exp(zc - top), torch.exp(zm - top)
            out[h, at:at + n] = (ec @ vc + em @ vm) / (ec.sum(1) + em.sum(1))[:, None]
        at += n
    return out.view(H * s["T"], D)
