"""The serving operators around the paged KV cache, as they are measured.

Four operators, each with a plain form in elementary torch operations and the
framework's own call (``own = True``):

  pages   page table and slot map of one step, built on the GPU from request
          lengths (b200kern.build_page_table)
  store   new K/V rows written into the cache by slot (b200kern.store_kv)
  tree    attention of a tree of drafted tokens over a cache
          (b200kern.tree_attention)
  scored  attention whose scores are capped by a tanh or biased by distance,
          under document and prefix masks: prompts
          (b200kern.flash_attention) and single tokens
          (b200kern.decode_attention)

Lengths come from a rule of the case alone and only their order from the seed,
so that ``work`` is exact for every seed.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _bk():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-metal_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import b200kern
    return b200kern


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a full batch: every request adds one token, 1 in 16 opens a page
        dict(name="pages_step", op="pages", B=256, ctx_lo=0, ctx_hi=8192, new_lo=1, new_hi=1, ps=16, spare=0),
        # a step that admits ragged prompts beside chunks of running ones, with room for more tokens than come
        dict(name="pages_prompts", op="pages", B=93, ctx_lo=0, ctx_hi=2000, new_lo=1, new_hi=4099, ps=16, spare=517),
        # the K/V rows of one decode step
        dict(name="store_step", op="store", N=201, pad=0, Hkv=8, D=128, ps=16, src="bf16", dst="bf16"),
        # the rows of ragged prompts, fp32 activations kept in an fp16 cache, padded at the end
        dict(name="store_prompts", op="store", N=60001, pad=517, Hkv=8, D=128, ps=16, src="fp32", dst="fp16"),
        # one user, eight drafted tokens, a short contiguous cache: latency
        dict(name="tree_single", op="tree", B=1, T=8, Hq=32, Hkv=8, D=128, ctx_lo=500, ctx_hi=500, ps=0, ragged=False,
             cap=0.0, dt="bf16"),
        # a serving batch with trees of different sizes over ragged contexts in pages
        dict(name="tree_batch", op="tree", B=16, T=26, Hq=32, Hkv=8, D=128, ctx_lo=1, ctx_hi=4096, ps=16, ragged=True,
             cap=0.0, dt="fp16"),
        # long contexts and wide trees: tensor cores and memory both count
        dict(name="tree_long", op="tree", B=32, T=64, Hq=32, Hkv=8, D=128, ctx_lo=8192, ctx_hi=32768, ps=64,
             ragged=False, cap=0.0, dt="bf16"),
        # fp32 buffers, every head its own cache, odd page size, capped scores
        dict(name="tree_fp32", op="tree", B=3, T=5, Hq=8, Hkv=8, D=64, ctx_lo=0, ctx_hi=777, ps=24, ragged=True,
             cap=30.0, dt="fp32"),
        # packed documents of ragged lengths, padded at the end of each row
        dict(name="packed_docs", op="flash", B=2, Hq=32, Hkv=8, S=8192, D=128, docs=11, pad=100, causal=True, cap=0.0,
             alibi=False, prefix=0, dt="bf16"),
        # causal prefill with capped scores, odd length
        dict(name="capped_prompt", op="flash", B=1, Hq=16, Hkv=8, S=6001, D=128, docs=0, pad=0, causal=True, cap=50.0,
             alibi=False, prefix=0, dt="fp16"),
        # a prefix every token sees, and scores biased by distance
        dict(name="prefix_bias", op="flash", B=3, Hq=12, Hkv=12, S=1111, D=64, docs=0, pad=0, causal=True, cap=0.0,
             alibi=True, prefix=300, dt="bf16"),
        # one token of each request over a paged cache, capped and biased
        dict(name="decode_capped", op="decode", B=64, Hq=32, Hkv=8, D=128, ctx_lo=1, ctx_hi=8192, ps=16, cap=30.0,
             alibi=True, dt="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "store", "tree", "tree", "flash", "flash", "decode"])
    if op == "pages":
        step = rng.random() < 0.5
        hi = 1 if step else _log(rng, 2, 4099)
        b = _log(rng, 1, 256)
        while b * hi > 300000:
            b = max(1, b // 2)
        lo = rng.choice([0, 2000])
        return dict(op=op, B=b, ctx_lo=rng.randrange(0, lo + 1), ctx_hi=lo + _log(rng, 1, 6000), new_lo=1, new_hi=hi,
                    ps=rng.choice([1, 8, 16, 24, 32, 64, 128]), spare=rng.choice([0, 1, 777]))
    if op == "store":
        src, dst = rng.choice([("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp16"), ("fp32", "bf16"), ("fp32", "fp32")])
        n = _log(rng, 1, 30000)
        return dict(op=op, N=n, pad=rng.choice([0, 1, 99]), Hkv=rng.choice([1, 2, 4, 8]),
                    D=rng.choice([64, 80, 128, 256]), ps=rng.choice([1, 16, 24, 64, 128]), src=src, dst=dst)
    if op == "tree":
        dt = rng.choice(["bf16", "fp16", "bf16", "fp16", "fp32"])
        hkv, rep = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
        t, b = _log(rng, 1, 64), _log(rng, 1, 32)
        hi = _log(rng, 1, 2000 if dt == "fp32" else 16384)
        while b * hi > (8192 if dt == "fp32" else 262144):
            b = max(1, b // 2)
        return dict(op=op, B=b, T=t, Hq=hkv * rep, Hkv=hkv, D=rng.choice([64, 128]),
                    ctx_lo=rng.randrange(0, hi + 1) // 2, ctx_hi=hi, ps=rng.choice([0, 16, 24, 64, 128]),
                    ragged=rng.random() < 0.5, cap=rng.choice([0.0, 0.0, 30.0, 50.0]), dt=dt)
    if op == "flash":
        s = _log(rng, 1, 6001)
        b = rng.choice([1, 2, 3]) if s < 3000 else 1
        hkv, rep = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4])
        causal = rng.random() < 0.75
        docs = rng.choice([0, 1, 3, 9]) if s >= 16 else 0
        return dict(op=op, B=b, Hq=hkv * rep, Hkv=hkv, S=s, D=rng.choice([64, 128]), docs=docs,
                    pad=s // 7 if docs and rng.random() < 0.5 else 0, causal=causal, cap=rng.choice([0.0, 30.0, 50.0]),
                    alibi=rng.random() < 0.5, prefix=s // 3 if causal and not docs and rng.random() < 0.5 else 0,
                    dt=rng.choice(["bf16", "fp16"]))
    b, hkv, rep = _log(rng, 1, 64), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
    hi = _log(rng, 1, 8192)
    return dict(op=op, B=b, Hq=hkv * rep, Hkv=hkv, D=rng.choice([64, 128]), ctx_lo=1, ctx_hi=hi,
                ps=rng.choice([0, 16, 24, 64]), cap=rng.choice([30.0, 50.0]), alibi=rng.random() < 0.5,
                dt=rng.choice(["bf16", "fp16"]))


# ---------------------------------------------------------------- lengths
def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread (the middle one when n == 1)."""
    if n == 1:
        return [(lo + hi) // 2]
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _doc_lens(total, n):
    """n document lengths that add up to total, the longest many times the shortest."""
    w = [1.0 + 0.5 * i for i in range(n)]
    lens = [int(total * x / sum(w)) for x in w]
    lens[-1] += total - sum(lens)
    return lens


def _shuffled(xs, rs):
    return [xs[i] for i in rs.permutation(len(xs))]


def _draft_lens(case):
    return _spread(1, case["T"], case["B"]) if case["ragged"] else [case["T"]] * case["B"]


def _pages_of(n, ps):
    return -(-n // ps)


# ---------------------------------------------------------------- prepare
def _i32(xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


def _cache(case, gen, dt, need, most, rs):
    """K and V of `need[b]` tokens a request, `most` at the most: [B, Hkv, S, D], or pages and their table."""
    B, Hkv, D, ps = case["B"], case["Hkv"], case["D"], case["ps"]
    if not ps:
        shape = (B, Hkv, most, D)
        table = None
    else:
        width = _pages_of(most, ps)
        count = [_pages_of(n, ps) for n in need]
        perm = rs.permutation(_pages_of(sum(need), ps) + B + 3)  # the same pool for every order of the lengths
        t = np.full((B, width), -1, np.int32)
        at = 0
        for b in range(B):
            t[b, :count[b]] = perm[at:at + count[b]]
            at += count[b]
        table = torch.from_numpy(t).cuda()
        shape = (len(perm), ps, Hkv, D)
    k = torch.randn(shape, generator=gen, device="cuda", dtype=dt)
    v = torch.randn(shape, generator=gen, device="cuda", dtype=dt)
    return k, v, table


def _tree_masks(B, T, rs):
    """Each drafted token sees itself and its ancestors in a random tree."""
    m = np.zeros((B, T, T), bool)
    for j in range(T):
        parent = rs.integers(-1, j, size=B)
        for b in range(B):
            if parent[b] >= 0:
                m[b, j] = m[b, parent[b]]
            m[b, j, j] = True
    return torch.from_numpy(m).cuda()


def prepare(case, seed):
    rs = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(int(rs.integers(1 << 62)))
    st = dict(case=case)
    op = case["op"]
    if op == "pages":
        B, ps = case["B"], case["ps"]
        ctx = _shuffled(_spread(case["ctx_lo"], case["ctx_hi"], B), rs)
        new = _shuffled(_spread(case["new_lo"], case["new_hi"], B), rs)
        have = [_pages_of(c, ps) for c in ctx]
        width = _pages_of(case["ctx_hi"] + case["new_hi"], ps) + 2
        total = sum(have) + sum(_pages_of(n, ps) + 1 for n in new)
        perm = rs.permutation(total).astype(np.int32)
        table = np.full((B, width), -1, np.int32)
        at = 0
        for b in range(B):
            table[b, :have[b]] = perm[at:at + have[b]]
            at += have[b]
        st.update(ctx=_i32(ctx), new=_i32(new), table=torch.from_numpy(table).cuda(),
                  free=torch.from_numpy(perm[at:].copy()).cuda(), max_tokens=sum(new) + case["spare"])
    elif op == "store":
        N, ps, Hkv, D = case["N"], case["ps"], case["Hkv"], case["D"]
        pages = _pages_of(N, ps) + 5
        order = rs.permutation(pages)[:_pages_of(N, ps)]  # tokens fill one page after another
        slots = (order[:, None].astype(np.int64) * ps + np.arange(ps)).reshape(-1)[:N]
        slots = np.concatenate([slots, np.full(case["pad"], -1, np.int64)])
        src, dst = _DT[case["src"]], _DT[case["dst"]]
        n = N + case["pad"]
        st.update(k=torch.randn(n, Hkv, D, generator=gen, device="cuda", dtype=src),
                  v=torch.randn(n, Hkv, D, generator=gen, device="cuda", dtype=src),
                  slots=torch.from_numpy(slots).cuda(),
                  kp=torch.zeros(pages, ps, Hkv, D, device="cuda", dtype=dst),
                  vp=torch.zeros(pages, ps, Hkv, D, device="cuda", dtype=dst))
    elif op == "tree":
        B, T, dt = case["B"], case["T"], _DT[case["dt"]]
        ctx = _shuffled(_spread(case["ctx_lo"], case["ctx_hi"], B), rs)
        dl = _shuffled(_draft_lens(case), rs)
        k, v, table = _cache(case, gen, dt, [c + n for c, n in zip(ctx, dl)], case["ctx_hi"] + T, rs)
        q = torch.randn(B, T, case["Hq"], case["D"], generator=gen, device="cuda") * (4.0 if case["cap"] else 1.0)
        st.update(q=q.to(dt), k=k, v=v, table=table, ctx=_i32(ctx), dl=_i32(dl) if case["ragged"] else None,
                  mask=_tree_masks(B, T, rs))
    elif op == "flash":
        B, Hq, Hkv, S, D, dt = (case[x] for x in ("B", "Hq", "Hkv", "S", "D", "dt"))
        q = torch.randn(B, Hq, S, D, generator=gen, device="cuda") * (4.0 if case["cap"] else 1.0)
        st.update(q=q.to(_DT[dt]), k=torch.randn(B, Hkv, S, D, generator=gen, device="cuda", dtype=_DT[dt]),
                  v=torch.randn(B, Hkv, S, D, generator=gen, device="cuda", dtype=_DT[dt]), docs=None, prefix=None)
        if case["docs"]:
            rows = [[0] + list(np.cumsum(_shuffled(_doc_lens(S - case["pad"], case["docs"]), rs))) for _ in range(B)]
            st["docs"] = _i32([[int(x) for x in r] for r in rows])
        if case["prefix"]:
            st["prefix"] = _i32(_shuffled(_spread(0, 2 * case["prefix"], B), rs))
        st["slopes"] = _slopes(Hq) if case["alibi"] else None
    else:
        B, dt = case["B"], _DT[case["dt"]]
        lens = _shuffled(_spread(case["ctx_lo"], case["ctx_hi"], B), rs)
        k, v, table = _cache(case, gen, dt, lens, case["ctx_hi"], rs)
        q = torch.randn(B, case["Hq"], case["D"], generator=gen, device="cuda") * 4.0
        st.update(q=q.to(dt), k=k, v=v, table=table, lens=_i32(lens),
                  slopes=_slopes(case["Hq"]) if case["alibi"] else None)
    torch.cuda.synchronize()
    return st


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device="cuda")


# -------------------------------------------------------------------- run
def run(state):
    return _OWN[state["case"]["op"]](state) if own else _PLAIN[state["case"]["op"]](state)


def _own_pages(st):
    return _bk().build_page_table(st["ctx"], st["new"], st["case"]["ps"], st["free"], st["table"], st["max_tokens"])


def _own_store(st):
    return _bk().store_kv(st["k"], st["v"], st["kp"], st["vp"], st["slots"])


def _own_tree(st):
    return _bk().tree_attention(st["q"], st["k"], st["v"], st["ctx"], st["mask"], draft_lens=st["dl"],
                                page_table=st["table"], softcap=st["case"]["cap"])


def _own_flash(st):
    return _bk().flash_attention(st["q"], st["k"], st["v"], causal=st["case"]["causal"], softcap=st["case"]["cap"],
                                 alibi_slopes=st["slopes"], doc_offsets=st["docs"], prefix_lens=st["prefix"])


def _own_decode(st):
    return _bk().decode_attention(st["q"], st["k"], st["v"], st["lens"], page_table=st["table"],
                                  softcap=st["case"]["cap"], alibi_slopes=st["slopes"])


def _plain_pages(st):
    ps, table, free, n = st["case"]["ps"], st["table"], st["free"].long(), st["max_tokens"]
    ctx, new = st["ctx"].long(), st["new"].long()
    offsets = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), torch.cumsum(new, 0)])
    have = (ctx + ps - 1) // ps
    need = (ctx + new + ps - 1) // ps - have
    base = torch.cumsum(need, 0) - need
    # the pages that this step opens
    col = torch.arange(table.shape[1], device="cuda")
    rank = col - have[:, None]
    opened = (rank >= 0) & (rank < need[:, None])
    page = free[(base[:, None] + rank).clamp(0, free.numel() - 1)]
    table.copy_(torch.where(opened, page.int(), table))
    # the slot of every new token
    t = torch.arange(n, device="cuda")
    b = torch.searchsorted(offsets[1:].contiguous(), t, right=True).clamp(max=len(ctx) - 1)
    pos = (ctx[b] + t - offsets[b]).clamp(0, table.shape[1] * ps - 1)
    slots = torch.where(t < offsets[-1], table[b, pos // ps].long() * ps + pos % ps, -1)
    return table, slots, offsets.int(), need.sum().int().reshape(1)


def _plain_store(st):
    kp, vp = st["kp"], st["vp"]
    live = st["slots"] >= 0
    at = st["slots"][live]
    kp.view(-1, *kp.shape[2:])[at] = st["k"][live].to(kp.dtype)
    vp.view(-1, *vp.shape[2:])[at] = st["v"][live].to(vp.dtype)
    return kp, vp


def _softmax_pv(s, hidden, v):
    """softmax of scores s over the keys that are not hidden, times v; rows that see nothing give 0."""
    s.masked_fill_(hidden, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == float("-inf"), 0.0, m)).exp_()
    return (p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _gathered(x, table, b0, b1):
    """Requests b0..b1 of a cache in fp32: [b, Hkv, S, D]."""
    if table is None:
        return x[b0:b1].float()
    t = table[b0:b1].long().clamp_min(0)
    rows = x[t]  # [b, pages, ps, Hkv, D]
    return rows.flatten(1, 2).transpose(1, 2).float()


def _plain_tree(st):
    c, q, mask = st["case"], st["q"], st["mask"]
    B, T, Hq, D = q.shape
    Hkv = c["Hkv"]
    rep = Hq // Hkv
    out = torch.empty_like(q)
    step = 4  # requests at a time
    for b0 in range(0, B, step):
        b1 = min(B, b0 + step)
        k, v = _gathered(st["k"], st["table"], b0, b1), _gathered(st["v"], st["table"], b0, b1)
        S = k.shape[2]
        qq = q[b0:b1].float().reshape(b1 - b0, T, Hkv, rep, D).permute(0, 2, 3, 1, 4)  # b, Hkv, rep, T, D
        s = (qq.flatten(2, 3) @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D))
        if c["cap"]:
            s = s.div_(c["cap"]).tanh_().mul_(c["cap"])
        ctx = st["ctx"][b0:b1].long()
        dl = st["dl"][b0:b1].long() if st["dl"] is not None else torch.full_like(ctx, T)
        j = torch.arange(S, device="cuda") - ctx[:, None]  # place among the drafted tokens
        drafted = (j >= 0) & (j < dl[:, None])
        seen = torch.gather(mask[b0:b1], 2, j.clamp(0, T - 1)[:, None, :].expand(-1, T, -1))
        vis = (j < 0)[:, None, :] | (seen & drafted[:, None, :])
        vis = vis & (torch.arange(T, device="cuda") < dl[:, None])[:, :, None]
        hidden = ~vis[:, None, None].expand(-1, 1, rep, -1, -1).reshape(b1 - b0, 1, rep * T, S)
        v = v.masked_fill(~((j < 0) | drafted)[:, None, :, None], 0.0)
        o = _softmax_pv(s, hidden, v)
        out[b0:b1] = o.view(b1 - b0, Hkv, rep, T, D).permute(0, 3, 1, 2, 4).reshape(b1 - b0, T, Hq, D).to(q.dtype)
    return out


def _ranges(st, b):
    """First and one past the last key that each query of prompt b sees."""
    c = st["case"]
    S = c["S"]
    i = torch.arange(S, device="cuda")
    lo, hi = torch.zeros_like(i), torch.full_like(i, S)
    if st["docs"] is not None:
        off = st["docs"][b].long()
        d = torch.searchsorted(off[1:].contiguous(), i, right=True)
        inside = d < off.numel() - 1
        d = d.clamp(max=off.numel() - 2)
        lo = torch.where(inside, off[d], 0)
        hi = torch.where(inside, off[d + 1], 0)
    if c["causal"]:
        last = i + 1
        if st["prefix"] is not None:
            last = torch.maximum(last, st["prefix"][b].long())
        hi = torch.minimum(hi, last)
    return lo, hi


def _plain_flash(st):
    c, q, k, v = st["case"], st["q"], st["k"], st["v"]
    B, Hq, S, D = q.shape
    rep = Hq // c["Hkv"]
    out = torch.empty_like(q)
    i = torch.arange(S, device="cuda")
    step = max(1, min(rep, (1 << 28) // (S * S)))
    while rep % step:  # query heads at a time, of one kv head
        step -= 1
    for b in range(B):
        lo, hi = _ranges(st, b)
        hidden = (i < lo[:, None]) | (i >= hi[:, None])
        far = (i[:, None] - i).abs().float() if st["slopes"] is not None else None
        for h in range(0, Hq, step):
            h1 = h + step
            kk, vv = k[b, h // rep].float(), v[b, h // rep].float()
            s = (q[b, h:h1].float() @ kk.t()).mul_(1.0 / math.sqrt(D))
            if c["cap"]:
                s = s.div_(c["cap"]).tanh_().mul_(c["cap"])
            if far is not None:
                s = s.sub_(st["slopes"][h:h1, None, None] * far)
            out[b, h:h1] = _softmax_pv(s, hidden, vv).to(q.dtype)
    return out


def _plain_decode(st):
    c, q = st["case"], st["q"]
    B, Hq, D = q.shape
    Hkv = c["Hkv"]
    out = torch.empty_like(q)
    step = 16
    for b0 in range(0, B, step):
        b1 = min(B, b0 + step)
        k, v = _gathered(st["k"], st["table"], b0, b1), _gathered(st["v"], st["table"], b0, b1)
        s = (q[b0:b1].float().view(b1 - b0, Hkv, Hq // Hkv, D) @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D))
        s = s.div_(c["cap"]).tanh_().mul_(c["cap"])
        j = torch.arange(k.shape[2], device="cuda")
        n = st["lens"][b0:b1].long()
        if st["slopes"] is not None:
            far = (n[:, None] - 1 - j).abs().float()
            s = s.sub_(st["slopes"].view(1, Hkv, -1, 1) * far[:, None, None, :])
        o = _softmax_pv(s, (j >= n[:, None])[:, None, None, :], v)
        out[b0:b1] = o.reshape(b1 - b0, Hq, D).to(q.dtype)
    return out


_PLAIN = dict(pages=_plain_pages, store=_plain_store, tree=_plain_tree, flash=_plain_flash, decode=_plain_decode)
_OWN = dict(pages=_own_pages, store=_own_store, tree=_own_tree, flash=_own_flash, decode=_own_decode)


# ------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "pages":
        ctx, new = _spread(case["ctx_lo"], case["ctx_hi"], case["B"]), _spread(case["new_lo"], case["new_hi"], case["B"])
        n = sum(new) + case["spare"]
        # lengths in, offsets and slots (8 bytes) out, about one page entry read or written per page touched
        pages = sum(_pages_of(x, case["ps"]) for x in new)
        return {"bytes": 12 * len(ctx) + 8 * n + 8 * pages, "flops": n}
    if op == "store":
        e = 2 * case["N"] * case["Hkv"] * case["D"]
        return {"bytes": e * (_ES[case["src"]] + _ES[case["dst"]]) + 8 * (case["N"] + case["pad"]), "flops": e}
    if op == "tree":
        ctx, dl = _spread(case["ctx_lo"], case["ctx_hi"], case["B"]), _draft_lens(case)
        keys = sum(ctx) + sum(dl)
        # both lists are shuffled on their own, so a mean draft length stands for each request's
        pairs = sum(ctx) * (sum(dl) / len(dl)) + sum(dl)
        q = case["B"] * case["T"] * case["Hq"] * case["D"]
        return {"bytes": _ES[case["dt"]] * (2 * keys * case["Hkv"] * case["D"] + 2 * q),
                "flops": 4 * pairs * case["Hq"] * case["D"]}
    if op == "flash":
        S = case["S"]
        lens = _doc_lens(S - case["pad"], case["docs"]) if case["docs"] else [S]
        pairs = case["B"] * sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        if case["prefix"]:
            pairs += sum(p * (p - 1) // 2 for p in _spread(0, 2 * case["prefix"], case["B"]))
        e = case["B"] * S * case["D"] * (2 * case["Hq"] + 2 * case["Hkv"])
        return {"bytes": e * _ES[case["dt"]], "flops": 4 * pairs * case["Hq"] * case["D"]}
    keys = sum(_spread(case["ctx_lo"], case["ctx_hi"], case["B"]))
    e = 2 * keys * case["Hkv"] * case["D"] + 2 * case["B"] * case["Hq"] * case["D"]
    return {"bytes": _ES[case["dt"]] * e, "flops": 4 * keys * case["Hq"] * case["D"]}


# ------------------------------------------------------------------ exact
def exact(case, seed):
    """The definitions, one request and head at a time, in 64 bits."""
    st = prepare(case, seed)
    return _EXACT[case["op"]](st)


def _exact_pages(st):
    ps, n = st["case"]["ps"], st["max_tokens"]
    ctx, new = st["ctx"].tolist(), st["new"].tolist()
    table, free = st["table"].cpu().numpy().copy(), st["free"].tolist()
    slots, offsets, used = [], [0], 0
    for b in range(len(ctx)):
        for pos in range(ctx[b], ctx[b] + new[b]):
            if pos % ps == 0:  # the first token of a page opens it
                table[b, pos // ps] = free[used]
                used += 1
            slots.append(int(table[b, pos // ps]) * ps + pos % ps)
        offsets.append(offsets[-1] + new[b])
    slots += [-1] * (n - len(slots))
    return (torch.from_numpy(table), torch.tensor(slots, dtype=torch.long), torch.tensor(offsets, dtype=torch.int32),
            torch.tensor([used], dtype=torch.int32))


def _exact_store(st):
    res = []
    slots = st["slots"].tolist()
    live = [n for n, s in enumerate(slots) if s >= 0]
    at = torch.tensor([slots[n] for n in live], device="cuda")
    live = torch.tensor(live, device="cuda")
    for x, pages in ((st["k"], st["kp"]), (st["v"], st["vp"])):
        flat = pages.double().reshape(-1, *pages.shape[2:])
        flat[at] = x.double()[live]
        res.append(flat.reshape(pages.shape))
    return tuple(res)


def _one_head(q, k, v, vis, cap, bias):
    """q [R, D], k/v [S, D], vis [R, S] -> [R, D] float64."""
    s = q.double() @ k.double().t() / math.sqrt(q.shape[-1])
    if cap:
        s = cap * torch.tanh(s / cap)
    if bias is not None:
        s = s + bias
    s = torch.where(vis, s, torch.tensor(float("-inf"), dtype=torch.float64, device="cuda"))
    o = torch.softmax(s, -1) @ v.double()
    return torch.where(vis.any(-1, keepdim=True), o, torch.zeros_like(o))


def _request_kv(st, b, hk, n):
    """K and V of head hk of request b: the first n keys, [n, D]."""
    if st["table"] is None:
        return st["k"][b, hk, :n], st["v"][b, hk, :n]
    ps = st["case"]["ps"]
    pages = st["table"][b, :_pages_of(n, ps)].long()
    return tuple(x[pages][:, :, hk].reshape(-1, x.shape[-1])[:n] for x in (st["k"], st["v"]))


def _exact_tree(st):
    c, q = st["case"], st["q"]
    B, T, Hq, D = q.shape
    rep = Hq // c["Hkv"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    ctx = st["ctx"].tolist()
    dl = st["dl"].tolist() if st["dl"] is not None else [T] * B
    for b in range(B):
        n = ctx[b] + dl[b]
        vis = torch.ones(dl[b], n, dtype=torch.bool, device="cuda")
        vis[:, ctx[b]:] = st["mask"][b, :dl[b], :dl[b]]
        for h in range(Hq):
            k, v = _request_kv(st, b, h // rep, n)
            out[b, :dl[b], h] = _one_head(q[b, :dl[b], h], k, v, vis, c["cap"], None)
    return out


def _exact_flash(st):
    c, q = st["case"], st["q"]
    B, Hq, S, D = q.shape
    rep = Hq // c["Hkv"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    pos = torch.arange(S, device="cuda")
    for b in range(B):
        doc = torch.zeros(S, dtype=torch.long, device="cuda")
        if st["docs"] is not None:
            doc -= 1
            off = st["docs"][b].tolist()
            for d in range(len(off) - 1):
                doc[off[d]:off[d + 1]] = d
        vis = (doc[:, None] == doc) & (doc >= 0)[:, None]
        if c["causal"]:
            first = int(st["prefix"][b]) if st["prefix"] is not None else 0
            vis &= (pos <= pos[:, None]) | (pos < first)
        for h in range(Hq):
            bias = None
            if st["slopes"] is not None:
                bias = -st["slopes"][h].double() * (pos[:, None] - pos).abs().double()
            out[b, h] = _one_head(q[b, h], st["k"][b, h // rep], st["v"][b, h // rep], vis, c["cap"], bias)
    return out


def _exact_decode(st):
    c, q = st["case"], st["q"]
    B, Hq, D = q.shape
    rep = Hq // c["Hkv"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["lens"].tolist()):
        far = torch.arange(n - 1, -1, -1, device="cuda").double()[None]
        vis = torch.ones(1, n, dtype=torch.bool, device="cuda")
        for h in range(Hq):
            k, v = _request_kv(st, b, h // rep, n)
            bias = -st["slopes"][h].double() * far if st["slopes"] is not None else None
            out[b, h] = _one_head(q[b, h:h + 1], k, v, vis, c["cap"], bias)[0]
    return out


_EXACT = dict(pages=_exact_pages, store=_exact_store, tree=_exact_tree, flash=_exact_flash, decode=_exact_decode)
