"""Values at the edges of the capped, biased and tree attention: slopes of either
sign, pages in every tile and what they may cost.  Against the float64 oracle,
within the bound that oracle/scored.py derives."""
import ctypes
import math

import pytest
import torch

import b200kern as bk
from b200kern import _lib, attention, errors
from oracle import scored

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _rand(g, *shape, dt=F32, big=1.0):
    return (torch.randn(*shape, generator=g) * big).to(dt)


def _i32(a, dev):
    return torch.tensor(a, dtype=torch.int32, device=dev)


def _pages(k, v, ps, gen):
    """A contiguous cache [B, Hkv, S, D] as shuffled pages and their table."""
    B, Hkv, S, D = k.shape
    width = -(-S // ps)
    table = torch.randperm(B * width, generator=gen).reshape(B, width).to(torch.int32)
    out = []
    for x in (k, v):
        pad = torch.zeros(B, Hkv, width * ps, D, dtype=x.dtype)
        pad[:, :, :S] = x
        p = torch.empty(B * width, ps, Hkv, D, dtype=x.dtype)
        p[table.reshape(-1).long()] = pad.view(B, Hkv, width, ps, D).permute(0, 2, 3, 1, 4).reshape(-1, ps, Hkv, D)
        out.append(p)
    return out[0], out[1], table


# --------------------------------------------------------- refusals
class _Cuda(torch.Tensor):
    """A CPU tensor that says it is on a GPU, to reach the checks behind the device's."""
    is_cuda = True


def _on_gpu(*shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Cuda)


@pytest.mark.parametrize("k,v,table", [
    ((2, 2, 8, 64), (2, 2, 9, 64), None), ((2, 2, 8, 64), (2, 1, 8, 64), None),  # caches of two shapes
    ((2, 2, 8, 32), (2, 2, 8, 32), None), ((2, 2, 8, 128), (2, 2, 8, 128), None),  # another head dim
    ((1, 2, 8, 64), (1, 2, 8, 64), None),                                          # fewer requests than q
    ((2, 8, 64), (2, 8, 64), None), ((2, 0, 8, 64), (2, 0, 8, 64), None),
    ((5, 16, 2, 64), (4, 16, 2, 64), (2, 3)),                                      # V has fewer pages
    ((5, 16, 2, 64), (5, 16, 2, 64), (1, 3)), ((5, 16, 2, 64), (5, 16, 2, 64), (6,)),
    ((5, 16, 2, 48), (5, 16, 2, 48), (2, 3))])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_decode_attention_refuses_shapes(k, v, table, cap):
    table = None if table is None else torch.zeros(table, dtype=torch.int32)
    with pytest.raises(errors.B2ShapeError):
        bk.decode_attention(_on_gpu(2, 4, 64), _on_gpu(*k), _on_gpu(*v), [1, 2], page_table=table, softcap=cap)


def test_decode_attention_refuses_other_devices():
    other = lambda *s: torch.zeros(*s, dtype=F16, device="meta").as_subclass(_Cuda)
    mine = _on_gpu(2, 2, 8, 64)
    for k, v in ((other(2, 2, 8, 64), mine), (mine, other(2, 2, 8, 64))):
        with pytest.raises(errors.B2ShapeError, match="meta"):
            bk.decode_attention(_on_gpu(2, 4, 64), k, v, [1, 2])
    with pytest.raises(errors.B2ShapeError, match="meta"):
        bk.decode_attention(_on_gpu(2, 4, 64), mine, mine, [1, 2], out=other(2, 4, 64))


def test_rows_beyond_31_bits_refused_without_gpu():
    """Head dims off the tensor cores count a kv head's rows (queries times query heads) in 32 bits."""
    s = _lib.strides_arg((8, 8, 8))
    call = lambda S, Hq: _lib.load().b2_flash_attn_fwd_scored(8, 8, 8, 8, 1, Hq, 1, S, 4, 8, s, s, s, s, 1.0, 0, 0, 1.0,
                                                              None, None, 0, None, 0, None)
    assert call(1 << 24, 128) == errors.ERR_UNSUPPORTED and b"rows a kv head" in _lib.load().b2_last_error()
    assert call(1 << 24, 65535) == errors.ERR_UNSUPPORTED


# ------------------------------------------------------------- caps
def test_caps_reach_the_kernels_in_range():
    """A cap is a Python float; fp32 knows neither 1e-60 (would be 0: no cap) nor 1e60 (infinite: refused)."""
    assert attention._cap(0) == 0.0 and attention._cap(30) == 30.0
    assert attention._cap(1e-60) == 1e-30 and attention._cap(1e60) == 1e30


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 64), (F32, 64), (F16, 256)])
@pytest.mark.parametrize("cap", [1e-60, 1e-300, 1e60, 1e300])
@pytest.mark.parametrize("binding", [True, False])
def test_caps_beyond_fp32(cuda, dt, D, cap, binding, monkeypatch):
    """Such caps leave all scores equal, or change none; with and without the C++ argument handling."""
    if not binding:
        monkeypatch.setattr(_lib, "fast", lambda: None)
    g = torch.Generator().manual_seed(D)
    q, k, v = (_rand(g, 1, 2, 130, D, dt=dt) for _ in range(3))
    dq, dk, dv = q.to(cuda), k.to(cuda), v.to(cuda)
    n = _i32([129], cuda)
    tri = torch.ones(1, 1, dtype=torch.bool, device=cuda)
    got = [bk.flash_attention(dq, dk, dv, softcap=cap)[0], bk.decode_attention(dq[:, :, 7], dk, dv, n + 1, softcap=cap)[0],
           bk.tree_attention(dq[:, :, 7][:, None].contiguous(), dk, dv, n, tri, softcap=cap)[0, 0]]
    sc = 0.0 if cap < 1 else 1 / math.sqrt(D)
    for h in range(2):
        o, av, mag = scored.rows(q[0, h], k[0, h], v[0, h], torch.ones(130, 130, dtype=torch.bool), sc)
        lim = scored.bound(o, av, mag, dt, 130, D, min(cap, float(mag.max())))
        assert bool(((got[0][h].double().cpu() - o).abs() <= lim).all())
        for x in got[1:]:
            assert bool(((x[h].double().cpu() - o[7]).abs() <= lim[7]).all())


# ----------------------------------------------------------- slopes
def _signed(h):
    """Slopes of both signs, up to 1/2."""
    return torch.tensor([(-1.0) ** i * 2.0 ** (-1.0 - 5.0 * i / h) for i in range(h)], dtype=F32)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64), (BF16, 80)])
@pytest.mark.parametrize("causal,docs,prefix,cap", [(True, None, None, 0.0), (False, None, None, 0.0),
                                                    (True, [0, 130, 140, 290], None, 0.0),
                                                    (False, [20, 150, 300], None, 20.0), (True, None, 170, 20.0)])
def test_prompt_slopes_of_either_sign(cuda, dt, D, causal, docs, prefix, cap):
    """s - slope |i - j| for any sign of the slope, on the diagonal, at documents' ends and between them."""
    g = torch.Generator().manual_seed(D)
    Hq, Hkv, S = 6, 3, 300
    q, k, v = _rand(g, 1, Hq, S, D, dt=dt, big=3.0), _rand(g, 1, Hkv, S, D, dt=dt), _rand(g, 1, Hkv, S, D, dt=dt)
    sl = _signed(Hq)
    out = bk.flash_attention(q.to(cuda), k.to(cuda), v.to(cuda), causal=causal, softcap=cap, alibi_slopes=sl.to(cuda),
                             doc_offsets=None if docs is None else _i32([docs], cuda),
                             prefix_lens=None if prefix is None else _i32([prefix], cuda)).double().cpu()
    vis = scored.ranges(S, S, causal, 0, docs, None if prefix is None else [prefix])
    far = (torch.arange(S).double()[:, None] - torch.arange(S).double()).abs()
    for h in range(Hq):
        o, av, mag = scored.rows(q[0, h], k[0, h // 2], v[0, h // 2], vis, 1 / math.sqrt(D), cap, -sl[h].double() * far)
        lim = scored.bound(o, av, mag, dt, S, D, cap, abs(float(sl[h])) * S)
        err = (out[0, h] - o).abs()
        assert bool((err <= lim).all()), f"h={h}: {(err / lim).max():.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64), (F16, 256)])
@pytest.mark.parametrize("rep", [1, 4, 12, 16])
@pytest.mark.parametrize("ps", [0, 16, 24])
def test_token_slopes_of_either_sign(cuda, dt, D, rep, ps):
    _token_slopes(cuda, dt, D, rep, ps)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("rep", [40, 100])
def test_token_slopes_of_either_sign_many_heads(cuda, dt, D, rep):
    _token_slopes(cuda, dt, D, rep, 16)


def _token_slopes(cuda, dt, D, rep, ps):
    g = torch.Generator().manual_seed(rep + D)
    lens = [300, 1, 129]
    B, Hkv, S = len(lens), 2, max(lens)
    Hq = rep * Hkv
    q, k, v = _rand(g, B, Hq, D, dt=dt, big=3.0), _rand(g, B, Hkv, S, D, dt=dt), _rand(g, B, Hkv, S, D, dt=dt)
    kc, vc, table = (k, v, None) if not ps else _pages(k, v, ps, g)
    sl = _signed(Hq)
    out = bk.decode_attention(q.to(cuda), kc.to(cuda), vc.to(cuda), _i32(lens, cuda), alibi_slopes=sl.to(cuda),
                              page_table=None if table is None else table.to(cuda)).double().cpu()
    for b, n in enumerate(lens):
        far = (n - 1 - torch.arange(n).double())[None]
        for h in range(Hq):
            o, av, mag = scored.rows(q[b, h:h + 1], k[b, h // rep, :n], v[b, h // rep, :n],
                                     torch.ones(1, n, dtype=torch.bool), 1 / math.sqrt(D), 0.0, -sl[h].double() * far)
            lim = scored.bound(o, av, mag, dt, n, D, 0.0, abs(float(sl[h])) * n)
            assert bool(((out[b, h] - o[0]).abs() <= lim[0]).all()), (b, h)


# ------------------------------------- infinities and NaN that a row sees
def _same_kind(out, ref):
    """Infinite and NaN where ref is, in kind and sign."""
    return torch.equal(torch.isnan(out), torch.isnan(ref)) and torch.equal(out == math.inf, ref == math.inf) and \
        torch.equal(out == -math.inf, ref == -math.inf)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 2, 2), (2, 8, 2), (3, 24, 2), (5, 8, 1), (30, 8, 2)])
@pytest.mark.parametrize("ps", [0, 12, 16])
def test_tree_visible_infinities(cuda, dt, D, T, Hq, Hkv, ps):
    """V of context keys holds infinities and NaN: +inf, -inf, both, NaN, an infinity that meets a drafted token's of
    the other sign; elsewhere nothing changes.  Rows stand in their tile four times, twice, once and in pairs."""
    g = torch.Generator().manual_seed(T + D)
    for ctx in (150, 3000):
        q = _rand(g, 2, T, Hq, D, dt=dt)
        k, v = _rand(g, 2, Hkv, ctx + T, D, dt=dt), _rand(g, 2, Hkv, ctx + T, D, dt=dt)
        clean, bad = v, v.clone()
        mask = torch.tril(torch.ones(T, T, dtype=torch.bool))
        for key, col, x in ((0, 1, math.inf), (ctx // 2, 2, -math.inf), (37, 3, math.inf), (ctx - 1, 3, -math.inf),
                            (ctx // 3, 4, math.nan), (ctx - 20, D - 1, math.inf), (ctx - 90, D - 1, math.inf),
                            (ctx, 6, -math.inf), (60, 6, math.inf), (ctx + T - 1, 7, -math.inf), (101, D // 2, math.inf)):
            bad[0, :, key, col] = x
        res = []
        for x in (clean, bad):
            kc, vc, table = (k, x, None) if not ps else _pages(k, x, ps, torch.Generator().manual_seed(1))
            res.append(bk.tree_attention(q.to(cuda), kc.to(cuda), vc.to(cuda), _i32([ctx, ctx - 7], cuda), mask.to(cuda),
                                         page_table=None if table is None else table.to(cuda)).float().cpu())
        want = res[0].clone()
        want[0, :, :, [1, D - 1, D // 2]] = math.inf
        want[0, :, :, 2] = -math.inf
        want[0, :, :, [3, 4, 6]] = math.nan
        want[0, -1, :, 7] = -math.inf
        assert _same_kind(res[1], want), ctx
        fine = torch.isfinite(want)
        assert torch.equal(res[1][fine], want[fine])


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 128), (F16, 64)])
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 8, 2), (12, 8, 2), (30, 8, 2), (60, 8, 2), (33, 4, 1)])
@pytest.mark.parametrize("ps", [0, 16])
def test_tree_infinities_of_small_weight(cuda, dt, D, T, Hq, Hkv, ps):
    """Visible infinities whose weights are far below fp16's smallest (scores up to 50 below the row's largest), but not
    below fp32's."""
    g = torch.Generator().manual_seed(T + D)
    ctx = 700
    q, k, v = _rand(g, 1, T, Hq, D, dt=dt, big=5.0), _rand(g, 1, Hkv, ctx + T, D, dt=dt), _rand(g, 1, Hkv, ctx + T, D, dt=dt)
    mask = torch.tril(torch.ones(T, T, dtype=torch.bool))

    def run(x):
        kc, vc, table = (k, x, None) if not ps else _pages(k, x, ps, torch.Generator().manual_seed(1))
        return bk.tree_attention(q.to(cuda), kc.to(cuda), vc.to(cuda), _i32([ctx], cuda), mask.to(cuda),
                                 page_table=None if table is None else table.to(cuda)).float().cpu()
    bad = v.clone()
    for key in range(0, 640, 64):
        bad[0, :, key, key // 64] = math.inf if key % 128 else -math.inf
    bad[0, :, 650, D - 1], bad[0, :, 30, D - 1] = math.inf, -math.inf
    want = run(v)
    want[..., 0:10:2], want[..., 1:10:2], want[..., D - 1] = -math.inf, math.inf, math.nan
    out = run(bad)
    assert _same_kind(out, want)
    fine = torch.isfinite(want)
    assert torch.equal(out[fine], want[fine])


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D,window", [(BF16, 128, 0), (F16, 64, 0), (F32, 64, 0), (F16, 256, 0), (BF16, 64, 90)])
@pytest.mark.parametrize("rep", [1, 4, 12])
@pytest.mark.parametrize("cap,alibi", [(20.0, False), (0.0, True)])
def test_token_visible_infinities(cuda, dt, D, window, rep, cap, alibi):
    g = torch.Generator().manual_seed(rep + D)
    n, Hkv = 400, 2
    q, k, v = _rand(g, 2, rep * Hkv, D, dt=dt), _rand(g, 2, Hkv, n, D, dt=dt), _rand(g, 2, Hkv, n, D, dt=dt)
    sl = _signed(rep * Hkv).abs().to(cuda) / 16 if alibi else None
    run = lambda x: bk.decode_attention(q.to(cuda), k.to(cuda), x.to(cuda), _i32([n, n - 3], cuda), softcap=cap,
                                        alibi_slopes=sl, window=window).float().cpu()
    bad = v.clone()
    for key, col, x in ((n - 1, 1, math.inf), (n - 40, 2, -math.inf), (n - 70, 3, math.inf), (n - 5, 3, -math.inf),
                        (n - 33, 4, math.nan), (n - 90, D - 1, math.inf)):
        bad[0, :, key, col] = x
    want = run(v)
    want[0, :, [1, D - 1]] = math.inf
    want[0, :, 2] = -math.inf
    want[0, :, [3, 4]] = math.nan
    out = run(bad)
    assert _same_kind(out, want)
    fine = torch.isfinite(want)
    assert torch.equal(out[fine], want[fine])


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("causal,cap,alibi", [(False, 0.0, False), (True, 0.0, True), (True, 30.0, False),
                                              (False, 30.0, True)])
def test_prompt_nan_scores(cuda, dt, D, causal, cap, alibi):
    """A NaN in K of one key, each key in turn: all rows that see it are NaN, the others as without it.  An infinite
    score without a cap is NaN as well (inf - inf in the softmax)."""
    g = torch.Generator().manual_seed(D)
    S = 140
    q, k, v = (_rand(g, 1, 1, S, D, dt=dt).expand(S, 1, S, D) for _ in range(3))
    sl = torch.tensor([0.01], device=cuda) if alibi else None
    docs = _i32([[0, S]], cuda).expand(S, 2).contiguous()
    run = lambda x: bk.flash_attention(q.to(cuda), x.to(cuda), v.to(cuda), causal=causal, softcap=cap, alibi_slopes=sl,
                                       doc_offsets=docs).float().cpu()
    clean = run(k)
    sees = torch.arange(S)[None] >= torch.arange(S)[:, None] if causal else torch.ones(S, S, dtype=torch.bool)
    for x in (math.nan, math.inf):
        k2 = k.clone()
        k2[torch.arange(S), 0, torch.arange(S), 0] = x
        out = run(k2)[:, 0]
        sick = sees if math.isnan(x) else sees & (q[0, 0, :, 0] > 0)[None]  # -inf: the key has weight 0
        if cap and x == math.inf:
            assert torch.isfinite(out).all()
            continue
        assert torch.isnan(out[sick]).all()
        hidden = ~sees
        assert torch.equal(out[hidden], clean[:, 0][hidden])
        assert torch.isfinite(out[~sick]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D,window", [(BF16, 128, 0), (F16, 64, 0), (F32, 64, 0), (F16, 256, 0), (BF16, 64, 200)])
@pytest.mark.parametrize("rep", [1, 4, 16])
@pytest.mark.parametrize("cap,alibi", [(30.0, False), (0.0, True)])
def test_token_nan_scores(cuda, dt, D, window, rep, cap, alibi):
    g = torch.Generator().manual_seed(D + rep)
    S = 140
    q = _rand(g, 1, 2 * rep, D, dt=dt).expand(S, 2 * rep, D)
    k, v = (_rand(g, 1, 2, S, D, dt=dt).expand(S, 2, S, D) for _ in range(2))
    k2 = k.clone()
    k2[torch.arange(S), 0, torch.arange(S), 0] = math.nan  # kv head 0 only
    sl = _signed(2 * rep).abs().to(cuda) / 16 if alibi else None
    run = lambda x: bk.decode_attention(q.contiguous().to(cuda), x.to(cuda), v.to(cuda), _i32([S] * S, cuda), softcap=cap,
                                        alibi_slopes=sl, window=window).float().cpu()
    out = run(k2)
    assert torch.isnan(out[:, :rep]).all()
    assert torch.equal(out[:, rep:], run(k)[:, rep:])


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("T,rep", [(1, 4), (4, 4), (4, 12), (2, 40), (9, 16)])
def test_tree_nan_scores(cuda, dt, D, T, rep):
    g = torch.Generator().manual_seed(D + T)
    S = 140
    q = _rand(g, 1, T, 2 * rep, D, dt=dt).expand(S, T, 2 * rep, D)
    k, v = (_rand(g, 1, 2, S + T, D, dt=dt).expand(S, 2, S + T, D) for _ in range(2))
    k2 = k.clone()
    k2[torch.arange(S), 0, torch.arange(S), 0] = math.nan
    k2[:, 1, S + T - 1] = math.nan  # kv head 1: a drafted token that only the last row sees
    mask = torch.tril(torch.ones(T, T, dtype=torch.bool)).to(cuda)
    run = lambda x: bk.tree_attention(q.to(cuda), x.to(cuda), v.to(cuda), _i32([S] * S, cuda), mask).float().cpu()
    out, clean = run(k2), run(k)
    assert torch.isnan(out[:, :, :rep]).all()
    assert torch.isnan(out[:, -1, rep:]).all()
    assert torch.equal(out[:, :-1, rep:], clean[:, :-1, rep:])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("D", [64, 80])
def test_infinities_of_no_weight(cuda, dt, D):
    """An infinity in V of a key that a row sees with a weight far below fp32's smallest is in its output, as an
    infinity or as NaN (0 times infinity)."""
    g = torch.Generator().manual_seed(D)
    S = 400
    q, k, v = (_rand(g, 1, 2, S, D, dt=dt) for _ in range(3))
    bad = v.clone()
    bad[:, :, 0, 3], bad[:, :, S - 1, 4] = math.inf, -math.inf
    slope = torch.tensor([2.0, 4.0], device=cuda)  # 800 to 1600 over the prompt
    run = lambda x: bk.flash_attention(q.to(cuda), k.to(cuda), x.to(cuda), causal=True, alibi_slopes=slope).cpu()[0]
    clean, out = run(v), run(bad)
    assert not torch.isfinite(out[:, :, 3]).any()
    assert torch.isfinite(out[:, :-1, 4]).all() and (out[:, -1, 4] == -math.inf).all()
    # a tree whose first context key scores 128 or more below the rest
    q2 = torch.full((1, 3, 2, D), 4.0, dtype=dt)
    k2 = k.abs()
    k2[:, :, 0] = -4
    tree = lambda x: bk.tree_attention(q2.to(cuda), k2.to(cuda), x.to(cuda), _i32([S - 3], cuda),
                                       torch.tril(torch.ones(3, 3, dtype=torch.bool, device=cuda))).cpu()[0]
    clean, out = tree(v), tree(bad)
    assert not torch.isfinite(out[..., 3]).any()
    assert torch.isfinite(out[:-1, :, 4]).all() and not torch.isfinite(out[-1, :, 4]).any()
    rest = [d for d in range(D) if d not in (3, 4)]
    assert torch.equal(out[..., rest], clean[..., rest])


# ------------------------------------------------------------- prefixes
@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64), (BF16, 80)])
def test_prefix_of_a_document_that_begins_before_the_row(cuda, dt, D):
    """Offsets may lie before the row's first token; a document's prefix counts from where it begins."""
    g = torch.Generator().manual_seed(D)
    S, docs, prefix = 300, [[-400, 130, 300], [-5, 2, 290]], [[460, 60], [3, 2 ** 31 - 1]]
    q, k, v = (_rand(g, 2, 2, S, D, dt=dt, big=2.0) for _ in range(3))
    out = bk.flash_attention(q.to(cuda), k.to(cuda), v.to(cuda), causal=True, doc_offsets=_i32(docs, cuda),
                             prefix_lens=_i32(prefix, cuda)).double().cpu()
    for b in range(2):
        vis = scored.ranges(S, S, True, 0, docs[b], prefix[b])
        for h in range(2):
            o, av, mag = scored.rows(q[b, h], k[b, h], v[b, h], vis, 1 / math.sqrt(D))
            assert bool(((out[b, h] - o).abs() <= scored.bound(o, av, mag, dt, S, D)).all()), (b, h)


# --------------------------------- infinities and NaN that a row must not see
@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("kw", [dict(causal=True, docs=[0, 600]), dict(causal=True, docs=[0, 3, 130, 131, 400, 555]),
                                dict(docs=[20, 150, 384, 590]), dict(causal=True, window=100, cap=20.0),
                                dict(causal=True, window=1, docs=[0, 600]), dict(causal=True, prefix=300, cap=30.0),
                                dict(causal=True, alibi=True), dict(docs=[0, 200, 600], alibi=True, cap=9.0)])
@pytest.mark.parametrize("far", [False, True])
def test_prompt_hidden_values(cuda, dt, D, kw, far):
    """Infinities and NaN in V of keys all over the prompt, in different columns (far: only at both ends): each row
    shows those of the keys it sees, and nothing of the others."""
    g = torch.Generator().manual_seed(D)
    S, Hq, Hkv = 600, 4, 2
    q, k, v = (_rand(g, 1, h, S, D, dt=dt) for h in (Hq, Hkv, Hkv))
    where = [(0, 1, math.nan), (599, 2, math.inf)] + ([] if far else [(128, 3, math.inf), (127, 4, -math.inf),
             (300, 5, math.nan), (301, 3, -math.inf), (450, D - 1, math.inf)])
    vis = scored.ranges(S, S, kw.get("causal", False), kw.get("window", 0), kw.get("docs"),
                        [kw["prefix"]] if "prefix" in kw else None)
    sl = _slopes(Hq) if kw.get("alibi") else None
    bad, finite = v.clone(), v.clone()
    want = torch.zeros(Hkv, S, D)
    for key, col, x in where:
        bad[:, :, key, col] = x
        finite[:, :, key, col] = 0
        want[:, vis[:, key], col] += x
    bad[0, 1, 400] = math.inf  # a whole row, in one kv head only
    finite[0, 1, 400] = 0
    want[1][vis[:, 400]] += math.inf
    out = bk.flash_attention(q.to(cuda), k.to(cuda), bad.to(cuda), causal=kw.get("causal", False),
                             window=kw.get("window", 0), softcap=kw.get("cap", 0.0),
                             alibi_slopes=None if sl is None else sl.to(cuda),
                             doc_offsets=_i32([kw["docs"]], cuda) if "docs" in kw else _i32([[0, S]], cuda),
                             prefix_lens=_i32([[kw["prefix"]]], cuda) if "prefix" in kw else None).double().cpu()[0]
    pos = torch.arange(S).double()
    for h in range(Hq):
        w = want[h // 2]
        bias = None if sl is None else -sl[h].double() * (pos[:, None] - pos).abs()
        o, av, mag = scored.rows(q[0, h], k[0, h // 2], finite[0, h // 2], vis, 1 / math.sqrt(D), kw.get("cap", 0.0), bias)
        lim = scored.bound(o, av, mag, dt, S, D, kw.get("cap", 0.0), 0.0 if sl is None else float(sl[h]) * S)
        fine = w == 0
        assert bool(((out[h] - o).abs() <= lim)[fine].all()), h
        assert _same_kind(out[h][~fine], w[~fine].double()), h


def _slopes(h):
    """Gentle ones: no visible key's weight falls to 0 in fp32, which would make NaN of its infinity."""
    return torch.tensor([2.0 ** -(4 + i) for i in range(h)], dtype=F32)


@pytest.mark.gpu
def test_prompt_hidden_values_many_turns(cuda):
    """More units than 31 turns of all CTAs: rows of every turn are looked at again."""
    g = torch.Generator(device=cuda).manual_seed(1)
    B, H, S, D = 16, 64, 1200, 64
    q, k, v = (torch.randn(B, H, S, D, generator=g, device=cuda).bfloat16() for _ in range(3))
    docs = _i32([[0, 500, 1190]] * B, cuda)
    run = lambda: bk.flash_attention(q, k, v, causal=True, doc_offsets=docs)
    clean = run()
    v[:, :, 1190:] = math.nan
    v[:, :, 500, 7] = math.inf
    out = run()
    far = 2.0 ** -6  # two outputs, each within the bound of weights rounded to 16 bits, |o| up to 4 in their rows
    sees = torch.zeros(S, D, dtype=torch.bool, device=cuda)
    sees[500:1190, 7] = True
    assert (out[:, :, sees] == math.inf).all()
    assert not out[:, :, 1190:].any()
    diff = (out.float() - clean.float()).abs()[:, :, ~sees]
    assert bool((diff <= far * (1 + clean.float().abs()[:, :, ~sees])).all())


@pytest.mark.gpu
@pytest.mark.parametrize("D,B", [(64, 300), (128, 600)])
def test_prompt_hidden_values_many_rounds(cuda, D, B):
    """More units than the list of rows to compute anew has room for at once."""
    g = torch.Generator(device=cuda).manual_seed(2)
    q, k, v = (torch.randn(B, 256, 2, D, generator=g, device=cuda).bfloat16() for _ in range(3))
    first = v[:, :, 0].clone()
    v[:, :, 1, ::2] = math.inf
    out = bk.flash_attention(q, k, v, causal=True, doc_offsets=_i32([[0, 2]] * B, cuda))
    assert torch.equal(out[:, :, 0], first)  # its only key
    assert (out[:, :, 1, ::2] == math.inf).all() and torch.isfinite(out[:, :, 1, 1::2]).all()


def _us(f, n=9):
    for _ in range(2):
        f()
    ev = [[torch.cuda.Event(enable_timing=True) for _ in range(2)] for _ in range(n)]
    for a, z in ev:
        a.record()
        f()
        z.record()
    torch.cuda.synchronize()
    return sorted(a.elapsed_time(z) for a, z in ev)[n // 2] * 1e3


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
def test_prompt_cost_of_what_is_not_finite(cuda, dt, D):
    """A NaN that the rows do see costs a look at their tiles' hidden keys, not their attention anew, and one that they
    must not see only the rows whose tiles hold it."""
    H, S = 16, 4096
    q, k, v = (torch.randn(1, H, S, D, device=cuda, dtype=dt) for _ in range(3))
    docs = _i32([[0, 4000]], cuda)
    run = lambda: _us(lambda: bk.flash_attention(q, k, v, causal=True, doc_offsets=docs))
    clean = run()
    v[:, :, 0, 5] = math.nan
    seen = run()
    v[:, :, 2000:4000] = math.nan
    most = run()
    v[:, :, :4000] = 0
    v[:, :, 4000:] = math.nan
    padding = run()
    assert seen <= 3 * clean and most <= 6 * clean + 2000 and padding <= 40 * clean, (clean, seen, most, padding)


# ------------------------------------------------------------ pages
@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (BF16, 256), (F32, 64)])
@pytest.mark.parametrize("ps", [1, 16, 24, 64, 100])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_token_pages_of_every_tile(cuda, dt, D, ps, cap):
    """Pages shuffled over many tiles; numbers outside the cache in the first, a middle and the last tile read as zeros
    and are recorded."""
    lib = _lib.load()
    code, stream = ctypes.c_uint(0), torch.cuda.current_stream().cuda_stream
    g = torch.Generator().manual_seed(D + ps)
    lens = [1000, 700, 64, 0]
    q, k, v = _rand(g, 4, 4, D, dt=dt), _rand(g, 4, 2, 1000, D, dt=dt), _rand(g, 4, 2, 1000, D, dt=dt)
    kp, vp, table = _pages(k, v, ps, g)
    run = lambda: bk.decode_attention(q.to(cuda), kp.to(cuda), vp.to(cuda), _i32(lens, cuda), page_table=table.to(cuda),
                                      softcap=cap).double().cpu()
    for change in (False, True):
        if change:
            for at, x in ((0, -1), (500 // ps, kp.shape[0]), (999 // ps, 2 ** 31 - 1)):
                table[0, at] = x
                k[0, :, at * ps:(at + 1) * ps] = 0
                v[0, :, at * ps:(at + 1) * ps] = 0
        out = run()
        st = lib.b2_device_error(stream, ctypes.byref(code))
        assert (code.value == 0xB2500001) if change else (st == 0 and code.value == 0)
        for b, n in enumerate(lens):
            for h in range(4):
                o, av, mag = scored.rows(q[b, h:h + 1], k[b, h // 2, :n], v[b, h // 2, :n],
                                         torch.ones(1, n, dtype=torch.bool), 1 / math.sqrt(D), cap)
                assert bool(((out[b, h] - o[0]).abs() <= scored.bound(o, av, mag, dt, n, D, cap)[0]).all()), (b, h)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("T", [2, 9, 40])
@pytest.mark.parametrize("ps", [8, 16, 24, 128])
def test_tree_pages_outside_in_every_tile(cuda, dt, D, T, ps):
    """Every third page number lies outside the cache: zeros there, call after call, whatever the ring held before."""
    lib = _lib.load()
    code, stream = ctypes.c_uint(0), torch.cuda.current_stream().cuda_stream
    g = torch.Generator().manual_seed(D + ps)
    ctx, S = [900, 130], 900 + T
    q, k, v = _rand(g, 2, T, 8, D, dt=dt), _rand(g, 2, 2, S, D, dt=dt), _rand(g, 2, 2, S, D, dt=dt)
    kp, vp, table = _pages(k, v, ps, g)
    mask = torch.tril(torch.ones(T, T, dtype=torch.bool))
    table[:, ::3] = torch.tensor([-1, 2 ** 31 - 1], dtype=torch.int32)[:, None]
    gone = (torch.arange(S) // ps) % 3 == 0
    k[:, :, gone] = 0
    v[:, :, gone] = 0
    run = lambda: bk.tree_attention(q.to(cuda), kp.to(cuda), vp.to(cuda), _i32(ctx, cuda), mask.to(cuda),
                                    page_table=table.to(cuda))
    out = run()
    for _ in range(5):
        assert torch.equal(run(), out)
    lib.b2_device_error(stream, ctypes.byref(code))
    assert code.value == 0xB2500001
    out = out.double().cpu()
    for b, n in enumerate(ctx):
        for h in range(8):
            o, av, mag = scored.tree(q[b, :, h], k[b, h // 4], v[b, h // 4], n, T, mask, 1 / math.sqrt(D))
            assert bool(((out[b, :, h] - o).abs() <= scored.bound(o, av, mag, dt, n + T, D)).all()), (b, h)


@pytest.mark.gpu
def test_token_pages_cost(cuda):
    """Single tokens over pages of 64 keys: the page table's latency does not stand before every tile (1.33 times the
    contiguous cache's time with the pages looked up a tile ahead, 1.94 with a check and a branch among the loads)."""
    B, Hq, Hkv, S, D, ps = 64, 32, 8, 4096, 128, 64
    q = torch.randn(B, Hq, D, device=cuda).bfloat16()
    k, v = (torch.randn(B, Hkv, S, D, device=cuda, dtype=BF16) for _ in range(2))
    lens = torch.full((B,), S, dtype=torch.int32, device=cuda)
    kp, vp = k.view(-1, ps, Hkv, D), v.view(-1, ps, Hkv, D)
    table = torch.randperm(B * S // ps, device=cuda).int().view(B, -1)

    def us(f):
        for _ in range(3):
            f()
        ev = [[torch.cuda.Event(enable_timing=True) for _ in range(2)] for _ in range(15)]
        for a, z in ev:
            a.record()
            f()
            z.record()
        torch.cuda.synchronize()
        return sorted(a.elapsed_time(z) for a, z in ev)[7]
    flat, paged = us(lambda: bk.decode_attention(q, k, v, lens)), us(
        lambda: bk.decode_attention(q, kp, vp, lens, page_table=table))
    assert paged <= 1.6 * flat, (paged, flat)


@pytest.mark.gpu
def test_edges_no_bounded_wait_ran_out(cuda):
    code = ctypes.c_uint(0)
    st = _lib.load().b2_device_error(torch.cuda.current_stream().cuda_stream, ctypes.byref(code))
    assert st == 0 and code.value == 0, hex(code.value)
