"""Attention of drafted-token trees over contiguous and paged caches: refusals
on the host (CPU), values on the GPU against the float64 oracle, within the
bound that oracle/scored.py derives from the arithmetic."""
import ctypes
import math

import pytest
import torch

import b200kern as bk
from b200kern import _lib, errors
from oracle import scored


# ---------------------------------------------------------------- refusals
def _args(B=2, T=3, Hq=4, Hkv=2, D=16, S=40, dt=torch.float32):
    z = lambda *s: torch.zeros(*s, dtype=dt)
    return dict(q=z(B, T, Hq, D), k_cache=z(B, Hkv, S, D), v_cache=z(B, Hkv, S, D),
                context_lens=torch.zeros(B, dtype=torch.int32), tree_mask=torch.ones(T, T, dtype=torch.bool))


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(2, 3, 4)), errors.B2ShapeError), (dict(q=torch.zeros(2, 3, 5, 16)), errors.B2ShapeError),
    (dict(q=torch.zeros(2, 3, 4, 16, dtype=torch.float64)), errors.B2DtypeError),
    (dict(v_cache=torch.zeros(2, 2, 40, 16).half()), errors.B2DtypeError),
    (dict(k_cache=torch.zeros(2, 2, 40, 8), v_cache=torch.zeros(2, 2, 40, 8)), errors.B2ShapeError),
    (dict(k_cache=torch.zeros(1, 2, 40, 16), v_cache=torch.zeros(1, 2, 40, 16)), errors.B2ShapeError),
    (dict(tree_mask=torch.ones(3, 4, dtype=torch.bool)), errors.B2ShapeError),
    (dict(tree_mask=torch.ones(3, 3)), errors.B2ShapeError),
    (dict(context_lens=torch.zeros(3, dtype=torch.int32)), errors.B2ShapeError),
    (dict(context_lens=torch.zeros(2, dtype=torch.int64)), errors.B2ShapeError),
    (dict(draft_lens=torch.zeros(2, dtype=torch.int64)), errors.B2ShapeError),
    (dict(page_table=torch.zeros(3, 1, dtype=torch.int32)), errors.B2ShapeError),
    (dict(softcap=-1.0), errors.B2ShapeError), (dict(softcap=math.inf), errors.B2ShapeError),
    ({}, errors.B2ShapeError)])  # in order, but on the CPU
def test_tree_attention_refuses(change, error):
    with pytest.raises(error):
        bk.tree_attention(**{**_args(), **change})


def test_c_entry_refuses_without_gpu():
    lib = _lib.load()
    s = _lib.strides_arg((8, 8, 8))

    def call(B=1, T=2, Hq=4, Hkv=2, D=16, keys=32, ps=0, mp=0, ms=0, scale=1.0, cap=0.0, qd=0, kd=0, q=1, table=None):
        return lib.b2_tree_attn(q, 1, 1, 1, table, 1, None, 1, ms, None, B, T, Hq, Hkv, D, keys, ps, mp, 4, s, s, s, s,
                                scale, cap, qd, kd, None)
    assert call(Hq=5) == errors.ERR_INVALID
    assert call(D=257) == errors.ERR_UNSUPPORTED
    assert call(qd=3) == errors.ERR_DTYPE
    assert call(ms=3) == errors.ERR_INVALID
    assert call(scale=math.nan) == errors.ERR_INVALID
    assert call(cap=-2.0) == errors.ERR_INVALID
    assert call(ps=16, mp=2) == errors.ERR_INVALID              # no table
    assert call(ps=16, mp=1, table=1) == errors.ERR_INVALID     # more keys than the table holds
    assert call(q=None) == errors.ERR_INVALID
    assert call(B=70000) == errors.ERR_UNSUPPORTED
    assert call(T=0, q=None) == errors.OK


# ------------------------------------------------------------------ values
def _masks(B, T, gen):
    """Random trees: every token sees itself and its ancestors."""
    m = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for j in range(T):
            parent = int(torch.randint(-1, j, (1,), generator=gen)) if j else -1
            if parent >= 0:
                m[b, j] = m[b, parent]
            m[b, j, j] = True
    return m


def _paged(k, v, ps, gen, spare=2):
    """A contiguous cache as shuffled pages; what no key fills is NaN."""
    B, Hkv, S, D = k.shape
    width = -(-S // ps)
    n = B * width + spare
    table = torch.randperm(n, generator=gen)[:B * width].reshape(B, width).to(torch.int32)
    out = []
    for x in (k, v):
        p = torch.full((n, ps, Hkv, D), math.nan, dtype=x.dtype)
        pad = torch.full((B, Hkv, width * ps, D), math.nan, dtype=x.dtype)
        pad[:, :, :S] = x
        p[table.reshape(-1).long()] = pad.view(B, Hkv, width, ps, D).permute(0, 2, 3, 1, 4).reshape(-1, ps, Hkv, D)
        out.append(p)
    return out[0], out[1], table


def _check(out, q, k, v, ctx, dl, mask, scale, cap, dtype):
    """Every row against the oracle, within its bound."""
    B, T, Hq, D = q.shape
    rep = Hq // k.shape[1]
    out = out.double().cpu()
    for b in range(B):
        m = mask[b] if mask.dim() == 3 else mask
        c = min(max(ctx[b], 0), k.shape[2])
        n = min(min(max(dl[b], 0), T), k.shape[2] - c)
        for h in range(Hq):
            o, av, mag = scored.tree(q[b, :, h], k[b, h // rep], v[b, h // rep], c, n, m, scale, cap)
            lim = scored.bound(o, av, mag, dtype, c + n, D, cap)
            err = (out[b, :, h] - o).abs()
            assert bool((err <= lim).all()), f"b={b} h={h}: {(err / lim).max().item():.3g} of the bound"
            assert not out[b, n:, h].any()


def _run(cuda, B, T, Hq, Hkv, D, ctx, dl, qd, kd, ps=0, cap=0.0, seed=0, shared=False, scale=None, big=1.0):
    gen = torch.Generator().manual_seed(seed + T + D)
    S = max(c + n for c, n in zip(ctx, dl)) if ctx else 0
    S = max(S, 1)
    q = (torch.randn(B, T, Hq, D, generator=gen) * big).to(qd)
    k, v = (torch.randn(B, Hkv, S, D, generator=gen).to(kd) for _ in range(2))
    for b in range(B):  # behind a request's tokens there is nothing to read
        k[b, :, max(ctx[b] + dl[b], 0):] = math.nan
        v[b, :, max(ctx[b] + dl[b], 0):] = math.nan
    mask = _masks(B, T, gen)
    if shared:
        mask = mask[0]
    i = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)
    kc, vc, table = k, v, None
    if ps:
        kc, vc, table = _paged(k, v, ps, gen)
        table = table.to(cuda)
    full = all(n == T for n in dl)
    out = bk.tree_attention(q.to(cuda), kc.to(cuda), vc.to(cuda), i(ctx), mask.to(cuda),
                            draft_lens=None if full else i(dl), page_table=table, softcap=cap, scale=scale)
    assert out.dtype == qd and out.shape == q.shape
    _check(out, q, k, v, ctx, dl, mask, 1 / math.sqrt(D) if scale is None else scale, cap, qd)


F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("qd,kd", [(BF16, BF16), (F16, F16), (F32, F32), (F32, F16), (BF16, F32)])
@pytest.mark.parametrize("ps", [0, 16, 24])
@pytest.mark.parametrize("T,Hq,Hkv,D,cap", [(1, 4, 4, 64, 0.0), (5, 8, 2, 128, 30.0), (33, 4, 1, 64, 0.0),
                                            (9, 2, 2, 80, 0.0), (3, 2, 1, 256, 5.0)])
def test_tree(cuda, qd, kd, ps, T, Hq, Hkv, D, cap):
    """Ragged contexts from none to several tiles, trees of all sizes, one of them empty."""
    _run(cuda, 5, T, Hq, Hkv, D, [0, 1, 127, 300, 640], [T, max(T - 1, 0), 0, T // 2, T], qd, kd, ps, cap)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("T,Hq,Hkv", [(64, 8, 2), (130, 2, 2), (17, 16, 1), (31, 8, 1), (200, 4, 2)])
def test_tree_rows_past_a_tile(cuda, dt, T, Hq, Hkv):
    """More rows than one tile has, trees wider than a tile of keys, drafted tokens across tile borders."""
    _run(cuda, 2, T, Hq, Hkv, 128, [100, 333], [T, T - 3], dt, dt, 64, shared=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("ctx", [1, 63, 64, 65, 128, 129, 191, 255, 256, 1000, 5000])
def test_tree_context_lengths(cuda, dt, ctx):
    """Around the tiles' ends, alone and beside a longer request."""
    _run(cuda, 1, 7, 8, 2, 128, [ctx], [7], dt, dt)
    _run(cuda, 2, 7, 8, 2, 64, [ctx, 2 * ctx + 1], [7, 6], dt, dt, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("ps", [1, 3, 4, 8, 12, 32, 64, 100, 128])
@pytest.mark.parametrize("T,Hq,Hkv,cap", [(4, 8, 2, 0.0), (12, 8, 2, 20.0), (25, 4, 1, 0.0), (80, 4, 2, 0.0)])
def test_tree_page_sizes(cuda, dt, D, ps, T, Hq, Hkv, cap):
    """Every way to load the cache; 16 to 160 rows a group: rows in the tile four times, twice, once, two tiles."""
    _run(cuda, 3, T, Hq, Hkv, D, [0, 130, 517], [T, T - 1, T], dt, dt, ps, cap)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("ps", [0, 12, 16])
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 1, 1), (2, 6, 2), (4, 2, 1), (8, 3, 3), (1, 7, 1), (3, 3, 1)])
@pytest.mark.parametrize("cap", [0.0, 10.0])
def test_tree_few_rows(cuda, dt, D, ps, T, Hq, Hkv, cap):
    """One to nine rows a group: around the eight that share a warp's lanes."""
    _run(cuda, 4, T, Hq, Hkv, D, [0, 31, 400, 129], [T, T, T - 1, T], dt, dt, ps, cap, big=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("T,Hq,Hkv", [(6, 3, 1), (4, 10, 2), (9, 7, 1), (3, 24, 1), (2, 40, 2), (2, 130, 1), (11, 48, 4)])
def test_tree_head_groups(cuda, dt, T, Hq, Hkv):
    """Groups that no power of two divides, and one of more heads than a tile has rows."""
    _run(cuda, 2, T, Hq, Hkv, 64, [77, 300], [T, T], dt, dt, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("cap,big", [(50.0, 8.0), (1.0, 4.0), (30.0, 40.0)])
def test_tree_caps(cuda, dt, cap, big):
    """Scores far inside, around and far beyond the cap."""
    _run(cuda, 2, 6, 4, 2, 128, [200, 77], [6, 6], dt, dt, 16, cap=cap, big=big)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("cap", [1e-40, 1e-6, 2e3, 1e9, 3e38])
def test_tree_extreme_caps(cuda, dt, cap):
    """Caps that leave nothing of the scores, and caps that none of them feels: no larger errors than without."""
    gen = torch.Generator().manual_seed(11)
    q, k, v = torch.randn(1, 6, 4, 64, generator=gen).to(dt), *(torch.randn(1, 2, 206, 64, generator=gen).to(dt) for _ in range(2))
    q[0, 2] = 0
    mask = _masks(1, 6, gen)[0]
    out = bk.tree_attention(q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor([200], dtype=torch.int32, device=cuda),
                            mask.to(cuda), softcap=cap).double().cpu()
    for h in range(4):
        o, av, mag = scored.tree(q[0, :, h], k[0, h // 2], v[0, h // 2], 200, 6, mask, 0.125, cap)
        lim = scored.bound(o, av, mag, dt, 206, 64, min(cap, float(mag.max())))  # the tanh is off by 3e-7 of the score
        assert bool(((out[0, :, h] - o).abs() <= lim).all())


@pytest.mark.gpu
def test_tree_many_requests(cuda):
    """More requests than CTAs and than a scan's round, most of them short."""
    B = 700
    ctx = [(37 * i) % 90 for i in range(B)]
    _run(cuda, B, 2, 2, 1, 64, ctx, [1 + i % 2 for i in range(B)], BF16, BF16, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
def test_tree_hidden_values_do_not_count(cuda, dt):
    """A drafted token that another row must not see holds infinities and NaN: only the rows that see it may show
    them."""
    gen = torch.Generator().manual_seed(4)
    B, T, Hq, Hkv, D, ctx = 1, 8, 4, 2, 128, 150
    q = torch.randn(B, T, Hq, D, generator=gen).to(dt)
    k, v = (torch.randn(B, Hkv, ctx + T, D, generator=gen).to(dt) for _ in range(2))
    mask = torch.eye(T, dtype=torch.bool)
    mask[5] = torch.tensor([1, 0, 1, 0, 0, 1, 0, 0], dtype=torch.bool)
    mask[7, 7] = False  # a padded token: sees the context, nobody sees it
    for bad, where in ((math.inf, 2), (math.nan, 3), (-math.inf, 7)):
        k2, v2 = k.clone(), v.clone()
        v2[:, :, ctx + where, 5:9] = bad
        if where != 2:
            k2[:, :, ctx + where] = bad
        out = bk.tree_attention(q.to(cuda), k2.to(cuda), v2.to(cuda), torch.tensor([ctx], dtype=torch.int32, device=cuda),
                                mask.to(cuda)).cpu()
        sees = mask[:, where]
        ref = bk.tree_attention(q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor([ctx], dtype=torch.int32, device=cuda),
                                mask.to(cuda)).cpu()
        assert torch.isfinite(out[:, ~sees]).all()
        assert (out[:, ~sees].float() - ref[:, ~sees].float()).abs().max() <= 2.0 ** -7
        if where == 2:
            hit = out[:, sees].float()
            assert (hit[..., 5:9] == math.inf).all() and torch.isfinite(hit[..., :5]).all() and torch.isfinite(hit[..., 9:]).all()


@pytest.mark.gpu
def test_tree_rows_that_see_nothing(cuda):
    """No context and a mask row of zeros: 0, not NaN; and T = 0, B = 0."""
    for dt in (BF16, F32):
        q = torch.randn(1, 3, 2, 64).to(dt).to(cuda)
        k = torch.randn(1, 2, 3, 64).to(dt).to(cuda)
        mask = torch.tensor([[1, 0, 0], [0, 0, 0], [1, 0, 1]], dtype=torch.uint8, device=cuda)
        out = bk.tree_attention(q, k, k, torch.zeros(1, dtype=torch.int32, device=cuda), mask)
        assert not out[:, 1].any() and torch.equal(out[:, 0], k[:, :, 0])
        none = bk.tree_attention(q[:, :0], k, k, torch.zeros(1, dtype=torch.int32, device=cuda), mask[:0, :0])
        assert none.shape == (1, 0, 2, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
def test_tree_lengths_beyond_the_cache(cuda, dt):
    """Context and drafted tokens are clamped to the cache's end; negative lengths count as 0."""
    gen = torch.Generator().manual_seed(9)
    q = torch.randn(3, 4, 2, 64, generator=gen).to(dt)
    k, v = (torch.randn(3, 2, 50, 64, generator=gen).to(dt) for _ in range(2))
    mask = torch.tril(torch.ones(4, 4, dtype=torch.bool))
    ctx = [48, 60, -5]
    out = bk.tree_attention(q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor(ctx, dtype=torch.int32, device=cuda),
                            mask.to(cuda), draft_lens=torch.tensor([4, 9, 3], dtype=torch.int32, device=cuda))
    _check(out, q, k, v, ctx, [4, 9, 3], mask, 1 / 8, 0.0, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
def test_tree_strides(cuda, dt):
    """q cut out of a fused projection, a cache with its heads innermost, an out with strides refused."""
    gen = torch.Generator().manual_seed(2)
    B, T, Hq, Hkv, D, ctx = 2, 5, 8, 2, 64, [70, 20]
    qkv = torch.randn(B, T, (Hq + 2 * Hkv) * D, generator=gen).to(dt).to(cuda)
    q = qkv[..., :Hq * D].view(B, T, Hq, D)
    kv = torch.randn(B, 80, 2, Hkv, D, generator=gen).to(dt).to(cuda)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    mask = _masks(B, T, gen)
    i = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)
    out = torch.empty(B, T, Hq, D, dtype=dt, device=cuda)
    assert bk.tree_attention(q, k, v, i(ctx), mask.to(cuda), out=out) is out
    _check(out, q.cpu(), k.cpu(), v.cpu(), ctx, [T] * B, mask, 1 / 8, 0.0, dt)
    odd = torch.randn(B, T, Hq, D + 1, generator=gen).to(dt).to(cuda)[..., :D]  # rows at odd addresses
    _check(bk.tree_attention(odd, k, v, i(ctx), mask.to(cuda)), odd.cpu(), k.cpu(), v.cpu(), ctx, [T] * B, mask, 1 / 8,
           0.0, dt)
    with pytest.raises(errors.B2ShapeError):
        bk.tree_attention(q, k, v, i(ctx), mask.to(cuda), out=out.transpose(1, 2).contiguous().transpose(1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
def test_tree_page_numbers_outside_the_cache(cuda, dt):
    """Such pages read as zeros, from nowhere, and the device error word says so."""
    lib = _lib.load()
    code = ctypes.c_uint(0)
    stream = torch.cuda.current_stream().cuda_stream
    lib.b2_device_error(stream, ctypes.byref(code))
    gen = torch.Generator().manual_seed(7)
    B, T, Hq, Hkv, D, ps, ctx = 1, 4, 4, 2, 64, 16, 90
    q = torch.randn(B, T, Hq, D, generator=gen).to(dt)
    k, v = (torch.randn(B, Hkv, ctx + T, D, generator=gen).to(dt) for _ in range(2))
    kp, vp, table = _paged(k, v, ps, gen)
    table[0, 1], table[0, 3] = -1, kp.shape[0]
    out = bk.tree_attention(q.to(cuda), kp.to(cuda), vp.to(cuda), torch.tensor([ctx], dtype=torch.int32, device=cuda),
                            torch.ones(T, T, dtype=torch.bool, device=cuda), page_table=table.to(cuda)).double().cpu()
    assert lib.b2_device_error(stream, ctypes.byref(code)) == errors.ERR_TIMEOUT and code.value == 0xB2500001
    vis = torch.ones(T, ctx + T, dtype=torch.bool)
    for x in (k, v):
        x[:, :, 16:32] = 0
        x[:, :, 48:64] = 0
    for h in range(Hq):
        o, av, mag = scored.rows(q[0, :, h], k[0, h // 2], v[0, h // 2], vis, 1 / 8)
        assert bool(((out[0, :, h] - o).abs() <= scored.bound(o, av, mag, dt, ctx + T, D)).all())


@pytest.mark.gpu
def test_tree_one_token_is_decode(cuda):
    """T = 1: the same attention as decode_attention over the context and the token itself."""
    gen = torch.Generator().manual_seed(1)
    B, Hq, Hkv, D, S = 3, 16, 4, 128, 700
    q = torch.randn(B, 1, Hq, D, generator=gen).bfloat16().to(cuda)
    k, v = (torch.randn(B, Hkv, S, D, generator=gen).bfloat16().to(cuda) for _ in range(2))
    lens = torch.tensor([700, 1, 333], dtype=torch.int32, device=cuda)
    out = bk.tree_attention(q, k, v, lens - 1, torch.ones(1, 1, dtype=torch.bool, device=cuda))
    dec = bk.decode_attention(q[:, 0], k, v, lens)
    assert (out[:, 0].float() - dec.float()).abs().max() <= 2.0 ** -7


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
def test_tree_graphs_and_streams(cuda, dt):
    """Two captured calls and eager ones in between do not disturb one another; lengths change between replays; the
    same call gives the same bits."""
    gen = torch.Generator().manual_seed(3)
    B, T, Hq, Hkv, D = 3, 6, 8, 2, 128
    q = torch.randn(B, T, Hq, D, generator=gen).to(dt).to(cuda)
    k, v = (torch.randn(B, Hkv, 3000, D, generator=gen).to(dt).to(cuda) for _ in range(2))
    mask = _masks(B, T, gen).to(cuda)
    ctx = torch.tensor([10, 2000, 500], dtype=torch.int32, device=cuda)
    eager = lambda: bk.tree_attention(q, k, v, ctx, mask)
    eager()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(eager())
        graphs.append(g)
    for lens in ([10, 2000, 500], [2900, 0, 64]):
        ctx.copy_(torch.tensor(lens, dtype=torch.int32))
        ref = eager()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref) and torch.equal(eager(), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F16])
def test_tree_far_offsets(cuda, dt):
    """Pages whose element offsets pass 2^31."""
    gen = torch.Generator().manual_seed(6)
    ps, Hkv, D, T, ctx = 64, 8, 128, 5, 200
    n = 2 ** 31 // (ps * Hkv * D) + 8
    kp, vp = (torch.zeros(n, ps, Hkv, D, dtype=dt, device=cuda) for _ in range(2))
    table = torch.tensor([[n - 1, n - 5, 3, n - 2]], dtype=torch.int32)
    q = torch.randn(1, T, Hkv, D, generator=gen).to(dt)
    k, v = (torch.randn(1, Hkv, ctx + T, D, generator=gen).to(dt) for _ in range(2))
    slots = (table[0].long()[:, None] * ps + torch.arange(ps)).reshape(-1)[:ctx + T].to(cuda)
    bk.store_kv(k[0].transpose(0, 1).to(cuda), v[0].transpose(0, 1).to(cuda), kp, vp, slots)
    mask = _masks(1, T, gen)
    out = bk.tree_attention(q.to(cuda), kp, vp, torch.tensor([ctx], dtype=torch.int32, device=cuda), mask.to(cuda),
                            page_table=table.to(cuda))
    _check(out, q, k, v, [ctx], [T], mask, 1 / math.sqrt(D), 0.0, dt)


@pytest.mark.gpu
def test_tree_no_bounded_wait_ran_out(cuda):
    code = ctypes.c_uint(0)
    st = _lib.load().b2_device_error(torch.cuda.current_stream().cuda_stream, ctypes.byref(code))
    assert st == 0 and code.value == 0, hex(code.value)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("T,Hq,Hkv", [(2, 4, 1), (12, 8, 2), (25, 4, 1), (80, 4, 2)])
@pytest.mark.parametrize("ps", [0, 12, 16])
def test_tree_growing_maximum(cuda, dt, D, T, Hq, Hkv, ps):
    """Scores that rise by more than the rescaling threshold (8 in log2) with every 32 keys: O is rescaled several times
    within a tile."""
    gen = torch.Generator().manual_seed(T)
    ctx, B = 500, 1
    q, k, v = scored.growing(B, T, Hq, Hkv, ctx + T, D, dt, gen)
    mask = torch.tril(torch.ones(T, T, dtype=torch.bool))
    kc, vc, table = k, v, None
    if ps:
        kc, vc, table = _paged(k, v, ps, gen)
        table = table.to(cuda)
    out = bk.tree_attention(q.to(cuda), kc.to(cuda), vc.to(cuda), torch.tensor([ctx], dtype=torch.int32, device=cuda),
                            mask.to(cuda), page_table=table)
    _check(out, q, k, v, [ctx], [T], mask, 1 / math.sqrt(D), 0.0, dt)
