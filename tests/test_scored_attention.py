"""Capped and biased scores, document and prefix masks: refusals on the host
(CPU), values on the GPU against the float64 oracle, within the bound that
oracle/scored.py derives from the arithmetic."""
import ctypes
import math

import pytest
import torch

import b200kern as bk
from b200kern import _lib, errors
from oracle import attention as oatt
from oracle import scored

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


# ---------------------------------------------------------------- refusals
class _Cuda(torch.Tensor):
    """A CPU tensor that says it is on a GPU, to reach the checks behind the device's."""
    is_cuda = True


def _t(*shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Cuda)


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("kw,error", [
    (dict(softcap=-1.0), errors.B2ShapeError), (dict(softcap=math.nan), errors.B2ShapeError),
    (dict(alibi_slopes=torch.ones(3)), errors.B2ShapeError), (dict(alibi_slopes=torch.ones(4).half()), errors.B2ShapeError),
    (dict(doc_offsets=_i(2, 1)), errors.B2ShapeError), (dict(doc_offsets=_i(3, 3)), errors.B2ShapeError),
    (dict(doc_offsets=torch.zeros(2, 3)), errors.B2ShapeError),
    (dict(causal=True, prefix_lens=_i(3)), errors.B2ShapeError),
    (dict(causal=True, doc_offsets=_i(2, 3), prefix_lens=_i(2)), errors.B2ShapeError),
    (dict(prefix_lens=_i(2)), errors.B2ShapeError), (dict(causal=True, window=4, prefix_lens=_i(2)), errors.B2ShapeError),
    (dict(window=4, softcap=1.0), errors.B2ShapeError)])
def test_flash_attention_refuses(kw, error):
    with pytest.raises(error):
        bk.flash_attention(_t(2, 4, 8, 64), _t(2, 2, 8, 64), _t(2, 2, 8, 64), **kw)


def test_flash_attention_refuses_unequal_lengths():
    for kw in (dict(causal=True, softcap=1.0), dict(doc_offsets=_i(2, 2))):
        with pytest.raises(errors.B2ShapeError):
            bk.flash_attention(_t(2, 4, 8, 64), _t(2, 2, 9, 64), _t(2, 2, 9, 64), **kw)


@pytest.mark.parametrize("kw", [dict(softcap=-1.0), dict(softcap=math.inf), dict(alibi_slopes=torch.ones(2))])
def test_decode_attention_refuses(kw):
    with pytest.raises(errors.B2ShapeError):
        bk.decode_attention(_t(2, 4, 64), _t(2, 2, 8, 64), _t(2, 2, 8, 64), [1, 2], **kw)


def test_c_entries_refuse_without_gpu():
    lib = _lib.load()
    s = _lib.strides_arg((64, 64, 64))

    def fa(B=1, Hq=4, Hkv=2, S=8, K=8, D=64, causal=1, window=0, cap=0.0, docs=None, n=0, pre=None, dt=0, scale=1.0, q=1):
        return lib.b2_flash_attn_fwd_scored(q, 1, 1, 1, B, Hq, Hkv, S, K, D, s, s, s, s, scale, causal, window, cap, None,
                                            docs, n, pre, dt, None)
    assert fa(q=None) == errors.ERR_INVALID
    assert fa(Hq=5) == errors.ERR_INVALID
    assert fa(K=9) == errors.ERR_INVALID
    assert fa(causal=0, K=9, docs=1, n=1) == errors.ERR_INVALID
    assert fa(causal=0, window=3) == errors.ERR_INVALID
    assert fa(causal=0, pre=1) == errors.ERR_INVALID
    assert fa(window=3, pre=1) == errors.ERR_INVALID
    assert fa(docs=1, n=0) == errors.ERR_INVALID
    assert fa(cap=-1.0) == errors.ERR_INVALID
    assert fa(scale=math.inf) == errors.ERR_INVALID
    assert fa(dt=5) == errors.ERR_DTYPE
    assert fa(D=300) == errors.ERR_UNSUPPORTED
    assert fa(S=0, K=0) == errors.OK
    st = lib.b2_decode_attn_scored(1, 1, 1, 1, None, 1, None, 1, 4, 2, 64, 8, 0, 0, 0, s, s, None, 0, None, 1.0, -1.0,
                                   None, 0, 0, None)
    assert st == errors.ERR_INVALID


# ----------------------------------------------------------------- prompts
def _slopes(h):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], dtype=F32)


def _check_flash(cuda, q, k, v, causal=False, window=0, cap=0.0, slopes=None, docs=None, prefix=None, scale=None,
                 vis=None, out=None):
    """One call, every row of every head against the oracle."""
    B, Hq, S, D = q.shape
    rep, dt = Hq // k.shape[1], q.dtype
    dev = lambda t: None if t is None else t.to(cuda)
    if out is None:
        out = bk.flash_attention(dev(q), dev(k), dev(v), causal=causal, window=window, softcap=cap, scale=scale,
                                 alibi_slopes=dev(slopes), doc_offsets=dev(docs), prefix_lens=dev(prefix))
    assert out.dtype == dt and out.shape == q.shape
    out = out.double().cpu()
    sc = 1 / math.sqrt(D) if scale is None else scale
    pos, kpos = torch.arange(S).double(), torch.arange(k.shape[2]).double()
    far = (pos[:, None] - kpos).abs()
    for b in range(B):
        pre = None if prefix is None else prefix[b].reshape(-1).tolist()
        vis = scored.ranges(S, k.shape[2], causal, window, None if docs is None else docs[b].tolist(), pre)
        for h in range(Hq):
            bias = None if slopes is None else -slopes[h].double() * far
            o, av, mag = scored.rows(q[b, h], k[b, h // rep], v[b, h // rep], vis, sc, cap, bias)
            # a weight matters down to 2^-40; a bias beyond that hides its key anyway
            dist = 0.0 if slopes is None else min(float(slopes[h]) * S, 60.0)
            lim = scored.bound(o, av, mag, dt, k.shape[2], D, cap, dist)
            err = (out[b, h] - o).abs()
            assert bool((err <= lim).all()), f"b={b} h={h}: {(err / lim).max().item():.3g} of the bound"


def _qkv(B, Hq, Hkv, S, D, dt, seed, big=1.0, Skv=None):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(B, Hq, S, D, generator=g) * big).to(dt)
    k, v = (torch.randn(B, Hkv, S if Skv is None else Skv, D, generator=g).to(dt) for _ in range(2))
    return q, k, v


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64), (F32, 128), (BF16, 80), (F16, 256)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S,cap,alibi", [(1, 5.0, True), (127, 50.0, False), (128, 0.0, True), (300, 30.0, True),
                                         (513, 2.0, False)])
def test_capped_and_biased(cuda, dt, D, causal, S, cap, alibi):
    q, k, v = _qkv(2, 4, 2, S, D, dt, S + D, big=6.0)
    _check_flash(cuda, q, k, v, causal=causal, cap=cap, slopes=_slopes(4) if alibi else None)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("offsets", [
    [[0, 300], [0, 1]], [[0, 128, 300], [5, 130, 131]], [[0, 0, 0, 10, 200, 200], [100, 101, 102, 103, 104, 290]],
    [[0, 1, 2, 3, 4, 300], [299, 299, 299, 299, 299, 300]], [[0, 64, 127, 129, 256, 257], [0, 0, 0, 0, 0, 0]],
    [[-7, 20, 400, 500, 600, 700], [250, 250, 260, 261, 262, 900]]])
def test_documents(cuda, dt, D, causal, offsets):
    """Empty documents, documents of one token, across and at tile borders, padding before and behind, rows without
    any, offsets beyond the row."""
    q, k, v = _qkv(2, 4, 2, 300, D, dt, len(offsets[0]))
    _check_flash(cuda, q, k, v, causal=causal, docs=torch.tensor(offsets, dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 128), (F32, 128)])
def test_documents_with_everything(cuda, dt, D):
    q, k, v = _qkv(2, 8, 2, 700, D, dt, 11, big=4.0)
    docs = torch.tensor([[0, 130, 140, 600], [20, 300, 300, 700]], dtype=torch.int32)
    _check_flash(cuda, q, k, v, causal=True, docs=docs, cap=20.0, slopes=_slopes(8),
                 prefix=torch.tensor([[50, 3, 460], [0, 9, 150]], dtype=torch.int32))
    _check_flash(cuda, q, k, v, causal=True, docs=docs, window=100, cap=20.0)
    _check_flash(cuda, q, k, v, causal=False, docs=docs, slopes=_slopes(8))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 128), (F32, 64)])
@pytest.mark.parametrize("S,prefix", [(1, [1, 0, 5]), (129, [0, 128, 129]), (400, [1, 257, 1000]), (300, [-3, 40, 2 ** 31 - 1])])
def test_prefixes(cuda, dt, D, S, prefix):
    q, k, v = _qkv(3, 2, 2, S, D, dt, S)
    _check_flash(cuda, q, k, v, causal=True, prefix=torch.tensor(prefix, dtype=torch.int32))
    _check_flash(cuda, q, k, v, causal=True, prefix=torch.tensor(prefix, dtype=torch.int32), slopes=_slopes(2))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("S,Skv", [(5, 1), (130, 700), (700, 130), (64, 0)])
def test_other_key_counts(cuda, dt, S, Skv):
    """Cross attention (not causal), also over no keys at all."""
    q, k, v = _qkv(1, 4, 2, S, 64, dt, S, Skv=Skv, big=3.0)
    _check_flash(cuda, q, k, v, cap=10.0, slopes=_slopes(4))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.5])
def test_scales_of_any_sign(cuda, dt, scale):
    q, k, v = _qkv(1, 2, 1, 200, 64, dt, 5)
    _check_flash(cuda, q, k, v, causal=True, cap=8.0, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64)])
def test_hidden_values_do_not_count(cuda, dt, D):
    """Infinities and NaN in padding, in another document and behind the query reach nobody who must not see them,
    and reach those who do."""
    q, k, v = _qkv(1, 4, 2, 600, D, dt, 3)
    docs = torch.tensor([[10, 200, 450, 580]], dtype=torch.int32)
    clean = bk.flash_attention(q.to(cuda), k.to(cuda), v.to(cuda), causal=True, doc_offsets=docs.to(cuda)).cpu()
    q2, k2, v2 = q.clone(), k.clone(), v.clone()
    for x in (q2, k2, v2):
        x[:, :, :10] = math.nan
        x[:, :, 580:] = math.inf
    v2[:, :, 300, 7] = math.inf       # seen by the queries 300 .. 449 of the second document
    v2[:, :, 440, 9] = math.nan
    out = bk.flash_attention(q2.to(cuda), k2.to(cuda), v2.to(cuda), causal=True, doc_offsets=docs.to(cuda)).cpu()
    far = 2.0 ** -6
    assert not out[:, :, :10].any() and not out[:, :, 580:].any()
    assert torch.isfinite(out[:, :, :300]).all() and torch.isfinite(out[:, :, 450:]).all()
    assert (out[:, :, :300].float() - clean[:, :, :300].float()).abs().max() <= far
    assert (out[:, :, 450:].float() - clean[:, :, 450:].float()).abs().max() <= far
    assert (out[:, :, 300:450, 7] == math.inf).all() and torch.isnan(out[:, :, 440:450, 9]).all()
    rest = [d for d in range(D) if d not in (7, 9)]
    assert (out[:, :, 300:450][..., rest].float() - clean[:, :, 300:450][..., rest].float()).abs().max() <= far
    assert torch.isfinite(out[:, :, 300:440, 9]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
def test_strided_and_given_out(cuda, dt):
    """q, k, v as views of one projection [B, S, H, D], an out of that layout, odd addresses."""
    g = torch.Generator().manual_seed(1)
    B, S, Hq, Hkv, D = 2, 250, 4, 2, 64
    for odd in (0, 1):
        qkv = torch.randn(B, S, (Hq + 2 * Hkv) * D + 8, generator=g).to(dt)[..., odd:]
        part = lambda a, n: qkv[..., a * D:(a + n) * D].unflatten(2, (n, D)).transpose(1, 2)
        q, k, v = part(0, Hq), part(Hq, Hkv), part(Hq + Hkv, Hkv)
        dq = qkv.to(cuda)
        dpart = lambda a, n: dq[..., a * D:(a + n) * D].unflatten(2, (n, D)).transpose(1, 2)
        o = torch.full((B, S, Hq, D), 7.0, dtype=dt, device=cuda).transpose(1, 2)
        docs = torch.tensor([[0, 100, 250], [0, 240, 240]], dtype=torch.int32)
        res = bk.flash_attention(dpart(0, Hq), dpart(Hq, Hkv), dpart(Hq + Hkv, Hkv), causal=True, out=o,
                                 doc_offsets=docs.to(cuda), softcap=30.0)
        assert res is o
        _check_flash(cuda, q, k, v, causal=True, docs=docs, cap=30.0, out=o)


@pytest.mark.gpu
def test_many_tiles_and_heads(cuda):
    """Q-tile pairs (a grid of more than one CTA per SM), long documents beside short ones."""
    q, k, v = _qkv(2, 16, 4, 2500, 128, BF16, 8)
    docs = torch.tensor([[0, 1700, 1710, 2400, 2500], [3, 256, 1024, 1025, 2049]], dtype=torch.int32)
    _check_flash(cuda, q, k, v, causal=True, docs=docs)
    _check_flash(cuda, q, k, v, causal=True, cap=50.0, slopes=_slopes(16))


@pytest.mark.gpu
def test_graph_follows_offsets(cuda):
    q, k, v = (t.to(cuda) for t in _qkv(1, 4, 2, 400, 128, BF16, 2))
    docs = torch.tensor([[0, 100, 400]], dtype=torch.int32, device=cuda)
    run = lambda: bk.flash_attention(q, k, v, causal=True, doc_offsets=docs, softcap=20.0)
    run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for off in ([0, 100, 400], [0, 128, 129], [50, 60, 300]):
        docs.copy_(torch.tensor([off], dtype=torch.int32))
        g.replay()
        assert torch.equal(out, run())


# ----------------------------------------------------------- single tokens
@pytest.mark.gpu
@pytest.mark.parametrize("qd,kd", [(BF16, BF16), (F16, F16), (F32, F32), (F32, F16)])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("B,Hq,Hkv,S,D,cap,alibi,window", [
    (1, 8, 2, 70, 64, 30.0, False, 0), (3, 16, 1, 900, 128, 5.0, True, 0), (2, 4, 4, 300, 256, 0.0, True, 90),
    (40, 8, 2, 200, 128, 50.0, True, 0)])
def test_decode(cuda, qd, kd, paged, B, Hq, Hkv, S, D, cap, alibi, window):
    g = torch.Generator().manual_seed(S + B)
    q = (torch.randn(B, Hq, D, generator=g) * 5).to(qd)
    k, v = (torch.randn(B, Hkv, S, D, generator=g).to(kd) for _ in range(2))
    lens = torch.randint(0, S + 1, (B,), generator=g)
    lens[0] = S
    slopes = _slopes(Hq) if alibi else None
    kc, vc, table = k, v, None
    if paged:
        ps = 24
        width = -(-S // ps)
        table = torch.randperm(B * width, generator=g).reshape(B, width).to(torch.int32)
        pages = []
        for x in (k, v):
            pad = torch.zeros(B, Hkv, width * ps, D, dtype=kd)
            pad[:, :, :S] = x
            pg = torch.empty(B * width, ps, Hkv, D, dtype=kd)
            pg[table.reshape(-1).long()] = pad.view(B, Hkv, width, ps, D).permute(0, 2, 3, 1, 4).reshape(-1, ps, Hkv, D)
            pages.append(pg)
        kc, vc = pages
        table = table.to(cuda)
    out = bk.decode_attention(q.to(cuda), kc.to(cuda), vc.to(cuda), lens.to(cuda), page_table=table, softcap=cap,
                              alibi_slopes=None if slopes is None else slopes.to(cuda), window=window).double().cpu()
    for b in range(B):
        n = int(lens[b])
        vis = torch.zeros(1, S, dtype=torch.bool)
        vis[0, max(0, n - window) if window else 0:n] = True
        far = (n - 1 - torch.arange(S).double()).abs()[None]
        for h in range(Hq):
            bias = None if slopes is None else -slopes[h].double() * far
            o, av, mag = scored.rows(q[b, h:h + 1], k[b, h // (Hq // Hkv)], v[b, h // (Hq // Hkv)], vis, 1 / math.sqrt(D),
                                     cap, bias)
            # the type whose roundings show: 16 bits of weights where q and cache are, else q's
            lim = scored.bound(o, av, mag, qd, S, D, cap, 0.0 if slopes is None else min(float(slopes[h]) * S, 60.0))
            assert bool(((out[b, h:h + 1] - o).abs() <= lim).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D,window", [(BF16, 64, 0), (F16, 128, 0), (F32, 64, 0), (BF16, 128, 150), (F16, 256, 0)])
@pytest.mark.parametrize("cap", [1e-40, 1e-6, 2e3, 1e9, 3e38])
def test_extreme_caps(cuda, dt, D, window, cap):
    """Caps that leave nothing of the scores, and caps that none of them feels: no larger errors than without."""
    g = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn(1, 2, 200, D, generator=g).to(dt) for _ in range(3))
    q[:, :, 199] = 0
    vis = scored.ranges(200, 200, True, window)
    out = bk.flash_attention(q.to(cuda), k.to(cuda), v.to(cuda), causal=True, window=window, softcap=cap).double().cpu()
    one = bk.decode_attention(q[:, :, 150].to(cuda), k.to(cuda), v.to(cuda), torch.tensor([200], device=cuda),
                              softcap=cap, window=window).double().cpu()
    for h in range(2):
        for got, qq, vv in ((out[0, h], q[0, h], vis), (one[:, h], q[0, h, 150:151], vis[199:])):
            o, av, mag = scored.rows(qq, k[0, h], v[0, h], vv, 1 / math.sqrt(D), cap)
            lim = scored.bound(o, av, mag, dt, 200, D, min(cap, float(mag.max())))  # the tanh is off by 3e-7 of the score
            assert bool(((got - o).abs() <= lim).all()), (h, ((got - o).abs() / lim).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("ps", [1, 4, 8, 12, 16, 32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv,cap,alibi", [(8, 8, 30.0, False), (6, 2, 0.0, True), (40, 1, 20.0, True)])
def test_decode_page_sizes(cuda, dt, D, ps, Hq, Hkv, cap, alibi):
    """Every way to load the cache, with infinities behind the last key."""
    g = torch.Generator().manual_seed(ps + D)
    lens = [0, 1, 129, 777]
    B, S = len(lens), max(lens)
    q = (torch.randn(B, Hq, D, generator=g) * 3).to(dt)
    k, v = (torch.randn(B, Hkv, S, D, generator=g).to(dt) for _ in range(2))
    width = -(-S // ps)
    table = torch.randperm(B * width + 1, generator=g)[:B * width].reshape(B, width)
    pages = []
    for x in (k, v):
        pg = torch.full((B * width + 1, ps, Hkv, D), math.inf, dtype=dt)
        for b, n in enumerate(lens):
            at = torch.arange(n)
            pg[table[b, at // ps], at % ps] = x[b, :, :n].transpose(0, 1)
        pages.append(pg.to(cuda))
    slopes = _slopes(Hq) if alibi else None
    out = bk.decode_attention(q.to(cuda), *pages, torch.tensor(lens, device=cuda), softcap=cap,
                              page_table=table.to(torch.int32).to(cuda),
                              alibi_slopes=None if slopes is None else slopes.to(cuda)).double().cpu()
    for b, n in enumerate(lens):
        far = (n - 1 - torch.arange(n).double())[None]
        for h in range(Hq):
            o, av, mag = scored.rows(q[b, h:h + 1], k[b, h // (Hq // Hkv), :n], v[b, h // (Hq // Hkv), :n],
                                     torch.ones(1, n, dtype=torch.bool), 1 / math.sqrt(D), cap,
                                     None if slopes is None else -slopes[h].double() * far)
            lim = scored.bound(o, av, mag, dt, n, D, cap, 0.0 if slopes is None else min(float(slopes[h]) * S, 60.0))
            assert bool(((out[b, h:h + 1] - o).abs() <= lim).all()), (b, h)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
def test_decode_rope_and_score_forms(cuda, dt):
    """RoPE and a query position together with cap and bias (distances count from q_pos)."""
    g = torch.Generator().manual_seed(0)
    B, Hq, Hkv, S, D = 2, 4, 2, 400, 64
    q = (torch.randn(B, Hq, D, generator=g) * 3).to(dt)
    k, v = (torch.randn(B, Hkv, S, D, generator=g).to(dt) for _ in range(2))
    lens, qpos = [400, 123], [350, 122]
    freqs = 1.0 / 10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)
    out = bk.decode_attention(q.to(cuda), k.to(cuda), v.to(cuda), lens, q_pos=qpos, rope_freqs=freqs.float(), softcap=9.0,
                              alibi_slopes=_slopes(Hq).to(cuda)).double().cpu()
    for b in range(B):
        n = lens[b]
        kr = torch.from_numpy(oatt.rope_rotate(k[b].double().numpy(), torch.arange(S).double().numpy(), freqs.float().double().numpy()))
        for h in range(Hq):
            qr = torch.from_numpy(oatt.rope_rotate(q[b, h:h + 1].double().numpy(), qpos[b], freqs.float().double().numpy()))
            vis = (torch.arange(S) < n)[None]
            bias = -_slopes(Hq)[h].double() * (qpos[b] - torch.arange(S).double()).abs()[None]
            o, av, mag = scored.rows(qr, kr[h // 2], v[b, h // 2], vis, 1 / 8, 9.0, bias)
            # rotated q and K are rounded once more: half a step of each, on scores of mag
            extra = 4 * torch.finfo(dt).eps / 2 * mag * av if dt != F32 else 4 * 2.0 ** -22 * mag * av
            assert bool(((out[b, h:h + 1] - o).abs() <= scored.bound(o, av, mag, dt, S, D, 9.0, 60.0) + extra).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
def test_decode_page_numbers_outside_the_cache(cuda, dt):
    """Read as zeros, from nowhere, and recorded in the device error word (also without score forms)."""
    lib = _lib.load()
    code, stream = ctypes.c_uint(0), torch.cuda.current_stream().cuda_stream
    lib.b2_device_error(stream, ctypes.byref(code))
    g = torch.Generator().manual_seed(5)
    kp, vp = (torch.randn(3, 16, 1, 64, generator=g).to(dt) for _ in range(2))
    q = torch.randn(1, 2, 64, generator=g).to(dt)
    table = torch.tensor([[2, -1, 0, 3]], dtype=torch.int32)
    for cap in (0.0, 4.0):
        out = bk.decode_attention(q.to(cuda), kp.to(cuda), vp.to(cuda), [60], page_table=table.to(cuda),
                                  softcap=cap).double().cpu()
        assert lib.b2_device_error(stream, ctypes.byref(code)) == errors.ERR_TIMEOUT and code.value == 0xB2500001
        zero = torch.zeros(16, 64, dtype=dt)
        k = torch.cat([kp[2, :, 0], zero, kp[0, :, 0], zero])[:60]
        v = torch.cat([vp[2, :, 0], zero, vp[0, :, 0], zero])[:60]
        o, av, mag = scored.rows(q[0], k, v, torch.ones(2, 60, dtype=torch.bool), 1 / 8, cap)
        assert bool(((out[0] - o).abs() <= scored.bound(o, av, mag, dt, 60, 64, cap)).all())


@pytest.mark.gpu
def test_scored_no_bounded_wait_ran_out(cuda):
    code = ctypes.c_uint(0)
    st = _lib.load().b2_device_error(torch.cuda.current_stream().cuda_stream, ctypes.byref(code))
    assert st == 0 and code.value == 0, hex(code.value)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("S", [300, 513])
@pytest.mark.parametrize("alibi", [False, True])
def test_growing_maximum(cuda, dt, D, S, alibi):
    """Scores that rise by more than the rescaling threshold (8 in log2) with every 32 keys, in the order in which the
    keys are taken (a bias takes them from the last one back): O is rescaled several times within a tile, in pieces of
    32 keys and in halves of 64.  Prompts, and single tokens with 2, 12 and 40 rows a kv head."""
    g = torch.Generator().manual_seed(S)
    q, k, v = scored.growing(1, S, 4, 2, S, D, dt, g, down=alibi)
    q = q.transpose(1, 2).contiguous()
    slopes = _slopes(4) / 64 if alibi else None
    docs = torch.tensor([[0, 70, S - 3]], dtype=torch.int32)
    for kw in (dict(docs=docs), dict(docs=docs, causal=True), dict(causal=True, window=200), dict(prefix=torch.tensor(
            [260], dtype=torch.int32), causal=True)):
        _check_flash(cuda, q, k, v, slopes=slopes, **kw)
    for rep in (2, 12, 40):
        q1, k, v = scored.growing(1, 3, 2 * rep, 2, S, D, dt, g, down=alibi)
        sl = _slopes(2 * rep) / 64 if alibi else torch.zeros(2 * rep)
        out = bk.decode_attention(q1[:, 2].to(cuda), k.to(cuda), v.to(cuda), torch.tensor([S], dtype=torch.int32, device=cuda),
                                  alibi_slopes=sl.to(cuda)).double().cpu()
        for h in range(2 * rep):
            bias = -sl[h].double() * (S - 1 - torch.arange(S).double())[None]
            o, av, mag = scored.rows(q1[0, 2, h:h + 1], k[0, h // rep], v[0, h // rep], torch.ones(1, S, dtype=torch.bool),
                                     1 / math.sqrt(D), 0.0, bias)
            assert bool(((out[0, h] - o[0]).abs() <= scored.bound(o, av, mag, dt, S, D, 0.0, float(sl[h]) * S)[0]).all()), (rep, h)
