"""Page table, slot map and K/V rows of a step: refusals on the host (CPU) and
results on the GPU, which are whole numbers or one rounding and so exact."""
import numpy as np
import pytest
import torch

import b200kern as bk
from b200kern import _lib, errors


# ---------------------------------------------------------------- refusals
def _table_args(B=3, width=4):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    return dict(context_lens=i(B), new_lens=i(B), page_size=16, free_pages=i(5), page_table=i(B, width), max_tokens=8)


@pytest.mark.parametrize("change", [
    dict(context_lens=torch.zeros(3, dtype=torch.int64)), dict(new_lens=torch.zeros(2, dtype=torch.int32)),
    dict(new_lens=torch.zeros(3, 1, dtype=torch.int32)), dict(page_table=torch.zeros(2, 4, dtype=torch.int32)),
    dict(page_table=torch.zeros(4, 3, dtype=torch.int32).t()), dict(page_table=torch.zeros(3, 4)),
    dict(page_table=torch.zeros(1, 4, dtype=torch.int32).expand(3, 4)), dict(page_size=0), dict(max_tokens=-1),
    dict(free_pages=torch.zeros(10, dtype=torch.int32)[::2]), {}])
def test_build_page_table_refuses(change):
    """Wrong types, shapes and strides; the last case is in order but on the CPU."""
    with pytest.raises(errors.B2ShapeError):
        bk.build_page_table(**{**_table_args(), **change})


def _store_args(N=4, dt=torch.float32, ct=torch.float16):
    r, c = torch.zeros(N, 2, 8, dtype=dt), torch.zeros(3, 4, 2, 8, dtype=ct)
    return dict(k=r, v=r.clone(), k_pages=c, v_pages=c.clone(), slots=torch.zeros(N, dtype=torch.int64))


@pytest.mark.parametrize("change,error", [
    (dict(k=torch.zeros(4, 2, 9)), errors.B2ShapeError), (dict(v=torch.zeros(5, 2, 8)), errors.B2ShapeError),
    (dict(slots=torch.zeros(4, dtype=torch.int32)), errors.B2ShapeError),
    (dict(slots=torch.zeros(5, dtype=torch.int64)), errors.B2ShapeError),
    (dict(k_pages=torch.zeros(3, 4, 1, 8, dtype=torch.float16)), errors.B2ShapeError),
    (dict(k_pages=torch.zeros(1, 4, 2, 8, dtype=torch.float16).expand(3, 4, 2, 8)), errors.B2ShapeError),
    (dict(v_pages=torch.zeros(3, 4, 2, 8, dtype=torch.bfloat16)), errors.B2DtypeError),
    (dict(k=torch.zeros(4, 2, 8).half(), v=torch.zeros(4, 2, 8).half(), k_pages=torch.zeros(3, 4, 2, 8),
          v_pages=torch.zeros(3, 4, 2, 8)), errors.B2DtypeError),
    ({}, errors.B2ShapeError)])
def test_store_kv_refuses(change, error):
    with pytest.raises(error):
        bk.store_kv(**{**_store_args(), **change})


def test_c_entries_refuse_without_gpu():
    lib = _lib.load()
    s2, s3 = _lib.strides_arg((1, 1, 1)), _lib.strides_arg((1, 1, 1))
    tab = lambda *sizes, table=1: lib.b2_build_page_table(1, 1, 1, table, 1, 1, 1, *sizes, None)
    assert tab(2, 0, 1, 4, 4, 8) == errors.ERR_INVALID       # page size
    assert tab(2, 16, 1, 4, 3, 8) == errors.ERR_INVALID      # rows overlap
    assert tab(2, 16, 1, 4, 4, 1 << 31) == errors.ERR_INVALID
    assert tab(2, 16, 1, 4, 4, 8, table=None) == errors.ERR_INVALID
    st = lambda n, ps, a, b, k=1: lib.b2_store_kv(k, 1, 1, 1, 1, n, 2, 8, 3, ps, s2, s2, s3, s3, a, b, None)
    assert st(4, 0, 0, 0) == errors.ERR_INVALID
    assert st(4, 16, 0, 1) == errors.ERR_DTYPE               # fp16 rows into a bf16 cache
    assert st(4, 16, 0, 2) == errors.ERR_DTYPE
    assert st(4, 16, 0, 0, k=None) == errors.ERR_INVALID
    assert st(0, 16, 0, 0, k=None) == errors.OK              # no rows: nothing to do


# ------------------------------------------------------------------ tables
def _build_ref(ctx, new, ps, free, table, max_tokens):
    """One token after another: the first token of a page that the request does not hold opens it."""
    table = table.copy()
    slots, offsets, used = [], [0], 0
    for b in range(len(ctx)):
        c, n = max(int(ctx[b]), 0), max(int(new[b]), 0)
        opened = {}
        for pos in range(c, c + n):
            pi = pos // ps
            if pi >= -(-c // ps) and pi not in opened:
                opened[pi] = int(free[used]) if used < len(free) else -1
                used += 1
                if pi < table.shape[1]:
                    table[b, pi] = opened[pi]
            page = -1 if pi >= table.shape[1] else int(table[b, pi])
            slots.append(page * ps + pos % ps if page >= 0 else -1)
        offsets.append(offsets[-1] + n)
    assert len(slots) <= max_tokens
    return table, np.array(slots + [-1] * (max_tokens - len(slots))), np.array(offsets), used


def _case(rs, B, ctx_hi, new_hi, ps, extra=2):
    ctx, new = rs.integers(0, ctx_hi + 1, B), rs.integers(0, new_hi + 1, B)
    have = -(-ctx // ps)
    width = int(max(1, (-(-(ctx + new) // ps)).max(initial=0) + extra))
    total = int(have.sum() + (new // ps + 2).sum())
    perm = rs.permutation(total)
    table = np.full((B, width), -7)
    at = 0
    for b in range(B):
        table[b, :have[b]] = perm[at:at + have[b]]
        at += have[b]
    return ctx, new, perm[at:], table


def _run_table(cuda, ctx, new, ps, free, table, max_tokens, pad=0):
    i = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=cuda)
    wide = torch.full((table.shape[0], table.shape[1] + pad), 99, dtype=torch.int32, device=cuda)
    t = wide[:, :table.shape[1]]
    t.copy_(i(table))
    out, slots, offsets, used = bk.build_page_table(i(ctx), i(new), ps, i(free), t, max_tokens)
    assert out is t and (wide[:, table.shape[1]:] == 99).all()
    return t.cpu().numpy(), slots.cpu().numpy(), offsets.cpu().numpy(), int(used)


def _check_table(cuda, ctx, new, ps, free, table, max_tokens, pad=0):
    got = _run_table(cuda, ctx, new, ps, free, table, max_tokens, pad)
    ref = _build_ref(ctx, new, ps, free, table, max_tokens)
    for a, b in zip(got, ref):
        assert np.array_equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("B,ctx_hi,new_hi,ps", [
    (1, 0, 1, 16), (1, 5, 0, 16), (7, 100, 33, 1), (64, 3000, 1, 16), (256, 500, 300, 24), (1023, 90, 3, 8),
    (1024, 90, 5, 16), (1025, 40, 4, 128), (3000, 64, 2, 16), (5, 10, 9000, 64)])
def test_build_page_table(cuda, B, ctx_hi, new_hi, ps):
    """Around the scan's rounds (1024 requests) and the CTAs' 1024 tokens, requests without new tokens among them."""
    rs = np.random.default_rng(B + ps)
    ctx, new, free, table = _case(rs, B, ctx_hi, new_hi, ps)
    n = int(new.sum())
    _check_table(cuda, ctx, new, ps, free, table, n + int(rs.integers(0, 3)) * 700, pad=B % 3)


@pytest.mark.gpu
def test_build_page_table_edges(cuda):
    """No requests, no room, negative lengths, too few free pages, a table that is too narrow."""
    empty = np.zeros(0, int)
    t, s, o, u = _run_table(cuda, empty, empty, 16, [3], np.zeros((0, 4), int), 5)
    assert (s == -1).all() and o.tolist() == [0] and u == 0
    t, s, o, u = _run_table(cuda, [3], [0], 16, empty, np.array([[5]]), 0)
    assert t.tolist() == [[5]] and o.tolist() == [0, 0] and u == 0
    _check_table(cuda, [-4, 20, 7], [18, -3, 30], 16, [9, 8, 7, 6, 5, 4], np.array([[-1] * 4, [1, 2, -1, -1], [3, -1, -1, -1]]), 60)
    _check_table(cuda, [16, 30], [40, 40], 16, [11, 12], np.array([[1, -1, -1, -1, -1], [2, 3, -1, -1, -1]]), 90)
    _check_table(cuda, [16, 30], [40, 40], 16, np.arange(20, 40), np.array([[1, -1], [2, 3]]), 90)


@pytest.mark.gpu
def test_build_page_table_large_page_numbers(cuda):
    """Slots pass 32 bits where page * page_size does."""
    free = np.array([2 ** 31 - 1, 2 ** 30])
    _check_table(cuda, [0, 127], [3, 2], 128, free, np.array([[-1, -1], [2 ** 31 - 2, -1]]), 5)


@pytest.mark.gpu
def test_build_page_table_graph_follows_lengths(cuda):
    """A captured step reads the lengths of each replay, also on a stream of its own."""
    rs = np.random.default_rng(0)
    i = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=cuda)
    ctx, new, free, table = _case(rs, 50, 200, 40, 16, extra=20)
    free = np.concatenate([free, np.arange(9000, 9400)])
    c, n, f, t = i(ctx), i(new), i(free), i(table)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        bk.build_page_table(c, n, 16, f, t.clone(), 3000)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            _, slots, offsets, used = bk.build_page_table(c, n, 16, f, t, 3000)
    for _ in range(3):
        new = rs.integers(0, 50, 50)
        n.copy_(i(new))
        t.copy_(i(table))
        graph.replay()
        torch.cuda.synchronize()
        ref = _build_ref(ctx, new, 16, free, table, 3000)
        assert np.array_equal(t.cpu().numpy(), ref[0]) and np.array_equal(slots.cpu().numpy(), ref[1])
        assert np.array_equal(offsets.cpu().numpy(), ref[2]) and int(used) == ref[3]


# -------------------------------------------------------------------- rows
@pytest.mark.gpu
@pytest.mark.parametrize("src,dst", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                     (torch.float32, torch.float32), (torch.float32, torch.float16),
                                     (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("N,Hkv,D,ps", [(1, 1, 1, 1), (1, 8, 128, 16), (77, 2, 64, 24), (700, 3, 80, 16), (33, 5, 7, 3),
                                        (2500, 8, 128, 64), (40, 40, 256, 16)])
def test_store_kv(cuda, src, dst, N, Hkv, D, ps):
    """Bit for bit what one rounding gives; every other element of the cache stays, and slots outside it are passed
    over."""
    gen = torch.Generator().manual_seed(N + D)
    pages = -(-N // ps) + 2
    slots = torch.randperm(pages * ps, generator=gen)[:N]
    if N > 4:
        slots[N // 2], slots[0], slots[-1] = -1, pages * ps, 1 << 40
    k, v = (torch.randn(N, Hkv, D, generator=gen).to(src) for _ in range(2))
    kp, vp = (torch.randn(pages, ps, Hkv, D, generator=gen).to(dst) for _ in range(2))
    kd, vd = kp.to(cuda), vp.to(cuda)
    out = bk.store_kv(k.to(cuda), v.to(cuda), kd, vd, slots.to(cuda))
    assert out[0] is kd and out[1] is vd
    live = (slots >= 0) & (slots < pages * ps)
    for x, p, d in ((k, kp, kd), (v, vp, vd)):
        p.view(-1, Hkv, D)[slots[live]] = x[live].to(dst)
        assert torch.equal(d.cpu(), p)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1])
def test_store_kv_strides(cuda, shift):
    """Rows cut out of a fused qkv projection, and a contiguous cache [B, Hkv, S, D] as pages of size S; with `shift`
    the rows start at an odd element, so 16-byte accesses are out."""
    gen = torch.Generator().manual_seed(3)
    N, Hkv, D, B, S = 50, 4, 64, 3, 40
    qkv = torch.randn(N, 3 * Hkv * D + 8, generator=gen).bfloat16().to(cuda)
    k = qkv[:, Hkv * D + shift:2 * Hkv * D + shift].view(N, Hkv, D)
    v = qkv[:, 2 * Hkv * D + shift:3 * Hkv * D + shift].view(N, Hkv, D)
    kc = torch.zeros(B, Hkv, S, D, dtype=torch.bfloat16, device=cuda)
    vc = torch.zeros(B, Hkv, S, D + 8, dtype=torch.bfloat16, device=cuda)[..., :D]
    slots = torch.randperm(B * S, generator=gen)[:N].to(cuda)
    bk.store_kv(k, v, kc.transpose(1, 2), vc.transpose(1, 2), slots)
    for x, c in ((k, kc), (v, vc)):
        ref = torch.zeros(B * S, Hkv, D, dtype=torch.bfloat16, device=cuda)
        ref[slots] = x
        assert torch.equal(c.transpose(1, 2).reshape(B * S, Hkv, D), ref)


@pytest.mark.gpu
def test_store_kv_far_offsets(cuda):
    """Element offsets past 2^31: the last page of a cache of 4.3 GB a side."""
    pages, ps, Hkv, D = 2100, 1024, 8, 128
    kp = torch.zeros(pages, ps, Hkv, D, dtype=torch.bfloat16, device=cuda)
    vp = torch.zeros_like(kp)
    k, v = (torch.randn(2, Hkv, D, device=cuda).bfloat16() for _ in range(2))
    bk.store_kv(k, v, kp, vp, torch.tensor([pages * ps - 1, pages * ps - 3], device=cuda))
    assert torch.equal(kp[-1, -1], k[0]) and torch.equal(kp[-1, -3], k[1]) and torch.equal(vp[-1, -1], v[0])
    assert int((kp[-1] != 0).sum()) == int((k != 0).sum()) and not kp[:2].any()


@pytest.mark.gpu
def test_paged_cache_takes_another_stream(cuda):
    stream = torch.cuda.Stream()
    kp = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device=cuda)
    vp = torch.zeros_like(kp)
    k = torch.randn(10, 2, 64, device=cuda).half()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        bk.store_kv(k, k, kp, vp, torch.arange(20, 30, device=cuda))
    stream.synchronize()
    assert torch.equal(kp.view(64, 2, 64)[20:30], k) and torch.equal(vp, kp)
