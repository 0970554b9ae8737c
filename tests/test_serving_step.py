"""A serving loop over one paged cache, its operators used together: the page
table of each step, the K/V rows stored by slot, the prompt's attention, then
steps of drafted trees and of single tokens.  Every output is checked against
float64 attention over the request's tokens, kept on the host in order."""
import math

import pytest
import torch

import b200kern as bk
from oracle import scored

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Host:
    """What each request holds, in order: the oracle's cache."""

    def __init__(self, B, Hkv, D, dt):
        self.k = [torch.empty(0, Hkv, D, dtype=dt) for _ in range(B)]
        self.v = [torch.empty(0, Hkv, D, dtype=dt) for _ in range(B)]

    def lens(self):
        return [len(x) for x in self.k]

    def append(self, k, v, new):
        at = 0
        for b, n in enumerate(new):
            self.k[b] = torch.cat([self.k[b], k[at:at + n]])
            self.v[b] = torch.cat([self.v[b], v[at:at + n]])
            at += n

    def keep(self, lens):
        for b, n in enumerate(lens):
            self.k[b], self.v[b] = self.k[b][:n], self.v[b][:n]


def _near(out, q, k, v, vis, scale, cap, dt, bias=None, dist=0.0):
    """out, q [R, Hq, D]; k, v [S, Hkv, D]."""
    Hq, Hkv, S, D = q.shape[1], k.shape[1], k.shape[0], q.shape[2]
    for h in range(Hq):
        o, av, mag = scored.rows(q[:, h], k[:, h * Hkv // Hq], v[:, h * Hkv // Hq], vis, scale, cap,
                                 None if bias is None else bias[h])
        lim = scored.bound(o, av, mag, dt, S, D, cap, dist)
        assert bool(((out[:, h].double().cpu() - o).abs() <= lim).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D,ps", [(BF16, 128, 16), (F16, 64, 64), (BF16, 64, 12), (F32, 64, 16)])
@pytest.mark.parametrize("cap", [0.0, 25.0])
def test_serving_loop(cuda, dt, D, ps, cap):
    """Packed prompts, three rounds of drafting in which a part of each tree is kept, then single tokens."""
    gen = torch.Generator().manual_seed(D + ps)
    B, Hq, Hkv, T, scale = 4, 8, 2, 6, 1 / math.sqrt(D)
    prompts = [37, 1, 260, 130]
    width, n_pages = 40, 160
    i = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)
    rand = lambda *s: torch.randn(*s, generator=gen).to(dt)
    host = Host(B, Hkv, D, dt)
    # what the allocator's pages held before: anything
    kp, vp = (torch.full((n_pages, ps, Hkv, D), math.nan, dtype=dt, device=cuda) for _ in range(2))
    free = torch.randperm(n_pages, generator=gen).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device=cuda)

    def store(new, k, v):
        """A step's bookkeeping and its rows; returns the request lengths before it."""
        nonlocal free
        ctx = host.lens()
        _, slots, offsets, used = bk.build_page_table(i(ctx), i(new), ps, free.to(cuda), table, k.shape[0])
        bk.store_kv(k.to(cuda), v.to(cuda), kp, vp, slots)
        assert offsets.tolist() == [sum(new[:b]) for b in range(B + 1)]
        free = free[int(used):]
        host.append(k, v, new)
        return ctx

    # prompts, packed into one row
    N = sum(prompts)
    q, k, v = rand(N, Hq, D), rand(N, Hkv, D), rand(N, Hkv, D)
    store(prompts, k, v)
    docs = [sum(prompts[:b]) for b in range(B + 1)]
    lay = lambda x: x.transpose(0, 1)[None].to(cuda)
    out = bk.flash_attention(lay(q), lay(k), lay(v), causal=True, softcap=cap, doc_offsets=i([docs]))[0].transpose(0, 1)
    _near(out, q, k, v, scored.ranges(N, N, True, 0, docs), scale, cap, dt)

    for step in range(3):
        # drafting: a tree of T tokens per request, request 1 drafts fewer
        new = [T, T - 2, T, T]
        n = sum(new)
        q, k, v = rand(B, T, Hq, D), rand(n, Hkv, D), rand(n, Hkv, D)
        ctx = store(new, k, v)
        mask = torch.eye(T, dtype=torch.bool)
        for t in range(1, T):
            mask[t] |= mask[int(torch.randint(0, t, (1,), generator=gen))]
        out = bk.tree_attention(q.to(cuda), kp, vp, i(ctx), mask.to(cuda), draft_lens=i(new), page_table=table,
                                softcap=cap)
        for b in range(B):
            vis = torch.ones(new[b], ctx[b] + new[b], dtype=torch.bool)
            vis[:, ctx[b]:] = mask[:new[b], :new[b]]
            _near(out[b, :new[b]], q[b, :new[b]], host.k[b], host.v[b], vis, scale, cap, dt)
            assert not out[b, new[b]:].any()
        # kept: the first tokens of the tree; what the others opened is given back
        kept = [c + 1 + (step + b) % 3 for b, c in enumerate(ctx)]
        lens = host.lens()
        for b in range(B):
            first, last = -(-kept[b] // ps), -(-lens[b] // ps)
            free = torch.cat([free, table[b, first:last].cpu()])
        host.keep(kept)

    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(Hq)])
    for step in range(3):
        q, k, v = rand(B, Hq, D), rand(B, Hkv, D), rand(B, Hkv, D)
        store([1] * B, k, v)
        out = bk.decode_attention(q.to(cuda), kp, vp, i(host.lens()), page_table=table, softcap=cap,
                                  alibi_slopes=slopes.to(cuda))
        for b in range(B):
            s = len(host.k[b])
            far = (s - 1 - torch.arange(s).double())[None]
            _near(out[b][None], q[b][None], host.k[b], host.v[b], torch.ones(1, s, dtype=torch.bool), scale, cap, dt,
                  [-float(x) * far for x in slopes], min(0.5 * s, 60.0))


@pytest.mark.gpu
def test_serving_step_captured(cuda):
    """One step of page table, store and tree attention in a CUDA graph: each replay follows the lengths on the GPU,
    and a second graph with a workspace of its own runs between the replays of the first."""
    gen = torch.Generator().manual_seed(3)
    B, Hq, Hkv, D, T, ps, dt = 3, 8, 2, 64, 4, 16, BF16
    rand = lambda *s: torch.randn(*s, generator=gen).to(dt).to(cuda)

    def make(n_pages, width):
        kp, vp = (torch.zeros(n_pages, ps, Hkv, D, dtype=dt, device=cuda) for _ in range(2))
        table = torch.randperm(n_pages, generator=gen)[:B * width].reshape(B, width).to(torch.int32).to(cuda)
        ctx, new = (torch.zeros(B, dtype=torch.int32, device=cuda) for _ in range(2))
        free = torch.arange(n_pages, dtype=torch.int32, device=cuda)
        q, k, v = rand(B, T, Hq, D), rand(B * T, Hkv, D), rand(B * T, Hkv, D)
        mask = torch.ones(T, T, dtype=torch.bool, device=cuda).tril()
        old = rand(B, Hkv, width * ps, D), rand(B, Hkv, width * ps, D)

        def step():
            t, slots, _, _ = bk.build_page_table(ctx, new, ps, free, table, B * T)
            bk.store_kv(k, v, kp, vp, slots)
            return bk.tree_attention(q, kp, vp, ctx, mask, draft_lens=new, page_table=t)

        def fill(c, n, seed):
            ctx.copy_(torch.tensor(c, dtype=torch.int32))
            new.copy_(torch.tensor(n, dtype=torch.int32))
            g = torch.Generator().manual_seed(seed)
            perm = torch.randperm(n_pages, generator=g).to(torch.int32)
            held = [-(-x // ps) for x in c]
            table.fill_(-1)
            at = 0
            for b in range(B):
                table[b, :held[b]] = perm[at:at + held[b]].to(cuda)
                at += held[b]
            free[:n_pages - at] = perm[at:].to(cuda)
            for x in (q, k, v):
                x.copy_(torch.randn(x.shape, generator=g).to(dt))
            for pages, o in ((kp, old[0]), (vp, old[1])):
                for b in range(B):
                    pos = torch.arange(c[b], device=cuda)
                    pages[table[b].long()[pos // ps], pos % ps] = o[b, :, :c[b]].transpose(0, 1)

        def check(out, c, n):
            at = 0
            for b in range(B):
                kk, vv = (torch.cat([o[b, :, :c[b]].transpose(0, 1), x[at:at + n[b]]]).cpu()
                          for o, x in ((old[0], k), (old[1], v)))
                vis = torch.ones(n[b], c[b] + n[b], dtype=torch.bool)
                vis[:, c[b]:] = mask[:n[b], :n[b]].cpu()
                _near(out[b, :n[b]], q[b, :n[b]].cpu(), kk, vv, vis, 1 / math.sqrt(D), 0.0, dt)
                assert not out[b, n[b]:].any()
                at += n[b]
        return step, fill, check

    graphs = []
    for n_pages, width in ((60, 12), (150, 40)):
        step, fill, check = make(n_pages, width)
        fill([0] * B, [T] * B, 0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, fill, check))
    for seed, c, n in ((1, [0, 5, 100], [4, 3, 4]), (2, [16, 15, 180], [1, 0, 4]), (3, [130, 0, 0], [4, 4, 4])):
        for graph, out, fill, check in graphs:
            fill(c, n, seed)
        for graph, out, fill, check in graphs:
            graph.replay()
        for graph, out, fill, check in graphs:
            check(out, c, n)
