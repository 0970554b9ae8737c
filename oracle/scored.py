"""Oracle for attention with masks, capped and biased scores (torch, float64).

TEST INFRASTRUCTURE ONLY: imported by tests/ for the right values.  Never the
product.  The definition, one (request, head) at a time:

  s_ij = cap tanh(scale q_i.k_j / cap) + bias_ij      (cap 0: scale q_i.k_j)
  o_i  = sum_j w_ij v_j,  w_i = softmax of s_i over the visible keys j

A hidden key does not count whatever its K and V hold; a row that sees nothing
gives 0.  Beside o, ``rows`` returns what an error bound needs: sum_j w_ij
|v_j| and the largest sum_d |q_id k_jd| |scale| of a row's visible keys.
"""
import torch


def rows(q, k, v, vis, scale, cap=0.0, bias=None):
    """q [R, D], k / v [S, D], vis bool [R, S] -> o, |w||v| [R, D], |q||k| [R, 1] in float64."""
    q, k, v = q.double(), k.double(), v.double()
    seen = vis.any(0)
    k, v = (torch.where(seen[:, None], x, torch.zeros_like(x)) for x in (k, v))
    if k.shape[0] == 0:
        z = torch.zeros_like(q)
        return z, z.clone(), z[:, :1].clone()
    s = (q * scale) @ k.t()
    if cap:
        s = cap * torch.tanh(s / cap)
    if bias is not None:
        s = s + bias
    s = torch.where(vis, s, torch.full_like(s, -torch.inf))
    w = torch.where(vis.any(1, keepdim=True), torch.softmax(s, 1), torch.zeros_like(s))
    mag = torch.where(vis, (q.abs() * abs(scale)) @ k.abs().t(), torch.zeros_like(s)).amax(1, keepdim=True)
    return w @ v, w @ v.abs(), mag


def tree(q, k, v, context, draft, mask, scale, cap=0.0):
    """Drafted tokens q [T, D] of one request and head over its keys k / v [context + draft, D] (float64).

    mask bool [T, T]; tokens t >= draft give 0."""
    T, n = q.shape[0], context + draft
    vis = torch.zeros(T, n, dtype=torch.bool, device=q.device)
    vis[:draft, :context] = True
    vis[:draft, context:] = mask[:draft, :draft].bool()
    return rows(q, k[:n], v[:n], vis, scale, cap)


def ranges(S, Skv, causal=False, window=0, docs=None, prefix=None):
    """vis bool [S, Skv] of a prompt: causal, sliding window, documents (offsets, ascending) and a prefix length per
    document (without documents: one)."""
    vis = torch.zeros(S, Skv, dtype=torch.bool)
    pieces = [(0, max(S, Skv))] if docs is None else list(zip(docs[:-1], docs[1:]))
    for d, (a, z) in enumerate(pieces):
        for i in range(max(a, 0), min(z, S)):
            hi = z
            if causal:
                hi = min(z, max(i + 1, a + (prefix[d] if prefix is not None else 0)))
            lo = max(a, i - window + 1) if window else a
            vis[i, max(lo, 0):min(hi, Skv)] = True
    return vis


def bound(o, av, mag, dtype, keys, D, cap=0.0, dist=0.0):
    """How far an output may be off, from the arithmetic (per element).

    Scores: D fp32 products and sums, (D + 4) 2^-24 |q||k|; a cap adds 3e-7 of
    itself, a distance bias its own rounding, 2^-23 of its size ``dist``.  A
    score error e changes an output by at most 2 e sum w|v|.  Weights: fp32
    exponentials and sums of ``keys`` terms, and in the 16-bit kernels one
    rounding of each weight (half a step) and a cubic of 7.5e-5 in the
    exponential.  The output itself is rounded once."""
    half = torch.finfo(dtype).eps / 2
    serr = (D + 4) * 2.0 ** -24 * mag + cap * 3e-7 + dist * 2.0 ** -23
    weights = (keys + 16) * 2.0 ** -24 + (half + 1e-4 if dtype != torch.float32 else 0.0)
    return half * o.abs() + av * (2 * serr + weights) + 1e-30


def growing(B, T, Hq, Hkv, S, D, dtype, gen, down=False):
    """q [B, T, Hq, D], k and v [B, Hkv, S, D] whose scores (scale D^-1/2) rise by 6 to 9 (8.6 to 13 in log2) with every
    32 keys, towards the last key, or with ``down`` towards the first; each row at its own rate."""
    q = (1.0 + torch.arange(T)[:, None] % 3 / 4).expand(T, Hq)[None, ..., None].expand(B, T, Hq, D)
    step = torch.arange(S) // 32
    step = step.flip(0) if down else step
    k = (6.0 / D ** 0.5 * step)[None, None, :, None].expand(B, Hkv, S, D) + torch.randn(B, Hkv, S, D, generator=gen) / 16
    v = torch.randn(B, Hkv, S, D, generator=gen)
    return q.to(dtype).contiguous(), k.to(dtype), v.to(dtype)
