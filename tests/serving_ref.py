"""Definitions of the serving operators in 64 bits, and their tolerances (imported
by the tests; not a test module)."""

import math

import torch

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
# half a unit in the last place, relative: 11 and 8 significant bits (the value
# halfway from 1 to its upper neighbour, 1 + 2^-11 and 1 + 2^-8, is off by that much)
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attend(q, k, v, scale, visible=None):
    """q [R,hd], k and v [n,hd] -> (out, lse, prob, spread) in 64 bits; ``spread`` is
    sum_u p_u |v_u|.  Only visible keys enter any sum; no key: zeros and -inf."""
    q, k, v = q.double(), k.double(), v.double()
    R, n = q.shape[0], k.shape[0]
    if visible is None:
        visible = torch.ones(R, n, dtype=torch.bool, device=q.device)
    used = visible.any(0)
    k, v, visible = k[used], v[used], visible[:, used]
    prob = torch.zeros(R, n, dtype=torch.float64, device=q.device)
    if k.shape[0] == 0:
        zero = torch.zeros(R, q.shape[1], dtype=torch.float64, device=q.device)
        return zero, torch.full((R,), -math.inf, dtype=torch.float64, device=q.device), prob, zero
    s = (q @ k.T * scale).masked_fill(~visible, -math.inf)
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None])
    prob[:, used] = p
    return p @ v, lse, prob, p @ v.abs()


def out_bound(dtype, ref, spread, n_keys, v_max):
    """Largest error of an attention output: each probability rounded to ``dtype``
    (relative UNIT; in fp16 also 2^-25 of the row's largest below its normal range, per key),
    the output rounded once more, and 1e-5 of the spread for fp32 scores, exponentials
    and sums (scores of a few tens at most)."""
    u = UNIT[dtype]
    tiny = n_keys * 2.0 ** -25 * v_max if dtype == torch.float16 else 0.0
    store = 2.0 ** -25 if dtype == torch.float16 else 0.0   # output below fp16's normal range
    return u * (1 + 2 * u) * (spread + ref.abs()) + 1e-5 * spread + tiny + store


def prompt_ref(q, k, v, lens, scale):
    """(out [T,Hq,hd], lse [T,Hq], bound [T,Hq,hd]) of packed causal prompts."""
    T, Hq, hd = q.shape
    g = Hq // k.shape[1]
    out = torch.zeros(T, Hq, hd, dtype=torch.float64, device=q.device)
    lse = torch.zeros(T, Hq, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    a = 0
    for n in lens:
        causal = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        for h in range(Hq):
            if n == 0:
                continue
            vh = v[a:a + n, h // g]
            o, ls, _, spread = attend(q[a:a + n, h], k[a:a + n, h // g], vh, scale, causal)
            out[a:a + n, h], lse[a:a + n, h] = o, ls
            bound[a:a + n, h] = out_bound(q.dtype, o, spread, n, float(vh.abs().max()))
        a += n
    return out, lse, bound


def decode_ref(q, pk, pv, kc, vc, lengths, scale):
    """(out, bound, weights [B,Hkv,C]) of one decode step over prefix and caches."""
    B, Hq, hd = q.shape
    C, Hkv = kc.shape[1], kc.shape[2]
    g = Hq // Hkv
    P = pk.shape[0]
    out = torch.zeros(B, Hq, hd, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    weights = torch.zeros(B, Hkv, C, dtype=torch.float64, device=q.device)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), C)
        for j in range(Hkv):
            hs = slice(j * g, (j + 1) * g)
            k = torch.cat([pk[:, j], kc[b, :n, j]])
            v = torch.cat([pv[:, j], vc[b, :n, j]])
            o, _, prob, spread = attend(q[b, hs], k, v, scale)
            out[b, hs] = o
            vmax = float(v.abs().max()) if v.numel() else 0.0
            bound[b, hs] = out_bound(q.dtype, o, spread, P + n, vmax)
            weights[b, j, :n] = prob[:, P:].sum(0)
    return out, bound, weights


def evict_ref(weights, lengths, capacity, budget, recent):
    """Kept rows per (sequence, head): a nested list of ascending row indices."""
    kept = []
    for b, row in enumerate(weights.tolist()):
        n = min(max(int(lengths[b]), 0), capacity)
        per_head = []
        for w in row:
            if n <= budget:
                per_head.append(list(range(n)))
                continue
            old = [(-math.inf if math.isnan(x) else x) for x in w[:n - recent]]
            best = sorted(range(n - recent), key=lambda i: (-old[i], i))[:budget - recent]
            per_head.append(sorted(best) + list(range(n - recent, n)))
        kept.append(per_head)
    return kept
