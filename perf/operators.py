"""Cases and plain forms of the serving operators: attention over packed prompts,
attention of new tokens over a shared prefix and each sequence's own cache, and
eviction from that cache by accumulated attention weight.

``run`` computes an operator in its plain form (elementary torch operations in
32 bits, rounded once at the end) unless ``own`` is true: then it makes the call
a user of the framework makes.  ``exact`` computes the same outputs from the
operators' definitions in 64 bits.
"""

import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


# ------------------------------------------------------------------ the cases

def _prompt(name, dtype, q_heads, kv_heads, head_dim, lens, lse=False):
    return {"name": name, "op": "prompt_attn", "dtype": dtype, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "lens": ",".join(str(n) for n in lens), "lse": lse}


def _decode(name, dtype, q_heads, kv_heads, head_dim, batch, prefix, capacity, len_lo, len_hi, weights):
    return {"name": name, "op": "shared_prefix_attn", "dtype": dtype, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "batch": batch, "prefix": prefix,
            "capacity": capacity, "len_lo": len_lo, "len_hi": len_hi, "weights": weights}


def _evict(name, dtype, kv_heads, head_dim, batch, capacity, len_lo, len_hi, budget, recent):
    return {"name": name, "op": "cache_evict", "dtype": dtype, "kv_heads": kv_heads, "head_dim": head_dim,
            "batch": batch, "capacity": capacity, "len_lo": len_lo, "len_hi": len_hi, "budget": budget,
            "recent": recent}


def listed():
    many = [1 + (i * 97) % 256 for i in range(94)] + [0, 1]
    return [
        # one short request on its own: launch latency
        _prompt("prompt_one_short", "float16", 8, 2, 64, [61]),
        # a burst of short chat turns, one of them empty, admitted together
        _prompt("prompt_many_short", "bfloat16", 32, 8, 128, many),
        # the framework's 8 x 2048 x 1024 layer (16 heads of 64) with ragged prompts, one head per group
        _prompt("prompt_batch_hd64", "float16", 16, 16, 64, [2048, 1901, 2047, 1024, 1777, 2048, 1500, 333]),
        # a mixed batch of documents and questions with grouped heads
        _prompt("prompt_mixed_grouped", "bfloat16", 32, 8, 128, [4096, 3001, 1733, 911, 500, 129, 64, 1], True),
        # one long document with a shorter one beside it: the tensor-bound end
        _prompt("prompt_long", "bfloat16", 32, 4, 128, [16384, 2049]),
        # one sequence decoding after a short system prompt: latency
        _decode("decode_one", "bfloat16", 16, 2, 128, 1, 512, 1024, 700, 700, False),
        # many users behind one long document, short answers so far: the shared part dominates
        _decode("decode_long_prefix", "bfloat16", 32, 8, 128, 64, 32768, 512, 0, 512, False),
        # many users behind a system prompt with long conversations of their own, weights kept for eviction
        _decode("decode_long_caches", "float16", 32, 8, 128, 128, 2048, 4096, 1000, 4096, True),
        # ungrouped heads of 64, odd sizes, some sequences just started
        _decode("decode_ungrouped_hd64", "float16", 16, 16, 64, 33, 1001, 2100, 0, 2100, True),
        # a small batch trimming a short cache: latency
        _evict("evict_small", "bfloat16", 4, 64, 2, 256, 200, 256, 128, 32),
        # a full serving batch cut to half its cache, some sequences below the budget
        _evict("evict_batch", "bfloat16", 8, 128, 64, 4096, 1500, 4096, 2048, 256),
        # few sequences with a very long cache of odd capacity
        _evict("evict_long", "float16", 8, 128, 4, 65537, 60000, 65537, 8192, 1024),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    group = rng.choice([1, 1, 2, 3, 4, 4, 7, 8, 8, 16])
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    while group * kv > 32:
        kv //= 2
    return group * kv, kv


def draw(rng):
    dtype = rng.choice(["float16", "bfloat16"])
    q_heads, kv_heads = _heads(rng)
    head_dim = rng.choice([64, 64, 128, 128, 128, 40, 80, 96, 192, 256])
    op = rng.choice(["prompt_attn", "prompt_attn", "shared_prefix_attn", "shared_prefix_attn", "cache_evict"])
    if op == "prompt_attn":
        longest = _log_int(rng, 1, 8192)
        count = _log_int(rng, 1, 64)
        budget = 8.0e11 / (2.0 * q_heads * head_dim)   # multiply-adds: below prompt_long's
        lens = [longest]
        used = longest ** 2
        for _ in range(count - 1):
            n = rng.choice([0, 1, rng.randint(1, longest), rng.randint(1, longest), longest])
            if used + n * n > budget or sum(lens) + n > 60000:
                break
            lens.append(n)
            used += n * n
        rng.shuffle(lens)
        case = _prompt("", dtype, q_heads, kv_heads, head_dim, lens, rng.random() < 0.3)
    else:
        batch = _log_int(rng, 1, 192)
        room = 5.0e8 / (batch * kv_heads * head_dim)    # cached keys per sequence: below decode_long_caches'
        hi_cap = int(max(2, min(20000, room)))
        capacity = _log_int(rng, min(64, hi_cap), hi_cap)
        len_hi = rng.choice([capacity, rng.randint(1, capacity)])
        len_lo = rng.choice([0, len_hi, rng.randint(0, len_hi)])
        if op == "shared_prefix_attn":
            prefix = rng.choice([0, _log_int(rng, 1, 32768), _log_int(rng, 64, 32768), _log_int(rng, 512, 8192)])
            prefix = int(min(prefix, 6.0e7 / (batch * q_heads)))
            case = _decode("", dtype, q_heads, kv_heads, head_dim, batch, prefix, capacity, len_lo, len_hi,
                           rng.random() < 0.5)
        else:
            budget = _log_int(rng, 1, capacity)
            recent = rng.choice([0, min(budget, 32), rng.randint(0, budget), budget])
            case = _evict("", dtype, kv_heads, head_dim, batch, capacity, len_lo, len_hi, budget, recent)
    case.pop("name")
    return case


def _prompt_lens(case):
    return [int(n) for n in case["lens"].split(",")]


def _cache_lens(case):
    rng = random.Random(case["batch"] * 1000003 + case["len_lo"] * 1009 + case["len_hi"])
    return [rng.randint(case["len_lo"], case["len_hi"]) for _ in range(case["batch"])]


def work(case):
    hd, hkv = case["head_dim"], case["kv_heads"]
    if case["op"] == "prompt_attn":
        lens = _prompt_lens(case)
        t, hq = sum(lens), case["q_heads"]
        pairs = sum(n * (n + 1) // 2 for n in lens)
        moved = 2 * t * hd * (2 * hq + 2 * hkv) + (4 * t * hq if case["lse"] else 0)
        return {"bytes": moved, "flops": 4 * hq * hd * pairs}
    b, cap, lens = case["batch"], case["capacity"], _cache_lens(case)
    if case["op"] == "shared_prefix_attn":
        hq, p = case["q_heads"], case["prefix"]
        moved = 2 * (2 * b * hq * hd) + 2 * 2 * hkv * hd * (p + sum(lens)) + 4 * b
        moved += 8 * b * hkv * cap if case["weights"] else 0
        return {"bytes": moved, "flops": 4 * hq * hd * (b * p + sum(lens))}
    budget, recent = case["budget"], case["recent"]
    kept = [min(n, budget) for n in lens]
    scanned = sum(n - recent for n in lens if n > budget)  # the recent tokens' weights are only copied
    moved = 4 * hkv * scanned                              # weights read to choose
    moved += 2 * 2 * hkv * hd * (sum(kept) + b * budget)   # kept rows read, every output row written
    moved += hkv * (4 * sum(kept) + 8 * b * budget) + 8 * b
    return {"bytes": moved, "flops": hkv * scanned}


# ------------------------------------------------------------------ the inputs

def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, hd, hkv = _DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)

    if case["op"] == "prompt_attn":
        # q, k and v are slices of one packed projection, as the framework's QKV product writes it
        hq, t = case["q_heads"], sum(_prompt_lens(case))
        packed = normal(t, (hq + 2 * hkv) * hd).view(t, hq + 2 * hkv, hd)
        return {"q": packed[:, :hq], "k": packed[:, hq:hq + hkv], "v": packed[:, hq + hkv:]}
    b, cap = case["batch"], case["capacity"]
    lens = torch.tensor(_cache_lens(case), dtype=torch.int32, device=dev)
    x = {"k_cache": torch.empty(b, cap, hkv, hd, dtype=dtype, device=dev),
         "v_cache": torch.empty(b, cap, hkv, hd, dtype=dtype, device=dev), "lengths": lens}
    for i in range(b):
        x["k_cache"][i] = normal(cap, hkv, hd)
        x["v_cache"][i] = normal(cap, hkv, hd)
    if case["op"] == "shared_prefix_attn":
        x["q"] = normal(b, case["q_heads"], hd)
        x["prefix_k"], x["prefix_v"] = normal(case["prefix"], hkv, hd), normal(case["prefix"], hkv, hd)
        if not case["weights"]:
            return x
    # accumulated attention weights: heavy-tailed, an eighth of them exact zeros (keys whose
    # probabilities underflowed, or that no query has seen yet)
    w = torch.exp(2.0 * torch.randn((b, hkv, cap), generator=gen, device=dev) - 4.0)
    x["key_weights"] = w * (torch.rand((b, hkv, cap), generator=gen, device=dev) >= 0.125)
    return x


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own and case["op"] == "prompt_attn":
        from tiktok_techjam_2026_track3_b200 import ops
        # the batch's work plan: built once per batch, used by every layer
        state["plan"] = ops.PromptPlan(_prompt_lens(case), case["q_heads"], case["kv_heads"],
                                       case["head_dim"], state["q"].device)
    return state


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------------ the framework's calls

def _own_prompt(s):
    from tiktok_techjam_2026_track3_b200 import ops
    return ops.prompt_attn(s["q"], s["k"], s["v"], s["plan"], return_lse=s["case"]["lse"])


def _own_decode(s):
    from tiktok_techjam_2026_track3_b200 import ops
    return ops.shared_prefix_attn(s["q"], s["prefix_k"], s["prefix_v"], s["k_cache"], s["v_cache"],
                                  s["lengths"], key_weights=s.get("key_weights"))


def _own_evict(s):
    from tiktok_techjam_2026_track3_b200 import ops
    return tuple(ops.cache_evict(s["k_cache"], s["v_cache"], s["key_weights"], s["lengths"],
                                 s["case"]["budget"], s["case"]["recent"]))


# ------------------------------------------------------------------ the plain forms

def _plain_prompt(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    hq, hkv, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    g, scale = hq // hkv, hd ** -0.5
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    start = 0
    for n in _prompt_lens(case):
        kf = k[start:start + n].float().permute(1, 2, 0)          # [Hkv, hd, n]
        vf = v[start:start + n].float().permute(1, 0, 2)          # [Hkv, n, hd]
        for lo in range(0, n, 1024):
            hi = min(n, lo + 1024)
            m = hi - lo
            qf = q[start + lo:start + hi].float().view(m, hkv, g, hd).permute(1, 2, 0, 3).reshape(hkv, g * m, hd)
            sc = (torch.matmul(qf, kf[:, :, :hi]) * scale).view(hkv, g, m, hi)
            later = torch.arange(hi, device=q.device) > torch.arange(lo, hi, device=q.device)[:, None]
            sc.masked_fill_(later, float("-inf"))
            top = sc.amax(-1, keepdim=True)
            p = torch.exp(sc.sub_(top))
            total = p.sum(-1, keepdim=True)
            o = torch.matmul(p.view(hkv, g * m, hi), vf[:, :hi]).view(hkv, g, m, hd) / total
            out[start + lo:start + hi] = o.permute(2, 0, 1, 3).reshape(m, hq, hd).to(q.dtype)
            lse[start + lo:start + hi] = (top + torch.log(total))[..., 0].permute(2, 0, 1).reshape(m, hq)
        start += n
    return (out, lse) if case["lse"] else out


def _plain_decode(s):
    case, q = s["case"], s["q"]
    b, hq, hkv, hd, p = case["batch"], case["q_heads"], case["kv_heads"], case["head_dim"], case["prefix"]
    g, cap = hq // hkv, case["capacity"]
    qf = q.float().view(b, hkv, g, hd) * hd ** -0.5
    # prefix: one product per head group for the whole batch
    rows = qf.permute(1, 0, 2, 3).reshape(hkv, b * g, hd)
    sp = torch.matmul(rows, s["prefix_k"].float().permute(1, 2, 0)).view(hkv, b, g, p).permute(1, 0, 2, 3)
    sc = torch.matmul(qf, s["k_cache"].float().permute(0, 2, 3, 1))
    unused = torch.arange(cap, device=q.device) >= s["lengths"][:, None]
    sc = sc.masked_fill(unused[:, None, None, :], float("-inf"))
    both = torch.cat([sp, sc], -1)
    top = both.amax(-1, keepdim=True)
    e = torch.exp(both - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    prob = e / torch.where(total == 0, torch.ones_like(total), total)
    pp, pc = prob[..., :p], prob[..., p:]
    o = torch.matmul(pp.permute(1, 0, 2, 3).reshape(hkv, b * g, p), s["prefix_v"].float().permute(1, 0, 2))
    o = o.view(hkv, b, g, hd).permute(1, 0, 2, 3) + torch.matmul(pc, s["v_cache"].float().permute(0, 2, 1, 3))
    out = o.reshape(b, hq, hd).to(q.dtype)
    return (out, s["key_weights"] + pc.sum(2)) if case["weights"] else out


def _plain_evict(s):
    case, w, lens = s["case"], s["key_weights"], s["lengths"].long()
    hkv, cap, budget, recent = case["kv_heads"], case["capacity"], case["budget"], case["recent"]
    dev = w.device
    pos = torch.arange(cap, device=dev)
    # rank: the recent tokens first, then by weight, the lowest index first among equals, unused rows last
    rank = torch.where(torch.isnan(w), torch.full_like(w, float("-inf")), w)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    kind = torch.where(pos >= lens[:, None], 2, torch.where(pos >= (lens - recent)[:, None], 0, 1))
    kind = kind[:, None, :].expand(-1, hkv, -1).gather(2, order)
    order = order.gather(2, torch.sort(kind, dim=-1, stable=True).indices)
    new_lens = torch.minimum(lens, torch.full_like(lens, budget))
    slot = torch.arange(budget, device=dev)
    kept = slot < new_lens[:, None, None]                                         # [B, 1, N]
    idx = torch.sort(torch.where(kept, order[..., :budget], cap), dim=-1).values  # ascending, unused last
    safe = idx.clamp(max=cap - 1)
    rows = safe.permute(0, 2, 1)[..., None].expand(-1, -1, -1, case["head_dim"])
    live = kept.expand(-1, hkv, -1)
    zero = ~live.permute(0, 2, 1)[..., None]
    k = s["k_cache"].gather(1, rows).masked_fill(zero, 0)
    v = s["v_cache"].gather(1, rows).masked_fill(zero, 0)
    weights = w.gather(2, safe).masked_fill(~live, 0)
    positions = idx.masked_fill(~live, -1).to(torch.int32)
    return k, v, weights, new_lens.to(torch.int32), positions


_OWN = {"prompt_attn": _own_prompt, "shared_prefix_attn": _own_decode, "cache_evict": _own_evict}
_PLAIN = {"prompt_attn": _plain_prompt, "shared_prefix_attn": _plain_decode, "cache_evict": _plain_evict}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_rows(q, keys, values):
    """softmax(q . keys / sqrt(hd)) values for q [R, hd], keys and values [n, hd], all in 64 bits."""
    logits = (q @ keys.T) / math.sqrt(q.shape[1])
    log_total = torch.logsumexp(logits, 1, keepdim=True)
    prob = torch.exp(logits - log_total)
    return prob @ values, log_total[:, 0], prob


def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "prompt_attn":
        lens, hq = _prompt_lens(case), case["q_heads"]
        group = hq // case["kv_heads"]
        out = torch.zeros(x["q"].shape, dtype=torch.float64, device=x["q"].device)
        lse = torch.zeros(x["q"].shape[:2], dtype=torch.float64, device=x["q"].device)
        first = 0
        for n in lens:
            for h in range(hq):
                key = x["k"][first:first + n, h // group].double()
                val = x["v"][first:first + n, h // group].double()
                for a in range(0, n, 2048):
                    z = min(n, a + 2048)
                    logits = (x["q"][first + a:first + z, h].double() @ key[:z].T) / math.sqrt(case["head_dim"])
                    logits[:, a:] += torch.full((z - a, z - a), float("-inf"), dtype=torch.float64,
                                                device=logits.device).triu(1)
                    total = torch.logsumexp(logits, 1, keepdim=True)
                    lse[first + a:first + z, h] = total[:, 0]
                    out[first + a:first + z, h] = torch.exp(logits - total) @ val[:z]
            first += n
        return (out, lse) if case["lse"] else out
    lens = [int(n) for n in x["lengths"].tolist()]
    if case["op"] == "shared_prefix_attn":
        group = case["q_heads"] // case["kv_heads"]
        out = torch.zeros(x["q"].shape, dtype=torch.float64, device=x["q"].device)
        weights = x["key_weights"].double() if case["weights"] else None
        for h in range(case["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            shared_k, shared_v = x["prefix_k"][:, h].double(), x["prefix_v"][:, h].double()
            for i, n in enumerate(lens):
                if n + case["prefix"] == 0:
                    continue
                key = torch.cat([shared_k, x["k_cache"][i, :n, h].double()])
                val = torch.cat([shared_v, x["v_cache"][i, :n, h].double()])
                out[i, heads], _, prob = _exact_rows(x["q"][i, heads].double(), key, val)
                if weights is not None:
                    weights[i, h, :n] += prob[:, case["prefix"]:].sum(0)
        return (out, weights) if case["weights"] else out
    budget, recent, hkv = case["budget"], case["recent"], case["kv_heads"]
    w = x["key_weights"].double().cpu().numpy()
    positions = np.full((case["batch"], hkv, budget), -1, dtype=np.int64)
    for i, n in enumerate(lens):
        for h in range(hkv):
            if n <= budget:
                positions[i, h, :n] = np.arange(n)
            else:
                old = w[i, h, :n - recent]
                best = np.argsort(-old, kind="stable")[:budget - recent]
                positions[i, h] = np.concatenate([np.sort(best), np.arange(n - recent, n)])
    pos = torch.from_numpy(positions).to(x["k_cache"].device)
    k = torch.zeros(case["batch"], budget, hkv, case["head_dim"], dtype=torch.float64, device=pos.device)
    v = torch.zeros_like(k)
    weights = torch.zeros(pos.shape, dtype=torch.float64, device=pos.device)
    for i, n in enumerate(lens):
        m = min(n, budget)
        for h in range(hkv):
            at = pos[i, h, :m]
            k[i, :m, h], v[i, :m, h] = x["k_cache"][i, at, h].double(), x["v_cache"][i, at, h].double()
            weights[i, h, :m] = x["key_weights"][i, h, at].double()
    return k, v, weights, torch.tensor([min(n, budget) for n in lens], dtype=torch.int32, device=pos.device), \
        pos.to(torch.int32)
