"""Serving operators on the GPU at the edges of what they accept: workspaces at any
allowed address, scores of minus infinity, infinities and NaN in long prompts, the decode
step's kernels right behind the ones that wrote its inputs."""

import math

import pytest
import torch

from serving_ref import DT, attend, decode_ref, out_bound
from tiktok_techjam_2026_track3_b200 import _lib, ops

pytestmark = pytest.mark.gpu

# (B, P, C, Hq, Hkv, hd): the prefix on the tensor-core tiles at every padded head_dim, and in the caches' line
STEPS = [(130, 513, 3, 32, 8, 128), (300, 1025, 0, 16, 16, 64), (140, 900, 5, 8, 2, 256), (40, 4099, 33, 24, 3, 80),
         (3, 300, 200, 8, 2, 128)]


def randn(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def decode_case(B, P, C, Hq, Hkv, hd, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return (randn(gen, dtype, B, Hq, hd), randn(gen, dtype, P, Hkv, hd), randn(gen, dtype, P, Hkv, hd),
            randn(gen, dtype, B, C, Hkv, hd), randn(gen, dtype, B, C, Hkv, hd))


def check(got, ref, bound, what=""):
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)          # NaN counts as bad
    assert not bool(bad.any()), (what, int(bad.sum()), float(err[bad].max()), float((err / bound.clamp_min(1e-30)).max()))


# ------------------------------------------------------------------ workspaces

@pytest.mark.parametrize("offset", [0, 16, 32, 48, 240])
@pytest.mark.parametrize("B,P,C,Hq,Hkv,hd", STEPS)
def test_decode_workspace_at_any_16_byte_boundary(B, P, C, Hq, Hkv, hd, offset):
    """A workspace of exactly the size asked for gives the same bits wherever it starts, is
    not left, and may be used again."""
    args = decode_case(B, P, C, Hq, Hkv, hd, torch.bfloat16, 1)
    lens = torch.tensor([i % (C + 1) for i in range(B)], dtype=torch.int32).cuda()
    w = torch.rand(B, Hkv, C, generator=torch.Generator().manual_seed(2)).cuda()
    want = ops.shared_prefix_attn(*args, lens, key_weights=w, return_lse=True)
    need = _lib.load().ttj_shared_prefix_attn_workspace_size(B, P, C, Hq, Hkv, hd, 1)
    arena = torch.full((need + 1024,), 0x5A, dtype=torch.uint8, device="cuda")
    base = 256 + offset - arena.data_ptr() % 256
    base += 256 if base < 256 else 0
    own = arena[base:base + need]
    assert own.data_ptr() % 256 == offset
    for _ in range(2):
        got = ops.shared_prefix_attn(*args, lens, key_weights=w, return_lse=True, workspace=own)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert bool((arena[:base] == 0x5A).all()) and bool((arena[base + need:] == 0x5A).all())
    ops.check_device_status(own.device)


def test_workspaces_the_kernels_could_not_use_are_refused():
    """Host memory and strided views: an error before any launch, from every call that takes one."""
    args = decode_case(3, 300, 200, 8, 2, 128, torch.bfloat16, 1)
    lens = torch.tensor([200, 0, 7], dtype=torch.int32).cuda()
    x = torch.randn(2, 64, 256, device="cuda").half()
    w = {n: torch.randn(s, device="cuda").half() * 0.05 for n, s in
         (("w_qkv", (768, 256)), ("b_qkv", (768,)), ("w_o", (256, 256)), ("b_o", (256,)))}
    block = dict(w, ln1_w=torch.ones_like(w["b_o"]), ln1_b=w["b_o"], ln2_w=torch.ones_like(w["b_o"]), ln2_b=w["b_o"],
                 w_in=w["w_qkv"][:512].contiguous(), b_in=w["b_qkv"][:512].contiguous(),
                 w_out=torch.randn(256, 512, device="cuda").half() * 0.05, b_out=w["b_o"])
    q8, s8 = ops.quantize_weight(w["w_qkv"])
    o8, so = ops.quantize_weight(w["w_o"])
    bf = (w["b_qkv"].float(), w["b_o"].float())
    calls = [lambda ws: ops.shared_prefix_attn(*args, lens, workspace=ws),
             lambda ws: ops.attn_layer(x, w["w_qkv"], w["b_qkv"], w["w_o"], w["b_o"], 4, True, workspace=ws),
             lambda ws: ops.transformer_block(x, block, 4, True, 1e-5, 1e-5, workspace=ws),
             lambda ws: ops.int8_attn_layer(x, q8, s8, bf[0], o8, so, bf[1], 4, True, workspace=ws)]
    n = 1 << 24
    for call in calls:
        want = call(None)
        assert torch.equal(call(torch.empty(n, dtype=torch.uint8, device="cuda")), want)
        assert torch.equal(call(torch.empty(n // 4, dtype=torch.float32, device="cuda")), want)
        for bad in (torch.empty(n, dtype=torch.uint8), torch.empty(n, 2, dtype=torch.uint8, device="cuda")[:, 0],
                    torch.empty(1, dtype=torch.uint8, device="cuda").expand(n)):
            with pytest.raises(RuntimeError, match="workspace must be a contiguous tensor on cuda"):
                call(bad)


# ------------------------------------------------------------------ scores of minus infinity

# (B, P, C, Hq, Hkv, hd, lengths): the caches' line alone, with the prefix in it, and behind the prefix's tiles at
# every padded head_dim and both row tiles (a group above 8 takes 16 rows)
FAINT = [(2, 0, 64, 4, 2, 64, [17, 64]), (2, 40, 33, 2, 2, 128, [1, 33]), (3, 33, 20, 24, 2, 64, [1, 17, 20]),
         (2, 130, 50, 4, 2, 256, [1, 49]), (300, 1025, 17, 16, 16, 64, [1, 17, 16] * 100),
         (130, 513, 33, 32, 8, 128, [1, 17] * 65), (140, 900, 17, 8, 2, 256, [1, 17] * 70)]


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("where", ["last cached key", "every cached key", "every prefix key", "last prefix range",
                                   "every key"])
@pytest.mark.parametrize("B,P,C,Hq,Hkv,hd,lengths", FAINT)
def test_keys_that_score_minus_infinity_weigh_nothing(dt, where, B, P, C, Hq, Hkv, hd, lengths):
    """Such a key is as good as absent beside others, also where a partial result (a cache's or a
    prefix range's) holds no other key; a row of such keys alone gets zeros, as one without keys."""
    q, pk, pv, kc, vc = decode_case(B, P, C, Hq, Hkv, hd, DT[dt], P + C)
    q[..., 5] = q[..., 5].abs() + 0.5            # times -inf: a score of -inf in every head
    if where == "last cached key":
        for b, n in enumerate(lengths):
            kc[b, n - 1, :, 5] = -math.inf
    if where in ("every cached key", "every key"):
        kc[..., 5] = -math.inf
    if where in ("every prefix key", "every key"):
        pk[..., 5] = -math.inf
    if where == "last prefix range":
        pk[P // 2:, :, 5] = -math.inf
    w = torch.rand(B, Hkv, C, generator=torch.Generator().manual_seed(3)).cuda()
    lens = torch.tensor(lengths, dtype=torch.int32).cuda()
    out, new_w, lse = ops.shared_prefix_attn(q, pk, pv, kc, vc, lens, key_weights=w, return_lse=True)
    ref, bound, prob = decode_ref(q, pk, pv, kc, vc, lengths, hd ** -0.5)
    assert bool(torch.isfinite(ref).all()) and bool(torch.isfinite(bound).all())
    check(out, ref, bound)
    want = w.double() + prob                     # fp32 scores and sums, then one fp32 addition
    assert bool(((new_w.double() - want).abs() <= 4e-5 * prob + 2.0 ** -23 * want.abs()).all())
    alone = where == "every key" or (where == "every cached key" and P == 0)
    assert bool((lse == -math.inf).all()) == alone and not bool(torch.isnan(lse).any())
    if alone:
        assert not bool(out.any()) and torch.equal(new_w, w)
    ops.check_device_status(q.device)


def test_the_types_lowest_value_as_a_mask():
    """Keys filled with the lowest bfloat16 value: their scores overflow to minus infinity."""
    B, P, C, Hq, Hkv, hd = 130, 513, 40, 32, 8, 128
    q, pk, pv, kc, vc = decode_case(B, P, C, Hq, Hkv, hd, torch.bfloat16, 9)
    q = q.abs() + 1
    lengths = [(5 * b) % (C + 1) for b in range(B)]
    kc[:, ::2] = torch.finfo(torch.bfloat16).min
    pk[400:] = torch.finfo(torch.bfloat16).min
    out = ops.shared_prefix_attn(q, pk, pv, kc, vc, torch.tensor(lengths, dtype=torch.int32).cuda())
    # the overflow is the inputs' own: in 64 bits these scores are finite and far below the others
    ref, bound, _ = decode_ref(q, pk, pv, kc, vc, lengths, hd ** -0.5)
    check(out, ref, bound)


def test_an_infinite_value_of_a_key_without_weight_still_gives_nan():
    """0 times infinity, as in the definition: the value of a key that a row attends is not masked."""
    q, pk, pv, kc, vc = decode_case(2, 40, 33, 4, 2, 64, torch.float16, 4)
    q[..., 5] = q[..., 5].abs() + 0.5
    kc[0, 0, :, 5], vc[0, 0, :, 7] = -math.inf, math.inf
    out = ops.shared_prefix_attn(q, pk, pv, kc, vc, torch.tensor([1, 33], dtype=torch.int32).cuda())
    assert bool(torch.isnan(out[0, :, 7]).all()) and bool(torch.isfinite(out[0, :, :7]).all())
    assert bool(torch.isfinite(out[0, :, 8:]).all()) and bool(torch.isfinite(out[1]).all())


# ------------------------------------------------------------------ later tokens' infinities and NaN

def prompt_case(lens, Hq, Hkv, hd, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    packed = randn(gen, dtype, sum(lens), Hq + 2 * Hkv, hd)
    return packed[:, :Hq], packed[:, Hq:Hq + Hkv].clone(), packed[:, Hq + Hkv:].clone()


def check_rows(out, q, k, v, first, rows):
    """Rows `rows` of the prompt that starts at row `first` against their own keys alone in 64 bits;
    where the definition gives an infinity or NaN, the same one."""
    Hq, Hkv, hd = q.shape[1], k.shape[1], q.shape[2]
    for i in rows:
        n = slice(first, first + i + 1)
        for h in range(Hq):
            vh = v[n, h * Hkv // Hq]
            ref, _, prob, spread = attend(q[first + i:first + i + 1, h], k[n, h * Hkv // Hq], vh, hd ** -0.5)
            vmax = float(vh[torch.isfinite(vh)].abs().max())
            got, ref = out[first + i, h].double(), ref[0]
            ok = torch.isfinite(ref)
            assert torch.equal(torch.isnan(got), torch.isnan(ref)), (i, h)
            assert torch.equal(got[torch.isinf(ref)], ref[torch.isinf(ref)]), (i, h)
            bound = out_bound(q.dtype, ref, spread[0], i + 1, vmax)
            assert bool(((got - ref).abs() <= bound)[ok].all()), (i, h, float(((got - ref).abs() / bound)[ok].max()))


HEADS = [(2, 2, 64), (8, 2, 64), (7, 1, 40), (4, 2, 128), (6, 2, 96), (2, 1, 256), (3, 1, 200)]


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,hd", HEADS)
def test_later_infinities_leave_long_prompts_as_they_are(dt, Hq, Hkv, hd):
    """Single values late in a long prompt (and in a short one beside it): every row before each
    of them keeps its result, the columns without one bit for bit."""
    lens = [130, 9000, 60]
    q, k, v = prompt_case(lens, Hq, Hkv, hd, DT[dt], hd)
    plan = ops.PromptPlan(lens, Hq, Hkv, hd, q.device)
    clean = ops.prompt_attn(q, k, v, plan)
    bad = [(8957, 3, math.nan), (8960, 4, math.inf), (8999, 5, -math.inf), (4477, 6, math.nan)]
    for at, col, x in bad:
        v[130 + at, :, col] = x
    v[100, :, 1] = math.inf
    out = ops.prompt_attn(q, k, v, plan)
    check_rows(out, q, k, v, 130, [4400, 4476, 4477, 4478, 8895, 8900, 8956, 8957, 8959, 8960, 8998, 8999])
    check_rows(out, q, k, v, 0, [90, 99, 100, 129])
    for col in range(hd):
        hit = [at for at, c, _ in bad if c == col]
        end = 130 + hit[0] if hit else len(out)
        if col != 1:
            near = slice(130 + hit[0] - 160, end) if hit else slice(0, 0)   # rows that may have been formed again
            rest = torch.ones(len(out), dtype=torch.bool, device=out.device)
            rest[near], rest[end:] = False, False
            assert torch.equal(out[rest][..., col], clean[rest][..., col]), col
            assert bool(torch.isfinite(out[:end, :, col].float()).all())
    ops.check_device_status(q.device)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,hd", HEADS)
def test_infinities_that_a_row_sees_meet_later_ones(dt, Hq, Hkv, hd):
    """Columns that a row's own keys make infinite or NaN, others that only later keys do, rows
    whose scores are NaN, and prompts without one finite column."""
    lens = [400, 257, 300]
    q, k, v = prompt_case(lens, Hq, Hkv, hd, DT[dt], hd + 1)
    inf, nan = math.inf, math.nan
    for at, col, x in [(5, 0, inf), (300, 0, nan), (7, 1, inf), (290, 1, -inf), (9, 2, -inf), (310, 2, -inf), (20, 3, nan),
                       (305, 3, inf), (30, 4, inf), (200, 4, -inf), (320, 4, inf), (333, 5, nan), (390, 6, inf)]:
        v[at, :, col] = x
    k[280, :, 0] = nan                            # scores of the rows from there on
    v[400 + 100] = inf                            # every column, more than once
    v[400 + 250] = inf
    v[400 + 255] = -inf
    v[657 + 50:657 + 300:50, :, 7] = inf          # a column infinite again and again
    k[657 + 10, :, 1] = inf                       # scores of both infinities
    out = ops.prompt_attn(q, k, v, ops.PromptPlan(lens, Hq, Hkv, hd, q.device))
    check_rows(out, q, k, v, 0, [0, 4, 5, 6, 8, 19, 20, 25, 199, 200, 255, 256, 270, 279])
    assert bool(torch.isnan(out[280:400].float()).all())
    check_rows(out, q, k, v, 400, [0, 99, 100, 200, 249, 250, 254, 255, 256])
    check_rows(out, q, k, v, 657, [0, 9])
    k[657 + 10, :, 1] = 0
    out = ops.prompt_attn(q, k, v, ops.PromptPlan(lens, Hq, Hkv, hd, q.device))
    check_rows(out, q, k, v, 657, [0, 9, 49, 50, 51, 99, 100, 128, 255, 256, 299])
    ops.check_device_status(q.device)


@pytest.mark.parametrize("Hq,Hkv,hd", [(4, 1, 64), (4, 1, 128), (2, 1, 256)])
def test_repair_of_a_very_long_prompt_ends_no_wait(Hq, Hkv, hd):
    """One value near the end of 200000 tokens: forming its tile's rows again takes longer than a
    key tile's step, with other prompts' work behind it in the same blocks."""
    n, lens = 200000, [200000] + [90] * 300
    q, k, v = prompt_case(lens, Hq, Hkv, hd, torch.float16, 5)
    plan = ops.PromptPlan(lens, Hq, Hkv, hd, q.device)
    clean = ops.prompt_attn(q, k, v, plan)
    v[n - 70, :, 2] = math.nan
    out = ops.prompt_attn(q, k, v, plan)
    ops.check_device_status(q.device)
    assert torch.equal(out[n:], clean[n:]) and torch.equal(out[:n - 300], clean[:n - 300])
    check_rows(out, q, k, v, 0, [n - 200, n - 128, n - 71, n - 70, n - 1])


# ------------------------------------------------------------------ right behind the kernels that write the inputs

def step_chain(q, pk, pv, kc, vc, lens, w, budget):
    """Eviction, then a decode step on what it wrote (lengths, rows and weights), then another."""
    kept = ops.cache_evict(kc, vc, w, lens, budget, 3)
    out, w1 = ops.shared_prefix_attn(q, pk, pv, kept.k, kept.v, kept.lengths, key_weights=kept.key_weights)
    out2, w2 = ops.shared_prefix_attn(out, pk, pv, kept.k, kept.v, kept.lengths, key_weights=w1)
    return kept.lengths, kept.positions, out, w1, out2, w2


@pytest.mark.parametrize("B,P,C,Hq,Hkv,hd,budget", [(130, 513, 40, 32, 8, 128, 17), (33, 26001, 40, 32, 8, 128, 20),
                                                    (300, 1025, 24, 16, 16, 64, 10), (140, 900, 25, 8, 2, 256, 11)])
def test_decode_behind_the_kernels_that_write_its_inputs(B, P, C, Hq, Hkv, hd, budget):
    """With the prefix on the tiles the caches' kernel starts without a wait of its own: chains of
    calls on a side stream and in a graph, inputs changed in between, give what each step gives alone."""
    sets = []
    for seed in (1, 2):
        q, pk, pv, kc, vc = decode_case(B, P, C, Hq, Hkv, hd, torch.bfloat16, seed)
        lens = torch.tensor([(i * (3 + seed)) % (C + 1) for i in range(B)], dtype=torch.int32).cuda()
        sets.append((q, pk, pv, kc, vc, lens, torch.rand(B, Hkv, C, generator=torch.Generator().manual_seed(seed)).cuda()))
    want = []
    for x in sets:
        kept = ops.cache_evict(*x[3:5], x[6], x[5], budget, 3)
        torch.cuda.synchronize()
        out, w1 = ops.shared_prefix_attn(*x[:3], kept.k, kept.v, kept.lengths, key_weights=kept.key_weights)
        torch.cuda.synchronize()
        out2, w2 = ops.shared_prefix_attn(out, *x[1:3], kept.k, kept.v, kept.lengths, key_weights=w1)
        torch.cuda.synchronize()
        want.append((kept.lengths, kept.positions, out, w1, out2, w2))
    held = tuple(t.clone() for t in sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    with torch.cuda.stream(side):
        for i in range(20):
            for h, t in zip(held, sets[i % 2]):
                h.copy_(t)
            got.append(step_chain(*held, budget))
    side.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2])), i
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step_chain(*held, budget)
    for i in range(10):
        for h, t in zip(held, sets[i % 2]):
            h.copy_(t)
        graph.replay()
        snap = [t.clone() for t in res]
        assert all(torch.equal(a, b) for a, b in zip(snap, want[i % 2])), i
    ops.check_device_status(side.device)


# ------------------------------------------------------------------ wide groups over caches larger than L2

@pytest.mark.parametrize("Hq,Hkv,hd", [(32, 1, 128), (40, 2, 64)])
def test_wide_groups_over_caches_larger_than_l2(Hq, Hkv, hd):
    """A group of several row tiles reads its cache once per tile."""
    B, C = 70, 8192 * 128 // (Hkv * hd)
    gen = torch.Generator(device="cuda").manual_seed(8)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda").bfloat16()
    q, kc, vc = normal(B, Hq, hd), normal(B, C, Hkv, hd), normal(B, C, Hkv, hd)
    none = kc.new_empty(0, Hkv, hd)
    assert kc.numel() * 4 > 126 << 20
    lengths = [C - 37 * b for b in range(B)]
    w = torch.rand(B, Hkv, C, generator=gen, device="cuda")
    out, new_w = ops.shared_prefix_attn(q, none, none, kc, vc, torch.tensor(lengths, dtype=torch.int32).cuda(), key_weights=w)
    ref, bound, prob = decode_ref(q, none, none, kc, vc, lengths, hd ** -0.5)
    check(out, ref, bound)
    want = w.double() + prob
    assert bool(((new_w.double() - want).abs() <= 4e-5 * prob + 2.0 ** -23 * want.abs()).all())
    ops.check_device_status(q.device)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,hd", HEADS)
def test_an_infinite_value_without_weight_meets_later_ones(dt, Hq, Hkv, hd):
    """A key that scores minus infinity and whose value is infinite: 0 times infinity is NaN, also
    where a later token's infinity falls into the same column and tile."""
    lens = [300, 130]
    q, k, v = prompt_case(lens, Hq, Hkv, hd, DT[dt], hd + 2)
    q = q.clone()
    q[:300, :, 2] = q[:300, :, 2].abs() + 0.5
    k[60, :, 2] = -math.inf
    for at, col in ((60, 3), (100, 3), (61, 4), (100, 4), (270, 4), (290, 3)):
        v[at, :, col] = math.inf
    v[300 + 20, :, 4] = math.inf
    v[300 + 90, :, 4] = math.inf
    out = ops.prompt_attn(q, k, v, ops.PromptPlan(lens, Hq, Hkv, hd, q.device))
    check_rows(out, q, k, v, 0, [0, 59, 60, 61, 62, 99, 100, 127, 128, 255, 256, 269, 270, 289, 290, 299])
    check_rows(out, q, k, v, 300, [0, 19, 20, 89, 90, 129])
    ops.check_device_status(q.device)
