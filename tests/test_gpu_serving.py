"""Serving operators on the GPU against their definitions in 64 bits: causal
attention over packed prompts, decode attention over a shared prefix and
per-sequence caches, eviction by accumulated attention weight."""

import math

import pytest
import torch

from serving_ref import DT, decode_ref, evict_ref, prompt_ref
from tiktok_techjam_2026_track3_b200 import ops

pytestmark = pytest.mark.gpu


def randn(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def check(got, ref, bound, what=""):
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)          # NaN counts as bad
    assert not bool(bad.any()), (what, int(bad.sum()), float(err[bad].max()), float((err / bound.clamp_min(1e-30)).max()))


# ------------------------------------------------------------------ prompts

def prompt_case(lens, Hq, Hkv, hd, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    packed = randn(gen, dtype, sum(lens), Hq + 2 * Hkv, hd)   # q | k | v as the projection writes them
    return packed[:, :Hq], packed[:, Hq:Hq + Hkv], packed[:, Hq + Hkv:]


PROMPTS = [  # (lens, Hq, Hkv, hd)
    ([1], 1, 1, 64), ([2, 1, 1], 4, 2, 64), ([61], 8, 2, 64), ([0, 5, 0, 0, 130, 0], 4, 4, 64),
    ([127, 128, 129], 4, 4, 64), ([255, 256, 257], 2, 1, 128), ([300, 1, 77], 8, 1, 128),
    ([33, 200], 7, 1, 64), ([17, 100, 40], 6, 2, 128), ([400], 5, 5, 40), ([129, 31], 12, 4, 96),
    ([256, 3], 16, 1, 8), ([500, 12], 4, 2, 256), ([130, 1], 3, 1, 200), ([64] * 9, 32, 2, 64),
    ([20, 30], 128, 1, 64), ([20, 30], 65, 1, 128), ([5, 9, 100], 24, 8, 80), ([1000, 700, 3], 4, 1, 64),
    ([1025], 2, 2, 128), ([600, 300], 8, 4, 192), (list(range(40)), 8, 2, 128),
]


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,Hq,Hkv,hd", PROMPTS)
def test_prompt_attn_matches_definition(dt, lens, Hq, Hkv, hd):
    q, k, v = prompt_case(lens, Hq, Hkv, hd, DT[dt], sum(lens) + Hq * hd)
    plan = ops.PromptPlan(lens, Hq, Hkv, hd, q.device)
    out, lse = ops.prompt_attn(q, k, v, plan, return_lse=True)
    ref, ref_lse, bound = prompt_ref(q, k, v, lens, hd ** -0.5)
    check(out, ref, bound)
    assert float((lse.double() - ref_lse).abs().max()) <= 2e-5 * (1 + float(ref_lse.abs().max()))
    assert torch.equal(ops.prompt_attn(q, k, v, plan), out)   # and without the sums, bit for bit
    ops.check_device_status(q.device)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,Hq,Hkv,hd", [([300, 2, 129], 4, 2, 64), ([300, 2, 129], 4, 1, 128),
                                            ([300, 140], 2, 1, 256)])
def test_other_prompts_contents_never_matter(dt, lens, Hq, Hkv, hd):
    """Infinities and NaN in one prompt leave the others' results as they are."""
    q, k, v = (t.clone() for t in prompt_case(lens, Hq, Hkv, hd, DT[dt], 3))
    plan = ops.PromptPlan(lens, Hq, Hkv, hd, q.device)
    clean = ops.prompt_attn(q, k, v, plan)
    first = lens[0]
    for t, bad in ((q, math.nan), (k, math.inf), (v, math.nan)):
        t[first:first + lens[1]] = bad
    dirty = ops.prompt_attn(q, k, v, plan)
    assert torch.equal(dirty[:first], clean[:first])
    assert torch.equal(dirty[first + lens[1]:], clean[first + lens[1]:])


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,hd", [(2, 2, 64), (4, 1, 64), (7, 1, 40), (4, 2, 128), (6, 2, 96), (2, 1, 256)])
@pytest.mark.parametrize("what,bad", [("v", math.nan), ("v", -math.inf), ("k", math.nan), ("kv", math.nan)])
def test_later_tokens_of_the_prompt_never_matter(dt, Hq, Hkv, hd, what, bad):
    """An infinity or NaN in a token's key or value reaches the rows from that token on
    and no earlier one (which meet it only behind the causal mask)."""
    lens, tokens = [300, 70, 129], (17, 130, 255, 298)
    q, k, v = (t.clone() for t in prompt_case(lens, Hq, Hkv, hd, DT[dt], 17))
    plan = ops.PromptPlan(lens, Hq, Hkv, hd, q.device)
    for t in tokens:
        dirty_k, dirty_v = k.clone(), v.clone()
        if "k" in what:
            dirty_k[t] = bad
        if "v" in what:
            dirty_v[t, :, 3] = bad
        out = ops.prompt_attn(q, dirty_k, dirty_v, plan)
        ref, _, bound = prompt_ref(q[:t], k[:t], v[:t], [t], hd ** -0.5)
        check(out[:t], ref, bound, t)
        hit = out[t:300].float()
        if what == "v":
            assert not bool(torch.isfinite(hit[..., 3]).any()) and bool(torch.isfinite(hit[..., :3]).all())
        else:
            assert bool(torch.isnan(hit).all())
        assert bool(torch.isfinite(out[300:].float()).all())
    ops.check_device_status(q.device)


@pytest.mark.parametrize("hd,g", [(64, 1), (64, 4), (128, 2), (256, 1)])
def test_prompt_attn_is_one_prompt_at_a_time(hd, g):
    """Packing changes nothing: each prompt alone gives the same rows."""
    lens, Hkv = [200, 1, 333], 2
    q, k, v = prompt_case(lens, Hkv * g, Hkv, hd, torch.bfloat16, 11)
    out = ops.prompt_attn(q, k, v, ops.PromptPlan(lens, Hkv * g, Hkv, hd, q.device))
    a = 0
    for n in lens:
        one = ops.prompt_attn(q[a:a + n], k[a:a + n], v[a:a + n], ops.PromptPlan([n], Hkv * g, Hkv, hd, q.device))
        assert torch.equal(one, out[a:a + n])
        a += n


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_attn_strides_scale_and_extremes(hd):
    lens, Hq, Hkv = [150, 60], 4, 2
    q, k, v = prompt_case(lens, Hq, Hkv, hd, torch.float16, 5)
    plan = ops.PromptPlan(lens, Hq, Hkv, hd, q.device)
    want = ops.prompt_attn(q, k, v, plan, scale=0.3)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]   # [H,T,hd] storage
    assert torch.equal(ops.prompt_attn(*heads_first, plan, scale=0.3), want)
    wide = torch.zeros(sum(lens), Hkv, 2 * hd + 8, dtype=torch.float16, device=q.device)
    wide[..., 8:8 + hd] = k                                                             # rows with gaps
    assert torch.equal(ops.prompt_attn(q, wide[..., 8:8 + hd], v, plan, scale=0.3), want)
    odd = torch.zeros(sum(lens), Hkv, hd + 3, dtype=torch.float16, device=q.device)
    odd[..., 3:] = v                                                                    # unaligned rows: copied
    assert torch.equal(ops.prompt_attn(q, k, odd[..., 3:], plan, scale=0.3), want)
    into = torch.empty_like(want)
    assert ops.prompt_attn(q, k, v, plan, scale=0.3, out=into) is into and torch.equal(into, want)
    ref, _, bound = prompt_ref(q, k, v, lens, 0.3)
    check(want, ref, bound)
    big = ops.prompt_attn(q * 40, k, v, plan, scale=1.0)                                # one key takes all
    ref, _, bound = prompt_ref(q * 40, k, v, lens, 1.0)
    # scores up to ~2000: fp32 rounds them by up to 2^-13, which moves each probability by as much
    check(big, ref, bound + 2.0 ** -12 * float(v.abs().max()))
    faint = ops.prompt_attn(q, k, v, plan, scale=1e-30)                                 # plain running means
    ref, _, bound = prompt_ref(q, k, v, lens, 1e-30)
    check(faint, ref, bound)


@pytest.mark.parametrize("Hq,Hkv,hd", [(4, 1, 128), (16, 16, 64)])
def test_prompt_attn_many_items_per_block(Hq, Hkv, hd):
    """Far more work items than blocks, of very different lengths."""
    gen = torch.Generator().manual_seed(9)
    lens = [int(n) for n in torch.randint(0, 400, (150,), generator=gen)]
    q, k, v = prompt_case(lens, Hq, Hkv, hd, torch.bfloat16, 10)
    plan = ops.PromptPlan(lens, Hq, Hkv, hd, q.device)
    out = ops.prompt_attn(q, k, v, plan)
    ref, _, bound = prompt_ref(q, k, v, lens, hd ** -0.5)
    check(out, ref, bound)
    assert torch.equal(ops.prompt_attn(q, k, v, plan), out)
    ops.check_device_status(q.device)


def test_prompt_attn_equals_dense_attention_on_equal_lengths():
    """Equal lengths, one head per group: the dense kernel's problem."""
    B, S, H, hd = 3, 320, 4, 64
    gen = torch.Generator().manual_seed(1)
    qkv = randn(gen, torch.float16, B, S, 3 * H * hd)
    dense = ops.flash_attn(qkv, H, True).view(B * S, H, hd)
    packed = qkv.view(B * S, 3 * H, hd)
    plan = ops.PromptPlan([S] * B, H, H, hd, qkv.device)
    out = ops.prompt_attn(packed[:, :H], packed[:, H:2 * H], packed[:, 2 * H:], plan)
    assert float((out.float() - dense.float()).abs().max()) <= 2e-3


def test_prompt_attn_empty_and_refusals():
    dev = torch.device("cuda")
    e = torch.empty(0, 4, 64, dtype=torch.float16, device=dev)
    for lens in ([], [0, 0]):
        plan = ops.PromptPlan(lens, 4, 2, 64, dev)
        out, lse = ops.prompt_attn(e, e[:, :2], e[:, :2], plan, return_lse=True)
        assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    q, k, v = prompt_case([5], 4, 2, 64, torch.float16, 1)
    plan = ops.PromptPlan([5], 4, 2, 64, dev)
    with pytest.raises(RuntimeError, match="q must be"):
        ops.prompt_attn(q[:4], k, v, plan)
    with pytest.raises(RuntimeError, match="k must be"):
        ops.prompt_attn(q, q, v, plan)
    with pytest.raises(RuntimeError, match="v must be torch.float16"):
        ops.prompt_attn(q, k, v.bfloat16(), plan)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        ops.prompt_attn(q.float(), k.float(), v.float(), plan)
    with pytest.raises(RuntimeError, match="CUDA tensor|on cuda"):
        ops.prompt_attn(q.cpu(), k.cpu(), v.cpu(), plan)
    with pytest.raises(RuntimeError, match="out must"):
        ops.prompt_attn(q, k, v, plan, out=torch.empty(5, 4, 64, device=dev))
    qc = q.contiguous()
    with pytest.raises(RuntimeError, match="alias"):
        ops.prompt_attn(qc, k, v, plan, out=qc)
    for scale in (math.inf, math.nan, 0.0, -1.0):
        with pytest.raises(RuntimeError, match="scale"):
            ops.prompt_attn(q, k, v, plan, scale=scale)


# ------------------------------------------------------------------ decode

def decode_case(B, P, C, Hq, Hkv, hd, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return (randn(gen, dtype, B, Hq, hd), randn(gen, dtype, P, Hkv, hd), randn(gen, dtype, P, Hkv, hd),
            randn(gen, dtype, B, C, Hkv, hd), randn(gen, dtype, B, C, Hkv, hd))


def check_decode(args, lengths, weights=None, scale=None):
    q = args[0]
    lens = torch.tensor(lengths, dtype=torch.int32, device=q.device)
    s = q.shape[2] ** -0.5 if scale is None else scale
    ref, bound, w = decode_ref(*args, lengths, s)
    if weights is None:
        out = ops.shared_prefix_attn(*args, lens, scale=scale)
    else:
        before = weights.clone()
        out, neww = ops.shared_prefix_attn(*args, lens, key_weights=weights, scale=scale)
        assert torch.equal(weights, before)
        # this step's part: fp32 scores and sums, 4e-5 relative; then one fp32 addition
        want = weights.double() + w
        assert bool(((neww.double() - want).abs() <= 4e-5 * w + 2.0 ** -23 * want.abs()).all())
        for b, n in enumerate(lengths):
            n = min(max(n, 0), weights.shape[2])
            assert torch.equal(neww[b, :, n:], weights[b, :, n:])
        assert torch.equal(ops.shared_prefix_attn(*args, lens, scale=scale), out)
    check(out, ref, bound)
    ops.check_device_status(q.device)
    return out


DECODES = [  # (B, P, C, Hq, Hkv, hd, lengths)
    (1, 0, 1, 1, 1, 64, [1]), (1, 1, 1, 1, 1, 64, [0]), (2, 0, 8, 2, 2, 64, [0, 8]), (1, 512, 1024, 16, 2, 128, [700]),
    (3, 130, 70, 8, 2, 128, [0, 70, 33]), (5, 127, 65, 4, 4, 64, [64, 65, 1, 0, 63]), (7, 300, 200, 7, 1, 128, [200] * 7),
    (2, 64, 129, 12, 4, 96, [128, 129]), (33, 257, 40, 6, 2, 40, list(range(33))), (2, 100, 50, 128, 1, 64, [50, 13]),
    (2, 90, 50, 65, 1, 128, [49, 1]), (4, 1000, 300, 8, 4, 256, [300, 0, 299, 17]), (3, 50, 60, 4, 4, 8, [60, 1, 31]),
    (2, 70, 0, 4, 2, 128, [0, 0]), (70, 129, 5, 4, 2, 128, [i % 6 for i in range(70)]), (1, 3000, 2000, 5, 1, 192, [1999]),
    (4, 0, 3000, 8, 2, 128, [2999, 1, 1024, 2048]), (130, 600, 3, 2, 2, 64, [3] * 130), (2, 33, 20, 48, 3, 128, [20, 9]),
    (9, 2049, 700, 32, 8, 128, [0, 1, 16, 17, 255, 256, 257, 511, 700]),
]


# enough rows and prefix for the tensor-core tiles: one and several ranges and row tiles, a group wider than a tile's
# share, every padded head_dim; the last beside its caches (a part of the SMs each)
DECODES_TILES = [
    (130, 513, 3, 32, 8, 128), (300, 1025, 0, 16, 16, 64), (140, 900, 5, 8, 2, 256), (40, 4099, 33, 24, 3, 80),
    (5, 20001, 9, 128, 1, 64), (33, 26001, 40, 32, 8, 128),
]


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("B,P,C,Hq,Hkv,hd", DECODES_TILES)
def test_decode_behind_a_long_prefix(dt, B, P, C, Hq, Hkv, hd):
    args = decode_case(B, P, C, Hq, Hkv, hd, DT[dt], B + P + C)
    w = torch.rand(B, Hkv, C, generator=torch.Generator().manual_seed(1)).cuda()
    check_decode(args, [(7 * i) % (C + 1) for i in range(B)], w)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("B,P,C,Hq,Hkv,hd,lengths", DECODES)
def test_decode_matches_definition(dt, B, P, C, Hq, Hkv, hd, lengths):
    args = decode_case(B, P, C, Hq, Hkv, hd, DT[dt], B + P + C)
    check_decode(args, lengths)
    w = torch.rand(B, Hkv, C, generator=torch.Generator().manual_seed(1)).cuda()
    check_decode(args, lengths, w)


@pytest.mark.parametrize("hd,Hq,Hkv", [(64, 4, 4), (128, 8, 2), (256, 4, 2)])
def test_unused_cache_rows_may_hold_anything(hd, Hq, Hkv):
    B, P, C = 4, 200, 150
    lengths = [0, 150, 33, 128]
    args = decode_case(B, P, C, Hq, Hkv, hd, torch.bfloat16, 8)
    w = torch.rand(B, Hkv, C).cuda()
    clean = check_decode(args, lengths, w)
    for b, n in enumerate(lengths):
        args[3][b, n:] = math.nan
        args[4][b, n:] = math.inf if b % 2 else math.nan
    lens = torch.tensor(lengths, dtype=torch.int32).cuda()
    out, _ = ops.shared_prefix_attn(*args, lens, key_weights=w)
    assert torch.equal(out, clean)
    # another sequence's query and cache do not matter either
    args[0][1], args[3][1], args[4][1] = math.nan, math.nan, math.nan
    out = ops.shared_prefix_attn(*args, lens)
    keep = [0, 2, 3]
    assert torch.equal(out[keep], clean[keep])


def test_decode_no_key_gives_zeros_and_lengths_are_clamped():
    args = decode_case(3, 0, 20, 4, 2, 64, torch.float16, 2)
    out = check_decode(args, [0, -5, 20], torch.zeros(3, 2, 20, device="cuda"))
    assert bool((out[:2] == 0).all())
    lens = torch.tensor([99, 21, 20], dtype=torch.int32).cuda()
    full = torch.tensor([20, 20, 20], dtype=torch.int32).cuda()
    assert torch.equal(ops.shared_prefix_attn(*args, lens), ops.shared_prefix_attn(*args, full))
    e = decode_case(2, 0, 0, 4, 2, 64, torch.float16, 2)
    assert bool((ops.shared_prefix_attn(*e, torch.zeros(2, dtype=torch.int32, device="cuda")) == 0).all())


def test_decode_strides_and_layouts():
    args = decode_case(3, 140, 90, 8, 2, 128, torch.bfloat16, 4)
    lens = torch.tensor([90, 0, 41], dtype=torch.int32).cuda()
    w = torch.rand(3, 2, 90).cuda()
    want, want_w = ops.shared_prefix_attn(*args, lens, key_weights=w)
    q, pk, pv, kc, vc = args
    heads_first = [kc.transpose(1, 2).contiguous().transpose(1, 2), vc.transpose(1, 2).contiguous().transpose(1, 2)]
    pf = [pk.transpose(0, 1).contiguous().transpose(0, 1), pv.transpose(0, 1).contiguous().transpose(0, 1)]
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    got, got_w = ops.shared_prefix_attn(qt, *pf, *heads_first, lens, key_weights=w)
    assert torch.equal(got, want) and torch.equal(got_w, want_w)
    both = torch.stack([kc, vc], 2)                                  # [B,C,2,Hkv,hd]
    got, got_w = ops.shared_prefix_attn(q, pk, pv, both[:, :, 0], both[:, :, 1], lens, key_weights=w)
    assert torch.equal(got, want) and torch.equal(got_w, want_w)


@pytest.mark.parametrize("scale", [1e-30, 0.01, 1.0])
def test_decode_scales(scale):
    args = decode_case(2, 200, 100, 8, 2, 128, torch.bfloat16, 6)
    check_decode(args, [100, 37], torch.zeros(2, 2, 100, device="cuda"), scale=scale)


def test_decode_offsets_past_32_bits():
    """A cache whose last rows lie beyond 2^32 bytes (and 2^31 elements)."""
    B, C, Hkv, hd = 2, 1200000, 8, 128
    k = torch.zeros(B, C, Hkv, hd, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    lens = torch.tensor([5, C], dtype=torch.int32).cuda()
    q = torch.ones(B, Hkv, hd, dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, Hkv, hd, dtype=torch.bfloat16, device="cuda")
    k[1, C - 1, 7] = 4.0          # score 4 * 128 / sqrt(128) ~ 45: takes the whole softmax of head 7
    v[1, C - 1] = 2.0
    w = torch.zeros(B, Hkv, C, device="cuda")
    out, neww = ops.shared_prefix_attn(q, none, none, k, v, lens, key_weights=w)
    assert float((out[1, 7].float() - 2).abs().max()) < 0.01
    assert float(out[1, :7].float().abs().max()) < 1e-4 and bool((out[0] == 0).all())
    assert float(neww[1, 7, C - 1]) > 0.999 and abs(float(neww[1, 0].double().sum()) - 1) < 1e-3
    kept = ops.cache_evict(k, v, neww, lens, 16, 2)
    assert kept.lengths.tolist() == [5, 16]
    assert kept.positions[1, 7, -2:].tolist() == [C - 2, C - 1] and bool((kept.v[1, 15] == 2).all())


def test_decode_refusals():
    q, pk, pv, kc, vc = decode_case(2, 10, 6, 4, 2, 64, torch.float16, 1)
    lens = torch.tensor([6, 2], dtype=torch.int32).cuda()
    with pytest.raises(RuntimeError, match="prefix_v must be"):
        ops.shared_prefix_attn(q, pk, pv[:9], kc, vc, lens)
    with pytest.raises(RuntimeError, match="multiple of num_kv_heads"):
        ops.shared_prefix_attn(q[:, :3], pk, pv, kc, vc, lens)
    with pytest.raises(RuntimeError, match="lengths must be int32"):
        ops.shared_prefix_attn(q, pk, pv, kc, vc, lens.long())
    with pytest.raises(RuntimeError, match="key_weights must be float32"):
        ops.shared_prefix_attn(q, pk, pv, kc, vc, lens, key_weights=torch.zeros(2, 2, 5, device="cuda"))
    with pytest.raises(RuntimeError, match="v_cache must be torch.float16"):
        ops.shared_prefix_attn(q, pk, pv, kc, vc.bfloat16(), lens)
    with pytest.raises(RuntimeError, match="scale"):
        ops.shared_prefix_attn(q, pk, pv, kc, vc, lens, scale=0.0)
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.shared_prefix_attn(q[..., :12], pk[..., :12], pv[..., :12], kc[..., :12], vc[..., :12], lens)
    assert ops.shared_prefix_attn(q[:0], pk, pv, kc[:0], vc[:0], lens[:0]).shape == (0, 4, 64)


# ------------------------------------------------------------------ eviction

def check_evict(k, v, w, lengths, budget, recent, out=None):
    lens = torch.tensor(lengths, dtype=torch.int32).cuda()
    B, C, H, hd = k.shape
    got = ops.cache_evict(k, v, w, lens, budget, recent, out=out)
    kept = evict_ref(w.cpu(), lengths, C, budget, recent)
    pos = got.positions.cpu()
    for b in range(B):
        for h in range(H):
            idx = kept[b][h]
            n = len(idx)
            assert pos[b, h].tolist() == idx + [-1] * (budget - n), (b, h)
            at = torch.tensor(idx, dtype=torch.long, device="cuda")
            for t, src in ((got.k, k), (got.v, v)):
                assert torch.equal(t[b, :n, h], src[b, at, h])
                assert not bool(t[b, n:budget, h].any())
            assert torch.equal(got.key_weights[b, h, :n].nan_to_num(nan=-1.0), w[b, h, at].nan_to_num(nan=-1.0))
            assert not bool(got.key_weights[b, h, n:].any())
        assert int(got.lengths[b]) == len(kept[b][0])
    return got


def cache_case(B, C, H, hd, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    w = torch.exp(2 * torch.randn(B, H, C, generator=gen) - 4) * (torch.rand(B, H, C, generator=gen) > 0.2)
    return randn(gen, dtype, B, C, H, hd), randn(gen, dtype, B, C, H, hd), w.cuda()


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("B,C,H,hd,lengths,budget,recent", [
    (1, 1, 1, 64, [1], 1, 0), (2, 10, 2, 8, [10, 3], 4, 1), (2, 256, 4, 64, [200, 256], 128, 32),
    (3, 777, 2, 128, [777, 0, 500], 333, 333), (3, 777, 2, 128, [776, 40, 501], 500, 0),
    (2, 1025, 3, 40, [1025, 1024], 1, 1), (2, 1025, 3, 96, [1025, 1024], 1, 0), (1, 5000, 2, 256, [4999], 4998, 100),
    (2, 300, 2, 64, [300, 299], 400, 50), (4, 2048, 1, 80, [2048, 2047, 1030, 1], 1024, 7),
    (1, 33000, 2, 8, [33000], 20000, 500), (2, 64, 40, 128, [-3, 99], 17, 16),
])
def test_evict_matches_definition(dt, B, C, H, hd, lengths, budget, recent):
    check_evict(*cache_case(B, C, H, hd, DT[dt], C + budget), lengths, budget, recent)


@pytest.mark.parametrize("hd", [40, 64, 128, 200])
def test_evict_many_caches_and_rows(hd):
    """More kept rows than the choosing blocks copy, more caches than there are SMs; some below the budget."""
    B, C = 40, 900
    lengths = [(97 * b) % (C + 1) for b in range(B)]
    check_evict(*cache_case(B, C, 4, hd, torch.bfloat16, hd), lengths, 640, 17)


def test_evict_ties_and_special_weights():
    B, C, H, hd = 5, 700, 2, 64
    k, v, _ = cache_case(B, C, H, hd, torch.float16, 1)
    w = torch.zeros(B, H, C)
    w[1] = torch.randint(0, 3, (H, C), generator=torch.Generator().manual_seed(2)).float()   # many ties
    w[2, :, ::3], w[2, :, 1::3], w[2, :, 2::3] = math.nan, -math.inf, -1.0
    w[3, :, ::2] = -0.0                                                                       # equals +0
    w[4] = torch.randn(H, C, generator=torch.Generator().manual_seed(3)) * 1e-42              # subnormal, both signs
    w[4, :, 5], w[4, :, 600] = math.inf, 3e38
    w = w.cuda()
    for budget, recent in ((1, 0), (250, 30), (300, 0), (699, 1)):
        check_evict(k, v, w, [700, 700, 700, 699, 700], budget, recent)


@pytest.mark.parametrize("C", [900, 4096, 9001, 40000, 90001])  # every row count per thread, clusters of 1 to 8 blocks
def test_evict_search_ranges(C):
    """The key that cuts lies among positive, zero or negative weights; within one value's ties; in a tiny range."""
    g = torch.Generator().manual_seed(C)
    H, hd, n = 2, 8, C - 3
    k, v, _ = cache_case(6, C, H, hd, torch.float16, 1)
    x = torch.randn(6, H, C, generator=g)
    w = x.exp()                                                   # 0: positive over a wide range
    w[1] = x[1].relu()                                            # half zeros
    w[2] = x[2]                                                   # both signs
    w[3] = -1.0 - x[3].abs()                                      # negative only
    w[4] = torch.where(x[4] > 0, 1.0 + 2.0 ** -23, 1.0)           # two neighbouring values
    w[5] = 7.5                                                    # one value
    w = w.cuda()
    for budget, recent in ((n // 7, 5), (n // 2 + n // 4, 64), (n - 1, 0), (50, 50)):
        check_evict(k, v, w, [n] * 6, budget, recent)


def test_evict_into_an_existing_cache_and_layouts():
    k, v, w = cache_case(3, 200, 2, 128, torch.bfloat16, 7)
    into = torch.full((3, 150, 2, 2, 128), 7.0, dtype=torch.bfloat16, device="cuda")          # k and v interleaved
    got = check_evict(k, v, w, [200, 60, 199], 100, 10, out=(into[:, :, 0], into[:, :, 1]))
    assert got.k.data_ptr() == into.data_ptr() and bool((into[:, 100:] == 7).all())
    kh, vh = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))                 # [B,H,C,hd] storage
    check_evict(kh, vh, w, [200, 60, 199], 100, 10)


def test_evict_refusals():
    k, v, w = cache_case(2, 20, 2, 64, torch.float16, 1)
    lens = torch.tensor([20, 20], dtype=torch.int32).cuda()
    for budget, recent in ((0, 0), (5, 6), (5, -1)):
        with pytest.raises(RuntimeError, match="budget must be positive"):
            ops.cache_evict(k, v, w, lens, budget, recent)
    with pytest.raises(RuntimeError, match="alias"):
        ops.cache_evict(k, v, w, lens, 5, 1, out=(k, v))
    o = torch.empty_like(k)
    with pytest.raises(RuntimeError, match="alias"):
        ops.cache_evict(k, v, w, lens, 5, 1, out=(o, o))
    with pytest.raises(RuntimeError, match="k_out must be"):
        ops.cache_evict(k, v, w, lens, 5, 1, out=(o[:, :4], v[:, :4]))
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        ops.cache_evict(k.float(), v.float(), w, lens, 5, 1)
    with pytest.raises(RuntimeError, match="key_weights must be"):
        ops.cache_evict(k, v, w.half(), lens, 5, 1)
    assert ops.cache_evict(k[:0], v[:0], w[:0], lens[:0], 5, 1).lengths.shape == (0,)


# ------------------------------------------------------------------ streams, graphs

def test_serving_ops_on_a_side_stream_and_in_a_graph():
    args = decode_case(3, 300, 200, 8, 2, 128, torch.bfloat16, 12)
    lens = torch.tensor([200, 3, 90], dtype=torch.int32).cuda()
    w = torch.rand(3, 2, 200).cuda()
    q, k, v = prompt_case([90, 3, 200], 8, 2, 128, torch.bfloat16, 13)
    plan = ops.PromptPlan([90, 3, 200], 8, 2, 128, q.device)

    def everything():
        o, neww = ops.shared_prefix_attn(*args, lens, key_weights=w)
        return (ops.prompt_attn(q, k, v, plan), o, neww, *ops.cache_evict(args[3], args[4], neww, lens, 64, 16))

    want = everything()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = everything()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = everything()
    for t in held:
        t.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_decode_lse_joins_two_key_sets():
    """return_lse: the results over the prefix and over the caches join to the result over both."""
    q, pk, pv, kc, vc = decode_case(5, 150, 90, 8, 2, 128, torch.float16, 21)
    lens = torch.tensor([90, 0, 1, 44, 64], dtype=torch.int32).cuda()
    both, lse = ops.shared_prefix_attn(q, pk, pv, kc, vc, lens, return_lse=True)
    a, la = ops.shared_prefix_attn(q, pk, pv, kc[:, :0], vc[:, :0], lens, return_lse=True)
    b, neww, lb = ops.shared_prefix_attn(q, pk[:0], pv[:0], kc, vc, lens, key_weights=torch.zeros(5, 2, 90).cuda(),
                                         return_lse=True)
    assert bool((lb[1] == -math.inf).all()) and neww.shape == (5, 2, 90)
    assert float((torch.logaddexp(la, lb) - lse).abs().max()) <= 2e-5 * (1 + float(lse.abs().max()))
    wa, wb = torch.exp(la - lse)[..., None], torch.exp(lb - lse)[..., None]
    # three roundings to fp16 of values below max |v|, each probability rounded once more
    tol = 4 * 2.0 ** -11 * float(torch.cat([pv.flatten(), vc.flatten()]).abs().max())
    assert float((wa * a.float() + wb * b.float() - both.float()).abs().max()) <= tol
