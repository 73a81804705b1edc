"""CachedAttention step by step within derived bounds, on weights whose attention is far
from uniform: a cache left out, or weights left at zero, would show in every dtype."""

import pytest
import torch

from serving_ref import UNIT, attend, out_bound
from tiktok_techjam_2026_track3_b200 import CachedAttention, ops

pytestmark = pytest.mark.gpu


def sharp_layer(d_model, hq, hkv, dtype):
    """Scores with a standard deviation of about 3 (torch's default weights give 1/3)."""
    layer = CachedAttention(d_model, hq, hkv).to("cuda", dtype).eval()
    with torch.no_grad():
        layer.qkv_proj.weight[:(hq + hkv) * layer.head_dim] *= 3
    return layer


def check_qkv(layer, x, parts):
    """The projection against 64 bits: one rounding, and fp32 sums."""
    w, b = layer.qkv_proj.weight.double(), layer.qkv_proj.bias.double()
    ref = (x.double() @ w.T + b).view(len(x), -1, layer.head_dim)
    size = (x.double().abs() @ w.abs().T + b.abs()).view(ref.shape)
    got = torch.cat(parts, 1).double()
    assert bool(((got - ref).abs() <= UNIT[x.dtype] * ref.abs() + 1e-5 * size).all())


def context(layer, q, k, v):
    """(context, bound, probabilities, lse) of one token q [Hq,hd] over k, v [n,Hkv,hd] as stored, in 64 bits."""
    g = layer.num_heads // layer.num_kv_heads
    outs, bounds, probs, spreads, lses = [], [], [], [], []
    for h in range(layer.num_heads):
        vh = v[:, h // g]
        o, lse, p, spread = attend(q[h:h + 1], k[:, h // g], vh, layer.head_dim ** -0.5)
        outs.append(o[0])
        bounds.append(out_bound(q.dtype, o[0], spread[0], len(vh), float(vh.abs().max())))
        probs.append(p[0])
        spreads.append(spread[0])
        lses.append(lse)
    return torch.stack(outs), torch.stack(bounds), torch.stack(probs), torch.stack(spreads), torch.stack(lses)


def output(layer, ctx, ctx_bound):
    """The projection of a context known to within ctx_bound: (y, bound)."""
    w, b = layer.out_proj.weight.double(), layer.out_proj.bias.double()
    ctx, ctx_bound = ctx.flatten(), ctx_bound.flatten()
    y = ctx @ w.T + b
    moved = ctx_bound @ w.abs().T
    return y, moved + UNIT[layer.out_proj.weight.dtype] * (y.abs() + moved) + 1e-5 * (ctx.abs() @ w.abs().T + b.abs())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d_model,P", [(8, 2, 512, 70), (4, 4, 256, 0), (4, 1, 512, 300)])
def test_every_step_within_its_bound(dtype, hq, hkv, d_model, P):
    torch.manual_seed(P + hq)
    layer = sharp_layer(d_model, hq, hkv, dtype)
    g, lens, u = hq // hkv, [40, 0, 9, 130], UNIT[dtype]
    rand = lambda n: torch.randn(n, d_model, device="cuda").to(dtype)
    with torch.inference_mode():
        xp, x = rand(P), rand(sum(lens))
        prefix = layer.encode_prefix(xp) if P else None
        none = x.new_empty(0, hkv, layer.head_dim)
        pk, pv = (prefix.k, prefix.v) if P else (none, none)
        q, k, v = layer._qkv(x)
        check_qkv(layer, x, (q, k, v))
        cache = layer.new_cache(len(lens), 160)
        y = layer.prefill(x, lens, cache, prefix)
        a = 0
        for b, n in enumerate(lens):
            assert torch.equal(cache.k[b, :n], k[a:a + n]) and torch.equal(cache.v[b, :n], v[a:a + n])
            for i in range(a, a + n):
                ctx, bound, _, spread, lse = context(layer, q[i], torch.cat([pk, k[a:i + 1]]), torch.cat([pv, v[a:i + 1]]))
                if P:
                    # Each part was rounded before the join and their sum once more (together at most
                    # u of the spread beyond out_bound's own rounding); the share, a logistic function of
                    # two lse of 2e-5 relative each, moves the result by at most a quarter of that times
                    # the parts' distance, itself at most the values' range.
                    reach = 2 * float(torch.cat([pv, v[a:i + 1]]).abs().max())
                    bound = bound + u * (1 + 2 * u) * spread + 1e-5 * (1 + lse.abs()) * reach
                want, most = output(layer, ctx, bound)
                assert bool(((y[i].double() - want).abs() <= most).all()), (b, i)
            a += n
        seen_without, seen_zero = False, True
        for step in range(5):
            if step == 3:
                cache.evict(32, 8)
            xt, weights = rand(len(lens)), cache.key_weights.clone()
            q, _, _ = layer._qkv(xt)
            y = layer.decode(xt, cache, prefix)
            for b, n in enumerate(cache.host_lengths):
                ctx, bound, prob, _, _ = context(layer, q[b], torch.cat([pk, cache.k[b, :n]]), torch.cat([pv, cache.v[b, :n]]))
                want, most = output(layer, ctx, bound)
                assert bool(((y[b].double() - want).abs() <= most).all()), (step, b)
                added = prob[:, P:].view(hkv, g, n).sum(1)
                sums = weights[b, :, :n].double() + added
                limit = 4e-5 * added + 2.0 ** -23 * sums.abs()
                assert bool(((cache.key_weights[b, :, :n].double() - sums).abs() <= limit).all()), (step, b)
                # the bounds tell: weights never added, the cache left out
                seen_zero &= bool((added > limit).any())
                if P:
                    rest, _ = output(layer, *context(layer, q[b], pk, pv)[:2])
                    seen_without |= bool(((rest - want).abs() > 2 * most).any())
        assert seen_zero and (seen_without or not P)
    ops.check_device_status(y.device)
