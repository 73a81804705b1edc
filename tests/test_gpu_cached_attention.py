"""A serving session through CachedAttention (packed prompts behind a shared prefix,
decode steps, eviction) against the same layer restated in 64 bits."""

import pytest
import torch

from serving_ref import attend
from tiktok_techjam_2026_track3_b200 import CachedAttention, ops

pytestmark = pytest.mark.gpu


class Restated:
    """Per-sequence lists of (key, value) rows per head, 64-bit arithmetic on the
    device layer's 16-bit weights and inputs; keys and values rounded as stored."""

    def __init__(self, layer):
        self.layer = layer
        self.w = {k: v.double() for k, v in layer.state_dict().items()}

    def qkv(self, x):
        hq, hkv, hd = self.layer.num_heads, self.layer.num_kv_heads, self.layer.head_dim
        p = (x.double() @ self.w["qkv_proj.weight"].T + self.w["qkv_proj.bias"]).to(x.dtype).view(len(x), -1, hd)
        return p[:, :hq], p[:, hq:hq + hkv], p[:, hq + hkv:]

    def attend(self, q, k, v):
        """q [Hq,hd] over k, v [n,Hkv,hd] -> (context [Hq*hd], probabilities [Hq,n])"""
        g = self.layer.num_heads // self.layer.num_kv_heads
        outs, probs = [], []
        for h in range(self.layer.num_heads):
            o, _, p, _ = attend(q[h:h + 1], k[:, h // g], v[:, h // g], self.layer.head_dim ** -0.5)
            outs.append(o[0])
            probs.append(p[0])
        return torch.cat(outs), torch.stack(probs)

    def out(self, ctx):
        return ctx @ self.w["out_proj.weight"].T + self.w["out_proj.bias"]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d_model,P", [(8, 2, 512, 70), (4, 4, 256, 0), (4, 1, 512, 300)])
def test_session_matches_restated_layer(dtype, hq, hkv, d_model, P):
    torch.manual_seed(hq * P + d_model)
    layer = CachedAttention(d_model, hq, hkv).to("cuda", dtype).eval()
    ref = Restated(layer)
    lens = [40, 0, 9, 130]
    B, C = len(lens), 160
    rand = lambda n: torch.randn(n, d_model, device="cuda").to(dtype)
    # projections, attention and output are each rounded once to `dtype` here and there:
    # a few units of values of magnitude ~1
    tol = 8 * (2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8)
    with torch.inference_mode():
        xp, x = rand(P), rand(sum(lens))
        prefix = layer.encode_prefix(xp) if P else None
        cache = layer.new_cache(B, C)
        y = layer.prefill(x, lens, cache, prefix)
        _, pk, pv = ref.qkv(xp) if P else (None, x.new_empty(0, hkv, d_model // hq), x.new_empty(0, hkv, d_model // hq))
        q, k, v = ref.qkv(x)
        a = 0
        want = []
        for n in lens:
            for i in range(a, a + n):
                ctx, _ = ref.attend(q[i], torch.cat([pk, k[a:i + 1]]), torch.cat([pv, v[a:i + 1]]))
                want.append(ref.out(ctx))
            a += n
        assert float((y.double() - torch.stack(want)).abs().max()) <= tol
        assert cache.host_lengths == lens and cache.lengths.tolist() == lens
        for step in range(4):
            if step == 2:
                before = [(cache.k.clone(), cache.v.clone(), cache.key_weights.clone())][0]
                positions = cache.evict(32, 8)
                assert cache.host_lengths == [32, 2, 11, 32] == cache.lengths.tolist()
                for b, n in enumerate(cache.host_lengths):
                    for h in range(hkv):
                        at = positions[b, h, :n].long()
                        assert torch.equal(cache.k[b, :n, h], before[0][b, at, h])
                        assert torch.equal(cache.v[b, :n, h], before[1][b, at, h])
                        assert torch.equal(cache.key_weights[b, h, :n], before[2][b, h, at])
            xt = rand(B)
            weights = cache.key_weights.clone()
            y = layer.decode(xt, cache, prefix)
            q, _, _ = ref.qkv(xt)
            for b, n in enumerate(cache.host_lengths):
                kk, vv = torch.cat([pk, cache.k[b, :n]]), torch.cat([pv, cache.v[b, :n]])
                ctx, prob = ref.attend(q[b], kk, vv)
                assert float((y[b].double() - ref.out(ctx)).abs().max()) <= tol
                got = (cache.key_weights - weights)[b, :, :n].double()
                assert float((got - prob[:, P:].view(hkv, hq // hkv, n).sum(1)).abs().max()) <= 2 * tol
    ops.check_device_status(y.device)


def test_a_full_cache_is_refused_on_the_host():
    layer = CachedAttention(256, 4, 2).to("cuda", torch.float16).eval()
    cache = layer.new_cache(2, 8)
    x = torch.randn(9, 256, device="cuda", dtype=torch.float16)
    with torch.inference_mode():
        with pytest.raises(RuntimeError, match="full"):
            layer.prefill(x, [9, 0], cache)
        layer.prefill(x, [8, 1], cache)
        with pytest.raises(RuntimeError, match="full"):
            layer.decode(x[:2], cache)
        with pytest.raises(RuntimeError, match="empty"):
            layer.prefill(x, [4, 5], cache)
        with pytest.raises(RuntimeError, match="exceeds"):
            cache.evict(9, 1)
        cache.evict(4, 1)
        assert layer.decode(x[:2], cache).shape == (2, 256) and cache.host_lengths == [5, 2]
