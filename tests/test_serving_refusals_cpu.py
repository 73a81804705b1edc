"""What the serving entry points refuse, or leave as it was, before anything reaches a GPU."""

import ctypes as C

import pytest
import torch

from tiktok_techjam_2026_track3_b200 import CachedAttention, SequenceCache, SharedPrefix, _lib, ops


def test_workspaces_that_would_be_used_are_dense_and_on_the_device():
    """The kernels get a workspace's address alone."""
    here, there = torch.device("cpu"), torch.device("cuda", 0)
    own = torch.empty(64, dtype=torch.float32)
    assert ops._workspace(own, 256, here) is own
    assert ops._workspace(own, 0, here) is own
    fresh = ops._workspace(own, 257, here)                    # too small: replaced, as without one
    assert fresh.numel() == 257 and fresh.dtype == torch.uint8
    assert ops._workspace(None, 8, here).numel() == 8
    for bad, need in ((own, 256), (torch.empty(64), 1)):      # a host address
        with pytest.raises(RuntimeError, match="workspace must be a contiguous tensor on cuda:0"):
            ops._workspace(bad, need, there)
    for bad in (own[::2], torch.empty(1).expand(64), torch.empty(8, 8)[:, :4]):
        with pytest.raises(RuntimeError, match="workspace must be a contiguous"):
            ops._workspace(bad, bad.numel() * 4, here)


# ------------------------------------------------------------------ the cached attention layer

@pytest.fixture
def layer(monkeypatch):
    """A layer whose projections run on the CPU, so that its calls reach the operators (which
    refuse CPU tensors)."""
    monkeypatch.setattr(ops, "linear", torch.nn.functional.linear)
    return CachedAttention(256, 4, 2).half()


def test_prefill_refuses_a_plan_of_other_lengths(layer):
    """Equal totals are not enough: such a plan's rows would attend across prompts."""
    cache = layer.new_cache(2, 16)
    x = torch.randn(9, 256).half()
    for other in ([5, 4], [9, 0], [4, 5, 0], [4, 4]):
        with pytest.raises(RuntimeError, match="other prompt lengths"):
            layer.prefill(x, [4, 5], cache, plan=layer.plan(other))
    with pytest.raises(RuntimeError, match="9 tokens, seq_lens 8"):
        layer.prefill(x, [4, 4], cache)
    for lens in ([4, 5], torch.tensor([4, 5])):               # accepted up to the operator itself
        with pytest.raises(RuntimeError, match="no CPU path"):
            layer.prefill(x, lens, layer.new_cache(2, 16), plan=layer.plan([4, 5]))


def state(cache):
    return cache.host_lengths, cache.lengths.tolist(), cache.key_weights.clone()


def test_a_refused_prefill_leaves_the_cache_empty(layer):
    cache = layer.new_cache(2, 16)
    x = torch.randn(9, 256).half()
    for args in (dict(x=x, seq_lens=[4, 5]), dict(x=x, seq_lens=[4, 5], plan=layer.plan([4, 5])),
                 dict(x=x, seq_lens=[4, 5], prefix=SharedPrefix(x, x)), dict(x=x[:, :8], seq_lens=[4, 5])):
        with pytest.raises(RuntimeError):
            layer.prefill(cache=cache, **args)
        assert cache.host_lengths == [0, 0] and cache.lengths.tolist() == [0, 0]


def test_a_refused_decode_leaves_the_cache_as_it_was(layer, monkeypatch):
    cache = layer.new_cache(2, 16)
    cache.extend([3, 0], torch.randn(3, 2, 64).half(), torch.randn(3, 2, 64).half())
    cache.key_weights[0, :, :3] = 0.5
    before, rows = state(cache), cache.k[0, :3].clone()
    bad = torch.zeros(4, 1, 64, dtype=torch.float16)
    for prefix in (None, SharedPrefix(bad, bad), SharedPrefix(bad.float(), bad)):
        with pytest.raises(RuntimeError):
            layer.decode(torch.randn(2, 256).half(), cache, prefix)
        now = state(cache)
        assert now[:2] == before[:2] and torch.equal(now[2], before[2]) and torch.equal(cache.k[0, :3], rows)
    # and where the attention is accepted but the output projection fails
    monkeypatch.setattr(ops, "shared_prefix_attn", lambda q, *a, key_weights: (q[:, :1], key_weights + 1))
    with pytest.raises(RuntimeError):
        layer.decode(torch.randn(2, 256).half(), cache)
    now = state(cache)
    assert now[:2] == before[:2] and torch.equal(now[2], before[2])


def test_cache_rows_are_never_spread_over_sequences():
    """One row for several places, other heads, another type: refused, nothing appended."""
    cache = SequenceCache(2, 8, 2, 64, torch.float16, torch.device("cpu"))
    row = lambda n, h=2, hd=64: torch.randn(n, h, hd).half()
    cache.extend([1, 0], row(1), row(1))
    for k, v in ((row(1), row(1)), (row(2), row(1)), (row(1), row(2)), (row(2, 1), row(2, 1)), (row(2, 2, 1), row(2)),
                 (row(2), row(2).float()), (row(3), row(3))):
        with pytest.raises(RuntimeError, match="must be torch.float16"):
            cache.append(k, v)
        with pytest.raises(RuntimeError, match="must be torch.float16"):
            cache.extend([2, 0], k, v)
    with pytest.raises(RuntimeError, match="cannot take -1 rows"):
        cache.extend([2, -1], row(1), row(1))
    assert cache.host_lengths == [1, 0] and cache.lengths.tolist() == [1, 0]
    k = row(2)
    cache.append(k, k)
    cache.extend([1, 2], row(3), row(3))
    assert cache.host_lengths == [3, 3] and torch.equal(cache.k[0, 1], k[0]) and torch.equal(cache.v[1, 0], k[1])


def test_evict_refuses_to_write_the_lengths_it_reads():
    """Every head's blocks read a sequence's length; the first one writes the new one."""
    at = lambda i: (i + 1) << 40   # never dereferenced
    a = _lib.CacheEvictArgs(
        k_cache=at(0), v_cache=at(1), key_weights=at(2), lengths=at(3), k_out=at(4), v_out=at(5), weights_out=at(6),
        positions_out=at(8), batch=2, capacity=8, num_kv_heads=2, head_dim=64, budget=4, recent=1,
        k_seq_stride=1024, k_row_stride=128, k_head_stride=64, v_seq_stride=1024, v_row_stride=128, v_head_stride=64,
        k_out_seq_stride=512, k_out_row_stride=128, k_out_head_stride=64, v_out_seq_stride=512, v_out_row_stride=128,
        v_out_head_stride=64)
    lib = _lib.load()
    for out in (at(3), at(3) + 4, at(3) - 4):
        a.lengths_out = out
        assert lib.ttj_cache_evict(C.byref(a), None) == -1
        assert b"lengths_out must not alias lengths" in lib.ttj_last_error()
