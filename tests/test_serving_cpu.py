"""The serving entry points without a GPU: the prompt plan, struct layouts and the
argument checks that fail before anything reaches the device."""

import ctypes as C
import random
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from tiktok_techjam_2026_track3_b200 import _lib, ops

HEADER = Path(__file__).resolve().parent.parent / "include" / "ttj_attn.h"


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("cname,pyname", [("ttj_prompt_attn_args", "PromptAttnArgs"),
                                          ("ttj_shared_prefix_attn_args", "SharedPrefixAttnArgs"),
                                          ("ttj_cache_evict_args", "CacheEvictArgs")])
def test_struct_layout_matches_header(tmp_path, cname, pyname):
    cls = getattr(_lib, pyname)
    fields = [f for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(
        ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){",
         f'printf("%zu\\n", sizeof({cname}));'] +
        [f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields] + ["return 0;}"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got[0] == C.sizeof(cls) and got[1:] == [getattr(cls, f).offset for f in fields]


@pytest.mark.parametrize("Hq,Hkv,hd", [(4, 4, 64), (8, 2, 128), (7, 1, 64), (128, 1, 64), (6, 2, 256), (65, 1, 200)])
def test_plan_covers_every_token_once(Hq, Hkv, hd):
    rng = random.Random(Hq * hd)
    lens = [rng.choice([0, 1, 2, 127, 128, 129, rng.randint(0, 700)]) for _ in range(30)]
    plan = ops.PromptPlan(lens, Hq, Hkv, hd, "cpu")
    starts, seen, a = [], [], 0
    for n in lens:
        starts.append(a)
        a += n
    limit = (2 if hd <= 128 else 1) * (128 // (Hq // Hkv))
    reach = []
    for q_row, rows, k_row, _ in plan.table[:plan.entries].tolist():
        assert 1 <= rows <= limit and k_row in starts
        owner = max(i for i, s in enumerate(starts) if s == k_row and lens[i] > 0)
        assert k_row <= q_row and q_row + rows <= k_row + lens[owner]
        seen += range(q_row, q_row + rows)
        reach.append(q_row + rows - k_row)
    assert sorted(seen) == list(range(sum(lens))) and plan.tokens == sum(lens)
    assert reach == sorted(reach, reverse=True)


def test_plan_refusals():
    for args, text in ((([5, -1], 4, 2, 64), "negative"), (([5], 4, 3, 64), "multiple of num_kv_heads"),
                       (([5], 0, 0, 64), "multiple of num_kv_heads"), (([5], 4, 2, 12), "head_dim"),
                       (([5], 4, 2, 264), "head_dim"), (([5], 258, 2, 64), "128 query heads"),
                       (([1 << 40], 4, 2, 64), "length"), (([8000000] * 300, 4, 2, 64), "2\\^31")):
        with pytest.raises(RuntimeError, match=text):
            ops.PromptPlan(*args, "cpu")
    assert ops.PromptPlan([], 4, 2, 64, "cpu").entries == 0
    assert ops.PromptPlan(torch.tensor([3, 0, 4]), 4, 2, 64, "cpu").seq_lens == (3, 0, 4)


def _bad(call, base, code, text, **change):
    a = type(base)(**{**{f: getattr(base, f) for f, _ in base._fields_}, **change})
    assert call(C.byref(a), None) == code, (change, _lib.load().ttj_last_error())
    assert text in _lib.load().ttj_last_error(), _lib.load().ttj_last_error()


def test_c_argument_checks_without_a_device():
    lib = _lib.load()
    at = lambda i: (i + 1) << 40   # never dereferenced
    p = _lib.PromptAttnArgs(q=at(0), k=at(1), v=at(2), out=at(3), plan=at(4), plan_entries=1, tokens=4,
                            num_heads=4, num_kv_heads=2, head_dim=64, q_token_stride=512, q_head_stride=64,
                            k_token_stride=512, k_head_stride=64, v_token_stride=512, v_head_stride=64,
                            scale=0.125, dtype=0)
    f = lib.ttj_prompt_attn_fwd
    assert f(None, None) == -1
    _bad(f, p, -1, b"dtype", dtype=2)
    _bad(f, p, -1, b"non-NULL", plan=None)
    _bad(f, p, -1, b"plan does not belong", plan_entries=0)
    _bad(f, p, -1, b"plan does not belong", plan_entries=5)
    _bad(f, p, -1, b"multiple of num_kv_heads", num_heads=5)
    _bad(f, p, -2, b"128 query heads", num_heads=516)
    _bad(f, p, -2, b"head_dim", head_dim=20)
    _bad(f, p, -2, b"q strides", q_token_stride=516)
    _bad(f, p, -2, b"k strides", k_head_stride=0)
    _bad(f, p, -2, b"v strides", v_token_stride=1 << 45)
    _bad(f, p, -3, b"aligned", v=at(2) + 8)
    _bad(f, p, -1, b"alias", out=at(0) + 512)
    _bad(f, p, -2, b"2^31", tokens=1 << 31)
    d = _lib.SharedPrefixAttnArgs(
        q=at(0), prefix_k=at(1), prefix_v=at(2), k_cache=at(3), v_cache=at(4), lengths=at(5), out=at(6),
        workspace=at(7), workspace_bytes=1 << 39, batch=2, prefix_len=8, capacity=8, num_heads=4, num_kv_heads=2,
        head_dim=64, q_seq_stride=256, q_head_stride=64, prefix_k_row_stride=128, prefix_k_head_stride=64,
        prefix_v_row_stride=128, prefix_v_head_stride=64, k_seq_stride=1024, k_row_stride=128, k_head_stride=64,
        v_seq_stride=1024, v_row_stride=128, v_head_stride=64, scale=0.125, dtype=1)
    f = lib.ttj_shared_prefix_attn_fwd
    assert f(None, None) == -1
    _bad(f, d, -1, b"non-NULL", lengths=None)
    _bad(f, d, -1, b"go together", key_weights=at(8))
    _bad(f, d, -1, b"alias", key_weights=at(8), key_weights_out=at(8) + 64)
    _bad(f, d, -2, b"k_cache strides", k_row_stride=100)
    _bad(f, d, -2, b"prefix_v strides", prefix_v_head_stride=-64)
    _bad(f, d, -6, b"workspace", workspace=None, key_weights=at(8), key_weights_out=at(9))
    _bad(f, d, -6, b"workspace", workspace_bytes=1, key_weights=at(8), key_weights_out=at(9))
    _bad(f, d, -2, b"maximum", capacity=1 << 31)
    _bad(f, d, -1, b"negative", prefix_len=-1)
    assert lib.ttj_shared_prefix_attn_workspace_size(0, 8, 8, 4, 2, 64, 1) == 0
    assert lib.ttj_shared_prefix_attn_workspace_size(1 << 40, 8, 1 << 30, 4, 2, 64, 1) == 0
    e = _lib.CacheEvictArgs(
        k_cache=at(0), v_cache=at(1), key_weights=at(2), lengths=at(3), k_out=at(4), v_out=at(5), weights_out=at(6),
        lengths_out=at(7), positions_out=at(8), batch=2, capacity=8, num_kv_heads=2, head_dim=64, budget=4, recent=1,
        k_seq_stride=1024, k_row_stride=128, k_head_stride=64, v_seq_stride=1024, v_row_stride=128, v_head_stride=64,
        k_out_seq_stride=512, k_out_row_stride=128, k_out_head_stride=64, v_out_seq_stride=512, v_out_row_stride=128,
        v_out_head_stride=64)
    f = lib.ttj_cache_evict
    assert f(None, None) == -1
    _bad(f, e, -1, b"budget", budget=0)
    _bad(f, e, -1, b"recent", recent=5)
    _bad(f, e, -1, b"non-NULL", positions_out=None)
    _bad(f, e, -1, b"alias", k_out=at(1))
    _bad(f, e, -1, b"alias", v_out=at(4))
    _bad(f, e, -1, b"alias", weights_out=at(2))
    _bad(f, e, -3, b"aligned", k_out=at(4) + 2)
    _bad(f, e, -2, b"k_out strides", k_out_row_stride=4)


def test_cpu_tensors_are_refused():
    plan = ops.PromptPlan([4], 4, 2, 64, "cpu")
    q, kv = torch.zeros(4, 4, 64, dtype=torch.float16), torch.zeros(4, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.prompt_attn(q, kv, kv, plan)
    cache = torch.zeros(4, 3, 2, 64, dtype=torch.float16)
    lens = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.shared_prefix_attn(q, kv, kv, cache, cache, lens)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.cache_evict(cache, cache, torch.zeros(4, 2, 3), lens, 2, 1)
