"""Serving operators on the GPU at the edges of what they accept: workspaces at any
allowed address, scores of minus infinity, infinities and NaN in long prompts, the decode
step's kernels right behind the ones that wrote its inputs."""

import math

import pytest
import torch

from serving_ref import DT
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
