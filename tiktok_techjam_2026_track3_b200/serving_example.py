"""A serving session on random weights: four prompts behind a shared prefix, 128 decode
steps, the caches cut to 256 rows when one is full.

    python -m tiktok_techjam_2026_track3_b200.serving_example
"""

from __future__ import annotations

import torch

from . import ops
from .serving import CachedAttention


def main() -> int:
    torch.manual_seed(0)
    layer = CachedAttention(1024, 8, 2).to("cuda", torch.bfloat16).eval()
    lens = [300, 17, 0, 128]
    with torch.inference_mode():
        prefix = layer.encode_prefix(torch.randn(500, 1024, device="cuda", dtype=torch.bfloat16))
        cache = layer.new_cache(len(lens), 384)
        x = torch.randn(sum(lens), 1024, device="cuda", dtype=torch.bfloat16)
        y = layer.prefill(x, lens, cache, prefix)
        print(f"prefill: {tuple(y.shape)}, cache lengths {cache.host_lengths}")
        for step in range(1, 129):
            if max(cache.host_lengths) == cache.capacity:
                cache.evict(256, 64)
                print(f"evicted before step {step}: cache lengths {cache.host_lengths}")
            token = torch.randn(len(lens), 1024, device="cuda", dtype=torch.bfloat16)
            y = layer.decode(token, cache, prefix)
        print(f"decode: {step} steps, {tuple(y.shape)}, cache lengths {cache.host_lengths}")
    ops.check_device_status(y.device)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
