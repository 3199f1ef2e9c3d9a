"""A model's key / value cache held in 4 or 8 bits, for decoding.

The reference decodes with HuggingFace's `generate` (Inference/GenerateTexts.py:19), whose cache holds the model's dtype; this one takes
0.5625 (4 bits) or 1.0625 (8 bits) bytes per value, scales included, and its tokens are written in place - nothing is
concatenated as a sequence grows.  `branchgan.generate.generate(..., cache_bits=)` decodes through it; the operators are
ops.kv_cache_append / kv_cache_read / kv_cache_attention.
"""
import torch

from . import _capi as C
from . import ops


class QuantizedKVCache:
    """n_layers caches of (batch, heads, capacity, head_dim) keys and values in one buffer."""

    def __init__(self, n_layers, batch, heads, capacity, head_dim, bits=4, device="cuda"):
        tile = C.lib().bg_kv_cache_tile_bytes(int(bits), int(head_dim))
        if tile == 0:
            raise ValueError(f"a quantised cache takes bits 4 or 8 and head sizes 32, 64, 128 or 256, got bits={bits}, head_dim={head_dim}")
        if min(n_layers, batch, heads, capacity) < 1:
            raise ValueError(f"QuantizedKVCache: n_layers={n_layers}, batch={batch}, heads={heads}, capacity={capacity}")
        self.bits, self.head_dim, self.capacity = int(bits), int(head_dim), int(capacity)
        tiles = -(-int(capacity) // ops.KV_TILE)
        self.data = torch.zeros((n_layers, batch, heads, tiles * tile), dtype=torch.uint8, device=device)
        self._layers = [ops.KVCacheLayer(d, self.bits, self.head_dim, self.capacity) for d in self.data]

    def layer(self, i):
        return self._layers[i]

    def __len__(self):
        return self.data.shape[0]

    @property
    def nbytes(self):
        return self.data.numel()
