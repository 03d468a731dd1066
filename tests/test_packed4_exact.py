"""4-bit storage where bits can get lost: operands that need more than 16 bits, probabilities far below the
largest, scores of any size, values next to far larger ones.  Inputs are made so that a rounding of an
operand shows in the result; references are in 64 bits, from the packed values themselves."""
import math

import numpy as np
import pytest
import torch

from test_packed4 import BF16, F16, F32, attention_bound, attention_ref, half_step, random_packed

import anima_attn
from anima_attn import Packed4, _lib as L


def codes_of(n):
    """Whole numbers in [-8, 7], [..., K] -> packed codes [..., K/2] (word and nibble order of anima_attn.h)."""
    n = np.asarray(n)
    lead, K = n.shape[:-1], n.shape[-1]
    c = (n + 8).astype(np.uint32).reshape(lead + (K // 128, 4, 4, 8))  # g, i, e
    words = np.zeros(lead + (K // 128, 16), np.uint32)
    for g in range(4):
        for i in range(4):
            for e in range(8):
                words[..., 4 * i + g] |= c[..., g, i, e] << np.uint32(4 * ((e >> 1) + 4 * (e & 1)))
    return words.astype("<u4").view(np.uint8).reshape(lead + (K // 2,))


def packed(n, s, device="cuda"):
    """Codes n [..., K] and scales s [..., K/32] -> (Packed4, the values in 64 bits)."""
    n, s = np.asarray(n), np.asarray(s).astype(np.float16)
    return (Packed4(torch.from_numpy(codes_of(n)).to(device), torch.from_numpy(s).to(device)),
            n * np.repeat(s.astype(np.float64), 32, -1))


def every_head(p, BH):
    """One head's packed rows [1, S, 128], for every head."""
    return Packed4(*(t.expand(BH, -1, -1).contiguous() for t in p))


def way(BH, Sq, Skv):
    """How a call is read: directly, or by tiles of 128 keys for units of one or two tiles of 128 rows."""
    if Sq <= 16 or BH * Sq * max(Skv, 256) <= 1 << (20 + (Skv >= 4096) + (Skv >= 32768)):
        return "direct"
    return "tile1" if Sq <= 128 else "tile2"


WAYS = [("direct", 1, 1), ("direct", 2, 9), ("tile1", 40, 128), ("tile1", 70, 65), ("tile2", 1, 4200), ("tile2", 16, 300)]


# ------------------------------------------------------------------ scratch
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [L.DTYPE_F16, L.DTYPE_BF16])
@pytest.mark.parametrize("B,H,Sq,Skv", [(2, 16, 4096, 512), (2, 16, 16384, 512), (2, 16, 4096, 65536), (1, 1, 1 << 17, 1 << 20)])
def test_a_packed_cache_is_not_written_out(dtype, B, H, Sq, Skv):
    """Scratch is for slices' partial results: none where the query tiles alone fill the device, and never
    near the 256 bytes a key and side of a cache in 16 bits."""
    assert L.lib.anima_attn_kv4_workspace_size(dtype, B, H, Sq, Skv) == 0
    for sq in (1, 8, 64, 200):
        assert L.lib.anima_attn_kv4_workspace_size(dtype, 1, 1, sq, 1 << 20) <= 64 * (sq + 255) * 130 * 4
