"""The ways of the attention over packed K and V, each reached on purpose: rows read directly, and tiles for one and
two query tiles, whole and in slices.  The way follows from a call's sizes (csrc/attn_kv4.cu, rows_path), and every
case says which one it means."""
import math

import numpy as np
import pytest
import torch

from test_packed4 import BF16, F16, F32, attention_ref, half_step, random_packed
from test_packed4_exact import every_head, packed, way

import anima_attn


def bound(out, pv, top, dtype):
    """One rounding bound for every way.  A score is a sum of at most 256 exact products and 16 scaled ones, each
    rounded by one fp32 step of sum |q k| scale at most: 512 steps with the scale's and the merges'.  An exponential
    is off by 2^-20; P in two bf16 parts and V in two by 2^-16; sums, rescaling and merges by 2^-17.  Numerator and
    denominator: twice.  The result is rounded once to its type."""
    c = 2 * (512 * 2.0 ** -23 * top + 2.0 ** -20 + 2.0 ** -16 + 2.0 ** -17)
    return pv * c * (1 + c) + np.abs(out) * half_step(dtype) + (6e-8 if dtype == F16 else 1e-37)


def check(want_way, B, H, Sq, Skv, dtype, lens=None, q=None, kv=None, seed=0):
    """One cache for all heads, other rows in each; q and (k, k's values) may be given."""
    BH = B * H
    assert way(BH, Sq, Skv) == want_way
    if q is None:
        q = torch.randn(BH, Sq, 128, generator=torch.Generator().manual_seed(seed))
    q = q.to(dtype).cuda()
    k, kvals = random_packed((1, Skv, 128), seed + 1) if kv is None else kv
    v, vvals = random_packed((1, Skv, 128), seed + 2)
    k, v = every_head(k, BH), every_head(v, BH)
    vl = None
    if lens is not None:
        vl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for b, n in enumerate(lens):  # what lies behind a length never counts
            for t in (k, v):
                t.scales.view(B, H, Skv, 4)[b, :, max(n, 0):] = float("nan")
                t.codes.view(B, H, Skv, 64)[b, :, max(n, 0):] = 0xF1
    kr, vr = (np.broadcast_to(t, (BH,) + t.shape[1:]) for t in (kvals, vvals))
    out, pv, top = attention_ref(q.double().cpu().numpy(), kr, vr, B, H, lens, 1 / math.sqrt(128))
    for odt in (dtype, F32):
        got = anima_attn.attention_core_kv4(q, k, v, B, H, kv_valid_len=vl, out_dtype=odt)
        err, tol = np.abs(got.double().cpu().numpy() - out), bound(out, pv, top, odt)
        assert (err <= tol).all(), (odt, float((err / tol).max()), np.argwhere(~(err <= tol))[:3])
        for b, n in enumerate(lens or ()):
            assert n > 0 or (got[b] == 0).all()
    assert anima_attn.status() == 0


def heads_for_tiles(Sq, Skv):
    """Heads with which Sq > 16 rows and Skv < 4096 keys pass the direct way's work, an even number."""
    return 2 * ((1 << 20) // (2 * Sq * max(Skv, 256)) + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Sq", [17, 64, 127, 128, 129, 257])
@pytest.mark.parametrize("Skv", [1, 2, 63, 64, 65, 127, 128, 129, 193, 333])
def test_tiles(Sq, Skv, dtype):
    check("tile1" if Sq <= 128 else "tile2", 1, heads_for_tiles(Sq, Skv), Sq, Skv, dtype, seed=Sq + Skv)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Sq", [17, 128, 129, 257])
@pytest.mark.parametrize("lens", [[0, 1], [129, 64], [65, 0], [200, 63], [-5, 300]])
def test_tiles_masked(Sq, lens, dtype):
    H = (heads_for_tiles(Sq, 200) + 1) // 2 + 1
    check("tile1" if Sq <= 128 else "tile2", 2, H, Sq, 200, dtype, lens=lens, seed=Sq)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("want,Sq,Skv", [("tile1", 120, 9000), ("tile1", 128, 33000), ("tile2", 300, 9001), ("tile2", 129, 9000)])
@pytest.mark.parametrize("lens", [None, [9000, 1], [0, 130], [65, 8999], [4481, 0]])
def test_tiles_in_slices(want, Sq, Skv, lens, dtype):
    """One or two units, their keys in slices, of which lengths leave some without a key."""
    check(want, 2, 1, Sq, Skv, dtype, lens=lens, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("want,Sq,H,Skv", [("tile1", 100, 200, 200), ("tile1", 17, 310, 200), ("tile2", 2307, 32, 133), ("tile2", 300, 161, 70)])
def test_more_units_than_multiprocessors(want, Sq, H, Skv, dtype):
    check(want, 1, H, Sq, Skv, dtype, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,H,Sq,Skv,lens", [(1, 4, 1000, 200, None), (2, 2, 511, 500, [500, 33]), (2, 1, 200, 5000, [0, 4999]), (1, 1, 64, 60000, None),
                                             (1, 2, 16, 70001, None)])
def test_many_rows_read_directly(B, H, Sq, Skv, lens, dtype):
    check("direct", B, H, Sq, Skv, dtype, lens=lens, seed=5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("want,B,H,Sq,Skv", [("direct", 1, 2, 1, 700), ("direct", 1, 2, 12, 700), ("tile1", 1, 80, 100, 700), ("tile2", 1, 16, 300, 700),
                                             ("tile1", 2, 1, 120, 9000), ("tile2", 2, 1, 300, 9000)])
@pytest.mark.parametrize("up", [True, False])
def test_maxima_that_jump(want, B, H, Sq, Skv, up, dtype):
    """Keys whose size grows from one tile of 64 to the next, so that a row's maximum rises by far more than 8 log2
    units at every tile and what was summed is scaled down each time, and keys that shrink, so that it never does."""
    tiles = (Skv + 63) // 64
    size = 2.0 ** (np.minimum(np.arange(tiles), 9) * 0.6)
    size = np.repeat(size if up else size[::-1], 64)[:Skv]
    rng = np.random.default_rng(6)
    k = packed(rng.integers(-8, 8, (1, Skv, 128)), 0.1 * size[None, :, None] * rng.uniform(0.9, 1.1, (1, Skv, 4)))
    check(want, B, H, Sq, Skv, dtype, kv=k, seed=7)
