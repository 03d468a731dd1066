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
    """Scratch is for partial results: none for slices where the query tiles alone fill the device, 128 KB a
    multiprocessor for chains of more than 8192 keys, and never the 256 bytes a key and side of a cache in 16 bits."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert L.lib.anima_attn_kv4_workspace_size(dtype, B, H, Sq, Skv) <= (sms * 256 * 512 if Skv > 8192 else 0)
    for sq in (1, 8, 64, 200):
        assert L.lib.anima_attn_kv4_workspace_size(dtype, 1, 1, sq, 1 << 20) <= 64 * (sq + 255) * 130 * 4 + sms * 256 * 512


# ------------------------------------------------------------------ attention: K, V and P keep their bits
def crafted(way_, BH, Sq, dtype, q, k, v, scale=1.0):
    """One cache for all heads, the same rows in each head: the result against 64 bits.
    Tolerance: P is held in two bf16 parts, P (1 + 2^-17), and times V in two bf16 parts loses the product
    of the lower parts, 2^-9 each; an exponential is off by 2^-22 and its argument, here of scores that
    fp32 holds exactly, by 2^-22 more; a handful of fp32 sums.  Together below 2^-16 of sum p |v|.
    The result is rounded once."""
    (kp, kv), (vp, vv) = k, v
    assert way(BH, Sq, kv.shape[1]) == way_
    qd = q[None].expand(BH, -1, -1).to(dtype).contiguous().cuda()
    assert torch.equal(qd[0].double().cpu(), q.double())  # the type holds q
    got = anima_attn.attention_core_kv4(qd, every_head(kp, BH), every_head(vp, BH), 1, BH, scale=scale)
    out, pv, _ = attention_ref(q.double().numpy()[None], kv, vv, 1, 1, None, scale)
    err = np.abs(got.double().cpu().numpy() - out)
    tol = pv * 2.0 ** -16 + np.abs(out) * half_step(dtype) + (3e-8 if dtype == F16 else 0.0)
    assert (err <= tol).all(), float((err / np.maximum(tol, 1e-300)).max())
    assert anima_attn.status() == 0


def two_keys(a, sa, b, sb):
    """Two keys (or values) whose 128 entries are a sa and b sb."""
    return packed(np.stack([np.full(128, a), np.full(128, b)])[None], np.stack([np.full(4, sa), np.full(4, sb)])[None])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("way_,BH,Sq", WAYS)
def test_keys_keep_their_bits(way_, BH, Sq, dtype):
    """7 (1 + 2^-10) needs 13 bits.  Against a key of 7 the score differs by 128 * 7 * 2^-10 = 0.875; of
    keys rounded to 16 bits it would by 1, or by 0."""
    q = torch.zeros(Sq, 128)
    q[:, 37] = 128.0
    crafted(way_, BH, Sq, dtype, q, two_keys(7, 1 + 2.0 ** -10, 7, 1.0), two_keys(1, 1.0, -1, 1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("way_,BH,Sq", WAYS)
def test_values_keep_their_bits(way_, BH, Sq, dtype):
    """Equal weights on 7 (1 + 2^-10) and -7: what is left is what the 13th bit holds."""
    crafted(way_, BH, Sq, dtype, torch.zeros(Sq, 128), two_keys(0, 1.0, 0, 1.0), two_keys(7, 1 + 2.0 ** -10, -7, 1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("way_,BH,Sq", WAYS)
def test_probabilities_keep_their_bits(way_, BH, Sq, dtype):
    """Weights 1 and p, p near 1/2, on values 1 and -2: 1 - 2 p is left, near 0."""
    q = torch.zeros(Sq, 128)
    step = 2.0 ** -11 if dtype == F16 else 2.0 ** -8
    q[:, 5] = 0.6875 + step * (torch.arange(Sq) % 23 - 11)
    crafted(way_, BH, Sq, dtype, q, two_keys(0, 1.0, -1, 1.0), two_keys(1, 1.0, -2, 1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("BH,Sq", [(75, 17), (75, 3), (38, 257)])
@pytest.mark.parametrize("ahead", [16.5, 17.5, 20.0, 30.0])
def test_a_long_cache_keeps_its_tail(dtype, BH, Sq, ahead):
    """65536 keys of which one is `ahead` above the others, e^ahead times their weight, and has a value of
    zero, theirs being 1: the others' share is a small number, and relative to it (it is sum p |v|) the
    weights have to be right.  Sums of 65536 equal terms in fp32: each addition rounds by half a step, at
    most 65536 / 16 additions of one accumulator on the tensor core and 4096 in a thread's sum."""
    N = 65536
    n = np.zeros((1, N, 128), np.int64)
    n[0, 5, 0] = -8
    k, kv = packed(n, np.full((1, N, 4), -ahead / 8))
    n = np.ones((1, N, 128), np.int64)
    n[0, 5] = 0
    v, _ = packed(n, np.ones((1, N, 4)))
    q = torch.zeros(BH, Sq, 128, dtype=dtype, device="cuda")
    q[:, :, 0] = 1
    got = anima_attn.attention_core_kv4(q, every_head(k, BH), every_head(v, BH), 1, BH, scale=1.0).double().cpu().numpy()
    w = (N - 1) * math.exp(-kv[0, 5, 0])
    want = w / (1 + w)
    tol = want * (2.0 ** -16 + 2 * 4096 * 2.0 ** -24 + half_step(dtype)) + (3e-8 if dtype == F16 else 0.0)
    assert np.abs(got - want).max() <= tol, (float(np.abs(got - want).max()), want)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e8, 1e10, 1e20, 1e30])
@pytest.mark.parametrize("BH,Sq,Skv", [(1, 1, 700), (2, 11, 700), (40, 100, 700), (16, 300, 700), (1, 100, 65000), (2, 200, 9000)])
def test_rows_of_huge_scores(size, BH, Sq, Skv):
    """bf16 rows whose scores are so large that one key takes all: the output is that key's value.  A row
    is compared where the best key is ahead by more than the scores' own rounding (512 fp32 steps of
    sum |q| |k| scale) and 40."""
    g = torch.Generator().manual_seed(21)
    q = (torch.randn(BH, Sq, 128, generator=g) * size).to(BF16).cuda()
    k, kv = random_packed((1, Skv, 128), 22)
    v, vv = random_packed((1, Skv, 128), 23)
    got = anima_attn.attention_core_kv4(q, every_head(k, BH), every_head(v, BH), 1, BH)[0].transpose(0, 1).double().cpu().numpy()
    sc = 1 / math.sqrt(128)
    qd = q.double().cpu().numpy().reshape(-1, 128)
    s = qd @ kv[0].T * sc
    top2 = np.partition(s, Skv - 2, -1)[:, -2:]
    far = top2[:, 1] - top2[:, 0] > 512 * 2.0 ** -23 * (np.abs(qd) @ np.abs(kv[0]).T * sc).max(-1) + 40
    assert far.mean() > 0.95
    want = vv[0][s.argmax(-1)]
    err = np.abs(got.reshape(-1, 128) - want)
    assert (err[far] <= np.abs(want[far]) * (half_step(BF16) + 2.0 ** -16)).all(), float(np.nanmax(err[far]))
    assert anima_attn.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scale", [1e-45, 1e-30, 3e38])
@pytest.mark.parametrize("BH,Sq", [(2, 1), (2, 9), (40, 128), (16, 300), (2, 3000)])
def test_scales_at_the_ends_of_fp32(dtype, scale, BH, Sq):
    """Equal scores, keys cut off in the middle of a tile: the mean of the values, whatever the scale.
    Rounding: weights of 1 are exact, sums of at most 333 values in fp32, the result once."""
    Skv, n = 333, 201
    k, _ = random_packed((1, Skv, 128), 51)
    v, vv = random_packed((1, Skv, 128), 52)
    q = torch.zeros(BH, Sq, 128, dtype=dtype, device="cuda")
    got = anima_attn.attention_core_kv4(q, every_head(k, BH), every_head(v, BH), 1, BH, scale=scale,
                                        kv_valid_len=torch.tensor([n], dtype=torch.int32, device="cuda")).double().cpu().numpy()
    want, size = vv[0, :n].mean(0), np.abs(vv[0, :n]).mean(0)
    assert (np.abs(got - want) <= np.abs(want) * half_step(dtype) + size * 400 * 2.0 ** -23 + (3e-8 if dtype == F16 else 0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Sq", [1, 5])
def test_a_large_query_value_leaves_the_others(dtype, Sq):
    """One value of a row is far larger than the others and meets keys of zero there: the scores are
    the others' alone (bound: as for any direct call, of sum |q| |k|, where it has no part)."""
    rng = np.random.default_rng(31)
    BH, Skv = 2, 300
    n = rng.integers(-8, 8, (BH, Skv, 128))
    n[..., 3] = 0
    k, kv = packed(n, rng.uniform(50, 100, (BH, Skv, 4)))
    v, vv = random_packed((BH, Skv, 128), 32)
    q = torch.randn(BH, Sq, 128, generator=torch.Generator().manual_seed(33)) * 2.0 ** -7
    q[..., 3] = 60000.0 if dtype == F16 else 1e9
    q = q.to(dtype)
    got = anima_attn.attention_core_kv4(q.cuda(), k, v, 1, BH).double().cpu().numpy()
    out, pv, top = attention_ref(q.double().numpy(), kv, vv, 1, BH, None, 1 / math.sqrt(128))
    err, tol = np.abs(got - out), attention_bound(out, pv, top, dtype, True)
    assert (err <= tol).all(), float((err / tol).max())


# ------------------------------------------------------------------ fp32 results
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,H,Sq,Skv,lens", [(2, 3, 1, 77, None), (1, 2, 1, 20011, None), (2, 2, 9, 300, [300, 0]), (1, 1, 5, 9000, [5000]),
                                             (2, 20, 128, 200, [200, 63]), (1, 2, 2100, 300, None), (2, 1, 300, 5000, [0, 4999]),
                                             (3, 13, 2049, 130, [0, 130, 40])])
def test_fp32_results(B, H, Sq, Skv, lens, dtype):
    """out_dtype float32, in each way, whole and in slices: the result before any 16-bit rounding.  Bound: scores
    by 512 fp32 steps of sum |q k| scale, exponentials by 2^-20, P in two bf16 parts and V's parts by
    2^-16, sums and merges by 2^-17; numerator and denominator, so twice."""
    g = torch.Generator().manual_seed(61)
    q = torch.randn(B * H, Sq, 128, generator=g).to(dtype).cuda()
    k, kv = random_packed((1, Skv, 128), 62)
    v, vv = random_packed((1, Skv, 128), 63)
    k, v = every_head(k, B * H), every_head(v, B * H)
    kv, vv = (np.broadcast_to(t, (B * H,) + t.shape[1:]) for t in (kv, vv))
    vl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = anima_attn.attention_core_kv4(q, k, v, B, H, kv_valid_len=vl, out_dtype=F32)
    assert got.dtype == F32 and got.shape == (B, Sq, H, 128)
    out, pv, top = attention_ref(q.double().cpu().numpy(), kv, vv, B, H, lens, 1 / math.sqrt(128))
    err = np.abs(got.double().cpu().numpy() - out)
    tol = pv * 2 * (512 * 2.0 ** -23 * top + 2.0 ** -20 + 2.0 ** -16 + 2.0 ** -17) + 1e-37
    assert (err <= tol).all(), float((err / np.maximum(tol, 1e-300)).max())
    if np.abs(out).max() > 0:
        assert np.linalg.norm(err) <= 2.0 ** -15 * np.linalg.norm(out)  # a 16-bit rounding alone is 2^-12 and more
    # the 16-bit result is this one rounded
    assert torch.equal(anima_attn.attention_core_kv4(q, k, v, B, H, kv_valid_len=vl), got.to(dtype))
    buf = torch.full((B, H + 1, Sq + 1, 136), 7.0, device="cuda")
    view = buf[:, :H, 1:, :128]
    assert anima_attn.attention_core_kv4(q, k, v, B, H, kv_valid_len=vl, out=view, out_layout="bhsd", out_dtype=F32) is view
    assert torch.equal(view.transpose(1, 2), got)
    view.fill_(7.0)
    assert (buf == 7).all()


@pytest.mark.gpu
def test_cached_kv_results_are_fp32_by_default():
    """attention_cached_kv over packed K/V writes fp32 results, as it does over 16-bit ones; other types are
    theirs rounded."""
    from anima_attn.ops import attention_cached_kv, prologue
    g = torch.Generator(device="cuda").manual_seed(64)
    B, S, H, N = 2, 300, 2, 130
    q = torch.randn(B, S, H, 128, device="cuda", generator=g)
    k, kv = random_packed((B * H, N, 128), 65)
    v, vv = random_packed((B * H, N, 128), 66)
    got = attention_cached_kv(q, k, v)
    qh, _, _ = prologue(q, None, None, None, None, None, 1e-6, True, False, F16)
    out, _, _ = attention_ref(qh.double().cpu().numpy(), kv, vv, B, H, None, 1 / math.sqrt(128))
    assert got.dtype == F32 and np.linalg.norm(got.double().cpu().numpy() - out) <= 2.0 ** -15 * np.linalg.norm(out)
    assert torch.equal(attention_cached_kv(q, k, v, out_dtype=F16), got.half())
    for dt in (F32, F16, BF16):
        buf = torch.empty(B, S, H, 128, dtype=dt, device="cuda")
        assert attention_cached_kv(q, k, v, out=buf) is buf and torch.equal(buf, got.to(dt))
    for bad in (torch.empty(2 * B, S, H, 128, dtype=dt, device="cuda") for dt in (F32, F16, BF16)):
        with pytest.raises(ValueError):
            attention_cached_kv(q, k, v, out=bad)
    with pytest.raises(ValueError):
        attention_cached_kv(q[:1], k, v)
    one = torch.empty(2, 1, S, H, 128, dtype=BF16, device="cuda")  # would broadcast
    with pytest.raises(ValueError):
        attention_cached_kv(q, k, v, out=one.expand(2, B, S, H, 128))


def test_output_types_that_are_refused(monkeypatch):
    monkeypatch.setattr(anima_attn.packed, "_here", lambda *ts: 0)
    q = torch.zeros(4, 3, 128, dtype=F16)
    k = Packed4(torch.zeros(4, 5, 64, dtype=torch.uint8), torch.zeros(4, 5, 4, dtype=F16))
    for kw in ({"out_dtype": BF16}, {"out_dtype": torch.float64}, {"out": torch.zeros(2, 3, 2, 128)},
               {"out_dtype": F32, "out": torch.zeros(2, 3, 2, 128, dtype=F16)}):
        with pytest.raises(ValueError):
            anima_attn.attention_core_kv4(q, k, k, 2, 2, **kw)


# ------------------------------------------------------------------ matvec4: every value keeps its bits
def matvec_bound_each(ax, aw, K, y, out_dtype, steps=0):
    """Rounding bound of one result of sum |x| |w| alone, wherever the other values of a group lie.  A
    value is three bf16 parts, together exact; their products with whole numbers are exact.  A group's 3 x
    32 products are summed by the tensor core (one fp32 step each), K/32 scaled sums are rounded, at most 8
    warps', the three parts', the addend: 96 + K/32 + 16 steps.  `steps` more for what x itself is off by.
    Results and sums below fp32's normal range round to multiples of 2^-149."""
    S = ax @ np.swapaxes(aw, -1, -2)
    return S * 2.0 ** -23 * (96 + K / 32 + 16 + steps) + (K / 32 + 16) * 2.0 ** -148 + np.abs(y) * half_step(out_dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 3, 8, 9])
@pytest.mark.parametrize("size", [1e3, 1e5, 1e8, 1e20, 3.4e38])
def test_matvec_outliers_leave_the_others(size, M):
    """A group's largest value meets weights of zero: what is left is the other values' sum, to fp32's
    accuracy (relative to sum |x| |w|, in which the large value has no part)."""
    rng = np.random.default_rng(41)
    N, K = 50, 384
    n = rng.integers(-8, 8, (N, K))
    n[:, [7, 40, 200]] = 0
    w, wv = packed(n, rng.uniform(0.01, 0.1, (N, K // 32)))
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(42))
    x[:, 7], x[:, 40], x[:, 200] = size, -size, size / 3
    y = anima_attn.matvec4(x.cuda(), w).double().cpu().numpy()
    xv = x.double().numpy()
    want = xv @ wv.T
    err, tol = np.abs(y - want), matvec_bound_each(np.abs(xv), np.abs(wv), K, want, F32)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("std", [1e-43, 1e-38, 1e-30, 1e30, 2e36])
def test_matvec_over_the_range_of_fp32(std):
    g = torch.Generator().manual_seed(43)
    w, wv = random_packed((64, 256), 44, std=0.05)
    x = torch.randn(2, 256, generator=g) * std
    y = anima_attn.matvec4(x.cuda(), w).double().cpu().numpy()
    xv = x.double().numpy()
    want = xv @ wv.T
    err, tol = np.abs(y - want), matvec_bound_each(np.abs(xv), np.abs(wv), 256, want, F32)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.gpu
def test_matvec_several_infinities():
    """Infinities of a group whose products agree give that infinity, as a sum in fp32 does."""
    n = np.ones((4, 256), np.int64)
    n[1], n[2, 9] = -1, 0
    w, _ = packed(n, np.full((4, 8), 0.5))
    x = torch.ones(1, 256)
    x[0, 9] = x[0, 20] = x[0, 100] = math.inf
    y = anima_attn.matvec4(x.cuda(), w).cpu()[0]
    assert y[0] == math.inf and y[1] == -math.inf and y[2].isnan() and y[3] == math.inf
    x[0, 20] = -math.inf
    assert anima_attn.matvec4(x.cuda(), w).isnan().all()
    # a NaN whose upper 16 bits alone are an infinity's
    x = torch.ones(1, 256)
    x.view(torch.int32)[0, 9] = 0x7F800001
    assert anima_attn.matvec4(x.cuda(), w).isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_matvec_silu_of_large_negative_values(dtype):
    """SiLU(-88) is -88 e^-88 = -5e-37, inside fp32's range; further down it goes to 0, and -infinity to NaN.
    Bound on x: 8 steps as elsewhere, and |x| + 2 steps for the rounding of the exponential of x."""
    w, wv = packed(np.ones((16, 128), np.int64), np.ones((16, 4)))
    for lo, hi in ((-88.6, -87.0), (-103.0, -88.5), (-87.0, -60.0)):
        x = torch.linspace(lo, hi, 128)[None].to(dtype)
        xv = x.double().numpy()
        sv = xv / (1 + np.exp(-xv))
        sv[xv < -88.72] = 0  # e^-x leaves fp32: below 2^-121 in the result
        y = anima_attn.matvec4(x.cuda(), w, silu=True).double().cpu().numpy()
        want = sv @ wv.T
        tol = matvec_bound_each(np.abs(sv), np.abs(wv), 128, want, F32, steps=8 + 105)
        near = (np.abs(xv + 88.72) < 0.01).sum() * 88.73 * math.exp(-88.71)  # may fall on either side
        assert (np.abs(y - want) <= tol + near).all()
    x = torch.full((1, 128), -math.inf, dtype=dtype)
    assert anima_attn.matvec4(x.cuda(), w, silu=True).isnan().all()


# ------------------------------------------------------------------ matvec4 in place
@pytest.mark.gpu
@pytest.mark.parametrize("E,N,K", [(1, 77, 128), (1, 33, 4096), (5, 96, 256), (3, 1003, 1024)])
@pytest.mark.parametrize("M", [1, 2, 9, 17])
@pytest.mark.parametrize("xdt", [F32, F16, BF16])
def test_matvec_adds_in_place(E, N, K, M, xdt):
    """out = add, the same tensor, over several passes of rows, several warps a tile and views: bit for bit what
    comes out beside it."""
    g = torch.Generator().manual_seed(71)
    w, _ = random_packed((E, N, K), 72, std=0.05)
    x = torch.randn(E, M, K, generator=g).to(xdt).cuda()
    add = torch.randn(E, M, N, generator=g).cuda()
    want = anima_attn.matvec4(x, w, add=add)
    inplace = add.clone()
    assert anima_attn.matvec4(x, w, add=inplace, out=inplace) is inplace and torch.equal(inplace, want)
    buf = torch.full((E, M + 1, N + 3), 7.0, device="cuda")
    view = buf[:, :M, 1:N + 1]
    view.copy_(add)
    anima_attn.matvec4(x, w, add=view, out=view)
    assert torch.equal(view, want)
    view.fill_(7.0)
    assert (buf == 7).all()
    if E == 1:  # accumulating into a gradient-like buffer, call after call
        a, b = torch.zeros(M, N, device="cuda"), torch.zeros(M, N, device="cuda")
        one = Packed4(w.codes[0], w.scales[0])
        for _ in range(3):
            anima_attn.matvec4(x[0], one, add=a, out=a)
            b = anima_attn.matvec4(x[0], one, add=b)
        assert torch.equal(a, b)


def test_the_addend_is_not_read_through_the_read_only_path():
    """out may be add: __ldg is only defined for memory that nothing writes while the kernel runs."""
    import os
    from conftest import PKG_ROOT
    with open(os.path.join(PKG_ROOT, "csrc", "packed4.cu")) as f:
        assert "__ldg(p.add" not in f.read()


@pytest.mark.gpu
@pytest.mark.parametrize("BH,Sq,N", [(2, 1, 200000), (75, 3, 200000), (75, 17, 200000), (38, 129, 200000), (1, 100, 1000000)])
@pytest.mark.parametrize("values", ["one", "two"])
def test_sums_over_a_long_cache(BH, Sq, N, values):
    """Values all alike: the result is that value whatever the weights are.  Chains of sums are of at most 8192
    keys (or of a warp's share of a cache): 128 tiles of 12 products, each cut off by a step of fp32 at most, of
    a sum that grows evenly, so half of that, 9.2e-5; weights and parts 2^-16, joining chains 64 half steps."""
    rng = np.random.default_rng(81)
    one, _ = packed(rng.integers(-8, 8, (1, 1000, 128)), np.full((1, 1000, 4), 0.1))
    k = Packed4(*(t.repeat(1, (N + 999) // 1000, 1)[:, :N].expand(BH, -1, -1).contiguous() for t in one))
    codes = torch.from_numpy(codes_of(np.full((1, 1, 128), 7))).cuda()
    v = Packed4(codes.expand(BH, N, -1).contiguous(), torch.full((BH, N, 4), 1 + 2.0 ** -10, dtype=F16, device="cuda"))
    if values == "two":  # the first half of the keys' values are twice the others', and so are the weights' halves
        v.scales[:, :N // 2] *= 2
        k.scales[:] = 0
    q = torch.randn(BH, Sq, 128, generator=torch.Generator().manual_seed(82)).to(F16).cuda()
    got = anima_attn.attention_core_kv4(q, k, v, 1, BH, out_dtype=F32).double()
    want = 7 * (1 + 2.0 ** -10) * (1.5 if values == "two" else 1.0)
    assert ((got - want).abs().max() / want).item() <= 9.2e-5 + 2.0 ** -16 + 64 * 2.0 ** -24
    assert anima_attn.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,H,Sq,Skv,lens", [(1, 80, 40, 20000, None), (2, 40, 20, 20000, [20000, 8192]), (2, 40, 20, 20000, [8193, 64]),
                                             (2, 40, 130, 20000, [100, 20000]), (2, 40, 20, 20000, [16385, 0])])
def test_runs_of_a_long_cache(B, H, Sq, Skv, lens, dtype):
    """Chains of more than 8192 keys go on as runs: whole, cut by lengths at, before and behind a run's end, with
    maxima that rise and fall from run to run (keys twice as large in the middle)."""
    size = np.ones(Skv)
    size[7000:9000], size[18000:] = 2.0, 0.1
    rng = np.random.default_rng(83)
    k, kv = packed(rng.integers(-8, 8, (1, Skv, 128)), 0.2 * size[None, :, None] * rng.uniform(0.9, 1.1, (1, Skv, 4)))
    v, vv = random_packed((1, Skv, 128), 84)
    BH = B * H
    q = torch.randn(BH, Sq, 128, generator=torch.Generator().manual_seed(85)).to(dtype).cuda()
    vl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = anima_attn.attention_core_kv4(q, every_head(k, BH), every_head(v, BH), B, H, kv_valid_len=vl, out_dtype=F32)
    kd, vd = torch.from_numpy(kv[0]).cuda(), torch.from_numpy(vv[0]).cuda()
    for b in range(B):
        n = Skv if lens is None else lens[b]
        for h in range(0, H, 13):
            if n == 0:
                assert (got[b, :, h] == 0).all()
                continue
            s = q[b * H + h].double() @ kd[:n].T / math.sqrt(128)
            p = torch.softmax(s, -1)
            top = (q[b * H + h].double().abs() @ kd[:n].abs().T / math.sqrt(128)).amax(-1, keepdim=True)
            tol = (p @ vd[:n].abs()) * (2 * (512 * 2.0 ** -23 * top + 2.0 ** -16) + 9.2e-5)
            assert ((got[b, :, h].double() - p @ vd[:n]).abs() <= tol).all()
    assert anima_attn.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1000000, 70], [0, 600001], [8192 * 64 + 1, 1]])
def test_slices_of_several_runs_masked(lens):
    """Slices so long that each is several runs, lengths that leave runs and slices empty: values all alike."""
    B, Sq, N = 2, 70, 1000000
    one, _ = packed(np.random.default_rng(86).integers(-8, 8, (1, 1000, 128)), np.full((1, 1000, 4), 0.1))
    k = Packed4(*(t.repeat(1, N // 1000, 1).expand(B, -1, -1).contiguous() for t in one))
    codes = torch.from_numpy(codes_of(np.full((1, 1, 128), 7))).cuda()
    v = Packed4(codes.expand(B, N, -1).contiguous(), torch.ones(B, N, 4, dtype=F16, device="cuda"))
    for b, n in enumerate(lens):
        k.scales[b, n:] = v.scales[b, n:] = float("nan")
    q = torch.randn(B, Sq, 128, generator=torch.Generator().manual_seed(87)).to(F16).cuda()
    vl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = anima_attn.attention_core_kv4(q, k, v, B, 1, kv_valid_len=vl, out_dtype=F32).double()
    assert way(B, Sq, N) == "tile1"
    for b, n in enumerate(lens):  # bound as in test_sums_over_a_long_cache
        assert ((got[b] - (7 if n else 0)).abs().max() / 7).item() <= 9.2e-5 + 2.0 ** -16 + 64 * 2.0 ** -24
    assert anima_attn.status() == 0
