"""4-bit storage: packing, attention over packed K/V, matrix-vector products with packed weights.

Every operator is compared with a plain implementation in 64 bits written from the format's
definition (include/anima_attn.h).  Tolerances are bounds of rounding, derived where they are used.
"""
import ctypes as ct
import math

import numpy as np
import pytest
import torch

from conftest import ATTN_REL_L2, rel_l2

import anima_attn
from anima_attn import Packed4, _lib as L
from anima_attn import packed as P

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------ the format in 64 bits
def pack_ref(x):
    """[..., K] 16-bit tensor -> (codes [..., K/2] uint8, scales [..., K/32] fp16) numpy arrays."""
    x = x.double().cpu().numpy()
    lead, K = x.shape[:-1], x.shape[-1]
    g = x.reshape(lead + (K // 32, 32))
    with np.errstate(all="ignore"):
        hi, lo = g.max(-1), g.min(-1)
        s = (np.where(hi >= -lo, hi, lo) / -8).astype(np.float16)
        s = np.where((np.abs(g) <= 65504).all(-1), s, np.float16(np.nan))
        n = np.floor(g / s.astype(np.float64)[..., None] + 0.5)
    n = np.where((s == 0)[..., None] | np.isnan(s)[..., None], 0, n)
    c = (np.clip(n, -8, 7) + 8).astype(np.uint32).reshape(lead + (K // 128, 4, 4, 8))  # g, i, e
    words = np.zeros(lead + (K // 128, 16), np.uint32)
    for gi in range(4):
        for i in range(4):
            for e in range(8):
                words[..., 4 * i + gi] |= c[..., gi, i, e] << np.uint32(4 * ((e >> 1) + 4 * (e & 1)))
    return words.astype("<u4").view(np.uint8).reshape(lead + (K // 2,)), s


def unpack_ref(codes, scales):
    """Values [..., K] in 64 bits of packed arrays (torch or numpy)."""
    codes, scales = (t.cpu().numpy() if torch.is_tensor(t) else t for t in (codes, scales))
    lead, K = codes.shape[:-1], 2 * codes.shape[-1]
    words = np.ascontiguousarray(codes).view("<u4").reshape(lead + (K // 128, 16))
    n = np.empty(lead + (K // 128, 4, 4, 8))
    for gi in range(4):
        for i in range(4):
            for e in range(8):
                n[..., gi, i, e] = (words[..., 4 * i + gi] >> np.uint32(4 * ((e >> 1) + 4 * (e & 1))) & 15).astype(float) - 8
    return (n.reshape(lead + (K // 32, 32)) * scales.astype(np.float64)[..., None]).reshape(lead + (K,))


def random_packed(shape, seed, dtype=F16, std=1.0, device="cuda"):
    """A packed tensor made by the reference, and its values in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    codes, scales = pack_ref(torch.randn(shape, generator=g).mul_(std).to(dtype))
    return Packed4(torch.from_numpy(codes).to(device), torch.from_numpy(scales).to(device)), unpack_ref(codes, scales)


def test_reference_format_by_hand():
    """Word and nibble order and the scale's sign, on one block worked out by hand."""
    x = torch.zeros(128, dtype=F16)
    x[0], x[1], x[9], x[34] = 8.0, -1.0, 3.0, -16.0
    codes, scales = pack_ref(x)
    assert scales.tolist() == [-1.0, 2.0, 0.0, 0.0]
    w = codes.view("<u4")
    # value 0 -> n = -8 -> code 0 at nibble 0 of word 0; value 1 -> n = 1 -> code 9 at nibble 4
    assert w[0] & 0xF == 0 and (w[0] >> 16) & 0xF == 9
    assert (w[4] >> 16) & 0xF == 8 - 3          # value 9: i = 1, e = 1, n = 3 / -1
    assert (w[1] >> 4) & 0xF == 0               # value 34: g = 1, i = 0, e = 2, n = -16 / 2
    assert w[2] == 0x88888888                   # an empty group
    np.testing.assert_array_equal(unpack_ref(codes, scales), x.double().numpy())


# ------------------------------------------------------------------ refusals (no GPU needed)
A = 1 << 20  # an aligned address that no refused call reads


def _quant(**kw):
    a = dict(x=A, dtype=L.DTYPE_F16, n=(1, 1, 4), s=(0, 0, 128), K=128, codes=A, scales=A)
    a.update(kw)
    return L.lib.anima_quantize4(a["x"], a["dtype"], *a["n"], *a["s"], a["K"], a["codes"], a["scales"], None)


@pytest.mark.parametrize("kw,want", [
    (dict(dtype=L.DTYPE_F32), L.ERR_ARG), (dict(dtype=9), L.ERR_ARG), (dict(K=64), L.ERR_SHAPE),
    (dict(K=0), L.ERR_SHAPE), (dict(K=-128), L.ERR_SHAPE), (dict(n=(1, -1, 4)), L.ERR_SHAPE),
    (dict(n=(1 << 30, 1 << 30, 4)), L.ERR_SHAPE), (dict(x=None), L.ERR_ARG), (dict(codes=None), L.ERR_ARG),
    (dict(scales=None), L.ERR_ARG), (dict(x=A + 2), L.ERR_ARG), (dict(codes=A + 8), L.ERR_ARG),
    (dict(scales=A + 4), L.ERR_ARG), (dict(s=(0, 0, 132)), L.ERR_ARG), (dict(s=(0, -128, 128)), L.ERR_ARG),
    (dict(n=(0, 1, 4), x=None), L.OK)])
def test_quantize_refusals(kw, want):
    assert _quant(**kw) == want


@pytest.mark.parametrize("args,want", [
    ((A, A, A, 7, 4, 128), L.ERR_ARG), ((A, A, A, L.DTYPE_F32, -1, 128), L.ERR_SHAPE),
    ((A, A, A, L.DTYPE_F32, 4, 100), L.ERR_SHAPE), ((None, A, A, L.DTYPE_F16, 4, 128), L.ERR_ARG),
    ((A, A, A + 4, L.DTYPE_F32, 4, 128), L.ERR_ARG), ((A, A + 2, A, L.DTYPE_F32, 4, 128), L.ERR_ARG),
    ((None, None, None, L.DTYPE_F16, 0, 128), L.OK)])
def test_dequantize_refusals(args, want):
    assert L.lib.anima_dequantize4(*args, None) == want


def _mv(**kw):
    a = L.Matvec4Args(A, L.DTYPE_F32, (0, 256), A, A, None, (0, 0), A, L.DTYPE_F32, (0, 16), 1, 1, 16, 256, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return L.lib.anima_matvec4(ct.byref(a), None)


@pytest.mark.parametrize("kw,want", [
    (dict(x_dtype=5), L.ERR_ARG), (dict(out_dtype=-1), L.ERR_ARG), (dict(K=192), L.ERR_SHAPE),
    (dict(K=0), L.ERR_SHAPE), (dict(K=32768 + 128), L.ERR_SHAPE), (dict(M=-1), L.ERR_SHAPE),
    (dict(E=1 << 30, N=1 << 30), L.ERR_SHAPE), (dict(N=(1 << 31) - 5), L.ERR_SHAPE), (dict(x=None), L.ERR_ARG), (dict(out=None), L.ERR_ARG),
    (dict(codes=A + 4), L.ERR_ARG), (dict(scales=A + 2), L.ERR_ARG), (dict(add=A + 2), L.ERR_ARG),
    (dict(x=A + 2), L.ERR_ARG), (dict(N=0, x=None), L.OK), (dict(M=0), L.OK), (dict(E=0), L.OK)])
def test_matvec_refusals(kw, want):
    assert _mv(**kw) == want
    assert L.lib.anima_matvec4(None, None) == L.ERR_ARG


def _attn(**kw):
    a = L.AttnKv4Args(A, A, A, A, A, L.DTYPE_F16, A, (128, 128, 128), 1, 1, 1, 1, 128, 0.1, 0, None, None, 0)
    for k, v in kw.items():
        if k == "out_stride":
            a.out_stride[:] = v
        else:
            setattr(a, k, v)
    return L.lib.anima_attn_kv4_fwd(ct.byref(a), None)


@pytest.mark.parametrize("kw,want", [
    (dict(q=None), L.ERR_ARG), (dict(v_scales=None), L.ERR_ARG), (dict(out=None), L.ERR_ARG),
    (dict(dtype=L.DTYPE_F32), L.ERR_ARG), (dict(D=64), L.ERR_SHAPE), (dict(B=0), L.ERR_SHAPE),
    (dict(S_q=0), L.ERR_SHAPE), (dict(S_kv=0), L.ERR_SHAPE), (dict(flags=L.FLAG_MASK), L.ERR_ARG),
    (dict(scale=0.0), L.ERR_ARG), (dict(scale=-0.3), L.ERR_ARG), (dict(scale=math.inf), L.ERR_ARG),
    (dict(scale=math.nan), L.ERR_ARG), (dict(flags=L.FLAG_CAUSAL), L.ERR_ARG), (dict(out_stride=(128, 128, 4)), L.ERR_ARG),
    (dict(out_stride=(-128, 128, 128)), L.ERR_ARG), (dict(q=A + 8), L.ERR_ARG), (dict(out=A + 8), L.ERR_ARG),
    (dict(k_codes=A + 8), L.ERR_ARG), (dict(k_scales=A + 4), L.ERR_ARG), (dict(workspace=A + 64), L.ERR_ARG),
    (dict(B=1 << 20, H=1 << 20), L.ERR_SHAPE), (dict(S_q=(1 << 31) - 1), L.ERR_SHAPE),
    (dict(S_kv=(1 << 30) + 1), L.ERR_SHAPE)])
def test_attention_refusals(kw, want):
    assert _attn(**kw) == want
    assert L.lib.anima_attn_kv4_fwd(None, None) == L.ERR_ARG


@pytest.mark.parametrize("cls,cname", [(L.Matvec4Args, "AnimaMatvec4Args"), (L.AttnKv4Args, "AnimaAttnKv4Args")])
def test_struct_layouts(cls, cname, tmp_path):
    from test_abi import _c_layout
    c = _c_layout(cname, [f for f, _ in cls._fields_], tmp_path)
    assert c["size"] == ct.sizeof(cls)
    for f, _ in cls._fields_:
        assert c[f] == getattr(cls, f).offset, f


def test_packed_argument_layouts():
    """The bytes that the Python entries pass are the structures of the header."""
    m = P._MATVEC_ARGS.pack(1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18)
    a = L.Matvec4Args(1, 2, (3, 4), 5, 6, 7, (8, 9), 10, 11, (12, 13), 14, 15, 16, 17, 18)
    assert len(m) == ct.sizeof(a) and bytes(a) == m
    m = P._ATTN_ARGS.pack(1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 0.5, 16, 17, 18, 19)
    a = L.AttnKv4Args(1, 2, 3, 4, 5, 6, 7, (8, 9, 10), 11, 12, 13, 14, 15, 0.5, 16, 17, 18, 19)
    assert len(m) == ct.sizeof(a) and bytes(a) == m


@pytest.fixture
def any_device(monkeypatch):
    """Lets the argument checks of the Python entries run on CPU tensors; the library is not called."""
    monkeypatch.setattr(P, "_here", lambda *ts: 0)


def _pk(*shape):
    return Packed4(torch.zeros(shape[:-1] + (shape[-1] // 2,), dtype=torch.uint8),
                   torch.zeros(shape[:-1] + (shape[-1] // 32,), dtype=F16))


def test_python_refusals(any_device):
    bad = pytest.raises(ValueError)
    h = torch.zeros(4, 256, dtype=F16)
    for x in (h.float(), h[:, :100], h.t(), torch.zeros(2, 130, dtype=F16)[:, 1:129],
              torch.zeros(2, 132, dtype=F16)[:, :128], torch.zeros(4, 2, 4, 2, 4, 2, 4, 128, dtype=F16)[:, 0, :, 0, :, 0]):
        with bad:
            anima_attn.quantize4(x)
    with bad:
        anima_attn.quantize4(h, out=_pk(4, 128))
    with bad:
        anima_attn.dequantize4(_pk(4, 128), torch.float64)
    with bad:
        anima_attn.dequantize4(Packed4(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(3, 4, dtype=F16)))
    with bad:
        anima_attn.dequantize4(Packed4(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 4, dtype=F16)))
    with bad:
        anima_attn.dequantize4(Packed4(torch.zeros((), dtype=torch.uint8), torch.zeros((), dtype=F16)))
    with bad:
        anima_attn.dequantize4(Packed4(torch.zeros(64, dtype=torch.uint8), torch.zeros((), dtype=F16)))
    w, ws = _pk(32, 256), _pk(3, 32, 256)
    for x, p, kw in ((torch.zeros(2, 128), w, {}), (torch.zeros(2, 2, 256), w, {}), (torch.zeros(2, 256), ws, {}),
                     (torch.zeros(2, 2, 256), ws, {}), (torch.zeros(2, 256, dtype=torch.float64), w, {}),
                     (torch.zeros(256, 2).t(), w, {}), (torch.zeros(2, 256), w, {"out_dtype": torch.float64}),
                     (torch.zeros(2, 256), w, {"out": torch.zeros(2, 31)}),
                     (torch.zeros(2, 256), w, {"out": torch.zeros(32, 2).t()}),
                     (torch.zeros(2, 256), w, {"out": torch.zeros(32).expand(2, 32)}),
                     (torch.zeros(2, 256), w, {"add": torch.zeros(3, 32)}),
                     (torch.zeros(2, 256), w, {"add": torch.zeros(2, 1)}),
                     (torch.zeros(2, 256), w, {"add": torch.zeros(32, dtype=F16)})):
        with bad:
            anima_attn.matvec4(x, p, **kw)
    q, k = torch.zeros(4, 3, 128, dtype=F16), _pk(4, 5, 128)
    for a, kw in (((q.float(), k, k, 2, 2), {}), ((q, k, k, 1, 2), {}), ((q, _pk(4, 5, 256), k, 2, 2), {}),
                  ((q, k, _pk(4, 6, 128), 2, 2), {}), ((q, _pk(4, 0, 128), _pk(4, 0, 128), 2, 2), {}),
                  ((q.transpose(0, 1), k, k, 2, 2), {}), ((q, k, k, 2, 2), {"out_layout": "sbhd"}),
                  ((q, k, k, 2, 2), {"out": torch.zeros(2, 3, 2, 128)}),
                  ((q, k, k, 2, 2), {"out": torch.zeros(2, 1, 2, 128, dtype=F16).expand(2, 3, 2, 128)}),
                  ((q, k, k, 2, 2), {"kv_valid_len": torch.zeros(3)}),
                  ((q, k, k, 2, 2), {"scale": 0.0}), ((q, k, k, 2, 2), {"scale": -0.3}),
                  ((q, k, k, 2, 2), {"scale": math.nan})):
        with bad:
            anima_attn.attention_core_kv4(*a, **kw)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError):
        anima_attn.quantize4(torch.zeros(4, 128, dtype=F16))


@pytest.mark.parametrize("shape,stride,want", [
    ((4, 8, 128), (1024, 128, 1), [(1, 0), (1, 0), (32, 128)]),
    ((4, 8, 128), (2048, 128, 1), [(1, 0), (4, 2048), (8, 128)]),
    ((2, 1, 5, 3, 128), (9999, 7, 1024, 128, 1), [(2, 9999), (5, 1024), (3, 128)]),
    ((128,), (1,), [(1, 0), (1, 0), (1, 0)]),
    ((2, 3, 128), (0, 128, 1), [(1, 0), (2, 0), (3, 128)]),
    ((2, 2, 2, 2, 128), (8000, 2000, 700, 300, 1), None)])
def test_row_strides(shape, stride, want):
    x = torch.empty(20000, dtype=F16).as_strided(shape, stride)
    assert P._row_strides(x) == want


# ------------------------------------------------------------------ packing on the GPU
def check_pack(x):
    codes, scales = pack_ref(x)
    got = anima_attn.quantize4(x.cuda() if not x.is_cuda else x)
    np.testing.assert_array_equal(got.scales.cpu().numpy(), scales)
    np.testing.assert_array_equal(got.codes.cpu().numpy(), codes)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 128), (3, 128), (7, 1, 384), (1, 32768), (33, 2, 5, 256), (128,)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_quantize_and_back(shape, dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(shape, generator=g).to(dtype)
    got = check_pack(x)
    want = unpack_ref(*got)
    for dt in (F32, F16, BF16):
        y = anima_attn.dequantize4(got, dt)
        ref = torch.from_numpy(want).float().to(dt)  # n * s has at most 15 bits: exact in fp32
        assert torch.equal(y.cpu(), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_quantize_any_bits(dtype):
    """Random bit patterns: subnormals, infinities, NaN, magnitudes past fp16, all mixed, and
    groups whose members have similar exponents, where the quotients come near the borders."""
    rng = np.random.default_rng(2)
    wild = rng.integers(-32768, 32768, (512, 128), dtype=np.int16)
    near = (rng.integers(0, 0x7C00 if dtype == F16 else 0x4780, (4096, 4, 1)) + rng.integers(-600, 600, (4096, 4, 32)))
    near = np.clip(near, 0, 0x7BFF if dtype == F16 else 0x477F).astype(np.int16).reshape(4096, 128)
    near |= (rng.integers(0, 2, near.shape) << 15).astype(np.uint16).view(np.int16)
    for bits in (wild, near):
        check_pack(torch.from_numpy(bits.copy()).view(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_quantize_ties_and_edges(dtype):
    x = torch.zeros(12, 128, dtype=dtype)
    x[0, :32] = torch.arange(32) / 4 - 4          # exact halves of the scale
    x[1, :32], x[1, 0] = 3.0, -3.0                # both signs reach the largest magnitude
    x[2, 5], x[2, 40] = float("inf"), float("nan")
    x[3, 64:96] = 65504.0                         # bf16 rounds this up past fp16: NaN scale
    x[4] = 2.0 ** -24
    x[5, 0], x[5, 1] = 2.0 ** -21, 2.0 ** -24     # a subnormal scale
    x[6, 7] = -0.0
    x[7, 0], x[7, 1] = 2.0 ** -22, -2.0 ** -24    # the scale rounds to zero or to 2^-24
    x[8] = torch.linspace(-1, 1, 128)
    check_pack(x)


@pytest.mark.gpu
def test_quantize_strided_views():
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(2, 9, 3, 4, 128, generator=g).to(F16).cuda()
    check_pack(qkv[:, :, 1])                       # [B, S, H, D] slice of a fused projection
    check_pack(qkv[:, 2:7, 2].transpose(1, 2))     # head-major view
    check_pack(qkv[0, 0, 0, 0].expand(5, 128))     # a repeated row
    big = torch.randn(6, 520, generator=g).to(BF16).cuda()
    check_pack(big[::2, 8:264])
    out = Packed4(torch.empty(5, 64, dtype=torch.uint8, device="cuda"), torch.empty(5, 4, dtype=F16, device="cuda"))
    assert anima_attn.quantize4(qkv[0, :5, 0, 0], out=out) is out
    np.testing.assert_array_equal(out.codes.cpu().numpy(), pack_ref(qkv[0, :5, 0, 0])[0])
    empty = anima_attn.quantize4(qkv[:0, :, 0])
    assert empty.shape == (0, 9, 4, 128) and anima_attn.dequantize4(empty).shape == (0, 9, 4, 128)


# ------------------------------------------------------------------ matrix-vector products
def matvec_bound(ax, aw, K, y, out_dtype, silu):
    """Rounding bound of one result, with S = sum |x| |w|.  Products are exact.  A group's 32 are
    summed by the tensor core (one truncation, a step of fp32, per product and addition: 64), then
    K/32 scaled sums, at most 8 warps and 4 digits, the addend and the scale's product are
    rounded: K/32 + 16 half steps, taken as steps.  fp32 rows enter as whole numbers of 2^(E - 30) per
    group of 32, 2^E at most twice the group's largest magnitude: half of that per value.  SiLU
    adds 8 steps on x (expf 2, sum, quotient, and the argument's)."""
    step = 2.0 ** -23
    S = ax @ np.swapaxes(aw, -1, -2)
    top = np.repeat(ax.reshape(ax.shape[:-1] + (K // 32, 32)).max(-1), 32, -1)
    T = top @ np.swapaxes(aw, -1, -2)
    return 1.01 * S * step * (64 + K / 32 + 16 + (8 if silu else 0)) + T * 2.0 ** -30 + np.abs(y) * half_step(out_dtype) + 1e-37 + \
        (6e-8 if out_dtype == F16 else 0.0)  # fp16 subnormals


def check_matvec(E, M, N, K, xdt=F32, odt=F32, silu=False, add=False, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    w, wv = random_packed((E, N, K), seed + 1, std=0.05)
    x = (torch.randn(E, M, K, generator=g) * std).to(xdt).cuda()
    ad = torch.randn(M, N, generator=g).cuda() if add else None
    got = anima_attn.matvec4(x, w, silu=silu, add=ad, out_dtype=odt)
    assert got.shape == (E, M, N) and got.dtype == odt
    xv = x.double().cpu().numpy()
    if silu:
        xv = xv / (1 + np.exp(-xv))
    y = xv @ np.swapaxes(wv, -1, -2)
    ax = np.abs(xv)
    if add:
        y = y + ad.double().cpu().numpy()
    tol = matvec_bound(ax, np.abs(wv), K, y, odt, silu)
    if add:
        tol = tol + np.abs(ad.double().cpu().numpy()) * 2.0 ** -23
    err = np.abs(got.double().cpu().numpy() - y)
    assert (err <= tol).all(), (float((err / tol).max()), np.argwhere(err > tol)[:3])


@pytest.mark.gpu
@pytest.mark.parametrize("E,M,N,K", [(1, 1, 1, 128), (1, 1, 16, 128), (1, 2, 17, 256), (3, 2, 15, 128), (1, 1, 129, 2048),
                                     (2, 5, 100, 640), (84, 2, 96, 256), (1, 8, 33, 1152), (5, 1, 1003, 384)])
@pytest.mark.parametrize("xdt", [F32, F16, BF16])
def test_matvec(E, M, N, K, xdt):
    check_matvec(E, M, N, K, xdt)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 3, 5, 6, 8, 9, 16, 17, 33])
@pytest.mark.parametrize("xdt,silu", [(F32, False), (BF16, False), (F16, True)])
def test_matvec_rows(M, xdt, silu):
    """Every split of rows into blocks of columns, and into several passes."""
    check_matvec(1, M, 40, 512, xdt, silu=silu, seed=M)


@pytest.mark.gpu
@pytest.mark.parametrize("odt", [F32, F16, BF16])
@pytest.mark.parametrize("silu,add", [(True, False), (False, True), (True, True)])
def test_matvec_epilogue(odt, silu, add):
    check_matvec(4, 2, 200, 256, F32, odt, silu, add)
    check_matvec(1, 3, 50, 1024, BF16, odt, silu, add)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,xdt", [(1, 32768, F32), (8, 16384, F32), (16, 32768, BF16), (2, 8192, F16)])
def test_matvec_long_rows(M, K, xdt):
    check_matvec(1, M, 24, K, xdt)


@pytest.mark.gpu
def test_matvec_many_rows_of_w():
    check_matvec(1, 1, 70001, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("std", [1e-38, 1e-30, 1e30, 2e36])
def test_matvec_keeps_the_range_of_fp32(std):
    check_matvec(1, 2, 64, 256, F32, std=std)


@pytest.mark.gpu
def test_matvec_magnitudes_far_apart():
    """Groups of 1e-20, 1 and 1e20 side by side, and within a group values 2^20 apart."""
    w, wv = random_packed((40, 384), 8)
    x = torch.randn(3, 384, generator=torch.Generator().manual_seed(9))
    x[:, :128] *= 1e-20
    x[0, 256:] *= 1e20
    x[1, 128:] = 0
    x[2, ::3] *= 2.0 ** -20
    x[2, 5] = -2.0 ** -149
    y = anima_attn.matvec4(x.cuda(), w).double().cpu().numpy()
    xv = x.double().numpy()
    want = xv @ wv.T
    assert (np.abs(y - want) <= matvec_bound(np.abs(xv), np.abs(wv), 384, want, F32, False)).all()


@pytest.mark.gpu
def test_matvec_views_and_shapes():
    """Strided rows, an output view, an addend of one row and a vector x."""
    g = torch.Generator().manual_seed(5)
    w, wv = random_packed((3, 48, 256), 6, std=0.05)
    h = torch.randn(2, 3 * 256, generator=g).cuda()
    x = h.view(2, 3, 256).transpose(0, 1)               # [E, M, K] with rows 768 apart
    buf = torch.full((3, 2, 64), 7.0, device="cuda")
    add = torch.randn(48, generator=g).cuda()
    got = anima_attn.matvec4(x, w, out=buf[:, :, 8:56], add=add)
    y = x.double().cpu().numpy() @ np.swapaxes(wv, 1, 2) + add.double().cpu().numpy()
    tol = matvec_bound(np.abs(x.double().cpu().numpy()), np.abs(wv), 256, y, F32, False) + 1e-6
    assert got.data_ptr() == buf[:, :, 8:56].data_ptr() and (np.abs(got.double().cpu().numpy() - y) <= tol).all()
    assert (buf[:, :, :8] == 7).all() and (buf[:, :, 56:] == 7).all()
    one = Packed4(w.codes[1].contiguous(), w.scales[1].contiguous())
    v = anima_attn.matvec4(x[1, 0], one)
    assert v.shape == (48,)
    assert torch.equal(v, anima_attn.matvec4(x[1, :1], one)[0])
    assert torch.equal(anima_attn.matvec4(x[1], one)[0], v)  # a row's result does not depend on the others
    assert anima_attn.matvec4(x[1, :0], one).shape == (0, 48)


@pytest.mark.gpu
@pytest.mark.parametrize("xdt", [F16, BF16, F32])
def test_matvec_unaligned_rows(xdt):
    """Rows of x that start on any element, and a row repeated by a zero stride."""
    g = torch.Generator().manual_seed(10)
    w, wv = random_packed((50, 256), 11)
    buf = torch.randn(3, 259, generator=g).to(xdt).cuda()
    for x in (buf[:, 1:257], buf[:, 3:], buf[1:2, 1:257].expand(4, 256)):
        y = anima_attn.matvec4(x, w).double().cpu().numpy()
        xv = x.double().cpu().numpy()
        want = xv @ wv.T
        assert (np.abs(y - want) <= matvec_bound(np.abs(xv), np.abs(wv), 256, want, F32, False)).all()


@pytest.mark.gpu
def test_matvec_not_finite():
    """A NaN scale reaches its row of W only, a NaN or infinite x its row of x only."""
    w, wv = random_packed((32, 256), 7)
    w.scales[3, 2] = float("nan")
    x = torch.ones(3, 256, device="cuda")
    x[1, 5] = float("nan")
    y = anima_attn.matvec4(x, w).cpu()
    assert y[1].isnan().all() and y[0, 3].isnan() and y[2, 3].isnan()
    keep = [n for n in range(32) if n != 3]
    assert y[0, keep].isfinite().all() and torch.equal(y[0, keep], y[2, keep])
    x = torch.zeros(1, 256, device="cuda")
    x[0, 9] = float("inf")
    y, want = anima_attn.matvec4(x, w).cpu()[0], np.sign(wv[:, 9])
    for n in keep:
        assert y[n].isnan() if want[n] == 0 else y[n] == want[n] * float("inf")


# ------------------------------------------------------------------ attention
def attention_ref(q, kv, vv, B, H, lens, scale):
    """[B*H, S, 128] in 64 bits -> out [B, S_q, H, 128], and the pieces of its rounding bound:
    sum p |v| and the largest sum |q| |k| scale of a row's valid keys."""
    BH, Sq, D = q.shape
    out, pv, top = np.zeros((BH, Sq, D)), np.zeros((BH, Sq, D)), np.zeros((BH, Sq, 1))
    for bh in range(BH):
        n = kv.shape[1] if lens is None else max(0, min(int(lens[bh // H]), kv.shape[1]))
        if n == 0:
            continue
        s = q[bh] @ kv[bh, :n].T * scale
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[bh], pv[bh] = p @ vv[bh, :n], p @ np.abs(vv[bh, :n])
        top[bh] = (np.abs(q[bh]) @ np.abs(kv[bh, :n]).T * abs(scale)).max(-1, keepdims=True)
    def layout(t):
        return t.reshape(B, H, Sq, -1).transpose(0, 2, 1, 3)
    return layout(out), layout(pv), layout(top)


def few_rows(Sq):
    return Sq <= 16  # read the packed cache directly (csrc/attn_kv4.cu)


def attention_bound(out, pv, top, dtype, direct):
    """Rounding bound.  Directly from the packed cache: a score is off by at most 80 fp32 steps of
    sum |q k| scale (32 exact products a group, 4 scaled sums, the scale), plus 2^-20 for the
    exponential; p s in two bf16 parts by 2^-17; sums and merges by 2^-17 (hundreds of fp32
    half steps).  Numerator and denominator: twice.  Through the core, k, v and p are each rounded
    once to the type (half steps u): u top for the score, u for v, u for p, again doubled for
    the denominator's share, and the core's lazily settled exponentials 2^-12.
    The result is rounded once more."""
    u = half_step(dtype)
    if direct:
        c = 2 * (80 * 2.0 ** -23 * top + 2.0 ** -20 + 2.0 ** -17 + 2.0 ** -17)
    else:
        c = 2 * (u * top + 2.0 ** -12) + 2 * u
    return np.abs(out) * u + pv * c * (1 + c) + (6e-8 if dtype == F16 else 1e-37)


def check_attention(B, H, Sq, Skv, dtype, lens=None, layout="bshd", scale=None, seed=0, poison=True, std=1.0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(B * H, Sq, 128, generator=g) * std).to(dtype).cuda()
    k, kv = random_packed((B * H, Skv, 128), seed + 1)
    v, vv = random_packed((B * H, Skv, 128), seed + 2)
    vl = None
    if lens is not None:
        vl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        if poison:  # what lies behind a sample's length is never part of its result
            for b, n in enumerate(lens):
                for t in (k, v):
                    t.scales.view(B, H, Skv, 4)[b, :, max(n, 0):] = float("nan")
                    t.codes.view(B, H, Skv, 64)[b, :, max(n, 0):] = 0xF1
    got = anima_attn.attention_core_kv4(q, k, v, B, H, scale=scale, kv_valid_len=vl, out_layout=layout)
    assert got.dtype == dtype and anima_attn.status() == 0
    if layout == "bhsd":
        got = got.transpose(1, 2)
    sc = 1 / math.sqrt(128) if scale is None else scale
    out, pv, top = attention_ref(q.double().cpu().numpy(), kv, vv, B, H, lens, sc)
    err = np.abs(got.double().cpu().numpy() - out)
    tol = attention_bound(out, pv, top, dtype, few_rows(Sq))
    assert (err <= tol).all(), (float((err / tol).max()), np.argwhere(~(err <= tol))[:3])
    if np.abs(out).max() > 0:
        assert rel_l2(got.float().cpu().numpy(), out) <= ATTN_REL_L2
    if lens is not None:
        for b, n in enumerate(lens):
            if n <= 0:
                assert (got[b] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 2, 7, 8, 9, 16, 17, 31, 64, 65, 130, 300])
@pytest.mark.parametrize("Skv", [1, 15, 33, 128, 515])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention(Sq, Skv, dtype):
    check_attention(2, 3, Sq, Skv, dtype, seed=Sq + Skv)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 13, 40, 260])
@pytest.mark.parametrize("lens", [[0, 0, 0], [0, 1, 77], [77, 64, 32], [31, 33, 500], [-3, 16, 17]])
def test_attention_masked(Sq, lens):
    check_attention(3, 2, Sq, 77, F16, lens=lens)
    check_attention(3, 2, Sq, 300, BF16, lens=lens, layout="bhsd")


@pytest.mark.gpu
@pytest.mark.parametrize("Sq,Skv,B,H", [(1, 4096, 2, 16), (1, 20011, 1, 1), (5, 9000, 1, 3), (12, 5003, 2, 2),
                                        (200, 5000, 1, 2), (300, 5000, 1, 3), (1, 100, 8, 32)])
def test_attention_long_and_wide(Sq, Skv, B, H):
    check_attention(B, H, Sq, Skv, F16)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq,Skv,B,H,lens", [(1, 4103, 1, 37, None), (1, 4103, 2, 20, [4103, 130]), (1, 16411, 1, 20, None),
                                             (8, 8205, 1, 21, None), (1, 33001, 2, 6, [0, 33001]), (3, 4097, 1, 160, None),
                                             (1, 4100, 3, 40, [31, 0, 4100])])
def test_attention_clusters_and_slices(Sq, Skv, B, H, lens):
    """Unit counts that ask for clusters of every size, several rounds and slices of single CTAs."""
    check_attention(B, H, Sq, Skv, BF16 if H % 2 else F16, lens=lens)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq,Skv,lens", [(1, 20011, [5, 0]), (3, 20011, [20011, 700]), (200, 5000, [0, 130]),
                                         (200, 5000, [5000, 1]), (100, 5000, [4999, 257]), (300, 5000, [0, 130]),
                                         (300, 5000, [5000, 1]), (230, 5000, [4999, 257])])
def test_attention_masked_slices(Sq, Skv, lens):
    """Keys cut into slices, of which masks leave some without a key."""
    check_attention(2, 1, Sq, Skv, F16, lens=lens)
    check_attention(2, 1, Sq, Skv, BF16, lens=lens)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,H,Sq,Skv,lens", [(2, 16, 2307, 133, None), (3, 13, 2049, 130, [0, 130, 40]), (5, 40, 100, 300, [300, 0, 1, 0, 128]),
                                             (4, 2, 2186, 6, [6, 4, 2, 0]), (2, 4, 3812, 2, None)])
def test_attention_many_units(dtype, B, H, Sq, Skv, lens):
    """More units than SMs: the persistent grid of the tile kernel, and the unpacked core for fp16."""
    check_attention(B, H, Sq, Skv, dtype, lens=lens)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [64, 300])
def test_attention_rows_of_any_size(Sq):
    """bf16 query rows whose magnitudes differ by far, a zero row, and a row past fp16's range."""
    g = torch.Generator().manual_seed(12)
    q = torch.randn(2, Sq, 128, generator=g)
    q[0, 1] *= 1e-30
    q[0, 2] *= 1e6
    q[0, 3] = 0
    q[1, 5, 7] = 1e8
    q[1, 6, :64] *= 1e-6
    q = q.to(BF16).cuda()
    k, kv = random_packed((2, 4200, 128), 1)  # beyond the direct form's work for both Sq
    v, vv = random_packed((2, 4200, 128), 2)
    got = anima_attn.attention_core_kv4(q, k, v, 1, 2)
    out, pv, top = attention_ref(q.double().cpu().numpy(), kv, vv, 1, 2, None, 1 / math.sqrt(128))
    tol = attention_bound(out, pv, top, F16, False) + np.abs(out) * half_step(BF16)
    # Where a row's scores are so large that their own bound passes 1, the largest keys may trade
    # places: those rows are only checked to be an average of values.
    far = (half_step(F16) * top > 1).squeeze(-1)
    err = np.abs(got.double().cpu().numpy() - out)
    assert (err[~far] <= tol[~far]).all(), float((err / tol)[~far].max())
    assert np.abs(got.float().cpu().numpy()[far]).max() <= np.abs(vv).max() * 1.01 and far.sum() == 2


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 100])
def test_attention_sharp_and_flat(Sq):
    """Scores spread over hundreds (one key takes all) and nearly alike."""
    check_attention(1, 2, Sq, 200, F16, scale=2.0)
    check_attention(1, 2, Sq, 200, F16, scale=1e-6)
    check_attention(1, 2, Sq, 200, BF16, scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [3, 100, 1100])
def test_attention_output_views(Sq):
    """An output view is filled and nothing around it is touched."""
    g = torch.Generator().manual_seed(9)
    B, H, Skv = 2, 2, 50
    q = torch.randn(B * H, Sq, 128, generator=g).to(F16).cuda()
    k, _ = random_packed((B * H, Skv, 128), 1)
    v, _ = random_packed((B * H, Skv, 128), 2)
    want = anima_attn.attention_core_kv4(q, k, v, B, H)
    buf = torch.full((B, Sq + 2, H + 1, 128), 5.0, dtype=F16, device="cuda")
    view = buf[:, 1:Sq + 1, :H]
    assert anima_attn.attention_core_kv4(q, k, v, B, H, out=view).data_ptr() == view.data_ptr()
    assert torch.equal(view, want)
    view.fill_(5.0)
    assert (buf == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 12, 300])
def test_attention_repeats_bit_for_bit(Sq):
    g = torch.Generator().manual_seed(10)
    q = torch.randn(4, Sq, 128, generator=g).to(F16).cuda()
    k, _ = random_packed((4, 3000, 128), 1)
    v, _ = random_packed((4, 3000, 128), 2)
    first = anima_attn.attention_core_kv4(q, k, v, 2, 2)
    for _ in range(3):
        assert torch.equal(anima_attn.attention_core_kv4(q, k, v, 2, 2), first)


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Sq,Skv,dtype", [(1, 2, 1, 60, F16), (1, 2, 5, 60, BF16), (1, 1, 1, 20011, BF16), (1, 1, 4, 20011, F16),
                                              (1, 2, 40, 5000, F16), (1, 2, 200, 5000, BF16), (1, 2, 300, 5000, F16),
                                              (1, 4, 2000, 200, BF16),
                                              (2, 16, 2400, 130, F16)])
def test_attention_nan_reaches_its_rows_only(B, H, Sq, Skv, dtype):
    """A NaN query value reaches its row; a NaN scale of a key or a value reaches its head (a value's: its
    group's dims); nothing else changes.  Direct, in slices, by tiles and through the core."""
    g = torch.Generator().manual_seed(13)
    q = torch.randn(B * H, Sq, 128, generator=g).to(dtype).cuda()
    k, v = (Packed4(*(t.expand(B * H, -1, -1).contiguous() for t in random_packed((1, Skv, 128), s)[0])) for s in (1, 2))
    clean = anima_attn.attention_core_kv4(q, k, v, B, H)
    assert clean.isfinite().all()
    last = B * H - 1
    q2 = q.clone()
    q2[last, Sq - 1, 77] = float("nan")
    got = anima_attn.attention_core_kv4(q2, k, v, B, H)
    assert got[-1, -1, -1].isnan().all()
    got[-1, -1, -1] = clean[-1, -1, -1]
    assert torch.equal(got, clean)
    for which in (0, 1):
        bad = Packed4((k, v)[which].codes, (k, v)[which].scales.clone())
        bad.scales[last, Skv // 2, 1] = float("nan")
        got = anima_attn.attention_core_kv4(q, bad if which == 0 else k, bad if which == 1 else v, B, H)
        hit = got[-1, :, -1] if which == 0 else got[-1, :, -1, 32:64]
        assert hit.isnan().all()
        (got[-1, :, -1] if which == 0 else got[-1, :, -1, 32:64]).copy_(clean[-1, :, -1] if which == 0 else clean[-1, :, -1, 32:64])
        assert torch.equal(got, clean)


# ------------------------------------------------------------------ offsets past 32 bits
@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 3, 20])
def test_attention_offsets_past_32_bits(Sq):
    H, Skv = 72, 480000  # 2.2 GB of codes each for K and V
    g = torch.Generator(device="cuda").manual_seed(14)

    def cache():
        return Packed4(torch.randint(0, 256, (H, Skv, 64), dtype=torch.uint8, device="cuda", generator=g),
                       (torch.rand(H, Skv, 4, device="cuda", generator=g) * 0.2 + 0.1).half())
    k, v = cache(), cache()
    q = torch.randn(H, Sq, 128, device="cuda", generator=g).half()
    got = anima_attn.attention_core_kv4(q, k, v, 1, H)
    for h in (0, H - 1):
        kv, vv = (anima_attn.dequantize4(Packed4(t.codes[h:h + 1], t.scales[h:h + 1]), F32)[0].double() for t in (k, v))
        p = torch.softmax(q[h].double() @ kv.T / math.sqrt(128), -1)
        err, size = (got[0, :, h].double() - p @ vv).abs(), p @ vv.abs()
        assert (err <= 2.0 ** -11 * (p @ vv).abs() + 2.0 ** -9 * size + 6e-8).all()  # far inside a misread


@pytest.mark.gpu
def test_matvec_and_packing_offsets_past_32_bits():
    E, N, K = 3, 100000, 16384  # 2.4 GB of codes
    g = torch.Generator(device="cuda").manual_seed(15)
    w = Packed4(torch.randint(0, 256, (E, N, K // 2), dtype=torch.uint8, device="cuda", generator=g),
                (torch.rand(E, N, K // 32, device="cuda", generator=g) * 0.01).half())
    x = torch.randn(E, 1, K, device="cuda", generator=g)
    y = anima_attn.matvec4(x, w)
    for e, n in ((0, 0), (E - 1, N - 40)):
        wv = anima_attn.dequantize4(Packed4(w.codes[e, n:n + 40], w.scales[e, n:n + 40]), F32).double()
        want = (wv @ x[e, 0].double()).cpu().numpy()
        tol = matvec_bound(x[e].abs().double().cpu().numpy(), wv.abs().cpu().numpy(), K, want, F32, False)[0]
        assert (np.abs(y[e, 0, n:n + 40].double().cpu().numpy() - want) <= tol).all()
    del w, y
    rows = (1 << 31) // 128 + 37  # more than 2^31 values
    big = torch.empty(rows, 128, dtype=F16, device="cuda")
    big[:] = torch.randn(1, 128, device="cuda", generator=g).half()
    tail = torch.randn(64, 128, device="cuda", generator=g).half()
    big[-64:] = tail
    p = anima_attn.quantize4(big)
    want = anima_attn.quantize4(tail)
    assert torch.equal(p.codes[-64:], want.codes) and torch.equal(p.scales[-64:], want.scales)
    back = anima_attn.dequantize4(p)
    assert torch.equal(back[-64:], anima_attn.dequantize4(want)) and torch.equal(back[:1], back[rows // 2:rows // 2 + 1])


# ------------------------------------------------------------------ as they are used
@pytest.mark.gpu
@pytest.mark.parametrize("H,Sq,Skv", [(2, 1, 20011), (20, 1, 16411), (3, 300, 5000), (40, 2100, 130)])
def test_graphs_with_scratch(H, Sq, Skv):
    """Calls that need scratch (slices, unpacked K and V) in two graphs whose replays overlap."""
    g = torch.Generator().manual_seed(12)
    k, v = (Packed4(*(t.expand(H, -1, -1).contiguous() for t in random_packed((1, Skv, 128), s)[0])) for s in (1, 2))
    qs = [torch.randn(H, Sq, 128, generator=g).to(F16).cuda() for _ in range(2)]
    want = [anima_attn.attention_core_kv4(q, k, v, 1, H) for q in qs]
    graphs, outs, side = [], [], torch.cuda.Stream()
    for q in qs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            outs.append([anima_attn.attention_core_kv4(q, k, v, 1, H) for _ in range(2)])
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[n]) for n in range(2) for o in outs[n])
    assert anima_attn.status() == 0


@pytest.mark.gpu
def test_streams_and_graphs():
    """The operators on a side stream, and two graphs captured on one stream whose replays overlap
    on two: scratch belongs to a call, not to a stream."""
    g = torch.Generator().manual_seed(11)
    k, _ = random_packed((4, 700, 128), 1)
    v, _ = random_packed((4, 700, 128), 2)
    w, _ = random_packed((96, 512), 3)
    qs = [torch.randn(4, 300, 128, generator=g).to(F16).cuda() for _ in range(2)]
    xs = [torch.randn(2, 512, generator=g).cuda() for _ in range(2)]

    def work(n):
        packed = anima_attn.quantize4(qs[n])
        return (anima_attn.attention_core_kv4(qs[n], k, v, 2, 2), anima_attn.attention_core_kv4(qs[n][:, :4].contiguous(), k, v, 2, 2),
                anima_attn.matvec4(xs[n], w, silu=True), anima_attn.dequantize4(packed))

    want = [work(n) for n in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work(0)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs, outs = [], []
    for n in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            outs.append(work(n))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for n in range(2):
        assert all(torch.equal(a, b) for a, b in zip(outs[n], want[n]))
    assert anima_attn.status() == 0
