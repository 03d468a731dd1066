"""4-bit storage on the device: packing, attention over packed K/V, and matrix-vector
products with packed weights (include/anima_attn.h, "4-bit storage").

For what a sampling server keeps resident per prompt or per model and reads with few rows or
once a step: the cross-attention K/V of text contexts (AnimaDiT.context_cache(kv_bits=4))
and the adaLN modulation weights (AnimaDiT(adaln_bits=4)).  A packed value takes 4.5 bits:
groups of 32 along the last axis share an fp16 scale s = x* / -8, x* the group's value of
largest magnitude, and a code n = floor(x / s + 1/2) in [-8, 7] stands for n * s.

Like the rest of the package: CUDA tensors on the current device, calls enqueued on the
current torch stream, no fallback.
"""
from __future__ import annotations

import math
import struct
from functools import lru_cache
from typing import NamedTuple, Optional

import torch

from . import _lib as L
from .ops import _TORCH_DT

_HALF = (torch.float16, torch.bfloat16)

# The smallest of these calls run for a few microseconds on the GPU, so the host side is kept
# short: the argument structures of the C entries are packed in one step (native alignment,
# the layouts of _lib's Structures), and the stream is asked for as a raw handle.
_MATVEC_ARGS = struct.Struct("@Pi2qPPP2qPi2qiiiii0q")
_ATTN_ARGS = struct.Struct("@PPPPPiP3qiiiiifIPPQ")
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current = getattr(torch._C, "_cuda_getDevice", None)
_U8, _F16, _F32 = torch.uint8, torch.float16, torch.float32
_quantize, _dequantize = L.lib.anima_quantize4, L.lib.anima_dequantize4
_matvec, _attn = L.lib.anima_matvec4, L.lib.anima_attn_kv4_fwd
_SCALE = 1.0 / math.sqrt(128)


class Packed4(NamedTuple):
    """A packed tensor [..., K]: ``codes`` uint8 [..., K/2] and ``scales`` float16
    [..., K/32], both contiguous (word and nibble order in anima_attn.h)."""
    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape[:-1] + (2 * self.codes.shape[-1],)

    def copy_(self, src: "Packed4") -> "Packed4":
        self.codes.copy_(src.codes)
        self.scales.copy_(src.scales)
        return self


def _here(t, *ts) -> int:
    """The current stream of the current device, on which every tensor must be."""
    dev = t.get_device()  # -1 on the CPU
    if dev < 0 or dev != _current():
        raise ValueError("anima_attn ops take CUDA tensors on the current device")
    for u in ts:
        if u is not None and u.get_device() != dev:
            raise ValueError("anima_attn ops take CUDA tensors on the current device")
    return _raw_stream(dev)


def _check_packed(c: torch.Tensor, s: torch.Tensor, what: str) -> tuple:
    """The codes' shape [..., K/2], after checking that codes and scales belong together."""
    if c.dtype is not _U8 or s.dtype is not _F16 or not c.is_contiguous() or not s.is_contiguous():
        raise ValueError(f"{what}: packed codes are contiguous uint8, scales contiguous float16")
    cs, ss = tuple(c.shape), tuple(s.shape)
    half = cs[-1] if cs and ss else 0
    if half == 0 or half % 64 or ss[-1] * 16 != half or cs[:-1] != ss[:-1]:
        raise ValueError(f"{what}: codes [..., K/2] and scales [..., K/32], K a multiple of 128")
    return cs


@lru_cache(maxsize=1024)
def _kv4_workspace(dev: int, dtype: torch.dtype, B: int, H: int, Sq: int, Skv: int) -> int:
    return int(L.lib.anima_attn_kv4_workspace_size(_TORCH_DT[dtype], B, H, Sq, Skv))


def _lengths32(t: torch.Tensor, most: int) -> torch.Tensor:
    """Lengths of another type as int32: what int32 does not hold is cut to [0, most] first."""
    if t.is_floating_point():
        t = t.double()
    return t.clamp(0, most).to(torch.int32) if t.element_size() == 8 else t.to(torch.int32)


def _repeats(t: torch.Tensor) -> bool:
    """Whether an axis of a tensor to be written repeats the same memory (an expanded view)."""
    return 0 in t.stride() and any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride()))


def _row_strides(x: torch.Tensor) -> Optional[list]:
    """The leading axes of x as three (size, stride) pairs, outermost first, adjacent axes
    joined where they step as one; None if more than three remain."""
    axes = []
    for n, st in zip(x.shape[:-1], x.stride()[:-1]):
        if n == 1:
            continue
        if axes and axes[-1][1] == n * st:
            axes[-1] = (axes[-1][0] * n, st)
        else:
            axes.append((n, st))
    return [(1, 0)] * (3 - len(axes)) + axes if len(axes) <= 3 else None


def quantize4(x: torch.Tensor, out: Optional[Packed4] = None) -> Packed4:
    """Packs x [..., K] (float16 or bfloat16, K a multiple of 128) to 4 bits along its last axis.

    The last axis is contiguous; the others may have any strides that are multiples of 8
    elements and amount to at most three axes (a [B, S, H, 128] projection or a slice of
    one).  ``out`` is filled if given.  A group of 32 with a NaN or a magnitude above 65504 reads
    back as NaN."""
    stream = _here(x)
    if x.dtype not in _HALF:
        raise ValueError("x must be float16 or bfloat16")
    shape = tuple(x.shape)
    K = shape[-1] if shape else 0
    if K == 0 or K % 128:
        raise ValueError("the last axis must be a positive multiple of 128")
    lead = shape[:-1]
    if out is None:
        codes, scales = x.new_empty(lead + (K // 2,), dtype=_U8), x.new_empty(lead + (K // 32,), dtype=_F16)
        out = Packed4(codes, scales)
    else:
        codes, scales = out
        _here(x, codes, scales)
        if _check_packed(codes, scales, "out") != lead + (K // 2,):
            raise ValueError("out must be packed with x's shape")
    n = x.numel()
    if n == 0:
        return out
    n0 = n1 = 1
    s0 = s1 = 0
    if x.is_contiguous():
        n2, s2 = n // K, K
    else:
        axes = _row_strides(x)
        if x.stride(-1) != 1 or axes is None or any(s % 8 for _, s in axes):
            raise ValueError("x needs a contiguous last axis and at most three row strides, all multiples of 8")
        (n0, s0), (n1, s1), (n2, s2) = axes
    xp = x.data_ptr()
    if xp % 16:
        raise ValueError("x must be 16-byte aligned")
    rc = _quantize(xp, _TORCH_DT[x.dtype], n0, n1, n2, s0, s1, s2, K, codes.data_ptr(), scales.data_ptr(), stream)
    if rc:
        L.check(rc, "anima_quantize4")
    return out


def dequantize4(p: Packed4, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values [..., K] that a packed tensor stands for: exact in float32, rounded once in
    float16 and bfloat16."""
    codes, scales = p
    stream = _here(codes, scales)
    cs = _check_packed(codes, scales, "p")
    dt = _TORCH_DT.get(dtype)
    if dt is None:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    K = 2 * cs[-1]
    y = scales.new_empty(cs[:-1] + (K,), dtype=dtype)
    rc = _dequantize(codes.data_ptr(), scales.data_ptr(), y.data_ptr(), dt, y.numel() // K, K, stream)
    if rc:
        L.check(rc, "anima_dequantize4")
    return y


def matvec4(x: torch.Tensor, w: Packed4, silu: bool = False, add: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """x @ W.T for a few rows x and packed W, in one launch: SiLU of x first if ``silu``, ``add``
    added behind.

    w [N, K] with x [M, K] or [K]; or a stack w [E, N, K] with x [E, M, K].  x is float32,
    float16 or bfloat16 with a contiguous last axis (other strides are free); ``add`` is float32
    and broadcasts to the result [.., M, N] over its leading axes; the result has ``out``'s or
    ``out_dtype``'s type; ``out`` may be ``add`` itself, and overlaps no other operand.  Sums are
    fp32 over exact products, every value of x with all its bits; the result is rounded once.  8 float32 rows or 16 16-bit ones
    share a pass over W."""
    codes, scales = w
    stream = _here(x, codes, scales, add, out)
    ws, xs, xst = _check_packed(codes, scales, "w"), tuple(x.shape), x.stride()
    K, nd = 2 * ws[-1], len(xs)
    xdt = _TORCH_DT.get(x.dtype)
    if xdt is None:
        raise ValueError("x must be float32, float16 or bfloat16")
    E, M, xe, xm = 1, 1, 0, 0
    if len(ws) == 2 and (nd == 2 or nd == 1):
        if nd == 2:
            M, xm = xs[0], xst[0]
    elif len(ws) == 3 and nd == 3 and xs[0] == ws[0]:
        E, M, _ = xs
        xe, xm, _ = xst
    else:
        raise ValueError("w [N, K] takes x [M, K] or [K]; w [E, N, K] takes x [E, M, K]")
    N = ws[-2]
    if xs[-1] != K or xst[-1] != 1:
        raise ValueError(f"x needs a contiguous last axis of K = {K}")
    if K > 32768:
        raise ValueError("K must be at most 32768")
    shape = xs[:-1] + (N,)
    if out is None:
        odt = _TORCH_DT.get(out_dtype)
        if odt is None:
            raise ValueError("out_dtype must be float32, float16 or bfloat16")
        out = x.new_empty(shape, dtype=out_dtype)
        oe, om = M * N, N
    else:
        odt = _TORCH_DT.get(out.dtype)
        if tuple(out.shape) != shape or odt is None or (N > 1 and out.stride(-1) != 1) or _repeats(out):
            raise ValueError("out must be float32, float16 or bfloat16 of the result's shape, its last axis contiguous, none repeated")
        oe, om, _ = ((0, 0) + out.stride())[-3:]
    aptr = ae = am = 0
    if add is not None:
        ash, ast, na = tuple(add.shape), add.stride(), add.dim()
        if add.dtype is not _F32 or (N > 1 and (na == 0 or ash[-1] != N or ast[-1] != 1)):
            raise ValueError("add must be float32 with a contiguous last axis of N values")
        (ne, nm, nn), (ae, am, _) = ((1, 1, 1) + ash)[na:], ((0, 0, 0) + ast)[na:]
        if na > 3 or (ne != E and ne != 1) or (nm != M and nm != 1) or nn != N:
            raise ValueError("add must broadcast to the result")
        aptr, ae, am = add.data_ptr(), (0 if ne == 1 else ae), (0 if nm == 1 else am)
    a = _MATVEC_ARGS.pack(x.data_ptr(), xdt, xe, xm, codes.data_ptr(), scales.data_ptr(), aptr, ae, am,
                          out.data_ptr(), odt, oe, om, E, M, N, K, 1 if silu else 0)
    rc = _matvec(a, stream)
    if rc:
        L.check(rc, "anima_matvec4")
    return out


def attention_core_kv4(q: torch.Tensor, k: Packed4, v: Packed4, B: int, H: int,
                       scale: Optional[float] = None, kv_valid_len: Optional[torch.Tensor] = None,
                       out: Optional[torch.Tensor] = None, out_layout: str = "bshd",
                       out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """attention_core over packed K and V: softmax(q k^T * scale) v per head.

    q [B*H, S_q, 128] contiguous float16 or bfloat16, k/v packed [B*H, S_kv, 128].  Returns
    (or fills) ``out`` in ``out_dtype`` (q's type, or float32) and ``out_layout`` "bshd" [B, S_q, H,
    128] or "bhsd" [B, H, S_q, 128].  ``kv_valid_len`` [B], int32 best: keys at or past it do not count,
    whatever the cache holds there; a sample without any has zero rows.

    ``out`` overlaps no operand.  K and V enter exactly, probabilities to 2^-16; sums are fp32 and the
    result is rounded once (anima_attn_kv4_fwd)."""
    kc, ks = k
    vc, vs = v
    stream = _here(q, kc, ks, vc, vs, out)
    qs, qdt = tuple(q.shape), q.dtype
    if len(qs) != 3 or qdt not in _HALF or not q.is_contiguous():
        raise ValueError("q must be [B*H, S_q, 128], contiguous, float16 or bfloat16")
    BH, Sq, D = qs
    if BH != B * H or D != 128 or BH == 0 or Sq == 0:
        raise ValueError("q must be [B*H, S_q, 128] with at least one row")
    cs = _check_packed(kc, ks, "k")
    if cs != _check_packed(vc, vs, "v") or len(cs) != 3 or cs[0] != BH or cs[1] == 0 or cs[2] != 64:
        raise ValueError("k and v must be packed [B*H, S_kv, 128] with at least one key")
    Skv = cs[1]
    if out_layout == "bshd":
        shape = (B, Sq, H, D)
    elif out_layout == "bhsd":
        shape = (B, H, Sq, D)
    else:
        raise ValueError("out_layout must be 'bshd' or 'bhsd'")
    if out_dtype is None or out_dtype is qdt:
        odt, flags = qdt, 0
    elif out_dtype is _F32:
        odt, flags = _F32, L.FLAG_OUT_F32
    else:
        raise ValueError("out_dtype must be q's type or float32")
    if out is None:
        out = q.new_empty(shape, dtype=odt)
        ob, s1, s2, _ = out.stride()
    else:
        ob, s1, s2, sd = out.stride() if out.dim() == 4 else (0, 0, 0, 0)
        if tuple(out.shape) != shape or out.dtype is not odt or sd != 1 or _repeats(out):
            raise ValueError("out must have q's type (or out_dtype's), the layout's shape, a contiguous head dimension and no repeated axis")
    oh, os = (s2, s1) if out_layout == "bshd" else (s1, s2)
    scale = _SCALE if scale is None else float(scale)
    if not 2.0 ** -150 < scale <= 3.4028234663852886e38:
        raise ValueError("scale must be positive and a float32")
    vp = 0
    if kv_valid_len is not None:
        vl = kv_valid_len if kv_valid_len.dtype is torch.int32 else _lengths32(kv_valid_len, Skv)
        if vl.device != q.device:
            vl = vl.to(q.device)
        vl = vl.contiguous()
        if vl.numel() != B:
            raise ValueError("kv_valid_len must have B entries")
        flags, vp = flags | L.FLAG_MASK, vl.data_ptr()
    nbytes = _kv4_workspace(q.get_device(), qdt, B, H, Sq, Skv)
    # Scratch of this call alone, from the caching allocator: freed on return, its block goes
    # to work enqueued later on this stream, and a captured graph keeps it in its own pool.
    ws = q.new_empty(nbytes, dtype=_U8) if nbytes else None
    a = _ATTN_ARGS.pack(q.data_ptr(), kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), _TORCH_DT[qdt],
                        out.data_ptr(), ob, oh, os, B, H, Sq, Skv, D, scale, flags, vp,
                        0 if ws is None else ws.data_ptr(), nbytes)
    rc = _attn(a, stream)
    if rc:
        L.check(rc, "anima_attn_kv4_fwd")
    return out
