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
_U8, _F16 = torch.uint8, torch.float16


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


def _check_packed(p: Packed4, what: str) -> torch.Size:
    """The codes' shape [..., K/2], after checking that codes and scales belong together."""
    c, s = p
    if c.dtype is not _U8 or s.dtype is not _F16 or not c.is_contiguous() or not s.is_contiguous():
        raise ValueError(f"{what}: packed codes are contiguous uint8, scales contiguous float16")
    cs, ss = c.shape, s.shape
    half = cs[-1] if cs and ss else 0
    if half == 0 or half % 64 or ss[-1] * 16 != half or cs[:-1] != ss[:-1]:
        raise ValueError(f"{what}: codes [..., K/2] and scales [..., K/32], K a multiple of 128")
    return cs


@lru_cache(maxsize=1024)
def _kv4_workspace(dev: int, dtype: torch.dtype, B: int, H: int, Sq: int, Skv: int) -> int:
    return int(L.lib.anima_attn_kv4_workspace_size(_TORCH_DT[dtype], B, H, Sq, Skv))


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
    if x.dim() == 0 or x.shape[-1] == 0 or x.shape[-1] % 128:
        raise ValueError("the last axis must be a positive multiple of 128")
    K, lead = x.shape[-1], x.shape[:-1]
    if out is None:
        out = Packed4(x.new_empty(lead + (K // 2,), dtype=_U8), x.new_empty(lead + (K // 32,), dtype=_F16))
    else:
        _here(*out)
        _check_packed(out, "out")
        if out.codes.shape != lead + (K // 2,):
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
    if x.data_ptr() % 16:
        raise ValueError("x must be 16-byte aligned")
    rc = L.lib.anima_quantize4(x.data_ptr(), _TORCH_DT[x.dtype], n0, n1, n2, s0, s1, s2, K,
                               out.codes.data_ptr(), out.scales.data_ptr(), stream)
    if rc:
        L.check(rc, "anima_quantize4")
    return out


def dequantize4(p: Packed4, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values [..., K] that a packed tensor stands for: exact in float32, rounded once in
    float16 and bfloat16."""
    stream = _here(*p)
    cs = _check_packed(p, "p")
    if dtype not in _TORCH_DT:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    K = 2 * cs[-1]
    y = p.scales.new_empty(cs[:-1] + (K,), dtype=dtype)
    rc = L.lib.anima_dequantize4(p.codes.data_ptr(), p.scales.data_ptr(), y.data_ptr(),
                                 _TORCH_DT[dtype], y.numel() // K, K, stream)
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
    fp32 over exact products, and of float32 x only what is below 2^-31 of its group's largest
    is lost, so the result is an fp32 one rounded once.  8 float32 rows or 16 16-bit ones
    share a pass over W."""
    stream = _here(x, add, out, *w)
    ws = _check_packed(w, "w")
    K = 2 * ws[-1]
    if x.dtype not in _TORCH_DT:
        raise ValueError("x must be float32, float16 or bfloat16")
    if len(ws) == 2 and x.dim() in (1, 2):
        E, xv = 1, x if x.dim() == 2 else x.unsqueeze(0)
        M, xe, xm = xv.shape[0], 0, xv.stride(0)
    elif len(ws) == 3 and x.dim() == 3 and x.shape[0] == ws[0]:
        E, M, xe, xm = ws[0], x.shape[1], x.stride(0), x.stride(1)
    else:
        raise ValueError("w [N, K] takes x [M, K] or [K]; w [E, N, K] takes x [E, M, K]")
    N = ws[-2]
    if x.shape[-1] != K or x.stride(-1) != 1:
        raise ValueError(f"x needs a contiguous last axis of K = {K}")
    if K > 32768:
        raise ValueError("K must be at most 32768")
    shape = x.shape[:-1] + (N,)
    if out is None:
        if out_dtype not in _TORCH_DT:
            raise ValueError("out_dtype must be float32, float16 or bfloat16")
        out = x.new_empty(shape, dtype=out_dtype)
    elif out.shape != shape or out.dtype not in _TORCH_DT or (N > 1 and out.stride(-1) != 1) or _repeats(out):
        raise ValueError("out must be float32, float16 or bfloat16 of the result's shape, its last axis contiguous, none repeated")
    ostr = out.stride()
    oe, om = ((0, 0) if len(shape) == 1 else (0, ostr[0])) if len(ws) == 2 else (ostr[0], ostr[1])
    aptr = ae = am = 0
    if add is not None:
        if add.dtype != torch.float32 or (N > 1 and (add.dim() == 0 or add.shape[-1] != N or add.stride(-1) != 1)):
            raise ValueError("add must be float32 with a contiguous last axis of N values")
        try:
            av = add.expand(E, M, N)
        except RuntimeError:
            raise ValueError("add must broadcast to the result") from None
        aptr, (ae, am, _) = av.data_ptr(), av.stride()
    a = _MATVEC_ARGS.pack(x.data_ptr(), _TORCH_DT[x.dtype], xe, xm, w.codes.data_ptr(),
                          w.scales.data_ptr(), aptr, ae, am, out.data_ptr(), _TORCH_DT[out.dtype],
                          oe, om, E, M, N, K, 1 if silu else 0)
    rc = L.lib.anima_matvec4(a, stream)
    if rc:
        L.check(rc, "anima_matvec4")
    return out


def attention_core_kv4(q: torch.Tensor, k: Packed4, v: Packed4, B: int, H: int,
                       scale: Optional[float] = None, kv_valid_len: Optional[torch.Tensor] = None,
                       out: Optional[torch.Tensor] = None, out_layout: str = "bshd") -> torch.Tensor:
    """attention_core over packed K and V: softmax(q k^T * scale) v per head.

    q [B*H, S_q, 128] contiguous float16 or bfloat16, k/v packed [B*H, S_kv, 128].  Returns
    (or fills) ``out`` in q's type and ``out_layout`` "bshd" [B, S_q, H, 128] or "bhsd" [B, H,
    S_q, 128].  ``kv_valid_len`` int32 [B]: keys at or past it do not count, whatever the
    cache holds there; a sample without any has zero rows.

    ``out`` overlaps no operand.  Few query rows have fp32 accuracy up to the output's rounding;
    many run on fp16 operands (unpacked K and V, probabilities), whose products are summed in
    fp32 (anima_attn_kv4_fwd)."""
    stream = _here(q, kv_valid_len, out, *k, *v)
    if q.dim() != 3 or q.dtype not in _HALF or not q.is_contiguous():
        raise ValueError("q must be [B*H, S_q, 128], contiguous, float16 or bfloat16")
    BH, Sq, D = q.shape
    if BH != B * H or D != 128 or BH == 0 or Sq == 0:
        raise ValueError("q must be [B*H, S_q, 128] with at least one row")
    ks = _check_packed(k, "k")
    if ks != _check_packed(v, "v") or len(ks) != 3 or ks[0] != BH or ks[1] == 0 or ks[2] != 64:
        raise ValueError("k and v must be packed [B*H, S_kv, 128] with at least one key")
    Skv = ks[1]
    if out_layout not in ("bshd", "bhsd"):
        raise ValueError("out_layout must be 'bshd' or 'bhsd'")
    shape = (B, Sq, H, D) if out_layout == "bshd" else (B, H, Sq, D)
    if out is None:
        out = q.new_empty(shape)
    elif out.shape != shape or out.dtype != q.dtype or out.stride(3) != 1 or _repeats(out):
        raise ValueError("out must have q's type, the layout's shape, a contiguous head dimension and no repeated axis")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("scale must be positive")
    st = out.stride()
    strides = (st[0], st[2], st[1]) if out_layout == "bshd" else (st[0], st[1], st[2])
    flags, vl = 0, None
    if kv_valid_len is not None:
        vl = kv_valid_len if kv_valid_len.dtype is torch.int32 else kv_valid_len.to(torch.int32)
        vl = vl.contiguous()
        if vl.numel() != B:
            raise ValueError("kv_valid_len must have B entries")
        flags = L.FLAG_MASK
    nbytes = _kv4_workspace(q.get_device(), q.dtype, B, H, Sq, Skv)
    # Scratch of this call alone, from the caching allocator: freed on return, its block goes
    # to work enqueued later on this stream, and a captured graph keeps it in its own pool.
    ws = q.new_empty(nbytes, dtype=_U8) if nbytes else None
    a = _ATTN_ARGS.pack(q.data_ptr(), k.codes.data_ptr(), k.scales.data_ptr(), v.codes.data_ptr(),
                        v.scales.data_ptr(), _TORCH_DT[q.dtype], out.data_ptr(), *strides, B, H, Sq, Skv,
                        D, scale, flags, 0 if vl is None else vl.data_ptr(),
                        0 if ws is None else ws.data_ptr(), nbytes)
    rc = L.lib.anima_attn_kv4_fwd(a, stream)
    if rc:
        L.check(rc, "anima_attn_kv4_fwd")
    return out
