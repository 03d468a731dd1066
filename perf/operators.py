"""The 4-bit operators of the library as timed cases, with their plain forms.

Three operators share one storage format (the "packed" format, 4.5 bits per value):

  pack      quantize4 / dequantize4: rows of 16-bit values to 4-bit codes with one fp16 scale
            per 32 values, and back to the values that the codes stand for
  attention attention_core_kv4: softmax(q K^T * scale) V with K and V held packed
  matvec    matvec4: x W^T for a few rows x and packed weights W, optionally SiLU(x) first
            and an addend behind, for one matrix or a stack of matrices

Packed format of a row of K values (K a multiple of 128): group g holds values 32 g .. 32 g + 31.
Its scale is s = x* / -8 in fp16, where x* is the value of largest magnitude (the positive one
if both signs reach it); a value's code is n = floor(x / s + 1/2) clamped to [-8, 7] and
stands for n * s.  A group holding a value that fp16 cannot hold finitely gets a NaN scale.
Codes are stored as n + 8, eight to a 32-bit word and 16 words to a block of 128 values: word
4 i + g of a block holds values 32 g + 8 i + e, e = 0..7, with value e at nibble e / 2 + 4 (e % 2).

``own`` false computes the plain forms (fp32 torch operations, rounded once at the end); true
calls the library.
"""
import math
import os
import sys

import torch

own = False

D = 128       # head size of every attention of the library
GROUP = 32    # values that share a scale
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MAX_ATTN_FLOPS = 4 * 32 * D * 16384 * 512
MAX_CACHE_ROWS = 32 * 65536
MAX_WEIGHTS = 84 * 6144 * 256


def listed():
    return [
        # One query row against a text context of 512 tokens: the smallest call, latency counts.
        {"name": "attn 1x512", "op": "attn", "B": 2, "H": 16, "Sq": 1, "Skv": 512, "dtype": "f16", "mask": False},
        # One query row per head against a long cache: bound by reading the cache.
        {"name": "attn 1x65536", "op": "attn", "B": 2, "H": 16, "Sq": 1, "Skv": 65536, "dtype": "bf16", "mask": False},
        # A few rows, odd lengths, one sample without a valid key.
        {"name": "attn 7x1237 masked", "op": "attn", "B": 3, "H": 16, "Sq": 7, "Skv": 1237, "dtype": "bf16", "mask": True},
        # Cross-attention of a 256-token image into a padded context.
        {"name": "attn 256x512 masked", "op": "attn", "B": 2, "H": 16, "Sq": 256, "Skv": 512, "dtype": "f16", "mask": True},
        # Cross-attention of the 4096-token denoising step, the guidance pair as a batch.
        {"name": "attn 4096x512", "op": "attn", "B": 2, "H": 16, "Sq": 4096, "Skv": 512, "dtype": "f16", "mask": False},
        # The same of a 16384-token image.
        {"name": "attn 16384x512", "op": "attn", "B": 2, "H": 16, "Sq": 16384, "Skv": 512, "dtype": "f16", "mask": False},
        # One modulation-sized matrix and one row: latency counts.
        {"name": "matvec 6144x2048", "op": "matvec", "E": 1, "M": 1, "N": 6144, "K": 2048, "x": "f32", "out": "f32", "silu": True, "add": False},
        # First layers of all adaLN-LoRA modulations of a step, as one matrix; guidance pair.
        {"name": "matvec 21504x2048", "op": "matvec", "E": 1, "M": 2, "N": 21504, "K": 2048, "x": "f32", "out": "f32", "silu": True, "add": False},
        # Their second layers: 84 matrices, each with its own rows, and the shared addend.
        {"name": "matvec 84x6144x256", "op": "matvec", "E": 84, "M": 2, "N": 6144, "K": 256, "x": "f32", "out": "f32", "silu": False, "add": True},
        # Odd sizes, 16-bit rows and results.
        {"name": "matvec 1003x1152", "op": "matvec", "E": 1, "M": 7, "N": 1003, "K": 1152, "x": "bf16", "out": "bf16", "silu": False, "add": False},
        # K of one block's text context, packed and read back.
        {"name": "pack 16384x128", "op": "pack", "rows": 32 * 512, "K": 128, "dtype": "f16"},
        # The stack of second modulation layers, packed at load time and read back.
        {"name": "pack 516096x256", "op": "pack", "rows": 84 * 6144, "K": 256, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "matvec", "matvec", "pack"])
    if op == "attn":
        B, H = rng.randint(1, 4), rng.choice([1, 2, 4, 8, 16])
        Sq = _log(rng, 1, 16384)
        most = min(65536, MAX_CACHE_ROWS // (B * H), MAX_ATTN_FLOPS // (4 * B * H * D * Sq))
        return {"op": op, "B": B, "H": H, "Sq": Sq, "Skv": _log(rng, 1, most),
                "dtype": rng.choice(["f16", "bf16"]), "mask": rng.random() < 0.5}
    if op == "matvec":
        K = 128 * _log(rng, 1, 64)
        E = _log(rng, 1, 84)
        N = _log(rng, 1, min(21504, MAX_WEIGHTS // (K * E)))
        return {"op": op, "E": E, "M": _log(rng, 1, 16), "N": N, "K": K,
                "x": rng.choice(["f32", "f16", "bf16"]), "out": rng.choice(["f32", "f16", "bf16"]),
                "silu": rng.random() < 0.5, "add": rng.random() < 0.5}
    K = 128 * _log(rng, 1, 64)
    return {"op": op, "rows": _log(rng, 1, MAX_WEIGHTS // K), "K": K, "dtype": rng.choice(["f16", "bf16"])}


def _lens(case):
    """Valid keys per sample: from all down to none over the batch."""
    B, S = case["B"], case["Skv"]
    if not case["mask"]:
        return [S] * B
    return [S * (B - 1 - b) // (B - 1) for b in range(B)] if B > 1 else [(2 * S + 2) // 3]


def work(case):
    packed = 0.5 + 2 / GROUP  # bytes per packed value
    if case["op"] == "attn":
        B, H, Sq = case["B"], case["H"], case["Sq"]
        keys = sum(_lens(case))
        return {"bytes": int(2 * B * H * Sq * D * 2 + 2 * H * keys * D * packed),
                "flops": 4 * H * D * Sq * keys}
    if case["op"] == "matvec":
        E, M, N, K = case["E"], case["M"], case["N"], case["K"]
        size = {"f32": 4, "f16": 2, "bf16": 2}
        nbytes = E * N * K * packed + E * M * K * size[case["x"]] + E * M * N * size[case["out"]]
        return {"bytes": int(nbytes + (M * N * 4 if case["add"] else 0)), "flops": 2 * E * M * N * K}
    n = case["rows"] * case["K"]
    return {"bytes": int(n * (2 + packed + packed + 2)), "flops": 2 * n}


# ---------------------------------------------------------------- the packed format, plainly
def _pack(x):
    """[..., K] 16-bit -> (codes uint8 [..., K / 2], scales fp16 [..., K / 32])."""
    g = x.float().unflatten(-1, (-1, GROUP))
    hi, lo = g.amax(-1), g.amin(-1)
    s = (torch.where(hi >= -lo, hi, lo) / -8).half()
    s = torch.where(g.abs().amax(-1) <= 65504, s, torch.full_like(s, math.nan))
    # the quotient of two 16-bit values is at a border between codes exactly, or 2^-13 away from it
    n = torch.floor(g / s.float().unsqueeze(-1) + 0.5)
    n = torch.where(torch.isnan(n) | (s == 0).unsqueeze(-1), torch.zeros_like(n), n).clamp(-8, 7)
    n = (n + 8).to(torch.uint8).flatten(-2).unflatten(-1, (-1, 4, 4, 8))  # block, g, i, e
    n = n.transpose(-3, -2)  # words in the order i, g
    # byte b of a word holds nibbles 2 b and 2 b + 1; nibble p holds value 2 (p % 4) + p / 4
    low, high = n[..., [0, 4, 1, 5]], n[..., [2, 6, 3, 7]]
    return (low | (high << 4)).flatten(-4).contiguous(), s.contiguous()


def _numbers(codes):
    """[..., K / 2] codes -> [..., K] whole numbers n in [-8, 7], int16."""
    c = codes.unflatten(-1, (-1, 4, 4, 4)).to(torch.int16)  # block, i, g, byte
    n = torch.stack([c & 15, c >> 4], -1).flatten(-2) - 8   # ..., nibble
    n = n[..., [0, 4, 1, 5, 2, 6, 3, 7]]                    # ..., value
    return n.transpose(-3, -2).flatten(-4)


def _unpack(codes, scales):
    """The values that packed rows stand for, in fp32 (exact)."""
    return (_numbers(codes).float().unflatten(-1, (-1, GROUP)) * scales.float().unsqueeze(-1)).flatten(-2)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g).to(dtype)

    state = {"case": case}
    if case["op"] == "attn":
        dt, n = DTYPES[case["dtype"]], case["B"] * case["H"]
        state["q"] = normal(n, case["Sq"], D, dtype=dt)
        state["k"] = _pack(normal(n, case["Skv"], D, dtype=dt))
        state["v"] = _pack(normal(n, case["Skv"], D, dtype=dt))
        state["valid"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda") if case["mask"] else None
    elif case["op"] == "matvec":
        E, M, N, K = case["E"], case["M"], case["N"], case["K"]
        state["x"] = normal(E, M, K, dtype=DTYPES[case["x"]])
        state["w"] = _pack(normal(E, N, K, dtype=torch.bfloat16, std=0.02))
        state["add"] = normal(M, N) if case["add"] else None
    else:
        state["x"] = normal(case["rows"], case["K"], dtype=DTYPES[case["dtype"]])
    return state


def _library():
    if "anima_attn" not in sys.modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "anima-on-android_b200"))
    import anima_attn
    return anima_attn


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        lib = _library()
        if case["op"] == "attn":
            return lib.attention_core_kv4(state["q"], lib.Packed4(*state["k"]), lib.Packed4(*state["v"]),
                                          case["B"], case["H"], kv_valid_len=state["valid"])
        if case["op"] == "matvec":
            return lib.matvec4(state["x"], lib.Packed4(*state["w"]), silu=case["silu"], add=state["add"],
                               out_dtype=DTYPES[case["out"]])
        packed = lib.quantize4(state["x"])
        return {"values": lib.dequantize4(packed, state["x"].dtype), "scales": packed.scales}
    if case["op"] == "attn":
        return _attention(state["q"], state["k"], state["v"], case["B"], case["H"], state["valid"])
    if case["op"] == "matvec":
        x = state["x"].float()
        if case["silu"]:
            x = x / (1 + torch.exp(-x))
        y = x @ _unpack(*state["w"]).transpose(-1, -2)
        if state["add"] is not None:
            y = y + state["add"]
        return y.to(DTYPES[case["out"]])
    codes, scales = _pack(state["x"])
    return {"values": _unpack(codes, scales).to(state["x"].dtype), "scales": scales}


def _attention(q, k, v, B, H, valid):
    """[B H, Sq, D] rows against packed K and V -> [B, Sq, H, D] in q's type."""
    k, v = _unpack(*k), _unpack(*v)
    s = (q.float() @ k.transpose(-1, -2)) * (1 / math.sqrt(D))
    if valid is not None:
        beyond = torch.arange(k.shape[1], device=q.device) >= valid.repeat_interleave(H)[:, None]
        s = s.masked_fill(beyond[:, None, :], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)  # no key: a row of zeros
    return o.unflatten(0, (B, H)).transpose(1, 2).contiguous().to(q.dtype)


# ---------------------------------------------------------------- in 64 bits, from the definitions
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attn":
        B, H, Sq = case["B"], case["H"], case["Sq"]
        out = torch.zeros(B, Sq, H, D, dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lens(case)):
            for h in range(H if n else 0):
                k, v = (_values64(c[b * H + h, :n], s[b * H + h, :n]) for c, s in (state["k"], state["v"]))
                for lo in range(0, Sq, 4096):
                    a = state["q"][b * H + h, lo:lo + 4096].double() @ k.T / math.sqrt(D)
                    out[b, lo:lo + 4096, h] = torch.softmax(a, -1) @ v
        return out
    if case["op"] == "matvec":
        E = case["E"]
        x = state["x"].double()
        x = x * torch.sigmoid(x) if case["silu"] else x
        add = 0.0 if state["add"] is None else state["add"].double()
        return torch.stack([x[e] @ _values64(state["w"][0][e], state["w"][1][e]).T + add for e in range(E)])
    values, scales = [], []
    for x in state["x"].split(max(1, (1 << 25) // case["K"])):
        g = x.double().reshape(x.shape[0], -1, GROUP)
        top = g.max(-1).values
        big = torch.where(top >= g.abs().max(-1).values, top, g.min(-1).values)
        s = (big * -0.125).half().double()
        n = torch.where(s[..., None] == 0, 0.0, (g / s[..., None] + 0.5).floor()).clamp(-8, 7)
        values.append((n * s[..., None]).reshape(x.shape))
        scales.append(s)
    return {"values": torch.cat(values), "scales": torch.cat(scales)}


def _values64(codes, scales):
    """Values of packed rows [R, K] in 64 bits, read nibble by nibble from the format's words."""
    rows, half = codes.shape
    words = codes.reshape(rows, half // 64, 16, 4).long()
    words = words[..., 0] | words[..., 1] << 8 | words[..., 2] << 16 | words[..., 3] << 24
    out = torch.empty(rows, half // 64, 128, dtype=torch.float64, device=codes.device)
    s = scales.double().reshape(rows, half // 64, 4)
    for w in range(16):
        i, g = divmod(w, 4)
        for e in range(8):
            n = (words[:, :, w] >> 4 * (e // 2 + 4 * (e % 2)) & 15) - 8
            out[:, :, 32 * g + 8 * i + e] = n * s[:, :, g]
    return out.reshape(rows, 2 * half)
