"""4-bit storage inside the DiT step and the sampler: packed adaLN modulation weights
(AnimaDiT(adaln_bits=4)) and packed cross-attention K/V (context_cache(kv_bits=4))."""
import numpy as np
import pytest
import torch

from conftest import golden, rel_l2
from dit_cpu_attention import cpu_attention
from test_packed4 import matvec_bound, unpack_ref
from test_sampling import BLOCKS, _contexts, _model

STEP_REL_L2 = 1e-2  # the step's bar against its reference, as in test_dit.py


def test_refusals_without_a_gpu():
    from anima_attn.dit import AnimaDiT, DiTConfig, make_weights
    from anima_attn.sampling import EulerCFGSampler
    cfg = DiTConfig(blocks=1)
    w = make_weights(cfg, seed=1)
    with pytest.raises(ValueError):
        AnimaDiT(cfg, w, attn_fn=cpu_attention, adaln_bits=8)
    with pytest.raises(ValueError):
        AnimaDiT(cfg, w, attn_fn=cpu_attention, adaln_bits=4)  # CPU weights
    m = AnimaDiT(cfg, w, attn_fn=cpu_attention)
    cc, cu = _contexts()
    for bits in (4, 2):
        with pytest.raises(ValueError):
            m.context_cache(cc, cu, kv_bits=bits)
    with pytest.raises(ValueError):
        EulerCFGSampler(m, cc, cu, 5.0, (1, 16, 16, 16), graph=False, cache_context=False, kv_bits=4)


def _packed_model(seed=1234):
    from anima_attn.dit import AnimaDiT, DiTConfig, make_weights
    cfg = DiTConfig(blocks=BLOCKS)
    return AnimaDiT(cfg, make_weights(cfg, seed=seed, device="cuda"), adaln_bits=4)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 2, 9])
def test_modulations_from_packed_weights(B):
    """_all_mods with packed weights: SiLU, both layers and the addend, in 64 bits from the values that
    the packed weights stand for.  The hidden layer's own bound passes through the second layer."""
    torch.cuda.set_device(0)
    m = _packed_model()
    g = torch.Generator().manual_seed(4)
    emb = torch.randn(B, 1, 2048, generator=g).cuda()
    lora = torch.randn(B, 1, 3 * 2048, generator=g).cuda()
    got = m._all_mods(emb, lora).double().cpu().numpy()
    w1, w2 = (unpack_ref(*t) for t in m._mod_w)
    x = emb[:, 0].double().cpu().numpy()
    x = x / (1 + np.exp(-x))
    h = x @ w1.T
    eh = matvec_bound(np.abs(x), np.abs(w1), 2048, h, torch.float32, True)
    lo = lora[:, 0].double().cpu().numpy()
    n, lr = w2.shape[0], w2.shape[2]
    for e in range(n):
        he, ee = h[:, e * lr:(e + 1) * lr], eh[:, e * lr:(e + 1) * lr]
        y = he @ w2[e].T + lo
        tol = matvec_bound(np.abs(he), np.abs(w2[e]), lr, y, torch.float32, False) + ee @ np.abs(w2[e]).T + np.abs(lo) * 2.0 ** -23
        assert (np.abs(got[e] - y) <= tol).all(), e


@pytest.mark.gpu
def test_step_with_packed_modulations():
    """The step against the 16-bit model given the same (unpacked) modulation weights, and the memory."""
    import anima_attn
    from anima_attn.dit import AnimaDiT, DiTConfig, make_weights
    torch.cuda.set_device(0)
    m = _packed_model()
    assert not any("blocks." in k and "adaln_modulation" in k for k in m.w)
    held = sum(t.numel() * t.element_size() for p in m._mod_w for t in p)
    cfg = DiTConfig(blocks=BLOCKS)
    w = make_weights(cfg, seed=1234, device="cuda")
    v1, v2 = (anima_attn.dequantize4(p, torch.float16) for p in m._mod_w)
    full, lr = 0, cfg.adaln_lora
    i = 0
    for b in range(BLOCKS):
        for s in ("self_attn", "cross_attn", "mlp"):
            for layer, v in ((1, v1[i * lr:(i + 1) * lr]), (2, v2[i])):
                name = f"blocks.{b}.adaln_modulation_{s}.{layer}.weight"
                full += w[name].numel() * 2
                assert w[name].shape == v.shape
                w[name] = v
            i += 1
    assert held * 32 == full * 9  # 4.5 bits against 16
    ref = AnimaDiT(cfg, w)
    cc, cu = (t.cuda() for t in _contexts())
    x = torch.randn(1, 16, 32, 32, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    a = ref.euler_cfg_step(x, 0.8, 0.5, cc, cu, 5.0).cpu().numpy()
    b = m.euler_cfg_step(x, 0.8, 0.5, cc, cu, 5.0).cpu().numpy()
    assert anima_attn.status() == 0 and rel_l2(b, a) <= STEP_REL_L2


@pytest.mark.gpu
@pytest.mark.parametrize("fused_qkv", [True, False])
def test_step_with_packed_context(fused_qkv):
    """The step with a packed context cache against the same step with a 16-bit cache of the values that
    it stands for."""
    import anima_attn
    from anima_attn.dit import AnimaDiT, DiTConfig, make_weights
    torch.cuda.set_device(0)
    cfg = DiTConfig(blocks=BLOCKS)
    m = AnimaDiT(cfg, make_weights(cfg, seed=1234, device="cuda"), fused_qkv=fused_qkv)
    cc, cu = (t.cuda() for t in _contexts())
    x = torch.randn(1, 16, 32, 32, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    packed = m.context_cache(cc, cu, kv_bits=4)
    wide = {k: {"kh": anima_attn.dequantize4(e["k4"], cfg.gemm_dtype), "vh": anima_attn.dequantize4(e["v4"], cfg.gemm_dtype)}
            for k, e in packed.items()}
    exact = m.context_cache(cc, cu)
    for k, e in exact.items():  # within half a step of the group's scale, whose extreme is 8 steps
        for n in ("kh", "vh"):
            v = e[n].float().unflatten(-1, (4, 32))
            top = v.abs().amax(-1, keepdim=True)
            assert ((wide[k][n].float().unflatten(-1, (4, 32)) - v).abs() <= top / 8 * 1.01).all()
    a = m.euler_cfg_step(x, 0.8, 0.5, cc, cu, 5.0, ctx_cache=wide).cpu().numpy()
    b = m.euler_cfg_step(x, 0.8, 0.5, cc, cu, 5.0, ctx_cache=packed).cpu().numpy()
    assert anima_attn.status() == 0 and rel_l2(b, a) <= 1e-3  # as cached against uncached


@pytest.mark.gpu
def test_sampler_with_packed_storage():
    """Everything together as served: packed weights, packed context, one captured step replayed over a
    schedule, new prompts and back."""
    import anima_attn
    from anima_attn.sampling import EulerCFGSampler, run_ksampler
    torch.cuda.set_device(0)
    g = golden("sampler_small.npz")
    cc, cu = (t.cuda() for t in _contexts())
    m = _packed_model()
    s = EulerCFGSampler(m, cc, cu, float(g["cfg"]), (1, 16, 32, 32), graph=True, kv_bits=4)
    noise = torch.from_numpy(g["noise"]).cuda()
    first = s.sample(noise, g["sigmas"]).cpu().numpy()
    again = s.sample(noise, g["sigmas"]).cpu().numpy()
    assert np.isfinite(first).all() and np.array_equal(first, again)
    s.refresh_context(cu, cc)
    swapped = s.sample(noise, g["sigmas"]).cpu().numpy()
    assert not np.array_equal(swapped, first)
    s.refresh_context(cc, cu)
    assert np.array_equal(s.sample(noise, g["sigmas"]).cpu().numpy(), first)
    eager = EulerCFGSampler(m, cc, cu, float(g["cfg"]), (1, 16, 32, 32), graph=False, kv_bits=4)
    assert rel_l2(eager.sample(noise, g["sigmas"]).cpu().numpy(), first) <= 1e-6
    out = run_ksampler(m, cc, cu, 32, 32, steps=int(g["meta"][2]), cfg=float(g["cfg"]), seed=int(g["meta"][3]), kv_bits=4)
    assert rel_l2(out.cpu().numpy(), first) <= 1e-6 and anima_attn.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_attention_cached_kv_takes_packed_operands(out_dtype):
    import anima_attn
    from anima_attn.ops import attention_cached_kv, prologue
    torch.cuda.set_device(0)
    g = torch.Generator(device="cuda").manual_seed(5)
    B, S, H, N = 2, 96, 4, 77
    q = torch.randn(B, S, H, 128, device="cuda", generator=g)
    k, v = (torch.randn(B, N, H, 128, device="cuda", generator=g) for _ in range(2))
    qw = 1 + 0.1 * torch.randn(128, device="cuda", generator=g)
    _, kh, vh = prologue(None, k, v, None, qw, op_dtype=torch.float16)
    k4, v4 = anima_attn.quantize4(kh), anima_attn.quantize4(vh)
    valid = torch.tensor([77, 31], dtype=torch.int32, device="cuda")
    want = attention_cached_kv(q, anima_attn.dequantize4(k4), anima_attn.dequantize4(v4), qw, kv_valid_len=valid)
    got = attention_cached_kv(q, k4, v4, qw, kv_valid_len=valid, out_dtype=out_dtype)
    assert got.dtype == out_dtype and rel_l2(got.float().cpu().numpy(), want.cpu().numpy()) <= 5e-3
    out = torch.empty(B, S, H, 128, dtype=out_dtype, device="cuda")
    assert attention_cached_kv(q, k4, v4, qw, kv_valid_len=valid, out_dtype=out_dtype, out=out) is out
    assert torch.equal(out, got)
