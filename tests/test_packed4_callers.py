"""Callers of the 4-bit storage: what they hand on, and calls that had worked without it."""
import numpy as np
import pytest
import torch

from dit_cpu_attention import cpu_attention
from test_sampling import _contexts, _model


class TwoArgumentCache:
    """A model whose context_cache takes the two contexts, as it did before packed ones."""

    def __init__(self, model):
        self.model, self.calls = model, 0

    def context_cache(self, ctx_cond, ctx_uncond):
        self.calls += 1
        return self.model.context_cache(ctx_cond, ctx_uncond)

    def euler_cfg_step(self, *a, **kw):
        return self.model.euler_cfg_step(*a, **kw)


def test_sampler_with_a_model_of_its_own_cache():
    from anima_attn.sampling import EulerCFGSampler
    cc, cu = _contexts()
    m = _model("cpu", attn_fn=cpu_attention)
    x = torch.randn(1, 16, 16, 16, generator=torch.Generator().manual_seed(3))
    want = EulerCFGSampler(m, cc, cu, 5.0, x.shape, graph=False).sample(x, [0.8, 0.5]).clone()
    wrapped = TwoArgumentCache(m)
    s = EulerCFGSampler(wrapped, cc, cu, 5.0, x.shape, graph=False)
    assert torch.equal(s.sample(x, [0.8, 0.5]), want)
    s.refresh_context(cc, cu)
    assert wrapped.calls == 2 and torch.equal(s.sample(x, [0.8, 0.5]), want)


def test_ksampler_does_not_ignore_kv_bits():
    """kv_bits of a sampler that is handed in is the sampler's own: another one is refused."""
    from anima_attn.sampling import EulerCFGSampler, run_ksampler
    cc, cu = _contexts()
    m = _model("cpu", attn_fn=cpu_attention)
    s = EulerCFGSampler(m, cc, cu, 5.0, (1, 16, 16, 16), graph=False)
    with pytest.raises(ValueError):
        run_ksampler(m, cc, cu, 16, 16, steps=1, sampler=s, kv_bits=4)
    assert np.isfinite(run_ksampler(m, cc, cu, 16, 16, steps=1, sampler=s).numpy()).all()


def test_lengths_of_other_types():
    """Lengths as int32: what that type does not hold means all keys, or none."""
    from anima_attn.packed import _lengths32
    big = torch.tensor([-(1 << 40), -1, 0, 5, 77, 78, 1 << 31, 1 << 40, (1 << 63) - 1])
    assert _lengths32(big, 77).tolist() == [0, 0, 0, 5, 77, 77, 77, 77, 77]
    assert _lengths32(torch.tensor([-3.0, 5.5, 60000.0, float("inf")], dtype=torch.float16), 77).tolist() == [0, 5, 77, 77]
    assert _lengths32(torch.tensor([0, 200], dtype=torch.uint8), 77).tolist() == [0, 200]
    assert _lengths32(torch.tensor([True, False]), 77).tolist() == [1, 0]
    assert _lengths32(big, 77).dtype == torch.int32


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 9, 2200])
def test_lengths_of_other_types_and_devices(Sq):
    """int64 lengths past 2^31 (a mark for "all"), lengths on the host, float lengths: the int32 call's results."""
    import anima_attn
    from test_packed4 import random_packed
    B, H, S = 3, 2, 150
    q = torch.randn(B * H, Sq, 128, generator=torch.Generator().manual_seed(5)).half().cuda()
    k, v = random_packed((B * H, S, 128), 1)[0], random_packed((B * H, S, 128), 2)[0]
    want = anima_attn.attention_core_kv4(q, k, v, B, H, kv_valid_len=torch.tensor([S, 0, 70], dtype=torch.int32, device="cuda"))
    for lens in (torch.tensor([1 << 40, -(1 << 40), 70], device="cuda"), torch.tensor([S, 0, 70]), torch.tensor([S, 0, 70], dtype=torch.int32),
                 torch.tensor([float("inf"), 0, 70.5], device="cuda"), torch.tensor([[S, 0, 70]] * 2, dtype=torch.int32, device="cuda").t()[:, 0]):
        assert torch.equal(anima_attn.attention_core_kv4(q, k, v, B, H, kv_valid_len=lens), want)


@pytest.mark.parametrize("scale", [1e39, 1e-46, 0.0, -1.0, float("inf"), float("nan")])
def test_scales_that_float32_does_not_hold(scale, monkeypatch):
    import anima_attn
    from anima_attn import packed as P
    monkeypatch.setattr(P, "_here", lambda *ts: 0)
    k = anima_attn.Packed4(torch.zeros(4, 5, 64, dtype=torch.uint8), torch.zeros(4, 5, 4, dtype=torch.float16))
    with pytest.raises(ValueError):
        anima_attn.attention_core_kv4(torch.zeros(4, 3, 128, dtype=torch.float16), k, k, 2, 2, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("adaln_bits,kv_bits", [(4, 16), (16, 4), (4, 4)])
def test_what_four_bits_do_to_the_latent(adaln_bits, kv_bits):
    """The packed options against the golden latents of the 16-bit model.  They are outside the parity bar of
    1e-2: 4-bit storage is a choice of memory over exactness.  Bound: the largest of 32 normal values is
    2.4 deviations, the step an eighth of that, its rounding 0.085 of a value (step / sqrt 12); two layers of
    weights, or K and V, 0.12 of a modulation or of a cross-attention's result; twice that for what the later blocks
    and the guidance make of it."""
    import anima_attn
    from anima_attn.dit import AnimaDiT, DiTConfig, make_weights
    from anima_attn.sampling import EulerCFGSampler
    from conftest import golden, rel_l2
    from test_sampling import BLOCKS
    g = golden("sampler_small.npz")
    cfg = DiTConfig(blocks=BLOCKS)
    m = AnimaDiT(cfg, make_weights(cfg, seed=1234, device="cuda"), adaln_bits=adaln_bits)
    cc, cu = (t.cuda() for t in _contexts())
    s = EulerCFGSampler(m, cc, cu, float(g["cfg"]), (1, 16, 32, 32), graph=False, kv_bits=kv_bits)
    r = rel_l2(s.sample(torch.from_numpy(g["noise"]).cuda(), g["sigmas"]).cpu().numpy(), g["latent"])
    print(f"adaln_bits {adaln_bits}, kv_bits {kv_bits}: latent against the golden one {r:.2e}")
    assert r <= 0.25 and anima_attn.status() == 0
