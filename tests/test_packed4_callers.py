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
