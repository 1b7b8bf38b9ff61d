"""Tangents of the language-model operators: formed by the tensor library on every device, or refused - never lost."""
import pytest
import torch
from torch.autograd import forward_ad

import mxnet_b200 as mx

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def op(name):
    return mx.ops.get('_contrib_' + name).fn


def functions(device):
    rng = torch.Generator().manual_seed(3)
    draw = lambda *shape: torch.randn(*shape, generator=rng).to(device)   # noqa: E731
    freq, k = torch.tensor([1.0, 0.1], device=device), draw(1, 6, 1, 64)
    tok = torch.tensor([3, 0, 2, 1, 2, 3], device=device)
    return draw, [(draw(1, 6, 2, 64), lambda x: op('rotary_embedding')(x, torch.arange(6, device=device), freq)),
                  (draw(1, 6, 2, 64), lambda x: op('sldwin_attention')(x, k, k, window=3, sinks=1)),
                  (draw(1, 6, 1, 64), lambda x: op('sldwin_attention')(k, x, x * 2, window=3)),
                  (draw(6, 10), lambda x: torch.cat([t.reshape(-1) for t in op('token_log_probs')(x, tok, topk=3)[:3]]))]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('which', range(4))
def test_tangents_against_gradients(device, which):
    draw, cases = functions(device)
    x, f = cases[which]
    t = draw(*x.shape)
    with forward_ad.dual_level():
        out, tangent = forward_ad.unpack_dual(f(forward_ad.make_dual(x, t)))
    assert tangent is not None
    a = x.clone().requires_grad_(True)
    y = f(a)
    g = draw(*y.shape)
    dx, = torch.autograd.grad(y, a, g)
    # both are fp32 sums of up to 1000 products of order 1, of relative error 2^-22 each
    size = float((tangent.abs() * g.abs()).sum() + (dx.abs() * t.abs()).sum())
    assert abs(float((tangent * g).sum()) - float((dx * t).sum())) <= 1e-5 * size
    assert float((out - y).detach().abs().max()) <= 1e-5 * float(1 + y.detach().abs().max())


@pytest.mark.parametrize('device', DEVICES)
def test_caches_have_no_tangents(device):
    x = torch.randn(1, 2, 4, device=device)
    for dual in range(3):
        caches = [torch.zeros(1, 5, 2, 4, device=device) for _ in range(2)]
        with forward_ad.dual_level():
            a = [x, x.clone(), x.clone()]
            a[dual] = forward_ad.make_dual(a[dual], torch.ones_like(x))
            with pytest.raises(mx.base.MXNetError, match='no gradient'):
                op('sldwin_attention_step')(*a, *caches, torch.tensor([0], device=device))
            if dual:
                with pytest.raises(mx.base.MXNetError, match='no gradient'):
                    op('sldwin_cache_fill')(a[1][:, None], a[2][:, None], *caches)
        assert not bool(caches[0].any())
