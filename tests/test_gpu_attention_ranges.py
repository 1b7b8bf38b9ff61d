"""Attention gradients in fp16 where the values are far larger than 1: the scaled gradients of the scores stay in the type's range."""
import math

import pytest
import torch


import _transformer_oracle as oracle
from test_gpu_transformer_ops import run_attention

pytestmark = pytest.mark.gpu
HALF = torch.float16


def randn(*shape):
    return torch.randn(*shape, device='cuda').to(HALF)


def check(q, k, v, g, valid=None, window=0, sinks=0):
    """Against the definition, with the floor of the type's smallest step for dS: fp16 holds f dS to 2^-25, and f is 2^3 over the largest
    |dO| (to the power of two below it) or as much smaller as D |V| |dO| makes it: an error of a score's gradient of
    max(2^-28 |dO|, 2^-39 D |dO| |V|) times twice, for the powers of two that both are cut to."""
    got = run_attention(q, k, v, valid, window, sinks, g)
    want, bound = oracle.attention(q, k, v, valid, window, sinks, None, g, t=HALF)
    B, T, Hq, D = q.shape
    Hk = k.shape[2]
    gmax, vmax = float(g[g.isfinite()].abs().max()), float(v[v.isfinite()].abs().max())
    floor = 2 * max(2.0 ** -28 * gmax, 2.0 ** -39 * D * gmax * vmax) / math.sqrt(D)
    for b in range(B):
        n = T if valid is None else int(valid[b])
        seen = oracle.visible(n, window, sinks).double()
        for h in range(Hq):
            e = h * Hk // Hq
            bound[1][b, :n, h] += floor * (seen @ k[b, :n, e].double().cpu().abs())
            bound[2][b, :n, e] += floor * (seen.T @ q[b, :n, h].double().cpu().abs())
    for name, a, w, e in zip(('out', 'dq', 'dk', 'dv'), got, want, bound):
        assert float(w.abs().max()) < 65000, name             # what is asked for fits the type
        oracle.check(a, w, e, name)


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('T', [2, 128, 300])
@pytest.mark.parametrize('size', [130, 500])
def test_two_opposite_values(D, T, size):
    """dO of ones and values of +size and -size over all channels at equally weighted keys: f dS would be D size / 2 * 8."""
    q, k = randn(1, T, 2, D) / 64, randn(1, T, 2, D) / 64
    v = torch.full((1, T, 2, D), float(size), device='cuda', dtype=HALF)
    v[:, 1::2] *= -1
    check(q, k, v, torch.ones_like(q))


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('Hq,Hk,window,sinks', [(2, 2, 0, 0), (4, 1, 70, 3), (2, 1, 129, 130)])
@pytest.mark.parametrize('size,g', [(31, 1), (100, 1), (500, 0.01), (3000, 300), (20000, 0.01)])
def test_large_values(D, Hq, Hk, window, sinks, size, g):
    T = 391
    q, k = randn(2, T, Hq, D) / 64, randn(2, T, Hk, D) / 64
    sign = randn(2, T, Hk, 1).sign()
    v = (sign * size + randn(2, T, Hk, D)).to(HALF)           # coherent over the channels
    valid = torch.tensor([T, 250], dtype=torch.int32, device='cuda')
    dout = (torch.ones(2, T, Hq, D, device='cuda') * min(g, 2e6 / (size * D))).to(HALF)
    check(q, k, v, dout, valid, window, sinks)
    # what lies behind a sequence is not a value
    v2 = v.clone()
    v2[1, 250:] = math.inf
    for a, b in zip(run_attention(q, k, v, valid, window, sinks, dout), run_attention(q, k, v2, valid, window, sinks, dout)):
        assert torch.equal(a, b)


@pytest.mark.parametrize('D', [64, 128])
def test_one_large_value_leaves_the_other_tiles_their_digits(D):
    """A value near the type's largest in one late tile: queries that do not see it keep their gradients to the bit."""
    T = 640
    q, k, v, g = (randn(1, T, 1, D) for _ in range(4))
    base = run_attention(q, k, v, None, 100, 0, g)
    far = v.clone()
    far[:, 600, :, 3] = 60000.
    got = run_attention(q, k, far, None, 100, 0, g / 1000)
    ref = run_attention(q, k, v, None, 100, 0, g / 1000)
    # dQ of the query tiles whose keys end before the tile of 600, dK and dV of the key tiles that no query at 600 or later sees
    assert torch.equal(got[1][:, :512], ref[1][:, :512])
    assert torch.equal(got[2][:, :384], ref[2][:, :384]) and torch.equal(got[3][:, :384], ref[3][:, :384])
    check(q, k, far, (g / 1000).to(HALF), window=100)
    assert all(bool(t.isfinite().all()) for t in base + got)


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('scale', [1e-6, 1.0, 30000.0])
def test_ordinary_values_with_any_loss_scale(D, scale):
    T = 300
    q, k, v = (randn(1, T, 2, D) for _ in range(3))
    g = (randn(1, T, 2, D).clamp(-0.5, 0.5) * scale).to(HALF)
    if scale > 1:
        q, k = q / 64, k / 64
        v = v / 64
    check(q, k, v, g)
