"""Automatic mixed precision and the language-model operators: attention runs in the half type, lengths keep their digits, and
caches are updated where they are."""
import pytest
import torch

import mxnet_b200 as mx
from mxnet_b200 import amp, nd, sym

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


@pytest.fixture(params=['float16', 'bfloat16'])
def half(request):
    amp._reset()
    amp.init(request.param)
    yield getattr(torch, request.param)
    amp._reset()


def draw(device, *shape, dtype=torch.float32):
    return nd.NDArray(torch.randn(*shape).to(device=device, dtype=dtype))


@pytest.mark.parametrize('device', DEVICES)
def test_attention_runs_in_the_half_type(half, device):
    q, k, v = draw(device, 2, 9, 2, 64), draw(device, 2, 9, 1, 64, dtype=half), draw(device, 2, 9, 1, 64)
    want = mx.ops.get('_contrib_sldwin_attention').fn(q._data.to(half), k._data, v._data.to(half), window=4)
    for op in (nd.contrib.sldwin_attention, mx.npx.sldwin_attention):
        got = op(q, k, v, window=4)
        assert got._data.dtype == half and torch.equal(got._data, want)


@pytest.mark.parametrize('device', DEVICES)
def test_lengths_keep_their_digits(half, device):
    T = 4099                                    # neither half type holds 4097
    q = draw(device, 1, T, 1, 4, dtype=half)
    n = nd.NDArray(torch.tensor([4097.], device=device))
    got = nd.contrib.sldwin_attention(q, q, q, n, window=3)
    assert bool(got._data[:, 4096].any()) and not bool(got._data[:, 4097:].any())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('cache', [torch.float32, torch.float16, torch.bfloat16])
def test_caches_are_updated_where_they_are(half, device, cache):
    kc, vc = (nd.NDArray(torch.zeros(2, 7, 1, 64, device=device, dtype=cache)) for _ in range(2))
    k, v = draw(device, 2, 5, 1, 64, dtype=half), draw(device, 2, 5, 1, 64)
    nd.contrib.sldwin_cache_fill(k, v, kc, vc, sinks=1)
    assert torch.equal(kc._data[:, :5], k._data.to(cache)) and torch.equal(vc._data[:, :5], v._data.to(cache))
    q1, k1, v1 = draw(device, 2, 2, 64), draw(device, 2, 1, 64, dtype=half), draw(device, 2, 1, 64)
    at = nd.NDArray(torch.tensor([5, 5], device=device))
    out = nd.contrib.sldwin_attention_step(q1, k1, v1, kc, vc, at, sinks=1)
    assert out._data.dtype == cache and kc._data.dtype == cache
    assert torch.equal(kc._data[:, 5], k1._data.to(cache)) and torch.equal(vc._data[:, 5], v1._data.to(cache))


@pytest.mark.parametrize('listed', [dict(target_precision_ops=['_contrib_sldwin_attention_step', 'sgd_mom_update']),
                                    dict(fp32_ops=['sgd_mom_update'])])
def test_what_is_updated_in_place_is_not_cast_by_any_list(listed):
    amp._reset()
    amp.init('bfloat16', **listed)
    try:
        w, g, m = (nd.NDArray(torch.ones(3, dtype=torch.float32 if 'target_precision_ops' in listed else torch.bfloat16)) for _ in range(3))
        try:
            nd.sgd_mom_update(w, g, m, lr=0.5, momentum=0.5)
        except mx.base.MXNetError:
            pass                                # types that do not go together are refused, not lost
        else:
            assert not bool((m._data == 1).any())
    finally:
        amp._reset()


@pytest.mark.parametrize('target', ['float16', 'bfloat16'])
def test_converted_graphs_leave_lengths_alone(target):
    q, k, v, n = (sym.var(x) for x in ('q', 'k', 'v', 'n'))
    out = amp.convert_symbol(sym.contrib.sldwin_attention(q, k, v, n, window=3), target_dtype=target)
    a = {x: nd.NDArray(torch.randn(1, 4099, 1, 4)) for x in 'qkv'}
    got, = out.eval(n=nd.NDArray(torch.tensor([4097.])), **a)
    assert str(got.dtype) in (target, "<class 'numpy.%s'>" % target) and bool(got._data[:, 4096].any()) and not bool(got._data[:, 4097:].any())
