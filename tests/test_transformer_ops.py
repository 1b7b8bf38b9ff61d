"""Rotary positions, sliding-window attention with sinks, the rolling cache and token log probabilities on host arrays: against
their definitions in 64 bits, their refusals, and their places in the front ends."""
import math

import numpy as np
import pytest
import torch

import mxnet_b200 as mx
from mxnet_b200 import autograd, nd
from mxnet_b200.base import MXNetError

import _transformer_oracle as oracle


def arr(t):
    return nd.NDArray(t)


def randn(*shape, dtype=torch.float64):
    return torch.randn(*shape, dtype=torch.float64).to(dtype)


TINY = 1e-12


# ---------------------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('R', [2, 6, 10])
@pytest.mark.parametrize('per_sample', [False, True])
def test_rotary_against_the_definition(interleaved, R, per_sample):
    x = randn(3, 5, 2, 10)
    pos = torch.randint(-9, 1000000, (3, 5) if per_sample else (5,))
    freq = mx.nd.contrib.rotary_inv_freq(dim=R, dtype='float64')._data
    y = nd.contrib.rotary_embedding(arr(x), arr(pos), arr(freq), interleaved=interleaved, scale=1.25)
    oracle.check(y._data, oracle.rotary(x, pos, freq, interleaved, 1.25), torch.full(x.shape, 1e-9, dtype=torch.float64))


def test_rotary_gradient_is_the_rotation_back():
    x, pos, freq = randn(2, 4, 3, 8), torch.arange(4), torch.tensor([1.0, 0.3], dtype=torch.float64)
    f = lambda t: mx.ops.get('_contrib_rotary_embedding').fn(t, pos, freq, interleaved=True, scale=0.7)   # noqa: E731
    assert torch.autograd.gradcheck(f, x.requires_grad_(True))


@pytest.mark.parametrize('scaling,expect', [
    ('none', lambda i, f, s: f), ('linear', lambda i, f, s: f / s),
    ('ntk', lambda i, f, s: (10000.0 * s ** (16 / 14.0)) ** (-2.0 * i / 16))])
def test_rotary_frequencies(scaling, expect):
    got = mx.npx.rotary_inv_freq(dim=16, scaling=scaling, factor=8.0, dtype='float64').asnumpy()
    want = [expect(i, 10000.0 ** (-2.0 * i / 16), 8.0) for i in range(8)]
    np.testing.assert_allclose(got, want, rtol=1e-12)


def test_rotary_yarn_keeps_fast_pairs_and_interpolates_slow_ones():
    plain = mx.npx.rotary_inv_freq(dim=64, dtype='float64').asnumpy()
    got = mx.npx.rotary_inv_freq(dim=64, scaling='yarn', factor=16.0, original_length=4096, dtype='float64').asnumpy()
    turns = 4096 * plain / (2 * math.pi)
    ratio = got / plain
    # whole pairs bound the ramp: one pair beyond each end is certain
    assert (ratio[turns > 32 * 10000 ** (2 / 64)] == 1).all()
    np.testing.assert_allclose(ratio[turns < 1 / 10000 ** (2 / 64)], 1 / 16.0, rtol=1e-12)
    assert (np.diff(ratio) <= 1e-15).all()


# ------------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize('T,window,sinks', [(1, 0, 0), (7, 1, 0), (7, 1, 9), (9, 3, 1), (9, 0, 2), (9, 20, 0), (12, 4, 4)])
@pytest.mark.parametrize('Hq,Hk', [(2, 2), (6, 2), (3, 1)])
@pytest.mark.parametrize('ragged', [False, True])
def test_attention_against_the_definition(T, window, sinks, Hq, Hk, ragged):
    B, D = 4, 6
    q, k, v, g = randn(B, T, Hq, D), randn(B, T, Hk, D), randn(B, T, Hk, D), randn(B, T, Hq, D)
    valid = torch.tensor([0, 1, T, T + 5]) if ragged else None
    arrays = [arr(t.clone()) for t in (q, k, v)]
    for a in arrays:
        a.attach_grad()
    with autograd.record():
        out = nd.contrib.sldwin_attention(*arrays, *([arr(valid)] if ragged else []), window=window, sinks=sinks)
    out.backward(arr(g))
    want, _ = oracle.attention(q, k, v, valid, window, sinks, None, g)
    for name, got, w in zip(('out', 'dq', 'dk', 'dv'), [out._data] + [a.grad._data for a in arrays], want):
        oracle.check(got, w, torch.full(w.shape, TINY, dtype=torch.float64), name)


def test_attention_ignores_what_lies_behind_a_sequence():
    q, k, v = randn(2, 8, 2, 4), randn(2, 8, 2, 4), randn(2, 8, 2, 4)
    valid = torch.tensor([5, 0])
    clean = nd.contrib.sldwin_attention(arr(q), arr(k), arr(v), arr(valid), window=3)._data.clone()
    for t in (q, k, v):
        t[0, 5:], t[1] = math.nan, math.inf
    again = nd.contrib.sldwin_attention(arr(q), arr(k), arr(v), arr(valid), window=3)._data
    assert bool((clean == again).all()) and not bool(clean[1].any()) and not bool(clean[0, 5:].any())


def test_attention_gradient_against_differences():
    q, k, v = (randn(2, 5, h, 3).requires_grad_(True) for h in (4, 2, 2))
    fn = mx.ops.get('_contrib_sldwin_attention').fn
    assert torch.autograd.gradcheck(lambda *a: fn(*a, torch.tensor([5, 3]), window=2, sinks=1), (q, k, v))


# ----------------------------------------------------------------------------------------------------------- cache
@pytest.mark.parametrize('T,C,sinks', [(1, 1, 0), (5, 8, 2), (8, 8, 2), (20, 8, 2), (20, 3, 2), (3, 8, 5), (23, 7, 0)])
@pytest.mark.parametrize('ragged', [False, True])
def test_cache_fill_is_writing_one_row_after_another(T, C, sinks, ragged):
    B = 4
    k, v, kc, vc = randn(B, T, 2, 3), randn(B, T, 2, 3), randn(B, C, 2, 3), randn(B, C, 2, 3)
    valid = torch.tensor([0, 1, T // 2, T + 3]) if ragged else None
    want = oracle.fill(k, kc, valid, sinks), oracle.fill(v, vc, valid, sinks)
    a, b = arr(kc), arr(vc)
    r = nd.contrib.sldwin_cache_fill(arr(k), arr(v), a, b, *([arr(valid)] if ragged else []), sinks=sinks)
    assert torch.equal(a._data, want[0]) and torch.equal(b._data, want[1])
    assert r[0]._data.data_ptr() == kc.data_ptr() and r[1]._data.data_ptr() == vc.data_ptr()


@pytest.mark.parametrize('C,sinks,window', [(6, 0, 0), (6, 2, 0), (9, 2, 3), (40, 2, 5), (40, 0, 0), (2, 1, 1)])
def test_steps_against_the_definition(C, sinks, window):
    B, Hq, Hk, D = 5, 4, 2, 3
    kc, vc = torch.full((B, C, Hk, D), math.nan, dtype=torch.float64), torch.full((B, C, Hk, D), math.nan, dtype=torch.float64)
    for p in range(17):
        pos = torch.tensor([p, max(0, p - 3), -1, p, p])       # sequence 1 writes position 0 several times
        q, k, v = randn(B, Hq, D), randn(B, Hk, D), randn(B, Hk, D)
        want, _, wk, wv = oracle.step(q, k, v, kc, vc, pos, window, sinks)
        got = nd.contrib.sldwin_attention_step(arr(q), arr(k), arr(v), arr(kc), arr(vc), arr(pos), window=window, sinks=sinks)
        oracle.check(got._data, want, torch.full(want.shape, TINY, dtype=torch.float64))
        assert torch.equal(kc.nan_to_num(nan=7.0), wk.nan_to_num(nan=7.0)) and torch.equal(vc.nan_to_num(nan=7.0), wv.nan_to_num(nan=7.0))


def run_decoder(dev, dtype, npx, bound, T=23, more=9, window=5, sinks=2, D=8, Hq=4, Hk=2, V=50):
    """A prompt through rotation, attention and cache, then tokens one at a time, against the same tokens as one sequence."""
    torch.manual_seed(3)
    B = 2
    n = T + more
    x = {h: torch.randn(B, n, w, D, device=dev).to(dtype) for h, w in (('q', Hq), ('k', Hk), ('v', Hk))}
    head = (torch.randn(Hq * D, V, device=dev) / 4).to(dtype)
    toks = torch.randint(0, V, (B, n), device=dev)
    cls = mx.np.ndarray if npx else nd.NDArray
    ops = mx.npx if npx else nd.contrib
    a = lambda t: cls._from_tensor(t)   # noqa: E731
    freq = ops.rotary_inv_freq(dim=D, scaling='yarn', factor=4.0, original_length=16, ctx=mx.gpu(0) if dev != 'cpu' else mx.cpu())

    def turned(lo, hi):
        pos = a(torch.arange(lo, hi, device=dev))
        return [ops.rotary_embedding(a(x[h][:, lo:hi]), pos, freq) for h in 'qk'] + [a(x['v'][:, lo:hi])]

    def scored(out, lo, hi):
        logits = a((out._data.reshape(B, hi - lo, Hq * D).to(head.dtype)) @ head)
        return ops.token_log_probs(logits, a(toks[:, lo:hi]), topk=3)
    whole = ops.sldwin_attention(*turned(0, n), window=window, sinks=sinks)
    want = scored(whole, 0, n)
    C = sinks + window
    kc, vc = (a(torch.full((B, C, Hk, D), math.nan, device=dev).to(dtype)) for _ in range(2))
    q, k, v = turned(0, T)
    ops.sldwin_cache_fill(k, v, kc, vc, sinks=sinks)
    for p in range(T, n):
        q, k, v = turned(p, p + 1)
        at = a(torch.full((B,), p, device=dev))
        one = lambda t: a(t._data[:, 0])   # noqa: E731
        out = ops.sldwin_attention_step(one(q), one(k), one(v), kc, vc, at, window=window, sinks=sinks)
        err = (out._data.double() - whole._data[:, p].double()).abs().max()
        assert float(err) <= bound, (p, float(err))
        got = scored(a(out._data[:, None]), p, p + 1)
        for u, w in zip(got[:2], want[:2]):
            assert float((u._data[:, 0].double() - w._data[:, p].double()).abs().max()) <= 40 * bound


@pytest.mark.parametrize('npx', [False, True])
def test_a_decoder_step_by_step_is_the_whole_sequence(npx):
    # fp32 sums of at most 8 products in different orders, values of a few units: 1e-5 has two digits to spare
    run_decoder('cpu', torch.float32, npx, 1e-5)


# -------------------------------------------------------------------------------------------------------- log probs
@pytest.mark.parametrize('k', [0, 1, 5])
@pytest.mark.parametrize('V', [5, 37])
def test_log_probs_against_the_definition(k, V):
    x = randn(6, V) * 4
    x[1, ::2] = -math.inf
    x[2] = 0.5                                                   # ties
    x[3, 2] = 60.0                                               # certain
    tok = torch.randint(0, V, (6,))
    tok[0], tok[1], tok[3] = -1, 1, 2
    g = [randn(6), randn(6), randn(6, k) if k else None]
    xs = x.clone().requires_grad_(True)
    out = mx.ops.get('_contrib_token_log_probs').fn(xs, tok, topk=k)
    want, _ = oracle.log_probs(x, tok, k, -1, g)
    oracle.check(out[0], want[0], 1e-12 * want[0].abs(), 'log_prob')
    oracle.check(out[1], want[1], 1e-12 * want[1].abs() + 1e-14, 'entropy')
    if k:
        oracle.check(out[2], want[2], torch.full(want[2].shape, 1e-12, dtype=torch.float64), 'top')
        assert torch.equal(out[3], want[3])
    heads = [(out[0], g[0]), (out[1], g[1])] + ([(out[2].masked_fill(torch.isinf(out[2]), 0.0), g[2])] if k else [])
    gx, = torch.autograd.grad([h for h, _ in heads], xs, [w for _, w in heads])
    fin = torch.isfinite(x)
    ref = want[-1]
    if k:     # alternatives that are ruled out were taken out of the heads above
        g2 = [g[0], g[1], g[2].masked_fill(torch.isinf(want[2]), 0.0)]
        ref = oracle.log_probs(x, tok, k, -1, g2)[0][-1]
    assert float((gx - ref)[fin].abs().max()) < 1e-11 and not bool(gx[~fin].any())


def test_log_probs_of_hopeless_rows():
    x = randn(5, 8)
    x[0], x[1, 3], x[2, 3] = -math.inf, math.nan, math.inf
    tok = torch.tensor([2, 0, 0, 8, -7])
    lp, ent, top, ids = mx.ops.get('_contrib_token_log_probs').fn(x, tok, topk=2)
    assert lp[0] == -math.inf and ent[0] == 0 and (top[0] == -math.inf).all() and ids[0].tolist() == [0, 1]
    assert torch.isnan(lp[1:]).all() and torch.isnan(ent[1:3]).all() and torch.isfinite(ent[3:]).all()
    assert ids[1, 0] == 3 and ids[2, 0] == 3
    assert mx.ops.get('_contrib_token_log_probs').fn(x, tok, ignore_label=8)[0][3] == 0


def test_log_probs_shapes_types_and_gradcheck():
    x = randn(2, 3, 4, dtype=torch.float16)
    lp, ent = nd.contrib.token_log_probs(arr(x), arr(torch.zeros(2, 3)))
    assert lp.shape == (2, 3) and ent.shape == (2, 3) and lp.dtype == np.float32
    lp, ent, top, ids = mx.npx.token_log_probs(mx.np.array(np.ones((4,))), mx.np.ndarray._from_tensor(torch.tensor(2)), topk=4)
    assert lp.shape == () and top.shape == (4,) and ids.asnumpy().tolist() == [0, 1, 2, 3]
    fn = mx.ops.get('_contrib_token_log_probs').fn
    assert torch.autograd.gradcheck(lambda t: fn(t, torch.tensor([1, -1, 3]), topk=2)[:3], randn(3, 6).requires_grad_(True))


# -------------------------------------------------------------------------------------------------------- refusals
def _attention_args(**change):
    a = dict(query=torch.zeros(2, 4, 4, 8), key=torch.zeros(2, 4, 2, 8), value=torch.zeros(2, 4, 2, 8))
    a.update(change)
    return a


@pytest.mark.parametrize('change', [
    dict(query=torch.zeros(2, 4, 3, 8)), dict(query=torch.zeros(2, 5, 4, 8)), dict(key=torch.zeros(2, 4, 2, 7)),
    dict(value=torch.zeros(2, 4, 1, 8)), dict(query=torch.zeros(4, 4, 8)), dict(value=torch.zeros(2, 4, 2, 8).half()),
    dict(window=-1), dict(sinks=-1), dict(window=2.5), dict(valid_length=torch.zeros(3)), dict(value=None),
    dict(query=torch.zeros(2, 4, 4, 8).long(), key=torch.zeros(2, 4, 2, 8).long(), value=torch.zeros(2, 4, 2, 8).long())])
def test_attention_refuses(change):
    a = {k: (nd.NDArray(v) if isinstance(v, torch.Tensor) else v) for k, v in _attention_args(**change).items()}
    with pytest.raises(MXNetError):
        nd.contrib.sldwin_attention(**a)


@pytest.mark.parametrize('change', [
    dict(data=torch.zeros(2, 3, 8)), dict(data=torch.zeros(2, 3, 1, 8).long()), dict(positions=torch.zeros(2)), dict(positions=torch.zeros(3, 2)),
    dict(inv_freq=torch.zeros(5)), dict(inv_freq=torch.zeros(0)), dict(inv_freq=torch.zeros(2, 2)), dict(positions=None),
    dict(inv_freq=torch.zeros(4).long()), dict(positions=torch.zeros(3).bool())])
def test_rotary_refuses(change):
    a = dict(data=torch.zeros(2, 3, 1, 8), positions=torch.zeros(3), inv_freq=torch.zeros(4))
    a.update(change)
    with pytest.raises(MXNetError):
        nd.contrib.rotary_embedding(**{k: (nd.NDArray(v) if isinstance(v, torch.Tensor) else v) for k, v in a.items()})


@pytest.mark.parametrize('attrs', [dict(dim=3), dict(dim=0), dict(base=0), dict(factor=0.5), dict(scaling='other'), dict(dtype='float16'),
                                   dict(scaling='yarn', factor=2.0)])
def test_rotary_frequencies_refuse(attrs):
    with pytest.raises(MXNetError):
        mx.npx.rotary_inv_freq(**attrs)


@pytest.mark.parametrize('change,attrs', [
    (dict(key_cache=torch.zeros(2, 6, 2, 7)), {}), (dict(value_cache=torch.zeros(2, 5, 2, 8)), {}), (dict(key_cache=torch.zeros(3, 6, 2, 8)), {}),
    (dict(key_cache=torch.zeros(2, 6, 2, 8).half()), {}), ({}, dict(sinks=6)), ({}, dict(sinks=-1)),
    (dict(key_cache=torch.zeros(2, 6, 8, 2).transpose(2, 3)), {}), (dict(value_cache=torch.zeros(2, 1, 2, 8).expand(2, 6, 2, 8)), {})])
def test_caches_refuse(change, attrs):
    base = dict(key_cache=torch.zeros(2, 6, 2, 8), value_cache=torch.zeros(2, 6, 2, 8))
    base.update(change)
    caches = {k: nd.NDArray(v) for k, v in base.items()}
    with pytest.raises(MXNetError):
        nd.contrib.sldwin_cache_fill(arr(torch.zeros(2, 4, 2, 8)), arr(torch.zeros(2, 4, 2, 8)), **caches, **attrs)
    with pytest.raises(MXNetError):
        nd.contrib.sldwin_attention_step(arr(torch.zeros(2, 4, 8)), arr(torch.zeros(2, 2, 8)), arr(torch.zeros(2, 2, 8)),
                                         positions=arr(torch.zeros(2)), **caches, **attrs)


def test_caches_refuse_to_be_one_array():
    c = arr(torch.zeros(2, 6, 2, 8))
    with pytest.raises(MXNetError):
        nd.contrib.sldwin_cache_fill(arr(torch.zeros(2, 4, 2, 8)), arr(torch.zeros(2, 4, 2, 8)), c, c)
    with pytest.raises(MXNetError):
        nd.contrib.sldwin_attention_step(arr(torch.zeros(2, 4, 8)), arr(torch.zeros(2, 2, 8)), arr(torch.zeros(2, 2, 8)), c, c,
                                         arr(torch.zeros(2)))


def test_step_and_fill_refuse_to_be_recorded():
    q, k, kc = arr(torch.zeros(2, 4, 8)), arr(torch.zeros(2, 2, 8)), arr(torch.zeros(2, 6, 2, 8))
    q.attach_grad()
    with autograd.record(), pytest.raises(MXNetError):
        nd.contrib.sldwin_attention_step(q, k, k, kc, kc.copy(), arr(torch.zeros(2)))
    k4 = arr(torch.zeros(2, 3, 2, 8))
    k4.attach_grad()
    with autograd.record(), pytest.raises(MXNetError):
        nd.contrib.sldwin_cache_fill(k4, k4, kc, kc.copy())
    with pytest.raises(MXNetError):
        nd.contrib.sldwin_attention_step(q, k, k, kc, kc.copy(), arr(torch.zeros(3)))


@pytest.mark.parametrize('x,tok,attrs', [
    (torch.zeros(3, 4), torch.zeros(4), {}), (torch.zeros(3, 4).long(), torch.zeros(3), {}), (torch.zeros(3, 4), torch.zeros(3), dict(topk=5)),
    (torch.zeros(3, 40), torch.zeros(3), dict(topk=33)), (torch.zeros(3, 4), torch.zeros(3), dict(topk=-1)), (torch.zeros(3, 4), None, {}),
    (torch.zeros(3, 4), torch.zeros(3), dict(topk=1.5))])
def test_log_probs_refuse(x, tok, attrs):
    with pytest.raises(MXNetError):
        nd.contrib.token_log_probs(arr(x), *([arr(tok)] if tok is not None else []), **attrs)


@pytest.mark.parametrize('bad', [math.inf, -math.inf, math.nan])
def test_sizes_that_are_no_numbers_are_refused(bad):
    a = {k: nd.NDArray(v) for k, v in _attention_args().items()}
    for size in ('window', 'sinks'):
        with pytest.raises(MXNetError):
            nd.contrib.sldwin_attention(**a, **{size: bad})


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32, torch.float64])
def test_real_lengths_are_cut(dtype):
    q, k, v = (randn(4, 9, 2, 4) for _ in range(3))
    lengths = torch.tensor([-math.inf, 2.5, 7.0, math.inf]).to(dtype)
    whole = torch.tensor([0, 2, 7, 9])
    got, want = (nd.contrib.sldwin_attention(arr(q), arr(k), arr(v), arr(n), window=3)._data for n in (lengths, whole))
    assert torch.equal(got, want)
    caches = [torch.zeros(2, 4, 5, 2, 4, dtype=torch.float64) for _ in range(2)]
    for c, n in zip(caches, (lengths, whole)):
        nd.contrib.sldwin_cache_fill(arr(k), arr(v), arr(c[0]), arr(c[1]), arr(n), sinks=1)
    assert torch.equal(*caches)


# ------------------------------------------------------------------------------------------------- front ends, empty
def test_empty_arrays():
    z = lambda *s: arr(torch.zeros(*s))   # noqa: E731
    assert nd.contrib.rotary_embedding(z(0, 3, 2, 4), z(3), z(2)).shape == (0, 3, 2, 4)
    assert nd.contrib.sldwin_attention(z(2, 0, 2, 4), z(2, 0, 2, 4), z(2, 0, 2, 4)).shape == (2, 0, 2, 4)
    assert nd.contrib.sldwin_attention_step(z(0, 2, 4), z(0, 2, 4), z(0, 2, 4), z(0, 3, 2, 4), z(0, 3, 2, 4), z(0)).shape == (0, 2, 4)
    assert nd.contrib.token_log_probs(z(0, 5), z(0), topk=2)[2].shape == (0, 2)


def test_symbols_infer_shapes_and_run():
    q, k, v, pos, freq, x, t = (mx.sym.Variable(n) for n in ('q', 'k', 'v', 'pos', 'freq', 'x', 't'))
    r = mx.sym.contrib.rotary_embedding(q, pos, freq, interleaved=True)
    o = mx.sym.contrib.sldwin_attention(r, k, v, window=3, sinks=1)
    assert set(o.list_arguments()) == {'q', 'pos', 'freq', 'k', 'v'}
    again = mx.sym.load_json(o.tojson())
    _, outs, _ = again.infer_shape(q=(2, 5, 4, 8), k=(2, 5, 2, 8), v=(2, 5, 2, 8), pos=(5,), freq=(4,))
    assert outs == [(2, 5, 4, 8)]
    feed = {'q': randn(2, 5, 4, 8, dtype=torch.float32), 'k': randn(2, 5, 2, 8, dtype=torch.float32),
            'v': randn(2, 5, 2, 8, dtype=torch.float32), 'pos': torch.arange(5).float(), 'freq': torch.rand(4)}
    got = again.eval(**{n: arr(a) for n, a in feed.items()})[0]
    turned = nd.contrib.rotary_embedding(arr(feed['q']), arr(feed['pos']), arr(feed['freq']), interleaved=True)
    want = nd.contrib.sldwin_attention(turned, arr(feed['k']), arr(feed['v']), window=3, sinks=1)
    assert torch.equal(got._data, want._data)
    s = mx.sym.contrib.token_log_probs(x, t, topk=2)
    assert len(s.list_outputs()) == 4
    assert s.infer_shape(x=(3, 7), t=(3,))[1] == [(3,), (3,), (3, 2), (3, 2)]


def test_gradient_passes_of_odd_heads():
    """Head gradients of another shape and arrays outside of the graph are refused, no heads at all are no pass; several heads
    and second derivatives are what they were."""
    x = nd.array([[1.0, 2.0], [3.0, 4.0]])
    x.attach_grad()
    with autograd.record():
        y = x * x
    autograd.backward([])
    with pytest.raises(Exception):
        autograd.backward([y], [nd.ones((3, 2))])
    with autograd.record():
        y = x * x
    autograd.backward([y], [nd.ones((2, 2))])
    assert x.grad.asnumpy().tolist() == [[2, 4], [6, 8]]
    with autograd.record():
        y, z = x * x, 3 * x
    g = autograd.grad([y, z], [x], [nd.ones((2, 2)) * 2, nd.ones((2, 2))])[0]
    assert g.asnumpy().tolist() == [[7, 11], [15, 19]]
    with autograd.record():
        y = x * x * x
        first = autograd.grad(y, x, create_graph=True, retain_graph=True)
        second = autograd.grad(first, x)
    assert second.asnumpy().tolist() == [[6, 12], [18, 24]]
    with pytest.raises(Exception):                       # an array outside of the graph
        autograd.grad([nd.ones((2, 2))], [x])
