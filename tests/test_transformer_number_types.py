"""Whole-number arguments of the language-model operators, of any number type."""
import numpy as np
import pytest
import torch

import mxnet_b200 as mx
from mxnet_b200 import nd


def calls(number):
    rng = torch.Generator().manual_seed(1)
    q = nd.NDArray(torch.randn(1, 5, 2, 4, generator=rng))
    one = nd.NDArray(q._data[:, 0].clone())
    caches = [nd.NDArray(torch.zeros(1, 6, 2, 4)) for _ in range(2)]
    yield nd.contrib.sldwin_attention(q, q, q, window=number(3), sinks=number(1))
    yield from nd.contrib.sldwin_cache_fill(q, q, *caches, sinks=number(1))
    yield nd.contrib.sldwin_attention_step(one, one, one, *caches, nd.NDArray(torch.tensor([5])), window=number(3), sinks=number(1))
    yield from nd.contrib.token_log_probs(one, nd.NDArray(torch.tensor([[3, 0]])), topk=number(3), ignore_label=number(3))
    yield mx.npx.rotary_inv_freq(dim=number(4))


@pytest.mark.parametrize('number', [np.int64, np.int32, np.int8, np.uint8, np.float32, np.float64, np.float16, float])
def test_number_types(number):
    for a, b in zip(calls(number), calls(int)):
        assert torch.equal(a._data, b._data)


@pytest.mark.parametrize('bad', [True, np.bool_(True), 2.5, np.float32(2.5), '3', np.array([1, 2]), float('inf'), np.float32('nan'), 1 + 0j])
def test_what_is_not_a_whole_number_is_refused(bad):
    q = nd.NDArray(torch.zeros(1, 5, 2, 4))
    with pytest.raises(mx.base.MXNetError, match='whole number'):
        nd.contrib.sldwin_attention(q, q, q, window=bad)
    with pytest.raises(mx.base.MXNetError, match='whole number'):
        nd.contrib.token_log_probs(q, nd.NDArray(torch.zeros(1, 5, 2)), topk=bad)
    with pytest.raises(mx.base.MXNetError, match='whole number'):
        mx.npx.rotary_inv_freq(dim=bad)
