"""Blocks that update their arguments in place, captured as CUDA graphs: the caller's arrays hold what the eager loop writes."""
import pytest
import torch

import mxnet_b200 as mx
from mxnet_b200 import nd

from test_cached_op_writes import STATIC, Count, Decode, Sometimes, Step, decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype,D', [(torch.float16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.float16, 20)])
@pytest.mark.parametrize('flags', [{}, STATIC])
@pytest.mark.parametrize('caches,packed', [(1, False), (2, False), (1, True)])
def test_a_captured_decode_step_writes_the_callers_caches(dtype, D, flags, caches, packed):
    block = decode('cuda', dtype, flags, caches, packed, D=D)
    op = block._cached_op
    assert not op._disabled and len(op._graphs) == caches and all(g.placed for g in op._graphs.values())


@pytest.mark.parametrize('flags', [{}, STATIC])
def test_a_captured_fill_writes_the_callers_caches(flags):
    block = Decode(fill=True, sinks=2)
    block.hybridize(**flags)
    draw = lambda *shape: nd.NDArray(torch.randn(*shape, device='cuda').half())   # noqa: E731
    caches = [draw(2, 9, 1, 64) for _ in range(2)]
    want = [c.copy() for c in caches]
    n = nd.NDArray(torch.tensor([12, 3], device='cuda'))
    for i in range(8):
        k, v = draw(2, 12, 1, 64), draw(2, 12, 1, 64)
        got = block(k, k, v, *caches, n)
        nd.contrib.sldwin_cache_fill(k, v, *want, n, sinks=2)
        for a, c, b in zip(got, caches, want):
            assert a._data.data_ptr() == c._data.data_ptr() and torch.equal(c._data, b._data), i
    assert len(block._cached_op._graphs) == 1


@pytest.mark.parametrize('flags', [{}, STATIC])
def test_other_writes(flags):
    block = Count()
    block.hybridize(**flags)
    ctx = mx.gpu(0)
    x, total = nd.array([1., 2., 3.], ctx=ctx), nd.zeros((3,), ctx=ctx)
    for i in range(1, 9):
        twice, part = block(x, total)
        assert total._data.tolist() == [0, 2. * i, 3. * i] and twice._data.tolist() == [0, 4. * i, 6. * i], i
        assert part._data.tolist() == [2. * i, 3. * i]
    assert len(block._cached_op._graphs) == 1
    block = Step()
    block.hybridize(**flags)
    w, m, g = nd.ones((4,), ctx=ctx), nd.zeros((4,), ctx=ctx), nd.ones((4,), ctx=ctx) * 2
    w2, m2 = w.copy(), m.copy()
    for i in range(8):
        block(w, g, m)
        nd.sgd_mom_update(w2, g, m2, lr=0.5, momentum=0.5, out=w2)
        assert torch.equal(w._data, w2._data) and torch.equal(m._data, m2._data), i
    assert len(block._cached_op._graphs) == 1


def test_writes_that_only_the_capture_meets():
    block = Sometimes()
    block.hybridize(**STATIC)
    x, total = nd.ones((2,), ctx=mx.gpu(0)), nd.zeros((2,), ctx=mx.gpu(0))
    block(x, total)
    block(x, total)
    block.writes = True
    for i in range(1, 7):
        assert block(x, total)._data.tolist() == [1. + i] * 2 and total._data.tolist() == [float(i)] * 2
    assert len(block._cached_op._graphs) == 1
