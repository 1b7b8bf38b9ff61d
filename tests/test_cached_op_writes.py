"""Blocks that update their arguments in place (key/value caches, optimizer states) under ``hybridize()``: a captured block writes
where the caller holds the arrays.  A recorder of tensor operations stands in for CUDA graphs, so that the cached executor's own
code runs on the host; ``test_gpu_cached_op_writes.py`` runs the same blocks in real graphs."""
import contextlib

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from mxnet_b200 import autograd, nd
from mxnet_b200.gluon import HybridBlock, cached_op


class Recorder(TorchDispatchMode):
    def __init__(self, calls):
        super().__init__()
        self.calls, self.before = calls, []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        for a, form in zip(args, func._schema.arguments):
            if form.alias_info is not None and form.alias_info.is_write:
                self.before.append((a, a.clone()))
        out = func(*args, **(kwargs or {}))
        self.calls.append((func, args, kwargs or {}, out))
        return out


class Graph(object):
    """What a captured graph does: the same operations on the same memory, every time."""

    def __init__(self):
        self.calls = []

    def replay(self):
        with torch.no_grad():
            for func, args, kwargs, out in self.calls:
                again = func(*args, **kwargs)
                for old, new in zip(*((o if isinstance(o, (tuple, list)) else (o,)) for o in (out, again))):
                    if isinstance(old, torch.Tensor) and old.untyped_storage().data_ptr() != new.untyped_storage().data_ptr():
                        old.copy_(new)


class Stream(object):
    def __init__(self, device=None):
        pass

    def wait_stream(self, other):
        pass


@contextlib.contextmanager
def capture(graph, pool=None, stream=None):
    recorder = Recorder(graph.calls)
    with recorder:
        yield
    with torch.no_grad():
        for t, was in reversed(recorder.before):        # a capture runs nothing
            t.copy_(was)


@pytest.fixture
def graphs(monkeypatch):
    """``CachedOp`` captures host arrays with the recorder."""
    for name, what in (('Stream', Stream), ('current_stream', lambda device=None: Stream()), ('CUDAGraph', Graph), ('graph', capture),
                       ('graph_pool_handle', lambda: None), ('stream', lambda s: contextlib.nullcontext())):
        monkeypatch.setattr(torch.cuda, name, what)
    monkeypatch.setattr(cached_op.CachedOp, '_use_graphs', lambda self, arrays: not self._disabled)


class Decode(HybridBlock):
    """One token of each sequence over the caches that it is given."""

    def __init__(self, fill=False, **step):
        super().__init__()
        self.fill, self.step = fill, step

    def forward(self, q, k, v, key_cache, value_cache, pos):
        if self.fill:
            return nd.contrib.sldwin_cache_fill(k, v, key_cache, value_cache, pos, sinks=self.step['sinks'])
        return nd.contrib.sldwin_attention_step(q, k, v, key_cache, value_cache, pos, **self.step)


def decode(device, dtype, flags, caches=1, packed=False, tokens=12, D=64):
    """Tokens one by one through a hybridized block and through the operator; returns the block.  ``caches``: sets of caches that
    take turns; ``packed``: keys and values lie in one array."""
    B, C, Hq, Hk = 3, 9, 4, 2
    step = {'window': 6, 'sinks': 2}
    rng = torch.Generator().manual_seed(5)
    draw = lambda *shape: torch.randn(*shape, generator=rng).to(device=device, dtype=dtype)   # noqa: E731

    def places(first):
        if packed:
            kv = nd.NDArray(first.clone())
            return [kv[0], kv[1]]
        return [nd.NDArray(t.clone()) for t in first]
    block = Decode(**step)
    block.hybridize(**flags)
    start = [draw(2, B, C, Hk, D) for _ in range(caches)]
    mine, want = [places(s) for s in start], [places(s) for s in start]
    for i in range(tokens * caches):
        q, k, v = (nd.NDArray(draw(B, h, D)) for h in (Hq, Hk, Hk))
        pos = nd.NDArray(torch.tensor([i // caches, i // caches + 7, -1], device=device))
        out = block(q, k, v, *mine[i % caches], pos)
        ref = nd.contrib.sldwin_attention_step(q, k, v, *want[i % caches], pos, **step)
        assert torch.equal(out._data, ref._data), i
        for a, b in zip(mine[i % caches], want[i % caches]):
            assert torch.equal(a._data, b._data), i
    return block


STATIC = {'static_alloc': True, 'static_shape': True}


@pytest.mark.parametrize('flags', [{}, STATIC])
@pytest.mark.parametrize('caches,packed', [(1, False), (2, False), (1, True), (7, False)])
def test_a_captured_decode_step_writes_the_callers_caches(graphs, flags, caches, packed):
    block = decode('cpu', torch.float32, flags, caches, packed)
    op = block._cached_op
    assert not op._disabled and len(op._graphs) == min(caches, 4) and all(g.placed for g in op._graphs.values())


@pytest.mark.parametrize('flags', [{}, STATIC])
def test_a_captured_fill_returns_the_callers_caches(graphs, flags):
    block = Decode(fill=True, sinks=2)
    block.hybridize(**flags)
    caches = [nd.NDArray(torch.zeros(2, 9, 1, 4)) for _ in range(2)]
    want = [nd.NDArray(torch.zeros(2, 9, 1, 4)) for _ in range(2)]
    n = nd.NDArray(torch.tensor([5, 3]))
    for i in range(8):
        k, v = (nd.NDArray(torch.randn(2, 5, 1, 4)) for _ in range(2))
        got = block(k, k, v, *caches, n)
        nd.contrib.sldwin_cache_fill(k, v, *want, n, sinks=2)
        for a, c, b in zip(got, caches, want):
            assert a._data.data_ptr() == c._data.data_ptr() and torch.equal(a._data, b._data), i
    assert len(block._cached_op._graphs) == 1


class Count(HybridBlock):
    """Adds to one argument with the array's own operators."""

    def forward(self, x, total):
        total += x
        total[0:1] = x[0:1] * 0
        return total * 2, total[1:]


@pytest.mark.parametrize('flags', [{}, STATIC])
def test_writes_of_the_arrays_own_operators(graphs, flags):
    block = Count()
    block.hybridize(**flags)
    x, total = nd.NDArray(torch.tensor([1., 2., 3.])), nd.NDArray(torch.zeros(3))
    for i in range(1, 9):
        twice, part = block(x, total)
        assert total._data.tolist() == [0, 2. * i, 3. * i] and twice._data.tolist() == [0, 4. * i, 6. * i], i
        assert part._data.tolist() == [2. * i, 3. * i] and part._data.data_ptr() == total._data.data_ptr() + 4
    assert len(block._cached_op._graphs) == 1
    block = Count()
    block.hybridize(**flags)
    for i in range(1, 9):                               # under record() such a block is not captured
        with autograd.record():
            block(x, total)
        assert total._data.tolist() == [0, 2. * (8 + i), 3. * (8 + i)], i
    assert len(block._cached_op._graphs) == 0


class Step(HybridBlock):
    def forward(self, weight, grad, mom):
        return nd.sgd_mom_update(weight, grad, mom, lr=0.5, momentum=0.5, out=weight)


@pytest.mark.parametrize('flags', [{}, STATIC])
def test_optimizer_states_as_arguments(graphs, flags):
    block = Step()
    block.hybridize(**flags)
    w, m, g = (nd.NDArray(torch.ones(4) * a) for a in (1, 0, 2))
    w2, m2 = w.copy(), m.copy()
    for i in range(8):
        out = block(w, g, m)
        nd.sgd_mom_update(w2, g, m2, lr=0.5, momentum=0.5, out=w2)
        assert torch.equal(w._data, w2._data) and torch.equal(m._data, m2._data) and torch.equal(out._data, w2._data), i
    assert len(block._cached_op._graphs) == 1


class Sometimes(HybridBlock):
    """Writes only once its own switch is on: the eager calls do not show it."""
    writes = False

    def forward(self, x, total):
        if self.writes:
            total += x
        return x + total


def test_writes_that_only_the_capture_meets(graphs):
    block = Sometimes()
    block.hybridize(**STATIC)
    x, total = nd.NDArray(torch.ones(2)), nd.NDArray(torch.zeros(2))
    block(x, total)
    block(x, total)
    block.writes = True
    for i in range(1, 7):
        assert block(x, total)._data.tolist() == [1. + i] * 2 and total._data.tolist() == [float(i)] * 2
    assert len(block._cached_op._graphs) == 1


class Replaces(HybridBlock):
    """Gives its argument another tensor."""

    def forward(self, x, w):
        x[0] = w[0]
        return x * 1


def test_an_argument_that_gets_another_tensor_keeps_the_block_eager(graphs):
    block = Replaces()
    block.hybridize(**STATIC)
    w = nd.NDArray(torch.tensor([5., 6.]))
    w.attach_grad()
    for _ in range(6):
        x = nd.NDArray(torch.zeros(2))
        with autograd.record():
            block(x, w)
        assert x._data.tolist() == [5., 0.]
    assert len(block._cached_op._graphs) == 0


def test_the_executor_keeps_nobodys_caches(graphs):
    import weakref
    block = Decode(window=6, sinks=2)
    block.hybridize(**STATIC)
    q, k = nd.NDArray(torch.randn(1, 2, 8)), nd.NDArray(torch.randn(1, 1, 8))
    caches = [torch.zeros(1, 9, 1, 8) for _ in range(2)]
    for i in range(5):
        block(q, k, k, *(nd.NDArray(c) for c in caches), nd.NDArray(torch.tensor([i])))
    (graph,) = block._cached_op._graphs.values()
    graph.fwd.calls.clear()                            # a real graph holds addresses
    block._last_args = None
    held = [weakref.ref(c) for c in caches]
    del caches
    assert all(h() is None for h in held)
