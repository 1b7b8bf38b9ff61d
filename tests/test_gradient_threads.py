"""The thread that a gradient pass runs on: the same for the eager passes of a device and for the one that is captured."""
import threading
from types import SimpleNamespace

import pytest
import torch

import mxnet_b200 as mx
from mxnet_b200 import _state, autograd, nd


def on(*indexes):
    return [SimpleNamespace(device=torch.device('cuda', i)) for i in indexes]


def stays(scope):
    """Whether passes inside the scope run on the calling thread."""
    with scope:
        return not torch._C._is_multithreading_enabled()


def fresh(monkeypatch):
    monkeypatch.setattr(autograd, '_worked', set())
    monkeypatch.setattr(autograd, '_here', threading.local())


def test_a_captured_pass_runs_where_the_eager_ones_ran(monkeypatch):
    fresh(monkeypatch)
    first, second = torch.device('cuda', 0), torch.device('cuda', 1)
    assert stays(autograd.captured_pass(first))                     # no pass so far: the forward pass ran here
    assert stays(autograd._calling_thread(on(0, 0))) and stays(autograd.captured_pass(first))
    assert not stays(autograd._calling_thread(on(0, 1)))
    assert stays(autograd.captured_pass(first)) and not stays(autograd.captured_pass(second))
    seen = []
    other = threading.Thread(target=lambda: seen.extend([stays(autograd.captured_pass(first)), stays(autograd.captured_pass(second))]))
    other.start()
    other.join()
    assert seen == [False, False]                                   # that thread ran none itself
    assert torch._C._is_multithreading_enabled()


def test_the_setting_is_put_back_after_a_pass_that_raises():
    class Fails(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x * 2

        @staticmethod
        def backward(ctx, g):
            raise ValueError('no gradient today')
    x = torch.ones(2, requires_grad=True)
    for scope in (lambda: autograd.captured_pass(torch.device('cuda', 0)), lambda: autograd._calling_thread(on(0))):
        try:
            with scope():
                Fails.apply(x).sum().backward()
        except ValueError:
            pass
        assert torch._C._is_multithreading_enabled()


def test_a_graph_over_several_devices_keeps_its_workers(monkeypatch):
    fresh(monkeypatch)
    assert stays(autograd._calling_thread(on(0)))
    _state.state.crossed = True
    assert not stays(autograd._calling_thread(on(0)))
    assert stays(autograd._calling_thread(on(0)))                   # the next graph is another one
    nd.ones((2,)).as_in_context(mx.cpu(1))
    with autograd.record():
        nd.ones((2,)).as_in_context(mx.cpu(1))                      # one device by two names
    assert not _state.state.crossed


def test_a_pass_from_a_host_head_may_have_run_on_any_devices_worker(monkeypatch):
    fresh(monkeypatch)
    host = [SimpleNamespace(device=torch.device('cpu'))]
    assert not stays(autograd._calling_thread(on(0, 0) + host)) and stays(autograd.captured_pass(torch.device('cuda', 1)))
    assert stays(autograd._calling_thread(host)) is False and stays(autograd.captured_pass(torch.device('cuda', 1)))
    monkeypatch.setattr(torch.cuda, 'is_initialized', lambda: True)
    monkeypatch.setattr(torch.cuda, 'device_count', lambda: 2)
    autograd._calling_thread(host)
    assert not stays(autograd.captured_pass(torch.device('cuda', 1)))
    assert stays(autograd._calling_thread(on(1))) and stays(autograd.captured_pass(torch.device('cuda', 1)))


@pytest.mark.gpu
def test_a_recorded_copy_between_devices_is_seen():
    seen = []

    class Spy(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x * 2

        @staticmethod
        def backward(ctx, g):
            seen.append(threading.get_ident())
            return g * 2
    x = nd.ones((3,), ctx=mx.gpu(0))
    x.attach_grad()
    spied = lambda a: nd.NDArray(Spy.apply(a._data))                # noqa: E731
    for move in (lambda a: a, lambda a: a.as_in_context(mx.cpu()).as_in_context(mx.gpu(0)), lambda a: a.copyto(mx.cpu()).copyto(mx.gpu(0)),
                 lambda a: a):
        with autograd.record():
            with torch.enable_grad():
                y = move(spied(x)) * 3
        y.backward()
        assert x.grad._data.tolist() == [6.] * 3
    here = threading.get_ident()
    assert [s == here for s in seen] == [True, False, False, True]
