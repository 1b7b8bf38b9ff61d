"""A wait that ran out inside a kernel is raised where the host next waits for the device, not only by the operator's next call."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import mxnet_b200 as mx
from mxnet_b200 import engine, nd
from mxnet_b200.ops.cuda import sldwin_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Library(object):
    """Host memory in place of the word that the kernel library allocates."""

    def __init__(self):
        self.word, self.asked = ctypes.c_int(0), 0

    def mxb_report_word(self):
        self.asked += 1
        return ctypes.addressof(self.word)


@pytest.fixture
def library(monkeypatch):
    fake = Library()
    monkeypatch.setattr(sldwin_ops, 'lib', lambda: fake)
    monkeypatch.setattr(sldwin_ops, '_report', [])
    monkeypatch.setattr(engine, '_sync_checks', [])
    return fake


def test_a_report_is_raised_once_at_the_next_wait(library):
    assert sldwin_ops._error_word() == ctypes.addressof(library.word) == sldwin_ops._error_word() and library.asked == 1
    x = nd.zeros((2,))
    for wait in (nd.waitall, x.wait_to_read, sldwin_ops._error_word):
        wait()
        library.word.value = 1
        with pytest.raises(mx.base.MXNetError, match='time-out'):
            wait()
        assert library.word.value == 0
        wait()


def test_the_word_is_there_inside_a_capture(library, monkeypatch):
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    assert sldwin_ops._error_word() == ctypes.addressof(library.word)


def test_a_forked_child_does_not_look_at_the_devices_memory():
    run = subprocess.run([sys.executable, '-c', """
import os
from mxnet_b200 import engine, nd


def check():
    os.kill(os.getpid(), 9)                 # what reading memory would do that the child does not have


engine.at_sync(check)
pid = os.fork()
if pid == 0:
    nd.zeros((2,)).wait_to_read()
    nd.waitall()
    os._exit(0)
print('child', os.waitpid(pid, 0)[1], len(engine._sync_checks))
engine._sync_checks.clear()
"""], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and 'child 0 1' in run.stdout, run.stdout + run.stderr[-2000:]


CAPTURED = """
import torch
import mxnet_b200 as mx
from mxnet_b200 import nd
from mxnet_b200.ops.cuda import sldwin_ops

q = torch.randn(1, 200, 2, 64, device='cuda').half()
fn = mx.ops.get('_contrib_sldwin_attention').fn
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):                 # the word's own memory may be asked for inside a capture
    y = q * 2
    at = sldwin_ops._error_word()
graph.replay()
assert at and bool((y == q * 2).all())
want = fn(q, q, q, window=60)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = fn(q, q, q, window=60)
graph.replay()
a = nd.NDArray(y).asnumpy()
assert (a == want.cpu().numpy()).all()
for wait in (nd.NDArray(y).asnumpy, nd.NDArray(y).wait_to_read, nd.waitall):
    sldwin_ops._report[2].value = 1           # what a kernel writes whose wait ran out
    try:
        wait()
    except mx.base.MXNetError as e:
        assert 'time-out' in str(e)
    else:
        raise SystemExit('nothing raised')
    wait()
print('reported')
sldwin_ops._report[2].value = 1
"""


@pytest.mark.gpu
def test_reports_of_captured_calls():
    run = subprocess.run([sys.executable, '-c', CAPTURED], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and 'reported' in run.stdout, run.stdout + run.stderr[-3000:]
    assert 'time-out' in run.stderr            # the last one, at exit
