"""CUDA graphs of hybridized training blocks in processes that have done nothing before: whatever a capture needs to find set up,
the block's own eager calls have to have set up."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

TRAIN = """
import sys, threading
import mxnet_b200 as mx
from mxnet_b200 import autograd, gluon, nd
from mxnet_b200.gluon import nn


def train(static, ask):
    ctx = mx.gpu(0)
    net = nn.HybridSequential()
    net.add(nn.Conv2D(16, 3, padding=1, in_channels=8), nn.BatchNorm(in_channels=16), nn.Activation('relu'),
            nn.Dense(32, in_units=16 * 64), nn.Dropout(0.5), nn.Dense(4, in_units=32))
    net.initialize(ctx=ctx)
    net.hybridize(static_alloc=static, static_shape=static)
    trainer = gluon.Trainer(net.collect_params(), 'sgd', {'learning_rate': 0.01})
    x = nd.random.normal(shape=(8, 8, 8, 8), ctx=ctx)
    for _ in range(6):
        with autograd.record():
            y = net(x).square().mean()
        if ask == 'grad':
            ws = [p.data(ctx) for p in net.collect_params().values() if p.grad_req != 'null']
            autograd.grad(y, ws)
        else:
            y.backward()
            trainer.step(1)
        assert y.asnumpy() == y.asnumpy()
    op = net._cached_op
    print('graphs', [(g.fwd is not None, g.bwd is not None) for g in op._graphs.values()], op._disabled)


static, ask, thread = sys.argv[1] == 'static', sys.argv[2], sys.argv[3] == 'thread'
if thread:
    t = threading.Thread(target=train, args=(static, ask))
    t.start()
    t.join()
else:
    train(static, ask)
"""


@pytest.mark.parametrize('how', [('static', 'backward', 'main'), ('plain', 'backward', 'main'), ('static', 'grad', 'main'),
                                 ('static', 'backward', 'thread')])
def test_a_training_block_is_captured(how):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, '-c', TRAIN, *how], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    assert 'graphs [(True, True)] False' in run.stdout and 'capture failed' not in run.stderr, run.stdout + run.stderr[-2000:]
