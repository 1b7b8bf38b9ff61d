"""A kernel's setup on a device is over before any thread goes on to launch it (``ops/cuda/device_setup.h``)."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "device_setup.h"
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>

int main() {
  for (int round = 0; round < 20; ++round) {
    unsigned long long seen = 0;
    std::atomic<int> ready[2] = {{0}, {0}}, early{0}, arrived{0};
    std::vector<std::thread> threads;
    for (int i = 0; i < 8; ++i)
      threads.emplace_back([&, i] {
        const int device = i & 1;
        ++arrived;
        while (arrived < 8) {}
        if (mxb::FirstOnDevice first{&seen, device}) {
          std::this_thread::sleep_for(std::chrono::milliseconds(2));
          ready[device] = 1;
        }
        if (!ready[device]) ++early;             // launched before the setup
      });
    for (auto& t : threads) t.join();
    if (early || seen != 3) { std::printf("%d early, seen %llx\n", early.load(), seen); return 1; }
  }
  unsigned long long seen = 0;
  int calls = 0;
  auto launch = [&](int code) {
    if (mxb::FirstOnDevice first{&seen, 5}) {
      ++calls;
      if (int c = first.take(code)) return c;
    }
    return 0;
  };
  if (launch(7) != 7 || launch(7) != 7 || launch(0) != 0 || launch(7) != 0 || calls != 3 || seen != 32) return 2;
  std::printf("all checks passed\n");
  return 0;
}
"""


@pytest.mark.skipif(shutil.which('g++') is None, reason='needs a C++ compiler')
@pytest.mark.parametrize('flags', [[], ['-fsanitize=thread']])
def test_no_thread_launches_before_the_setup(tmp_path, flags):
    src, exe = tmp_path / 'setup.cc', str(tmp_path / 'setup')
    src.write_text(PROGRAM)
    r = subprocess.run(['g++', '-std=c++17', '-O1', '-g', '-pthread', '-I', os.path.join(ROOT, 'mxnet_b200', 'ops', 'cuda')] + flags +
                       [str(src), '-o', exe], capture_output=True, text=True)
    if r.returncode != 0 and ('sanitizer' in r.stderr or 'cannot find -l' in r.stderr):
        pytest.skip('sanitizer runtime not installed')
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and 'all checks passed' in r.stdout, r.stdout + r.stderr[-3000:]
    assert 'WARNING: ThreadSanitizer' not in r.stderr


def test_no_thread_gets_the_library_before_its_prototypes(monkeypatch):
    import threading
    import time
    import types
    from mxnet_b200.ops import cuda
    from mxnet_b200.ops.cuda import _signatures

    def declare(library):
        time.sleep(0.05)
        library.declared = True
    made, seen, start = [], [], threading.Barrier(6)

    def load(path):
        made.append(types.SimpleNamespace(declared=False))
        return made[-1]
    monkeypatch.setattr(cuda, '_lib', None)
    monkeypatch.setattr(cuda, 'LIB_PATH', __file__)
    monkeypatch.setattr(cuda.ctypes, 'CDLL', load)
    monkeypatch.setattr(_signatures, 'declare', declare)

    def call():
        start.wait()
        seen.append(cuda.lib().declared)
        time.sleep(0.01)
        seen.append(cuda.lib().declared)
    threads = [threading.Thread(target=call) for _ in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert seen == [True] * 12 and len(made) == 1


FIRST_CALLS = """
import threading
import torch
import mxnet_b200 as mx

fns = [mx.ops.get('_contrib_' + n).fn for n in ('sldwin_attention', 'sldwin_attention_step')]
q, g = torch.randn(2, 300, 4, 128, device='cuda').half(), torch.randn(2, 300, 4, 128, device='cuda').half()
cache = [torch.zeros(1, 70000, 1, 128, device='cuda', dtype=torch.half) for _ in range(8)]
torch.cuda.synchronize()
start, out, errors = threading.Barrier(8), [None] * 8, []


def call(i):
    try:
        a = q.clone().requires_grad_(True)
        start.wait()
        y = fns[0](a, a, a, window=100)
        d, = torch.autograd.grad(y, a, g)
        s = fns[1](q[:1, 0, :1], q[:1, 0, :1], q[:1, 0, :1], cache[i], torch.zeros_like(cache[i]), torch.tensor([69999], device='cuda'))
        torch.cuda.current_stream().synchronize()
        out[i] = (y.detach(), d, s)
    except Exception as e:
        errors.append(e)


threads = [threading.Thread(target=call, args=(i,)) for i in range(8)]
for t in threads:
    t.start()
for t in threads:
    t.join()
assert not errors, errors
assert all(torch.equal(a, b) for o in out[1:] for a, b in zip(o, out[0]))
print('all alike')
"""


@pytest.mark.gpu
def test_first_calls_of_many_threads():
    run = subprocess.run([sys.executable, '-c', FIRST_CALLS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and 'all alike' in run.stdout, run.stdout + run.stderr[-3000:]
