"""Helpers shared by the kernel wrappers."""
import functools

import torch
from torch.autograd.function import once_differentiable

from . import lib, ptr, stream_ptr, count_launch, check

DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def dt(t):
    return DT[t.dtype]


def f32(t):
    """fp32 contiguous view/copy of a small per-channel tensor."""
    return t if (t.dtype == torch.float32 and t.is_contiguous()) else t.float().contiguous()


def require(t, name, numel=None, dtype=None, device=None, shape=None):
    """Validate one kernel operand before its raw pointer crosses the C boundary: the kernels index
    from the sizes they are told, so a mis-sized or misplaced tensor must fail here, in Python."""
    if t is None:
        raise ValueError('%s is required' % name)
    if not t.is_cuda:
        raise ValueError('%s must live on a CUDA device' % name)
    if device is not None and t.device != device:
        raise ValueError('%s is on %s, expected %s' % (name, t.device, device))
    if not t.is_contiguous():
        raise ValueError('%s must be contiguous' % name)
    if dtype is not None and t.dtype != dtype:
        raise ValueError('%s has dtype %s, expected %s' % (name, t.dtype, dtype))
    if numel is not None and t.numel() != numel:
        raise ValueError('%s has %d elements, expected %d' % (name, t.numel(), numel))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError('%s has shape %s, expected %s' % (name, tuple(t.shape), tuple(shape)))
    return t


def job_wide(choice):
    """The autotuning verdict of rank 0 for every rank of a multi-process job: each rank times the candidates itself (so
    all of them reach this point together, after the same work), then adopts rank 0's choice, so that one layer runs the
    same kernel, with the same rounding, on every GPU of the job.  A single process returns its own verdict."""
    from ...parallel import dist
    if not dist.is_initialized() or dist.world_size() < 2:
        return bool(choice)
    flag = torch.tensor([1 if choice else 0], dtype=torch.int32, device='cuda')
    dist.broadcast_(flag, 0)
    return bool(int(flag.item()))


def on_device(t):
    """Context in which the device of ``t`` is the current one (the raw launchers start their kernels there); the caller's
    current device is put back on exit."""
    if t.get_device() == torch._C._cuda_getDevice():
        return _HERE
    return torch.cuda.device(t.device)


def raw_stream(t):
    """Handle of the current stream of the device of ``t``."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def address(t):
    """Address of a tensor's data for a launcher (0 = no tensor)."""
    return 0 if t is None else t.data_ptr()


def once(backward):
    """``backward`` of a Function whose gradient has no gradient: one that is asked for raises.  Without ``create_graph`` nothing
    can ask, and the guard (9 us of host time) stays out."""
    guarded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


class _Here(object):
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return None


_HERE = _Here()
