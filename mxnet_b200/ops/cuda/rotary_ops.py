"""Rotary position embedding on the sm_100a kernel (``rotary.cu``)."""
import torch

from . import lib, count_launch, check
from ._util import DT, on_device, once, raw_stream

_POS = {torch.float32: 0, torch.float64: 1, torch.int32: 2, torch.int64: 3}


def _run(x, positions, inv_freq, interleaved, scale, backward):
    B, T, H, D = x.shape
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    sb, st, sh, _ = x.stride()
    if positions.dim() == 2:
        pos_sb, pos_st = positions.stride()
    else:
        pos_sb, pos_st = 0, positions.stride(0)
    with on_device(x):
        check(lib().mxb_rotary(DT[x.dtype], x.data_ptr(), y.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), B, T, H, D,
                               2 * inv_freq.shape[0], sb, st, sh, pos_sb, pos_st, _POS[positions.dtype],
                               1 if inv_freq.dtype == torch.float64 else 0, interleaved, scale, backward, raw_stream(x)), 'rotary_embedding')
    count_launch(1)
    return y


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, inv_freq, interleaved, scale):
        ctx.save_for_backward(positions, inv_freq)
        ctx.args = (interleaved, scale)
        return _run(x, positions, inv_freq, interleaved, scale, 0)

    @staticmethod
    @once
    def backward(ctx, dy):
        positions, inv_freq = ctx.saved_tensors
        if dy.stride(3) != 1:
            dy = dy.contiguous()
        return _run(dy, positions, inv_freq, *ctx.args, 1), None, None, None, None


def rotary_embedding(x, positions, inv_freq, interleaved, scale):
    if positions.dtype not in _POS:
        positions = positions.to(torch.float32 if positions.is_floating_point() else torch.int64)
    if inv_freq.dtype not in (torch.float32, torch.float64):
        inv_freq = inv_freq.float()
    inv_freq = inv_freq.contiguous()
    if x.stride(3) != 1:
        x = x.contiguous()
    if x.requires_grad and torch.is_grad_enabled():
        return _Rotary.apply(x, positions, inv_freq, interleaved, scale)
    return _run(x, positions, inv_freq, interleaved, scale, 0)
