"""Sliding-window attention with sinks on the sm_100a kernels: whole sequences (``sldwin_attention.cu``), and the rolling
key/value cache with the attention of single tokens over it (``sldwin_cache.cu``)."""
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import lib, ptr, stream_ptr, count_launch, check
from ._util import dt, on_device

MAX_DIM = 256
_DIMS7, _DIMS6 = C.c_int * 7, C.c_int * 6
_S6, _S12 = C.c_int64 * 6, C.c_int64 * 12


_report = []          # a word of pinned host memory that the kernels set when a wait inside them ran out, and its reader


def _error_word():
    if not _report:
        if torch.cuda.is_current_stream_capturing():
            return C.c_void_p(0)                                  # a capture allows no allocation of host memory
        word = torch.zeros(1, dtype=torch.int32).pin_memory()
        _report.extend((word, C.c_void_p(word.data_ptr()), C.c_int.from_address(word.data_ptr())))
    elif _report[2].value:
        _report[2].value = 0
        raise RuntimeError('an earlier call reported a barrier time-out inside its kernel: its results are not valid')
    return _report[1]


def _rows(t):
    """``t`` as the kernels read it: adjacent channels, no two elements in one place (an expanded axis is written out), and
    where the rows are whole 16-byte units every row on a 16-byte boundary."""
    s0, s1, s2, s3 = t.stride()
    n0, n1, n2, n3 = t.shape
    unit = 16 // t.element_size()
    if s3 == 1 and (s0 > 0 or n0 == 1) and (s1 > 0 or n1 == 1) and (s2 > 0 or n2 == 1):
        if n3 % unit or (t.data_ptr() % 16 == 0 and (s0 % unit == 0 or n0 == 1) and (s1 % unit == 0 or n1 == 1) and
                         (s2 % unit == 0 or n2 == 1)):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _forward(q, k, v, valid, window, sinks, scale, keep):
    B, T, Hq, D = q.shape
    out = torch.empty((B, T, Hq, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, Hq, T), dtype=torch.float32, device=q.device) if keep else None
    dims = _DIMS7(B, T, Hq, k.shape[2], D, window, sinks)
    strides = _S12(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3])
    with on_device(q):
        check(lib().mxb_sldwin_forward(dt(q), ptr(q), ptr(k), ptr(v), ptr(valid), ptr(out), ptr(lse), dims, strides, scale,
                                       _error_word(), stream_ptr(q.device)), 'sldwin_attention')
    count_launch(1)
    return out, lse


class _SldwinAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, valid, window, sinks, scale):
        out, lse = _forward(q, k, v, valid, window, sinks, scale, True)
        ctx.save_for_backward(q, k, v, valid, out, lse)
        ctx.args = (window, sinks, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, valid, out, lse = ctx.saved_tensors
        window, sinks, scale = ctx.args
        B, T, Hq, D = q.shape
        Hk = k.shape[2]
        dout = _rows(dout)
        dq = torch.empty((B, T, Hq, D), dtype=q.dtype, device=q.device)
        dk = torch.empty((B, T, Hk, D), dtype=q.dtype, device=q.device)
        dv = torch.empty((B, T, Hk, D), dtype=q.dtype, device=q.device)
        delta = torch.empty(B * Hq * (T + (T + 127) // 128), dtype=torch.float32, device=q.device)
        dims = _DIMS7(B, T, Hq, Hk, D, window, sinks)
        strides = _S12(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *dout.stride()[:3])
        words = lib().mxb_sldwin_backward_parts(dt(q), dims)      # key gradients that several blocks sum up
        parts = torch.empty(words, dtype=torch.float32, device=q.device) if words else None
        with on_device(q):
            check(lib().mxb_sldwin_backward(dt(q), ptr(q), ptr(k), ptr(v), ptr(valid), ptr(out), ptr(dout), ptr(lse), ptr(delta), ptr(parts),
                                            ptr(dq), ptr(dk), ptr(dv), dims, strides, scale, _error_word(), stream_ptr(q.device)),
                  'sldwin_attention backward')
        count_launch(3 if words else 2)
        return dq, dk, dv, None, None, None, None


def attention(q, k, v, valid, window, sinks, scale):
    q, k, v = _rows(q), _rows(k), _rows(v)
    if valid is not None:
        valid = valid.to(torch.int32).contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _SldwinAttention.apply(q, k, v, valid, window, sinks, scale)
    return _forward(q, k, v, valid, window, sinks, scale, False)[0]


def cache_fill(k, v, key_cache, value_cache, valid, sinks):
    B, T, H, D = k.shape
    k, v = _rows(k), _rows(v)
    if valid is not None:
        valid = valid.to(torch.int32).contiguous()
    dims = _DIMS6(B, T, H, D, key_cache.shape[1], sinks)
    strides = _S12(*k.stride()[:3], *v.stride()[:3], *key_cache.stride()[:3], *value_cache.stride()[:3])
    with on_device(k):
        check(lib().mxb_cache_fill(dt(k), ptr(k), ptr(v), ptr(key_cache), ptr(value_cache), ptr(valid), dims, strides,
                                   stream_ptr(k.device)), 'sldwin_cache_fill')
    count_launch(1)


def attention_step(q, k, v, key_cache, value_cache, positions, window, sinks, scale):
    B, Hq, D = q.shape
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    positions = positions.to(torch.int64).contiguous()
    out = torch.empty((B, Hq, D), dtype=q.dtype, device=q.device)
    dims = _DIMS7(B, Hq, k.shape[1], D, key_cache.shape[1], window, sinks)
    strides = _S6(*key_cache.stride()[:3], *value_cache.stride()[:3])
    with on_device(q):
        check(lib().mxb_sldwin_step(dt(q), ptr(q), ptr(k), ptr(v), ptr(key_cache), ptr(value_cache), ptr(positions), ptr(out), dims,
                                    strides, scale, stream_ptr(q.device)), 'sldwin_attention_step')
    count_launch(1)
    return out
