"""Sliding-window attention with sinks on the sm_100a kernels: whole sequences (``sldwin_attention.cu``), and the rolling
key/value cache with the attention of single tokens over it (``sldwin_cache.cu``)."""
import ctypes as C

import torch

from . import lib, count_launch, check
from ...base import MXNetError
from ._util import DT, address, on_device, once, raw_stream

_I13, _I16, _I18, _I19 = C.c_int64 * 13, C.c_int64 * 16, C.c_int64 * 18, C.c_int64 * 19      # sizes, then strides


_report = []          # where kernels report a wait that ran out: the word of host memory, its address and its reader


def _error_word():
    """Address of the word; raises what an earlier call reported."""
    if not _report:
        at = lib().mxb_report_word()
        if not at:
            raise RuntimeError('no host memory for the reports of kernels')
        from ... import engine
        word = C.c_int.from_address(at)
        _report[:] = (word, at, word)
        engine.at_sync(_raise_reported)
    if _report[2].value:
        _raise_reported()
    return _report[1]


def _raise_reported():
    if _report[2].value:
        _report[2].value = 0
        raise MXNetError('an earlier call reported a barrier time-out inside its kernel: its results are not valid')


def _rows(t):
    """``t`` as the kernels read it: adjacent channels, no two elements in one place (an expanded axis is written out), and
    where the rows are whole 16-byte units every row on a 16-byte boundary."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
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
    dtype, dev = q.dtype, q.device
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((B, Hq, T), dtype=torch.float32, device=dev) if keep else None
    (q0, q1, q2, _), (k0, k1, k2, _), (v0, v1, v2, _) = q.stride(), k.stride(), v.stride()
    form = _I16(B, T, Hq, k.shape[2], D, window, sinks, q0, q1, q2, k0, k1, k2, v0, v1, v2)
    with on_device(q):
        check(lib().mxb_sldwin_forward(DT[dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), address(valid), out.data_ptr(), address(lse),
                                       form, scale, _error_word(), raw_stream(q)), 'sldwin_attention')
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
    @once
    def backward(ctx, dout):
        q, k, v, valid, out, lse = ctx.saved_tensors
        window, sinks, scale = ctx.args
        B, T, Hq, D = q.shape
        kshape = k.shape
        dtype, dev = q.dtype, q.device
        dout = _rows(dout)
        dq = torch.empty_like(q, memory_format=torch.contiguous_format)
        dk = torch.empty_like(k, memory_format=torch.contiguous_format)
        dv = torch.empty_like(v, memory_format=torch.contiguous_format)
        (q0, q1, q2, _), (k0, k1, k2, _), (v0, v1, v2, _), (g0, g1, g2, _) = q.stride(), k.stride(), v.stride(), dout.stride()
        form = _I19(B, T, Hq, kshape[2], D, window, sinks, q0, q1, q2, k0, k1, k2, v0, v1, v2, g0, g1, g2)
        L, code = lib(), DT[dtype]
        # workspace: rowsum(dO * O), the largest |dO| of each query tile and |V| of each key tile, then key gradients that several
        # blocks sum up
        tiles = (T + 127) // 128
        rows = (B * (Hq * (T + tiles) + kshape[2] * tiles) + 3) // 4 * 4
        parts = L.mxb_sldwin_backward_parts(code, form)
        work = torch.empty(rows + parts, dtype=torch.float32, device=dev)
        at = work.data_ptr()
        with on_device(q):
            check(L.mxb_sldwin_backward(code, q.data_ptr(), k.data_ptr(), v.data_ptr(), address(valid), out.data_ptr(), dout.data_ptr(),
                                        lse.data_ptr(), at, at + 4 * rows if parts else 0, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                        form, scale, _error_word(), raw_stream(q)), 'sldwin_attention backward')
        count_launch(2 + (parts > 0) + (dtype is torch.float16 and D in (64, 128) and 0 < scale < 1e30))
        return dq, dk, dv, None, None, None, None


def attention(q, k, v, valid, window, sinks, scale):
    q, k, v = _rows(q), _rows(k), _rows(v)
    if valid is not None:
        valid = _int32(valid)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _SldwinAttention.apply(q, k, v, valid, window, sinks, scale)
    return _forward(q, k, v, valid, window, sinks, scale, False)[0]


def _int32(valid):
    """Lengths as the kernels read them (real ones are cut, values beyond 32 bits stay beyond every length)."""
    if valid.dtype == torch.int32 and valid.is_contiguous():
        return valid
    # narrow and unsigned types do not hold the bounds below
    valid = valid.double() if valid.is_floating_point() else valid.long()
    return valid.clamp(-1, (1 << 31) - 128).to(torch.int32).contiguous()


def cache_fill(k, v, key_cache, value_cache, valid, sinks):
    B, T, H, D = k.shape
    k, v = _rows(k), _rows(v)
    if valid is not None:
        valid = _int32(valid)
    (k0, k1, k2, _), (v0, v1, v2, _), (a0, a1, a2, _), (b0, b1, b2, _) = k.stride(), v.stride(), key_cache.stride(), value_cache.stride()
    form = _I18(B, T, H, D, key_cache.shape[1], sinks, k0, k1, k2, v0, v1, v2, a0, a1, a2, b0, b1, b2)
    with on_device(k):
        check(lib().mxb_cache_fill(DT[k.dtype], k.data_ptr(), v.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), address(valid),
                                   form, raw_stream(k)), 'sldwin_cache_fill')
    count_launch(1)


def _dense(t):
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def attention_step(q, k, v, key_cache, value_cache, positions, window, sinks, scale):
    B, Hq, D = q.shape
    q, k, v = _dense(q), _dense(k), _dense(v)
    if positions.dtype != torch.int64 or not positions.is_contiguous():
        positions = positions.to(torch.int64).contiguous()
    out = torch.empty_like(q)
    (a0, a1, a2, _), (b0, b1, b2, _) = key_cache.stride(), value_cache.stride()
    form = _I13(B, Hq, k.shape[1], D, key_cache.shape[1], window, sinks, a0, a1, a2, b0, b1, b2)
    with on_device(q):
        check(lib().mxb_sldwin_step(DT[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
                                    positions.data_ptr(), out.data_ptr(), form, scale, raw_stream(q)), 'sldwin_attention_step')
    count_launch(1)
    return out
