"""Operators of decoder language models: rotary positions, causal attention over a sliding window with sinks (whole sequences,
and single tokens over a rolling key/value cache), and the log probabilities of given tokens.

They stand beside the reference's transformer helpers (``src/operator/contrib/transformer.cc``: interleaved products and the
``sldwin_atten_*`` family, which leave softmax, causality and caching to the caller) and its ``softmax`` / ``pick`` /
``topk`` chain.  On a GPU fp32, fp16 and bf16 arrays run on the kernels of ``ops/cuda``; other types, host arrays and
``MXNET_B200_KERNELS=0`` run the tensor-library form below, which computes in fp32 (fp64 for fp64 inputs)."""
from __future__ import annotations

import math
import numbers

import torch
from torch.autograd import forward_ad

from .registry import register
from .cuda import logprob_ops, rotary_ops, sldwin_ops
from .. import env
from ..base import MXNetError

_KERNEL_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_MAX_TOP = 32


def _need(ok, what, *args):
    if not ok:
        raise MXNetError(what % args if args else what)


def _kernels(t):
    # forward-mode differentiation runs through the tensor library: the kernels know no tangents
    return t.is_cuda and t.dtype in _KERNEL_TYPES and t.numel() > 0 and env.get('MXNET_B200_KERNELS') and forward_ad._current_level < 0


def _alike(first, second, third):
    """Floating-point arrays of one type on one device."""
    t, dev = first.dtype, first.get_device()
    return t is second.dtype and t is third.dtype and dev == second.get_device() and dev == third.get_device() and t.is_floating_point and \
        (dev >= 0 or first.device == second.device == third.device)


def _plain(t):
    """``t`` outside of its graph."""
    return t.detach() if t.requires_grad else t


def _same(name, first, **others):
    _need(first.is_floating_point(), '%s: floating-point arrays expected, got %s', name, first.dtype)
    for k, t in others.items():
        _need(t.dtype == first.dtype, '%s: %s has type %s, expected %s', name, k, t.dtype, first.dtype)
        _need(t.device == first.device, '%s: %s is on %s, expected %s', name, k, t.device, first.device)


def _whole(name, what, v):
    """``v`` as an int: whole numbers of any type that is not a truth value, real ones without a fraction."""
    if isinstance(v, numbers.Integral) and not isinstance(v, bool):
        return int(v)
    _need(isinstance(v, numbers.Real) and not isinstance(v, bool) and float(v).is_integer(), '%s: %s must be a whole number, got %r', name,
          what, v)
    return int(v)


def _work(t):
    """The type the tensor-library form computes in."""
    return t if t.dtype == torch.float64 else t.float()


# ------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------
@register('_npx_rotary_inv_freq', '_contrib_rotary_inv_freq', inputs=(),
          defaults={'dim': 64, 'base': 10000.0, 'scaling': 'none', 'factor': 1.0, 'original_length': 0, 'fast_turns': 32.0,
                    'slow_turns': 1.0, 'ctx': None, 'dtype': 'float32'})
def rotary_inv_freq(dim=64, base=10000.0, scaling='none', factor=1.0, original_length=0, fast_turns=32.0, slow_turns=1.0, ctx=None,
                    dtype='float32'):
    """Frequencies of :func:`rotary_embedding`: ``dim / 2`` angles per position, ``base ** (-2 i / dim)`` unscaled.

    ``scaling`` stretches them for contexts ``factor`` times as long as the model was trained on:

    * 'linear': every frequency divided by ``factor`` (positions are interpolated);
    * 'ntk': the base raised to ``base * factor ** (dim / (dim - 2))``, so the fastest pair keeps its frequency and the slowest
      one is divided by ``factor``;
    * 'yarn': by parts (the YaRN method) - a pair that turns at least ``fast_turns`` times over ``original_length`` positions is
      kept, one that turns at most ``slow_turns`` times is divided by ``factor``, with a linear ramp over the pairs between.
      (The method's temperature is the ``scale`` of :func:`rotary_embedding`: ``0.1 * log(factor) + 1``.)

    Computed in 64 bits; ``dtype`` is 'float32' or 'float64'."""
    from ..base import to_torch_dtype
    from ..device import current_device
    name = 'rotary_inv_freq'
    dim = _whole(name, 'dim', dim)
    td = to_torch_dtype(dtype)
    _need(dim >= 2 and dim % 2 == 0, '%s: dim must be even and at least 2, got %d', name, dim)
    _need(base > 0 and factor >= 1, '%s: base must be positive and factor at least 1, got %g and %g', name, base, factor)
    _need(scaling in ('none', 'linear', 'ntk', 'yarn'), "%s: scaling is 'none', 'linear', 'ntk' or 'yarn', got %r", name, scaling)
    _need(td in (torch.float32, torch.float64), '%s: dtype is float32 or float64, got %s', name, td)
    if scaling == 'ntk' and dim > 2:
        base = base * factor ** (dim / (dim - 2.0))
    f = [float(base) ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == 'linear':
        f = [x / factor for x in f]
    elif scaling == 'yarn':
        _need(original_length > 0 and fast_turns > slow_turns > 0 and base > 1,
              '%s: yarn needs original_length > 0, fast_turns > slow_turns > 0 and base > 1', name)

        def pair(turns):                         # the (real-valued) pair that makes that many turns over the original length
            return dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(0, math.floor(pair(fast_turns))), min(dim - 1, math.ceil(pair(slow_turns)))     # the ramp may end behind the last pair
        ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3))) for i in range(dim // 2)]
        f = [x * (1 - r) + x / factor * r for x, r in zip(f, ramp)]
    dev = (ctx if ctx is not None else current_device()).torch_device
    return torch.tensor(f, dtype=torch.float64).to(td).to(dev)


def _rotary_fits(data, positions, inv_freq):
    n, at, dev = data.shape, positions.shape, data.get_device()
    return len(n) == 4 and data.is_floating_point() and (at == n[:2] or at == n[1:2]) and inv_freq.dim() == 1 and \
        1 <= inv_freq.shape[0] <= n[3] // 2 and inv_freq.is_floating_point() and not positions.is_complex() and \
        positions.dtype is not torch.bool and positions.get_device() == dev and inv_freq.get_device() == dev and \
        (dev >= 0 or positions.device == data.device == inv_freq.device)


def _rotary_refuse(name, data, positions, inv_freq):
    _need(positions is not None and inv_freq is not None, '%s: data, positions and inv_freq are required', name)
    _need(data.dim() == 4, '%s: data must be (B, T, H, D), got %s', name, tuple(data.shape))
    _need(data.is_floating_point(), '%s: data must be floating point, got %s', name, data.dtype)
    B, T, H, D = data.shape
    _need(tuple(positions.shape) in ((T,), (B, T)), '%s: positions must be (%d,) or (%d, %d), got %s', name, T, B, T, tuple(positions.shape))
    _need(inv_freq.dim() == 1 and 1 <= inv_freq.shape[0] <= D // 2, '%s: inv_freq must be (R / 2,) with 2 <= R <= %d, got %s', name, D,
          tuple(inv_freq.shape))
    _need(inv_freq.is_floating_point() and not positions.is_complex() and positions.dtype != torch.bool,
          '%s: inv_freq must be floating point and positions numbers, got %s and %s', name, inv_freq.dtype, positions.dtype)
    raise MXNetError('%s: arrays on %s, %s and %s, expected one device' % (name, data.device, positions.device, inv_freq.device))


@register('_contrib_rotary_embedding', '_npx_rotary_embedding', inputs=('data', 'positions', 'inv_freq'),
          defaults={'interleaved': False, 'scale': 1.0})
def rotary_embedding(data, positions=None, inv_freq=None, interleaved=False, scale=1.0):
    """Rotates the channels of each head by angles that grow with the position.

    ``data``: (B, T, H, D), any strides over B, T and H.  ``positions``: (T,) for all samples or (B, T), whole or real numbers of
    either sign.  ``inv_freq``: (R / 2,) angles per position, R <= D (:func:`rotary_inv_freq`).  Of the first R channels the
    pairs (i, i + R / 2), or (2 i, 2 i + 1) with ``interleaved``, turn by ``positions * inv_freq[i]`` and are multiplied by
    ``scale``; the channels behind them pass through.  Angles are formed in 64 bits.  Returns a new (B, T, H, D) array;
    differentiable in ``data``."""
    name = 'rotary_embedding'
    if positions is None or inv_freq is None or not _rotary_fits(data, positions, inv_freq):
        _rotary_refuse(name, data, positions, inv_freq)
    B, T, H, D = data.shape
    positions, inv_freq, scale = _plain(positions), _plain(inv_freq), float(scale)
    if _kernels(data) and D <= 1024 and H <= 4096 and B * T < (1 << 30):
        return rotary_ops.rotary_embedding(data, positions, inv_freq, 1 if interleaved else 0, scale)
    R = 2 * inv_freq.shape[0]
    x = _work(data)
    angle = positions.double().unsqueeze(-1) * inv_freq.double()
    cos, sin = (angle.cos() * scale).to(x.dtype).unsqueeze(-2), (angle.sin() * scale).to(x.dtype).unsqueeze(-2)
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., R:]), dim=-1).to(data.dtype)


# ------------------------------------------------------------------------------------------
# sliding-window attention with sinks
# ------------------------------------------------------------------------------------------
def _window_args(name, window, sinks, scale, D):
    if type(window) is not int or type(sinks) is not int:
        window, sinks = _whole(name, 'window', 0 if window is None else window), _whole(name, 'sinks', 0 if sinks is None else sinks)
    if window < 0 or sinks < 0:
        _need(False, '%s: window and sinks must not be negative, got %d and %d', name, window, sinks)
    return window, sinks, 1.0 / math.sqrt(D) if scale is None else float(scale)


def _heads_fit(query, key, value, axes):
    qs, ks = query.shape, key.shape
    return len(qs) == axes and len(ks) == axes and ks == value.shape and qs[0] == ks[0] and (axes == 3 or qs[1] == ks[1]) and \
        qs[-1] == ks[-1] >= 1 and ks[-2] >= 1 and qs[-2] % ks[-2] == 0 and _alike(query, key, value)


def _heads_refuse(name, query, key, value, lead):
    _need(key is not None and value is not None, '%s: query, key and value are required', name)
    form = '(%s, H, D)' % ', '.join(lead)
    n = len(lead) + 2
    _need(query.dim() == n and key.dim() == n, '%s: query and key must be %s, got %s and %s', name, form, tuple(query.shape), tuple(key.shape))
    qs, ks = tuple(query.shape), tuple(key.shape)
    _need(qs[:-2] == ks[:-2] and qs[-1] == ks[-1] and ks == tuple(value.shape), '%s: query, key and value must agree in all but the heads, '
          'key and value in these too, got %s, %s and %s', name, qs, ks, tuple(value.shape))
    _need(ks[-2] >= 1 and qs[-2] % ks[-2] == 0, '%s: %d query heads are not a multiple of %d key heads', name, qs[-2], ks[-2])
    _need(qs[-1] >= 1, '%s: heads have no channels', name)
    _same(name, query, key=key, value=value)
    raise MXNetError('%s: bad arguments' % name)


def _lengths(name, valid_length, B, device):
    if valid_length is not None:
        if valid_length.shape != (B,) or valid_length.device != device:
            _need(tuple(valid_length.shape) in ((B,), (B, 1)), '%s: valid_length must be (%d,), got %s', name, B, tuple(valid_length.shape))
            _need(valid_length.device == device, '%s: valid_length is on %s, expected %s', name, valid_length.device, device)
            valid_length = valid_length.reshape(B)
        valid_length = _plain(valid_length)
    return valid_length


def _cut(valid, T):
    """Lengths as whole numbers from 0 to T (real ones are cut)."""
    return (valid.double() if valid.is_floating_point() else valid.long()).clamp(0, T).long()


def _grouped_softmax(score, seen):
    """Probabilities of ``score`` over the keys that are seen; a row that sees none gets zeros."""
    score = score.masked_fill(~seen, -math.inf)
    top = score.detach().amax(-1, keepdim=True)
    e = (score - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


@register('_contrib_sldwin_attention', '_npx_sldwin_attention', inputs=('query', 'key', 'value', 'valid_length'),
          defaults={'window': 0, 'sinks': 0, 'scale': None})
def sldwin_attention(query, key=None, value=None, valid_length=None, window=0, sinks=0, scale=None):
    """Causal multi-head attention over a sliding window, with a few first tokens that stay visible.

    ``query``: (B, T, Hq, D); ``key``, ``value``: (B, T, Hk, D), Hq a multiple of Hk (query heads ``h * Hk // Hq`` share a key
    head); any strides over B, T and H.  Query i sees key j when ``j <= i`` and ``i - j < window`` or ``j < sinks``; ``window=0``
    sees every ``j <= i``.  ``valid_length``: (B,) numbers of tokens (cut to whole ones in 0 .. T); the rows behind them take no
    part - what they hold does not matter - and their outputs and gradients are 0.  ``scale`` defaults to ``1 / sqrt(D)``.

    A query whose largest score is NaN or +inf gets NaN, one with nothing but -inf gets 0.  A value that is not finite may make
    rows of its sequence NaN that do not see it (0 times infinity).

    Returns (B, T, Hq, D); differentiable in query, key and value.  The (T, T) scores are not stored on the GPU."""
    name = 'sldwin_attention'
    if key is None or value is None or not _heads_fit(query, key, value, 4):
        _heads_refuse(name, query, key, value, ('B', 'T'))
    B, T, Hq, D = query.shape
    Hk = key.shape[2]
    window, sinks, scale = _window_args(name, window, sinks, scale, D)
    valid = _lengths(name, valid_length, B, query.device)
    if _kernels(query) and D <= 256 and T <= (1 << 30):
        # a window of T sees everything, and more sinks than T are T
        return sldwin_ops.attention(query, key, value, valid, min(window, T) or T, min(sinks, T), scale)
    if query.numel() == 0:
        return torch.zeros_like(query) + 0 * query
    G = Hq // Hk
    q = _work(query).reshape(B, T, Hk, G, D).permute(0, 2, 3, 1, 4)
    k, v = _work(key).permute(0, 2, 1, 3).unsqueeze(2), _work(value).permute(0, 2, 1, 3).unsqueeze(2)
    i = torch.arange(T, device=query.device)
    gap = i[:, None] - i[None, :]
    seen = gap >= 0
    if window:
        seen = seen & ((gap < window) | (i < sinks)[None, :])
    seen = seen.expand(B, 1, 1, T, T)
    if valid is not None:
        there = i[None, :] < _cut(valid, T)[:, None]
        seen = seen & there[:, None, None, :, None]
        gone = ~there[:, None, None, :, None]
        q, k, v = q.masked_fill(gone, 0.0), k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)
    out = torch.matmul(_grouped_softmax(torch.matmul(q, k.transpose(-1, -2)) * scale, seen), v)
    return out.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(query.dtype)


def _adjacent(t):
    """Channels next to one another, and no two elements of the array in one place."""
    s, n = t.stride(), t.shape
    return (s[3] == 1 or n[3] == 1) and (s[0] > 0 or n[0] == 1) and (s[1] > 0 or n[1] == 1) and (s[2] > 0 or n[2] == 1)


def _cache_args(name, key_cache, value_cache, B, Hk, D, sinks, like):
    if key_cache is not None and value_cache is not None and key_cache.dim() == 4:
        n = key_cache.shape
        if n[0] == B and n[2] == Hk and n[3] == D and n[1] > sinks and value_cache.shape == n and _alike(like, key_cache, value_cache) and \
                (B == 0 or (_adjacent(key_cache) and _adjacent(value_cache) and key_cache.data_ptr() != value_cache.data_ptr())):
            return
    _need(key_cache is not None and value_cache is not None, '%s: key_cache and value_cache are required', name)
    _need(key_cache.dim() == 4 and tuple(key_cache.shape[:1] + key_cache.shape[2:]) == (B, Hk, D) and value_cache.shape == key_cache.shape,
          '%s: caches must be (%d, C, %d, %d), got %s and %s', name, B, Hk, D, tuple(key_cache.shape), tuple(value_cache.shape))
    _same(name, like, key_cache=key_cache, value_cache=value_cache)
    _need(key_cache.shape[1] > sinks, '%s: a cache of %d rows has no room beside %d sinks', name, key_cache.shape[1], sinks)
    _need(key_cache.data_ptr() != value_cache.data_ptr(), '%s: keys and values need caches of their own', name)
    raise MXNetError('%s: the channels of a cache must be adjacent, and no axis an expanded one' % name)


def _no_gradient(name, *arrays):
    if torch.is_grad_enabled():
        _need(not any(a.requires_grad for a in arrays), '%s updates its caches in place and has no gradient: call it '
              'outside of autograd.record(), or on detached arrays', name)
    if forward_ad._current_level >= 0:
        _need(all(forward_ad.unpack_dual(a).tangent is None for a in arrays), '%s updates its caches in place and has no gradient in '
              'forward mode either', name)


def _written(*arrays):
    for a in arrays:
        if not a.is_inference():
            torch.autograd.graph.increment_version(a)


@register('_contrib_sldwin_cache_fill', '_npx_sldwin_cache_fill', inputs=('key', 'value', 'key_cache', 'value_cache', 'valid_length'),
          nout=2, defaults={'sinks': 0}, mutate=('key_cache', 'value_cache'))
def sldwin_cache_fill(key, value=None, key_cache=None, value_cache=None, valid_length=None, sinks=0):
    """Stores the keys and values of prompts in rolling caches, in place.

    ``key``, ``value``: (B, T, Hk, D) of positions 0 .. T - 1; ``key_cache``, ``value_cache``: (B, C, Hk, D), C > sinks.  A cache
    keeps position p in row p while ``p < sinks`` and in row ``sinks + (p - sinks) % (C - sinks)`` behind: of a prompt longer than
    the cache the sinks and the last ``C - sinks`` positions stay.  ``valid_length``: (B,) lengths of the prompts (clipped to
    0 .. T).  Rows of the caches that no position falls on are left as they were.  The caches may be views of larger arrays but must
    not overlap one another, the keys or the values.  Returns the caches; in a symbol an operator runs only where its outputs lead to
    a result, so that what reads the caches there takes them from here."""
    name = 'sldwin_cache_fill'
    _need(value is not None, '%s: key and value are required', name)
    _need(key.dim() == 4 and value.shape == key.shape, '%s: key and value must be (B, T, H, D), got %s and %s', name, tuple(key.shape),
          tuple(value.shape))
    B, T, Hk, D = key.shape
    sinks = _whole(name, 'sinks', 0 if sinks is None else sinks)
    _need(sinks >= 0, '%s: sinks must not be negative, got %d', name, sinks)
    _same(name, key, value=value)
    _cache_args(name, key_cache, value_cache, B, Hk, D, sinks, key)
    valid = _lengths(name, valid_length, B, key.device)
    _no_gradient(name, key, value, key_cache, value_cache)
    if key.numel() == 0:
        return key_cache, value_cache
    if _kernels(key) and B <= 65535:
        sldwin_ops.cache_fill(key, value, key_cache, value_cache, valid, sinks)
        _written(key_cache, value_cache)
        return key_cache, value_cache
    C = key_cache.shape[1]
    at = torch.arange(T, device=key.device).expand(B, T)
    n = (_cut(valid, T) if valid is not None else at.new_full((B,), T))[:, None]
    # the position that ends up in each row: the last one that falls on it
    row = torch.arange(C, device=key.device).expand(B, C)
    held = torch.where(row < sinks, row, n - 1 - torch.remainder(n - 1 - row, C - sinks))
    keep = ((held < n) & (held >= torch.where(row < sinks, 0, sinks)))[:, :, None, None]
    pick = held.clamp(0, T - 1)[:, :, None, None].expand(B, C, Hk, D)
    with torch.no_grad():
        for src, dst in ((key, key_cache), (value, value_cache)):
            dst.copy_(torch.where(keep, src.gather(1, pick), dst))
    return key_cache, value_cache


@register('_contrib_sldwin_attention_step', '_npx_sldwin_attention_step',
          inputs=('query', 'key', 'value', 'key_cache', 'value_cache', 'positions'),
          defaults={'window': 0, 'sinks': 0, 'scale': None}, mutate=('key_cache', 'value_cache'))
def sldwin_attention_step(query, key=None, value=None, key_cache=None, value_cache=None, positions=None, window=0, sinks=0, scale=None):
    """One new token of each sequence: stores its key and value in the rolling caches, in place, and attends over them.

    ``query``: (B, Hq, D); ``key``, ``value``: (B, Hk, D); ``key_cache``, ``value_cache``: (B, C, Hk, D) in the layout of
    :func:`sldwin_cache_fill` with the same ``sinks``; ``positions``: (B,) position of each new token, all earlier ones of its
    sequence being stored.  A negative position marks a place of the batch without a sequence: its output is 0 and its caches
    are left as they are.  The token sees what :func:`sldwin_attention` with the same ``window`` and ``sinks`` shows it, as far as
    the cache still holds it (the sinks and the last ``C - sinks`` positions); ``window=0`` sees all of that.  The caches must not
    overlap one another or the other arrays.

    A token whose largest score is NaN or +inf gets NaN; a value that is not finite may make the outputs of its sequence NaN (0 times
    infinity).  Returns (B, Hq, D).  Has no gradient.  In a hybridized block the caches may be arguments: a captured graph writes them
    where they are."""
    name = 'sldwin_attention_step'
    _need(positions is not None, '%s: positions are required', name)
    if key is None or value is None or not _heads_fit(query, key, value, 3):
        _heads_refuse(name, query, key, value, ('B',))
    B, Hq, D = query.shape
    Hk = key.shape[1]
    window, sinks, scale = _window_args(name, window, sinks, scale, D)
    _cache_args(name, key_cache, value_cache, B, Hk, D, sinks, query)
    if positions.shape != (B,) or positions.device != query.device:
        _need(tuple(positions.shape) in ((B,), (B, 1)) and positions.device == query.device, '%s: positions must be (%d,) on %s, got %s on %s',
              name, B, query.device, tuple(positions.shape), positions.device)
        positions = positions.reshape(B)
    _no_gradient(name, query, key, value, key_cache, value_cache)
    positions = _plain(positions)
    ring = key_cache.shape[1] - sinks
    window = min(window, ring) or ring
    if _kernels(query) and D <= 256:
        out = sldwin_ops.attention_step(query, key, value, key_cache, value_cache, positions, window, sinks, scale)
        _written(key_cache, value_cache)
        return out
    if query.numel() == 0:
        return torch.zeros_like(query)
    pos = positions.long()[:, None]
    with torch.no_grad():
        row = torch.arange(key_cache.shape[1], device=query.device)[None]
        mine = (row == torch.where(pos < sinks, pos, sinks + torch.remainder(pos - sinks, ring))) & (pos >= 0)
        for src, dst in ((key, key_cache), (value, value_cache)):
            dst.copy_(torch.where(mine[:, :, None, None], src[:, None], dst))
        held = torch.where(row < sinks, row, pos - torch.remainder(pos - row, ring))
        seen = (held <= pos) & ((row < sinks) | ((held >= sinks) & (pos - held < window))) & (pos >= 0)
        q = _work(query).reshape(B, Hk, Hq // Hk, D)
        hide = ~seen[:, None, :, None]                      # rows that were never written may hold anything
        k, v = (_work(c).permute(0, 2, 1, 3).masked_fill(hide, 0.0) for c in (key_cache, value_cache))
        p = _grouped_softmax(torch.matmul(q, k.transpose(-1, -2)) * scale, seen[:, None, None, :])
        return torch.matmul(p, v).reshape(B, Hq, D).to(query.dtype)


# ------------------------------------------------------------------------------------------
# scored tokens
# ------------------------------------------------------------------------------------------
def _log_probs_refuse(name, logits, tokens, k):
    _need(logits.dim() >= 1 and logits.is_floating_point(), '%s: logits must be floating-point (..., V), got %s of %s', name,
          tuple(logits.shape), logits.dtype)
    V, lead = logits.shape[-1], tuple(logits.shape[:-1])
    _need(tuple(tokens.shape) == lead, '%s: tokens must be %s, got %s', name, lead, tuple(tokens.shape))
    _need(V >= 1, '%s: logits have no entries', name)
    _need(0 <= k <= min(V, _MAX_TOP), '%s: topk must be between 0 and %d, got %d', name, min(V, _MAX_TOP), k)
    raise MXNetError('%s: tokens are on %s, expected %s' % (name, tokens.device, logits.device))


@register('_contrib_token_log_probs', '_npx_token_log_probs', inputs=('logits', 'tokens'),
          nout=lambda attrs: 4 if int(attrs.get('topk', 0) or 0) else 2, defaults={'topk': 0, 'ignore_label': -1})
def token_log_probs(logits, tokens=None, topk=0, ignore_label=-1):
    """Log probabilities of given tokens, the entropy of each distribution, and its most probable tokens.

    ``logits``: (..., V); ``tokens``: (...) token numbers.  Returns ``(log_prob, entropy)`` of shape (...) and, with ``topk`` = k
    (at most 32 and V), also ``(top_log_prob, top_token)`` of shape (..., k): the k largest in descending order, equal ones by the
    lower token number, as int64.  Results are fp32 (fp64 for fp64 logits).

    A token equal to ``ignore_label`` is padding: its log probability is 0 and no gradient flows through it.  Any other token
    outside 0 .. V - 1 gives NaN, and a NaN gradient of the row where its log probability has a gradient other than 0.  Tokens with a logit of -inf are ruled out; where all are, every log probability is -inf,
    the entropy 0 and the gradient 0.  A NaN or +inf in a row makes its results NaN (``top_token`` then lists NaN first).

    Differentiable in ``logits`` through log_prob, entropy and top_log_prob.  On a GPU one kernel reads the logits once for all
    outputs and one writes the gradient; probabilities are not stored."""
    name = 'token_log_probs'
    if tokens is None or type(topk) is not int or type(ignore_label) is not int:
        _need(tokens is not None, '%s: logits and tokens are required', name)
        topk, ignore_label = _whole(name, 'topk', 0 if topk is None else topk), _whole(name, 'ignore_label', ignore_label)
    k, ignore = topk, ignore_label
    shape = logits.shape
    if not (len(shape) >= 1 and logits.is_floating_point() and tokens.shape == shape[:-1] and shape[-1] >= 1 and
            0 <= k <= min(shape[-1], _MAX_TOP) and tokens.device == logits.device):
        _log_probs_refuse(name, logits, tokens, k)
    V, lead = shape[-1], shape[:-1]
    flat = len(shape) == 2
    tok, x = _plain(tokens), logits
    if not flat:
        tok, x = tok.reshape(-1), x.reshape(-1, V)
    if tok.dtype != torch.int64:
        tok = tok.long()
    if _kernels(logits) and V < (1 << 31) - 1024:
        res = logprob_ops.token_log_probs(x if x.is_contiguous() else x.contiguous(), tok.contiguous(), k, ignore)
    else:
        res = _token_log_probs(_work(x), tok, k, ignore)
    return res if flat else tuple(r.reshape(lead if i < 2 else lead + (k,)) for i, r in enumerate(res))


class _NoSuchToken(torch.autograd.Function):
    """NaN where a token is not ``known``; so is its gradient where one is asked for, but in rows in which nothing is possible."""
    @staticmethod
    def forward(ctx, x, known, empty):
        ctx.save_for_backward(known, empty)
        ctx.known = known
        return x.masked_fill(~known, math.nan)

    @staticmethod
    def backward(ctx, g):
        known, empty = ctx.saved_tensors
        return torch.where(known, g, torch.zeros_like(g).masked_fill((g != 0) & ~empty, math.nan)), None, None

    @staticmethod
    def jvp(ctx, dx, *_):
        return dx.masked_fill(~ctx.known, math.nan)


def _token_log_probs(x, tok, k, ignore):
    V = x.shape[1]
    bad = (torch.isnan(x) | (x == math.inf)).any(-1, keepdim=True)
    top = x.detach().masked_fill(torch.isnan(x), -math.inf).amax(-1, keepdim=True)
    empty = (top == -math.inf) & ~bad
    shifted = x - torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    out = shifted == -math.inf
    e = shifted.masked_fill(out, 0.0).exp().masked_fill(out, 0.0)
    first = torch.argmax(x.detach().masked_fill(torch.isnan(x), -math.inf), dim=-1, keepdim=True)
    # of the total all but one largest element (which counts 1) are summed: log1p keeps the digits of a sure token
    others = (e - torch.zeros_like(e).scatter(-1, first, 1.0) * e).sum(-1, keepdim=True)
    own = torch.where(empty, torch.ones_like(others), e.gather(-1, first))
    total = own + others
    # log(own) carries the gradient of the largest element and is 0 in value
    log_total = own.log() + torch.log1p(others / own)
    nan = torch.where(bad, torch.full_like(others, math.nan), torch.zeros_like(others))
    logp = shifted - log_total + nan
    p = e / total
    entropy = (log_total - (p * shifted.masked_fill(out, 0.0)).sum(-1, keepdim=True) + nan).masked_fill(empty, 0.0).squeeze(-1)
    known = (tok >= 0) & (tok < V)
    chosen = logp.gather(-1, tok.clamp(0, V - 1)[:, None]).squeeze(-1)
    chosen = _NoSuchToken.apply(chosen, known, empty.squeeze(-1))
    chosen = torch.where(empty.squeeze(-1) & known, torch.full_like(chosen, -math.inf), chosen)
    chosen = torch.where(tok == ignore, torch.zeros_like(chosen), chosen)
    if not k:
        return chosen, entropy
    order = torch.sort(x.detach(), dim=-1, descending=True, stable=True)[1][:, :k]
    best = logp.gather(-1, order)
    return chosen, entropy, torch.where(empty, torch.full_like(best, -math.inf), best), order
