"""The sm_100a kernels of rotary positions, sliding-window attention with sinks, the rolling cache and token log probabilities,
against their definitions in 64 bits with bounds derived from the roundings each computation makes (``_transformer_oracle.py``)."""
import math

import pytest
import torch

import mxnet_b200 as mx
from mxnet_b200 import autograd, nd
from mxnet_b200.ops import cuda as kernels

import _transformer_oracle as oracle
from test_transformer_ops import run_decoder

pytestmark = pytest.mark.gpu
HALF = [torch.float16, torch.bfloat16]


def dev():
    return torch.device('cuda', 0)


def randn(*shape, dtype):
    return torch.randn(*shape, device=dev()).to(dtype)


def op(name):
    return mx.ops.get('_contrib_' + name).fn


# ---------------------------------------------------------------------------------------------------------- rotary
def rotary_bound(x, want, t):
    """One rounding of the result, and fp32 angles and products: sin and cos to 2^-22 absolute, two products and a sum."""
    return oracle.half(t) * want.abs() + 1e-6 * x.double().cpu().abs().amax(-1, keepdim=True) + oracle.least(t)


@pytest.mark.parametrize('dtype', HALF + [torch.float32])
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('B,T,H,D,R', [(1, 1, 1, 2, 2), (2, 3, 5, 64, 64), (3, 33, 2, 80, 20), (1, 700, 3, 128, 32), (2, 9, 17, 96, 96),
                                       (4, 1, 12, 64, 16), (1, 5, 1, 256, 256), (2, 7, 3, 30, 14)])
def test_rotary(dtype, interleaved, B, T, H, D, R):
    before = kernels.launches()
    x, g = randn(B, T, H, D, dtype=dtype).requires_grad_(True), randn(B, T, H, D, dtype=dtype)
    pos = torch.randint(-5, 1000000, (B, T), device=dev())
    freq = torch.rand(R // 2, device=dev())
    y = op('rotary_embedding')(x, pos, freq, interleaved=interleaved, scale=0.75)
    y.backward(g)
    assert kernels.launches() == before + 2
    want = oracle.rotary(x.detach().cpu(), pos.cpu(), freq.cpu(), interleaved, 0.75)
    back = oracle.rotary(g.cpu(), -pos.cpu(), freq.cpu(), interleaved, 0.75)
    oracle.check(y, want, rotary_bound(x.detach(), want, dtype), 'out')
    oracle.check(x.grad, back, rotary_bound(g, back, dtype), 'grad')


def test_rotary_of_the_widest_heads():
    x = randn(1, 9700, 1, 1024, dtype=torch.bfloat16)             # many tokens for each block, the largest table
    pos, freq = torch.arange(9700, device=dev()), torch.rand(512, device=dev()) ** 4
    got = op('rotary_embedding')(x, pos, freq)
    at = torch.cat([torch.arange(40), torch.arange(4000, 4040), torch.arange(9660, 9700)])
    want = oracle.rotary(x[:, at].cpu(), pos[at].cpu(), freq.cpu())
    oracle.check(got[:, at], want, rotary_bound(x[:, at], want, torch.bfloat16))


@pytest.mark.parametrize('pos_dtype', [torch.int32, torch.int64, torch.float32, torch.float64, torch.int16])
@pytest.mark.parametrize('freq_dtype', [torch.float32, torch.float64])
def test_rotary_takes_views_and_number_types(pos_dtype, freq_dtype):
    qkv = randn(2, 6, 9, 64, dtype=torch.bfloat16)
    freq = torch.rand(16, device=dev(), dtype=freq_dtype)
    pos = torch.arange(12, device=dev())[::2].to(pos_dtype)
    for x in (qkv[:, :, 2:5], qkv[:, 1:].transpose(1, 2)[:, :6, :, :], qkv[:, :, :, 3:61], qkv[:, ::2, ::4].expand(2, 3, 3, 64)[:, :, :, ::2]):
        p = pos[:x.shape[1]] if x.shape[1] <= 6 else torch.arange(x.shape[1], device=dev()).to(pos_dtype)
        want = oracle.rotary(x.cpu(), p.cpu(), freq.cpu()[:x.shape[3] // 2])
        got = op('rotary_embedding')(x, p, freq[:x.shape[3] // 2])
        oracle.check(got, want, rotary_bound(x, want, torch.bfloat16))


# ------------------------------------------------------------------------------------------------------- attention
def run_attention(q, k, v, valid, window, sinks, g, scale=None):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = op('sldwin_attention')(q, k, v, valid, window=window, sinks=sinks, scale=scale)
    grads = torch.autograd.grad(out, (q, k, v), g)
    return (out,) + grads


def check_attention(q, k, v, valid, window, sinks, g, scale=None):
    got = run_attention(q, k, v, valid, window, sinks, g, scale)
    want, bound = oracle.attention(q, k, v, valid, window, sinks, scale, g, t=q.dtype)
    for n, a, w, b in zip(('out', 'dq', 'dk', 'dv'), got, want, bound):
        oracle.check(a, w, b, n)
    return got


@pytest.mark.parametrize('dtype', HALF + [torch.float32])
@pytest.mark.parametrize('D', [64, 128, 40])
@pytest.mark.parametrize('T,window,sinks', [(1, 0, 0), (2, 1, 1), (77, 32, 1), (128, 0, 0), (129, 5, 130), (300, 128, 4), (391, 100, 140),
                                            (513, 0, 0), (640, 1, 0), (530, 257, 3)])
def test_attention(dtype, D, T, window, sinks):
    B, Hq, Hk = 1, 4, 2
    q, k, v, g = (randn(B, T, h, D, dtype=dtype) for h in (Hq, Hk, Hk, Hq))
    check_attention(q, k, v, None, window, sinks, g)


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('Hq,Hk', [(1, 1), (3, 3), (3, 1), (7, 1), (16, 2), (5, 5)])
def test_attention_head_groups(dtype, D, Hq, Hk):
    q, k, v, g = (randn(2, 260, h, D, dtype=dtype) for h in (Hq, Hk, Hk, Hq))
    check_attention(q, k, v, None, 70, 2, g)


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('D', [64, 128, 72])
@pytest.mark.parametrize('window,sinks', [(0, 0), (50, 0), (200, 131)])
def test_attention_ragged_and_what_lies_behind(dtype, D, window, sinks):
    T = 391
    valid = torch.tensor([0, 1, 127, 128, 129, 300, T, T + 9, -4], dtype=torch.int32, device=dev())
    q, k, v, g = (randn(9, T, h, D, dtype=dtype) for h in (2, 1, 1, 2))
    got = check_attention(q, k, v, valid, window, sinks, g)
    behind = (torch.arange(T, device=dev())[None] >= valid[:, None])[:, :, None, None]
    for fill in (math.nan, math.inf, -math.inf):
        again = run_attention(*(t.masked_fill(behind, fill) for t in (q, k, v)), valid, window, sinks, g.masked_fill(behind, fill))
        for n, a, b in zip(('out', 'dq', 'dk', 'dv'), got, again):
            assert torch.equal(a, b), (n, fill)
            assert not bool(b.masked_select(behind.expand_as(b)).any())


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('Hq,Hk,window,sinks', [(3, 3, 0, 0), (4, 2, 70, 3), (3, 3, 129, 65)])
def test_attention_of_many_short_sequences(dtype, Hq, Hk, window, sinks):
    T = 520
    valid = torch.tensor([0, 1, 2, 63, 64, 65, 66, 127, 128, 129, 191, 192, 193, 256, 257, 383, 385, 449, 513, T, T + 1, 300, 320, 500],
                         dtype=torch.int32, device=dev())
    q, k, v, g = (randn(24, T, h, 64, dtype=dtype) for h in (Hq, Hk, Hk, Hq))
    got = check_attention(q, k, v, valid, window, sinks, g)
    behind = (torch.arange(T, device=dev())[None] >= valid[:, None])[:, :, None, None]
    for fill in (math.nan, math.inf):
        again = run_attention(*(t.masked_fill(behind, fill) for t in (q, k, v)), valid, window, sinks, g.masked_fill(behind, fill))
        assert all(torch.equal(a, b) for a, b in zip(got, again)), fill


@pytest.mark.parametrize('D', [64, 128])
def test_attention_of_short_sequences_over_and_over(D):
    """Short walks one after another, without a pause: the loading warp is done before the others have their TMEM."""
    T = 512
    valid = torch.randint(0, T + 1, (16,), device=dev(), dtype=torch.int32)
    q, k, v, g = (randn(16, T, 12, D, dtype=torch.float16) for _ in range(4))
    want = check_attention(q[:4], k[:4], v[:4], valid[:4], 0, 0, g[:4])
    first = run_attention(q, k, v, valid, 0, 0, g)
    assert all(torch.equal(a, b[:4]) for a, b in zip(want[:2], first[:2]))
    same = torch.ones((), dtype=torch.bool, device=dev())
    for _ in range(300):
        for a, b in zip(first, run_attention(q, k, v, valid, 0, 0, g)):
            same &= (a == b).all()
    assert bool(same)


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('Hq,Hk,window,sinks', [(2, 1, 0, 0), (1, 1, 2049, 3), (3, 3, 2048, 130)])
def test_attention_long_walks_of_small_heads(dtype, Hq, Hk, window, sinks):
    q, k, v, g = (randn(1, 2500, h, 64, dtype=dtype) for h in (Hq, Hk, Hk, Hq))
    check_attention(q, k, v, torch.tensor([2390], dtype=torch.int32, device=dev()), window, sinks, g)


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('B,T,Hq,Hk,D,sinks', [(60, 900, 1, 1, 64, 130), (20, 1300, 4, 4, 128, 4), (160, 600, 2, 1, 64, 1)])
def test_attention_with_sinks_seen_by_many_later_tiles(dtype, B, T, Hq, Hk, D, sinks):
    valid = torch.randint(0, T + 1, (B,), device=dev(), dtype=torch.int32)
    valid[:2] = T
    q, k, v, g = (randn(B, T, h, D, dtype=dtype) for h in (Hq, Hk, Hk, Hq))
    check_attention(q, k, v, valid, 64, sinks, g)


@pytest.mark.parametrize('dtype', [torch.uint8, torch.int16, torch.int64, torch.float32, torch.float64])
def test_lengths_of_any_number_type(dtype):
    q, k, v = (randn(3, 140, 2, 64, dtype=torch.float16) for _ in range(3))
    lengths = torch.tensor([0, 97, 140], device=dev())
    want = op('sldwin_attention')(q, k, v, lengths.to(torch.int32), window=33)
    assert torch.equal(op('sldwin_attention')(q, k, v, lengths.to(dtype), window=33), want)
    assert torch.equal(op('sldwin_attention')(q, k, v, lengths.to(dtype).reshape(3, 1), window=33), want)
    if dtype in (torch.int64, torch.float64):      # numbers that 32 bits do not hold are beyond every length, or below 0
        huge = torch.tensor([-(10 ** 12), 97, 10 ** 12], device=dev()).to(dtype)
        assert torch.equal(op('sldwin_attention')(q, k, v, huge, window=33), want)
    caches = [torch.zeros(2, 3, 50, 2, 64, device=dev(), dtype=torch.float16) for _ in range(2)]
    op('sldwin_cache_fill')(k, v, caches[0][0], caches[0][1], lengths.to(torch.int32), sinks=2)
    op('sldwin_cache_fill')(k, v, caches[1][0], caches[1][1], lengths.to(dtype), sinks=2)
    assert torch.equal(*caches)


@pytest.mark.parametrize('dtype', HALF)
def test_lengths_of_half_types(dtype):
    q, k, v = (randn(3, 140, 2, 64, dtype=torch.float16) for _ in range(3))
    lengths = torch.tensor([-math.inf, 97, math.inf], device=dev()).to(dtype)
    want = op('sldwin_attention')(q, k, v, torch.tensor([0, 97, 140], dtype=torch.int32, device=dev()), window=33)
    assert torch.equal(op('sldwin_attention')(q, k, v, lengths, window=33), want)


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('D', [64, 128, 72])
@pytest.mark.parametrize('j', [0, 1, 5, 130, 131, 191])
def test_attention_with_keys_that_are_not_finite(dtype, D, j):
    """A key of NaN makes the rows NaN that see it, one that scores -inf weighs nothing, one that scores +inf makes rows NaN; the
    other rows keep their bits.  Hidden values weigh nothing however large they are."""
    T, window = 300, 140
    q, k, v = (randn(1, T, h, D, dtype=dtype) for h in (2, 1, 1))
    q[..., 0] = q[..., 0].abs() + 0.25
    i = torch.arange(T, device=dev())
    sees = (i >= j) & (i - j < window)
    base = op('sldwin_attention')(q, k, v, window=window)
    large = v.clone()
    large[:, j] = torch.finfo(dtype).max
    got = op('sldwin_attention')(q, k, large, window=window)
    assert torch.equal(got[:, ~sees], base[:, ~sees])
    for x in (math.nan, math.inf):
        bad = k.clone()
        bad[:, j, :, 0] = x
        got = op('sldwin_attention')(q, bad, v, window=window)
        assert torch.equal(got[:, ~sees], base[:, ~sees]) and bool(torch.isnan(got[:, sees]).all()), x
    bad = k.clone()
    bad[:, j, :, 0] = -math.inf
    got = op('sldwin_attention')(q, bad, v, window=window)
    mask = (oracle.visible(T, window, 0) & (i.cpu() != j)[None, :])[None, None]
    P = (torch.einsum('bihd,bjgd->bhij', q.double(), k.double()).cpu() / math.sqrt(D)).masked_fill(~mask, -math.inf).softmax(-1).nan_to_num(nan=0.0)
    V = v.double().cpu()[:, :, 0]
    want = torch.einsum('bhij,bjd->bihd', P, V)
    half = oracle.half(dtype)
    bound = (half + oracle.FP32) * torch.einsum('bhij,bjd->bihd', P, V.abs()) + half * want.abs() + oracle.least(dtype)
    oracle.check(got, want, bound, 'out')


def test_second_derivatives_are_refused():
    x = randn(2, 5, 3, 64, dtype=torch.float16)
    pos, freq = torch.arange(5, device=dev()), torch.rand(4, device=dev())
    tok = torch.zeros(10, dtype=torch.int64, device=dev())
    for f in (lambda a: op('rotary_embedding')(a, pos, freq), lambda a: op('sldwin_attention')(a, a, a),
              lambda a: op('token_log_probs')(a.reshape(10, -1), tok)[0]):
        a = x.clone().requires_grad_(True)
        first, = torch.autograd.grad(f(a).float().square().sum(), a)
        again, = torch.autograd.grad(f(a).float().square().sum(), a, create_graph=True)
        assert torch.equal(first, again)
        with pytest.raises(RuntimeError, match='once_differentiable'):
            again.float().sum().backward()


def test_a_reported_time_out_is_raised_by_the_next_call():
    from mxnet_b200.ops.cuda import sldwin_ops
    q = randn(1, 20, 1, 64, dtype=torch.float16)
    want = op('sldwin_attention')(q, q, q)
    sldwin_ops._report[2].value = 1               # what a kernel writes whose wait ran out
    with pytest.raises(RuntimeError, match='time-out'):
        op('sldwin_attention')(q, q, q)
    assert torch.equal(op('sldwin_attention')(q, q, q), want)


@pytest.mark.parametrize('D', [64, 128, 20])
def test_attention_takes_views(D):
    T, dtype = 200, torch.bfloat16
    qkv = randn(2, T, 8, D, dtype=dtype)
    g = randn(2, T, 4, D, dtype=dtype)
    want = run_attention(*(t.contiguous() for t in (qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:])), None, 60, 3, g)
    heads_first = qkv.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.empty(2 * T * 8 * D + 1, device=dev(), dtype=dtype)[1:].view(2, T, 8, D).copy_(qkv)      # not on a 16-byte boundary
    for base in (qkv, heads_first, odd):
        got = run_attention(base[:, :, :4], base[:, :, 4:6], base[:, :, 6:], None, 60, 3, g.transpose(1, 2).contiguous().transpose(1, 2))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    # one key head for all, given as an expanded view; the gradient of an expanded output
    k1, v1 = qkv[:, :, 4:5], qkv[:, :, 6:7]
    g1 = g[:, :1, :1].expand(2, T, 4, D)
    got = run_attention(qkv[:, :, :4], k1.expand(2, T, 2, D), v1.expand(2, T, 2, D), None, 60, 3, g1)
    ref = run_attention(qkv[:, :, :4].contiguous(), k1.expand(2, T, 2, D).contiguous(), v1.expand(2, T, 2, D).contiguous(), None, 60, 3,
                        g1.contiguous())
    for a, b in zip(got, ref):
        assert torch.equal(a, b)


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('D', [64, 128])
def test_attention_with_large_scores(dtype, D):
    """Rows dominated by one key, far apart in size: the running maximum moves by hundreds from tile to tile."""
    T = 400
    q, k, v, g = (randn(1, T, 2, D, dtype=dtype) for _ in range(4))
    k = (k * torch.linspace(0.1, 12, T, device=dev())[None, :, None, None]).to(dtype)
    q[:, ::3] *= 4
    # the score is a sum of D products of up to 2^7 in size: its fp32 error is up to D 2^-24 of the sum of their absolute
    # values, which moves a probability by as much again
    mag = (torch.einsum('bihd,bjhd->bhij', q.double().abs(), k.double().abs()) / math.sqrt(D)).max()
    room = float(mag) * 2 ** -20
    got = run_attention(q, k, v, None, 150, 4, g)
    want, bound = oracle.attention(q, k, v, None, 150, 4, None, g, t=dtype)
    for n, a, w, b in zip(('out', 'dq', 'dk', 'dv'), got, want, bound):
        oracle.check(a, w, b * (1 + room / oracle.half(dtype)), n)


def test_attention_scale_and_negative_scale():
    q, k, v, g = (randn(1, 150, 2, 64, dtype=torch.float16) for _ in range(4))
    check_attention(q, k, v, None, 40, 1, g, scale=0.3)
    check_attention(q, k, v, None, 40, 1, g, scale=-0.1)
    check_attention(q, k, v, None, 40, 1, g, scale=0.0)


def test_attention_gradient_against_differences():
    q, k, v = (randn(1, 37, h, 64, dtype=torch.float32) for h in (2, 1, 1))
    g = randn(1, 37, 2, 64, dtype=torch.float32)
    got = run_attention(q, k, v, None, 9, 2, g)[1:]
    for i, grad in enumerate(got):
        d = torch.randn_like((q, k, v)[i])
        up, down = [list((q, k, v)) for _ in range(2)]
        up[i], down[i] = up[i] + 1e-3 * d, down[i] - 1e-3 * d
        f = lambda a: (oracle.attention(*a, None, 9, 2)[0][0] * g.double().cpu()).sum()   # noqa: E731
        num, ana = float(f(up) - f(down)) / 2e-3, float((grad.double() * d.double()).sum())
        # third-order term of the difference ~ 1e-6 of the gradient's size, fp32 sums of it ~ 1e-5
        assert abs(num - ana) <= 1e-4 * float(grad.double().norm() * d.double().norm())


@pytest.mark.parametrize('D', [64, 128])
def test_attention_is_repeatable_and_runs_on_other_streams(D):
    q, k, v, g = (randn(2, 500, h, D, dtype=torch.bfloat16) for h in (6, 2, 2, 6))
    want = run_attention(q, k, v, None, 130, 4, g)
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run_attention(q, k, v, None, 130, 4, g))
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(r, want):
            assert torch.equal(a, b)


def test_attention_and_log_probs_in_captured_graphs():
    q, k, v, g = (randn(1, 200, 2, 64, dtype=torch.float16) for _ in range(4))
    x, tok = randn(4, 1000, dtype=torch.float16), torch.arange(4, device=dev())

    def work():
        return run_attention(q, k, v, None, 64, 2, g) + op('token_log_probs')(x, tok, topk=4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((work(), graph))
    for t in (q, k, v, g, x):
        t.copy_(torch.randn_like(t))
    want = [t.clone() for t in work()]
    for outs, graph in graphs:
        graph.replay()
    for outs, graph in graphs:
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


# ----------------------------------------------------------------------------------------------------------- cache
@pytest.mark.parametrize('dtype', HALF + [torch.float32])
@pytest.mark.parametrize('D', [64, 20, 3])
@pytest.mark.parametrize('T,C,sinks', [(1, 1, 0), (70, 128, 3), (70, 33, 3), (300, 33, 32), (16, 128, 20)])
def test_cache_fill(dtype, D, T, C, sinks):
    B = 4
    valid = torch.tensor([0, 1, T // 2, T + 3], device=dev())
    kv = randn(B, T, 4, D, dtype=dtype)
    cache = randn(B, 2, C, 2, D, dtype=dtype)
    for n in (None, valid):
        kc, vc = cache[:, 0].clone(), cache[:, 1].transpose(1, 2).contiguous().transpose(1, 2)
        want = oracle.fill(kv[:, :, :2], kc, n, sinks), oracle.fill(kv[:, :, 2:], vc, n, sinks)
        op('sldwin_cache_fill')(kv[:, :, :2], kv[:, :, 2:], kc, vc, n, sinks=sinks)
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


@pytest.mark.parametrize('dtype', HALF + [torch.float32])
@pytest.mark.parametrize('D', [64, 128, 40])
@pytest.mark.parametrize('Hq,Hk', [(2, 2), (8, 1), (6, 2), (17, 1), (32, 2)])
@pytest.mark.parametrize('C,sinks,window', [(1, 0, 0), (40, 4, 0), (700, 4, 300), (700, 33, 0), (1500, 0, 1499)])
def test_step(dtype, D, Hq, Hk, C, sinks, window):
    pos = torch.tensor([0, 1, sinks, C - 1, C, 3 * C + 7, -1, 10 ** 11 + 1], device=dev())
    B = len(pos)
    q, k, v = (randn(B, h, D, dtype=dtype) for h in (Hq, Hk, Hk))
    kc, vc = randn(B, C, Hk, D, dtype=dtype), randn(B, Hk, C, D, dtype=dtype).transpose(1, 2)
    for b, p in enumerate(pos.tolist()):          # rows that no position has reached yet hold anything
        kc[b, max(p, 0):], vc[b, max(p, 0):] = math.nan, math.inf
    held = pos.clamp(max=3 * C + 7)               # the far position repeats a near one: the oracle walks all positions
    held[-1] = sinks + C + (10 ** 11 + 1 - sinks) % (C - sinks) if C > sinks else 0
    held[-1] += (-(held[-1] - (10 ** 11 + 1))) % (C - sinks)
    want, bound, wk, wv = oracle.step(q, k, v, kc, vc, held.tolist(), window, sinks, t=dtype)
    got = op('sldwin_attention_step')(q, k, v, kc, vc, pos, window=window, sinks=sinks)
    oracle.check(got, want, bound)
    assert torch.equal(kc.nan_to_num(nan=7.), wk.nan_to_num(nan=7.)) and torch.equal(vc.nan_to_num(posinf=7.), wv.nan_to_num(posinf=7.))


def test_step_keeps_sequences_apart_and_replays_in_graphs():
    B, C = 3, 90
    q, k, v = (randn(B, h, 64, dtype=torch.bfloat16) for h in (4, 2, 2))
    kc, vc = randn(B, C, 2, 64, dtype=torch.bfloat16), randn(B, C, 2, 64, dtype=torch.bfloat16)
    pos = torch.tensor([5, 200, -3], dtype=torch.int64, device=dev())
    step = lambda: op('sldwin_attention_step')(q, k, v, kc, vc, pos, window=50, sinks=2)   # noqa: E731
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for p in ([6, 201, 0], [7, 202, 1]):
        pos.copy_(torch.tensor(p))
        for t in (q, k, v):
            t.copy_(torch.randn_like(t))
        want, bound, wk, wv = oracle.step(q, k, v, kc, vc, p, 50, 2, t=torch.bfloat16)
        graph.replay()
        oracle.check(out, want, bound)
        assert torch.equal(kc, wk) and torch.equal(vc, wv)


@pytest.mark.parametrize('npx', [False, True])
@pytest.mark.parametrize('dtype,bound', [(torch.float32, 1e-5), (torch.bfloat16, 6e-2), (torch.float16, 8e-3)])
def test_a_decoder_step_by_step_is_the_whole_sequence(npx, dtype, bound):
    # outputs of up to 4 in size: both sides round probabilities and the output, 4 half steps of 4 in all (bf16: 4 * 4 * 2^-8)
    run_decoder('cuda', dtype, npx, bound)
    run_decoder('cuda', dtype, npx, bound, T=150, more=9, window=140, sinks=3, D=64)


def test_step_of_one_long_sequence():
    """Few key heads and very many keys: the widest clusters."""
    C, D = 70000, 128
    q, k, v = (randn(1, h, D, dtype=torch.bfloat16) for h in (4, 2, 2))
    kc, vc = randn(1, C, 2, D, dtype=torch.bfloat16), randn(1, C, 2, D, dtype=torch.bfloat16)
    for window, pos in ((0, C - 1), (60000, 5 * C + 3), (300, 3 * C)):
        got = op('sldwin_attention_step')(q, k, v, kc, vc, torch.tensor([pos], device=dev()), window=window, sinks=4)
        # the definition on the rows that are seen, in 64 bits
        held = torch.arange(C, device=dev())
        held = torch.where(held < 4, held, pos - (pos - held) % (C - 4))
        seen = (held <= pos) & ((held < 4) | ((held >= 4) & ((pos - held < window) if window else (held >= 0))))
        K, V = kc[0, seen].double().repeat_interleave(2, 1), vc[0, seen].double().repeat_interleave(2, 1)
        P = (torch.einsum('hd,khd->hk', q[0].double(), K) / math.sqrt(D)).softmax(-1)
        want = torch.einsum('hk,khd->hd', P, V).cpu()[None]
        mass = torch.einsum('hk,khd->hd', P, V.abs()).cpu()[None]
        e = oracle.half(torch.bfloat16)
        oracle.check(got, want, (e + oracle.FP32) * mass + e * want.abs())


def test_caches_beyond_two_to_the_31_elements():
    B, C, H, D = 3, 90000, 64, 128                # sample 2 starts at element 1.47e9, its last row lies behind 2^31
    kc, vc = (torch.zeros(B, C, H, D, dtype=torch.float16, device=dev()) for _ in range(2))
    k, v = (randn(B, 100, H, D, dtype=torch.float16) for _ in range(2))
    q1, k1, v1 = (randn(B, H, D, dtype=torch.float16) for _ in range(3))
    op('sldwin_cache_fill')(k, v, kc, vc, sinks=4)
    assert torch.equal(kc[:, :100], k) and torch.equal(vc[:, :100], v)
    kc[:, -100:], vc[:, -100:] = k, v
    got = op('sldwin_attention_step')(q1, k1, v1, kc, vc, torch.full((B,), C - 1, device=dev()), window=60, sinks=4)
    assert torch.equal(kc[:, -1], k1) and torch.equal(vc[:, -1], v1)
    at = [0, 1, 2, 3] + list(range(C - 60, C))
    K, V = kc[:, at].double(), vc[:, at].double()
    P = (torch.einsum('bhd,bkhd->bhk', q1.double(), K) / math.sqrt(D)).softmax(-1)
    want, mass = (torch.einsum('bhk,bkhd->bhd', P, t).cpu() for t in (V, V.abs()))
    e = oracle.half(torch.float16)
    oracle.check(got, want, (e + oracle.FP32) * mass + e * want.abs() + oracle.least(torch.float16))


# -------------------------------------------------------------------------------------------------------- log probs
def check_log_probs(x, tok, k, ignore=-1, grads=True):
    N = x.shape[0]
    g = [torch.randn(N, device=dev()), torch.randn(N, device=dev()), torch.randn(N, k, device=dev()) if k else None] if grads else None
    xs = x.detach().requires_grad_(bool(grads))
    out = op('token_log_probs')(xs, tok, topk=k, ignore_label=ignore)
    want, bound = oracle.log_probs(x, tok, k, ignore, g, t=x.dtype)
    oracle.check(out[0], want[0], bound[0], 'log_prob')
    oracle.check(out[1], want[1], bound[1], 'entropy')
    if k:
        oracle.check(out[2], want[2], bound[2], 'top_log_prob')
        assert torch.equal(out[3].cpu(), want[3])
    if grads:
        dx, = torch.autograd.grad(out[:3] if k else out, xs, g[:3] if k else g[:2])
        oracle.check(dx, want[-1], bound[-1], 'dx')
    return out


@pytest.mark.parametrize('dtype', HALF + [torch.float32])
@pytest.mark.parametrize('V,k', [(1, 1), (2, 0), (7, 7), (33, 32), (1000, 5), (4099, 0), (33278, 20), (131072, 32), (50001, 1)])
def test_log_probs(dtype, V, k):
    x = (torch.randn(6, V, device=dev()) * 3).to(dtype)
    tok = torch.randint(0, V, (6,), device=dev())
    tok[4] = -1
    check_log_probs(x, tok, k)


@pytest.mark.parametrize('dtype', HALF + [torch.float32])
def test_log_probs_ties_masks_and_certain_tokens(dtype):
    V = 5003
    x = (torch.randn(8, V, device=dev()) * 2).to(dtype)
    x[0] = 1.5                                       # all equal
    x[1] = (torch.arange(V, device=dev()) % 7).to(dtype)
    x[2] = torch.linspace(-9, 9, V, device=dev()).to(dtype)       # every element a new maximum
    x[3, 77] = 40.0                                  # almost certain
    x[4] = -math.inf
    x[4, [5, 4000]] = 2.0                            # two choices
    x[5, 100:] = -math.inf
    x[6] = torch.finfo(dtype).min                    # masked by the type's lowest value
    x[6, 9:40] = 1.0
    x[7] = x[2].flip(0)
    tok = torch.tensor([0, 6, V - 1, 77, 4000, 3, 12, 0], device=dev())
    check_log_probs(x, tok, 6)
    check_log_probs(x, tok, 32)
    check_log_probs(x, tok, 0)


def test_log_probs_of_hopeless_rows():
    x = randn(5, 300, dtype=torch.bfloat16)
    x[0], x[1, 3], x[2, 3] = -math.inf, math.nan, math.inf
    x[4, :5] = math.nan
    x[4, 5:] = -math.inf
    tok = torch.tensor([2, 0, 0, 300, -7], device=dev())
    xs = x.requires_grad_(True)
    lp, ent, top, ids = op('token_log_probs')(xs, tok, topk=2)
    assert lp[0] == -math.inf and ent[0] == 0 and (top[0] == -math.inf).all() and ids[0].tolist() == [0, 1]
    assert torch.isnan(lp[1:]).all() and torch.isnan(ent[[1, 2, 4]]).all() and torch.isfinite(ent[3])
    assert ids[1, 0] == 3 and ids[2, 0] == 3 and ids[4].tolist() == [0, 1]
    g, = torch.autograd.grad((lp, ent, top), xs, (torch.ones_like(lp), torch.ones_like(ent), torch.ones_like(top)))
    assert not bool(g[0].any()) and torch.isnan(g[1:3]).any(-1).all() and torch.isnan(g[3]).any()
    lp = op('token_log_probs')(x.detach(), tok, ignore_label=300)[0]
    assert lp[3] == 0


@pytest.mark.parametrize('grads', [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
def test_log_probs_gradient_through_some_outputs(grads):
    x = (torch.randn(3, 777, device=dev()) * 2).to(torch.float16).requires_grad_(True)
    tok = torch.tensor([3, 4, 776], device=dev())
    out = op('token_log_probs')(x, tok, topk=3)
    g = [torch.randn(3, device=dev()), torch.randn(3, device=dev()), torch.randn(3, 3, device=dev())]
    heads = [i for i, use in enumerate(grads) if use]
    dx, = torch.autograd.grad([out[i] for i in heads], x, [g[i] for i in heads])
    want, bound = oracle.log_probs(x.detach(), tok, 3, -1, [t if use else None for t, use in zip(g, grads)], t=torch.float16)
    oracle.check(dx, want[-1], bound[-1])


def test_log_probs_of_views_and_leading_shapes():
    base = (torch.randn(2, 5, 1001, device=dev()) * 3).to(torch.bfloat16)
    tok = torch.randint(0, 1001, (2, 4), device=dev(), dtype=torch.int32)
    for x in (base[:, :-1], base.transpose(0, 1)[:4].transpose(0, 1), base[:, 1:]):
        lp, ent, top, ids = op('token_log_probs')(x, tok, topk=4)
        want, bound = oracle.log_probs(x.reshape(8, -1), tok.reshape(-1), 4, t=torch.bfloat16)
        oracle.check(lp.reshape(-1), want[0], bound[0])
        assert torch.equal(ids.reshape(8, 4).cpu(), want[3])
    odd = torch.empty(1001 * 3 + 1, device=dev(), dtype=torch.bfloat16)[1:].view(3, 1001).copy_(base[0, :3])
    check_log_probs(odd, tok.reshape(-1)[:3].long(), 4)


def test_log_probs_of_many_rows():
    x = (torch.randn(20000, 65, device=dev()) * 3).to(torch.float16)
    tok = torch.randint(0, 65, (20000,), device=dev())
    out = op('token_log_probs')(x, tok, topk=3)
    lp = torch.log_softmax(x.double(), -1)
    want = lp.gather(-1, tok[:, None])[:, 0]
    assert float(((out[0].double() - want).abs() / (1 + want.abs())).max()) < 2e-6
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :3]
    assert torch.equal(out[3], order)


# --------------------------------------------------------------------------------------------------------- refusals
def test_refusals_name_the_operator():
    q = nd.NDArray(torch.zeros(1, 4, 2, 64, device=dev()))
    with pytest.raises(mx.base.MXNetError, match='sldwin_attention'):
        nd.contrib.sldwin_attention(q, nd.NDArray(torch.zeros(1, 4, 2, 64)), q)
    with pytest.raises(mx.base.MXNetError, match='rotary_embedding'):
        nd.contrib.rotary_embedding(q, nd.NDArray(torch.zeros(4)), nd.NDArray(torch.ones(4, device=dev())))
    with pytest.raises(mx.base.MXNetError, match='token_log_probs'):
        nd.contrib.token_log_probs(q, nd.NDArray(torch.zeros(1, 4, 2)))
    q.attach_grad()
    with autograd.record(), pytest.raises(mx.base.MXNetError, match='sldwin_cache_fill'):
        nd.contrib.sldwin_cache_fill(q, q, nd.NDArray(torch.zeros(1, 8, 2, 64, device=dev())), nd.NDArray(torch.zeros(1, 8, 2, 64, device=dev())))


def test_second_derivatives_are_refused_not_wrong():
    x = randn(2, 50, dtype=torch.float32).requires_grad_(True)
    lp, _ = op('token_log_probs')(x, torch.tensor([1, 2], device=dev()))
    g, = torch.autograd.grad(lp.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_a_gradient_pass_of_one_device_runs_on_the_calling_thread():
    import threading
    seen = []

    class Spy(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x * 2

        @staticmethod
        def backward(ctx, g):
            seen.append(threading.get_ident())
            return g * 2
    x = nd.NDArray(torch.ones(3, device=dev()))
    x.attach_grad()
    for ask in (lambda y: y.backward(), lambda y: autograd.grad(y, x, nd.NDArray(torch.ones(3, device=dev())))):
        with autograd.record():
            with torch.enable_grad():
                y = nd.NDArray(Spy.apply(x._data))
        ask(y)
    assert seen == [threading.get_ident()] * 2 and x.grad._data.tolist() == [4.0 / 2] * 3
    assert torch._C._is_multithreading_enabled() if hasattr(torch._C, '_is_multithreading_enabled') else True
