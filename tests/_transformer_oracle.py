"""The language-model operators from their definitions in 64 bits, one element or row at a time, with bounds on the error that
rounding to a type may cause.  ``half(t)``: half a step of type ``t`` relative to the value; ``FP32``: room for the fp32
arithmetic around it (sums of a few hundred products and exponentials of relative error 2^-22)."""
import math

import torch

FP32 = 2e-5


def half(t):
    return torch.finfo(t).eps / 2 if t != torch.float64 else 0.0


def least(t):
    """Half of the smallest step of the type, reached below its normal range; the fp32 arithmetic of the kernels flushes what is
    below 2^-126 to zero, in each of up to 2^10 terms of a few units' weight (2^-113; bf16 has fp32's range)."""
    return max(torch.finfo(t).smallest_normal * torch.finfo(t).eps, 0.0 if t == torch.float64 else 2.0 ** -113)


def rotary(x, positions, inv_freq, interleaved=False, scale=1.0):
    B, T, H, D = x.shape
    R = 2 * inv_freq.shape[0]
    y = x.double().clone()
    pos = positions.double().expand(B, T)
    for i in range(R // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
        t = (pos * float(inv_freq[i].double()))[:, :, None]
        xa, xb = x[..., a].double(), x[..., b].double()
        y[..., a] = scale * (xa * torch.cos(t) - xb * torch.sin(t))
        y[..., b] = scale * (xb * torch.cos(t) + xa * torch.sin(t))
    return y


def sees(i, j, window, sinks):
    return j <= i and (not window or i - j < window or j < sinks)


def visible(n, window, sinks):
    i, j = torch.arange(n)[:, None], torch.arange(n)[None, :]
    s = j <= i
    return s & ((i - j < window) | (j < sinks)) if window else s


def attention(q, k, v, valid=None, window=0, sinks=0, scale=None, dout=None, t=torch.float64):
    """Outputs (out[, dq, dk, dv]) and, beside each, how far a computation in type ``t`` may be from it."""
    B, T, Hq, D = q.shape
    Hk = k.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    e = half(t)
    c = 0.0 if t == torch.float64 else (FP32 if t != torch.float32 else 4e-6)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    bo = torch.zeros_like(out)
    dq, bq = torch.zeros_like(out), torch.zeros_like(out)
    dk, dv, bk, bv = (torch.zeros(B, T, Hk, D, dtype=torch.float64) for _ in range(4))
    for b in range(B):
        n = T if valid is None else max(0, min(T, int(valid[b])))
        if n == 0:
            continue
        mask = visible(n, window, sinks)
        for h in range(Hq):
            g = h * Hk // Hq
            Q, K, V = q[b, :n, h], k[b, :n, g], v[b, :n, g]
            P = (Q @ K.T * scale).masked_fill(~mask, -math.inf).softmax(-1)
            O = P @ V
            out[b, :n, h] = O
            bo[b, :n, h] = (e + c) * (P @ V.abs()) + e * O.abs()
            if dout is not None:
                G = dout[b, :n, h].double().cpu()
                dP = G @ V.T
                delta = (G * O).sum(-1, keepdim=True)
                dS = P * (dP - delta) * scale
                # dS is rounded once; delta comes from the rounded output, dP and the score from fp32 sums
                bs = (e + c) * dS.abs() + P * abs(scale) * (e * (G * O).abs().sum(-1, keepdim=True) + c * (G.abs() @ V.abs().T))
                dq[b, :n, h] = dS @ K
                bq[b, :n, h] = bs @ K.abs()
                dk[b, :n, g] += dS.T @ Q
                bk[b, :n, g] += bs.T @ Q.abs()
                dv[b, :n, g] += P.T @ G
                bv[b, :n, g] += (e + c) * (P.T @ G.abs())
    if dout is None:
        return (out,), (bo + least(t),)
    return (out, dq, dk, dv), (bo + least(t), bq + e * dq.abs() + least(t), bk + e * dk.abs() + least(t), bv + e * dv.abs() + least(t))


def place(p, sinks, capacity):
    return p if p < sinks else sinks + (p - sinks) % (capacity - sinks)


def fill(k, key_cache, valid, sinks):
    """The cache after the prompts' rows were written one after another."""
    c = key_cache.clone()
    for b in range(k.shape[0]):
        for p in range(max(0, min(k.shape[1], int(valid[b]))) if valid is not None else k.shape[1]):
            c[b, place(p, sinks, c.shape[1])] = k[b, p]
    return c


def step(q, k, v, key_cache, value_cache, positions, window=0, sinks=0, scale=None, t=torch.float64):
    """(out, bound, key cache, value cache) after one token."""
    B, Hq, D = q.shape
    Hk, C = k.shape[1], key_cache.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    kc, vc = key_cache.clone(), value_cache.clone()
    out, bound = torch.zeros(B, Hq, D, dtype=torch.float64), torch.zeros(B, Hq, D, dtype=torch.float64)
    e, c = half(t), (0.0 if t == torch.float64 else FP32)
    for b in range(B):
        p = int(positions[b])
        if p < 0:
            continue
        kc[b, place(p, sinks, C)], vc[b, place(p, sinks, C)] = k[b], v[b]
        held = [j for j in range(p + 1) if sees(p, j, window, sinks) and (j < sinks or j > p - (C - sinks))]
        at = [place(j, sinks, C) for j in held]
        for h in range(Hq):
            K, V = kc[b, at, h * Hk // Hq].double().cpu(), vc[b, at, h * Hk // Hq].double().cpu()
            P = (K @ q[b, h].double().cpu() * scale).softmax(0)
            out[b, h] = P @ V
            bound[b, h] = (e + c) * (P @ V.abs()) + e * out[b, h].abs() + least(t)
    return out, bound, kc, vc


def log_probs(x, tokens, k=0, ignore=-1, grads=None, t=torch.float64):
    """Rows [N, V]: (log_prob, entropy[, top, ids][, dx]) and the bounds of the floating ones.  Each log probability is a sum of
    two terms of one sign, (m - x) and log(total), each good to a few 2^-22 relative: the exponentials' arguments carry half a
    step of up to 2^5 and sums of them half a step of their own."""
    x = x.double().cpu()
    tokens = tokens.cpu()
    N, V = x.shape
    r = 0.0 if t == torch.float64 else 3e-6
    m, first = x.max(-1, keepdim=True)
    others = (x - m).exp().scatter(-1, first, 0.0).sum(-1, keepdim=True)      # 64 bits run out too where one token is sure
    lp = (x - m) - torch.log1p(others)
    p = lp.exp()
    plogp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    H = -plogp.sum(-1)
    got = torch.stack([torch.zeros(()).double() if int(tok) == ignore else lp[i, int(tok)] for i, tok in enumerate(tokens)])
    out, bound = [got, H], [r * got.abs(), 2 * r * H + 1e-30]
    ids = None
    if k:
        ids = torch.argsort(-x, dim=-1, stable=True)[:, :k]
        top = lp.gather(-1, ids)
        out += [top, ids]
        bound += [r * top.abs().nan_to_num(posinf=0.0), None]
    if grads is not None:
        gl, ge, gt = (None if g is None else g.double().cpu() for g in grads)
        gl = torch.zeros(N).double() if gl is None else torch.where(tokens == ignore, torch.zeros_like(gl), gl)
        ge = torch.zeros(N).double() if ge is None else ge
        own, mag = torch.zeros_like(x), torch.zeros_like(x)
        for i in range(N):
            if int(tokens[i]) != ignore:
                own[i, int(tokens[i])] += gl[i]
            if gt is not None:
                for j in range(k):
                    own[i, ids[i, j]] += gt[i, j]
        mag = own.abs().sum(-1, keepdim=True)
        tail = torch.where(p > 0, p * (ge[:, None] * (lp + H[:, None])), torch.zeros_like(p))
        dx = own - p * own.sum(-1, keepdim=True) - tail
        size = own.abs() + p * mag + torch.where(p > 0, p * ge.abs()[:, None] * (lp.abs() + H[:, None]), torch.zeros_like(p))
        # p itself is exp of a difference of up to 2^6 in size, rounded to fp32: 2^6 * 2^-24 relative, and the terms' own steps
        out.append(dx)
        bound.append((4 * r) * size + half(t) * dx.abs() + least(t) + (1e-37 if t != torch.float64 else 0.0))
    return out, bound


def check(got, want, bound, what=''):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert bool((torch.isnan(got) == nan).all()), '%s: NaN in other places' % what
    inf = torch.isinf(want)
    assert bool((got[inf] == want[inf]).all()) and bool((torch.isinf(got) == inf).all()), '%s: infinities in other places' % what
    off = (got - want).abs()
    fine = ~(nan | inf)
    bad = (off > bound) & fine
    if bool(bad.any()):
        at = int(torch.where(fine, off / bound.clamp(min=1e-300), torch.zeros_like(off)).argmax())
        raise AssertionError('%s: %d of %d beyond the bound; worst got %.9g, want %.9g, bound %.3g' % (
            what, int(bad.sum()), bad.numel(), got.reshape(-1)[at], want.reshape(-1)[at], bound.reshape(-1)[at]))
