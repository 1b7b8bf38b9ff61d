"""Tokens outside of the vocabulary: NaN log probabilities, whose gradients poison a row only where they are asked for."""
import math

import pytest
import torch

import _transformer_oracle as oracle
import mxnet_b200 as mx

V = 300


def op():
    return mx.ops.get('_contrib_token_log_probs').fn


def gradients(device, dtype, use, tok, x, g):
    x = x.to(device=device, dtype=dtype).requires_grad_(True)
    lp, ent, top, _ = op()(x, tok.to(device), topk=5)
    assert torch.isnan(lp).tolist() == [bool(t < 0 or t >= V) and int(t) != -1 for t in tok]
    heads = {'log_prob': lp, 'entropy': ent, 'top': top}
    dx, = torch.autograd.grad([heads[u] for u in use], x, [g[u].to(device=device, dtype=heads[u].dtype) for u in use])
    return dx


def check(device, dtype):
    t = torch.float32 if dtype == torch.float64 else dtype         # the oracle has 64 bits itself: no bound of its own for them
    rng = torch.Generator().manual_seed(2)
    x = torch.randn(6, V, generator=rng).to(dtype)
    x[5] = -math.inf
    tok = torch.tensor([3, -100, V, -1, 2 ** 40, -100])
    inside = torch.tensor([3, 0, 0, -1, 0, 0])
    g = {'log_prob': torch.randn(6, generator=rng), 'entropy': torch.randn(6, generator=rng), 'top': torch.randn(6, 5, generator=rng)}
    for use in (['entropy'], ['top'], ['entropy', 'top']):         # nothing asks about the tokens
        dx = gradients(device, dtype, use, tok, x, g)
        grads = [None] + [g[u][:5] if u in use else None for u in ('entropy', 'top')]
        want, bound = oracle.log_probs(x[:5], inside[:5], 5, grads=grads, t=t)
        oracle.check(dx[:5], want[-1], bound[-1], str(use))
        assert not bool(dx[5].any())
    # gradients of 0, as a mask behind the operator gives them
    quiet = dict(g, log_prob=torch.where(tok == inside, g['log_prob'], torch.zeros(6)))
    dx = gradients(device, dtype, ['log_prob', 'entropy', 'top'], tok, x, quiet)
    want, bound = oracle.log_probs(x[:5], inside[:5], 5, grads=[quiet[u][:5] for u in ('log_prob', 'entropy', 'top')], t=t)
    oracle.check(dx[:5], want[-1], bound[-1], 'masked')
    assert not bool(dx[5].any())
    dx = gradients(device, dtype, ['log_prob', 'entropy', 'top'], tok, x, g)
    assert torch.isnan(dx).all(-1).tolist() == [False, True, True, False, True, False]
    assert torch.isfinite(dx[[0, 3, 5]]).all() and not bool(dx[5].any())


@pytest.mark.parametrize('dtype', [torch.float32, torch.float64])
def test_unknown_tokens(dtype):
    check('cpu', dtype)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
def test_unknown_tokens_on_the_kernels(dtype):
    check('cuda', dtype)


def test_the_gradient_of_known_tokens_still_has_one():
    x = torch.randn(3, 7, dtype=torch.float64, requires_grad=True)
    tok = torch.tensor([0, 6, -1])
    assert torch.autograd.gradcheck(lambda a: op()(a, tok)[0], x) and torch.autograd.gradgradcheck(lambda a: op()(a, tok)[0], x)
