"""Log probabilities of tokens, entropy and top alternatives on the sm_100a kernels (``logprobs.cu``)."""
import torch

from . import lib, count_launch, check
from ._util import DT, address, on_device, once, raw_stream


def _forward(x, tokens, k, ignore, keep):
    rows, cols = x.shape
    dev = x.device
    lp = torch.empty(rows, dtype=torch.float32, device=dev)
    ent = torch.empty_like(lp)
    top_lp = torch.empty((rows, k), dtype=torch.float32, device=dev) if k else None
    top_id = torch.empty((rows, k), dtype=torch.int64, device=dev) if k else None
    stat = torch.empty((rows, 3), dtype=torch.float32, device=dev) if keep else None
    with on_device(x):
        check(lib().mxb_logprob_forward(DT[x.dtype], x.data_ptr(), tokens.data_ptr(), lp.data_ptr(), ent.data_ptr(), address(top_lp),
                                        address(top_id), address(stat), rows, cols, k, ignore, raw_stream(x)), 'token_log_probs')
    count_launch(1)
    return lp, ent, top_lp, top_id, stat


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tokens, k, ignore):
        lp, ent, top_lp, top_id, stat = _forward(x, tokens, k, ignore, True)
        ctx.save_for_backward(x, tokens, stat, top_id)
        ctx.args = (k, ignore)
        ctx.set_materialize_grads(False)
        if not k:
            return lp, ent
        ctx.mark_non_differentiable(top_id)
        return lp, ent, top_lp, top_id

    @staticmethod
    @once
    def backward(ctx, g_lp, g_ent, g_top=None, _=None):
        x, tokens, stat, top_id = ctx.saved_tensors
        k, ignore = ctx.args
        rows, cols = x.shape
        g_lp, g_ent, g_top = (None if g is None else g.contiguous() for g in (g_lp, g_ent, g_top))
        dx = torch.empty_like(x)
        with on_device(x):
            check(lib().mxb_logprob_backward(DT[x.dtype], x.data_ptr(), dx.data_ptr(), tokens.data_ptr(), stat.data_ptr(), address(g_lp),
                                             address(g_ent), address(g_top), address(top_id), rows, cols, k, ignore, raw_stream(x)),
                  'token_log_probs backward')
        count_launch(1)
        return dx, None, None, None


def token_log_probs(x, tokens, k, ignore):
    """``x``: [rows, cols] contiguous, ``tokens``: [rows] int64 contiguous."""
    if x.requires_grad and torch.is_grad_enabled():
        return _TokenLogProbs.apply(x, tokens, k, ignore)
    lp, ent, top_lp, top_id, _ = _forward(x, tokens, k, ignore, False)
    return (lp, ent, top_lp, top_id) if k else (lp, ent)
