"""Fused loss terms of the world-model update on the GPU (lib/world_model.py:463-528).

``kl_pair``: both KL terms between the unimix'ed posterior and prior (dynamics: gradient to the prior
only; representation: to the posterior only) from one forward and one backward kernel.
``mse_rows``: 0.5 * mean squared reconstruction error per frame.
``distill_topk_rows``: a student's logits against a teacher's stored top logits.
Host tensors (and class counts other than 32) take the eager formulas of ``WorldModel``.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native as N


class _KLPairFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, post, prior, eps, free_nats):
        post, prior = post.contiguous(), prior.contiguous()
        rows, L, K = post.shape
        out = torch.empty(2, rows, dtype=torch.float32, device=post.device)
        N.check(N.lib().drm_kl_pair_forward(post.data_ptr(), prior.data_ptr(), rows, L, K, eps, free_nats, out[0].data_ptr(),
                                            out[1].data_ptr(), N.stream_ptr(post.device)), "drm_kl_pair_forward")
        ctx.save_for_backward(post, prior)
        ctx.eps, ctx.free_nats = eps, free_nats
        return out[0], out[1]

    @staticmethod
    def backward(ctx, g_dyn, g_rep):
        post, prior = ctx.saved_tensors
        rows, L, K = post.shape
        d_post, d_prior = torch.empty_like(post), torch.empty_like(prior)
        g_dyn = None if g_dyn is None else g_dyn.contiguous()
        g_rep = None if g_rep is None else g_rep.contiguous()
        N.check(N.lib().drm_kl_pair_backward(post.data_ptr(), prior.data_ptr(), rows, L, K, ctx.eps, ctx.free_nats, N.ptr(g_dyn),
                                             N.ptr(g_rep), d_post.data_ptr(), d_prior.data_ptr(), N.stream_ptr(post.device)),
                "drm_kl_pair_backward")
        return d_post, d_prior, None, None


def kl_pair(post_logits: torch.Tensor, prior_logits: torch.Tensor, unimix_eps: float, free_nats: float):
    """(dynamics rows, representation rows), each (rows,): sum over latents of max(KL, free_nats)."""
    return _KLPairFn.apply(post_logits.float(), prior_logits.float(), float(unimix_eps), float(free_nats))


class _MseRowsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x_hat, x):
        x_hat, x = x_hat.contiguous(), x.contiguous()
        rows = x_hat.shape[0]
        E = x_hat.numel() // max(rows, 1)
        out = torch.empty(rows, dtype=torch.float32, device=x_hat.device)
        N.check(N.lib().drm_mse_rows_forward(x_hat.data_ptr(), x.data_ptr(), rows, E, out.data_ptr(), N.stream_ptr(x_hat.device)),
                "drm_mse_rows_forward")
        ctx.save_for_backward(x_hat, x)
        return out

    @staticmethod
    def backward(ctx, g):
        x_hat, x = ctx.saved_tensors
        rows = x_hat.shape[0]
        d = torch.empty_like(x_hat)
        N.check(N.lib().drm_mse_rows_backward(x_hat.data_ptr(), x.data_ptr(), rows, x_hat.numel() // max(rows, 1),
                                              g.contiguous().data_ptr(), d.data_ptr(), N.stream_ptr(x_hat.device)),
                "drm_mse_rows_backward")
        return d, None


def mse_rows(x_hat: torch.Tensor, x_true: torch.Tensor) -> torch.Tensor:
    """0.5 * mean over all but the first dimension of (x_hat - x_true)^2; gradient to ``x_hat`` only."""
    return _MseRowsFn.apply(x_hat.float(), x_true.detach().float())


class _CriticLossRowsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, slow_logits, returns, lo, hi, reg):
        rows, nb = logits.shape
        out = torch.empty(rows, dtype=torch.float32, device=logits.device)
        N.check(N.lib().drm_critic_loss_forward(logits.data_ptr(), N.ptr(slow_logits), returns.data_ptr(), rows, nb, lo, hi, reg,
                                                out.data_ptr(), N.stream_ptr(logits.device)), "drm_critic_loss_forward")
        ctx.save_for_backward(logits, slow_logits, returns)
        ctx.conf = (lo, hi, reg)
        return out

    @staticmethod
    def backward(ctx, g):
        logits, slow_logits, returns = ctx.saved_tensors
        lo, hi, reg = ctx.conf
        rows, nb = logits.shape
        d = torch.empty_like(logits)
        N.check(N.lib().drm_critic_loss_backward(logits.data_ptr(), N.ptr(slow_logits), returns.data_ptr(), g.contiguous().data_ptr(),
                                                 rows, nb, lo, hi, reg, d.data_ptr(), N.stream_ptr(logits.device)),
                "drm_critic_loss_backward")
        return d, None, None, None, None, None


def critic_loss_rows(logits: torch.Tensor, slow_logits, returns: torch.Tensor, bucket_min: float, bucket_max: float,
                     reg: float) -> torch.Tensor:
    """Per-state critic loss (two-hot cross-entropy + reg * KL towards the slow critic), (rows,); gradient to
    ``logits`` only."""
    nb = logits.shape[-1]
    slow2 = None if slow_logits is None else slow_logits.detach().reshape(-1, nb).float().contiguous()
    return _CriticLossRowsFn.apply(logits.reshape(-1, nb).float().contiguous(), slow2,
                                   returns.detach().reshape(-1).float().contiguous(), float(bucket_min), float(bucket_max), float(reg))


def _distill_grad(ctx, g):
    logits, top_indices, p, row = ctx.saved_tensors
    return N.distill_topk_backward(logits, top_indices, p, row, g.contiguous(), ctx.temperature), None, None, None, None


_distill_grad_once = once_differentiable(_distill_grad)


class _DistillTopkRowsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_values, top_indices, top_lse, temperature):
        loss, p, row = N.distill_topk_forward(logits, top_values, top_indices, top_lse, temperature)
        ctx.save_for_backward(logits, top_indices, p, row)
        ctx.temperature = temperature
        return loss

    @staticmethod
    def backward(ctx, g):
        # (the wrapper that refuses a second differentiation is only needed where one could follow)
        return _distill_grad_once(ctx, g) if torch.is_grad_enabled() else _distill_grad(ctx, g)


def _list_of(t: torch.Tensor, dtype, rows: int, k: int) -> torch.Tensor:
    """A list (rows, k), dense, in ``dtype``, without derivatives; the tensor itself where it is that."""
    t = t.detach() if t.requires_grad or N.in_dual_level() else t
    if t.dtype == dtype and t.dim() == 2 and t.is_contiguous():
        return t
    return t.to(dtype).reshape(rows, k).contiguous()


def _distill_topk_rows_host(s, values, idx, lse, temperature):
    """The formula in tensor operations (autograd forms its gradient)."""
    vocab = s.shape[1]
    here = (idx >= 0) & (idx < vocab)
    t = torch.where(here, values / temperature, torch.full_like(values, float("-inf")))
    none = ~here.any(1) if lse is not None else ~(here & ((values != float("-inf")))).any(1)
    t = t.masked_fill(none.unsqueeze(1), 0.0)
    logp = t - (torch.logsumexp(t, 1) if lse is None else lse).unsqueeze(1)
    logp = logp.masked_fill(~here, float("-inf"))
    p = logp.exp()
    logq = torch.log_softmax(s.masked_fill(none.unsqueeze(1), 0.0) / temperature, 1)
    listed = torch.gather(logq, 1, torch.where(here, idx, torch.zeros_like(idx)))
    loss = torch.where(p == 0, torch.zeros_like(p), p * (logp - listed)).sum(1)
    if lse is not None:
        mass = p.sum(1)
        rest = (1.0 - mass).clamp_min(0.0)
        seen = torch.zeros(s.shape[0], vocab + 1, dtype=torch.bool).scatter_(1, torch.where(here, idx, torch.full_like(idx, vocab)), True)[:, :vocab]
        open_ = ~seen & (logq > float("-inf"))
        live = (rest > 0) & open_.any(1)
        log_rest = torch.logsumexp(torch.where(open_ | ~live.unsqueeze(1), logq, torch.full_like(logq, float("-inf"))), 1)
        loss = loss + torch.where(live, rest * (torch.log1p(-torch.where(live, mass, torch.zeros_like(mass))) - log_rest), torch.zeros_like(rest))
    return torch.where(none, torch.zeros_like(loss), loss)


def distill_topk_rows(logits: torch.Tensor, top_values: torch.Tensor, top_indices: torch.Tensor, temperature: float = 1.0,
                      top_lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Distillation loss per row, (rows,) fp32, of student logits (rows, V) against the teacher's listed logits: KL divergence of
    softmax(logits / temperature) from the teacher's probabilities; gradient to ``logits`` only (once).

    logits: fp32, bf16 or fp16, any leading shape and row stride.  top_values, top_indices (rows, k): the teacher's listed logits and
    their positions, k <= 1024; entries whose index is outside [0, V) are absent, a row with none has loss 0 and gradient 0.
    Without ``top_lse`` the teacher is the softmax over the listed entries.  With ``top_lse`` (rows,), the log-sum-exp of the
    teacher's whole row of logits / temperature, its listed probabilities keep their size and the rest of its mass is compared with
    the student's mass outside the list.  (The factor temperature**2 that keeps gradients comparable is the caller's.)"""
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise N.NativeError(f"distill_topk_rows: rows of at least one logit, got shape {tuple(logits.shape)}")
    if not 1e-6 <= float(temperature) <= 1e6:
        raise ValueError(f"distill_topk_rows: temperature {temperature}")
    for name, t in (("top_values", top_values), ("top_indices", top_indices)):
        if t.dim() < 1 or t.shape[:-1] != logits.shape[:-1] or t.shape != top_indices.shape:
            raise N.NativeError(f"distill_topk_rows: {name} {tuple(t.shape)} does not match logits {tuple(logits.shape)}")
    if top_indices.dtype not in (torch.int64, torch.int32) or top_values.dtype not in N.DTYPE_ID:
        raise N.NativeError(f"distill_topk_rows: top_values {top_values.dtype} / top_indices {top_indices.dtype}")
    if top_lse is not None and (top_lse.shape != logits.shape[:-1] or not top_lse.is_floating_point()):
        raise N.NativeError(f"distill_topk_rows: top_lse {tuple(top_lse.shape)} does not match logits {tuple(logits.shape)}")
    k = top_indices.shape[-1]
    rows = logits.numel() // logits.shape[-1]
    values, indices = _list_of(top_values, torch.float32, rows, k), _list_of(top_indices, torch.int64, rows, k)
    lse = None if top_lse is None else top_lse.detach().float().reshape(-1).contiguous()
    if logits.is_cuda:
        if N.wants_grad(logits):
            return _DistillTopkRowsFn.apply(N.as_rows(logits), values, indices, lse, float(temperature))
        return N.distill_topk_forward(N.as_rows(logits), values, indices, lse, float(temperature))[0]
    N.dtype_id(logits, "logits")
    return _distill_topk_rows_host(logits.reshape(rows, -1).float(), values, indices, lse, float(temperature))


def fused_ok(t: torch.Tensor, classes: int = 32) -> bool:
    return t.is_cuda and t.dtype == torch.float32 and classes == 32
