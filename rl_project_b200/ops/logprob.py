"""Fused LM-head -> log-softmax -> gather (kernel: csrc/logprob.cu).

``linear_logprobs(h, W, targets)`` returns per-token ``log p(target)`` (and
optionally the entropy) without ever building an fp32 ``[N, V]`` tensor:
logits exist only in bf16; when the own GEMM runs the LM-head forward its
epilogue also writes each row's online log-sum-exp statistics per 256-column
chunk, so a small merge pass gives the outputs without re-reading the logits
(otherwise the kernel makes ONE pass over each row for the forward), and the
backward rewrites the same buffer in
place with ``g * (onehot - softmax)`` before the two GEMMs that produce
``dh`` and ``dW``.  When ``N * V`` bf16 logits exceed the keep budget, rows
are processed in chunks and recomputed in backward.

Replaces ``F.cross_entropy`` at ``src/forgeline/models/transformer/model.py:154``
and ``token_logprobs_from_logits`` at ``src/forgeline/models/policy.py:47-50``.

``token_logprobs(logits, targets, top)`` (csrc/token_logprob.cu) takes logits that exist already (a serving step's, a
Hugging Face model's) and returns the targets' log-probs, the entropy and the ``top`` alternatives, differentiably.
"""

from __future__ import annotations

import os
from typing import List, NamedTuple, Optional, Tuple

import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn.functional as F

from rl_project_b200.ops._ext import native

KEEP_BUDGET_BYTES = int(float(os.environ.get("RLB_LOGITS_KEEP_GB", "24")) * (1 << 30))
CHUNK_ROWS = int(os.environ.get("RLB_LOGITS_CHUNK_ROWS", "16384"))


from rl_project_b200.ops.linear import matmul_nn, matmul_tn  # noqa: E402


def _gemm_nt(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """a [M, K] @ b[N, K]^T -> [M, N]."""
    from rl_project_b200.ops.linear import matmul_nt

    return matmul_nt(a, b)


class _LinearLogprob(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, W, targets, with_entropy):
        N = h.shape[0]
        V = W.shape[0]
        keep = N * V * 2 <= KEEP_BUDGET_BYTES
        step = N if keep else max(1, min(N, CHUNK_ROWS))
        lse_parts, lp_parts, ent_parts, kept = [], [], [], []
        from rl_project_b200.ops import gemm

        for s in range(0, N, step):
            hs = h[s:s + step]
            if hs.is_cuda and gemm.lse_fusable(hs, W):
                # the GEMM's epilogue writes per-chunk row statistics: no second pass over the logits
                logits, stats = gemm.gemm_nt_lse(hs, W)
                outs = native().logprob_combine(stats, logits, targets[s:s + step], with_entropy, None)
            else:
                logits = _gemm_nt(hs, W)
                outs = native().logprob_fwd(logits, targets[s:s + step], with_entropy, None)
            lse_parts.append(outs[0])
            lp_parts.append(outs[1])
            if with_entropy:
                ent_parts.append(outs[2])
            if keep:
                kept.append(logits)
        lse = torch.cat(lse_parts)
        lp = torch.cat(lp_parts)
        ent = torch.cat(ent_parts) if with_entropy else None
        ctx.keep = keep
        ctx.step = step
        ctx.with_entropy = with_entropy
        ctx.kept = kept
        ctx.save_for_backward(h, W, targets, lse, ent if ent is not None else torch.empty(0))
        ctx.mark_non_differentiable(lse)
        if with_entropy:
            return lp, ent
        return lp, lse

    @staticmethod
    def backward(ctx, g_lp, g_second):
        h, W, targets, lse, ent = ctx.saved_tensors
        g_ent = g_second if ctx.with_entropy else None
        N = h.shape[0]
        step = ctx.step
        dh = torch.empty_like(h)
        dW32: Optional[torch.Tensor] = None
        dW16: Optional[torch.Tensor] = None
        g_lp = g_lp.float().contiguous() if g_lp is not None else None
        g_ent = g_ent.float().contiguous() if g_ent is not None else None
        for i, s in enumerate(range(0, N, step)):
            logits = ctx.kept[i] if ctx.keep else _gemm_nt(h[s:s + step], W)
            native().logprob_bwd_(logits, targets[s:s + step], lse[s:s + step],
                                  g_lp[s:s + step] if g_lp is not None else None,
                                  ent[s:s + step] if ctx.with_entropy else None,
                                  g_ent[s:s + step] if g_ent is not None else None, 1.0)
            dh[s:s + step] = matmul_nn(logits, W)
            part = matmul_tn(logits, h[s:s + step])
            if N <= step:
                dW16 = part
            else:
                dW32 = part.float() if dW32 is None else dW32.add_(part.float())
            del logits
        ctx.kept = []
        dW = dW16 if dW16 is not None else dW32.to(W.dtype)
        return dh, dW, None, None


def linear_logprobs_reference(h: torch.Tensor, W: torch.Tensor, targets: torch.Tensor, with_entropy: bool = False):
    logits = (h.float() @ W.float().t())
    logp = torch.log_softmax(logits, dim=-1)
    safe = targets.clamp(min=0)
    lp = logp.gather(-1, safe.unsqueeze(-1)).squeeze(-1) * (targets >= 0).float()
    if with_entropy:
        ent = -(logp.exp() * logp).sum(-1)
        return lp, ent
    return lp, torch.logsumexp(logits, dim=-1)


def linear_logprobs(h: torch.Tensor, W: torch.Tensor, targets: torch.Tensor,
                    with_entropy: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``h [N, d]``, ``W [V, d]``, ``targets [N]`` (-1 = ignore) -> ``(lp [N], lse [N] | entropy [N])``."""
    targets = targets.reshape(-1).to(torch.long).contiguous()
    h2 = h.reshape(-1, h.shape[-1])
    if h2.is_cuda and h2.dtype == torch.bfloat16:
        Wc = W if W.dtype == torch.bfloat16 else W.to(torch.bfloat16)
        return _LinearLogprob.apply(h2.contiguous(), Wc, targets, with_entropy)
    if h2.is_cuda:
        native()
    return linear_logprobs_reference(h2, W, targets, with_entropy)


def linear_cross_entropy(h: torch.Tensor, W: torch.Tensor, targets: torch.Tensor,
                         ignore_index: int = -1) -> torch.Tensor:
    """Mean token cross-entropy of ``h @ W^T`` against ``targets`` (``ignore_index`` skipped)."""
    t = targets.reshape(-1).to(torch.long)
    if ignore_index != -1:
        t = torch.where(t == ignore_index, torch.full_like(t, -1), t)
    lp, _ = linear_logprobs(h, W, t)
    n = (t >= 0).sum().clamp(min=1)
    return -(lp.sum() / n)


def logprobs_from_logits(logits: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """Token log-probs from already materialised logits ``[..., V]`` (any device)."""
    flat = logits.reshape(-1, logits.shape[-1])
    t = targets.reshape(-1).to(torch.long)
    lp = -F.cross_entropy(flat.float(), t, reduction="none", ignore_index=-1)
    return lp.view(targets.shape)


# ---------------------------------------------------------------- log-probs, entropy and alternatives from logits
TOP_MOST = 64


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor  # [...] fp32: log p(target), 0 where the target is -1
    entropy: torch.Tensor  # [...] fp32
    top_logprobs: torch.Tensor  # [..., top] fp32, falling
    top_ids: torch.Tensor  # [..., top] int64, the lowest id first among equal logits


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, targets, top, status):
        lp, ent, top_lp, top_ids, m, ls = native().token_logprob(x, targets, top, True, status)
        ctx.top = top
        ctx.save_for_backward(x, targets, m, ls, ent, top_ids)
        ctx.mark_non_differentiable(top_ids)
        ctx.set_materialize_grads(False)
        return lp, ent, top_lp, top_ids

    @staticmethod
    def backward(ctx, g_lp, g_ent, g_top, _):
        grads = [g.float().contiguous() if g is not None else None for g in (g_lp, g_ent, g_top)]
        if not torch.is_grad_enabled():
            return native().token_logprob_bwd(*ctx.saved_tensors, *grads), None, None, None
        # a gradient that is itself to be differentiated (create_graph): the plain form's
        x, targets = ctx.saved_tensors[:2]
        outs = _token_logprobs_reference(x, _within(targets, x.shape[-1]), ctx.top)[:3]
        outs, grads = zip(*((o, g) for o, g in zip(outs, grads) if g is not None))
        return torch.autograd.grad(outs, x, grads, create_graph=True)[0], None, None, None


def _within(targets: torch.Tensor, V: int) -> torch.Tensor:
    """Targets without those outside the vocabulary."""
    return targets.masked_fill(targets >= V, -1)


def _plainly(x: torch.Tensor) -> bool:
    """Whether the call is under a transform that kernels do not go through: torch.func's, or forward-mode AD."""
    return torch._C._are_functorch_transforms_active() or forward_ad.unpack_dual(x).tangent is not None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0,
                   status: Optional[torch.Tensor] = None) -> TokenLogprobs:
    """``logits [..., V]`` (fp32, bf16 or fp16) and ``targets [...]`` (-1: none) -> :class:`TokenLogprobs`.

    One pass over the logits; gradients flow to them from the log-probs, the entropy and the alternatives' log-probs.
    Entries of -inf are tokens that cannot occur; a row of nothing else has log-probs -inf, entropy 0 and no
    gradient, a row with NaN or +inf gives NaN.  ``top`` is at most 64.  A target outside the vocabulary has log-prob
    0 and is reported in ``status`` or the device's index-error word (on CPU: ``IndexError``).  Second derivatives
    (``create_graph``), forward-mode AD and ``torch.func`` transforms go through the plain form, in several passes and
    without that report.
    """
    V = logits.shape[-1]
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"logits: fp32, bf16 or fp16, got {logits.dtype}")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} do not match logits {tuple(logits.shape)}")
    if not 0 <= top <= min(TOP_MOST, V):
        raise ValueError(f"top must be 0 to {TOP_MOST} and no more than the vocabulary ({V}), got {top}")
    x = logits.reshape(-1, V)
    t = targets.reshape(-1).to(torch.long).contiguous()
    shape = targets.shape
    if _plainly(x):
        lp, ent, top_lp, ids = _token_logprobs_reference(x, _within(t, V), int(top))
    elif x.is_cuda:
        x = x if x.stride(1) == 1 else x.contiguous()
        if x.requires_grad and torch.is_grad_enabled():
            lp, ent, top_lp, ids = _TokenLogprobs.apply(x, t, int(top), status)
        else:
            lp, ent, top_lp, ids = native().token_logprob(x.detach(), t, int(top), False, status)
    else:
        if t.numel() and t.max() >= V:
            raise IndexError("a target lies outside the vocabulary")
        lp, ent, top_lp, ids = _token_logprobs_reference(x, t, int(top))
    if logits.dim() == 2:
        return TokenLogprobs(lp, ent, top_lp, ids)
    return TokenLogprobs(lp.view(shape), ent.view(shape), top_lp.view(*shape, top), ids.view(*shape, top))


def _token_logprobs_reference(x: torch.Tensor, t: torch.Tensor, top: int):
    x = x.float()
    dead = (x == float("-inf")).all(-1, keepdim=True)
    logp = torch.where(dead, torch.zeros_like(x), x).log_softmax(-1)
    lp = logp.gather(-1, t.clamp(min=0)[:, None])[:, 0]
    p = logp.exp()
    ent = -torch.where(p == 0, torch.zeros_like(p), p * logp.masked_fill(p == 0, 0.0)).sum(-1)
    if top:
        ids = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, :top]
    else:
        ids = torch.empty(x.shape[0], 0, dtype=torch.long, device=x.device)
    inf, zero = torch.full_like(lp, float("-inf")), torch.zeros_like(lp)
    lp = torch.where(t >= 0, torch.where(dead[:, 0], inf, lp), zero)
    return lp, torch.where(dead[:, 0], zero, ent), logp.gather(-1, ids).masked_fill(dead, float("-inf")), ids
