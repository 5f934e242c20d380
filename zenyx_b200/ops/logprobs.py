"""Operators on the logits of a language-model head, over ``csrc/head/logprobs.cu``:

* ``token_logprobs``: log-probabilities of given tokens, the entropy, and the most likely alternatives (scoring,
  policy gradients, writing down a teacher), differentiable;
* ``distill_topk`` / ``distill_topk_fwd_bwd_``: the divergence from a teacher of which only the top log-probabilities were
  kept, and its gradient.

Logits are [..., V] in bf16, fp16 or fp32 with contiguous columns (rows may be strided and start anywhere); results
are fp32. CPU tensors take a PyTorch form of the same formulas (fp64 logits are computed in fp64 there). The
reference has neither: its loss is whatever criterion the caller passes to ``Trainer.train_step``
(zenyx/train/trainer.py:36-49).

Rows and values that stand for nothing:

* a row whose target lies outside [0, V) (``ignore_index`` included) is left out: its log-probability, entropy and
  gradient are 0, it has no alternatives, and its logits are not looked at;
* a logit of -inf has probability 0 and is no alternative. Missing alternatives have token -1 and log-probability -inf;
* a row whose logits are all -inf has log-probability -inf, entropy 0 and no gradient;
* a row that holds +inf or NaN has NaN everywhere and no alternatives.

Gradients are reverse-mode and of first order: tensors with forward-mode tangents and function transforms are refused.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _ext

MAX_TOP = 128          # most alternatives of a row
MAX_VOCAB = 400000     # most columns
MIN_TEMPERATURE, MAX_TEMPERATURE = 1e-4, 1e4
_NEG = float("-inf")


class TokenLogprobs(NamedTuple):
    logprobs: Optional[torch.Tensor]       # [...] of the given tokens; None without targets
    entropy: torch.Tensor                  # [...], in nats
    top_logprobs: Optional[torch.Tensor]   # [..., top_k], largest first; None for top_k = 0
    top_ids: Optional[torch.Tensor]        # [..., top_k] int64; equal logits: the lower token first


# ------------------------------------------------------------------------------------------------
# Checks
# ------------------------------------------------------------------------------------------------


_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check_no_tangent(name: str, t: torch.Tensor) -> None:
    if forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{name}: there is no forward-mode derivative")


def _check_logits(logits: torch.Tensor, temperature: float) -> None:
    _check_no_tangent("logits", logits)
    if logits.dtype not in _TYPES and (logits.is_cuda or logits.dtype != torch.float64):
        raise TypeError(f"logits are bf16, fp16 or fp32 (fp64 on the CPU), not {logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_VOCAB:
        raise ValueError(f"logits are [..., V] with 1 <= V <= {MAX_VOCAB}, not {tuple(logits.shape)}")
    if not MIN_TEMPERATURE <= temperature <= MAX_TEMPERATURE:
        raise ValueError(f"the temperature lies in [{MIN_TEMPERATURE:g}, {MAX_TEMPERATURE:g}], not {temperature}")


def _check_ids(name: str, ids: torch.Tensor, shape, logits: torch.Tensor) -> None:
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} are int64 or int32, not {ids.dtype}")
    if ids.shape != torch.Size(shape):
        raise ValueError(f"{name} have shape {tuple(ids.shape)}, expected {tuple(shape)}")
    if ids.device != logits.device:
        raise ValueError(f"{name} are on {ids.device}, the logits on {logits.device}")


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """[..., V] -> [rows, V] with contiguous columns (a copy only where the strides leave no other way)."""
    x = logits.reshape(-1, logits.shape[-1]) if logits.dim() != 2 else logits
    return x if x.shape[1] == 1 or x.stride(1) == 1 else x.contiguous()


def _wide(x: torch.Tensor) -> torch.Tensor:
    return x if x.dtype == torch.float64 else x.float()


# ------------------------------------------------------------------------------------------------
# Token log-probabilities
# ------------------------------------------------------------------------------------------------


def token_logprobs_fwd(logits: torch.Tensor, targets: Optional[torch.Tensor], top_k: int,
                       temperature: float) -> Tuple[TokenLogprobs, torch.Tensor]:
    """logits [rows, V], targets [rows] or None. Returns the results and the row statistics that
    ``token_logprobs_bwd`` takes: [rows, 2], the maximum and the sum of the exponentials (0: no gradient)."""
    T, V = logits.shape
    dev = logits.device
    if _ext.use_cuda_kernels(logits):
        lp = torch.empty(T, device=dev, dtype=torch.float32) if targets is not None else None
        entropy = torch.empty(T, device=dev, dtype=torch.float32)
        stats = torch.empty(T, 2, device=dev, dtype=torch.float32)
        top = ids = None
        if top_k > 0:
            top = torch.empty(T, top_k, device=dev, dtype=torch.float32)
            ids = torch.empty(T, top_k, device=dev, dtype=torch.int64)
        _ext.C().token_logprobs_fwd(logits, targets.contiguous() if targets is not None else None, lp, entropy, stats,
                                    top, ids, temperature)
        return TokenLogprobs(lp, entropy, top, ids), stats
    x = _wide(logits)
    live = torch.ones(T, dtype=torch.bool)
    if targets is not None:
        live = (targets >= 0) & (targets < V)
    m = x.amax(dim=1).masked_fill(~live, 0.0)
    empty, bad = m == _NEG, torch.isnan(m) | (m == float("inf"))
    m0 = torch.where(empty | bad, torch.zeros_like(m), m)
    z = ((x - m0[:, None]) / temperature).masked_fill(~live[:, None], 0.0)
    e = z.exp()
    l = e.sum(dim=1).masked_fill(bad, float("nan"))
    log_l = l.log()
    entropy = log_l - torch.where(e == 0, 0.0, e * z).sum(dim=1) / l
    entropy = entropy.masked_fill(empty | ~live, 0.0)
    stats = torch.stack([m, l.masked_fill(empty | ~live, 0.0)], dim=1)
    z = z - torch.where(empty, 0.0, log_l)[:, None]
    lp = None
    if targets is not None:
        lp = z.gather(1, targets.clamp(0, V - 1).long()[:, None])[:, 0].masked_fill(~live, 0.0)
    top = ids = None
    if top_k > 0:
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top_k]
        top = z.gather(1, ids).masked_fill(~live[:, None], _NEG)
        ids = ids.masked_fill((x.gather(1, ids) == _NEG) | ~live[:, None] | torch.isnan(top), -1)
    return TokenLogprobs(lp, entropy, top, ids), stats


def token_logprobs_bwd(logits: torch.Tensor, targets: Optional[torch.Tensor], out: TokenLogprobs, stats: torch.Tensor,
                       d_logprobs: Optional[torch.Tensor], d_entropy: Optional[torch.Tensor],
                       d_top: Optional[torch.Tensor], temperature: float,
                       d_logits: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient with respect to the logits [rows, V] (their type) from the gradients of the three results, each of
    which may be absent. ``d_logits`` may be the logits themselves."""
    if d_logits is None:
        d_logits = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
    if _ext.use_cuda_kernels(logits):
        def fp32(g):
            return g.to(torch.float32).contiguous() if g is not None else None

        _ext.C().token_logprobs_bwd(logits, targets.contiguous() if targets is not None else None, out.entropy, stats,
                                    out.top_ids, fp32(d_logprobs), fp32(d_entropy), fp32(d_top), d_logits, temperature)
        if not d_logits.is_inference():     # a backward that has kept these logits is an error now instead of wrong
            torch.autograd.graph.increment_version(d_logits)
        return d_logits
    x = _wide(logits)
    m, l = stats[:, 0], stats[:, 1]
    live = l != 0
    z = ((x - m[:, None]) / temperature).masked_fill(~live[:, None], 0.0)
    p = z.exp() / l[:, None]
    g = torch.zeros_like(p)
    if d_entropy is not None:
        z = z - l.log()[:, None]
        g -= d_entropy[:, None] * torch.where(p == 0, 0.0, p * (z + out.entropy[:, None]))
    if d_logprobs is not None:
        hit = (targets >= 0) & (targets < x.shape[1])
        d = d_logprobs.masked_fill(~hit, 0.0)[:, None]
        g -= d * p
        g.scatter_add_(1, targets.clamp(0, x.shape[1] - 1).long()[:, None], d)
    if d_top is not None:
        d = d_top.masked_fill(out.top_ids < 0, 0.0)
        g -= d.sum(dim=1, keepdim=True) * p
        g.scatter_add_(1, out.top_ids.clamp(min=0), d)
    return d_logits.copy_((g / temperature).masked_fill(~live[:, None], 0.0))


class _TokenLogprobsFn(torch.autograd.Function):
    """CPU tensors; the CUDA form is an autograd function of the extension."""

    @staticmethod
    def forward(ctx, logits, targets, top_k, temperature):
        out, stats = token_logprobs_fwd(logits, targets, top_k, temperature)
        ctx.save_for_backward(logits, targets, out.entropy, out.top_ids, stats)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if out.top_ids is not None:
            ctx.mark_non_differentiable(out.top_ids)
        return tuple(out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_logprobs, d_entropy, d_top, _):
        logits, targets, entropy, ids, stats = ctx.saved_tensors
        if d_logprobs is None and d_entropy is None and d_top is None:
            return None, None, None, None
        out = TokenLogprobs(None, entropy, None, ids)
        return token_logprobs_bwd(logits, targets, out, stats, d_logprobs, d_entropy, d_top, ctx.temperature), None, None, None


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *, top_k: int = 0,
                   temperature: float = 1.0, ignore_index: int = -100) -> TokenLogprobs:
    """Log-probabilities of ``targets`` [...] under softmax(logits [..., V] / temperature), its entropy, and the
    ``top_k`` (at most 128) most likely tokens with their log-probabilities.

    Differentiable with respect to the logits through the log-probabilities, the entropy and the alternatives'
    log-probabilities. Rows whose target is ``ignore_index`` (or any other number outside [0, V)) are left out;
    without targets every row counts and ``logprobs`` is None.
    """
    if logits.is_cuda:      # the extension checks the same
        return TokenLogprobs(*_ext.C().token_logprobs(logits, targets, top_k, temperature, ignore_index))
    _check_logits(logits, temperature)
    V, shape = logits.shape[-1], logits.shape[:-1]
    if not 0 <= top_k <= min(V, MAX_TOP):
        raise ValueError(f"top_k lies in [0, min(V, {MAX_TOP})], not {top_k}")
    if 0 <= ignore_index < V:
        raise ValueError(f"ignore_index {ignore_index} is a token")
    if targets is not None:
        _check_ids("targets", targets, shape, logits)
    if targets is not None:
        targets = targets.reshape(-1)
    lp, entropy, top, ids = _TokenLogprobsFn.apply(_rows(logits), targets, int(top_k), float(temperature))
    return TokenLogprobs(lp.view(shape) if lp is not None else None, entropy.view(shape),
                         top.view(*shape, top_k) if top is not None else None,
                         ids.view(*shape, top_k) if ids is not None else None)


# ------------------------------------------------------------------------------------------------
# Distillation from a teacher's top logits
# ------------------------------------------------------------------------------------------------


def _check_teacher(logits, values, ids, tail: str) -> None:
    if tail not in ("renormalize", "bucket"):
        raise ValueError(f"tail is 'renormalize' or 'bucket', not {tail!r}")
    K = ids.shape[-1] if ids.dim() > 0 else 0
    if not 1 <= K <= MAX_TOP:
        raise ValueError(f"teacher_ids are [..., K] with 1 <= K <= {MAX_TOP}, not {tuple(ids.shape)}")
    _check_ids("teacher_ids", ids, (*logits.shape[:-1], K), logits)
    if values.dtype not in _TYPES and (logits.is_cuda or values.dtype != torch.float64):
        raise TypeError(f"teacher_logprobs are bf16, fp16 or fp32, not {values.dtype}")
    if values.shape != ids.shape:
        raise ValueError(f"teacher_logprobs have shape {tuple(values.shape)}, teacher_ids {tuple(ids.shape)}")
    if values.device != logits.device:
        raise ValueError(f"teacher_logprobs are on {values.device}, the logits on {logits.device}")
    if values.requires_grad and torch.is_grad_enabled():
        raise ValueError("the teacher gets no gradient: detach teacher_logprobs")
    _check_no_tangent("teacher_logprobs", values)


def _distill_torch(x, values, ids, temperature: float, bucket: bool):
    """(losses, their gradient with respect to x) in the type of x, which is fp32 or fp64."""
    T, V = x.shape
    there = (ids >= 0) & (ids < V)
    at = torch.where(there, ids, 0).long()
    v = values.to(x.dtype).masked_fill(~there, _NEG)
    if bucket:
        live = there.any(dim=1)
        q = v.exp()
    else:
        top = v.amax(dim=1, keepdim=True)
        live = (top != _NEG)[:, 0]
        q = (v - top.masked_fill(~live[:, None], 0.0)).exp()
        q = q / q.sum(dim=1, keepdim=True).masked_fill(~live[:, None], 1.0)
    m = x.amax(dim=1, keepdim=True)
    none = m == _NEG
    lse = torch.logsumexp((x - m.masked_fill(none, 0.0)) / temperature, dim=1, keepdim=True)
    lp = (x - m.masked_fill(none, 0.0)) / temperature - lse.masked_fill(none, 0.0)
    loss = torch.where(q == 0, 0.0, q * (q.log() - lp.gather(1, at))).sum(dim=1)
    grad = lp.exp()
    if bucket:
        total = v.double().exp().sum(dim=1, keepdim=True)     # a peaked teacher leaves few digits of the remainder in 32 bits
        rest, total = (1.0 - total).clamp(min=0.0).to(x.dtype), total.to(x.dtype)
        inside = torch.zeros_like(x).scatter_add_(1, at, there.to(x.dtype)) > 0
        outside = lp.masked_fill(inside, _NEG)
        log_rest = torch.logsumexp(outside, dim=1, keepdim=True)
        some = (rest > 0) & (log_rest != _NEG)
        loss = loss + torch.where(some, rest * (rest.log() - log_rest), 0.0)[:, 0]
        # the weights in the loss add up to 1, except where the remainder is not among them
        grad = grad * torch.where(some, 1.0, total) - torch.where(some & (outside != _NEG), rest * (outside - log_rest).exp(), 0.0)
    grad = grad.scatter_add(1, at, -q) / temperature
    return loss.masked_fill(~live, 0.0), grad.masked_fill(~live[:, None], 0.0)


def distill_topk_fwd_bwd_(logits: torch.Tensor, teacher_logprobs: torch.Tensor, teacher_ids: torch.Tensor,
                          grad_scale: float, *, temperature: float = 1.0, tail: str = "renormalize",
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Overwrites `logits` [rows, V] (or fills `out`, which leaves them alone) with grad_scale * d(sum of
    losses)/d(logits); returns the per-row losses (fp32), without a gradient of their own. What the losses are: see
    ``distill_topk``."""
    if logits.is_cuda:      # the extension checks the same
        return _ext.C().distill_topk_fwd_bwd(logits, teacher_logprobs, teacher_ids, grad_scale, temperature, tail, out)
    _check_logits(logits, temperature)
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits are [rows, V] with contiguous columns")
    _check_teacher(logits, teacher_logprobs, teacher_ids, tail)
    out = logits if out is None else out
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out has the shape, type and device of the logits")
    loss, grad = _distill_torch(_wide(logits.detach()), teacher_logprobs.detach(), teacher_ids, temperature, tail == "bucket")
    out.copy_(grad * grad_scale)
    return loss


class _DistillFn(torch.autograd.Function):
    """CPU tensors; the CUDA form is an autograd function of the extension."""

    @staticmethod
    def forward(ctx, logits, values, ids, temperature, bucket):
        ctx.meta = (temperature, bucket)
        ctx.save_for_backward(logits, values, ids)
        return _distill_torch(_wide(logits), values, ids, temperature, bucket)[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_loss):
        logits, values, ids = ctx.saved_tensors
        grad = _distill_torch(_wide(logits), values, ids, *ctx.meta)[1]
        return (grad * d_loss[:, None]).to(logits.dtype), None, None, None, None


def distill_topk(logits: torch.Tensor, teacher_logprobs: torch.Tensor, teacher_ids: torch.Tensor, *,
                 temperature: float = 1.0, tail: str = "renormalize") -> torch.Tensor:
    """Per-row divergences [...] (fp32, in nats) from a teacher to p = softmax(logits [..., V] / temperature),
    differentiable with respect to the logits. The teacher is known by the log-probabilities [..., K] of K (at most
    128) of its tokens, as ``token_logprobs(teacher, top_k=K, temperature=temperature)`` writes them down.

    ``tail="renormalize"``: q = softmax(teacher_logprobs) over the K tokens (so logits do as well),
    sum_k q_k (log q_k - log p_k). ``tail="bucket"``: q = exp(teacher_logprobs), and all other tokens are one, with
    what is left of either distribution: + q_r (log q_r - log p_r), where q_r = max(0, 1 - sum_k q_k); it is left out
    where the student has nothing outside the K tokens. Values in bf16 or fp16 may add up to more than 1 by their
    rounding: the loss takes them as they are.

    Entries whose token lies outside [0, V) (-1) are absent, whatever their value; a row without entries (or, for
    ``renormalize``, with values of -inf only) is left out: loss and gradient 0. A token that is named twice gets
    the sum of both. The loss is infinite where the student's logit of a token with q > 0 is -inf. Softened
    targets are usually weighted with temperature^2: that is left to the caller.
    """
    if logits.is_cuda:      # the extension checks the same
        return _ext.C().distill_topk_loss(logits, teacher_logprobs, teacher_ids, temperature, tail)
    _check_logits(logits, temperature)
    _check_teacher(logits, teacher_logprobs, teacher_ids, tail)
    K = teacher_ids.shape[-1]
    loss = _DistillFn.apply(_rows(logits), teacher_logprobs.detach().reshape(-1, K), teacher_ids.reshape(-1, K),
                            float(temperature), tail == "bucket")
    return loss.view(logits.shape[:-1])
