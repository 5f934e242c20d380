"""Plain 64-bit forms of the operators in zenyx_b200/ops/logprobs.py, row by row, and the tolerances their results are held to.

Tolerances (u = 2^-24, half a step of fp32; t_out = eps(type) / 2, half a step of the output's type):

* an exponential 2^d is off by 2^-22 of itself (the hardware's, with a margin of two), and its argument
  d = (x - m) log2(e) / t by 3 u |d| (a subtraction, a product, the factor's own rounding): relative 3 u ln 2 |d| < 2.1 u |d|;
* a sum of V exponentials adds one rounding a term along the longest chain, ceil(V / 128) + 16: a row of up to 128 vectors of
  16 bytes has a thread for each of them (eight terms at most, four sums of two), a longer one 128 threads or more, and a
  tree joins a thread's sums (2), the warp (5), the block (3) and the cluster (3). l is off by
  rel(V) = (ceil(V / 128) + 16) u + 2^-22 + 2.1 u <|d|> where <|d|>, the mean over the distribution, is at most log2(V) plus
  a few: 32 covers V <= 2^20.
  logprob = (x - m) / t - ln l: rel(V) plus the rounding of the result, u |logprob|;
* the entropy's second sum has terms 2^d d of one sign: <|d|> times the same relative error, and one product more;
* p is off by 2 rel(V) + 2.1 u |d| of itself; gradients add at most one more rounding for each of the at most 260
  coefficients that are summed up (their absolute sum times 260 u), and t_out of the result for its type.
"""
import math

import torch

U = 2.0 ** -24
NEG = float("-inf")


def rel_sum(V):
    return (math.ceil(V / 128) + 16) * U + 2.0 ** -22 + 2.1 * U * 32


def smallest(dtype):
    """Half of the smallest step near zero (bf16 and fp32 results below 2^-126 may be flushed)."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def logprobs(x, targets, top_k, t):
    """(logprobs, entropy, top_logprobs, top_ids, live, p, lp) in fp64 of logits x [T, V] (any float type)."""
    x = x.detach().double()
    T, V = x.shape
    live = torch.ones(T, dtype=torch.bool, device=x.device)
    if targets is not None:
        live = (targets >= 0) & (targets < V)
    m = x.amax(1)
    bad = (torch.isnan(x).any(1) | (x == float("inf")).any(1)) & live
    empty = (m == NEG) & live
    good = live & ~bad & ~empty
    z = torch.where(good[:, None], (x - torch.where(good, m, 0.0)[:, None]) / t, 0.0)
    lp = z - torch.log(torch.exp(z).sum(1))[:, None]
    p = torch.exp(lp)
    plp = torch.where(p > 0, p * lp, 0.0)
    h = -plp.sum(1)
    h = torch.where(good, h, 0.0)
    h[bad] = float("nan")
    lp = torch.where(good[:, None], lp, NEG)
    lp[bad] = float("nan")
    p = torch.where(good[:, None], p, 0.0)
    out = None
    if targets is not None:
        out = lp.gather(1, targets.long().clamp(0, V - 1)[:, None])[:, 0]
        out[~live] = 0.0
    top = ids = None
    if top_k:
        order = torch.sort(torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=NEG), dim=1, descending=True, stable=True).indices
        ids = order[:, :top_k].clone()
        top = lp.gather(1, ids)
        top[~live] = NEG
        ids[(top == NEG) | torch.isnan(top)] = -1
    return out, h, top, ids, good, p, lp


def logprobs_grad(x, targets, top_k, t, d_lp, d_h, d_top):
    """(gradient, bound of what an fp32 computation of it may be off by, without the output's rounding)."""
    _, h, top, ids, good, p, lp = logprobs(x, targets, top_k, t)
    T, V = x.shape
    g = torch.zeros(T, V, dtype=torch.float64, device=x.device)
    size = torch.zeros(T, dtype=torch.float64, device=x.device)
    sparse = torch.zeros_like(g)
    lpf = torch.where(torch.isinf(lp), 0.0, lp)
    if d_h is not None:
        w = torch.where(good, d_h.double(), 0.0)
        g -= w[:, None] * p * (lpf + h[:, None])
        dense = w.abs()[:, None] * (lpf.abs() + h[:, None] + 1)
    else:
        dense = torch.zeros_like(g)
    if d_lp is not None:
        d = torch.where(good, d_lp.double(), 0.0)
        g -= d[:, None] * p
        sparse.scatter_add_(1, targets.long().clamp(0, V - 1)[:, None], d[:, None])
        size += d.abs()
    if d_top is not None:
        d = torch.where(good[:, None] & (ids >= 0), d_top.double(), 0.0)
        g -= d.sum(1)[:, None] * p
        sparse.scatter_add_(1, ids.clamp(min=0), d)
        size += d.abs().sum(1)
    g += sparse
    rel = 2 * rel_sum(V) + 2.1 * U * 1.4427 * lpf.abs()
    off = (p * (rel + 260 * U) * (size[:, None] + dense) + 260 * U * (sparse != 0) * size[:, None] + 8 * U * g.abs()) / t
    return torch.where(good[:, None], g / t, 0.0), off


def distill(x, values, ids, t, tail):
    """(loss, its gradient, bound of the loss, bound of the gradient) in fp64."""
    x = x.detach().double()
    T, V = x.shape
    loss = torch.zeros(T, dtype=torch.float64)
    loss_off = torch.zeros(T, dtype=torch.float64)
    grad = torch.zeros(T, V, dtype=torch.float64)
    off = torch.zeros(T, V, dtype=torch.float64)
    x, v, ids = x.cpu(), values.detach().double().cpu(), ids.long().cpu()
    r = rel_sum(V)
    for i in range(T):
        at = [k for k in range(ids.shape[1]) if 0 <= int(ids[i, k]) < V]
        if not at:
            continue
        col, val = ids[i, at], v[i, at]
        if tail == "renormalize":
            if bool((val == NEG).all()):
                continue
            q = torch.softmax(val, 0)
        else:
            q = val.exp()
        # from the maximum: ln V is lost beside the type's lowest value, in 64 bits too
        top = float(x[i].max())
        z = (x[i] - (top if math.isfinite(top) else 0.0)) / t
        lp = z - torch.logsumexp(z, 0) if bool((x[i] != NEG).any()) else z
        p = lp.exp()
        spread = torch.where(torch.isinf(lp), 0.0, lp).abs()
        terms = torch.where(q > 0, q * (q.log() - lp[col]), 0.0)
        total = terms.sum()
        size = torch.where(q > 0, q * (q.log().abs() + spread[col] + 1), 0.0).sum()
        g = p.clone()
        w = p.clone()
        q_rest, lift = 0.0, 0.0
        # d(-sum w_k log p_k)/dx_j = (sum of the weights w_k in the loss) p_j - w_j
        weights = float(q.sum()) if tail == "bucket" else 1.0
        outside = torch.ones(V, dtype=torch.bool)
        outside[col] = False
        if tail == "bucket":
            q_rest = max(0.0, 1.0 - float(q.sum()))
            if bool((x[i][outside] != NEG).any()):
                inside_rest = torch.where(outside, z, NEG)
                log_rest = torch.logsumexp(inside_rest, 0) - torch.logsumexp(z, 0)
                share = torch.exp(inside_rest - torch.logsumexp(inside_rest, 0))
                if q_rest > 0:
                    total = total + q_rest * (math.log(q_rest) - log_rest)
                    weights = 1.0
                    g -= q_rest * share
                # 1 - sum q in 32 bits: off by 140 u, whatever is left of it
                lift = 140 * U
                size = size + q_rest * (abs(math.log(q_rest)) if q_rest > 0 else 0.0) + q_rest * abs(float(log_rest))
                loss_off[i] += lift * (abs(float(log_rest)) + 18 + (abs(math.log(q_rest)) if q_rest > 0 else 0.0))
                w += (q_rest + lift / r) * share
        g += (weights - 1.0) * p
        g.scatter_add_(0, col, -q)
        w.scatter_add_(0, col, q)
        loss[i], grad[i] = total, g / t
        loss_off[i] += (4 * r + 140 * U) * float(size)
        off[i] = w * (4 * r + 2.1 * U * 1.4427 * 2 * spread + 140 * U) / t
    return loss, grad, loss_off, off


def check(got, ref, off, what=""):
    """Equal NaNs and infinities, and every other value within `off` + the rounding to its type."""
    ref = ref.to(got.device)
    off = off.to(got.device) if torch.is_tensor(off) else torch.full_like(ref, off)
    g = got.detach().double()
    assert g.shape == ref.shape, what
    # what lies half a step beyond the type's largest number rounds to infinity
    last = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    ref = torch.where(ref.abs() >= last, ref.sign() * float("inf"), ref)
    assert torch.equal(torch.isnan(g), torch.isnan(ref)), f"{what}: NaN in other places"
    whole = torch.isinf(ref)
    assert torch.equal(g[whole], ref[whole]) and not bool(torch.isinf(g[~whole]).any()), f"{what}: infinities"
    fine = ~(whole | torch.isnan(ref))
    room = off[fine] * 1.0 + ref[fine].abs() * (torch.finfo(got.dtype).eps / 2) * 1.001 + smallest(got.dtype)
    worst = ((g[fine] - ref[fine]).abs() / room)
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, f"{what}: {float(worst.max()):.3g} of the tolerance"


def logprob_off(ref, h, V):
    return rel_sum(V) * 1.5 + 4 * U * ref.abs()


def entropy_off(h, V):
    # <|d|> = (H - ln l) / ln 2 is below 1.45 H, the log below rel_sum
    return rel_sum(V) * (1.5 + 4 * h)
