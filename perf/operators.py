"""Operators on the logits of a language-model head, as cases that can be timed and compared.

A case is a dict of plain values. ``prepare(case, seed)`` makes what a user's program holds before the call,
``run(state)`` is one pass: the framework's entry points where ``own`` is true, elementary torch in 32 bits otherwise.
``exact(case, seed)`` is the same pass from the definition in 64 bits, ``work(case)`` the bytes and operations the
pass cannot do without. ``listed()`` are the cases quoted in the documentation, ``draw(rng)`` gives more of the same
ranges.

Two kinds of work, on logits ``x`` [rows, vocab] at temperature t (z = x / t, lse = log sum exp z, p = exp(z - lse)):

* ``logprobs``  ``token_logprobs``: per row z - lse of a given token, the entropy of p, and the ``top`` most likely
                tokens with their log-probabilities (ties: the lower token first); with ``backward`` also the gradient
                of all of it with respect to the logits. Rows whose target is the ignore index are left out.
* ``distill``   ``distill_topk_fwd_bwd_``: the Kullback-Leibler divergence from a teacher, of which the ``top`` most likely
                tokens and their log-probabilities were written down, to p, and its gradient. ``renormalize`` makes
                the teacher's tokens a distribution of their own; ``bucket`` takes all other tokens as one.
                Entries of -1 are absent; rows without an entry are left out.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100
NEG = float("-inf")


def listed():
    return [
        # scoring with the 8B shape: one chunk of its LM head, log-probabilities and entropies (perplexity, rewards)
        dict(name="score_head_chunk", kind="logprobs", rows=4096, vocab=128256, dtype="bf16", top=0, backward=False,
             ignored=0.0, banned=0.0, temperature=1.0),
        # a teacher writes down its 64 most likely tokens for the same chunk; padding at the end of the sequences
        dict(name="teacher_head_chunk", kind="logprobs", rows=4096, vocab=128256, dtype="bf16", top=64, backward=False,
             ignored=0.05, banned=0.0, temperature=1.0),
        # one generated token and its 20 alternatives, some tokens forbidden: latency
        dict(name="one_token", kind="logprobs", rows=1, vocab=128256, dtype="bf16", top=20, backward=False, ignored=0.0,
             banned=0.01, temperature=0.7),
        # a batch of generated tokens, logits already in fp32 behind a sampler's penalties
        dict(name="batch_of_tokens", kind="logprobs", rows=64, vocab=128256, dtype="fp32", top=20, backward=False,
             ignored=0.0, banned=0.01, temperature=1.0),
        # a policy-gradient step with an entropy bonus on the 8B shape: forward, then the gradient
        dict(name="policy_step", kind="logprobs", rows=2048, vocab=128256, dtype="bf16", top=0, backward=True,
             ignored=0.3, banned=0.0, temperature=1.0),
        # a vocabulary that no vector divides (rows start on odd addresses), alternatives with a gradient
        dict(name="policy_step_odd_vocab", kind="logprobs", rows=999, vocab=50257, dtype="fp16", top=5, backward=True,
             ignored=0.1, banned=0.0, temperature=1.3),
        # a mid-sized model's logits in fp32, forward and gradient
        dict(name="policy_step_fp32", kind="logprobs", rows=1024, vocab=32000, dtype="fp32", top=0, backward=True,
             ignored=0.0, banned=0.0, temperature=1.0),
        # distillation on one chunk of the 8B shape's head
        dict(name="distill_head_chunk", kind="distill", rows=4096, vocab=128256, dtype="bf16", top=64, tail="bucket",
             ids="int32", values="fp32", absent=0.05, temperature=1.0),
        # softened distributions, odd vocabulary, few alternatives
        dict(name="distill_odd_vocab", kind="distill", rows=777, vocab=50257, dtype="bf16", top=17, tail="renormalize",
             ids="int64", values="fp32", absent=0.1, temperature=2.0),
        # a mid-sized model, fp32 logits, the most alternatives
        dict(name="distill_fp32", kind="distill", rows=1024, vocab=32000, dtype="fp32", top=128, tail="bucket",
             ids="int64", values="bf16", absent=0.0, temperature=1.0),
        # the fine-tuning example's vocabulary: a step that is all latency
        dict(name="distill_tiny", kind="distill", rows=256, vocab=512, dtype="bf16", top=8, tail="renormalize",
             ids="int64", values="fp32", absent=0.0, temperature=1.0),
    ]


MOST_BYTES = 4096 * 128256 * 2


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    size = 4 if dtype == "fp32" else 2
    vocab = _log(rng, 512, 160000)
    if rng.random() < 0.5:
        vocab = max(512, vocab // 128 * 128)
    rows = _log(rng, 1, min(8192, MOST_BYTES // (vocab * size)))
    c = dict(kind=rng.choice(("logprobs", "logprobs", "distill")), rows=rows, vocab=vocab, dtype=dtype,
             temperature=rng.choice((1.0, 1.0, 0.6, 1.5, 2.0)))
    if c["kind"] == "logprobs":
        c.update(top=rng.choice((0, 0, 1, _log(rng, 2, 128))), backward=rng.random() < 0.5,
                 ignored=rng.choice((0.0, 0.1, 0.5)), banned=rng.choice((0.0, 0.01, 0.3)))
    else:
        c.update(top=_log(rng, 1, 128), tail=rng.choice(("bucket", "renormalize")), ids=rng.choice(("int32", "int64")),
                 values=rng.choice(("fp32", "bf16")), absent=rng.choice((0.0, 0.1, 0.5)))
    return c


# ------------------------------------------------------------------------------------------------


def _logits(case, gen):
    """What a trained head gives: a spread of a few units, the frequent (low) tokens above the rare ones."""
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=gen, device="cuda").mul_(2.0)
    return x.sub_(torch.arange(vocab, device="cuda", dtype=torch.float32).add_(1.0).log_().mul_(0.5))


def _some_rows(share, rows, gen):
    """About that share of the rows, never the first: a call without a live row measures nothing."""
    some = torch.rand(rows, generator=gen, device="cuda") < share
    some[0] = False
    return some


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    x = _logits(case, gen)
    if case["kind"] == "logprobs":
        targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        # the model has learnt something: the given token stands out, more in some rows than in others
        lift = torch.rand(rows, 1, generator=gen, device="cuda").mul_(12.0)
        x.scatter_add_(1, targets[:, None], lift)
        if case["banned"] > 0:
            x.masked_fill_((torch.rand(vocab, generator=gen, device="cuda") < case["banned"])[None, :], NEG)
        if case["ignored"] > 0:
            targets.masked_fill_(_some_rows(case["ignored"], rows, gen), IGNORE)
        s = dict(case=case, logits=x.to(dtype), targets=targets)
        if case["backward"]:
            s["logits"].requires_grad_(True)
            s["grads"] = [torch.randn(rows, generator=gen, device="cuda"),
                          torch.randn(rows, generator=gen, device="cuda").mul_(0.01)]
            if case["top"] > 0:
                s["grads"].append(torch.randn(rows, case["top"], generator=gen, device="cuda"))
        return s
    # the teacher agrees with the student up to some noise
    teacher = torch.randn(rows, vocab, generator=gen, device="cuda").add_(x).div_(case["temperature"])
    values, ids = teacher.topk(case["top"], dim=1)
    values = values - torch.logsumexp(teacher, dim=1, keepdim=True)
    del teacher
    if case["absent"] > 0:
        ids.masked_fill_(_some_rows(case["absent"], rows, gen)[:, None], -1)
        # some rows have fewer alternatives than others
        least = 1 + (torch.rand(rows, 1, generator=gen, device="cuda") * 4 * case["top"]).long()
        ids.masked_fill_(torch.arange(case["top"], device="cuda")[None, :] >= least, -1)
    x = x.to(dtype)
    return dict(case=case, logits=x, grad=torch.empty_like(x), values=values.to(DTYPES[case["values"]]),
                ids=ids.to(torch.int32 if case["ids"] == "int32" else torch.int64), scale=1.0 / rows)


def run(state):
    case = state["case"]
    if case["kind"] == "logprobs":
        return _run_logprobs(state, case)
    return _run_distill(state, case)


def _run_logprobs(s, case):
    if own:
        from zenyx_b200.ops.logprobs import token_logprobs

        out = token_logprobs(s["logits"], s["targets"], top_k=case["top"], temperature=case["temperature"],
                             ignore_index=IGNORE)
        outs = [out.logprobs, out.entropy] + ([out.top_logprobs, out.top_ids] if case["top"] > 0 else [])
        if case["backward"]:
            outs.append(torch.autograd.grad([o for o in outs if o.requires_grad], s["logits"], s["grads"])[0])
        return outs
    return _plain_logprobs(s, case)


def _plain_logprobs(s, case):
    t = case["temperature"]
    raw, targets = s["logits"].detach(), s["targets"]
    live = (targets >= 0) & (targets < raw.shape[1])
    at = targets.clamp(0, raw.shape[1] - 1)[:, None]
    z = raw.float() / t
    top = z.amax(dim=1, keepdim=True)
    z = z - top
    e = z.exp()
    total = e.sum(dim=1, keepdim=True)
    lp = z - total.log()
    p = e / total
    del z, e
    logprobs = torch.where(live, lp.gather(1, at)[:, 0], 0.0)
    plogp = torch.where(p > 0, p * lp, 0.0)
    entropy = torch.where(live, -plogp.sum(dim=1), 0.0)
    outs = [logprobs, entropy]
    k = case["top"]
    if k > 0:
        # order-preserving whole numbers of the logits, the column below them: no two are alike
        bits = (raw.float() + 0.0).view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32)
        key += (1 << 31) - torch.arange(raw.shape[1], device=raw.device)
        ids = key.topk(k, dim=1).indices
        del key, bits
        top_lp = lp.gather(1, ids)
        there = live[:, None] & (top_lp > NEG)
        ids = torch.where(there, ids, -1)
        outs += [torch.where(there, top_lp, NEG), ids]
    if case["backward"]:
        g, h = [torch.where(live, x, 0.0)[:, None] for x in s["grads"][:2]]
        d = -h * (plogp + p * entropy[:, None])
        coefficient = g
        if k > 0:
            c = torch.where(there, s["grads"][2], 0.0)
            coefficient = g + c.sum(dim=1, keepdim=True)
            d.scatter_add_(1, ids.clamp(min=0), c)
        d -= coefficient * p
        d.scatter_add_(1, at, g)
        outs.append((d / t).to(raw.dtype))
    return outs


def _run_distill(s, case):
    if own:
        from zenyx_b200.ops.logprobs import distill_topk_fwd_bwd_

        loss = distill_topk_fwd_bwd_(s["logits"], s["values"], s["ids"], s["scale"], temperature=case["temperature"],
                                     tail=case["tail"], out=s["grad"])
        return [loss, s["grad"]]
    return _plain_distill(s, case)


def _plain_distill(s, case):
    t = case["temperature"]
    x, ids = s["logits"], s["ids"].long()
    there = (ids >= 0) & (ids < x.shape[1])
    at = torch.where(there, ids, 0)
    v = torch.where(there, s["values"].float(), NEG)
    live = there.any(dim=1)
    z = x.float() / t
    z = z - z.amax(dim=1, keepdim=True)
    e = z.exp()
    total = e.sum(dim=1, keepdim=True)
    lse = total.log()
    if case["tail"] == "renormalize":
        q = (v - torch.where(live[:, None], v.amax(dim=1, keepdim=True), 0.0)).exp()
        q = q / q.sum(dim=1, keepdim=True).clamp(min=1e-30)
    else:
        q = v.exp()
    lp = z.gather(1, at) - lse
    loss = torch.where(q > 0, q * (q.log() - lp), 0.0).sum(dim=1)
    p = e / total
    del z, e
    if case["tail"] == "bucket":
        q_rest = (1.0 - q.sum(dim=1)).clamp(min=0.0)
        outside = torch.ones_like(p).scatter_reduce_(1, at, 1.0 - there.float(), "amin")
        p_rest = (p * outside).sum(dim=1)
        log_rest = torch.where(q_rest > 0, q_rest * (q_rest.log() - p_rest.log()), 0.0)
        loss = loss + torch.where(p_rest > 0, log_rest, 0.0)
        ratio = torch.where(p_rest > 0, q_rest / p_rest, 0.0)
        p -= p * outside * ratio[:, None]
        del outside
    p.scatter_add_(1, at, -q)
    grad = torch.where(live[:, None], p * (s["scale"] / t), 0.0)
    return [torch.where(live, loss, 0.0), grad.to(x.dtype)]


# ------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    x = s["logits"].detach().double()
    if case["kind"] == "logprobs":
        return _exact_logprobs(case, s, x)
    return _exact_distill(case, s, x)


def _exact_logprobs(case, s, x):
    rows, vocab = x.shape
    t, k, targets = case["temperature"], case["top"], s["targets"]
    live = targets != IGNORE
    row = torch.arange(rows, device=x.device)
    y = torch.where(live, targets, torch.zeros_like(targets))
    lp = torch.log_softmax(x / t, dim=1)
    p = lp.exp()
    finite = torch.where(torch.isinf(lp), torch.zeros_like(lp), lp)
    h = -(p * finite).sum(dim=1)
    outs = [lp[row, y] * live if not case["banned"] else torch.where(live, lp[row, y], torch.zeros_like(h)), h * live]
    if k:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
        best = torch.gather(lp, 1, order)
        keep = live[:, None] & ~torch.isinf(best)
        outs.append(best.masked_fill(~keep, NEG))
        outs.append(order.masked_fill(~keep, -1))
    if case["backward"]:
        g = s["grads"][0].double() * live
        w = s["grads"][1].double() * live
        d = -p * g[:, None] - w[:, None] * p * (finite + h[:, None])
        d[row, y] += g
        if k:
            c = s["grads"][2].double() * keep
            d -= p * c.sum(dim=1)[:, None]
            d[row[:, None], order] += c      # the columns of one row are distinct
        outs.append(d / t)
    return outs


def _exact_distill(case, s, x):
    rows, vocab = x.shape
    t = case["temperature"]
    ids, values = s["ids"].long(), s["values"].double()
    valid = ids != -1
    live = valid.any(dim=1)
    row = torch.arange(rows, device=x.device)[:, None].expand_as(ids)
    teacher = torch.zeros_like(x)
    if case["tail"] == "renormalize":
        weight = torch.softmax(values.masked_fill(~valid, NEG), dim=1)
    else:
        weight = values.exp()
    teacher[row[valid], ids[valid]] = weight[valid]      # the columns of one row are distinct
    member = torch.zeros(rows, vocab, dtype=torch.bool, device=x.device)
    member[row[valid], ids[valid]] = True
    lp = torch.log_softmax(x / t, dim=1)
    loss = (torch.xlogy(teacher, teacher) - teacher * lp).sum(dim=1)
    grad = lp.exp() - teacher
    if case["tail"] == "bucket":
        rest = torch.clamp(1.0 - teacher.sum(dim=1), min=0.0)
        log_rest = torch.logsumexp(lp.masked_fill(member, NEG), dim=1)
        loss += torch.xlogy(rest, rest) - rest * log_rest
        inside = torch.exp(lp - log_rest[:, None]).masked_fill(member, 0.0)
        grad -= rest[:, None] * inside
    grad = grad * (s["scale"] / t)
    return [loss.masked_fill(~live, 0.0), grad.masked_fill(~live[:, None], 0.0)]


def work(case):
    rows, vocab, k = case["rows"], case["vocab"], case["top"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "logprobs":
        live = rows * (1.0 - case["ignored"])
        read = live * vocab * size + rows * 8
        write = rows * 8 + rows * k * 12
        flops = 5.0 * live * vocab                       # subtract, exponential, two sums, one product
        if case["backward"]:
            read += rows * 8 + rows * k * 4
            write += rows * vocab * size
            flops += 6.0 * live * vocab
        return {"bytes": read + write, "flops": flops}
    live = rows * (1.0 - case["absent"])
    entry = (4 if case["ids"] == "int32" else 8) + (2 if case["values"] == "bf16" else 4)
    return {"bytes": live * vocab * size + rows * vocab * size + rows * k * entry + rows * 4,
            "flops": 6.0 * live * vocab}
