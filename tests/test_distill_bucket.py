"""The gradient of the bucket form of distillation is the derivative of its loss, whatever the weights and the remainder
add up to: teachers whose rounded weights exceed 1, students with nothing outside the teacher's tokens.

The gradient is held to that of 64-bit autograd through the documented loss, within the bounds of _logprobs_oracle.py."""
import math

import pytest
import torch

import _logprobs_oracle as oracle
from zenyx_b200.ops.logprobs import distill_topk, distill_topk_fwd_bwd_

NEG = float("-inf")


def _loss(x, values, ids, t):
    """Per-row losses as documented, for rows with every entry present."""
    lp = torch.log_softmax(x / t, 1)
    q = values.double().exp()
    rows = (q * (values.double() - lp.gather(1, ids))).sum(1)
    rest = (1.0 - q.sum(1)).clamp(min=0.0)
    outside = torch.ones_like(lp, dtype=torch.bool).scatter(1, ids, False) & (x != NEG)
    parts = []
    for i in range(x.shape[0]):
        some = bool(outside[i].any()) and float(rest[i]) > 0
        parts.append(rest[i] * (rest[i].log() - torch.logsumexp(lp[i][outside[i]], 0)) if some else 0.0 * rest[i])
    return rows + torch.stack(parts)


def _case(T, V, K, dtype, device, value_type, above, seed=0):
    """Rows in turn: the whole vocabulary, the teacher's tokens alone, the teacher's tokens and one more."""
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, V, generator=gen) * 2).to(dtype)
    ids = torch.stack([torch.randperm(V, generator=gen)[:K] for _ in range(T)])
    values = (torch.log_softmax(torch.randn(T, K, generator=gen) * 2, 1) + above).to(value_type)
    for i in range(T):
        if i % 3 and V > K:
            keep = torch.zeros(V, dtype=torch.bool)
            keep[ids[i]] = True
            if i % 3 == 2:
                keep[(~keep).nonzero()[0]] = True
            x[i, ~keep] = NEG
    return x.to(device), values.to(device), ids.to(device)


def _check(x, values, ids, t, scale=0.5):
    a = x.detach().double().cpu().requires_grad_(True)
    v, k = values.cpu(), ids.cpu()
    ref = _loss(a, v, k, t)
    (grad,) = torch.autograd.grad(ref.sum(), a)
    ref = ref.detach()
    grad = torch.where(a.detach() == NEG, torch.where(torch.zeros_like(grad).scatter(1, k, 1.0) > 0, grad, 0.0), grad)
    _, same, off, grad_off = oracle.distill(x, values, ids, t, "bucket")
    assert float((same - grad).abs().max()) < 1e-13
    out = torch.full_like(x, 3.0)
    loss = distill_topk_fwd_bwd_(x, values, ids, scale, temperature=t, tail="bucket", out=out)
    oracle.check(loss, ref, off, "loss")
    oracle.check(out, grad * scale, grad_off * scale, "gradient")
    b = x.detach().requires_grad_(True)
    loss = distill_topk(b, values, ids, temperature=t, tail="bucket")
    (got,) = torch.autograd.grad(loss.sum(), b)
    oracle.check(loss, ref, off, "loss of the autograd form")
    oracle.check(got, grad, grad_off, "gradient of the autograd form")
    # a gradient through a softmax adds up to nothing
    g, half = got.double().cpu(), torch.finfo(x.dtype).eps / 2
    room = (grad_off + grad.abs() * half * 1.001 + oracle.smallest(x.dtype)).sum(1)
    assert bool((g.sum(1).abs() <= room).all())


SIZES = [(3, 2, 2), (6, 4, 2), (6, 130, 128), (6, 1000, 17)]


@pytest.mark.parametrize("value_type,above", [(torch.bfloat16, 0.0), (torch.float16, 0.0), (torch.float32, 0.05), (torch.float32, -0.7)])
@pytest.mark.parametrize("T,V,K", SIZES)
def test_gradient_of_the_cpu_form(T, V, K, value_type, above):
    for dtype in (torch.float64, torch.float32, torch.bfloat16):
        _check(*_case(T, V, K, dtype, "cpu", value_type, above), t=1.0)
    _check(*_case(T, V, K, torch.float32, "cpu", value_type, above, seed=1), t=1.7)


@pytest.mark.parametrize("above", [0.05, -0.3])
def test_cpu_form_by_differences(above):
    x, values, ids = _case(6, 9, 3, torch.float64, "cpu", torch.float64, above)
    free = torch.nan_to_num(x, neginf=0.0).requires_grad_(True)
    assert torch.autograd.gradcheck(
        lambda v: distill_topk(torch.where(x == NEG, NEG, v), values, ids, temperature=1.3, tail="bucket"), (free,))


def test_two_rows_by_hand():
    out = torch.empty(1, 4)
    ids = torch.tensor([[0, 1]])
    v = torch.full((1, 2), math.log(0.5)).bfloat16()         # exp of the rounded values: 0.50088 each
    distill_topk_fwd_bwd_(torch.zeros(1, 4), v, ids, 1.0, tail="bucket", out=out)
    q = v.double().exp()
    want = q.sum() * 0.25 - torch.tensor([float(q[0, 0]), float(q[0, 1]), 0.0, 0.0])
    assert float(q.sum()) > 1.001 and torch.allclose(out[0].double(), want.double(), rtol=0, atol=1e-6)
    x = torch.tensor([[1.0, 0.0, NEG, NEG]])
    distill_topk_fwd_bwd_(x, torch.log(torch.tensor([[0.5, 0.25]])), ids, 1.0, tail="bucket", out=out)
    p = 1 / (1 + math.exp(-1.0))
    want = torch.tensor([0.75 * p - 0.5, 0.75 * (1 - p) - 0.25, 0.0, 0.0])
    assert torch.allclose(out[0], want, rtol=0, atol=1e-6)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("t", [1.0, 1.5])
@pytest.mark.parametrize("V,K", [(9, 2), (1000, 40), (50257, 128)])
def test_the_remainder_of_a_peaked_teacher(device, V, K, t):
    """What the bucket has left is off by half a step where it is small, and by the roundings of a sum of 128 weights
    (140 u, u = 2^-24) of at least a quarter, 560 u of itself, where it is not. So is its part of the gradient,
    q_r p_j / p_r, on top of the bounds of the logits' own sums (_logprobs_oracle.py)."""
    U = oracle.U
    left = [0.9, 0.3, 0.26, 0.24, 0.1, 1e-2, 1e-3, 1e-4, 1e-5, 1e-6, 3e-7]
    gen = torch.Generator().manual_seed(K)
    T = len(left)
    ids = torch.stack([torch.randperm(V, generator=gen)[:K] for _ in range(T)])
    spread = torch.softmax(torch.randn(T, K, generator=gen, dtype=torch.float64), 1)
    left = torch.tensor(left, dtype=torch.float64)[:, None]
    values = torch.log(spread * (1 - left)).float()
    # the student has learnt most of it: twice the teacher's remainder lies outside
    z = torch.randn(T, V, generator=gen, dtype=torch.float64).scatter(1, ids, NEG)
    z = (torch.log_softmax(z, 1) + torch.log(2 * left)).scatter(1, ids, values.double() + 0.3 * torch.randn(T, K, generator=gen))
    x = (z * t).float()
    a = x.double().requires_grad_(True)
    ref = _loss(a, values, ids, t)
    (grad,) = torch.autograd.grad(ref.sum(), a)
    rest = 1 - values.double().exp().sum(1)
    assert bool((rest > 2e-7).all())
    lp = torch.log_softmax(x.double() / t, 1)
    outside = lp.scatter(1, ids, NEG)
    share = torch.softmax(outside, 1)
    r = oracle.rel_sum(V)
    rounding = 4 * r + 2.1 * U * 1.4427 * 2 * lp.abs() + 140 * U
    inside = torch.zeros_like(lp).scatter(1, ids, values.double().exp())
    off = ((lp.exp() + inside) * rounding + rest[:, None] * share * (rounding + 560 * U)) / t
    loss = distill_topk_fwd_bwd_(x.to(device), values.to(device), ids.to(device), 1.0, temperature=t, tail="bucket",
                                 out=(out := torch.empty(T, V, device=device)))
    oracle.check(out, grad, off, "gradient")
    terms = inside * (inside.clamp(min=1e-300).log().abs() + lp.abs() + 1)
    log_rest = torch.logsumexp(outside, 1)
    size = terms.sum(1) + rest * (rest.log().abs() + log_rest.abs())
    # d(q_r (log q_r - log p_r)) = (log q_r + 1 - log p_r) dq_r
    off = (4 * r + 140 * U) * size + 560 * U * rest * (rest.log().abs() + 1 + log_rest.abs())
    oracle.check(loss, ref.detach(), off, "loss")


@pytest.mark.gpu
@pytest.mark.parametrize("value_type,above", [(torch.bfloat16, 0.0), (torch.float16, 0.0), (torch.float32, 0.05), (torch.float32, -0.7)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,V,K", SIZES + [(6, 50257, 64), (3, 128256, 128)])
def test_gradient_of_the_kernels(T, V, K, dtype, value_type, above):
    from zenyx_b200.ops import _ext

    for t in (1.0, 1.7):
        _check(*_case(T, V, K, dtype, "cuda", value_type, above, seed=V), t=t)
    _ext.check_status()
