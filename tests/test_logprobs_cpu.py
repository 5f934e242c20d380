"""Token log-probabilities and distillation on CPU tensors: values, gradients by differences, refusals."""
import math

import pytest
import torch

import _logprobs_oracle as oracle
from zenyx_b200.ops import logprobs as ops
from zenyx_b200.ops.logprobs import distill_topk, distill_topk_fwd_bwd_, token_logprobs

NEG = float("-inf")


def _case(T, V, seed=0, dtype=torch.float64):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, V, generator=gen, dtype=torch.float64) * 3).to(dtype)
    y = torch.randint(0, V, (T,), generator=gen)
    return x, y, gen


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,V,K", [(1, 1, 1), (5, 7, 7), (4, 300, 20), (3, 1000, 128)])
def test_logprobs_values(dtype, T, V, K):
    x, y, _ = _case(T, V, dtype=dtype)
    y[0] = -100
    out = token_logprobs(x, y, top_k=K, temperature=0.7)
    lp, h, top, ids, *_ = oracle.logprobs(x, y, K, 0.7)
    oracle.check(out.logprobs, lp, oracle.logprob_off(lp, h, V), "logprobs")
    oracle.check(out.entropy, h, oracle.entropy_off(h, V), "entropy")
    oracle.check(out.top_logprobs, top, oracle.rel_sum(V) * 1.5 + 4 * oracle.U * 60, "top")
    assert torch.equal(out.top_ids, ids)


def test_logprobs_rows_that_stand_for_nothing():
    V = 9
    x = torch.zeros(6, V)
    x[0] = NEG                       # nothing is left
    x[1, 3:] = NEG                   # three alternatives, all alike
    x[2] = float("nan")              # left out: not looked at
    x[3, 4] = float("nan")
    x[4, 4] = float("inf")
    x[5] = torch.finfo(torch.float32).min
    x[5, 2] = -0.0
    y = torch.tensor([1, 4, -100, 0, 4, 2])
    x.requires_grad_(True)
    out = token_logprobs(x, y, top_k=5)
    assert out.logprobs[0] == NEG and out.entropy[0] == 0 and out.top_ids[0].tolist() == [-1] * 5
    assert out.logprobs[1] == NEG and abs(out.entropy[1].item() - math.log(3)) < 1e-6
    assert out.top_ids[1].tolist() == [0, 1, 2, -1, -1] and out.top_logprobs[1, 3] == NEG
    assert out.logprobs[2] == 0 and out.entropy[2] == 0 and (out.top_ids[2] == -1).all() and (out.top_logprobs[2] == NEG).all()
    for r in (3, 4):
        assert out.logprobs[r].isnan() and out.entropy[r].isnan() and (out.top_ids[r] == -1).all()
        assert out.top_logprobs[r].isnan().all()
    assert out.logprobs[5] == 0 and out.top_ids[5].tolist() == [2, 0, 1, 3, 4]
    rows = torch.tensor([0, 1, 2, 5])
    (out.logprobs[rows].sum() + out.entropy[rows].sum()).backward()
    assert torch.equal(x.grad[0], torch.zeros(V)) and torch.equal(x.grad[2], torch.zeros(V))
    assert torch.isfinite(x.grad[1]).all() and torch.isfinite(x.grad[5]).all()


def test_logprobs_gradient_by_differences():
    x, y, gen = _case(4, 11)
    y[1] = -100
    x[2, 3] = NEG
    y[2] = 5
    x.requires_grad_(True)
    w = torch.randn(4, 3, generator=gen, dtype=torch.float64)

    def f(v):
        v = torch.where(x.detach() == NEG, NEG, v)
        out = token_logprobs(v, y, top_k=3, temperature=1.7)
        top = torch.where(out.top_ids >= 0, out.top_logprobs, 0.0)
        return (out.logprobs * w[:, 0]).sum() + (out.entropy * w[:, 1]).sum() + (top * w).sum()

    assert torch.autograd.gradcheck(f, (torch.nan_to_num(x.detach(), neginf=0.0).requires_grad_(True),))


def test_logprobs_gradient_of_part_of_the_results():
    x, y, gen = _case(3, 40)
    for pick in ("logprobs", "entropy", "top_logprobs"):
        a = x.clone().requires_grad_(True)
        getattr(token_logprobs(a, y, top_k=4), pick).sum().backward()
        ones = torch.ones(3, dtype=torch.float64)
        g, off = oracle.logprobs_grad(x, y, 4, 1.0, ones if pick == "logprobs" else None, ones if pick == "entropy" else None,
                                      torch.ones(3, 4) if pick == "top_logprobs" else None)
        oracle.check(a.grad, g, off, pick)
    out = token_logprobs(x.clone().requires_grad_(True), top_k=2)
    assert out.logprobs is None and out.entropy.requires_grad and not out.top_ids.requires_grad


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_distill_values_and_differences(tail):
    x, _, gen = _case(5, 13)
    teacher = torch.randn(5, 13, generator=gen, dtype=torch.float64)
    values, ids = torch.log_softmax(teacher, 1).topk(4)
    ids = ids.clone()
    ids[1] = -1
    ids[2, 2:] = 13                   # out of range: absent
    ids[3, 1] = ids[3, 0]             # named twice
    values = values.clone()
    values[2, 2:] = float("nan")
    loss = distill_topk(x, values, ids, temperature=1.3, tail=tail)
    ref, grad, off, grad_off = oracle.distill(x, values, ids, 1.3, tail)
    oracle.check(loss, ref, off, "loss")
    assert loss[1] == 0
    a = x.clone().requires_grad_(True)
    w = torch.randn(5, generator=gen, dtype=torch.float64)
    (distill_topk(a, values, ids, temperature=1.3, tail=tail) * w).sum().backward()
    oracle.check(a.grad, grad * w[:, None], grad_off * w.abs()[:, None], "gradient")
    assert torch.autograd.gradcheck(lambda v: distill_topk(v, values, ids, temperature=1.3, tail=tail), (a,))
    b, out = x.clone(), torch.empty_like(x)
    l1 = distill_topk_fwd_bwd_(b, values, ids, 0.25, temperature=1.3, tail=tail, out=out)
    assert torch.equal(b, x) and torch.equal(l1, loss)
    l2 = distill_topk_fwd_bwd_(b, values, ids, 0.25, temperature=1.3, tail=tail)
    assert torch.equal(b, out) and torch.equal(l2, loss)
    oracle.check(out, grad * 0.25, grad_off, "scaled gradient")


def test_distill_rows_that_stand_for_nothing():
    x = torch.zeros(4, 6)
    x[1, 2] = NEG
    x[3] = NEG
    values = torch.log(torch.tensor([[0.5, 0.25]])).repeat(4, 1)
    ids = torch.tensor([[0, 1], [2, 1], [-1, -1], [0, 1]])
    x[2] = float("nan")
    for tail in ("renormalize", "bucket"):
        out = torch.empty_like(x)
        loss = distill_topk_fwd_bwd_(x, values, ids, 1.0, tail=tail, out=out)
        assert loss[1] == float("inf") and loss[2] == 0 and loss[3] == float("inf") and torch.isfinite(loss[0])
        assert torch.isfinite(out).all() and (out[2] == 0).all() and (out[1, 2] < 0)
        assert (out[3, 2:] == 0).all()
    # the student has nothing outside the teacher's tokens
    y = torch.full((1, 6), NEG)
    y[0, :2] = 1.0
    loss = distill_topk(y, values[:1], ids[:1], tail="bucket")
    q = torch.tensor([0.5, 0.25], dtype=torch.float64)
    assert abs(loss.item() - float((q * (q.log() - math.log(0.5))).sum())) < 1e-6
    none = distill_topk(y, torch.full((1, 2), NEG), ids[:1], tail="renormalize")
    assert none.item() == 0


def test_a_teacher_written_down_is_its_own_best_student():
    """token_logprobs of a teacher feeds distill_topk: loss and gradient vanish at the teacher."""
    x, _, _ = _case(6, 50)
    t = 1.5
    out = token_logprobs(x, top_k=8, temperature=t)
    a = x.clone().requires_grad_(True)
    loss = distill_topk(a, out.top_logprobs, out.top_ids, temperature=t, tail="bucket")
    loss.sum().backward()
    assert loss.abs().max() < 1e-14 and a.grad.abs().max() < 1e-15
    shaped = token_logprobs(x.view(2, 3, 50), torch.zeros(2, 3, dtype=torch.int32), top_k=8, temperature=t)
    assert shaped.top_ids.shape == (2, 3, 8) and shaped.logprobs.shape == (2, 3)
    assert torch.equal(shaped.top_ids.view(6, 8), out.top_ids)
    assert token_logprobs(x[0], torch.tensor(3)).logprobs.shape == ()
    empty = token_logprobs(x[:0], torch.zeros(0, dtype=torch.int64), top_k=2)
    assert empty.top_ids.shape == (0, 2)


def test_refusals():
    x, y, _ = _case(3, 20, dtype=torch.float32)
    ids = torch.zeros(3, 2, dtype=torch.int64)
    v = torch.zeros(3, 2)
    for bad in (dict(top_k=21), dict(top_k=-1), dict(temperature=0.0), dict(temperature=float("nan")),
                dict(temperature=float("inf")), dict(ignore_index=5)):
        with pytest.raises(ValueError):
            token_logprobs(x, y, **bad)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(1, 200), top_k=129)
    with pytest.raises(ValueError):
        token_logprobs(x, y[:2])
    with pytest.raises(TypeError):
        token_logprobs(x, y.float())
    with pytest.raises(TypeError):
        token_logprobs(x.long(), y)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(3, 0), None)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(1, 1).expand(1, ops.MAX_VOCAB + 1), None)
    for bad in (lambda: distill_topk(x, v, ids, tail="drop"), lambda: distill_topk(x, v[:, :1], ids),
                lambda: distill_topk(x, v[:2], ids[:2]), lambda: distill_topk(x, v, ids, temperature=-1.0),
                lambda: distill_topk(x, v[:, :0], ids[:, :0]),
                lambda: distill_topk(x, torch.zeros(3, 129), torch.zeros(3, 129, dtype=torch.int64)),
                lambda: distill_topk(x, v.requires_grad_(True), ids),
                lambda: distill_topk_fwd_bwd_(x, v.detach(), ids, 1.0, out=torch.zeros(3, 21)),
                lambda: distill_topk_fwd_bwd_(x, v.detach(), ids, 1.0, out=torch.zeros(3, 20, dtype=torch.bfloat16)),
                lambda: distill_topk_fwd_bwd_(x.t(), torch.zeros(20, 2), torch.zeros(20, 2, dtype=torch.int64), 1.0),
                lambda: distill_topk_fwd_bwd_(x[None], v.detach()[None], ids[None], 1.0)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        distill_topk(x, v.detach(), ids.float())
    with pytest.raises(TypeError):
        distill_topk(x, v.detach().long(), ids)
