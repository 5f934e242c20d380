"""The operators on rows of logits as autograd functions: the CPU form and the CUDA form notice, refuse and return the same."""
import pytest
import torch
from torch.autograd import forward_ad

from zenyx_b200.ops.logprobs import distill_topk, distill_topk_fwd_bwd_, token_logprobs

both = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])


def _case(device, shape=(2, 3), V=50, K=4, ids=torch.int64, values=torch.float32):
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(*shape, V, generator=gen)
    y = torch.randint(0, V, shape, generator=gen)
    v, k = torch.log_softmax(torch.randn(*shape, V, generator=gen), -1).topk(K)
    return x.to(device), y.to(device), v.to(values).to(device), k.to(ids).to(device)


@both
@pytest.mark.parametrize("shape", [(6,), (2, 3)])
@pytest.mark.parametrize("kind", [(torch.int64, torch.float32), (torch.int32, torch.bfloat16)])
@pytest.mark.parametrize("which", ["teacher_ids", "teacher_logprobs"])
def test_a_teacher_overwritten_before_the_backward_is_noticed(device, shape, kind, which):
    x, _, v, k = _case(device, shape, ids=kind[0], values=kind[1])
    x.requires_grad_(True)
    for tail in ("renormalize", "bucket"):
        loss = distill_topk(x, v, k, tail=tail)
        (k if which == "teacher_ids" else v).zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.sum().backward()


@both
def test_targets_overwritten_before_the_backward_are_noticed(device):
    x, y, _, _ = _case(device)
    x.requires_grad_(True)
    out = token_logprobs(x, y)
    y.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.logprobs.sum().backward()


@both
def test_a_teacher_that_had_to_be_copied_may_be_overwritten(device):
    x, _, v, k = _case(device)
    x.requires_grad_(True)
    (want,) = torch.autograd.grad(distill_topk(x, v, k).sum(), x)
    v2, k2 = v.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(0, 1).contiguous().transpose(0, 1)
    loss = distill_topk(x, v2, k2)
    v2.zero_()
    k2.zero_()
    (got,) = torch.autograd.grad(loss.sum(), x)
    assert torch.equal(got, want)


@both
def test_leaves_that_want_a_gradient_are_not_overwritten(device):
    x, _, v, k = _case(device, (6,))
    leaf, kept = x.clone().requires_grad_(True), x.clone()
    for write in (lambda: distill_topk_fwd_bwd_(leaf, v, k, 1.0), lambda: distill_topk_fwd_bwd_(leaf[:], v, k, 1.0),
                  lambda: distill_topk_fwd_bwd_(x, v, k, 1.0, out=leaf)):
        with pytest.raises(RuntimeError, match="leaf Variable that requires grad"):
            write()
    assert torch.equal(leaf, kept) and torch.equal(x, kept)
    want = torch.empty_like(x)
    loss = distill_topk_fwd_bwd_(x, v, k, 1.0, out=want)
    with torch.no_grad():                       # what an optimizer may do
        assert torch.equal(distill_topk_fwd_bwd_(leaf, v, k, 1.0), loss)
    assert torch.equal(leaf, want)
    inner = kept.clone().requires_grad_(True) * 1.0
    out = distill_topk_fwd_bwd_(inner, v, k, 1.0)
    assert torch.equal(out, loss) and not out.requires_grad and torch.equal(inner, want)


@both
@pytest.mark.parametrize("wants_grad", [False, True])
def test_tangents_are_refused_and_not_dropped(device, wants_grad):
    x, y, v, k = _case(device, (6,))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.clone().requires_grad_(wants_grad), torch.ones_like(x))
        teacher = forward_ad.make_dual(v.clone(), torch.ones_like(v))
        calls = [lambda: token_logprobs(dual, y, top_k=2), lambda: token_logprobs(dual), lambda: distill_topk(dual, v, k),
                 lambda: distill_topk(x, teacher, k), lambda: distill_topk_fwd_bwd_(x.clone(), teacher, k, 1.0),
                 lambda: distill_topk_fwd_bwd_(dual, v, k, 1.0, out=torch.empty_like(x))]
        for call in calls:
            with pytest.raises(NotImplementedError):
                call()
            with pytest.raises(NotImplementedError), torch.no_grad():
                call()
        token_logprobs(x, y)            # what has no tangent goes through
        distill_topk(x, v, k)


@both
def test_function_transforms_are_refused(device):
    x, y, v, k = _case(device, (6,))
    for f in (lambda z: token_logprobs(z, y).logprobs.sum(), lambda z: token_logprobs(z).entropy.sum(),
              lambda z: distill_topk(z, v, k).sum()):
        with pytest.raises(RuntimeError):
            torch.func.grad(f)(x)
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))
    for f in (lambda z: token_logprobs(z).entropy, lambda z: distill_topk(z, v[0], k[0])):
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x)


@pytest.mark.gpu
def test_kernels_of_a_backward_pass_are_counted():
    from zenyx_b200.ops import _ext

    x, y, v, k = _case("cuda")
    x.requires_grad_(True)
    start = _ext.launch_count
    out, loss = token_logprobs(x, y, top_k=2), distill_topk(x, v, k)
    assert _ext.launch_count == start + 2
    out.entropy.sum().backward()
    loss.sum().backward()
    assert _ext.launch_count == start + 4
