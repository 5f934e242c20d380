"""Results of the operators on rows of logits lie where their definitions put them, and calls at the ends of what is allowed."""
import io

import pytest
import torch

from zenyx_b200.ops.logprobs import distill_topk_fwd_bwd_, token_logprobs

both = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
dtypes = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])


@both
@dtypes
@pytest.mark.parametrize("V", [2, 300, 9001])
def test_no_entropy_below_nothing_and_no_probability_above_one(device, dtype, V):
    """One token with all of the mass, near zero and far from it, where roundings would pass the end of the range."""
    gen = torch.Generator().manual_seed(V)
    T = 400
    size = torch.exp(torch.rand(T, generator=gen) * 13 + 1).clamp(max=6e4 if dtype == torch.float16 else 7e5)
    sign = torch.where(torch.rand(T, generator=gen) < 0.5, -1.0, 1.0)
    y = torch.randint(0, V, (T,), generator=gen)
    x = (torch.randn(T, V, generator=gen) - 200 + (sign * size)[:, None]).clamp(min=-6e4 if dtype == torch.float16 else -8e5)
    x.scatter_(1, y[:, None], (sign * size)[:, None])
    x, y = x.to(dtype).to(device), y.to(device)
    for t in (1.0, 0.7, 3.0):
        out = token_logprobs(x, y, top_k=2, temperature=t)
        assert bool((out.entropy >= 0).all()) and bool((out.logprobs <= 0).all()) and bool((out.top_logprobs <= 0).all())
        assert bool((out.logprobs.exp() <= 1).all())


@both
@pytest.mark.parametrize("T", [1, 3, 4000])
def test_results_have_storages_of_their_own(device, T):
    """What is written to a file is the result and no more, whatever the size of the call."""
    x = torch.randn(T, 60, device=device)
    y = torch.randint(0, 60, (T,), device=device)
    for wants_grad in (False, True):
        out = token_logprobs(x.clone().requires_grad_(wants_grad), y, top_k=2)
        assert len({t.untyped_storage().data_ptr() for t in out}) == 4
        for t in out:
            assert t.storage_offset() == 0 and t.untyped_storage().nbytes() == t.numel() * t.element_size()
            file = io.BytesIO()
            torch.save(t.detach(), file)
            assert file.tell() < t.numel() * t.element_size() + 2048


@pytest.mark.gpu
def test_more_blocks_than_a_grid_holds_are_refused():
    """2^30 + 1 rows (one row, many times) of a vocabulary that takes four blocks a row."""
    x = torch.zeros(1, 400000, device="cuda").expand((1 << 30) + 1, 400000)
    with pytest.raises(RuntimeError, match="launch failed"):
        token_logprobs(x)
    torch.cuda.synchronize()
    assert float(token_logprobs(x[:3]).entropy.max()) > 12      # nothing is left behind


@both
@dtypes
@pytest.mark.parametrize("V,gap", [(100, 0), (101, 3), (50257, 1)])
def test_logits_and_gradient_side_by_side(device, dtype, V, gap):
    """Rows of one buffer: the logits in their first columns, the gradient behind them, and the other way round."""
    T = 5
    x = (torch.randn(T, V, device=device) * 2).to(dtype)
    ids = torch.randint(0, V, (T, 3), device=device)
    values = torch.full((T, 3), -2.0, device=device)
    want = torch.empty_like(x)
    loss = distill_topk_fwd_bwd_(x.clone(), values, ids, 1.0, out=want)
    for logits_first in (True, False):
        buffer = torch.full((T, 2 * V + gap + 5), 9.0, device=device, dtype=dtype)
        a, b = buffer[:, :V], buffer[:, V + gap: 2 * V + gap]
        logits, out = (a, b) if logits_first else (b, a)
        logits.copy_(x)
        got = distill_topk_fwd_bwd_(logits, values, ids, 1.0, out=out)
        assert torch.equal(logits, x) and bool((buffer[:, 2 * V + gap:] == 9).all()) and bool((buffer[:, V: V + gap] == 9).all())
        # rows at other addresses are summed up in another order: V / 128 + 16 roundings along the longest chain, twice
        rel = 2 * (V / 128 + 16) * 2.0 ** -24 + 2.0 ** -20
        assert bool(((got - loss).abs() <= rel * (1 + loss.abs())).all())
        off = (out.float() - want.float()).abs()
        assert bool((off <= (want.float().abs() + 0.5) * rel + want.float().abs() * torch.finfo(dtype).eps).all())


@pytest.mark.gpu
def test_gradients_that_cross_the_logits_are_refused():
    flat = torch.zeros(5 * 220, device="cuda")
    ids, values = torch.zeros(3, 2, device="cuda", dtype=torch.int64), torch.zeros(3, 2, device="cuda")

    def rows(first):
        return flat.as_strided((3, 100), (220, 1), first)

    for first in (110 - 99, 110 + 1, 110 + 99, 110 + 121, 110 + 220):     # the last two reach the next row's logits
        with pytest.raises(RuntimeError, match="overlaps"):
            distill_topk_fwd_bwd_(rows(110), values, ids, 1.0, out=rows(first))
    for first in (110 - 100, 110 + 100, 110 + 120):
        distill_topk_fwd_bwd_(rows(110), values, ids, 1.0, out=rows(first))
    with pytest.raises(RuntimeError, match="overlaps"):                    # rows at another distance
        distill_topk_fwd_bwd_(rows(110), values, ids, 1.0, out=flat.as_strided((3, 100), (230, 1), 210))


@pytest.mark.gpu
@dtypes
@pytest.mark.parametrize("rows", [1, 3])
def test_the_largest_vocabulary(dtype, rows):
    """Every form at the most columns, at an address that no vector divides: eight blocks a row with 200 KB each."""
    import _logprobs_oracle as oracle
    from zenyx_b200.ops import _ext
    from zenyx_b200.ops.logprobs import MAX_TOP, MAX_VOCAB, distill_topk

    V, K = MAX_VOCAB, MAX_TOP
    flat = torch.randn(rows * (V + 1) + 1, device="cuda").mul_(3).to(dtype)
    x = flat[1:].as_strided((rows, V), (V + 1, 1), 1)
    y = torch.randint(0, V, (rows,), device="cuda")
    y[-1] = V - 1
    lp, h, top, ids, *_ = oracle.logprobs(x, y, K, 0.8)
    a = x.detach().requires_grad_(True)
    out = token_logprobs(a, y, top_k=K, temperature=0.8)
    assert torch.equal(out.top_ids, ids)
    oracle.check(out.logprobs, lp, oracle.logprob_off(lp, h, V), "logprobs")
    oracle.check(out.entropy, h, oracle.entropy_off(h, V), "entropy")
    g = [torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda"), torch.randn(rows, K, device="cuda")]
    (got,) = torch.autograd.grad([out.logprobs, out.entropy, out.top_logprobs], a, g)
    oracle.check(got, *oracle.logprobs_grad(x, y, K, 0.8, *g), "gradient")
    values = out.top_logprobs.detach() - 0.1
    for tail in ("renormalize", "bucket"):
        ref, grad, off, grad_off = oracle.distill(x, values, ids, 1.3, tail)
        loss = distill_topk_fwd_bwd_(x, values, ids, 1.0, temperature=1.3, tail=tail, out=(d := torch.empty_like(got)))
        oracle.check(loss, ref, off, "loss")
        oracle.check(d, grad, grad_off, "gradient of the fused form")
        loss = distill_topk(a, values, ids, temperature=1.3, tail=tail)
        oracle.check(loss, ref, off, "loss")
        oracle.check(torch.autograd.grad(loss.sum(), a)[0], grad, grad_off, "gradient")
    _ext.check_status()
