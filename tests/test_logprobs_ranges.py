"""Results of the operators on rows of logits lie where their definitions put them, and calls at the ends of what is allowed."""
import io

import pytest
import torch

from zenyx_b200.ops.logprobs import token_logprobs

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
