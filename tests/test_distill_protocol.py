"""How the blocks of a cluster hand on rows in the distillation kernel (csrc/head/distill.cu)."""
import re
from pathlib import Path

import pytest
import torch

CSRC = Path(__file__).resolve().parent.parent / "csrc"


def test_arrivals_on_another_blocks_barrier_release():
    """What a block has read of its shared memory must come before its arrival on the barrier that lets another block write
    there again: the arrival is a release at the scope of the cluster."""
    seen = 0
    for path in [*CSRC.rglob("*.cu"), *CSRC.rglob("*.cuh")]:
        for op in re.findall(r"mbarrier\.arrive\S*shared::cluster\S*", path.read_text()):
            seen += 1
            assert ".release.cluster." in op, f"{path.name}: {op}"
    assert seen > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 50257), (torch.float32, 128256), (torch.float16, 262147)])
def test_rows_handed_on_while_most_are_left_out(dtype, V):
    """Two, eight and eight blocks a row. Rows that are left out have no exchange that would keep the blocks together; each
    row's loss and gradient are those of a call for that row alone, up to the order of the sums."""
    from zenyx_b200.ops import _ext
    from zenyx_b200.ops.logprobs import distill_topk_fwd_bwd_

    rows = 2000
    gen = torch.Generator(device="cuda").manual_seed(V)
    x = (torch.randn(4, V, generator=gen, device="cuda") * 3).to(dtype)
    ids = torch.randint(0, V, (rows, 3), generator=gen, device="cuda")
    values = torch.full((rows, 3), -1.5, device="cuda")
    ids[torch.rand(rows, generator=gen, device="cuda") < 0.98] = -1
    ids[-1, 0] = 5
    big = x.repeat(rows // 4, 1)
    loss = distill_topk_fwd_bwd_(big, values, ids, 1.0, tail="bucket")
    _ext.check_status()
    live = (ids >= 0).any(1)
    assert bool(live.any()) and not bool(loss[~live].any()) and bool((loss[live] > 0).all())
    for r in range(rows):
        if not live[r]:
            assert not bool(big[r].any())
            continue
        one = x[r % 4].clone()[None]
        alone = distill_topk_fwd_bwd_(one, values[r: r + 1], ids[r: r + 1], 1.0, tail="bucket")
        # a sum of V exponentials in any order: V / 128 + 16 roundings along its longest chain, twice; a weight is below 1 / 4
        rel = 2 * (V / 128 + 16) * 2.0 ** -24 + 2.0 ** -20
        assert abs(float(alone) - float(loss[r])) <= rel * (1 + abs(float(alone)))
        off = (one[0].float() - big[r].float()).abs()
        assert bool((off <= (one[0].float().abs() + 0.25) * rel + one[0].float().abs() * torch.finfo(dtype).eps + 2.0 ** -24).all())
    _ext.check_status()
