"""Scoring over a ring of ranks: each rank's part is what a single process gives for the same positions."""
import pytest
import torch

from zenyx_b200.models import LlamaConfig, LlamaModel
from zenyx_b200.ops.attention import RingContext, shard_sequence

B, S, V, K = 2, 512, 128, 3


def _model():
    cfg = LlamaConfig.tiny(n_layers=2, d_model=64, n_heads=2, n_kv_heads=1, ffn_dim=96, vocab_size=V)
    return LlamaModel(cfg, device="cpu", dtype=torch.float32, seed=7, head_chunk_tokens=100)


def _data():
    gen = torch.Generator().manual_seed(11)
    tokens = torch.randint(0, V, (B, S), generator=gen)
    targets = tokens.roll(-1, 1)
    targets[:, -1] = -100
    targets[1, 40:300] = -100
    return tokens, targets


def _score(rank, world, layout, tmp):
    tokens, targets = _data()
    model, ring = _model(), RingContext(rank=rank, degree=world, seq_len=S, layout=layout)
    cut = lambda x: shard_sequence(x, rank, world, layout).contiguous()  # noqa: E731
    scores = model.token_logprobs(cut(tokens), cut(targets), top_k=K, temperature=1.3, ring=ring)
    torch.save((tuple(scores), model.logits(cut(tokens), ring)), f"{tmp}/{rank}.pt")


@pytest.mark.parametrize("world,layout", [(2, "zigzag"), (2, "contiguous"), (4, "zigzag")])
def test_scores_over_a_ring_are_a_single_processs(tmp_path, world, layout):
    """Logits that are at most d apart have log-probabilities (of logits over a temperature above 1) at most 2 d apart and
    alternatives in the same order where their gaps exceed 2 d; entropies are at most 2 d (1 + the largest |ln p|)
    apart. d itself is the rounding of two layers in another order of sums: below 1e-4 for logits of a few units."""
    import test_dist_cpu

    test_dist_cpu.run_ranks(_score, world=world, args=(layout, str(tmp_path)))
    tokens, targets = _data()
    model = _model()
    want = model.token_logprobs(tokens, targets, top_k=K, temperature=1.3)
    logits = model.logits(tokens)
    for rank in range(world):
        cut = lambda x: shard_sequence(x, rank, world, layout)  # noqa: B023, E731
        (lp, h, top, ids), got_logits = torch.load(tmp_path / f"{rank}.pt")
        d = float((got_logits - cut(logits)).abs().max())
        assert d < 1e-4
        off = 2 * d + 1e-5
        assert lp.shape == (B, S // world) and ids.shape == (B, S // world, K)
        assert float((lp - cut(want.logprobs)).abs().max()) <= off
        least = float(torch.log_softmax(logits / 1.3, -1).abs().max())
        assert float((h - cut(want.entropy)).abs().max()) <= off * (1 + least)
        live = cut(targets) >= 0
        assert bool((lp[~live] == 0).all()) and bool((ids[~live] == -1).all())
        assert float((top - cut(want.top_logprobs))[live].abs().max()) <= off
        best = cut(logits).sort(-1, descending=True).values[..., : K + 1]
        clear = ((best[..., :-1] - best[..., 1:]) > 2 * d).all(-1) & live
        assert float(clear.float().sum()) > 0.5 * float(live.float().sum())
        assert torch.equal(ids[clear], cut(want.top_ids)[clear])
