"""Scoring over a ring of ranks: each rank's part is what a single process gives for the same positions."""
import pytest
import torch

from zenyx_b200.models import LlamaConfig, LlamaModel
from zenyx_b200.ops.attention import RingContext, shard_sequence

B, S, V, K = 2, 512, 128, 3


def _model(n_layers=2):
    cfg = LlamaConfig.tiny(n_layers=n_layers, d_model=64, n_heads=2, n_kv_heads=1, ffn_dim=96, vocab_size=V)
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


class _Peer:
    """A ring's buffers as the model's host code sees them (the CPU's ring does not use them)."""

    def __init__(self, sequences, log=None):
        self.kv_shape = (sequences, S, 1, 32)
        self.barrier = lambda: log.append("barrier")


@pytest.mark.parametrize("sequences", [1, 2, 3])
def test_more_sequences_than_the_rings_buffers_hold(monkeypatch, sequences):
    model = _model()
    gen = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, V, (5, S), generator=gen)
    want = model.token_logprobs(tokens, tokens, top_k=2)
    seen, layer = [], model._layer_forward
    monkeypatch.setattr(model, "_layer_forward", lambda l, h, B, *a, **kw: (seen.append(B), layer(l, h, B, *a, **kw))[1])
    ring = RingContext(rank=0, degree=1, seq_len=S, peer=_Peer(sequences))
    got = model.token_logprobs(tokens, tokens, top_k=2, ring=ring)
    assert max(seen) == sequences and sum(seen) == 5 * model.cfg.n_layers
    assert torch.equal(got.top_ids, want.top_ids) and torch.allclose(got.logprobs, want.logprobs, rtol=0, atol=1e-4)
    assert model.logits(tokens, ring).shape == (5, S, V)


def test_views_of_a_ring_slot_stay_inside_it():
    """One more sequence than the slot holds would lay K across V."""
    from zenyx_b200.parallel.peer import RingBuffers

    class Memory:
        def tensor(self, rank, offset, shape, dtype):
            return offset, shape

    ring = object.__new__(RingBuffers)
    ring.kv_shape, ring.n, ring.fp8_block_tokens, ring.dtype = (2, 8, 1, 4), 64, 0, torch.bfloat16
    ring.kv_bytes, ring.slot_bytes, ring.dkv_bytes = 128, 256, 256
    ring.staging, ring.kv, ring.dkv = torch.arange(256.0).view(2, 2, 64), Memory(), Memory()
    assert ring.kv_views(0, 1) == ((256, (2, 8, 1, 4)), (384, (2, 8, 1, 4)))
    assert ring.kv_views(0, 0, (1, 8, 1, 4))[1] == (128, (1, 8, 1, 4))
    k, v = ring.staged_kv(1, (1, 8, 1, 4))
    assert torch.equal(k.reshape(-1), torch.arange(128.0, 160)) and torch.equal(v.reshape(-1), torch.arange(192.0, 224))
    for bad in (lambda: ring.kv_views(0, 0, (3, 8, 1, 4)), lambda: ring.staged_kv(0, (3, 8, 1, 4)), lambda: ring.dkv_views(0, 0, (2, 9, 1, 4))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("n_layers", [1, 2, 3])
def test_a_slot_is_not_written_again_while_others_may_pull_from_it(monkeypatch, n_layers):
    """Layer l uses slot l % 2 and starts with a barrier behind its write. Between a slot's use and the next write to it
    there has to be a barrier of another layer, or one for itself."""
    model, log = _model(n_layers), []
    layer = model._layer_forward

    def seen(l, *a, **kw):
        log.append(l % 2)              # the write, and the barrier of ring_attn_forward behind it
        return layer(l, *a, **kw)

    monkeypatch.setattr(model, "_layer_forward", seen)
    ring = RingContext(rank=0, degree=1, seq_len=S, peer=_Peer(1, log))
    model.token_logprobs(torch.zeros(3, S, dtype=torch.long), ring=ring)
    model.logits(torch.zeros(1, S, dtype=torch.long), ring)
    assert sum(e != "barrier" for e in log) == 4 * n_layers
    assert all(a != b for a, b in zip(log, log[1:]))
