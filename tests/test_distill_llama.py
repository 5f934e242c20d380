"""Scoring and distillation through the flagship model, the engine and the Trainer: CPU in fp32 against autograd on the same
math, and on a GPU in bf16 against the logits that the model itself gives."""
import pytest
import torch

import _logprobs_oracle as oracle
import test_llama_cpu
from zenyx_b200.models import LlamaConfig, LlamaModel
from zenyx_b200.ops.logprobs import distill_topk
from zenyx_b200.train import Trainer, TrainerConfig


def _tiny(device="cpu", dtype=torch.float32, seed=0, **kw):
    cfg = LlamaConfig.tiny(n_layers=2, d_model=64, n_heads=2, n_kv_heads=1, ffn_dim=96, vocab_size=128)
    return LlamaModel(cfg, device=device, dtype=dtype, seed=seed, head_chunk_tokens=100, **kw)


def _tokens(B=2, S=128, V=128, device="cpu"):
    gen = torch.Generator().manual_seed(3)
    return torch.randint(0, V, (B, S), generator=gen).to(device)


def test_model_token_logprobs_match_its_logits():
    model, tokens = _tiny(), _tokens()
    targets = tokens.roll(-1, 1)
    targets[:, -1] = -100
    out = model.token_logprobs(tokens, targets, top_k=7, temperature=1.5)
    lp, h, top, ids, *_ = oracle.logprobs(model.logits(tokens).view(-1, 128), targets.view(-1), 7, 1.5)
    assert out.logprobs.shape == (2, 128) and out.top_ids.shape == (2, 128, 7)
    oracle.check(out.logprobs.view(-1), lp, oracle.logprob_off(lp, h, 128), "logprobs")
    oracle.check(out.entropy.view(-1), h, oracle.entropy_off(h, 128), "entropy")
    oracle.check(out.top_logprobs.view(-1, 7), top, oracle.rel_sum(128) * 1.5 + 4 * oracle.U * 20, "top")
    assert torch.equal(out.top_ids.view(-1, 7), ids)
    assert model.token_logprobs(tokens).logprobs is None
    with pytest.raises(ValueError):
        model.token_logprobs(tokens, targets[:, :-1])


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_model_distillation_against_autograd(monkeypatch, tail):
    teacher, model, tokens = _tiny(seed=5), _tiny(seed=1), _tokens()
    wrote = teacher.token_logprobs(tokens, top_k=6, temperature=2.0)
    ids = wrote.top_ids.clone()
    ids[1, 100:] = -1                           # padding
    loss_of = lambda logits, _: distill_topk(logits.double(), wrote.top_logprobs.double().view(-1, 6), ids.view(-1, 6),  # noqa: E731
                                             temperature=2.0, tail=tail).mean().float()
    monkeypatch.setattr(torch.nn.functional, "cross_entropy", loss_of)
    ref_loss, ref_grads = test_llama_cpu._torch_reference_loss(model, tokens, tokens)
    monkeypatch.undo()
    model.zero_grad()
    loss = model.forward_backward_distill(tokens, wrote.top_logprobs, ids, temperature=2.0, tail=tail)
    assert abs(loss.item() - ref_loss.item()) < 1e-5 * max(1.0, abs(ref_loss.item()))
    for n, _ in model.named_flat_parameters():
        err = (model.g(n) - ref_grads[n]).norm() / (ref_grads[n].norm() + 1e-12)
        assert err < 2e-4, (n, err.item())
    with pytest.raises(ValueError):
        model.forward_backward_distill(tokens, wrote.top_logprobs[:1], ids)


def test_trainer_distill_step_is_train_step_with_another_loss():
    cfg = LlamaConfig.tiny(n_layers=1, d_model=64, n_heads=2, n_kv_heads=1, ffn_dim=96, vocab_size=128)
    trainer = Trainer(cfg, TrainerConfig(lr=1e-3, seq_len=128, global_batch=2))
    tokens = _tokens()
    wrote = trainer.model.token_logprobs(tokens, top_k=4)
    before = trainer.model.w("lm_head.weight").clone()
    loss = trainer.distill_step(tokens, wrote.top_logprobs, wrote.top_ids.int(), tail="bucket")
    assert abs(loss) < 1e-2 and trainer.step == 1      # bf16 weights: the teacher is the model itself
    assert not torch.equal(before, trainer.model.w("lm_head.weight")) or loss == 0
    trainer.close()
    generic = Trainer(torch.nn.Linear(4, 4), TrainerConfig())
    with pytest.raises(ValueError):
        generic.distill_step(tokens, wrote.top_logprobs, wrote.top_ids)


@pytest.mark.gpu
def test_scoring_and_distillation_of_the_bf16_model():
    """The whole run as it is used: a teacher scores and writes down its tokens, a student's step on them. The head's
    weight gradient is dlogits^T h with h and dlogits in bf16: a rounding of dlogits is off by at most 2^-8 of itself, so
    the product's error stays below 2^-8 of |dlogits|^T |h|, plus fp32 sums over 512 tokens."""
    cfg = LlamaConfig.tiny(n_layers=2, d_model=256, n_heads=2, n_kv_heads=1, ffn_dim=512, vocab_size=1000)
    teacher = LlamaModel(cfg, device="cuda", seed=1, head_chunk_tokens=200)
    student = LlamaModel(cfg, device="cuda", seed=2, head_chunk_tokens=200)
    tokens = _tokens(2, 256, 1000, "cuda")
    targets = tokens.roll(-1, 1)
    targets[:, -1] = -100
    out = teacher.token_logprobs(tokens, targets, top_k=16, temperature=1.5)
    lp, h, top, ids, *_ = oracle.logprobs(teacher.logits(tokens).view(-1, 1000), targets.view(-1), 16, 1.5)
    oracle.check(out.logprobs.view(-1), lp, oracle.logprob_off(lp, h, 1000), "logprobs")
    assert torch.equal(out.top_ids.view(-1, 16), ids)
    logits = student.logits(tokens).view(-1, 1000)
    hn = student.forward(tokens).view(-1, cfg.d_model)
    ref, grad, off, grad_off = oracle.distill(logits, out.top_logprobs.view(-1, 16), out.top_ids.view(-1, 16), 1.5, "bucket")
    student.zero_grad()
    loss = student.forward_backward_distill(tokens, out.top_logprobs, out.top_ids, 1.0, temperature=1.5, tail="bucket")
    assert abs(loss.item() - ref.sum().item()) < off.sum().item() + 512 * 2.0 ** -24 * ref.abs().sum().item()
    got = student.g("lm_head.weight").double().cpu()
    hd = hn.double().cpu()
    want = grad.t() @ hd
    room = (grad.abs() * 2.0 ** -8 + grad_off).t() @ hd.abs() + 600 * 2.0 ** -24 * (grad.abs().t() @ hd.abs())
    assert bool(((got - want).abs() <= room).all()), float(((got - want).abs() / room).max())
    for n, _ in student.named_flat_parameters():
        assert torch.isfinite(student.g(n)).all(), n


@pytest.mark.gpu
def test_trainer_distill_step_on_the_gpu():
    from zenyx_b200.ops import _ext

    cfg = LlamaConfig.tiny(n_layers=2, d_model=256, n_heads=2, n_kv_heads=1, ffn_dim=512, vocab_size=1024)
    teacher = LlamaModel(cfg, device="cuda", seed=1)
    trainer = Trainer(cfg, TrainerConfig(lr=1e-3, seq_len=256, global_batch=2, max_grad_norm=1.0))
    tokens = _tokens(2, 256, 1024)
    wrote = teacher.token_logprobs(tokens.cuda(), top_k=8)
    for _ in range(2):      # teacher data from the host, as a file of it would come
        loss = trainer.distill_step(tokens, wrote.top_logprobs.cpu(), wrote.top_ids.int().cpu(), tail="bucket")
        assert loss == loss and loss > 0
    _ext.check_status()
    trainer.close()


def _distill_ranks(rank, world, cp, tmp):
    """Replicas, or one sequence over a ring: the tokens and what the teacher wrote down are cut the same way, so the loss
    and the scores are a single process's."""
    from zenyx_b200.ops.attention import shard_sequence

    cfg = LlamaConfig.tiny(n_layers=1, d_model=64, n_heads=2, n_kv_heads=1, ffn_dim=96, vocab_size=128)
    S = 512
    tokens = _tokens(2, S)
    teacher = LlamaModel(cfg, device="cpu", dtype=torch.float32, seed=9)
    wrote = teacher.token_logprobs(tokens, top_k=4)
    ids = wrote.top_ids.clone()
    ids[0, 30:50] = -1
    trainer = Trainer(cfg, TrainerConfig(lr=1e-2, seq_len=S, global_batch=2, ring_degree=cp, max_grad_norm=1.0, seed=4))
    ring = trainer.engine.ring
    if cp > 1:
        part = shard_sequence(tokens, ring.rank, cp, ring.layout)
        scores = trainer.model.token_logprobs(part, part, top_k=2, ring=ring)
        torch.save(tuple(scores), f"{tmp}/scores{rank}.pt")
    losses = [trainer.distill_step(tokens, wrote.top_logprobs, ids, tail="bucket") for _ in range(2)]
    torch.save((losses, trainer.model.w("lm_head.weight").clone(), ring.rank, ring.layout), f"{tmp}/{cp}_{world}_{rank}.pt")
    trainer.close()


@pytest.mark.parametrize("cp", [1, 2])
def test_distillation_on_two_ranks_is_that_of_one(tmp_path, cp):
    import test_dist_cpu

    test_dist_cpu.run_ranks(_distill_ranks, world=2, args=(cp, str(tmp_path)))
    _distill_ranks(0, 1, 1, str(tmp_path))
    one = torch.load(tmp_path / "1_1_0.pt")
    for rank in range(2):
        losses, head, *_ = torch.load(tmp_path / f"{cp}_2_{rank}.pt")
        # bf16 weights and activations in another order of sums: 2^-8 of a loss of a few units, twice that after a step
        assert max(abs(a - b) for a, b in zip(losses, one[0])) < 2 * 2.0 ** -8 * max(one[0])
        assert (head.float() - one[1].float()).abs().max() <= 3 * 1e-2      # two steps of Adam move a weight by lr each
    if cp == 2:
        for rank in range(2):
            scores = torch.load(tmp_path / f"scores{rank}.pt")
            assert scores[0].shape == (2, 256) and scores[3].shape == (2, 256, 2) and bool(torch.isfinite(scores[0]).all())
