"""What a distillation step of the Trainer weighs."""
import torch

from zenyx_b200.models import LlamaConfig
from zenyx_b200.train import Trainer, TrainerConfig


def test_loss_scale_of_a_distillation_step():
    """The loss of the first step, and the weight that the model's backward gets, are in proportion; 1 is the default."""
    cfg = LlamaConfig.tiny(n_layers=1, d_model=64, n_heads=2, n_kv_heads=1, ffn_dim=96, vocab_size=128)
    gen = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, 128, (2, 128), generator=gen)
    values, ids = torch.log_softmax(torch.randn(2, 128, 128, generator=gen) * 2, -1).topk(5)
    losses, weights = [], []
    for kw in ({}, {"loss_scale": 1.0}, {"loss_scale": 4.0}):
        trainer = Trainer(cfg, TrainerConfig(lr=1e-3, seq_len=128, global_batch=2))
        whole = trainer.model.forward_backward_distill

        def seen(tokens, values, ids, weight, *args, **kwargs):
            weights.append(weight)
            return whole(tokens, values, ids, weight, *args, **kwargs)

        trainer.model.forward_backward_distill = seen
        losses.append(trainer.distill_step(tokens, values, ids, temperature=2.0, tail="bucket", **kw))
        trainer.close()
    assert losses[0] == losses[1] > 0 and abs(losses[2] - 4 * losses[0]) <= 1e-6 * losses[2]
    assert weights[0] == weights[2] == 1 / 256 and weights[4] == weights[5] == 4 / 256
