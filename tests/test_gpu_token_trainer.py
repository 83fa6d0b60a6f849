"""A whole language model step (embedding, layers, projection, loss, gradients, update) against autograd in fp32."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _config(batch):
    from terapipe_b200.models import TransformerConfig
    return TransformerConfig(batch_size=batch, seq_len=96, n_layers=2, embedding_dim=256, num_attention_heads=4, n_devices=1)


def _oracle(trainer, tokens, labels, teacher):
    """Loss and gradients of the same model from the portable layers and torch's losses, with the trainer's 16-bit weights."""
    from terapipe_b200.models import TransformerLayer
    cfg = trainer.config
    layers = [TransformerLayer(cfg.embedding_dim, cfg.ffn_embedding_dim, cfg.num_attention_heads, device="cuda") for _ in range(cfg.n_layers)]
    state = trainer.engine.state_dict()
    for i, layer in enumerate(layers):
        layer.load_state_dict({k.split(".", 3)[3]: v.float() for k, v in state.items() if k.startswith(f"layers.layers.{i}.")})
    table = trainer.weight[:trainer.vocab].float().requires_grad_()
    x = torch.nn.functional.embedding(tokens.t(), table) * trainer.embed_scale
    for layer in layers:
        x, _, _ = layer.forward_slice(x)
    z = x @ table.t()
    y = labels.t()
    loss = torch.nn.functional.cross_entropy(z.flatten(0, 1), y.flatten(), ignore_index=trainer.ignore_id, reduction="none")
    if teacher is not None:
        w, t = trainer.teacher_weight, trainer.temperature
        ids, logits = (v.transpose(0, 1).flatten(0, 1) for v in teacher)
        p = torch.softmax(logits.masked_fill(ids < 0, -torch.inf) / t, -1)
        log_q = torch.log_softmax(z.flatten(0, 1) / t, -1).gather(1, ids.clamp(min=0).long())
        kl = torch.where(p > 0, p * (p.clamp(min=1e-30).log() - log_q), 0).sum(-1)
        loss = (1 - w) * loss + w * t * t * kl
    loss.mean().backward()
    grads = {f"layers.layers.{i}.{k}": v.grad for i, layer in enumerate(layers) for k, v in layer.named_parameters()}
    return loss.mean().item(), grads, table.grad


def _rel(a, b):
    return ((a.float() - b.float()).norm() / (b.float().norm() + 1e-12)).item()


@pytest.mark.parametrize("entries", [0, 7])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("vocab", [512, 1003])
def test_step_matches_autograd(vocab, dtype, entries):
    from terapipe_b200.runtime.token_trainer import TokenTrainer
    t = TokenTrainer(_config(3), vocab, 3, dtype=dtype, lr=1e-3, embed_scale=50.0, teacher_entries=entries, temperature=2.0,
                     teacher_weight=0.5, loss_scale=1024.0)
    g = torch.Generator().manual_seed(vocab)
    tokens = torch.randint(0, vocab, (3, 96), generator=g).cuda()
    labels = torch.randint(0, vocab, (3, 96), generator=g).cuda()
    labels[:, -5:] = -100
    teacher = None
    if entries:
        ids = torch.stack([torch.randperm(vocab, generator=g)[:entries] for _ in range(288)]).view(3, 96, entries)
        ids[:, :, -2:][:, ::3] = -1
        teacher = (ids.cuda(), torch.randn(3, 96, entries, generator=g).cuda() * 2)
    want, grads, table = _oracle(t, tokens, labels, teacher)
    # the engine's tolerances for the same stack: activations and gradients rounded to 16 bits in every layer
    tol = 2e-2 if dtype == "fp16" else 6e-2
    got = t.compute_grads(tokens, labels, teacher)
    assert abs(float(t.losses.mean()) - want) < tol * 0.2
    assert abs(t.evaluate(tokens, labels, teacher) - want) < tol * 0.2
    for name, ref in grads.items():
        assert _rel(got[name], ref) < tol, name
    assert _rel(got["embedding"], table) < tol
    assert got["embedding"].shape == (vocab, 256) and (t.grad[vocab:] == 0).all()
    # an update of Adam's first step is lr times the gradient's sign
    before = t.master.clone()
    t.train_step(tokens, labels, teacher)
    assert (t.master[vocab:] == 0).all() and (t.weight[vocab:] == 0).all()
    big = table.abs() > table.abs().mean()
    assert ((before - t.master)[:vocab][big] * table[big].sign() > 0).float().mean() > 0.99
    t.close()


def test_loss_falls_and_graphs_replay():
    """The step is captured after the first call: new tokens, labels and entries reach the replays."""
    from terapipe_b200.runtime.token_trainer import TokenTrainer
    t = TokenTrainer(_config(4), 300, 4, lr=1e-3, embed_scale=50.0, teacher_entries=4, teacher_weight=0.5)
    g = torch.Generator().manual_seed(0)
    losses = []
    for step in range(60):
        tokens = torch.randint(0, 300, (4, 96), generator=g)
        nxt = (7 * tokens + 3) % 300
        ids = torch.stack([nxt, (nxt + 1) % 300, (nxt + 2) % 300, torch.full_like(nxt, -1)], -1)
        losses.append(t.train_step(tokens, nxt, (ids, torch.tensor([5.0, 1.0, 0.0, 0.0]).expand(4, 96, 4))))
    assert t.engine._graph is not None
    assert losses[-1] < 0.5 * losses[0], losses[::10]
    t.close()


def test_default_labels_and_refusals():
    from terapipe_b200.runtime.token_trainer import TokenTrainer
    t = TokenTrainer(_config(2), 100, 2)
    tokens = torch.randint(0, 100, (2, 96))
    t.load(tokens)
    assert torch.equal(t.labels[:, :-1].cpu(), tokens[:, 1:]) and (t.labels[:, -1] == -100).all()
    for bad in (lambda: t.load(tokens[:, :50]), lambda: t.load(tokens, teacher=(tokens, tokens)),
                lambda: TokenTrainer(_config(2), 100, 3)):
        with pytest.raises(ValueError):
            bad()
    t.close()
