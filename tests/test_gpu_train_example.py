"""The training operators together: one step of examples/train_table.py
against the same step in 64 bits with torch's autograd, and a short run."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parent.parent / "examples" / "train_table.py"
    spec = importlib.util.spec_from_file_location("train_table", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("batch,tokens,dim", [(1, 3, 8), (37, 11, 64), (300, 20, 256)])
def test_step_against_autograd_in_64_bits(cuda, batch, tokens, dim):
    import torch

    E = _example()
    g = torch.Generator(device=cuda).manual_seed(batch)
    vocab, tau, lr, max_norm = 500, 0.05, 0.05, 1.0
    table = torch.randn(vocab, dim, generator=g, device=cuda) * 0.02
    topics = torch.randint(0, vocab // 16, (batch,), generator=g, device=cuda)
    left, right = E.texts(topics, tokens, vocab, g), E.texts(topics, tokens, vocab, g)

    w = table.double().requires_grad_()

    def vectors(ids):
        keep = (ids != E.PAD)[..., None]
        rows = w[ids.long()] * keep * dim ** 0.5
        pooled = rows.sum(1) / keep.sum(1).clamp(min=1)
        return pooled / pooled.norm(dim=1, keepdim=True)

    logits = vectors(left) @ vectors(right).t() / tau
    loss = -torch.log_softmax(logits, 1).diagonal().mean()
    loss.backward()
    norm = w.grad.norm()
    c = min(1.0, max_norm / max(float(norm), 1e-300))
    want = table.double() - lr * c * w.grad

    s = E.step(table, left, right, temperature=tau, lr=lr, max_norm=max_norm)
    # similarities are within 1e-5 (split products), so the logits within
    # 2e-4, and so the probabilities and each gradient in proportion
    assert abs(float(s.Loss) - float(loss)) <= 4e-4
    assert abs(float(s.Norm) - float(norm)) <= 2e-3 * float(norm) + 1e-5
    # a row's step is at most lr times the clipped norm
    assert float((table.double() - want).abs().max()) <= 2e-3 * lr * max_norm + 1e-6
    met = torch.unique(torch.cat([left, right]))
    met = met[met != E.PAD]
    assert int(s.Grad.Count) == len(met) and torch.equal(s.Grad.Ids[:len(met)], met)


def test_short_run_learns(cuda):
    E = _example()
    assert E.main(["--steps", "120", "--batch", "256", "--vocab", "4096", "--dim", "64"]) > 0.5
