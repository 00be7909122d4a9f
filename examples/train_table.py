"""Trains a table of static token vectors on pairs of texts: a text's vector is
the mean of its tokens' rows, scaled to unit length, and each text has to find
its partner among the batch's (a contrastive loss over the similarities).

Every step runs the training operators together, on the device and without a
synchronisation: lookup, similarity product, log probabilities (with the
hardest wrong partners), their gradient, the products back to the vectors, the
gradient of the rows met, clipping by the global norm, update.

    python examples/train_table.py --steps 200
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path
from typing import NamedTuple

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from ai_b200 import cluster, tensor, train  # noqa: E402

PAD = 0


class Step(NamedTuple):
    Loss: torch.Tensor      # mean of -log p(partner)
    Norm: torch.Tensor      # of the gradient, before clipping
    Hardest: torch.Tensor   # [batch, top] the most probable partners
    Grad: train.RowsGrad    # of the rows met, clipped


def encode(table: torch.Tensor, ids: torch.Tensor):
    """Unit vectors [batch, dim] of padded token ids, with what their gradient
    needs: the vectors' lengths and the texts' token counts."""
    rows = train.Embedding(table, ids, scale=table.shape[1] ** 0.5, padding=PAD, dtype=torch.float32)
    count = (ids != PAD).sum(1, keepdim=True).clamp(min=1)
    pooled = rows.sum(1) / count
    length = pooled.norm(dim=1, keepdim=True).clamp(min=1e-12)
    return cluster.Normalize(pooled), length, count


def encode_grad(dvec: torch.Tensor, vec: torch.Tensor, length: torch.Tensor, count: torch.Tensor, tokens: int):
    """The gradient of every token's row, [batch, tokens, dim]."""
    dpooled = (dvec - vec * (vec * dvec).sum(1, keepdim=True)) / length
    return (dpooled / count)[:, None, :].expand(-1, tokens, -1)


def step(table: torch.Tensor, left: torch.Tensor, right: torch.Tensor, temperature: float = 0.05, lr: float = 0.2,
         max_norm: float = 1.0, top: int = 4) -> Step:
    """One step on the pairs (left[i], right[i]) of int32 ids [batch, tokens]."""
    batch = left.shape[0]
    a, a_length, a_count = encode(table, left)
    b, b_length, b_count = encode(table, right)
    partner = torch.arange(batch, dtype=torch.int32, device=table.device)
    sims = cluster.Similarities(a, b)
    p = train.LogProbs(sims, partner, scale=1 / temperature, top=min(top, batch))
    share = torch.full((batch,), -1.0 / batch, device=table.device)
    dsims = train.LogProbsGrad(sims, partner, p.LogSum, share, scale=1 / temperature, peak=p.Peak)
    da, db = tensor.MatMul(dsims, b), tensor.MatMul(dsims.t(), a)
    dy = torch.cat([encode_grad(da, a, a_length, a_count, left.shape[1]),
                    encode_grad(db, b, b_length, b_count, right.shape[1])], 1)
    grad = train.EmbeddingGradRows(dy, torch.cat([left, right], 1), table.shape[0], scale=table.shape[1] ** 0.5,
                                   padding=PAD)
    norm = train.ClipGradNorm([grad.Rows], max_norm)
    # places past the rows met hold zeros, so they may go to any row
    table.index_add_(0, grad.Ids.clamp(min=0), grad.Rows.to(table.dtype), alpha=-lr)
    return Step(-p.LogProb.mean(), norm, p.TopIndex, grad)


def texts(topics: torch.Tensor, tokens: int, vocab: int, g: torch.Generator) -> torch.Tensor:
    """Padded ids of texts about the topics: a third of the words are the
    topic's own 16, the others anybody's."""
    n, dev = len(topics), topics.device
    own = 1 + (topics[:, None] * 16 + torch.randint(0, 16, (n, tokens), generator=g, device=dev)) % (vocab - 1)
    other = torch.randint(1, vocab, (n, tokens), generator=g, device=dev)
    ids = torch.where(torch.rand(n, tokens, generator=g, device=dev) < 1 / 3, own, other)
    length = torch.randint(tokens // 2, tokens + 1, (n, 1), generator=g, device=dev)
    return torch.where(torch.arange(tokens, device=dev) < length, ids, PAD).int()


def main(argv=None) -> float:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--batch", type=int, default=512)
    ap.add_argument("--tokens", type=int, default=48)
    ap.add_argument("--vocab", type=int, default=32768)
    ap.add_argument("--dim", type=int, default=256)
    a = ap.parse_args(argv)
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(0)
    table = torch.randn(a.vocab, a.dim, generator=g, device=dev) * 0.02
    found = 0.0
    for i in range(a.steps):
        topics = torch.randint(0, a.vocab // 16, (a.batch,), generator=g, device=dev)
        s = step(table, texts(topics, a.tokens, a.vocab, g), texts(topics, a.tokens, a.vocab, g))
        if i % 20 == 0 or i == a.steps - 1:
            found = float((s.Hardest[:, 0] == torch.arange(a.batch, device=dev)).float().mean())
            print(f"step {i:4d}  loss {float(s.Loss):.4f}  partner found {found:.3f}  gradient norm {float(s.Norm):.3f}")
    train.Check(dev)
    return found


if __name__ == "__main__":
    main()
