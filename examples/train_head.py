"""A training step's last part with the operators as they are used together.

A small language model of one recurrent layer: embeddings feed the RWKV-7
recurrence (``statetune_recurrent_fp32io16``), its output joins the residual
stream in the head's layer norm, and the loss is taken from the hidden rows:
cross entropy against the next token (prompt positions left out) plus the
divergence from a teacher's top logits. Neither loss makes the [tokens, vocab]
logits. Two ways to train:

* ``--mode full``: embeddings, projections, norm and head;
* ``--mode state``: only the initial state, everything else frozen (the weight
  gradients of the head are then never computed).

``--max-norm`` clips each step's gradients by their norm together.

    python examples/train_head.py [--mode state] [--steps 60] [--max-norm 1]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from flashrwkv_amd import (  # noqa: E402
    infer_layer_norm_forward_varlen,
    pretrain_clip_grad_norm,
    pretrain_layer_norm,
    pretrain_linear_cross_entropy,
    pretrain_linear_topk_distillation,
    statetune_recurrent_fp32io16,
)

IGNORE = -100


class Model(torch.nn.Module):
    """One recurrent layer between an embedding and a head, bf16."""

    def __init__(self, vocab: int, heads: int, head_size: int = 64):
        super().__init__()
        self.heads, self.head_size = heads, head_size
        c = heads * head_size

        def weight(*shape, std):
            return torch.nn.Parameter((torch.randn(*shape) * std).bfloat16())

        self.embedding = weight(vocab, c, std=1.0)
        self.tokens = weight(6 * c, c, std=0.5 * c ** -0.5)
        self.norm_weight = torch.nn.Parameter(torch.ones(c).bfloat16())
        self.norm_bias = torch.nn.Parameter(torch.zeros(c).bfloat16())
        self.head = weight(vocab, c, std=c ** -0.5)
        self.state = torch.nn.Parameter(torch.zeros(1, heads, head_size, head_size))

    def recurrence(self, ids: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """The recurrence's output and the residual stream it joins, [tokens, C] each, of
        one packed sequence."""
        n = ids.numel()
        stream = self.embedding[ids]
        r, decay, k, v, a, b = (
            t.contiguous().view(n, self.heads, self.head_size)
            for t in (stream @ self.tokens.t()).chunk(6, dim=1))
        a = torch.nn.functional.normalize(a, dim=2)
        offsets, starts, ends = (torch.tensor(x, dtype=torch.int32, device=ids.device)
                                 for x in ([0, 1], [0], [n]))
        out, *_ = statetune_recurrent_fp32io16(self.state, offsets, starts, ends, r, decay, k, v,
                                               -a, (a * torch.sigmoid(b)).contiguous())
        return out.reshape(n, -1), stream

    def hidden(self, ids: torch.Tensor) -> torch.Tensor:
        """Normed hidden rows [tokens, C], for training."""
        out, stream = self.recurrence(ids)
        rows, _ = pretrain_layer_norm(out, self.norm_weight, self.norm_bias, residual=stream)
        return rows


def step_loss(model: Model, ids, targets, teacher_logits, teacher_tokens, temperature=2.0):
    """Cross entropy plus distillation of one sequence, both from the hidden rows."""
    rows = model.hidden(ids)
    labels = pretrain_linear_cross_entropy(rows, model.head, targets, ignore_index=IGNORE)
    teacher = pretrain_linear_topk_distillation(rows, model.head, teacher_logits, teacher_tokens,
                                                temperature=temperature)
    return 0.5 * labels + 0.5 * teacher


@torch.no_grad()
def token_log_probs(model: Model, ids, targets):
    """Scoring: the log probability of each target, [tokens] fp32 (the rows as a
    serving loop would norm them)."""
    out, stream = model.recurrence(ids)
    rows, _ = infer_layer_norm_forward_varlen(out, model.norm_weight, model.norm_bias,
                                              residual=stream)
    return -pretrain_linear_cross_entropy(rows, model.head, targets, reduction="none")


def synthetic(vocab: int, tokens: int, top: int, device):
    """A sequence with a pattern to learn: each token names the next one, a third
    of the positions are prompt, the teacher lists the right token first."""
    gen = torch.Generator().manual_seed(5)
    follow = torch.randperm(vocab, generator=gen)
    ids = torch.empty(tokens, dtype=torch.int64)
    ids[0] = 1
    for i in range(1, tokens):
        ids[i] = follow[ids[i - 1]]
    right = follow[ids]
    targets = right.clone()
    targets[: tokens // 3] = IGNORE
    others = (right[:, None] + torch.arange(1, top)) % vocab
    teacher_tokens = torch.cat([right[:, None], others], 1)
    teacher_logits = torch.cat([torch.full((tokens, 1), 6.0), torch.zeros(tokens, top - 1)], 1)
    return [t.to(device) for t in (ids, targets, teacher_logits, teacher_tokens)]


def train(mode: str = "full", steps: int = 60, vocab: int = 1000, heads: int = 4,
          tokens: int = 192, top: int = 16, device: str = "cuda",
          max_norm: float | None = None) -> list[float]:
    """Trains on one synthetic sequence; the loss of every step."""
    torch.manual_seed(0)
    model = Model(vocab, heads).to(device)
    if mode == "state":
        for name, p in model.named_parameters():
            p.requires_grad_(name == "state")
    trained = [p for p in model.parameters() if p.requires_grad]
    optimizer = torch.optim.AdamW(trained, lr=2e-2 if mode == "state" else 3e-3)
    batch = synthetic(vocab, tokens, top, device)
    losses = []
    for _ in range(steps):
        optimizer.zero_grad(set_to_none=True)
        loss = step_loss(model, *batch)
        loss.backward()
        if max_norm is not None:
            pretrain_clip_grad_norm([p.grad for p in trained], max_norm)
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--mode", choices=("full", "state"), default="full")
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--max-norm", type=float)
    args = parser.parse_args()
    losses = train(args.mode, args.steps, max_norm=args.max_norm)
    for i in range(0, len(losses), max(1, len(losses) // 6)):
        print(f"step {i:4d}  loss {losses[i]:.4f}")
    print(f"last       loss {losses[-1]:.4f}")


if __name__ == "__main__":
    main()
