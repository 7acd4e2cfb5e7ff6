"""Policy and preference steps with the operators as they are used together.

The model of ``train_head.py`` (embedding, RWKV-7 recurrence, layer norm, head)
answers prompts that are packed one after another. A step takes the hidden rows to
the log probability and the entropy of each sampled token at the sampling
temperature (``pretrain_linear_log_probs``), those of an answer's tokens to the loss
(``pretrain_policy_loss`` with a reward an answer, or ``pretrain_preference_loss`` of
answers in pairs), and the gradients through ``pretrain_clip_grad_norm`` to the
optimizer. The [tokens, vocab] logits are never made.

    python examples/train_policy.py [--loss preference] [--mode state] [--steps 20]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))

from train_head import Model  # noqa: E402

from flashrwkv_amd import (  # noqa: E402
    pretrain_clip_grad_norm,
    pretrain_layer_norm,
    pretrain_linear_log_probs,
    pretrain_policy_loss,
    pretrain_preference_loss,
    statetune_recurrent_fp32io16,
)

TEMPERATURE = 0.8


def hidden_rows(model: Model, ids: torch.Tensor, cu_seqlens: torch.Tensor) -> torch.Tensor:
    """Normed hidden rows of packed sequences, each from the model's initial state."""
    n, sequences = ids.numel(), cu_seqlens.numel() - 1
    stream = model.embedding[ids]
    r, decay, k, v, a, b = (
        t.contiguous().view(n, model.heads, model.head_size)
        for t in (stream @ model.tokens.t()).chunk(6, dim=1))
    a = torch.nn.functional.normalize(a, dim=2)
    offsets = torch.arange(sequences + 1, dtype=torch.int32, device=ids.device)
    out, *_ = statetune_recurrent_fp32io16(
        model.state.expand(sequences, -1, -1, -1).contiguous(), offsets,
        cu_seqlens[:-1].contiguous(), cu_seqlens[1:].contiguous(), r, decay, k, v, -a,
        (a * torch.sigmoid(b)).contiguous())
    rows, _ = pretrain_layer_norm(out.reshape(n, -1), model.norm_weight, model.norm_bias,
                                  residual=stream)
    return rows


def scores(model: Model, batch: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Log probability and entropy of each next token, [tokens] fp32."""
    rows = hidden_rows(model, batch["ids"], batch["cu_seqlens"])
    return pretrain_linear_log_probs(rows, model.head, batch["next"], temperature=TEMPERATURE,
                                     entropy=True)


def step_loss(model: Model, batch: dict, loss: str) -> torch.Tensor:
    """One step's loss; batch holds what the policy that sampled and the reference gave."""
    log_probs, entropy = scores(model, batch)
    if loss == "preference":
        return pretrain_preference_loss(log_probs, batch["cu_seqlens"], mask=batch["answer"],
                                        reference_log_probs=batch["reference"], beta=0.1)[0]
    return pretrain_policy_loss(
        log_probs, batch["old"], batch["advantages"], reference_log_probs=batch["reference"],
        entropy=entropy, mask=batch["answer"], cu_seqlens=batch["cu_seqlens"], clip_low=0.2,
        clip_high=0.28, kl_weight=0.02, entropy_weight=1e-3, reduction="sequence_mean")


def synthetic(model: Model, vocab: int, answers: int, device) -> dict:
    """Ragged prompts with sampled answers; an answer's reward is the share of its tokens
    in the lower half of the vocabulary. Neighbours are pairs, the better one first."""
    gen = torch.Generator().manual_seed(3)
    lengths = torch.randint(20, 90, (answers,), generator=gen)
    prompts = (lengths.float() * 0.4).long()
    ids = torch.randint(vocab, (int(lengths.sum()),), generator=gen)
    sequences = list(ids.split(lengths.tolist()))
    better = [float((s[p:] < vocab // 2).float().mean()) for s, p in zip(sequences, prompts)]
    order = [i for p in range(0, answers, 2)
             for i in ((p, p + 1) if better[p] >= better[p + 1] else (p + 1, p))]
    sequences, lengths = [sequences[i] for i in order], lengths[order]
    ids, rewards = torch.cat(sequences), torch.tensor([better[i] for i in order])
    cu = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)])
    place = torch.arange(ids.numel()) - cu[:-1].repeat_interleave(lengths)
    prompt = prompts[order].repeat_interleave(lengths)
    last = place == lengths.repeat_interleave(lengths) - 1
    batch = {
        "ids": ids, "next": torch.where(last, -100, ids.roll(-1)),
        "answer": (place >= prompt - 1) & ~last, "cu_seqlens": cu.to(torch.int32),
        "advantages": (rewards - rewards.mean()) / rewards.std(),
    }
    batch = {name: t.to(device) for name, t in batch.items()}
    with torch.no_grad():
        batch["old"], _ = scores(model, batch)
    batch["reference"] = batch["old"].clone()
    return batch


def train(loss: str = "policy", mode: str = "full", steps: int = 20, vocab: int = 1000,
          heads: int = 4, answers: int = 16, max_norm: float = 1.0,
          device: str = "cuda") -> list[tuple[float, float]]:
    """Steps on one batch; loss and gradient norm of each."""
    torch.manual_seed(0)
    model = Model(vocab, heads).to(device)
    if mode == "state":
        for name, p in model.named_parameters():
            p.requires_grad_(name == "state")
    trained = [p for p in model.parameters() if p.requires_grad]
    optimizer = torch.optim.AdamW(trained, lr=1e-2 if mode == "state" else 1e-3)
    batch = synthetic(model, vocab, answers, device)
    seen = []
    for _ in range(steps):
        optimizer.zero_grad(set_to_none=True)
        value = step_loss(model, batch, loss)
        value.backward()
        norm = pretrain_clip_grad_norm([p.grad for p in trained if p.grad is not None], max_norm)
        optimizer.step()
        seen.append(torch.stack([value.detach(), norm]))
    return [tuple(x) for x in torch.stack(seen).tolist()]


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--loss", choices=("policy", "preference"), default="policy")
    parser.add_argument("--mode", choices=("full", "state"), default="full")
    parser.add_argument("--steps", type=int, default=20)
    args = parser.parse_args()
    for i, (value, norm) in enumerate(train(args.loss, args.mode, args.steps)):
        print(f"step {i:3d}  loss {value:9.5f}  gradient norm {norm:.4f}")


if __name__ == "__main__":
    main()
