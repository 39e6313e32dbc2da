"""Preference training of a small Mamba model on one GPU: the training operators together.

    python examples/preference_step.py [--steps 20] [--plain]

Every step runs a batch of answer pairs through ``MambaModel.forward_train`` (the scan's and the conv's gradients,
activations held in 8 bits unless ``--plain``), takes ``training.preference_loss`` against the frozen start, and
updates the weights. The data are synthetic: the chosen answer of a pair counts upwards from the prompt's last token,
the rejected one is random.
"""

from __future__ import annotations

import argparse
import copy
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from mamba_metal_b200 import MambaConfig, MambaModel, init_weights_, training  # noqa: E402

IGNORE = -100


def make_pairs(pairs: int, prompt: int, answer: int, vocab: int, generator: torch.Generator):
    """(input ids, labels), each (2 * pairs, prompt + answer - 1): chosen rows first; labels are the next tokens,
    IGNORE inside the prompt. The rejected answers are shorter, by up to half."""
    dev = generator.device
    rows = torch.randint(0, vocab, (pairs, prompt), generator=generator, device=dev).repeat(2, 1)
    steps = torch.arange(1, answer + 1, device=dev)
    good = (rows[:pairs, -1:] + steps) % vocab
    bad = torch.randint(0, vocab, (pairs, answer), generator=generator, device=dev)
    ids = torch.cat([rows, torch.cat([good, bad])], 1)
    labels = ids[:, 1:].clone()
    labels[:, :prompt - 1] = IGNORE
    short = torch.randint(0, answer // 2 + 1, (pairs,), generator=generator, device=dev)
    past = torch.arange(labels.shape[1], device=dev) >= labels.shape[1] - short[:, None]
    labels[pairs:][past] = IGNORE
    return ids[:, :-1], labels


@torch.no_grad()
def answer_logps(model: MambaModel, ids: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    """Log-probability of every row's answer: with a reference of 0 and beta 1 they are the loss's rewards."""
    zero = torch.zeros(ids.shape[0], device=ids.device)
    _, chosen, rejected = training.preference_loss(model.forward(ids), labels, zero, beta=1.0)
    return torch.cat([chosen, rejected])


def train(steps: int = 20, checkpoint8: bool = True, dtype: torch.dtype = torch.bfloat16, seed: int = 0, pairs: int = 4,
          prompt: int = 24, answer: int = 17, lr: float = 2e-3, device: str = "cuda:0") -> list[float]:
    cfg = MambaConfig(d_model=128, n_layer=3, vocab_size=256)
    model = init_weights_(MambaModel(cfg, dtype=dtype, device=device), seed=seed)
    reference = copy.deepcopy(model).requires_grad_(False)
    optimizer = torch.optim.Adam(model.parameters(), lr=lr)
    generator = torch.Generator(device=device).manual_seed(seed + 1)
    losses = []
    for _ in range(steps):
        ids, labels = make_pairs(pairs, prompt, answer, cfg.vocab_size, generator)
        ref = answer_logps(reference, ids, labels)
        logits = model.forward_train(ids, checkpoint8=checkpoint8)
        loss, chosen, rejected = training.preference_loss(logits, labels, ref, beta=0.1, label_smoothing=0.05)
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return [float(v) for v in losses]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--plain", action="store_true", help="hold activations as they are instead of in 8 bits")
    a = ap.parse_args()
    for i, v in enumerate(train(a.steps, checkpoint8=not a.plain)):
        print(f"step {i:3d}  loss {v:.4f}")


if __name__ == "__main__":
    main()
