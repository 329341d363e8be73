"""A student with window attention, distilled from a teacher with full
attention and then served from ring caches.

Teacher and student are the same small decoder of random weights (there is no
data here: tokens are random too), the student starting from the teacher's.
The teacher attends to everything; its top logits are kept as a CSR matrix,
from which the student, whose queries see a window and a few sinks, learns.
Then a prompt goes through the student at once, its keys and values into ring
caches, and tokens follow one at a time.

    python mlx-sparse_amd/examples/distill_window_student.py [--tokens 512] [--steps 20]
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch
from torch import nn

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import mlx_sparse as ms  # noqa: E402


class Cache:
    """Ring caches of all layers, and how many tokens each sequence holds."""

    def __init__(self, model: "Decoder", batch: int, window: int, sinks: int):
        weight = model.embedding.weight
        shape = (batch, sinks + window, model.kv_heads, model.dim)
        self.pairs = [(weight.new_zeros(shape), weight.new_zeros(shape)) for _ in model.blocks]
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=weight.device)


class Block(nn.Module):
    def __init__(self, width: int, heads: int, kv_heads: int, dim: int):
        super().__init__()
        self.split = [heads * dim, kv_heads * dim, kv_heads * dim]
        self.dim = dim
        self.norms = nn.ModuleList([nn.RMSNorm(width), nn.RMSNorm(width)])
        self.project = nn.Linear(width, sum(self.split), bias=False)
        self.join = nn.Linear(heads * dim, width, bias=False)
        self.expand = nn.Linear(width, 4 * width, bias=False)
        self.contract = nn.Linear(4 * width, width, bias=False)

    def forward(self, x, attend):
        """``attend(q, k, v)`` with operands of shape (..., heads, dim)."""
        q, k, v = (t.unflatten(-1, (-1, self.dim))  # views of one projection
                   for t in self.project(self.norms[0](x)).split(self.split, -1))
        x = x + self.join(attend(q, k, v).flatten(-2))
        return x + self.contract(nn.functional.silu(self.expand(self.norms[1](x))))


class Decoder(nn.Module):
    def __init__(self, vocab: int, width: int = 256, layers: int = 2, heads: int = 8,
                 kv_heads: int = 2, dim: int = 32):
        super().__init__()
        self.kv_heads, self.dim = kv_heads, dim
        self.embedding = nn.Embedding(vocab, width)
        self.blocks = nn.ModuleList(Block(width, heads, kv_heads, dim) for _ in range(layers))
        self.norm = nn.RMSNorm(width)
        self.head = nn.Linear(width, vocab, bias=False)

    def forward(self, tokens, *, window: int, sinks: int = 0, cache: Cache | None = None):
        """Logits of whole sequences, shape (batch, tokens, vocab); their keys
        and values go into ``cache`` where one is given."""
        x = self.embedding(tokens)
        for layer, block in enumerate(self.blocks):
            def attend(q, k, v):
                if cache is not None:
                    ms.window_cache_store(k, v, *cache.pairs[layer], sinks=sinks)
                return ms.window_attention(q, k, v, window=window, sinks=sinks)
            x = block(x, attend)
        if cache is not None:
            cache.lengths += tokens.shape[1]
        return self.head(self.norm(x))

    @torch.no_grad()
    def step(self, token, cache: Cache, *, window: int, sinks: int = 0):
        """Logits after one more token of each sequence, shape (batch, vocab)."""
        x = self.embedding(token)
        for pair, block in zip(cache.pairs, self.blocks):
            x = block(x, lambda q, k, v: ms.window_attention_step(
                q, k, v, *pair, cache.lengths, window=window, sinks=sinks))
        cache.lengths += 1
        return self.head(self.norm(x))


def top_logits(logits: torch.Tensor, kept: int) -> ms.CSRArray:
    """The ``kept`` largest logits of each row."""
    rows = logits.flatten(0, -2)
    values, columns = rows.topk(kept, dim=-1)
    columns, order = columns.sort(dim=-1)
    starts = torch.arange(0, (rows.shape[0] + 1) * kept, kept, dtype=torch.int32,
                          device=rows.device)
    return ms.csr_array((values.gather(-1, order).flatten(), columns.int().flatten(), starts),
                        tuple(rows.shape), sorted_indices=True)


def distill(teacher: Decoder, student: Decoder, batches, *, kept: int, window: int, sinks: int,
            temperature: float = 2.0, rate: float = 1e-3) -> list[float]:
    """One optimizer step a batch of tokens; the mean losses."""
    optimizer = torch.optim.AdamW(student.parameters(), lr=rate)
    means = []
    for tokens in batches:
        with torch.no_grad():
            target = top_logits(teacher(tokens, window=tokens.shape[1]), kept)
        logits = student(tokens, window=window, sinks=sinks)
        losses, gradient = ms.distill_value_and_grad(logits, target, 1.0 / tokens.numel(),
                                                     temperature=temperature)
        optimizer.zero_grad(set_to_none=True)
        logits.backward(gradient)
        optimizer.step()
        means.append(losses.mean().item())
    return means


@torch.no_grad()
def evaluate(teacher: Decoder, student: Decoder, tokens, *, kept: int, window: int,
             sinks: int) -> float:
    target = top_logits(teacher(tokens, window=tokens.shape[1]), kept)
    return ms.distill_loss(student(tokens, window=window, sinks=sinks), target).mean().item()


@torch.no_grad()
def generate(model: Decoder, prompt, count: int, *, window: int, sinks: int) -> torch.Tensor:
    """``count`` tokens after the prompt, the likeliest each time."""
    cache = Cache(model, prompt.shape[0], window, sinks)
    logits = model(prompt, window=window, sinks=sinks, cache=cache)[:, -1]
    tokens = [logits.argmax(-1)]
    while len(tokens) < count:
        tokens.append(model.step(tokens[-1], cache, window=window, sinks=sinks).argmax(-1))
    return torch.stack(tokens, 1)


def main(argv=None) -> None:
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, default in (("batch", 4), ("tokens", 512), ("steps", 20), ("vocab", 1000),
                          ("kept", 16), ("window", 64), ("sinks", 4), ("generate", 32)):
        parser.add_argument(f"--{name}", type=int, default=default)
    args = parser.parse_args(argv)
    device = ms.default_torch_device()
    torch.manual_seed(0)
    teacher = Decoder(args.vocab).to(device)
    student = Decoder(args.vocab).to(device)
    student.load_state_dict(teacher.state_dict())
    span = {"window": args.window, "sinks": args.sinks}
    batches = [torch.randint(args.vocab, (args.batch, args.tokens), device=device)
               for _ in range(args.steps + 1)]

    before = evaluate(teacher, student, batches[-1], kept=args.kept, **span)
    start = time.perf_counter()
    distill(teacher, student, batches[:-1], kept=args.kept, **span)
    seconds = time.perf_counter() - start
    after = evaluate(teacher, student, batches[-1], kept=args.kept, **span)
    print(f"{device.type}: divergence {before:.4f} -> {after:.4f} in {args.steps} steps "
          f"({1e3 * seconds / args.steps:.1f} ms each)")
    tokens = generate(student, batches[-1], args.generate, **span)
    print("generated", tokens[0, :10].tolist(), "...")


if __name__ == "__main__":
    main()
