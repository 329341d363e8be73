"""The distillation example, as a user runs it, at sizes of a test."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import torch

PATH = Path(__file__).resolve().parents[1] / "mlx-sparse_amd/examples/distill_window_student.py"


def load():
    spec = importlib.util.spec_from_file_location("distill_window_student", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def learns(device) -> None:
    """The divergence falls on tokens that were not trained on."""
    ex = load()
    torch.manual_seed(1)
    size = {"width": 64, "layers": 2, "heads": 4, "kv_heads": 2, "dim": 16}
    teacher, student = ex.Decoder(97, **size).to(device), ex.Decoder(97, **size).to(device)
    student.load_state_dict(teacher.state_dict())
    span = {"kept": 8, "window": 6, "sinks": 2}
    batches = [torch.randint(97, (3, 40), device=device) for _ in range(13)]
    before = ex.evaluate(teacher, student, batches[0], **span)
    means = ex.distill(teacher, student, batches[1:], **span)
    after = ex.evaluate(teacher, student, batches[0], **span)
    assert len(means) == 12 and before > 0 and after < before


def serves(device) -> None:
    """A prompt and steps from its caches give the logits of the whole
    sequence: float32 sums in another order, over two layers."""
    ex = load()
    torch.manual_seed(2)
    model = ex.Decoder(53, width=32, layers=2, heads=4, kv_heads=2, dim=8).to(device)
    tokens = torch.randint(53, (3, 41), device=device)
    span = {"window": 7, "sinks": 2}
    with torch.no_grad():
        want = model(tokens, **span)
        cache = ex.Cache(model, 3, **span)
        got = [model(tokens[:, :20], cache=cache, **span)]
        for i in range(20, 41):
            got.append(model.step(tokens[:, i], cache, **span)[:, None])
    got = torch.cat(got, 1)
    assert cache.lengths.tolist() == [41] * 3
    # a few hundred float32 roundings of values of the logits' size
    assert (got - want).abs().max() <= 2**-24 * 512 * want.abs().max()
    new = ex.generate(model, tokens, 5, **span)
    whole = tokens
    for i in range(5):
        with torch.no_grad():
            logits = model(whole, **span)[:, -1]
        top = logits.topk(2, -1).values
        sure = top[:, 0] - top[:, 1] > 2**-24 * 1024 * logits.abs().max()
        assert (logits.argmax(-1) == new[:, i])[sure].all()
        whole = torch.cat([whole, new[:, i:i + 1]], 1)
