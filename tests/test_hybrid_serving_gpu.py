"""examples/hybrid_serving.py: what the caches give token by token, across
forks and a compaction, is what a prefill of the whole text gives."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
import hybrid_serving  # noqa: E402

pytestmark = pytest.mark.gpu


def test_decoding_agrees_with_a_prefill_of_the_whole_text(gpu_device):
    """Both are the same function of the text; they round differently (chunks
    against single tokens, bf16 activations of 8 layers: each of the 16
    roundings to bf16 on the way moves the logits by some 2^-9 of their
    size, so 0.03 of it allows four times their root sum of squares)."""
    gen = torch.Generator().manual_seed(3)
    model = hybrid_serving.Model(device=gpu_device)
    server = hybrid_serving.Server(model, rows=3, device=gpu_device)
    texts = [torch.randint(0, model.vocab, (n,), generator=gen).tolist() for n in (33, 16, 70)]
    server.prefill(texts)
    for step in range(24):
        tokens = torch.randint(0, model.vocab, (3,), generator=gen).tolist()
        for row, t in enumerate(tokens):
            texts[row].append(t)
        logits = server.step(torch.tensor(tokens, device=gpu_device))
        if step == 6:
            server.fork([2, 2], [0, 1])
            texts[0], texts[1] = list(texts[2]), list(texts[2])
        if step == 12:
            held = {int(p) for p in server.table.flatten() if p >= 0}
            assert server.compact() == len(held)
            assert {int(p) for p in server.table.flatten() if p >= 0} == set(range(len(held)))
    fresh = hybrid_serving.Server(model, rows=3, device=gpu_device)
    want = fresh.prefill(texts)
    rel = ((logits.float() - want.float()).norm() / want.float().norm()).item()
    assert rel <= 0.03, rel


def test_main_runs(gpu_device, capsys):
    hybrid_serving.main()
    # 20 tokens after each prompt; row 1 went on as row 2
    assert "tokens cached: [57, 84, 84, 140]" in capsys.readouterr().out
