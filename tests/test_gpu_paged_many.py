"""Paged attention of many sequences whose rows form long tiles, and of steps
that mix all kinds of sequences.  Bounds as in paged_ref.py."""

from __future__ import annotations

import random

import pytest
import torch

from test_gpu_paged import BF, _case, _check, _run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count,layout,page", [(70, (16, 2, 256), 16), (130, (6, 2, 128), 32), (300, (8, 2, 64), 8),
                                               (600, (4, 1, 64), 8)])
def test_attention_long_tiles_of_many_sequences(device, count, layout, page):
    rng = random.Random(count)
    seqs = []
    for i in range(count):
        n = rng.choice([0, 1, 1, rng.randint(2, 9), rng.randint(20, 90) if i % 5 == 0 else 3])
        seqs.append((max(n, rng.choice([n, n + rng.randint(0, 40), rng.randint(0, 900) if i % 7 == 0 else 60])), n))
    seqs[-1] = (1700, 33)   # a long one at the end
    c, *rest = _case(device, *layout, page, seqs, BF, seed=count, gate=True, pad=2)
    out = torch.full(c["q"].shape, 9.0, dtype=BF, device=device)
    _check(c, *rest, _run_attention(c, out=out))
    assert bool((out[-2:] == 9.0).all())


@pytest.mark.parametrize("layout", [(16, 2, 256), (32, 8, 128)])
def test_attention_of_a_mixed_step(device, layout):
    # A prompt, a chunk over a long cache, verify blocks, decode rows and rows that rest.
    seqs = [(300, 300), (3000, 200)] + [(500 + 37 * i, 1 + i % 5) for i in range(20)] + [(100, 0), (0, 0)]
    seqs += [(30 * i + 1, 1) for i in range(40)]
    c, *rest = _case(device, *layout, 16, seqs, BF, seed=31, gate=True)
    _check(c, *rest, _run_attention(c))
