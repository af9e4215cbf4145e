"""Draft verification of entries that are no probabilities."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged import _ints

pytestmark = pytest.mark.gpu


def test_verify_entries_without_mass_are_never_drawn(device):
    from lightreason_amd.verify import verify_drafts

    # A rejected draft; target entries of 0 or less beside negative draft
    # entries: only tokens 2 and 3 have mass, whatever the draft's entries are.
    target = torch.tensor([[0.0, -1.0, 0.5, 0.5, -0.0, 0.0]], device=device).repeat(2, 1)
    draft = torch.tensor([[-3.0, -2.0, 0.25, 0.25, -1.0, 1.5]], device=device).repeat(2, 1)
    samples = torch.linspace(0, 0.999, 50, device=device)
    for s in samples:
        accepted, token = verify_drafts(torch.tensor([2, 5], device=device), target, _ints([0, 2], device),
                                        torch.full((2,), 0.5, device=device), s.reshape(1), draft=draft)
        assert accepted.item() == 0 and token.item() == (2 if float(s) < 0.5 else 3)
