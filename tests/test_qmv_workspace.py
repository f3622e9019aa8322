"""A caller's workspace of qmv_grouped is looked at before its size is believed: no GPU needed."""

from __future__ import annotations

import os

import pytest
import torch

from ironmule_amd import _native


@pytest.fixture(scope="module")
def probs():
    if not os.path.exists(_native.LIB_PATH):
        from ironmule_amd import build
        build.build()
    made = (_native.Problem * 1)()
    made[0].N, made[0].K, made[0].ldx, made[0].ldy = 512, 4096, 4096, 512
    return made


def test_a_workspace_that_is_not_what_it_should_be_is_refused(probs):
    """Its size is numel() * 4 bytes: of bytes that would be four times what is there, of every second value
    twice, and memory of another device is not the kernel's."""
    words = 1 << 16
    for bad in (torch.zeros(words, dtype=torch.uint8), torch.zeros(words, dtype=torch.bfloat16),
                torch.zeros(2 * words)[::2], torch.zeros(1).expand(words), torch.zeros(words, dtype=torch.float64)):
        with pytest.raises(ValueError, match="workspace"):
            _native._grouped_launch(probs, 1, 8, torch.bfloat16, torch.device("cpu"), None, bad)
    with pytest.raises(ValueError, match="workspace"):
        _native._grouped_launch(probs, 1, 8, torch.bfloat16, torch.device("cuda", 0), None, torch.zeros(words))
