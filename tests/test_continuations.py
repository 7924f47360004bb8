"""Continuations of shared prompts on a paged cache, sampled together."""

from __future__ import annotations

import torch

from tests.continuations_util import run


def test_continuations_are_sampled_forked_and_compacted():
    run("cpu", torch.float32)
