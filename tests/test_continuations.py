"""Continuations of shared prompts on a paged cache, sampled together."""

from __future__ import annotations

import torch

from tests.continuations_util import run, step_without_pages


def test_continuations_are_sampled_forked_and_compacted():
    run("cpu", torch.float32)


def test_a_step_that_finds_no_page_leaves_the_others_alone():
    step_without_pages("cpu")
