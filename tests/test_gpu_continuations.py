"""Continuations of shared prompts on the GPU, sampled together."""

from __future__ import annotations

import pytest
import torch

from tests.continuations_util import run, step_without_pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_continuations_are_sampled_forked_and_compacted(dtype):
    run("cuda", dtype)


def test_a_captured_step_between_forks_and_a_compaction():
    """The step is captured once and replayed; between its replays rows are
    released, forked and moved eagerly on the same tensors."""

    def captured(r):
        kept = [t.clone() for t in (*r.caches, r.counts, r.tables, r.context)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            r.step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = r.step()
        for t, was in zip((*r.caches, r.counts, r.tables, r.context), kept):
            t.copy_(was)

        def replay():
            graph.replay()
            torch.cuda.synchronize()
            return results

        return replay

    run("cuda", torch.bfloat16, captured)


def test_a_step_that_finds_no_page_leaves_the_others_alone():
    step_without_pages("cuda")

    def captured(step, state):
        kept = [t.clone() for t in state]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            slots = step()

        def replay():
            for _ in range(3):
                for t, was in zip(state, kept):
                    t.copy_(was)
                graph.replay()
                torch.cuda.synchronize()
            return slots

        return replay

    step_without_pages("cuda", captured)
