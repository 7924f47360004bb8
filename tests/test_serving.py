"""The operators of serving in 8 bits together, in their plain forms."""

from __future__ import annotations

import pytest
import torch

from tests.chunk_util import CODES
from tests.serving_util import Layer, serve


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("held", [None, *CODES])
def test_a_run(dtype, held):
    serve(Layer("cpu", dtype, held))
