"""How the int8 product's sums become results: step by step, exactly."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import pytest
import torch

import cuda_force_amd as cf

pytestmark = pytest.mark.gpu


def fp32(x: Fraction) -> Fraction:
    """The fp32 number nearest to x (of ordinary size), ties to even."""
    if x == 0:
        return x
    e = 0
    while abs(x) >= Fraction(2) ** (e + 1):
        e += 1
    while abs(x) < Fraction(2) ** e:
        e -= 1
    step = Fraction(2) ** (e - 23)
    return round(x / step) * step


@pytest.mark.parametrize("m,n,k", [(3, 24, 64), (40, 20, 128), (70, 24, 30)])
@pytest.mark.parametrize("biased", [True, False])
def test_sum_scale_fma_rounding(m, n, k, biased):
    gen = torch.Generator().manual_seed(m)
    x, w = (torch.randint(-127, 128, (r, k), generator=gen, dtype=torch.int8) for r in (m, n))
    xs, ws = (torch.rand(r, generator=gen) * 0.01 + 1e-4 for r in (m, n))
    bias = torch.randn(n, generator=gen) if biased else None
    y = cf.matmul_int8(x.cuda(), w.cuda(), xs.cuda(), ws.cuda(), None if bias is None else bias.cuda(), torch.float32)
    sums = (x.long() @ w.long().t()).tolist()
    exact = lambda t: [Fraction(float(v)) for v in t]  # noqa: E731
    fx, fw, fb = exact(xs), exact(ws), exact(bias) if biased else [Fraction(0)] * n
    want = np.array([[float(fp32(fp32(sums[i][j] * fx[i]) * fw[j] + fb[j])) for j in range(n)] for i in range(m)])
    assert (y.cpu().double().numpy() == want).all()
