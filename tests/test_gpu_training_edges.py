"""Calls of the training operators at the ends of what they take: magnitudes,
sizes, reports and recorded results, against the formulas in 64 bits with the
bounds derived in the modules they come from.
"""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_norm_grad import both, make

pytestmark = pytest.mark.gpu


# rows of one size: with a mean square of 10^28 to 10^34 or below 10^-26 the cube of its root's
# inverse leaves what fp32 holds, and with it a gradient that is formed from the cube
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size,eps", [(1e14, 1e-6), (1e15, 1e-6), (1e17, 1e-6), (1e-13, 0.0),
                                      (1e-17, 0.0)])
@pytest.mark.parametrize("inter", [True, False])
def test_head_norm_of_very_large_and_very_small_rows(size, eps, dtype, inter):
    a, w, cos, sin, pos = make(2, 9, 3, 2, 128, 64, dtype, seed=31)
    for n in ("q", "k"):
        a[n] = (a[n].float() * size).to(dtype)
    both(a, w, cos, sin, pos, inter, eps)


def test_head_norm_gradient_of_zero_rows_beside_a_small_eps():
    a, w, cos, sin, pos = make(1, 5, 2, 2, 64, 64, torch.float32, seed=32)
    a["q"][0, 2] = 0
    a["k"][0, 4, 1] = 0
    both(a, w, cos, sin, pos, True, 1e-28)
