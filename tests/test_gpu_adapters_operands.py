"""GPU: adapters on operands at the edges of what a binding takes, and values
at the edges of their types.  Bounds are those that test_gpu_adapters derives.
"""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import linear
from test_gpu_adapters import DEV, case, check

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("stride", [0, 1, 260, 267])
def test_a_single_row_of_any_stride(stride):
    """The row stride of one row means nothing, of the activations as of the others."""
    print(f"adapters: one row, stride {stride}", flush=True)
    x, (base,), banks, (held,), slots = case(1, 264, (40,), (16, 5), 16, torch.bfloat16, "one", seed=20)
    at = lambda t: t.clone().as_strided(t.shape, (stride, 1))
    y = at(base)
    linear.PackedLinearOperators().bind_adapters(at(x), banks, slots, y).launch()
    torch.cuda.synchronize()
    check(y, x, base, held, slots)
