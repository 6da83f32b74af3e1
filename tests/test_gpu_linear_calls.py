"""Calls of ``linear`` that its documentation allows and whose form is out of the ordinary (GPU):
rows far apart, buffers that do not fit, buffers that overlap."""

from __future__ import annotations

import pytest
import torch

from test_gpu_linear import make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("rows", ["bf16", "q8"])
def test_rows_that_span_4_gib_or_more(dev, rows):
    """Three rows 2 GiB apart: further than the kernels' 32-bit offsets reach."""
    from kappa_amd.qwen3 import Q8Rows, linear, prepack_linear

    T, K, N = 3, 256, 96
    x, w, _, _ = make(dev, T, K, N, "w8c", rows)
    p = prepack_linear(w)
    v = x.values if rows == "q8" else x
    stride = (1 << 31) // v.element_size()
    far = torch.empty((T - 1) * stride + K, dtype=v.dtype, device=dev).as_strided((T, K), (stride, 1))
    far.copy_(v)
    assert torch.equal(linear(Q8Rows(far, x.scale) if rows == "q8" else far, p), linear(x, p))
