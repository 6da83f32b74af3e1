"""Every kernel of ``linear`` at depth (GPU), at the sizes of linear_forms.py: results against
64 bits with the bound of test_gpu_linear.py."""

from __future__ import annotations

import pytest
import torch

from linear_forms import KINDS, SIZES, names
from test_gpu_linear import check, make, make_adapters

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda:0")


@pytest.mark.parametrize(
    "kind,size",
    [
        pytest.param(kind, size, id=f"{kind}-{'x'.join(map(str, size))}-{names(size)[k].replace(' ', '_')}")
        for k, kind in enumerate(KINDS)
        for size in SIZES
    ],
)
def test_every_kernel(dev, kind, size):
    from kappa_amd.qwen3 import linear, lora_batch, prepack_linear, prepack_lora

    T, K, N, L, R = size
    x, w, xd, wd = make(dev, T, K, N, *KINDS[kind])
    p, lora, kw = prepack_linear(w), None, {}
    if L:
        lora = make_adapters(dev, T, K, N, L, R)
        kw = dict(lora=prepack_lora(*lora[:3]), batch=lora_batch(lora[3], L))
    y = linear(x, p, **kw)
    check(y, xd, wd, K, lora, R)
    assert torch.equal(y, linear(x, p, **kw))
