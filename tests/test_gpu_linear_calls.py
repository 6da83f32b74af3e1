"""Calls of ``linear`` that its documentation allows and whose form is out of the ordinary (GPU):
rows far apart, buffers that overlap, the largest sizes."""

from __future__ import annotations

import ctypes

import pytest
import torch

from linear_forms import KINDS
from test_gpu_linear import check, make, make_adapters

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


def test_buffers_that_overlap_are_refused(dev):
    """C ABI: out on the rows, on the workspace, and the workspace on the rows; beside them, and
    in the gap between two rows, is fine."""
    from kappa_amd import _lib
    from kappa_amd.qwen3 import linear, prepack_linear
    from kappa_amd.qwen3.projection import _stream

    T, K, N = 2, 250, 96  # rows that are copied into the workspace
    x, w, _, _ = make(dev, T, K, N)
    p = prepack_linear(w)
    L, n = _lib.lib(), ctypes.c_size_t()
    rows = torch.zeros(T, 2048, dtype=torch.bfloat16, device=dev)
    rows[:, :K] = x
    _lib.check(L.kmoe_linear_call_bytes(p.struct, T, rows.data_ptr(), _lib.DTYPE_BF16, 2048, None, ctypes.byref(n)))
    assert 0 < n.value <= 2048
    ws, out = torch.empty(n.value, dtype=torch.uint8, device=dev), torch.empty(T, N, dtype=torch.bfloat16, device=dev)

    def call(o, s):
        return L.kmoe_linear(p.struct, T, rows.data_ptr(), _lib.DTYPE_BF16, 2048, None, None, None, o, s, n.value, _stream(dev))

    at, gap = rows.data_ptr(), rows.data_ptr() + 2 * 256
    assert call(at, ws.data_ptr()) == _lib.ERR_INVALID_ARG
    assert call(at + 4096 - 2, ws.data_ptr()) == _lib.ERR_INVALID_ARG
    assert call(ws.data_ptr(), ws.data_ptr()) == _lib.ERR_INVALID_ARG
    assert call(out.data_ptr(), at) == _lib.ERR_INVALID_ARG
    want = linear(x, p)
    _lib.check(call(out.data_ptr(), ws.data_ptr()))
    assert torch.equal(out, want)
    _lib.check(call(gap, gap + 1024))
    assert torch.equal(rows[0, 256 : 256 + T * N].view(T, N), want) and torch.equal(rows[:, :K], x)


LIMITS = [(1 << 20, 64, 40, 5, 8), (3, 64, 1 << 20, 2, 8), (70, 64, 1 << 20, 0, 0), (1, 65536, 32, 3, 16), (70, 65536, 32, 3, 16),
          (40, 128, 32, 1024, 256), (1100, 128, 32, 1024, 256)]  # fmt: skip


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,K,N,L,R", LIMITS)
def test_the_largest_sizes(dev, T, K, N, L, R, kind):
    """The limits of tokens, inputs, outputs, adapters and rank, one or two at a time."""
    from kappa_amd.qwen3 import linear, lora_batch, prepack_linear, prepack_lora

    x, w, xd, wd = make(dev, T, K, N, *KINDS[kind])
    lora, kw = None, {}
    if L:
        lora = make_adapters(dev, T, K, N, L, R)
        kw = dict(lora=prepack_lora(*lora[:3]), batch=lora_batch(lora[3], L))
    check(linear(x, prepack_linear(w), **kw), xd, wd, K, lora, R)


def test_one_more_than_the_largest_is_refused(dev):
    from kappa_amd.qwen3 import LoraAdapters, linear, lora_batch, prepack_linear

    def zeros(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype, device=dev)

    p = prepack_linear(zeros(8, 8))
    for call in (
        lambda: linear(zeros((1 << 20) + 1, 8), p), lambda: prepack_linear(zeros(65537, 1)),
        lambda: prepack_linear(zeros(1, (1 << 20) + 1)), lambda: lora_batch(zeros((1 << 20) + 1, dtype=torch.int32), 1),
        lambda: lora_batch(zeros(1, dtype=torch.int32), 1025), lambda: LoraAdapters.empty(1025, 1, 8, 8),
        lambda: LoraAdapters.empty(1, 257, 8, 8), lambda: linear(zeros(1 << 20, 2048), prepack_linear(zeros(2048, 8))),
    ):  # fmt: skip
        with pytest.raises(ValueError):
            call()
