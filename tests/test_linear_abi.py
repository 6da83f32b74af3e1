"""The C ABI of the residual norms and the projections on the host (CPU): refusals before any
HIP call, buffer sizes, and the host code under the sanitizers."""

from __future__ import annotations

import ctypes
import os
import shutil

import pytest
import torch

from conftest import ROOT, gpu_available
from kappa_amd import _lib
from test_host_sanitized import _build, _run

BF, F32, I8 = _lib.DTYPE_BF16, _lib.DTYPE_F32, _lib.DTYPE_I8
P = 0x1000


def desc(T=4, D=128, act=BF):
    return _lib.KmoeDesc(T, D, 1, 1, 1, act, _lib.IMPL_GATHER_EINSUM, 64, 0, _lib.KERNELS_AUTO)


def lin(K=256, N=96, dtype=I8, values=P, scale=P):
    return _lib.KmoeLinear(values, scale, dtype, K, N)


def lora(L=4, R=16, K=256, N=96, a=P, b=P, f=P):
    return _lib.KmoeLora(a, b, f, L, R, K, N)


def batch(T=4, L=4, order=P):
    return _lib.KmoeLoraBatch(P, order, P, P, T, L)


def got(st):
    return st, _lib.lib().kmoe_last_error().decode()


NO_DEVICE = pytest.mark.skipif(gpu_available(), reason="a valid call would reach the device")


@pytest.mark.parametrize(
    "over,frag",
    [
        (dict(x=None), "non-NULL"),
        (dict(res=None), "non-NULL"),
        (dict(h=None), "non-NULL"),
        (dict(out=None), "non-NULL"),
        (dict(out=P), "alias"),
        (dict(out=2 * P), "alias"),
        (dict(scale=None), "norm scale pointer"),
        (dict(sdt=I8), "norm scale dtype"),
        (dict(eps=float("nan")), "epsilon"),
        (dict(d=desc(T=-1)), "tokens"),
        (dict(d=desc(act=I8)), "act_dtype"),
    ],
)
def test_add_rms_norm_refusals(over, frag):
    a = dict(d=desc(), x=P, res=2 * P, scale=3 * P, sdt=BF, eps=1e-6, h=4 * P, out=5 * P)
    a.update(over)
    st, msg = got(_lib.lib().kmoe_add_rms_norm(a["d"], a["x"], a["res"], a["scale"], a["sdt"], a["eps"], a["h"],
                                               a["out"], None))  # fmt: skip
    assert st == _lib.ERR_INVALID_ARG and frag in msg


@pytest.mark.parametrize(
    "over,frag",
    [
        (dict(x=None), "non-NULL"),
        (dict(q=None), "non-NULL"),
        (dict(qs=None), "non-NULL"),
        (dict(res=None), "come together"),
        (dict(h=None), "come together"),
        (dict(q=4 * P), "alias"),
    ],
)
def test_add_rms_norm_q8_refusals(over, frag):
    a = dict(x=P, res=2 * P, h=4 * P, q=5 * P, qs=6 * P)
    a.update(over)
    st, msg = got(_lib.lib().kmoe_add_rms_norm_q8(desc(), a["x"], a["res"], 3 * P, BF, 1e-6, a["h"], a["q"], a["qs"],
                                                  None))  # fmt: skip
    assert st == _lib.ERR_INVALID_ARG and frag in msg


@pytest.mark.parametrize(
    "over,want,frag",
    [
        (dict(w=lin(dtype=F32)), _lib.ERR_INVALID_ARG, "BF16 or I8"),
        (dict(w=lin(dtype=9)), _lib.ERR_INVALID_ARG, "BF16 or I8"),
        (dict(w=lin(K=0)), _lib.ERR_INVALID_ARG, ">= 1"),
        (dict(w=lin(K=65537)), _lib.ERR_UNSUPPORTED, "too large"),
        (dict(w=lin(values=None)), _lib.ERR_INVALID_ARG, "non-NULL"),
        (dict(w=lin(values=P + 8)), _lib.ERR_INVALID_ARG, "16-byte"),
        (dict(T=-1), _lib.ERR_INVALID_ARG, "tokens"),
        (dict(xt=F32), _lib.ERR_INVALID_ARG, "BF16 or I8 rows"),
        (dict(xt=I8, xs=P, w=lin(dtype=BF)), _lib.ERR_INVALID_ARG, "int8 weights"),
        (dict(xt=I8), _lib.ERR_INVALID_ARG, "x_scale"),
        (dict(xs=P), _lib.ERR_INVALID_ARG, "x_scale"),
        (dict(stride=255), _lib.ERR_INVALID_ARG, "x_stride"),
        (dict(x=None), _lib.ERR_INVALID_ARG, "non-NULL"),
        (dict(out=None), _lib.ERR_INVALID_ARG, "non-NULL"),
        (dict(stride=1 << 29), _lib.ERR_UNSUPPORTED, "4 GiB"),
        (dict(stride=(1 << 63) - 1), _lib.ERR_UNSUPPORTED, "4 GiB"),
        (dict(ws=None, lora=lora(), batch=batch()), _lib.ERR_WORKSPACE_TOO_SMALL, "workspace"),
        (dict(n=16, lora=lora(), batch=batch()), _lib.ERR_WORKSPACE_TOO_SMALL, "workspace"),
        (dict(ws=None, stride=257), _lib.ERR_WORKSPACE_TOO_SMALL, "workspace"),
        (dict(ws=None, x=P + 2), _lib.ERR_WORKSPACE_TOO_SMALL, "workspace"),
        (dict(ws=P + 4), _lib.ERR_INVALID_ARG, "16-byte"),
        (dict(lora=lora()), _lib.ERR_INVALID_ARG, "come together"),
        (dict(batch=batch()), _lib.ERR_INVALID_ARG, "come together"),
        (dict(lora=lora(N=97), batch=batch()), _lib.ERR_INVALID_ARG, "the weights"),
        (dict(lora=lora(K=128), batch=batch()), _lib.ERR_INVALID_ARG, "the weights"),
        (dict(lora=lora(R=257), batch=batch()), _lib.ERR_UNSUPPORTED, "rank"),
        (dict(lora=lora(L=1025), batch=batch(L=1025)), _lib.ERR_UNSUPPORTED, "num_adapters"),
        (dict(lora=lora(b=None), batch=batch()), _lib.ERR_INVALID_ARG, "non-NULL"),
        (dict(lora=lora(), batch=batch(order=None)), _lib.ERR_INVALID_ARG, "non-NULL"),
        (dict(lora=lora(), batch=batch(T=5)), _lib.ERR_INVALID_ARG, "batch holds"),
        (dict(lora=lora(), batch=batch(L=3)), _lib.ERR_INVALID_ARG, "batch holds"),
    ],
)
def test_linear_refusals(over, want, frag):
    a = dict(w=lin(), T=4, x=P, xt=BF, stride=256, xs=None, lora=None, batch=None, out=P, ws=P, n=1 << 40)
    a.update(over)
    st, msg = got(_lib.lib().kmoe_linear(a["w"], a["T"], a["x"], a["xt"], a["stride"], a["xs"], a["lora"], a["batch"],
                                         a["out"], a["ws"], a["n"], None))  # fmt: skip
    assert st == want and frag in msg


def test_packing_refusals():
    L = _lib.lib()
    q = _lib.KmoeWeight(P, I8, P, F32, _lib.SCALE_CHANNEL)
    f = _lib.KmoeWeight(P, F32, None, F32, _lib.SCALE_NONE)
    b = _lib.KmoeWeight(P, BF, None, F32, _lib.SCALE_NONE)
    assert L.kmoe_linear_pack(f, lin(), None) == _lib.ERR_INVALID_ARG
    assert L.kmoe_linear_pack(b, lin(), None) == _lib.ERR_INVALID_ARG
    assert L.kmoe_linear_pack(q, lin(dtype=BF), None) == _lib.ERR_INVALID_ARG
    assert L.kmoe_linear_pack(q, lin(scale=None), None) == _lib.ERR_INVALID_ARG
    assert L.kmoe_linear_pack(None, lin(), None) == _lib.ERR_INVALID_ARG
    for first, count, rank in ((-1, 1, 8), (0, 5, 8), (4, 1, 8), (5, 0, 8), (0, 1, 17), (0, 1, 0), (0, -1, 8)):
        assert L.kmoe_lora_pack(lora(), first, count, rank, P, P, P, None) == _lib.ERR_INVALID_ARG
    assert L.kmoe_lora_pack(lora(), 0, 1, 8, P, None, P, None) == _lib.ERR_INVALID_ARG
    assert L.kmoe_lora_sort(None, batch(), P, 1 << 20, None) == _lib.ERR_INVALID_ARG
    assert L.kmoe_lora_sort(P, batch(), P, 19, None) == _lib.ERR_WORKSPACE_TOO_SMALL
    assert L.kmoe_lora_sort(P, batch(L=0), P, 1 << 20, None) == _lib.ERR_INVALID_ARG
    assert L.kmoe_lora_sort(P, batch(T=(1 << 20) + 1), P, 1 << 40, None) == _lib.ERR_UNSUPPORTED


@NO_DEVICE
def test_valid_calls_reach_the_device_check():
    L = _lib.lib()
    nodev = _lib.ERR_NO_DEVICE
    assert L.kmoe_add_rms_norm(desc(), P, 2 * P, 3 * P, BF, 1e-6, P, 5 * P, None) == nodev
    assert L.kmoe_add_rms_norm_q8(desc(), P, None, 3 * P, BF, 1e-6, None, 5 * P, 6 * P, None) == nodev
    assert L.kmoe_linear(lin(), 4, P, BF, 256, None, lora(), batch(), P, P, 1 << 40, None) == nodev
    assert L.kmoe_linear(lin(), 0, None, BF, 256, None, None, None, None, None, 0, None) == nodev
    assert L.kmoe_linear(lin(), 4, P, I8, 300, P, None, None, P, P, 1 << 40, None) == nodev
    assert L.kmoe_linear_pack(_lib.KmoeWeight(P, I8, P, BF, _lib.SCALE_TENSOR), lin(), None) == nodev
    assert L.kmoe_lora_pack(lora(), 3, 1, 16, P, P, P, None) == nodev
    assert L.kmoe_lora_sort(P, batch(), P, 20, None) == nodev


def test_sizes():
    L = _lib.lib()
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    assert L.kmoe_linear_pack_bytes(lin(K=2048, N=5120), a, b) == _lib.OK
    assert (a.value, b.value) == (2048 * 5120, 4 * 5120)
    assert L.kmoe_linear_pack_bytes(lin(K=100, N=33, dtype=BF), a, b) == _lib.OK
    assert (a.value, b.value) == (2 * 128 * 64, 4 * 64)
    assert L.kmoe_lora_pack_bytes(lora(L=3, R=8, K=100, N=33), a, b) == _lib.OK
    assert (a.value, b.value) == (3 * 2 * 128 * 32, 3 * 2 * 32 * 64)
    for l in (None, lora(K=4096)):
        before = 0
        for T in (0, 1, 63, 64, 65, 66, 300, 4096):
            w = lin(K=4096)
            assert L.kmoe_linear_workspace_bytes(w, T, BF, l, a) == _lib.OK
            assert a.value >= max(before, T * (2 * 4096 + (4 * 16 if l else 0)))
            before = a.value
            # what one call takes: nothing for aligned rows without adapters, but for partial sums
            for x, stride in ((P, 4096), (P + 2, 4096), (P, 4100), (P, 4104)):
                assert L.kmoe_linear_call_bytes(w, T, x, BF, stride, l, b) == _lib.OK
                assert b.value <= a.value
            assert L.kmoe_linear_call_bytes(w, T, P, BF, 4096, l, b) == _lib.OK
            if l is None:
                assert (b.value == 0) == (not 32 < T <= 64)
    assert L.kmoe_linear_call_bytes(lin(), 4, P, BF, -1, None, b) == _lib.ERR_INVALID_ARG


def test_the_workspace_of_many_tokens_serves_fewer():
    """The kernels change with the number of tokens, and so does what a call needs: partial sums
    for some sizes up to 64 tokens, none for others."""
    L = _lib.lib()
    most, call = ctypes.c_size_t(), ctypes.c_size_t()
    for K, N in ((8192, 4096), (8192, 3500), (65536, 64), (4096, 9216), (100, 20000)):
        for l in (None, lora(R=40, K=K, N=N)):
            for dtype, x_dtype in ((BF, BF), (I8, BF), (I8, I8)):
                w = lin(K=K, N=N, dtype=dtype)
                need = 0
                for T in range(1, 100):
                    for x in (P, P + 2):
                        assert L.kmoe_linear_call_bytes(w, T, x, x_dtype, K, l, call) == _lib.OK
                        need = max(need, call.value)
                    assert L.kmoe_linear_workspace_bytes(w, T, x_dtype, l, most) == _lib.OK
                    assert most.value >= need


def test_python_layer_refuses_cpu_tensors():
    from kappa_amd.qwen3 import LoraAdapters, add_rms_norm, add_rms_norm_q8, lora_batch, prepack_linear, prepack_lora

    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    s = torch.ones(64)
    for call in (
        lambda: add_rms_norm(x, x, s), lambda: add_rms_norm_q8(x, None, s), lambda: prepack_linear(x),
        lambda: prepack_lora(x[None], x[None]), lambda: lora_batch(torch.zeros(2, dtype=torch.int32), 1),
        lambda: LoraAdapters.empty(1, 8, 64, 64, device="cpu"),
    ):  # fmt: skip
        with pytest.raises(ValueError, match="HIP device"):
            call()


@pytest.mark.skipif(shutil.which(os.environ.get("CXX", "g++")) is None, reason="no C++ compiler")
def test_host_code_under_the_sanitizers(tmp_path):
    src = [os.path.join(ROOT, "kappa_amd", "csrc", f) for f in ("host.cpp", "linear_host.cpp")]
    exe = _build(tmp_path, [*src, os.path.join(ROOT, "tests", "sanitize", "linear_checks.cpp")], "linear_checks")
    r = _run(exe)
    assert r.returncode == 0 and "linear checks: ok" in r.stdout, r.stdout + r.stderr
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr
