"""Which kernels a projection's call runs, by its sizes and types (CPU): the sizes of
linear_forms.py take the kernels they are listed for, and between them every kernel, so that a
change of a threshold cannot leave one without a test on the GPU."""

from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest

from conftest import ROOT
from kappa_amd import _lib
from linear_forms import KINDS, SIZES, names
from test_host_sanitized import _build

# one launch: 1 to 3 row groups x 1 or 2 column groups and 4 x 1; two launches: 4 row groups; tiles:
# 5 sizes and the quarters, each of these with adapters too; the adapters' inner products: 3,
# whose rows are read once or again
KERNELS = 7 + 4 * 2 + 6 * 2 + 3 * 2

pytestmark = pytest.mark.skipif(shutil.which(os.environ.get("CXX", "g++")) is None, reason="no C++ compiler")


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    src = [os.path.join(ROOT, "kappa_amd", "csrc", f) for f in ("host.cpp", "linear_host.cpp")]
    exe = _build(tmp_path_factory.mktemp("forms"), [*src, os.path.join(ROOT, "tests", "sanitize", "linear_forms.cpp")],
                 "linear_forms")  # fmt: skip

    def run(sizes, kind):
        weights, rows = KINDS[kind]
        lines = [f"{T} {K} {N} {int(rows == 'q8')} {int(weights != 'bf16')} {L} {R}\n" for T, K, N, L, R in sizes]
        r = subprocess.run([exe], input="".join(lines), capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr
        return r.stdout.splitlines()

    return run


@pytest.mark.parametrize("k,kind", enumerate(KINDS))
def test_each_size_takes_its_kernels(choose, k, kind):
    assert dict(zip(SIZES, choose(SIZES, kind))) == {s: names(s)[k] for s in SIZES}


@pytest.mark.parametrize("k,kind", enumerate(KINDS))
def test_the_sizes_take_every_kernel(choose, k, kind):
    """What a sweep of sizes reaches, with reductions of every depth, is in the list (a deep one
    stands for the short one, whose loop the other tests' sizes run)."""
    have = {part for s in SIZES for part in names(s)[k].split(", ")}
    tokens = [1, 15, 16, 17, 24, 32, 33, 47, 48, 49, 63, 64, 65, 90, 128, 200, 333, 512, 700, 1024, 1040, 1500, 2048, 2900, 4096, 8192]
    sweep = [
        (T, K, N, L, R) for T in tokens for K in (64, 1024, 2560, 4096, 8192, 16384, 65536)
        for N in (64, 512, 2048, 4400, 5120, 6144, 9216, 20000, 151936) for L, R in ((0, 0), (1, 8), (8, 32), (64, 64), (64, 256))
    ]  # fmt: skip
    reached = {part for line in choose(sweep, kind) for part in line.split(", ")}
    assert len({r.replace(" deep", "") for r in reached}) == KERNELS
    missing = {r for r in reached if r not in have and r + " deep" not in have}
    assert not missing, sorted(missing)


def test_partial_sums_stay_bounded():
    """The workspace of up to 64 tokens: the rows' copy, the adapters' inner values and less than
    64 MB of partial sums, up to the largest weights."""
    L = _lib.lib()
    most, call = ctypes.c_size_t(), ctypes.c_size_t()
    for K, N in ((2048, 151936), (4096, 65536), (65536, 1 << 20), (65536, 64), (16384, 32768)):
        for R in (0, 16):
            lora = _lib.KmoeLora(None, None, None, 4, R, K, N) if R else None
            for dtype, x_dtype in ((_lib.DTYPE_BF16, _lib.DTYPE_BF16), (_lib.DTYPE_I8, _lib.DTYPE_BF16), (_lib.DTYPE_I8, _lib.DTYPE_I8)):
                w = _lib.KmoeLinear(None, None, dtype, K, N)
                need = 0
                for T in range(1, 70):
                    assert L.kmoe_linear_call_bytes(w, T, 0x1002, x_dtype, K, lora, call) == _lib.OK
                    need = max(need, call.value)
                    assert L.kmoe_linear_workspace_bytes(w, T, x_dtype, lora, most) == _lib.OK
                    assert need <= most.value <= (64 << 20) + T * (2 * K + 4 * 32) + 1024
