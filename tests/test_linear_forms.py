"""Which kernels a projection's call runs, by its sizes and types (CPU): the sizes of
linear_forms.py take the kernels they are listed for, and between them every kernel, so that a
change of a threshold cannot leave one without a test on the GPU."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from conftest import ROOT
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
