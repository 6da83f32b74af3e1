"""Packed weights, adapters and batches whose fields do not belong together (made by hand or by
dataclasses.replace) are refused before a kernel reads past a buffer (CPU: the check needs no
device); and so are an output and a workspace that overlap the rows or each other."""

from __future__ import annotations

import dataclasses
import os
import shutil

import pytest
import torch

from conftest import ROOT
from test_host_sanitized import _build, _run

from kappa_amd.qwen3 import LoraAdapters, LoraBatch, PackedLinear

K, N = 200, 40  # packed as 256 x 64
BF, I8, F32, I32 = torch.bfloat16, torch.int8, torch.float32, torch.int32


def packed(dtype=I8):
    return PackedLinear(torch.zeros(256 * 64, dtype=dtype), torch.zeros(64), K, N)


def adapters():
    # 3 adapters, rank 8 packed as 32
    return LoraAdapters(torch.zeros(3 * 256 * 32, dtype=BF), torch.zeros(3 * 64 * 32, dtype=BF), torch.zeros(3), 3, 8, K, N)


def batch():
    return LoraBatch(torch.zeros(3 * 5 + 4, dtype=I32), 5, 3)


@pytest.mark.parametrize("make", [packed, lambda: packed(BF), adapters, batch])
def test_what_fits_is_taken(make):
    m = make()
    assert m.struct is m.struct


@pytest.mark.parametrize(
    "make,over,match",
    [
        (packed, dict(values=torch.zeros(256 * 64 - 1, dtype=I8)), "values must be"),
        (packed, dict(values=torch.zeros(256 * 128, dtype=I8)[::2]), "values must be"),
        (packed, dict(values=torch.zeros(256 * 64)), "int8 or bfloat16"),
        (packed, dict(scale=torch.zeros(N)), "scale must be"),
        (packed, dict(scale=torch.zeros(64, dtype=BF)), "scale must be"),
        (packed, dict(scale=None), "scale must be"),
        (packed, dict(scale=torch.zeros(64, device="meta")), "scale must be"),
        (packed, dict(in_features=257), "values must be"),
        (packed, dict(out_features=65), "values must be"),
        (packed, dict(out_features=0), "out_features must be"),
        (adapters, dict(a=torch.zeros(3 * 256 * 32 - 1, dtype=BF)), "a must be"),
        (adapters, dict(b=torch.zeros(3 * 64 * 32 - 1, dtype=BF)), "b must be"),
        (adapters, dict(a=torch.zeros(3 * 256 * 32, dtype=torch.float16)), "a must be"),
        (adapters, dict(factor=torch.zeros(2)), "factor must be"),
        (adapters, dict(factor=torch.zeros(3, dtype=torch.float64)), "factor must be"),
        (adapters, dict(num_adapters=4), "a must be"),
        (adapters, dict(rank=33), "a must be"),
        (adapters, dict(rank=0), "must be >= 1"),
        (batch, dict(buffer=torch.zeros(3 * 5 + 3, dtype=I32)), "buffer must be"),
        (batch, dict(buffer=torch.zeros(3 * 5 + 4, dtype=torch.int64)), "buffer must be"),
        (batch, dict(tokens=6), "buffer must be"),
        (batch, dict(num_adapters=4), "buffer must be"),
    ],
)
def test_what_does_not_fit_is_refused(make, over, match):
    with pytest.raises(ValueError, match=match):
        dataclasses.replace(make(), **over).struct


@pytest.mark.skipif(shutil.which(os.environ.get("CXX", "g++")) is None, reason="no C++ compiler")
def test_overlaps(tmp_path):
    src = [os.path.join(ROOT, "kappa_amd", "csrc", f) for f in ("host.cpp", "linear_host.cpp")]
    exe = _build(tmp_path, [*src, os.path.join(ROOT, "tests", "sanitize", "linear_apart.cpp")], "linear_apart")
    r = _run(exe)
    assert r.returncode == 0 and "linear apart: ok" in r.stdout, r.stdout + r.stderr
