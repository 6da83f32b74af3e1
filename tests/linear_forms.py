"""Sizes of projections that take every kernel of ``linear``, with the kernel that each
takes per kind of product (bf16 rows with bf16 weights, with int8 weights, int8 rows):
tests/test_linear_forms.py checks the choice on the CPU, tests/test_gpu_linear_forms.py the
results. A name is the form (``linear_form``) with its row groups x column groups or its tile,
whether there are adapters, "deep" where the reduction takes further rounds of loads (the
tiles' rings: where stages are loaded again), and how the adapters' inner products are made.
"""

KINDS = {"bf16": ("bf16", "bf16"), "w8": ("w8c", "bf16"), "i8": ("w8c", "q8")}  # (weights, rows)

# (T, K, N, adapters, rank): the kernels, one name for all three kinds or one each
SIZES = {
    # one launch
    (1, 256, 5120, 0, 0): "one 1x2",
    (24, 256, 5120, 0, 0): "one 2x2",
    (40, 192, 4700, 0, 0): "one 3x2",
    (3, 7000, 300, 0, 0): "one 1x1 deep",
    (32, 4032, 300, 0, 0): "one 2x1 deep",
    (41, 2600, 300, 0, 0): "one 3x1 deep",
    (64, 4096, 96, 0, 0): ("split 4 deep", "split 4 deep", "one 4x1 deep"),
    (64, 2048, 130, 0, 0): "one 4x1",
    (1, 4096, 5120, 0, 0): "one 1x2 deep",
    (24, 4096, 5120, 0, 0): "one 2x2 deep",
    (40, 2600, 4700, 0, 0): "one 3x2 deep",
    # two launches, without adapters and with
    (8, 16500, 65, 0, 0): "split 1 deep",
    (24, 8320, 70, 0, 0): "split 2 deep",
    (48, 5500, 130, 0, 0): "split 3 deep",
    (64, 4224, 2048, 0, 0): "split 4 deep",
    (1, 4200, 130, 3, 16): "split 1 lora deep",
    (24, 4096, 257, 5, 40): "split 2 lora deep",
    (40, 2600, 130, 40, 8): "split 3 lora deep",
    (64, 4096, 2048, 16, 64): "split 4 lora deep",
    # too many partial sums for two launches
    (64, 1088, 140000, 3, 8): "64x128 lora deep, shrink 1",
    (32, 4600, 60000, 3, 8): (
        "32x64 lora deep, shrink 1 again", "32x64 lora deep, shrink 1 again", "split 2 lora deep",
    ),
    # tiles, their rings turning
    (129, 1216, 257, 0, 0): "32x64 deep",
    (80, 4200, 130, 3, 16): "32x64 lora deep, shrink 1 again",
    (700, 1216, 1300, 0, 0): "64x64 deep",
    (700, 1216, 2500, 7, 40): "64x64 lora deep, shrink 1",
    (1100, 1216, 3500, 0, 0): "64x128 deep",
    (1100, 1216, 3500, 7, 40): "64x128 lora deep, shrink 1",
    (1900, 1216, 3900, 0, 0): "128x128 deep",
    (1900, 1216, 3900, 7, 40): "128x128 lora deep, shrink 4",
    (2900, 1216, 3900, 0, 0): "256x256 deep",
    (2900, 1216, 3900, 7, 24): "256x256 lora deep, shrink 2",
    (4200, 1216, 4001, 0, 0): "256x256 quarters deep",
    (4200, 1216, 4001, 7, 40): "256x256 quarters lora deep, shrink 4",
    # the adapters' inner products where the rows stay in registers and where they are read again
    (2100, 192, 300, 5, 24): "32x64 lora, shrink 2",
    (2100, 2600, 130, 5, 24): "32x64 lora deep, shrink 2 again",
    (2100, 2600, 130, 5, 64): "32x64 lora deep, shrink 4 again",
    (300, 4200, 130, 40, 200): "32x64 lora deep, shrink 1 again",
}  # fmt: skip


def names(size):
    """The size's kernel per kind, in the order of KINDS."""
    n = SIZES[size]
    return (n, n, n) if isinstance(n, str) else n
