"""Projections of a decoder layer on MI355X, and the low-rank adapters of many requests
beside them.

``linear(x, w)`` is the ``x @ to_compute_dtype(w)`` of the reference's q, k, v and o
projections (kappa/qwen3/linear.py:10-25) with the heads side by side in the last axis. ``w`` is laid out
once by ``prepack_linear`` (bf16, or a ``Q8Weight`` whose scale multiplies the f32 sum);
``x`` is bf16 or the 8-bit rows of ``add_rms_norm_q8``.

Adapters (the reference has none): ``prepack_lora`` lays out the adapters of one projection,
``lora_batch`` sorts a step's tokens by adapter once, and every projection of the step takes
that batch::

    batch = lora_batch(adapter, num_adapters)          # adapter[t]: of token t, -1 for none
    qkv = linear(normed, w_qkv, lora=lora_qkv, batch=batch)

adds ``factor[a] * (x[t] @ a[a]) @ b[a]`` to token t's row. Like the rest of the package this
is for inference: no gradients.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from functools import cached_property
from typing import NamedTuple, Union

import torch

from .. import _lib
from .quant import Q8Weight, _require_cuda, is_q8_weight, weight_struct


class Q8Rows(NamedTuple):
    """Rows in int8 with one scale each: row ``t`` stands for ``values[t] * scale[t]``."""

    values: torch.Tensor  # [..., D] int8
    scale: torch.Tensor  # [..., 1] float32


def _stream(device: torch.device) -> int:
    """The current stream of ``device`` (the raw handle: a torch.cuda.Stream for it takes 2 us)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _elsewhere(device: torch.device) -> bool:
    """Whether ``device`` is not the current one, where launches go."""
    return device.index != torch._C._cuda_getDevice()


def _require_buffer(t: torch.Tensor, name: str, dtype: torch.dtype, n: int, device: torch.device) -> int:
    """The address of a buffer that the kernels take for ``n`` elements."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device or not t.is_contiguous() or t.numel() < n:
        what = f"{tuple(t.shape)} {t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n} elements on {device} (got {what})")
    return t.data_ptr()


class _WithStruct:
    """Keeps the C struct of a frozen dataclass after its first use, which checks that the buffers
    hold what the sizes say; copies make their own."""

    def __getstate__(self):
        state = dict(self.__dict__)
        state.pop("struct", None)
        return state


@dataclass(frozen=True)
class PackedLinear(_WithStruct):
    """A projection's weights in the gfx950 layout (include/kmoe.h, kmoe_linear_weight)."""

    values: torch.Tensor
    scale: torch.Tensor
    in_features: int
    out_features: int

    @cached_property
    def struct(self) -> _lib.KmoeLinear:
        dev, dtype = self.values.device, self.values.dtype
        if dtype not in (torch.int8, torch.bfloat16):
            raise ValueError(f"the packed values must be int8 or bfloat16 (got {dtype})")
        code = _lib.DTYPE_I8 if dtype == torch.int8 else _lib.DTYPE_BF16
        st = _lib.KmoeLinear(None, None, code, self.in_features, self.out_features)
        nv, ns = ctypes.c_size_t(), ctypes.c_size_t()
        _lib.check(_lib.lib().kmoe_linear_pack_bytes(st, ctypes.byref(nv), ctypes.byref(ns)))
        st.values = _require_buffer(self.values, "values", dtype, nv.value // dtype.itemsize, dev)
        st.scale = _require_buffer(self.scale, "scale", torch.float32, ns.value // 4, dev)
        return st

    @property
    def nbytes(self) -> int:
        return self.values.numel() * self.values.element_size() + 4 * self.scale.numel()


def prepack_linear(w: Union[torch.Tensor, Q8Weight]) -> PackedLinear:
    """One-time relayout of a projection's ``[in, out]`` weights for the MFMA kernels: bf16,
    or a ``Q8Weight`` with one scale or one per output channel (``[out]`` or ``[1, out]``).
    The copy holds the same values and does not follow later writes to ``w``."""
    v = w.values if is_q8_weight(w) else w
    _require_cuda(v, "w")
    if v.dim() != 2:
        raise ValueError(f"w must be [in, out] (got shape {tuple(v.shape)})")
    if not is_q8_weight(w) and v.dtype != torch.bfloat16:
        raise ValueError(f"w must be bfloat16 or a Q8Weight (got {v.dtype})")
    K, N = (int(s) for s in v.shape)
    dtype = torch.int8 if is_q8_weight(w) else torch.bfloat16
    code = _lib.DTYPE_I8 if is_q8_weight(w) else _lib.DTYPE_BF16
    st = _lib.KmoeLinear(None, None, code, K, N)
    nv, ns = ctypes.c_size_t(), ctypes.c_size_t()
    L = _lib.lib()
    _lib.check(L.kmoe_linear_pack_bytes(st, ctypes.byref(nv), ctypes.byref(ns)))
    with torch.cuda.device(v.device):
        src, keep = weight_struct(w, v.device, n_out=N, n_groups=None, name="w")
        values = torch.empty(nv.value // dtype.itemsize, dtype=dtype, device=v.device)
        scale = torch.empty(ns.value // 4, dtype=torch.float32, device=v.device)
        packed = PackedLinear(values, scale, K, N)
        _lib.check(L.kmoe_linear_pack(src, packed.struct, _stream(v.device)))
    return packed


@dataclass(frozen=True)
class LoraAdapters(_WithStruct):
    """The adapters of one projection in the gfx950 layout (include/kmoe.h, kmoe_lora)."""

    a: torch.Tensor
    b: torch.Tensor
    factor: torch.Tensor
    num_adapters: int
    rank: int
    in_features: int
    out_features: int

    @cached_property
    def struct(self) -> _lib.KmoeLora:
        dev = self.a.device
        st = _lib.KmoeLora(None, None, None, self.num_adapters, self.rank, self.in_features, self.out_features)
        na, nb = ctypes.c_size_t(), ctypes.c_size_t()
        _lib.check(_lib.lib().kmoe_lora_pack_bytes(st, ctypes.byref(na), ctypes.byref(nb)))
        st.a = _require_buffer(self.a, "a", torch.bfloat16, na.value // 2, dev)
        st.b = _require_buffer(self.b, "b", torch.bfloat16, nb.value // 2, dev)
        st.factor = _require_buffer(self.factor, "factor", torch.float32, self.num_adapters, dev)
        return st

    @staticmethod
    def empty(
        num_adapters: int, rank: int, in_features: int, out_features: int, *, device: Union[str, torch.device] = "cuda"
    ) -> LoraAdapters:
        """Slots that add nothing until ``store`` fills them; ``rank`` is the largest they take."""
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"the adapters must be on a HIP device (got {device})")
        st = _lib.KmoeLora(None, None, None, num_adapters, rank, in_features, out_features)
        na, nb = ctypes.c_size_t(), ctypes.c_size_t()
        _lib.check(_lib.lib().kmoe_lora_pack_bytes(st, ctypes.byref(na), ctypes.byref(nb)))
        a = torch.zeros(na.value // 2, dtype=torch.bfloat16, device=device)
        b = torch.zeros(nb.value // 2, dtype=torch.bfloat16, device=device)
        factor = torch.zeros(num_adapters, dtype=torch.float32, device=device)
        return LoraAdapters(a, b, factor, num_adapters, rank, in_features, out_features)

    def store(self, first: int, a: torch.Tensor, b: torch.Tensor, factor: Union[float, torch.Tensor]) -> None:
        """Fills the slots ``first ..`` from ``a`` ``[count, in, r]`` and ``b`` ``[count, r, out]``
        (bf16, ``r <= rank``; without the first axis: one slot) and ``factor`` (a number, or
        ``[count]``; an adapter's alpha / r)."""
        if a.dim() == 2 and b.dim() == 2:
            a, b = a.unsqueeze(0), b.unsqueeze(0)
        dev = self.a.device
        for name, t in (("a", a), ("b", b)):
            if t.device != dev or t.dtype != torch.bfloat16:
                raise ValueError(f"{name} must be bfloat16 on {dev} (got {t.dtype} on {t.device})")
        if a.dim() != 3 or b.dim() != 3:
            raise ValueError(f"a and b must be [count, in, r] and [count, r, out] (got {tuple(a.shape)}, {tuple(b.shape)})")
        count, K, r = (int(s) for s in a.shape)
        if K != self.in_features or tuple(b.shape) != (count, r, self.out_features):
            raise ValueError(
                f"a {tuple(a.shape)} and b {tuple(b.shape)} are not [count, {self.in_features}, r] and "
                f"[count, r, {self.out_features}]"
            )
        if isinstance(factor, torch.Tensor):
            if factor.numel() != count:
                raise ValueError(f"factor has {factor.numel()} entries for {count} adapters")
            f = factor.reshape(count).to(device=dev, dtype=torch.float32).contiguous()
        else:
            f = torch.full((count,), float(factor), dtype=torch.float32, device=dev)
        a, b = a.contiguous(), b.contiguous()
        with torch.cuda.device(dev):
            _lib.check(
                _lib.lib().kmoe_lora_pack(
                    self.struct, first, count, r, a.data_ptr(), b.data_ptr(), f.data_ptr(), _stream(dev)
                )
            )


def prepack_lora(a: torch.Tensor, b: torch.Tensor, factor: Union[float, torch.Tensor] = 1.0) -> LoraAdapters:
    """One-time relayout of a projection's adapters: ``a`` ``[L, in, rank]`` and ``b``
    ``[L, rank, out]`` in bf16 (adapters of smaller rank filled up with zeros, or
    ``LoraAdapters.empty`` and ``store``), ``factor`` a number or ``[L]``."""
    _require_cuda(a, "a")
    _require_cuda(b, "b")
    if a.dim() != 3 or b.dim() != 3:
        raise ValueError(f"a and b must be [L, in, rank] and [L, rank, out] (got {tuple(a.shape)}, {tuple(b.shape)})")
    L, K, r = (int(s) for s in a.shape)
    out = LoraAdapters.empty(L, r, K, int(b.shape[2]), device=a.device)
    out.store(0, a, b, factor)
    return out


@dataclass(frozen=True)
class LoraBatch(_WithStruct):
    """A step's tokens sorted by adapter (include/kmoe.h, kmoe_lora_batch)."""

    buffer: torch.Tensor  # int32: adapter, order and sorted [tokens], offsets [num_adapters + 1], the sort's scratch
    tokens: int
    num_adapters: int

    @cached_property
    def struct(self) -> _lib.KmoeLoraBatch:
        count = 3 * self.tokens + self.num_adapters + 1
        p, n = _require_buffer(self.buffer, "buffer", torch.int32, count, self.buffer.device), 4 * self.tokens
        return _lib.KmoeLoraBatch(p, p + n, p + 2 * n, p + 3 * n, self.tokens, self.num_adapters)


def lora_batch(adapter: torch.Tensor, num_adapters: int) -> LoraBatch:
    """Sorts the tokens by ``adapter`` (int32 or int64, one per token, on the device); a value
    outside ``[0, num_adapters)`` means none. The batch holds a copy of ``adapter``."""
    _require_cuda(adapter, "adapter")
    if adapter.dtype == torch.int64:
        adapter = adapter.clamp(-1, num_adapters).to(torch.int32)
    if adapter.dtype != torch.int32:
        raise ValueError(f"adapter must be int32 or int64 (got {adapter.dtype})")
    adapter = adapter.reshape(-1).contiguous()
    T, dev = adapter.numel(), adapter.device
    st = _lib.KmoeLoraBatch(None, None, None, None, T, num_adapters)
    L = _lib.lib()
    n = ctypes.c_size_t()
    _lib.check(L.kmoe_lora_sort_bytes(st, ctypes.byref(n)))
    with torch.cuda.device(dev):
        buf = torch.empty(3 * T + num_adapters + 1 + n.value // 4, dtype=torch.int32, device=dev)
        batch = LoraBatch(buf, T, num_adapters)
        scratch = buf.data_ptr() + 4 * (3 * T + num_adapters + 1)
        _lib.check(L.kmoe_lora_sort(adapter.data_ptr(), batch.struct, scratch, n.value, _stream(dev)))
    return batch


def linear(
    x: Union[torch.Tensor, Q8Rows],
    w: PackedLinear,
    *,
    lora: LoraAdapters | None = None,
    batch: LoraBatch | None = None,
) -> torch.Tensor:
    """``x @ w`` with the adapters of each token's request: ``[..., in]`` -> bf16 ``[..., out]``.

    ``x`` is bf16, or 8-bit rows (which need int8 weights). Sums are f32 (8-bit rows: exact),
    rounded once at the end. A row's bits do not depend on the other rows' adapters; up to 64
    tokens they do depend on whether ``lora`` is given at all, so a server whose requests may use
    adapters passes it on every step, also where all tokens have -1."""
    if not isinstance(w, PackedLinear):
        raise ValueError(f"w must be a PackedLinear from prepack_linear (got {type(w).__name__})")
    K = w.in_features
    xs = None
    if isinstance(x, Q8Rows):
        v, scale = x
        code = _lib.DTYPE_I8
        if v.dtype != torch.int8 or scale.dtype != torch.float32:
            raise ValueError(f"8-bit rows are int8 with float32 scales (got {v.dtype}, {scale.dtype})")
        if w.values.dtype != torch.int8:
            raise ValueError("8-bit rows need int8 weights")
    else:
        v, code = x, _lib.DTYPE_BF16
        if not isinstance(v, torch.Tensor) or v.dtype != torch.bfloat16:
            raise ValueError(f"x must be bfloat16 or Q8Rows (got {getattr(v, 'dtype', type(v).__name__)})")
    dev = w.values.device
    if v.device != dev:
        raise ValueError(f"x is on {v.device}, w on {dev}")
    if v.dim() < 1 or v.shape[-1] != K:
        raise ValueError(f"x has shape {tuple(v.shape)}, the weights take rows of {K}")
    shape = v.shape[:-1]
    T = v.numel() // K
    if code == _lib.DTYPE_I8:
        if scale.device != dev or scale.numel() != T:
            raise ValueError(f"the scales are {tuple(scale.shape)} on {scale.device}: one per row is wanted")
        scale = scale.contiguous()
        xs = scale.data_ptr()
    # rows of one stride are read where they are
    if not (v.dim() == 2 and v.stride(1) == 1 and v.stride(0) >= K):
        v = v.reshape(T, K)
        if v.stride(1) != 1 or v.stride(0) < K:
            v = v.contiguous()
    stride = v.stride(0) if T > 1 else K
    if stride > K and T * stride * v.element_size() >= 1 << 32:  # past the kernels' offsets
        v, stride = v.contiguous(), K
    if (lora is None) != (batch is None):
        raise ValueError("lora and batch come together")
    ls = bs = None
    if lora is not None:
        if not isinstance(lora, LoraAdapters) or not isinstance(batch, LoraBatch):
            raise ValueError("lora must be LoraAdapters from prepack_lora, batch a LoraBatch from lora_batch")
        if lora.a.device != dev or batch.buffer.device != dev:
            raise ValueError(f"the adapters are on {lora.a.device}, the batch on {batch.buffer.device}, w on {dev}")
        ls, bs = lora.struct, batch.struct
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return linear(x, w, lora=lora, batch=batch)
    L = _lib.lib()
    n = ctypes.c_size_t()
    _lib.check(L.kmoe_linear_call_bytes(w.struct, T, v.data_ptr(), code, stride, ls, ctypes.byref(n)))
    out = v.new_empty((*shape, w.out_features), dtype=torch.bfloat16)
    ws = v.new_empty(n.value, dtype=torch.uint8) if n.value else None
    _lib.check(
        L.kmoe_linear(
            w.struct, T, v.data_ptr(), code, stride, xs, ls, bs, out.data_ptr(),
            None if ws is None else ws.data_ptr(), n.value, _stream(dev),
        )
    )  # fmt: skip
    return out
