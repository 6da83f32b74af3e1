"""The steps either side of the MoE block in a Qwen3 MoE layer.

``rms_norm`` mirrors kappa/qwen3/norms.py:10-16 and ``moe_block_ffn`` the MoE
half of the layer (kappa/qwen3/block.py:71-82, 153-164, 196-207)::

    h2 = rms_norm(h, params.pre_ffn_norm)
    out = moe_swiglu_ffn(h2, router, gate_proj, up_proj, down_proj, cfg=cfg)
    return h + out

``moe_block_ffn`` runs the three steps as one C-ABI call (kmoe_forward_block):
the norm writes h2 once into the workspace and the combine kernel adds the
block's output to h, so the separate add and its [T, D] round trip disappear.
"""

from __future__ import annotations

import torch

from .. import _lib
from .architecture import Qwen3Config
from .ffn_moe import PackedExperts, _desc, _impl_and_capacity, _moe_forward, _norm_scale, _stream
from .projection import Q8Rows, _elsewhere
from .projection import _stream as _raw_stream
from .quant import Weight, kmoe_dtype


def rms_norm(
    x: torch.Tensor, scale: torch.Tensor, *, epsilon: float = 1e-6, out_dtype: torch.dtype | None = None
) -> torch.Tensor:
    """RMSNorm with a learnable ``scale`` (kappa/qwen3/norms.py:10-16): ``x * scale``
    after normalising by ``rsqrt(mean(x^2) + epsilon)``, computed in f32 and
    returned in ``x.dtype``."""
    if out_dtype is not None and out_dtype != x.dtype:
        raise ValueError(f"out_dtype must be x.dtype ({x.dtype}); got {out_dtype}")
    if x.device.type != "cuda":
        raise ValueError(f"x must be on a HIP device (got {x.device}); rms_norm has no CPU implementation")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"x must be bfloat16 or float32 (got {x.dtype})")
    d = int(x.shape[-1])
    T = x.numel() // d if d else 0
    xf = x.reshape(T, d).contiguous()
    sc = _norm_scale(scale, d, x.device)
    out = torch.empty((T, d), dtype=x.dtype, device=x.device)
    desc = _desc(T, d, 1, 1, 1, x.dtype)
    _lib.check(
        _lib.lib().kmoe_rms_norm(
            desc, xf.data_ptr(), sc.data_ptr(), kmoe_dtype(sc.dtype), float(epsilon), out.data_ptr(), _stream(x.device)
        )
    )
    return out.reshape(x.shape)


_CODE = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}


def _norm_inputs(x: torch.Tensor, residual: torch.Tensor | None, scale: torch.Tensor):
    """Contiguous x and residual, the norm scale, and kmoe_desc (the checks a serving loop pays
    for on every call are kept to attributes)."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"x must be a torch tensor on a HIP device (got {getattr(x, 'device', type(x))})")
    dtype, dev, shape = x.dtype, x.device, x.shape
    code = _CODE.get(dtype)
    if code is None:
        raise ValueError(f"x must be bfloat16 or float32 (got {dtype})")
    if not shape:
        raise ValueError("x must have at least one axis")
    if residual is not None:
        if (
            not isinstance(residual, torch.Tensor)
            or residual.shape != shape or residual.dtype != dtype or residual.device != dev
        ):  # fmt: skip
            raise ValueError(
                f"residual must be as x, {tuple(shape)} {dtype} on {dev} (got "
                f"{tuple(getattr(residual, 'shape', ()))} {getattr(residual, 'dtype', type(residual))} on "
                f"{getattr(residual, 'device', None)})"
            )
        residual = residual.contiguous()
    d = shape[-1]
    if not (
        isinstance(scale, torch.Tensor) and scale.shape == shape[-1:] and scale.dtype in _CODE
        and scale.device == dev and scale.is_contiguous()
    ):  # fmt: skip
        scale = _norm_scale(scale, d, dev)
    desc = _lib.KmoeDesc(x.numel() // d if d else 0, d, 1, 1, 1, code, _lib.IMPL_GATHER_EINSUM, 64, 0, _lib.KERNELS_AUTO)
    return x.contiguous(), residual, scale, desc


def add_rms_norm(
    x: torch.Tensor, residual: torch.Tensor, scale: torch.Tensor, *, epsilon: float = 1e-6
) -> tuple[torch.Tensor, torch.Tensor]:
    """The residual's addition and the norm after it, in one pass: ``(rms_norm(h, scale), h)``
    with ``h = x + residual`` (kappa/qwen3/block.py:71, 153, 196), bit for bit what the two
    steps give. ``x`` and ``residual`` are ``[..., D]`` of one type, bfloat16 or float32."""
    if residual is None:
        raise ValueError("add_rms_norm needs a residual (rms_norm takes none)")
    x, residual, sc, desc = _norm_inputs(x, residual, scale)
    dev = x.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return add_rms_norm(x, residual, sc, epsilon=epsilon)
    h, out = torch.empty_like(x), torch.empty_like(x)
    _lib.check(
        _lib.lib().kmoe_add_rms_norm(
            desc, x.data_ptr(), residual.data_ptr(), sc.data_ptr(), _CODE[sc.dtype], float(epsilon), h.data_ptr(),
            out.data_ptr(), _raw_stream(dev),
        )
    )  # fmt: skip
    return out, h


def add_rms_norm_q8(
    x: torch.Tensor, residual: torch.Tensor | None, scale: torch.Tensor, *, epsilon: float = 1e-6
) -> tuple[Q8Rows, torch.Tensor]:
    """``add_rms_norm`` with the normalised rows in 8 bits, for ``linear``: ``(rows, h)``. With
    ``v`` the normalised row in float32, ``rows.scale = max|v| / 127`` and ``rows.values =
    rint(v / rows.scale)``; a row with an infinity or a NaN has a NaN scale. ``residual`` may
    be None (``h`` is ``x``)."""
    x, residual, sc, desc = _norm_inputs(x, residual, scale)
    dev = x.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return add_rms_norm_q8(x, residual, sc, epsilon=epsilon)
    h = x if residual is None else torch.empty_like(x)
    q = torch.empty_like(x, dtype=torch.int8)
    s = x.new_empty((*x.shape[:-1], 1), dtype=torch.float32)
    _lib.check(
        _lib.lib().kmoe_add_rms_norm_q8(
            desc, x.data_ptr(), None if residual is None else residual.data_ptr(), sc.data_ptr(), _CODE[sc.dtype],
            float(epsilon), None if residual is None else h.data_ptr(), q.data_ptr(), s.data_ptr(), _raw_stream(dev),
        )
    )  # fmt: skip
    return Q8Rows(q, s), h


def moe_block_ffn(
    h: torch.Tensor,
    pre_ffn_norm: torch.Tensor,
    router_w: Weight,
    ffn_gate: Weight,
    ffn_up: Weight,
    ffn_down: Weight,
    *,
    cfg: Qwen3Config,
    epsilon: float = 1e-6,
    packed: PackedExperts | None = None,
) -> torch.Tensor:
    """``h + moe_swiglu_ffn(rms_norm(h, pre_ffn_norm), ...)`` (kappa/qwen3/block.py:196-207).

    ``h`` is the residual stream ``[B, T, D]``; the result has its shape and dtype."""
    if not cfg.use_moe:
        raise ValueError("moe_swiglu_ffn requires cfg.use_moe")
    b, t = int(h.shape[0]), int(h.shape[1])
    impl, capacity = _impl_and_capacity(cfg, b * t)
    return _moe_forward(
        h, router_w, ffn_gate, ffn_up, ffn_down,
        num_experts=cfg.num_experts, num_experts_per_tok=cfg.num_experts_per_tok, impl=impl,
        decode_threshold=cfg.moe_ragged_decode_token_threshold, packed=packed, capacity=capacity,
        norm=(pre_ffn_norm, epsilon),
    )  # fmt: skip
