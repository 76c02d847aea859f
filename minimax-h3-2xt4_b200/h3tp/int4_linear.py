"""Column-parallel linear with 4-bit weights and group scales, for few rows.

The modulation projections of a DiT (a handful of embedding rows into six vectors of the
hidden width for every block) and a text encoder's projections at a few tokens are bound
by their weights' bytes alone; here those are 4 bits each plus one scale (and, if wanted,
one zero point) for every `group` of them along K.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import ops


def _stored_scales(scales: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """fp32 scales in the type they are kept in, none of them 0.  Below fp16's normal numbers they
    are rounded up to its steps of 2^-24: rounded down, a scale would cut its largest weights off."""
    if dtype == torch.float16:
        step = 2.0 ** -24
        scales = torch.where(scales < torch.finfo(dtype).tiny, (scales / step).ceil().clamp(min=1) * step, scales)
    stored = scales.clamp(min=torch.finfo(torch.float32).tiny).to(dtype)
    if not torch.isfinite(stored).all():
        raise ValueError(f"weight: not finite, or beyond what scales of {dtype} reach")
    return stored


def quantize_int4(weight: torch.Tensor, group: int = 128, zero_points: bool = False,
                  scale_dtype: torch.dtype = torch.float32):
    """Rounds a weight [N, K] to 4-bit codes with one scale for each group along K.

    Symmetric (zero_points False): W = scale * (code - 8), scale = max|W| / 7 of the
    group.  With zero points: W = scale * (code - zero), the range [min(W, 0), max(W, 0)]
    over 15 steps.  The codes are chosen for the scales as stored (scale_dtype); weights
    that no finite scale of that type spans are refused.
    Returns (packed uint8 [N, ceil(K / 2)], scales [N, ceil(K / group)], zeros or None),
    as ops.int4_linear takes them, on the weight's device."""
    if weight.ndim != 2 or not weight.is_floating_point() or min(weight.shape) < 1:
        raise ValueError("weight: floating [N, K] required")
    if group not in ops.INT4_GROUPS:
        raise ValueError(f"group must be one of {ops.INT4_GROUPS}")
    if scale_dtype not in ops._TYPES:
        raise ValueError("scale_dtype must be fp32, fp16 or bf16")
    N, K = weight.shape
    groups = -(-K // group)
    w = torch.nn.functional.pad(weight.detach().float(), (0, groups * group - K)).unflatten(1, (groups, group))
    if zero_points:
        lo, hi = w.amin(2).clamp(max=0), w.amax(2).clamp(min=0)
        scales = _stored_scales(hi / 15 - lo / 15, scale_dtype)
        zeros = torch.round(-lo / scales.float()).clamp(0, 15)
    else:
        scales = _stored_scales(w.abs().amax(2) / 7, scale_dtype)
        zeros = None
    offset = 8.0 if zeros is None else zeros[:, :, None]
    code = torch.round(w / scales.float()[:, :, None] + offset).clamp(0, 15)
    code = code.to(torch.uint8).flatten(1)[:, :K]
    code = torch.nn.functional.pad(code, (0, K % 2))
    packed = (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous()
    return packed, scales, None if zeros is None else zeros.to(torch.uint8)


class ColumnParallelLinearINT4(nn.Module):
    """Column-parallel linear with 4-bit weights: output features split across TP ranks, no
    communication.  Input [..., in_features] fp16 or bf16 -> output [..., out_features //
    world] in `out_dtype` (None: the input's type; modulation tables are read as fp32).
    Meant for few rows; the INT8 projections serve the long sequences."""

    def __init__(self, in_features: int, out_features: int, rank: int = 0, world_size: int = 1,
                 group: int = 128, zero_points: bool = False, bias: bool = False,
                 scale_dtype: torch.dtype = torch.float32, out_dtype: Optional[torch.dtype] = None,
                 device: Optional[torch.device] = None, components: int = 1):
        super().__init__()
        if out_features % (world_size * components):
            raise ValueError("out_features must divide by the ranks and components")
        if group not in ops.INT4_GROUPS:
            raise ValueError(f"group must be one of {ops.INT4_GROUPS}")
        self.in_features = in_features
        self.out_features_per_rank = n = out_features // world_size
        self.rank, self.world_size, self.components = rank, world_size, components
        self.group, self.out_dtype = group, out_dtype
        device = torch.device(device) if device is not None else torch.device("cuda", rank)
        groups = -(-in_features // group)

        def held(*shape, dtype):
            return nn.Parameter(torch.empty(*shape, dtype=dtype, device=device), requires_grad=False)

        self.weight = held(n, (in_features + 1) // 2, dtype=torch.uint8)
        self.weight_scale = held(n, groups, dtype=scale_dtype)
        self.weight_zero = held(n, groups, dtype=torch.uint8) if zero_points else None
        self.bias = held(n, dtype=torch.float32) if bias else None

    def _rows(self, full):
        """This rank's rows of every component of a full tensor."""
        rows = self.out_features_per_rank * self.world_size
        if full.ndim < 1 or full.shape[0] != rows:
            raise ValueError(f"{rows} rows over all ranks required, got {tuple(full.shape)}")
        parts = full.chunk(self.components, 0)
        return torch.cat([p.chunk(self.world_size, 0)[self.rank] for p in parts], 0)

    def _load(self, **given):
        """Copies this rank's parts into the parameters, after all of them were checked."""
        parts = {name: part for name, part in given.items() if part is not None}
        for name, part in parts.items():
            held = getattr(self, name)
            if part.shape != held.shape or part.dtype != held.dtype:
                raise ValueError(f"{name}: {held.dtype} {tuple(held.shape)} a rank required, got "
                                 f"{part.dtype} {tuple(part.shape)}")
        for name, part in parts.items():
            getattr(self, name).data.copy_(part)

    def load_quantized(self, packed, scales, zeros=None, bias=None):
        """Loads this rank's rows of a full quantised weight (quantize_int4's three results)."""
        if (zeros is None) != (self.weight_zero is None) or (bias is None) != (self.bias is None):
            raise ValueError("zero points and bias must be given exactly where the module holds them")
        if zeros is not None and zeros.numel() and int(zeros.max()) > 15:
            raise ValueError("zero points must lie between 0 and 15")
        self._load(weight=self._rows(packed), weight_scale=self._rows(scales),
                   weight_zero=None if zeros is None else self._rows(zeros),
                   bias=None if bias is None else self._rows(bias))

    def load_from_full(self, full_weight: torch.Tensor, bias=None):
        """Quantises this rank's rows of a full floating weight and loads them."""
        if (bias is None) != (self.bias is None):
            raise ValueError("a bias must be given exactly where the module holds one")
        packed, scales, zeros = quantize_int4(self._rows(full_weight), self.group, self.weight_zero is not None,
                                              self.weight_scale.dtype)
        self._load(weight=packed, weight_scale=scales, weight_zero=zeros,
                   bias=None if bias is None else self._rows(bias).float())

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.ndim < 1 or x.shape[-1] != self.in_features:
            raise ValueError(f"x: in_features {self.in_features} required, got {tuple(x.shape)}")
        y = ops.int4_linear(x.reshape(-1, self.in_features), self.weight, self.weight_scale,
                            self.weight_zero, group=self.group, bias=self.bias,
                            out_dtype=self.out_dtype)
        return y.reshape(*x.shape[:-1], self.out_features_per_rank)
