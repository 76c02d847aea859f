"""QK norm and rotary positions over several axes, on the QKV projection's output
(the counterpart of the reference's fused kernel, patches/tilelang_fp32_rms_rope.py).

Images and video turn the pairs of a head by several positions at once (time, height,
width): every pair belongs to one axis and turns by that axis's position times the pair's
frequency.  RotaryAxes is the plan (which axis and which frequency each pair has);
qk_norm_rope applies it, after a per-head RMS norm, to q and k, and packed_qk_norm_rope
to the packed [q | k | v] rows that ColumnParallelLinearINT8 returns, in place.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import ops

MAX_HEAD_DIM = 256


class RotaryAxes:
    """Which axis turns which pair of a head, and how fast.

    head_dim: elements of a head (<= 256); sections: the elements each axis turns (even
    numbers, in total at most head_dim; the rest of the head is normed and not turned).
    theta: the base of the frequencies, or one for each axis.
    pairing: 'interleaved' pairs elements (2p, 2p + 1), 'half' (p, p + R / 2) of the R
    turned elements.
    order: 'chunked' gives each axis a run of consecutive pairs; 'interleaved' deals the
    pairs to the axes in turn while an axis has pairs left, then to the first that has.
    frequencies: 'per_axis' counts each axis's pairs from 0, theta^(-2 j / section);
    'shared' gives pair p of the whole head theta^(-2 p / R).  inv_freq (R / 2 numbers)
    overrides both, for scaled frequencies.

    The plan lives on the host and travels with each launch: it serves every device and
    stream, and a captured graph keeps its own copy."""

    def __init__(self, head_dim: int, sections, theta=10000.0, *, pairing: str = "interleaved",
                 order: str = "chunked", frequencies: str = "per_axis", inv_freq=None):
        sections = tuple(int(s) for s in sections)
        if not 2 <= head_dim <= MAX_HEAD_DIM:
            raise ValueError(f"head_dim must lie between 2 and {MAX_HEAD_DIM}")
        if not sections or any(s < 0 or s % 2 for s in sections) or not 0 < sum(sections) <= head_dim:
            raise ValueError("sections must be even and add up to at most head_dim")
        if pairing not in ("interleaved", "half"):
            raise ValueError("pairing must be 'interleaved' or 'half'")
        if order not in ("chunked", "interleaved"):
            raise ValueError("order must be 'chunked' or 'interleaved'")
        if frequencies not in ("per_axis", "shared"):
            raise ValueError("frequencies must be 'per_axis' or 'shared'")
        self.head_dim = int(head_dim)
        self.sections = sections
        self.n_axes = len(sections)
        self.pairs = sum(sections) // 2
        self.half = int(pairing == "half")
        self.axis_of_pair = self._deal(order)
        if inv_freq is None:
            inv_freq = self._frequencies(theta, frequencies)
        self.inv_freq = tuple(float(f) for f in inv_freq)
        if len(self.inv_freq) != self.pairs or not all(map(math.isfinite, self.inv_freq)):
            raise ValueError(f"inv_freq: {self.pairs} finite numbers required")
        # turns per position: the kernel reduces whole turns away in 64 bits
        self.turns = (ctypes.c_double * self.pairs)(*(f / (2 * math.pi) for f in self.inv_freq))
        self.axis = (ctypes.c_uint8 * self.pairs)(*self.axis_of_pair)

    def _deal(self, order):
        left = [s // 2 for s in self.sections]
        if order == "chunked":
            return tuple(a for a, n in enumerate(left) for _ in range(n))
        dealt = []
        for p in range(self.pairs):
            a = p % self.n_axes
            if not left[a]:
                a = next(j for j, n in enumerate(left) if n)
            left[a] -= 1
            dealt.append(a)
        return tuple(dealt)

    def _frequencies(self, theta, frequencies):
        bases = [float(theta)] * self.n_axes if isinstance(theta, (int, float)) else [float(t) for t in theta]
        if len(bases) != self.n_axes or not all(b > 0 for b in bases):
            raise ValueError("theta must be positive, one number or one for each axis")
        seen = [0] * self.n_axes
        out = []
        for p, a in enumerate(self.axis_of_pair):
            j, total = (p, 2 * self.pairs) if frequencies == "shared" else (seen[a], self.sections[a])
            out.append(bases[a] ** (-2.0 * j / total))
            seen[a] += 1
        return out


def qk_norm_rope(q, k, positions, axes: RotaryAxes, *, q_weight=None, k_weight=None, eps=1e-6,
                 norm=True, out_q=None, out_k=None):
    """q [S, Hq, D] and k [S, Hk, D] (k may be None, Hk may differ), fp32, fp16 or bf16, any
    token and head strides: each head times rsqrt(mean(x^2) + eps) and its weight (fp32
    [D] or None; norm=False skips the norm), then turned by `axes` at `positions`
    (int32, int64 or fp32 [S, axes]; [S] for a single axis).  Everything between the load
    and the one rounding of the result is fp32, the angles 64 bits until they are reduced.

    Returns (q', k') in fresh [S, H, D] tensors, or in out_q / out_k: any strides without
    overlap (a head-major view, say), or the input itself for an update in place."""
    return ops.qk_norm_rope(q, k, positions, axes, q_weight=q_weight, k_weight=k_weight, eps=eps,
                            norm=norm, out_q=out_q, out_k=out_k)


def packed_qk_norm_rope(qkv, heads: int, kv_heads: int, positions, axes: RotaryAxes, *,
                        q_weight=None, k_weight=None, eps=1e-6, norm=True):
    """qk_norm_rope in place on packed rows [S, (heads + 2 kv_heads) * D] = [q | k | v] of one
    rank's QKV projection.  Returns the views (q, k, v), each [S, H, D]."""
    D = axes.head_dim
    if not isinstance(qkv, torch.Tensor):
        raise ValueError("qkv: tensor required")
    if qkv.ndim != 2 or qkv.shape[1] != (heads + 2 * kv_heads) * D:
        raise ValueError(f"qkv: [S, {(heads + 2 * kv_heads) * D}] required, got {tuple(qkv.shape)}")
    a, b = heads * D, (heads + kv_heads) * D
    q = qkv[:, :a].unflatten(1, (heads, D))
    k = qkv[:, a:b].unflatten(1, (kv_heads, D))
    v = qkv[:, b:].unflatten(1, (kv_heads, D))
    qk_norm_rope(q, k, positions, axes, q_weight=q_weight, k_weight=k_weight, eps=eps, norm=norm,
                 out_q=q, out_k=k)
    return q, k, v
