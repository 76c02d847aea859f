"""torch front end of the C ABI: validates tensors, allocates outputs on the input's
device, and enqueues the sm_100a kernels on the current CUDA stream.

Every function here launches native kernels; none has a CPU path.  Scales follow
the reference's shapes: activation scales [M, 1] fp32, weight scales [N, 1] fp32.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _native as N


def launch_count() -> int:
    """Kernels enqueued so far by this process (one per native call)."""
    return N.launch_count()


def sm_clock_probe(out: torch.Tensor, ns: int, stream: torch.cuda.Stream) -> None:
    """Enqueues the SM clock probe on `stream`: a 32-thread kernel that sleeps `ns`
    nanoseconds and writes [elapsed ns, SM cycles] into `out` (int64 [2], on the GPU),
    so that cycles / ns is the SM clock while other kernels ran beside it."""
    out = _need(out, torch.int64, "out", 1)
    if out.numel() != 2:
        raise ValueError("out must hold 2 int64 values")
    N.call("h3_sm_clock_probe", int(ns), out.data_ptr(), stream.cuda_stream)


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _need(t: torch.Tensor, dtype, name: str, ndim: int | None = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name}: CUDA tensor required (the INT8 path has no CPU fallback)")
    if t.dtype != dtype:
        raise ValueError(f"{name}: {dtype} required, got {t.dtype}")
    if ndim is not None and t.ndim != ndim:
        raise ValueError(f"{name}: {ndim}-D tensor required")
    return t.contiguous()


def _vec(t: torch.Tensor, n: int, name: str) -> torch.Tensor:
    t = _need(t, torch.float32, name)
    if t.numel() != n:
        raise ValueError(f"{name}: {n} values required, got {t.numel()}")
    return t if t.ndim == 1 else t.reshape(-1)


INPUT_KINDS = {"gateup_f16": N.IN_GATEUP_F16, "act_f32": N.IN_ACT_F32, "act_f16": N.IN_ACT_F16}
DIVISIONS = {"rn": N.DIV_RN, "fast": N.DIV_FAST}


def _out(out, shape, dtype, device, name):
    """A caller-provided output buffer (contiguous, exact shape / dtype / device), or a
    fresh one."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if (out.dtype != dtype or tuple(out.shape) != tuple(shape) or not out.is_contiguous()
            or out.device != device):
        raise ValueError(f"{name}: contiguous {dtype} {tuple(shape)} buffer on {device} required")
    return out


def _producer_input(x: torch.Tensor, kind: str):
    k = INPUT_KINDS[kind]
    x = _need(x, torch.float32 if k == N.IN_ACT_F32 else torch.float16, "x", 2)
    width = x.shape[1] // 2 if k == N.IN_GATEUP_F16 else x.shape[1]
    return x, k, x.shape[0], width


# ----------------------------------------------------------------------------
# column path
# ----------------------------------------------------------------------------
def column_quantize(x: torch.Tensor, convrot: bool = True, out_q=None, out_scale=None):
    """Rotation (optional) + per-row INT8 quantisation of the column input.
    Returns (q int8 [M, K], scale fp32 [M, 1])."""
    x = _need(x, torch.float16, "x", 2)
    M, K = x.shape
    q = _out(out_q, (M, K), torch.int8, x.device, "out_q")
    s = _out(out_scale, (M, 1), torch.float32, x.device, "out_scale")
    N.call("h3_column_quantize", x.data_ptr(), M, K, int(bool(convrot)), q.data_ptr(),
           s.data_ptr(), _stream(x))
    return q, s


def modulated_norm_quantize(x, weight, eps: float, shift, scale, labels=None, convrot=True,
                            quantize=True, want_h=False):
    """Modulated RMSNorm (tilelang_dit_fusion.py:11-37) fused with the column
    activation quantiser: x fp16 [M, K] -> (codes int8 [M, K], row_scale fp32 [M, 1],
    h fp16 [M, K] or None).  quantize=False returns (None, None, h)."""
    x = _need(x, torch.float16, "x", 2)
    M, K = x.shape
    w = _vec(weight, K, "norm weight")
    shift = _need(shift, torch.float32, "shift", 2)
    scale = _need(scale, torch.float32, "scale", 2)
    if shift.shape != scale.shape or shift.shape[1] != K:
        raise ValueError("shift / scale tables must be [modulation_rows, K]")
    lab = None
    if labels is not None:
        lab = _need(labels, torch.int32, "labels", 1)
        if lab.numel() != M:
            raise ValueError("one label per row required")
    elif shift.shape[0] != 1:
        raise ValueError("labels required for a multi-row modulation table")
    q = s = h = None
    if quantize:
        q = torch.empty((M, K), dtype=torch.int8, device=x.device)
        s = torch.empty((M, 1), dtype=torch.float32, device=x.device)
    if want_h or not quantize:
        h = torch.empty((M, K), dtype=torch.float16, device=x.device)
    N.call("h3_modulated_norm_quantize", x.data_ptr(), M, K, w.data_ptr(), float(eps),
           shift.data_ptr(), scale.data_ptr(), shift.shape[0], _ptr(lab), int(bool(convrot)),
           _ptr(q), _ptr(s), _ptr(h), _stream(x))
    return q, s, h


def int8_gemm_i32(q: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """Exact INT32 q @ w.T on the tensor cores (tcgen05 kind::i8)."""
    q = _need(q, torch.int8, "q", 2)
    w = _need(w, torch.int8, "weight", 2)
    M, K = q.shape
    if w.shape[1] != K:
        raise ValueError("Input and weight inner dimensions must match")
    out = torch.empty((M, w.shape[0]), dtype=torch.int32, device=q.device)
    N.call("h3_int8_gemm_i32", q.data_ptr(), w.data_ptr(), M, w.shape[0], K, out.data_ptr(),
           _stream(q))
    return out


def int8_gemm_column(q, w, row_scale, weight_scale, bias=None) -> torch.Tensor:
    """INT8 GEMM + ordered column epilogue, fp16 [M, N]."""
    q = _need(q, torch.int8, "q", 2)
    w = _need(w, torch.int8, "weight", 2)
    M, K = q.shape
    Nn = w.shape[0]
    if w.shape[1] != K:
        raise ValueError("Input and weight inner dimensions must match")
    a = _vec(row_scale, M, "row_scale")
    ws = _need(weight_scale, torch.float32, "weight_scale").reshape(-1)
    if ws.numel() not in (1, Nn):
        raise ValueError("INT8 weight scale must be scalar or per-output-channel")
    b = None if bias is None else _vec(bias, Nn, "bias")
    out = torch.empty((M, Nn), dtype=torch.float16, device=q.device)
    N.call("h3_int8_gemm_column", q.data_ptr(), w.data_ptr(), M, Nn, K, a.data_ptr(),
           ws.data_ptr(), ws.numel(), _ptr(b), out.data_ptr(), _stream(q))
    return out


def int8_gemm_swiglu(q, w, row_scale, weight_scale, bias=None, out_dtype=torch.float32, out=None):
    """FC1 GEMM with the FP32 SwiGLU epilogue; w is [gate_r | up_r]; output
    [M, w.shape[0] // 2] in out_dtype (fp32 keeps the reference's bits)."""
    q = _need(q, torch.int8, "q", 2)
    w = _need(w, torch.int8, "weight", 2)
    M, K = q.shape
    Np = w.shape[0]
    if w.shape[1] != K or Np % 2:
        raise ValueError("SwiGLU weight must be [2*n, K] with matching K")
    a = _vec(row_scale, M, "row_scale")
    ws = _vec(weight_scale, Np, "weight_scale")
    b = None if bias is None else _vec(bias, Np, "bias")
    kind = {torch.float32: N.OUT_F32, torch.float16: N.OUT_F16}[out_dtype]
    out = _out(out, (M, Np // 2), out_dtype, q.device, "out")
    N.call("h3_int8_gemm_swiglu", q.data_ptr(), w.data_ptr(), M, Np, K, a.data_ptr(),
           ws.data_ptr(), _ptr(b), kind, out.data_ptr(), _stream(q))
    return out


def column_dequantize(acc, row_scale, weight_scale) -> torch.Tensor:
    """tilelang_column_epilogue.dequantize: f16(C * (A * W))."""
    acc = _need(acc, torch.int32, "accumulator", 2)
    M, Nn = acc.shape
    a = _vec(row_scale, M, "row_scale")
    ws = _need(weight_scale, torch.float32, "weight_scale").reshape(-1)
    if ws.numel() not in (1, Nn):
        raise ValueError("Scalar or channel scale required")
    out = torch.empty((M, Nn), dtype=torch.float16, device=acc.device)
    N.call("h3_column_dequantize", acc.data_ptr(), M, Nn, a.data_ptr(), ws.data_ptr(),
           ws.numel(), out.data_ptr(), _stream(acc))
    return out


# ----------------------------------------------------------------------------
# FC2 producer
# ----------------------------------------------------------------------------
def swiglu_rotate_max(x, kind="gateup_f16", store=True):
    """Phase 'stored' (store=True) or 'maximum'.  Returns (rotated fp32 or None,
    row_max fp32 [M, 1])."""
    x, k, M, W = _producer_input(x, kind)
    rot = torch.empty((M, W), dtype=torch.float32, device=x.device) if store else None
    m = torch.empty((M, 1), dtype=torch.float32, device=x.device)
    N.call("h3_swiglu_rotate_max", x.data_ptr(), k, M, W, _ptr(rot), m.data_ptr(), _stream(x))
    return rot, m


def swiglu_rotate_quantize(x, row_max, kind="gateup_f16", division="rn"):
    """Phase 'recompute': codes of the rotated activation under the reduced row max."""
    x, k, M, W = _producer_input(x, kind)
    m = _vec(row_max, M, "row_max")
    q = torch.empty((M, W), dtype=torch.int8, device=x.device)
    s = torch.empty((M, 1), dtype=torch.float32, device=x.device)
    N.call("h3_swiglu_rotate_quantize", x.data_ptr(), k, M, W, m.data_ptr(),
           DIVISIONS[division], q.data_ptr(), s.data_ptr(), _stream(x))
    return q, s


def swiglu_rotate_quantize_local(x, kind="gateup_f16", division="rn"):
    """TP=1 single pass.  Returns (q, scale [M, 1], row_max [M, 1])."""
    x, k, M, W = _producer_input(x, kind)
    q = torch.empty((M, W), dtype=torch.int8, device=x.device)
    s = torch.empty((M, 1), dtype=torch.float32, device=x.device)
    m = torch.empty((M, 1), dtype=torch.float32, device=x.device)
    N.call("h3_swiglu_rotate_quantize_local", x.data_ptr(), k, M, W, DIVISIONS[division],
           q.data_ptr(), s.data_ptr(), m.data_ptr(), _stream(x))
    return q, s, m


PEER_PRODUCER_MAX_WIDTH = 16384  # H3_PEER_PRODUCER_MAX_WIDTH


def swiglu_rotate_quantize_peer(x, bases, world: int, rank: int, slots_off: int, epoch: int,
                                kind="gateup_f16", division="rn", want_max=False, out_q=None,
                                out_scale=None):
    """TP>1 single pass (h3_swiglu_rotate_quantize_peer): the row maxima are exchanged
    with the other ranks over peer memory inside the kernel.  Returns (q, scale [M, 1],
    row_max [M, 1] of the global maxima or None)."""
    x, k, M, W = _producer_input(x, kind)
    q = _out(out_q, (M, W), torch.int8, x.device, "out_q")
    s = _out(out_scale, (M, 1), torch.float32, x.device, "out_scale")
    m = torch.empty((M, 1), dtype=torch.float32, device=x.device) if want_max else None
    arr = (ctypes.c_void_p * world)(*bases)
    N.call("h3_swiglu_rotate_quantize_peer", x.data_ptr(), k, M, W, arr, world, rank,
           int(slots_off), int(epoch), DIVISIONS[division], q.data_ptr(), s.data_ptr(), _ptr(m),
           _stream(x))
    return q, s, m


def row_quantize(rotated, row_max, width=None, start=0, division="rn"):
    """tilelang_row_quant.quantize: codes of rotated[:, start:start+width]."""
    rotated = _need(rotated, torch.float32, "rotated", 2)
    M, stride = rotated.shape
    width = stride - start if width is None else int(width)
    m = _vec(row_max, M, "row_max")
    q = torch.empty((M, width), dtype=torch.int8, device=rotated.device)
    s = torch.empty((M, 1), dtype=torch.float32, device=rotated.device)
    N.call("h3_row_quantize", rotated.data_ptr(), M, width, stride, int(start), m.data_ptr(),
           DIVISIONS[division], q.data_ptr(), s.data_ptr(), _stream(rotated))
    return q, s


# ----------------------------------------------------------------------------
# row path
# ----------------------------------------------------------------------------
def transport_shift(full_k: int) -> int:
    return int(N.load().h3_transport_shift(int(full_k)))


def int8_gemm_row_encode(q, w, shift: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """INT8 GEMM + scaled-FP16 encode: f16(acc * 2^-shift), [M, N].  `out` (contiguous
    fp16 [M, N], e.g. a peer-mapped transport buffer) receives the payload if given."""
    q = _need(q, torch.int8, "q", 2)
    w = _need(w, torch.int8, "weight", 2)
    M, K = q.shape
    if w.shape[1] != K:
        raise ValueError("Input and weight inner dimensions must match")
    if out is None:
        out = torch.empty((M, w.shape[0]), dtype=torch.float16, device=q.device)
    elif (out.dtype != torch.float16 or tuple(out.shape) != (M, w.shape[0])
          or not out.is_contiguous() or out.device != q.device):
        raise ValueError("out must be a contiguous fp16 [M, N] tensor on the input's device")
    N.call("h3_int8_gemm_row_encode", q.data_ptr(), w.data_ptr(), M, w.shape[0], K, int(shift),
           out.data_ptr(), _stream(q))
    return out


def int8_gemm_row_encode_push(q, w, shift: int, bases, world: int, rank: int,
                              partial_off: int) -> None:
    """INT8 GEMM + scaled-FP16 encode with every output row stored into the peer-mapped
    buffer of the rank that owns it (h3_int8_gemm_row_encode_push): the reduce-scatter
    of the partials fused into the GEMM epilogue."""
    q = _need(q, torch.int8, "q", 2)
    w = _need(w, torch.int8, "weight", 2)
    M, K = q.shape
    if w.shape[1] != K:
        raise ValueError("Input and weight inner dimensions must match")
    arr = (ctypes.c_void_p * world)(*bases)
    N.call("h3_int8_gemm_row_encode_push", q.data_ptr(), w.data_ptr(), M, w.shape[0], K,
           int(shift), arr, world, rank, int(partial_off), _stream(q))


def _gate_args(residual, gate, labels, M, Nn):
    if residual is None:
        return None, None, 0, None
    residual = _need(residual, torch.float16, "residual", 2)
    if residual.shape != (M, Nn):
        raise ValueError("residual shape mismatch")
    if gate is None:
        return residual, None, 0, None
    gate = _need(gate, torch.float32, "gate", 2)
    if gate.shape[1] != Nn:
        raise ValueError("gate table width mismatch")
    lab = None
    if labels is not None:
        lab = _need(labels, torch.int32, "labels", 1)
        if lab.numel() != M:
            raise ValueError("one label per row required")
    elif gate.shape[0] != 1:
        raise ValueError("labels required for a multi-row gate table")
    return residual, gate, gate.shape[0], lab


def int8_gemm_row_dequant(q, w, row_scale, weight_scale, out_dtype=torch.float32,
                          residual=None, gate=None, labels=None):
    """TP=1 row GEMM, exact INT32 + fused dequant.  With `residual` the gated residual
    is updated in place and returned; otherwise a new [M, N] tensor in out_dtype."""
    q = _need(q, torch.int8, "q", 2)
    w = _need(w, torch.int8, "weight", 2)
    M, K = q.shape
    Nn = w.shape[0]
    if w.shape[1] != K:
        raise ValueError("Input and weight inner dimensions must match")
    a = _vec(row_scale, M, "row_scale")
    ws = _vec(weight_scale, Nn, "weight_scale")
    if residual is not None:
        if not residual.is_contiguous():
            raise ValueError("residual must be contiguous (updated in place)")
        res, g, grows, lab = _gate_args(residual, gate, labels, M, Nn)
        N.call("h3_int8_gemm_row_dequant", q.data_ptr(), w.data_ptr(), M, Nn, K, a.data_ptr(),
               ws.data_ptr(), N.OUT_RESIDUAL, None, res.data_ptr(), _ptr(g), grows, _ptr(lab),
               _stream(q))
        return residual
    kind = {torch.float32: N.OUT_F32, torch.float16: N.OUT_F16}[out_dtype]
    out = torch.empty((M, Nn), dtype=out_dtype, device=q.device)
    N.call("h3_int8_gemm_row_dequant", q.data_ptr(), w.data_ptr(), M, Nn, K, a.data_ptr(),
           ws.data_ptr(), kind, out.data_ptr(), None, None, 0, None, _stream(q))
    return out


def fp16_encode(partial: torch.Tensor, shift: int) -> torch.Tensor:
    p = _need(partial, torch.int32, "partial")
    out = torch.empty(p.shape, dtype=torch.float16, device=p.device)
    N.call("h3_fp16_encode", p.data_ptr(), p.numel(), int(shift), out.data_ptr(), _stream(p))
    return out


def fp16_decode(payload: torch.Tensor, shift: int) -> torch.Tensor:
    y = _need(payload, torch.float16, "payload")
    out = torch.empty(y.shape, dtype=torch.int32, device=y.device)
    N.call("h3_fp16_decode", y.data_ptr(), y.numel(), int(shift), out.data_ptr(), _stream(y))
    return out


def row_reduce_finish(parts, shift, row_scale, weight_scale, out_dtype=torch.float32,
                      residual=None, gate=None, labels=None):
    """parts: fp16 [world, rows, N] (or [rows, N] for an already reduced payload).
    Fixed-order fp32 sum + one fp16 rounding, decode, dequant, then store or gated
    residual update (residual updated in place and returned)."""
    parts = _need(parts, torch.float16, "parts")
    if parts.ndim == 2:
        parts = parts.unsqueeze(0)
    world, M, Nn = parts.shape
    a = _vec(row_scale, M, "row_scale")
    ws = _vec(weight_scale, Nn, "weight_scale")
    if residual is not None:
        if not residual.is_contiguous():
            raise ValueError("residual must be contiguous (updated in place)")
        res, g, grows, lab = _gate_args(residual, gate, labels, M, Nn)
        N.call("h3_row_reduce_finish", parts.data_ptr(), world, M * Nn, M, Nn, int(shift),
               a.data_ptr(), ws.data_ptr(), N.OUT_RESIDUAL, None, res.data_ptr(), _ptr(g),
               grows, _ptr(lab), _stream(parts))
        return residual
    kind = {torch.float32: N.OUT_F32, torch.float16: N.OUT_F16}[out_dtype]
    out = torch.empty((M, Nn), dtype=out_dtype, device=parts.device)
    N.call("h3_row_reduce_finish", parts.data_ptr(), world, M * Nn, M, Nn, int(shift),
           a.data_ptr(), ws.data_ptr(), kind, out.data_ptr(), None, None, 0, None,
           _stream(parts))
    return out


# ----------------------------------------------------------------------------
# packed INT8 transport ('int8_gather')
# ----------------------------------------------------------------------------
def pack8_pitch(width: int) -> int:
    """Bytes per row of a packed payload: 128 codes + 4 scale bytes per 128 columns."""
    if width % 128:
        raise ValueError("Whole group128 outputs required")
    return width // 128 * 132


def int8_gemm_row_pack8(q, w, out: torch.Tensor | None = None) -> torch.Tensor:
    """INT8 GEMM with the group-128 INT8 pack fused: uint8 [M, N/128*132]."""
    q = _need(q, torch.int8, "q", 2)
    w = _need(w, torch.int8, "weight", 2)
    M, K = q.shape
    if w.shape[1] != K:
        raise ValueError("Input and weight inner dimensions must match")
    pitch = pack8_pitch(w.shape[0])
    if out is None:
        out = torch.empty((M, pitch), dtype=torch.uint8, device=q.device)
    elif (out.dtype != torch.uint8 or tuple(out.shape) != (M, pitch) or not out.is_contiguous()
          or out.device != q.device):
        raise ValueError("out must be a contiguous uint8 [M, N/128*132] tensor on q's device")
    N.call("h3_int8_gemm_row_pack8", q.data_ptr(), w.data_ptr(), M, w.shape[0], K,
           out.data_ptr(), _stream(q))
    return out


def pack8(partial) -> torch.Tensor:
    """Group-128 INT8 pack of an INT32 partial (pack_int8): uint8 [rows, width/128*132]."""
    p = _need(partial, torch.int32, "partial", 2)
    rows, width = p.shape
    out = torch.empty((rows, pack8_pitch(width)), dtype=torch.uint8, device=p.device)
    N.call("h3_pack8", p.data_ptr(), rows, width, out.data_ptr(), _stream(p))
    return out


def unpack8_finish(parts, width: int, row_scale=None, weight_scale=None, out_dtype=torch.float32,
                   residual=None, gate=None, labels=None):
    """parts: uint8 [world, rows, pitch] (or [rows, pitch]).  Rank-order reconstruction,
    then the row epilogue; out_dtype torch.int32 returns the restored sums."""
    parts = _need(parts, torch.uint8, "parts")
    if parts.ndim == 2:
        parts = parts.unsqueeze(0)
    world, M, pitch = parts.shape
    if pitch != pack8_pitch(width):
        raise ValueError("payload pitch does not match the width")
    if out_dtype == torch.int32 and residual is None:
        out = torch.empty((M, width), dtype=torch.int32, device=parts.device)
        N.call("h3_unpack8_finish", parts.data_ptr(), world, M * pitch, M, width, None, None,
               N.OUT_I32, out.data_ptr(), None, None, 0, None, _stream(parts))
        return out
    a = _vec(row_scale, M, "row_scale")
    ws = _vec(weight_scale, width, "weight_scale")
    if residual is not None:
        if not residual.is_contiguous():
            raise ValueError("residual must be contiguous (updated in place)")
        res, g, grows, lab = _gate_args(residual, gate, labels, M, width)
        N.call("h3_unpack8_finish", parts.data_ptr(), world, M * pitch, M, width, a.data_ptr(),
               ws.data_ptr(), N.OUT_RESIDUAL, None, res.data_ptr(), _ptr(g), grows, _ptr(lab),
               _stream(parts))
        return residual
    kind = {torch.float32: N.OUT_F32, torch.float16: N.OUT_F16}[out_dtype]
    out = torch.empty((M, width), dtype=out_dtype, device=parts.device)
    N.call("h3_unpack8_finish", parts.data_ptr(), world, M * pitch, M, width, a.data_ptr(),
           ws.data_ptr(), kind, out.data_ptr(), None, None, 0, None, _stream(parts))
    return out


def dequantize_i32(acc, row_scale, weight_scale, out_dtype=torch.float32, bias=None):
    """parallel_int8.dequantize order: ((acc * a) * w) + bias."""
    acc = _need(acc, torch.int32, "accumulator", 2)
    M, Nn = acc.shape
    a = _vec(row_scale, M, "activation_scale")
    ws = _need(weight_scale, torch.float32, "weight_scale").reshape(-1)
    if ws.numel() not in (1, Nn):
        raise ValueError("INT8 weight scale must be scalar or per-output-channel")
    b = None if bias is None else _vec(bias, Nn, "bias")
    kind = {torch.float32: N.OUT_F32, torch.float16: N.OUT_F16}[out_dtype]
    out = torch.empty((M, Nn), dtype=out_dtype, device=acc.device)
    N.call("h3_dequantize_i32", acc.data_ptr(), M, Nn, a.data_ptr(), ws.data_ptr(), ws.numel(),
           _ptr(b), kind, out.data_ptr(), _stream(acc))
    return out


def gated_add(residual, branch, gate=None, labels=None):
    """X = f16(fma(f16(branch), G[label], X)) in place (gate_kernel,
    tilelang_dit_fusion.py:39-53); branch fp32 or fp16 [M, N]; returns residual."""
    if not residual.is_contiguous():
        raise ValueError("residual must be contiguous (updated in place)")
    if branch.dtype not in (torch.float32, torch.float16):
        raise ValueError("branch must be fp32 or fp16")
    b = _need(branch, branch.dtype, "branch", 2)
    M, Nn = b.shape
    res, g, grows, lab = _gate_args(residual, gate, labels, M, Nn)
    kind = N.OUT_F32 if b.dtype == torch.float32 else N.OUT_F16
    N.call("h3_gated_add", b.data_ptr(), kind, M, Nn, res.data_ptr(), _ptr(g), grows, _ptr(lab),
           _stream(b))
    return residual


# ----------------------------------------------------------------------------
# operators of a block around its projections
# ----------------------------------------------------------------------------
_TYPES = {torch.float32: N.TYPE_F32, torch.float16: N.TYPE_F16, torch.bfloat16: N.TYPE_BF16}
_NORM_KINDS = {"rms": N.NORM_RMS, "layer": N.NORM_LAYER}
_POSITIONS = {torch.int32: N.POS_I32, torch.int64: N.POS_I64, torch.float32: N.POS_F32}


def _raw_stream(device: torch.device) -> int:
    """The handle of the device's current stream (without a Stream object: a call on one row
    or token is bound by its host side)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _inference(where: str, device, tensors, names) -> None:
    """Everything given is a tensor on `device`, none that autograd would have to follow."""
    grad = torch.is_grad_enabled()
    for t, name in zip(tensors, names):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name}: tensor required")
        if t.device != device:
            raise ValueError(f"{name}: on {t.device}, the call runs on {device}")
        if grad and t.requires_grad:
            raise ValueError(f"{where} has no backward ({name} requires a gradient): call it under "
                             "torch.no_grad()")


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The addresses [first, last) that a strided tensor's elements lie in."""
    if t.numel() == 0:
        return 0, 0
    if t.is_contiguous():
        last = t.numel()
    else:
        last = sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1
    return t.data_ptr(), t.data_ptr() + last * t.element_size()


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a1 <= b0 or b1 <= a0


_NORM_TENSORS = ("x", "branch", "gate", "labels", "shift", "scale", "out")
_POST_TENSORS, _PRE_TENSORS = ("post weight", "post bias"), ("pre weight", "pre bias")
_ROPE_TENSORS = ("q", "k", "positions", "q_weight", "k_weight", "out_q", "out_k")
_INT4_TENSORS = ("x", "weight", "scales", "zeros", "bias")


class NormSpec(NamedTuple):
    """A norm over the last dimension: kind 'rms' (v * rsqrt(mean(v^2) + eps)) or 'layer'
    ((v - mean) * rsqrt(var + eps)), times `weight`, plus `bias` (fp32 [width] or None)."""
    kind: str = "rms"
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    eps: float = 1e-6


def _norm_args(spec: Optional[NormSpec], width: int, name: str):
    if spec is None:
        return N.NORM_NONE, None, None, 0.0
    if spec.kind not in _NORM_KINDS:
        raise ValueError(f"{name}: norm kind must be 'rms' or 'layer'")
    if not spec.eps >= 0.0:
        raise ValueError(f"{name}: eps must not be negative")
    w = None if spec.weight is None else _vec(spec.weight, width, f"{name} weight")
    b = None if spec.bias is None else _vec(spec.bias, width, f"{name} bias")
    return _NORM_KINDS[spec.kind], w, b, float(spec.eps)


def _table(t, rows, width: int, name: str):
    """A modulation table [rows, width] with unit stride inside a row (a slice of a wider
    table is read in place)."""
    if t is None:
        return None, 0
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float32 or t.ndim != 2:
        raise ValueError(f"{name}: fp32 CUDA table [rows, {width}] required")
    if t.shape[1] != width or t.shape[0] != rows:
        raise ValueError(f"{name}: table [{rows}, {width}] required, got {tuple(t.shape)}")
    if t.stride(1) != 1 and width > 1:
        t = t.contiguous()
    return t, t.stride(0)


def residual_norm(x, branch=None, gate=None, labels=None, *, post: Optional[NormSpec] = None,
                  pre: Optional[NormSpec] = None, shift=None, scale=None,
                  residual_scale: float = 1.0, out=None, quantize=False, convrot=True):
    """Residual update joined with the norms before and after it, one pass over each row:

        b  = post(branch)                                       (post None: the branch itself)
        x' = residual_scale * x + gate[label] * b
        h  = pre(x') * (1 + scale[label]) + shift[label]        (pre None: not computed)

    x [M, N] (N <= 32768) is fp32, fp16 or bf16; branch has x's type or fp32.  x' is
    written over x unless `out` (another [M, N] of x's type) is given, rounded once;
    without a branch x is left as it is and only `pre` runs.  h comes in x's type or,
    with quantize, as the INT8 codes and row scales that
    ColumnParallelLinearINT8.forward_quantized takes (convrot: of the row rotated by
    ConvRot256, N % 256 == 0).  Statistics, x' and h stay in fp32 until those roundings.

    gate, shift, scale: fp32 tables [R, N], all of the same R (slices of one wider table
    are read in place); labels: int32 [M], needed unless R is 1.  A label out of range
    reads row 0 and sets the device error word.  x' must not lie over a table, a norm's
    weight or the labels: every row reads those (refused).

    Returns (x', h or codes or None, row_scale [M, 1] or None)."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.ndim != 2 or x.dtype not in _TYPES:
        raise ValueError("x: 2-D CUDA tensor of fp32, fp16 or bf16 required")
    if not x.is_contiguous():
        raise ValueError("x must be contiguous (updated in place)")
    M, width = x.shape
    if not 1 <= width <= 32768:
        raise ValueError("x: a width of 1 to 32768 is required")
    dev = x.device
    if pre is None and (quantize or shift is not None or scale is not None):
        raise ValueError("shift, scale and quantize belong to the pre-norm: give pre")
    if quantize and convrot and width % 256:
        raise ValueError("ConvRot256 needs a width that is a multiple of 256")
    _inference("residual_norm", dev, (x, branch, gate, labels, shift, scale, out), _NORM_TENSORS)
    if branch is None:
        if pre is None or post is not None or gate is not None or out is not None \
                or residual_scale != 1.0:
            raise ValueError("without a branch only the pre-norm of x applies")
        xo = None
    else:
        if branch.dtype not in (x.dtype, torch.float32) or branch.shape != x.shape:
            raise ValueError(f"branch: {tuple(x.shape)} of {x.dtype} or fp32 required")
        branch = branch.contiguous()
        xo = x if out is None else _out(out, x.shape, x.dtype, dev, "out")
        # all three are contiguous: their addresses and sizes say whether they overlap
        at, size = xo.data_ptr(), x.nbytes
        b_at = branch.data_ptr()
        if at < b_at + branch.nbytes and b_at < at + size or xo is not x and 0 < abs(at - x.data_ptr()) < size:
            raise ValueError("out must be x itself or overlap neither x nor the branch")
    rows = next((t.shape[0] for t in (gate, shift, scale)
                 if isinstance(t, torch.Tensor) and t.ndim == 2), 1)
    g, g_ld = _table(gate, rows, width, "gate")
    sh, sh_ld = _table(shift, rows, width, "shift")
    sc, sc_ld = _table(scale, rows, width, "scale")
    if rows < 1:
        raise ValueError("the modulation tables must have a row")
    lab = None
    if rows > 1 or labels is not None:
        if labels is None:
            raise ValueError("labels required for a multi-row modulation table")
        lab = _need(labels, torch.int32, "labels", 1)
        if lab.numel() != M:
            raise ValueError("one label per row required")
    for spec, names in ((post, _POST_TENSORS), (pre, _PRE_TENSORS)):
        if spec is not None:
            if not isinstance(spec, NormSpec):
                raise ValueError("post and pre: NormSpec or None required")
            _inference("residual_norm", dev, (spec.weight, spec.bias), names)
    pk, pw, pb, pe = _norm_args(post, width, "post")
    nk, nw, nb, ne = _norm_args(pre, width, "pre")
    h = q = s = None
    if quantize:
        q = torch.empty((M, width), dtype=torch.int8, device=dev)
        s = torch.empty((M, 1), dtype=torch.float32, device=dev)
    elif pre is not None:
        h = torch.empty_like(x)
    if M == 0:
        return x if xo is None else xo, q if quantize else h, s
    kind = _TYPES[x.dtype]
    N.call("h3_residual_norm", x.data_ptr(), kind, _ptr(branch),
           kind if branch is None else _TYPES[branch.dtype], M, width, float(residual_scale),
           _ptr(g), g_ld, _ptr(sh), sh_ld, _ptr(sc), sc_ld, rows, _ptr(lab), pk, _ptr(pw), _ptr(pb),
           pe, nk, _ptr(nw), _ptr(nb), ne, _ptr(xo), _ptr(h), int(bool(convrot)), _ptr(q), _ptr(s),
           _raw_stream(dev))
    return x if xo is None else xo, q if quantize else h, s


def _heads(t, name: str, like=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.ndim != 3 or t.dtype not in _TYPES:
        raise ValueError(f"{name}: CUDA tensor [tokens, heads, head_dim] of fp32, fp16 or bf16 required")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}: unit stride inside a head required")
    if like is not None and (t.dtype != like.dtype or t.shape[0] != like.shape[0]
                             or t.shape[2] != like.shape[2]):
        raise ValueError(f"{name}: the token count, head_dim and type of q required")
    return t


def _head_windows_apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [tokens, heads, dim] views share no element: their spans are apart, or
    (views of one packed row) their heads lie in disjoint windows of one token stride."""
    if _apart(a, b):
        return True
    period = a.stride(0)
    if period != b.stride(0) or a.shape[0] < 2 and b.shape[0] < 2:
        return False
    wide = [(t.shape[1] - 1) * t.stride(1) + t.shape[2] for t in (a, b)]
    diff = b.data_ptr() - a.data_ptr()
    if diff % a.element_size() or min(a.stride(1), b.stride(1)) < 0:
        return False
    diff = diff // a.element_size() % period
    return max(wide) <= period and wide[0] <= diff and diff + wide[1] <= period


def _head_out(out, like, name: str):
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    _heads(out, name, like)
    if out.shape != like.shape:
        raise ValueError(f"{name}: {tuple(like.shape)} required")
    # distinct elements at distinct addresses: token-major or head-major
    (s, h, d), (ts, hs, _) = out.shape, out.stride()
    if out.numel() and not ((h == 1 or hs >= d) and (s == 1 or ts >= (h - 1) * hs + d)
                            or (s == 1 or ts >= d) and (h == 1 or hs >= (s - 1) * ts + d)):
        raise ValueError(f"{name}: overlapping strides")
    return out


def qk_norm_rope(q, k, positions, plan, *, q_weight=None, k_weight=None, eps: float = 1e-6,
                 norm: bool = True, out_q=None, out_k=None):
    """Per-head RMS norm and rotary positions of q [S, Hq, D] and k [S, Hk, D] (or None);
    h3tp.rms_rope documents the arguments.  Returns (q', k')."""
    _heads(q, "q")
    dev, (S, hq, D) = q.device, q.shape
    if not hasattr(plan, "head_dim"):
        raise ValueError("plan: RotaryAxes required")
    if D != plan.head_dim:
        raise ValueError(f"q: head_dim {plan.head_dim} of the plan required, got {D}")
    if k is not None:
        _heads(k, "k", q)
    if hq < 1 or (k is not None and k.shape[1] < 1):
        raise ValueError("at least one head required")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in _POSITIONS:
        raise ValueError("positions: int32, int64 or fp32 tensor required")
    if positions.ndim == 1 and plan.n_axes == 1:
        positions = positions.unsqueeze(1)
    if tuple(positions.shape) != (S, plan.n_axes):
        raise ValueError(f"positions: [{S}, {plan.n_axes}] required, got {tuple(positions.shape)}")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if not norm and (q_weight is not None or k_weight is not None):
        q_weight = k_weight = None
    _inference("qk_norm_rope", dev, (q, k, positions, q_weight, k_weight, out_q, out_k), _ROPE_TENSORS)
    positions = positions.contiguous()
    wq = None if q_weight is None else _vec(q_weight, D, "q_weight")
    wk = None if k_weight is None or k is None else _vec(k_weight, D, "k_weight")
    if out_q is not None or out_k is not None:
        _check_head_outs(q, k, out_q, out_k)
    oq = _head_out(out_q, q, "out_q")
    ok = None if k is None else _head_out(out_k, k, "out_k")
    if S == 0:
        return oq, ok
    (qt, qh, _), (qot, qoh, _) = q.stride(), oq.stride()
    (kt, kh, _), (kot, koh, _) = ((0, 0, 0),) * 2 if k is None else (k.stride(), ok.stride())
    N.call("h3_qk_norm_rope", q.data_ptr(), qt, qh, hq, oq.data_ptr(), qot, qoh, _ptr(k), kt, kh,
           0 if k is None else k.shape[1], _ptr(ok), kot, koh, S, D,
           _TYPES[q.dtype], positions.data_ptr(), _POSITIONS[positions.dtype], plan.n_axes,
           plan.turns, plan.axis, plan.pairs, plan.half, int(bool(norm)), _ptr(wq), _ptr(wk),
           float(eps), _raw_stream(dev))
    return oq, ok


def _check_head_outs(q, k, out_q, out_k) -> None:
    """Outputs that are given must be their own input, or share no element with an input
    or with each other."""
    if out_k is not None and k is None:
        raise ValueError("out_k without k")
    for out, own, other, name in ((out_q, q, k, "out_q"), (out_k, k, q, "out_k")):
        if out is None:
            continue
        _head_out(out, own, name)
        same = out.data_ptr() == own.data_ptr() and all(
            n == 1 or a == b for n, a, b in zip(own.shape, out.stride(), own.stride()))
        if not same and not _head_windows_apart(out, own):
            raise ValueError(f"{name} must be its input or not overlap it")
        if other is not None and not _head_windows_apart(out, other):
            raise ValueError(f"{name} overlaps the other input")
    if out_q is not None and out_k is not None and not _head_windows_apart(out_q, out_k):
        raise ValueError("out_q and out_k overlap")


INT4_GROUPS = (32, 64, 128)


def int4_linear(x, weight, scales, zeros=None, *, group: int = 128, bias=None, out_dtype=None):
    """y = x @ W.T + bias with W[n, k] = scales[n, k // group] * (code[n, k] - zero), codes of
    4 bits; x fp16 or bf16 [M, K], y [M, N] in x's type or fp32 (out_dtype).

    weight: contiguous uint8 [N, ceil(K / 2)], code k in the low nibble of byte k // 2 for
    even k and in the high one for odd k; scales: fp32, fp16 or bf16 [N, ceil(K / group)];
    zeros: uint8 of the same shape, None for 8 everywhere; bias: fp32 [N].  Zero points must
    lie between 0 and 15: the call does not read them on the host and larger ones give wrong
    products (ColumnParallelLinearINT4's loader refuses them).
    Meant for few rows (a token or a handful): the weight is read and unpacked once for every 16
    rows, or for every 32 where their x fits an SM's shared memory (K up to about 1200 for 32
    rows, 2900 for 17)."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.ndim != 2 \
            or x.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("x: 2-D CUDA tensor of fp16 or bf16 required")
    M, K = x.shape
    if group not in INT4_GROUPS:
        raise ValueError(f"group must be one of {INT4_GROUPS}")
    _inference("int4_linear", x.device, (x, weight, scales, zeros, bias), _INT4_TENSORS)
    if weight is None or weight.dtype != torch.uint8 or weight.ndim != 2 or not weight.is_contiguous() or K < 1 \
            or weight.shape[0] < 1 or weight.shape[1] != (K + 1) // 2:
        raise ValueError(f"weight: contiguous uint8 [N, {(K + 1) // 2}] required")
    n = weight.shape[0]
    shape = (n, -(-K // group))
    if scales is None or scales.dtype not in _TYPES or tuple(scales.shape) != shape:
        raise ValueError(f"scales: {shape} of fp32, fp16 or bf16 required")
    if zeros is not None and (zeros.dtype != torch.uint8 or tuple(zeros.shape) != shape):
        raise ValueError(f"zeros: uint8 {shape} required")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in (x.dtype, torch.float32):
        raise ValueError("out_dtype must be x's type or fp32")
    if K > 1 and x.stride(1) != 1 or x.stride(0) < K:
        x = x.contiguous()
    scales = scales.contiguous()
    zeros = None if zeros is None else zeros.contiguous()
    b = None if bias is None else _vec(bias, n, "bias")
    out = torch.empty((M, n), dtype=out_dtype, device=x.device)
    if M == 0:
        return out
    N.call("h3_int4_linear", x.data_ptr(), _TYPES[x.dtype], x.stride(0) if M > 1 else K, M, K,
           weight.data_ptr(), n, scales.data_ptr(), _TYPES[scales.dtype], _ptr(zeros), group,
           _ptr(b), out.data_ptr(), _TYPES[out_dtype], _raw_stream(x.device))
    return out


def peer_reduce(bases, world: int, rank: int, flags_off: int, partial_off: int, final_off: int,
                rows: int, width: int, shift: int, row_scale, weight_scale, residual,
                gate=None, labels=None, epoch: int = 1, multicast: int = 0, pushed: bool = False):
    """Reduce + fused gated-residual epilogue of this rank's row block from every rank's
    partial, finished rows stored into the peers' final areas (h3_peer_reduce).  With a
    non-zero `multicast` address of the same buffers the sum is taken in the NVSwitch
    and the finished rows are broadcast through it (h3_peer_reduce_nvls).  pushed: the
    partials were owner-routed by int8_gemm_row_encode_push (h3_peer_reduce_pushed)."""
    a = _vec(row_scale, rows, "row_scale")
    ws = _vec(weight_scale, width, "weight_scale")
    if not residual.is_contiguous():
        raise ValueError("residual must be contiguous (updated in place)")
    res, g, grows, lab = _gate_args(residual, gate, labels, rows, width)
    arr = (ctypes.c_void_p * world)(*bases)
    if multicast:
        N.call("h3_peer_reduce_nvls", arr, int(multicast), world, rank, flags_off, partial_off,
               final_off, rows, width, int(shift), a.data_ptr(), ws.data_ptr(), res.data_ptr(),
               _ptr(g), grows, _ptr(lab), int(epoch), _stream(res))
        return residual
    N.call("h3_peer_reduce_pushed" if pushed else "h3_peer_reduce", arr, world, rank, flags_off,
           partial_off, final_off, rows, width, int(shift), a.data_ptr(), ws.data_ptr(),
           res.data_ptr(), _ptr(g), grows, _ptr(lab), int(epoch), _stream(res))
    return residual


def peer_signal(bases, world: int, rank: int, flags_off: int, which: int, epoch: int,
                publish: bool, like: torch.Tensor) -> None:
    """h3_peer_signal on the stream of `like`'s device: optionally publish flag `which`
    (0 ready, 1 done) of this rank to every rank, then wait (bounded) for every peer's."""
    arr = (ctypes.c_void_p * world)(*bases)
    N.call("h3_peer_signal", arr, world, rank, int(flags_off), int(which), int(epoch),
           1 if publish else 0, _stream(like))


def peer_reduce_staged(bases, world: int, rank: int, flags_off: int, stage_off: int,
                       own_off: int, final_off: int, rows: int, width: int, shift: int,
                       row_scale, weight_scale, residual, gate=None, labels=None,
                       epoch: int = 1):
    """The reduce of the copy-engine exchange (h3_peer_reduce_staged): the peers' rows of
    this rank's block from the staging slots, its own rows at own_off, the finished rows
    into this rank's own final area."""
    a = _vec(row_scale, rows, "row_scale")
    ws = _vec(weight_scale, width, "weight_scale")
    if not residual.is_contiguous():
        raise ValueError("residual must be contiguous (updated in place)")
    res, g, grows, lab = _gate_args(residual, gate, labels, rows, width)
    arr = (ctypes.c_void_p * world)(*bases)
    N.call("h3_peer_reduce_staged", arr, world, rank, int(flags_off), int(stage_off),
           int(own_off), int(final_off), rows, width, int(shift), a.data_ptr(), ws.data_ptr(),
           res.data_ptr(), _ptr(g), grows, _ptr(lab), int(epoch), _stream(res))
    return residual


def copy_async(dst: int, src: int, nbytes: int, like: torch.Tensor) -> None:
    """cudaMemcpyAsync of nbytes between device addresses (either may be a peer's mapped
    buffer) on the stream of `like`'s device."""
    N.call("h3_copy_async", int(dst), int(src), int(nbytes), _stream(like))


def peer_reduce_int8(bases, world: int, rank: int, flags_off: int, partial_off: int,
                     final_off: int, rows: int, width: int, row_scale, weight_scale, residual,
                     gate=None, labels=None, epoch: int = 1):
    """peer_reduce for packed INT8 payloads (h3_peer_reduce_int8)."""
    a = _vec(row_scale, rows, "row_scale")
    ws = _vec(weight_scale, width, "weight_scale")
    if not residual.is_contiguous():
        raise ValueError("residual must be contiguous (updated in place)")
    res, g, grows, lab = _gate_args(residual, gate, labels, rows, width)
    arr = (ctypes.c_void_p * world)(*bases)
    N.call("h3_peer_reduce_int8", arr, world, rank, flags_off, partial_off, final_off, rows, width,
           a.data_ptr(), ws.data_ptr(), res.data_ptr(), _ptr(g), grows, _ptr(lab), int(epoch),
           _stream(res))
    return residual


def peer_gather(bases, world: int, rank: int, flags_off: int, final_off: int, rows: int,
                width: int, residual, epoch: int = 1):
    """Copies the peers' finished row blocks into `residual` (h3_peer_gather)."""
    res = _need(residual, torch.float16, "residual", 2)
    if res.data_ptr() != residual.data_ptr() or tuple(res.shape) != (rows, width):
        raise ValueError("residual must be a contiguous fp16 [rows, width] tensor")
    arr = (ctypes.c_void_p * world)(*bases)
    N.call("h3_peer_gather", arr, world, rank, flags_off, final_off, rows, width, res.data_ptr(),
           int(epoch), _stream(res))
    return residual


def expf_compare(x: torch.Tensor):
    """(h3_expf(x), CUDA expf(x)) evaluated on the device."""
    x = _need(x, torch.float32, "x")
    ours = torch.empty_like(x)
    ref = torch.empty_like(x)
    N.call("h3_expf_compare", x.data_ptr(), x.numel(), ours.data_ptr(), ref.data_ptr(), _stream(x))
    return ours, ref


def silu_compare(g: torch.Tensor):
    """(fast, ieee, cuda_expf) evaluations of g / (1 + exp(-g)) on the device."""
    g = _need(g, torch.float32, "g")
    fast = torch.empty_like(g)
    ieee = torch.empty_like(g)
    cuda = torch.empty_like(g)
    N.call("h3_silu_compare", g.data_ptr(), g.numel(), fast.data_ptr(), ieee.data_ptr(),
           cuda.data_ptr(), _stream(g))
    return fast, ieee, cuda


def quant_compare(x: torch.Tensor, scale: torch.Tensor):
    """(kernel codes, IEEE-division codes) of x / scale, elementwise."""
    x = _need(x, torch.float32, "x")
    scale = _need(scale, torch.float32, "scale")
    if scale.numel() != x.numel():
        raise ValueError("one scale per value")
    fast = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    ieee = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    N.call("h3_quant_compare", x.data_ptr(), scale.data_ptr(), x.numel(), fast.data_ptr(),
           ieee.data_ptr(), _stream(x))
    return fast, ieee
