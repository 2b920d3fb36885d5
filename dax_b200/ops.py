"""Tensor-level wrappers over the C ABI: one function per kernel family.

These take CUDA ``torch.Tensor`` arguments, validate device/dtype/contiguity, allocate outputs with
torch (the library itself never allocates) and enqueue on the current CUDA stream.
"""
from __future__ import annotations

import functools
import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import I64x3, check, load

_DT = {torch.bfloat16: _lib.DAX_BF16, torch.float16: _lib.DAX_F16, torch.float32: _lib.DAX_F32,
       torch.int8: _lib.DAX_I8, torch.float8_e4m3fn: _lib.DAX_E4M3, torch.float8_e5m2: _lib.DAX_E5M2}

# "bf16" (alias "f16", the default): bf16 contractions; the mode that meets rel-L2 <= 1e-2 against fp32 SDPA;
# "sage": INT8 Q.K^T + FP8 P.V (the arithmetic of the reference's SAGE_ATTN backend; about 3.7e-2 on Gaussian data);
# "int8_bf16": INT8 Q.K^T + bf16 P.V (V unquantised; about 1e-2)
ATTN_MODES = {"sage": _lib.DAX_ATTN_QK_I8_PV_F8, "int8_fp8": _lib.DAX_ATTN_QK_I8_PV_F8,
              "bf16": _lib.DAX_ATTN_QK_BF16_PV_BF16, "f16": _lib.DAX_ATTN_QK_BF16_PV_BF16,
              "int8_bf16": _lib.DAX_ATTN_QK_I8_PV_BF16}


class _Trace:
    """Optional launch accounting: number of library kernels launched and, when timing is on, CUDA
    events around each wrapper on the stream it launches on (used by the benchmark's roofline leg)."""

    KERNELS_PER_CALL = {"layernorm_modulate_quant": 1, "linear_dynamic": 2, "quant_rowwise": 1, "gemm_dequant": 1, "rmsnorm_rope_pack": 1, "attn_prepare": 5, "attn_forward": 1}

    def __init__(self):
        self.launches = 0
        self.timing = False
        self.events = []

    def reset(self, timing: bool = False):
        self.launches, self.timing, self.events = 0, timing, []

    def begin(self, name, kernels=None):
        """``kernels``: how many this call launches, where that goes by its arguments."""
        self.launches += self.KERNELS_PER_CALL[name] if kernels is None else kernels
        if not self.timing:
            return None
        e0 = torch.cuda.Event(enable_timing=True)
        e0.record(torch.cuda.current_stream())
        return (name, e0)

    def end(self, tok, meta=None):
        if tok is None:
            return
        e1 = torch.cuda.Event(enable_timing=True)
        e1.record(torch.cuda.current_stream())
        self.events.append((tok[0], tok[1], e1, meta))

    def summary(self):
        """name -> (calls, total milliseconds, list of meta) after a device synchronise."""
        out = {}
        for name, e0, e1, meta in self.events:
            c, t, m = out.get(name, (0, 0.0, []))
            out[name] = (c + 1, t + e0.elapsed_time(e1), m + [meta])
        return out


TRACE = _Trace()


def _dt(dtype: torch.dtype) -> int:
    if dtype not in _DT:
        raise NotImplementedError(f"dax_b200: dtype {dtype} is not supported")
    return _DT[dtype]


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _need_cuda(*ts) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("dax_b200 operators run on CUDA tensors only; there is no CPU path")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _ptr_array(ptrs):
    """Host array of device pointers for the ``*_scatter`` entry points."""
    import ctypes
    return (ctypes.c_void_p * len(ptrs))(*[int(p) for p in ptrs])


def peer_copy(dst_ptr: int, src: torch.Tensor, stream: Optional[torch.cuda.Stream] = None) -> None:
    """Copy the contiguous tensor ``src`` to the device address ``dst_ptr`` (possibly another GPU's buffer) with the
    copy engines, on ``stream`` (default: the current stream)."""
    _need_cuda(src)
    assert src.is_contiguous()
    st = (stream or torch.cuda.current_stream()).cuda_stream
    check(load().dax_peer_copy(int(dst_ptr), src.data_ptr(), src.numel() * src.element_size(), st))


def quant_rowwise(x: torch.Tensor, q_dtype: torch.dtype, *, col_group: Optional[int] = None,
                  group_stride: int = 0, rows: Optional[int] = None, cols: Optional[int] = None,
                  ldx: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-token quantisation of a ``[M, K]`` matrix -> ``(q [M, K], scale [M, 1] fp32)``.

    With ``col_group``/``group_stride`` (and explicit ``rows``, ``cols``, ``ldx``) ``x`` is read as
    column groups living in separate slabs, see ``dax_quant_rowwise`` in ``include/dax_b200.h``."""
    _need_cuda(x)
    if col_group is None:
        x2 = x.reshape(-1, x.shape[-1])
        if x2.stride(-1) != 1:
            x2 = x2.contiguous()
        M, K = x2.shape
        ld, cg, gs = x2.stride(0) if M > 1 else K, K, 0
        src = x2
    else:
        M, K, ld, cg, gs, src = rows, cols, ldx, col_group, group_stride, x
    q = torch.empty((M, K), dtype=q_dtype, device=x.device)
    scale = torch.empty((M, 1), dtype=torch.float32, device=x.device)
    tok = TRACE.begin("quant_rowwise")
    check(load().dax_quant_rowwise(src.data_ptr(), _dt(x.dtype), M, K, ld, cg, gs, q.data_ptr(), _dt(q_dtype),
                                   scale.data_ptr(), _stream()))
    TRACE.end(tok, (M, K, x.element_size()))
    return q, scale


def gemm_dequant(qx: torch.Tensor, sx: torch.Tensor, qw: torch.Tensor, sw: torch.Tensor,
                 bias: Optional[torch.Tensor], out_dtype: torch.dtype, *, out: Optional[torch.Tensor] = None,
                 ldo: Optional[int] = None, out_col_group: Optional[int] = None, out_group_stride: int = 0,
                 row_sumsq: Optional[torch.Tensor] = None, acc_dump: Optional[torch.Tensor] = None,
                 act: Optional[str] = None, resid: Optional[torch.Tensor] = None,
                 gate: Optional[torch.Tensor] = None, group_ptrs=None) -> Optional[torch.Tensor]:
    """``out = cast((acc(qx @ qw.T) * sx) * sw) + bias`` on the tcgen05 INT8 / FP8 pipe, optionally followed
    by ``act="gelu_tanh"`` and / or the gated residual ``out = resid + gate * out`` (gate ``[N]`` fp32).
    With ``group_ptrs`` (device addresses, one per group of ``out_col_group`` columns, possibly peer mappings of
    other GPUs' buffers) row ``t`` of group ``g`` is stored at ``group_ptrs[g] + t * ldo``; nothing is returned."""
    _need_cuda(qx, sx, qw, sw, bias, out)
    M, K = qx.shape
    N = qw.shape[0]
    assert qw.shape[1] == K and qx.is_contiguous() and qw.is_contiguous()
    assert sx.numel() == M and sw.numel() == N and sx.dtype == torch.float32 and sw.dtype == torch.float32
    if group_ptrs is not None:
        assert out is None and row_sumsq is None and acc_dump is None and act is None and resid is None
        tok = TRACE.begin("gemm_dequant")
        check(load().dax_gemm_dequant_scatter(qx.data_ptr(), _dt(qx.dtype), sx.data_ptr(), qw.data_ptr(), _dt(qw.dtype),
                                              sw.data_ptr(), _ptr(bias), _dt(bias.dtype) if bias is not None else 0,
                                              _ptr_array(group_ptrs), len(group_ptrs), _dt(out_dtype), M, N, K, ldo,
                                              out_col_group, _stream()))
        TRACE.end(tok, (M, N, K))
        return None
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=qx.device)
        ldo = N
    if out_col_group is None:
        out_col_group = N
    if act not in (None, "gelu_tanh"):
        raise NotImplementedError(f"unknown activation {act!r}")
    if resid is not None:
        _need_cuda(resid, gate)
        assert resid.dtype == out_dtype and resid.stride(-1) == 1 and resid.shape == (M, N)
        assert gate is None or (gate.dtype == torch.float32 and gate.numel() == N and gate.is_contiguous())
    tok = TRACE.begin("gemm_dequant")
    check(load().dax_gemm_dequant_ex(qx.data_ptr(), _dt(qx.dtype), sx.data_ptr(), qw.data_ptr(), _dt(qw.dtype),
                                     sw.data_ptr(), _ptr(bias), _dt(bias.dtype) if bias is not None else 0,
                                     out.data_ptr(), _dt(out_dtype), M, N, K, ldo, out_col_group, out_group_stride,
                                     _ptr(row_sumsq), _ptr(acc_dump), 1 if act else 0, _ptr(resid),
                                     resid.stride(0) if resid is not None else 0, _ptr(gate), _stream()))
    TRACE.end(tok, (M, N, K))
    return out


def linear_dynamic(x: torch.Tensor, qw: torch.Tensor, sw: torch.Tensor, bias: Optional[torch.Tensor],
                   act_dtype: torch.dtype, out_dtype: torch.dtype) -> torch.Tensor:
    """``dynamic.Linear.forward`` in one library call: quantise ``x [M, K]`` per token, multiply by the
    quantised weight ``qw [N, K]``, de-quantise, add the bias.  The workspace comes from torch."""
    _need_cuda(x, qw, sw, bias)
    M, K = x.shape
    N = qw.shape[0]
    assert x.stride(1) == 1 and qw.is_contiguous()
    n = load().dax_linear_dynamic_workspace_bytes(M, K)
    ws = torch.empty(n + 256, dtype=torch.uint8, device=x.device)
    off = (-ws.data_ptr()) % 256
    out = torch.empty((M, N), dtype=out_dtype, device=x.device)
    tok = TRACE.begin("linear_dynamic")
    check(load().dax_linear_dynamic(x.data_ptr(), _dt(x.dtype), M, K, x.stride(0) if M > 1 else K, qw.data_ptr(),
                                    _dt(qw.dtype), _dt(act_dtype), sw.data_ptr(), _ptr(bias),
                                    _dt(bias.dtype) if bias is not None else 0, out.data_ptr(), _dt(out_dtype), N, N,
                                    ws.data_ptr() + off, n, _stream()))
    TRACE.end(tok, (M, N, K))
    return out


def layernorm_modulate_quant(x: torch.Tensor, *, eps: float = 1e-6, ln_weight: Optional[torch.Tensor] = None,
                             ln_bias: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None,
                             scale: Optional[torch.Tensor] = None, q_dtype: Optional[torch.dtype] = None,
                             want_y: bool = True):
    """``y = LN(x) [* w + b] [* (1 + scale) + shift]`` per token row of ``x [s, D]`` (all vectors ``[D]`` fp32),
    optionally with the per-token quantisation of ``y`` fused in.  Returns ``(y or None, q or None, qscale or None)``."""
    _need_cuda(x, ln_weight, ln_bias, shift, scale)
    s_, D = x.shape
    assert x.stride(1) == 1
    for v in (ln_weight, ln_bias, shift, scale):
        assert v is None or (v.dtype == torch.float32 and v.numel() == D and v.is_contiguous())
    y = torch.empty((s_, D), dtype=x.dtype, device=x.device) if want_y else None
    q = qs = None
    if q_dtype is not None:
        q = torch.empty((s_, D), dtype=q_dtype, device=x.device)
        qs = torch.empty((s_, 1), dtype=torch.float32, device=x.device)
    tok = TRACE.begin("layernorm_modulate_quant")
    check(load().dax_layernorm_modulate_quant(x.data_ptr(), _dt(x.dtype), s_, D, x.stride(0), _ptr(ln_weight),
                                              _ptr(ln_bias), _ptr(shift), _ptr(scale), float(eps), _ptr(y), D, _ptr(q),
                                              _dt(q_dtype) if q_dtype is not None else 0, _ptr(qs), _stream()))
    TRACE.end(tok, (s_, D))
    return y, q, qs


def rmsnorm_rope_pack(x: torch.Tensor, *, norm_weight: Optional[torch.Tensor], do_norm: bool, eps: float = 1e-6,
                      rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
                      token_offset: int = 0, row_sumsq: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None, ldo: Optional[int] = None,
                      col_group: Optional[int] = None, group_stride: int = 0, group_ptrs=None) -> Optional[torch.Tensor]:
    """RMSNorm over the full row + rotary embedding + write into a (possibly grouped) layout.  With ``group_ptrs``
    (one device address per column group, possibly in other GPUs' memory) row ``t`` of group ``g`` goes to
    ``group_ptrs[g] + t * ldo``."""
    _need_cuda(x, norm_weight, rope_cos, rope_sin, row_sumsq, out)
    s, D = x.shape
    assert x.stride(1) == 1
    if group_ptrs is not None:
        assert out is None and ldo is not None and col_group is not None
    elif out is None:
        out = torch.empty((s, D), dtype=x.dtype, device=x.device)
        ldo = D
    if col_group is None:
        col_group = D
    # the kernel reads the weight as 16-bit elements of x's dtype and the tables as fp32 [S_total, 64]
    if norm_weight is not None and (norm_weight.dtype != x.dtype or norm_weight.numel() != D or not norm_weight.is_contiguous()):
        raise ValueError(f"rmsnorm_rope_pack: norm_weight must be a contiguous [{D}] tensor of {x.dtype}, got "
                         f"{tuple(norm_weight.shape)} {norm_weight.dtype}")
    if (rope_cos is None) != (rope_sin is None):
        raise ValueError("rmsnorm_rope_pack: rope_cos and rope_sin come together")
    for tname, tab in (("rope_cos", rope_cos), ("rope_sin", rope_sin)):
        if tab is not None and (tab.dtype != torch.float32 or tab.dim() != 2 or tab.shape[1] != 64 or not tab.is_contiguous()
                                or token_offset + s > tab.shape[0]):
            raise ValueError(f"rmsnorm_rope_pack: {tname} must be a contiguous fp32 [>= {token_offset + s}, 64] table, got "
                             f"{tuple(tab.shape)} {tab.dtype}")
    if row_sumsq is not None and (row_sumsq.dtype != torch.float32 or row_sumsq.dim() != 2 or row_sumsq.shape[0] < s
                                  or not row_sumsq.is_contiguous()):
        raise ValueError(f"rmsnorm_rope_pack: row_sumsq must be a contiguous fp32 [>= {s}, n] tensor")
    n_part = row_sumsq.shape[1] if row_sumsq is not None else 0
    tok = TRACE.begin("rmsnorm_rope_pack")
    if group_ptrs is not None:
        check(load().dax_rmsnorm_rope_pack_scatter(x.data_ptr(), _dt(x.dtype), s, D, x.stride(0), _ptr(row_sumsq), n_part,
                                                   1 if do_norm else 0, _ptr(norm_weight), float(eps), _ptr(rope_cos),
                                                   _ptr(rope_sin), token_offset, _ptr_array(group_ptrs), len(group_ptrs),
                                                   ldo, col_group, _stream()))
        TRACE.end(tok, (s, D))
        return None
    check(load().dax_rmsnorm_rope_pack(x.data_ptr(), _dt(x.dtype), s, D, x.stride(0), _ptr(row_sumsq), n_part,
                                       1 if do_norm else 0, _ptr(norm_weight), float(eps), _ptr(rope_cos),
                                       _ptr(rope_sin), token_offset, out.data_ptr(), ldo, col_group, group_stride,
                                       _stream()))
    TRACE.end(tok, (s, D))
    return out


def _bhsd_strides(t: torch.Tensor) -> I64x3:
    assert t.dim() == 4 and t.shape[-1] == 128 and t.stride(-1) == 1, "expected [B, heads, S, 128], channels contiguous"
    return I64x3(t.stride(0), t.stride(1), t.stride(2))


class AttentionPlan:
    """Prepared operands of one attention call (workspace owned by torch)."""

    def __init__(self, B, heads, Sq, Sk, mode, workspace, dtype):
        self.B, self.heads, self.Sq, self.Sk, self.mode, self.workspace, self.dtype = B, heads, Sq, Sk, mode, workspace, dtype


_WS_CACHE = {}   # (device, B, heads, Sq, Sk, mode) -> buffer; insertion-ordered, a few most recent shapes
_WS_CACHE_ENTRIES = 4


def attn_workspace(B: int, heads: int, Sq: int, Sk: int, mode: int, device) -> torch.Tensor:
    """Workspace of one attention shape.  A block alternates between self-attention and cross-attention, so a few
    shapes stay cached; every plan of the same shape shares ONE buffer: a plan is valid until the next
    ``attn_prepare`` of that shape (on the same stream)."""
    n = load().dax_attn_workspace_bytes(B, heads, Sq, Sk, mode)
    if n == 0:
        check(_lib.DAX_ERR_INVALID)
    key = (str(device), B, heads, Sq, Sk, mode)
    ws = _WS_CACHE.pop(key, None)
    if ws is None:
        while len(_WS_CACHE) >= _WS_CACHE_ENTRIES:
            _WS_CACHE.pop(next(iter(_WS_CACHE)))
        ws = torch.empty(n + 1024, dtype=torch.uint8, device=device)
    _WS_CACHE[key] = ws  # most recently used last
    off = (-ws.data_ptr()) % 1024
    return ws[off:off + n]


def attn_prepare(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mode: str = "bf16",
                 sm_scale: Optional[float] = None, parts: str = "all") -> AttentionPlan:
    """q, k, v: ``[B, heads, S, 128]`` views (any batch/head/token strides) of bf16 or fp16.  ``parts``: "all", or
    "kv" (statistics, K and V operands) and "q" (Q operands) as two calls on the same shape, for callers whose K and
    V are complete before Q is."""
    _need_cuda(q, k, v)
    B, heads, Sq, d = q.shape
    Sk = k.shape[2]
    assert d == 128 and k.shape == v.shape and k.shape[:2] == q.shape[:2] and q.dtype == k.dtype == v.dtype
    m = ATTN_MODES[mode]
    ws = attn_workspace(B, heads, Sq, Sk, m, q.device)
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(d)
    tok = TRACE.begin("attn_prepare")
    TRACE.launches -= {"all": 0, "kv": 1, "q": 4}[parts]  # five kernels in all: four on the K / V side, one for Q
    check(load().dax_attn_prepare_parts(q.data_ptr(), k.data_ptr(), v.data_ptr(), _dt(q.dtype), B, heads, Sq, Sk,
                                        _bhsd_strides(q), _bhsd_strides(k), _bhsd_strides(v), float(sm_scale), m,
                                        {"all": 3, "kv": 1, "q": 2}[parts], ws.data_ptr(), ws.numel(), _stream()))
    TRACE.end(tok, (B, heads, Sq, Sk))
    return AttentionPlan(B, heads, Sq, Sk, m, ws, q.dtype)


def attn_forward(plan: AttentionPlan, out: torch.Tensor, q_begin: int = 0, q_end: Optional[int] = None,
                 n_ranges: int = 1, range_stride: int = 0) -> torch.Tensor:
    """Run the flash pass for the query rows ``[q_begin + r*range_stride, q_end + r*range_stride)``,
    ``r < n_ranges``, into ``out`` (a ``[B, heads, Sq, 128]`` view)."""
    _need_cuda(out)
    if q_end is None:
        q_end = plan.Sq
    assert out.shape == (plan.B, plan.heads, plan.Sq, 128) and out.dtype == plan.dtype
    tok = TRACE.begin("attn_forward")
    check(load().dax_attn_forward(out.data_ptr(), _dt(out.dtype), plan.B, plan.heads, plan.Sq, plan.Sk,
                                  _bhsd_strides(out), q_begin, q_end, n_ranges, range_stride, plan.mode,
                                  plan.workspace.data_ptr(),
                                  plan.workspace.numel(), _stream()))
    TRACE.end(tok, (plan.B, plan.heads, (q_end - q_begin) * n_ranges, plan.Sk))
    return out


def attn_forward_scatter(plan: AttentionPlan, dest_ptrs, rows_per_dest: int, head_stride: int, token_stride: int,
                         q_begin: int = 0, q_end: Optional[int] = None) -> None:
    """The flash pass (batch 1) with every query row written to the destination that owns it: row ``q`` of head
    ``h`` goes to ``dest_ptrs[q // rows_per_dest] + (q % rows_per_dest) * token_stride + h * head_stride``
    (elements of the plan's dtype).  The destinations may be other GPUs' buffers (peer mappings)."""
    assert plan.B == 1
    if q_end is None:
        q_end = plan.Sq
    tok = TRACE.begin("attn_forward")
    check(load().dax_attn_forward_scatter(_ptr_array(dest_ptrs), len(dest_ptrs), rows_per_dest, _dt(plan.dtype), plan.heads,
                                          plan.Sq, plan.Sk, head_stride, token_stride, q_begin, q_end, plan.mode,
                                          plan.workspace.data_ptr(), plan.workspace.numel(), _stream()))
    TRACE.end(tok, (plan.B, plan.heads, q_end - q_begin, plan.Sk))


def direct_attention_ok(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mode: str) -> bool:
    """Whether the in-place 16-bit kernel serves this call: bf16 mode and tensors, at least one tile of queries and
    keys, (batch, head) flattening to one stride."""
    B, heads = q.shape[:2]
    return (ATTN_MODES[mode] == _lib.DAX_ATTN_QK_BF16_PV_BF16 and q.dtype == torch.bfloat16 and q.shape[2] >= 128
            and k.shape[2] >= 128 and (B == 1 or all(t.stride(0) == heads * t.stride(1) for t in (q, k, v))))


def attention_direct(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: Optional[torch.Tensor] = None, *,
                     sm_scale: Optional[float] = None, dest_ptrs=None, rows_per_dest: int = 0, head_stride: int = 0,
                     token_stride: int = 0, q_begin: int = 0, q_end: Optional[int] = None, n_ranges: int = 1,
                     range_stride: int = 0) -> Optional[torch.Tensor]:
    """The 16-bit attention reading ``q, k, v`` (``[B, heads, S, 128]`` views, bf16 or fp16) in place: one kernel, no
    prepare step, no workspace.  Result into ``out`` (a ``[B, heads, Sq, 128]`` view; allocated token-major when
    omitted) or, with ``dest_ptrs``, scattered by destination like ``attn_forward_scatter``."""
    _need_cuda(q, k, v, out)
    B, heads, Sq, d = q.shape
    Sk = k.shape[2]
    assert d == 128 and k.shape == v.shape and k.shape[:2] == q.shape[:2] and q.dtype == k.dtype == v.dtype
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(d)
    if q_end is None:
        q_end = Sq
    if dest_ptrs is not None:
        o_ptr, o_str, table, n = None, I64x3(0, head_stride, token_stride), _ptr_array(dest_ptrs), len(dest_ptrs)
    else:
        if out is None:
            out = torch.empty((B, Sq, heads, d), dtype=q.dtype, device=q.device).transpose(1, 2)
        assert out.shape == (B, heads, Sq, 128) and out.dtype == q.dtype
        o_ptr, o_str, table, n = out.data_ptr(), _bhsd_strides(out), None, 0
    tok = TRACE.begin("attn_forward")
    check(load().dax_attn_forward_direct(q.data_ptr(), k.data_ptr(), v.data_ptr(), _dt(q.dtype), B, heads, Sq, Sk,
                                         _bhsd_strides(q), _bhsd_strides(k), _bhsd_strides(v), float(sm_scale), o_ptr, o_str,
                                         table, n, rows_per_dest, q_begin, q_end, n_ranges, range_stride, _stream()))
    TRACE.end(tok, (B, heads, (q_end - q_begin) * n_ranges, Sk))
    return out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mode: str = "bf16",
              sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Non-causal attention over ``[B, heads, S, 128]``; the result has the memory layout
    ``[B, S, heads, 128]`` (token-major, as the head->sequence exchange wants it) viewed as
    ``[B, heads, S, 128]``."""
    B, heads, Sq, d = q.shape
    if direct_attention_ok(q, k, v, mode):
        return attention_direct(q, k, v, out, sm_scale=sm_scale)  # the 16-bit mode reads its operands in place
    plan = attn_prepare(q, k, v, mode, sm_scale)
    if out is None:
        out = torch.empty((B, Sq, heads, d), dtype=q.dtype, device=q.device).transpose(1, 2)
    return attn_forward(plan, out)


# ---- training: operators with a gradient ---------------------------------------------------------------------------------
# The backward passes recompute what they need from the inputs and the row statistics that the forward passes return.
# Workspaces come from torch for every call (nothing is shared between calls, streams or captured graphs).
_get_device = getattr(torch._C, "_cuda_getDevice", None)  # torch.cuda.current_device() without its checks: the tensors are there


class _OnDevice:
    """Makes a device the current one for a call, if it is not (``torch.cuda.device`` costs as much as a launch)."""

    __slots__ = ("index", "previous")

    def __init__(self, index: int):
        self.index = index

    def __enter__(self) -> int:
        """The raw handle of the device's current stream."""
        self.previous = _get_device()
        if self.previous != self.index:
            torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc) -> None:
        if self.previous != self.index:
            torch.cuda.set_device(self.previous)


def _on_one_device(what: str, *ts) -> int:
    """The index of the device all tensors live on (the call goes to that device's current stream)."""
    dev = None
    for t in ts:
        if t is None:
            continue
        i = t.get_device()
        if i != dev:
            if i < 0:
                _need_cuda(t)
            if dev is not None:
                raise ValueError(f"{what}: tensors are on different devices, cuda:{dev} and {t.device}")
            dev = i
    return dev


def _rows(what: str, name: str, t: torch.Tensor) -> Tuple[torch.Tensor, int, int, int, int, int]:
    """``t [B, S, D]`` or ``[S, D]`` for the row kernels: ``(tensor, B, S, D, sample stride, token stride)``.  They want the
    channels contiguous and everything else in whole 16 bytes; a tensor that is not laid out like that is copied."""
    shape, strides = t.shape, t.stride()
    if len(shape) == 3:
        (B, S, D), (sb, ss, sd) = shape, strides
    elif len(shape) == 2:
        (S, D), (ss, sd), B, sb = shape, strides, 1, 0
    else:
        raise ValueError(f"{what}: {name} must be [B, S, D] or [S, D], got {list(shape)}")
    if t.dtype not in _ROW_PIECE:
        raise NotImplementedError(f"{what}: {name} must be bf16, fp16 or fp32, got {t.dtype}")
    # the stride of a dimension of one is never used, and torch may report anything for it
    sb, ss = sb if B > 1 else 0, ss if S > 1 else 0
    if sd != 1 or sb % _ROW_PIECE[t.dtype] or ss % _ROW_PIECE[t.dtype] or t.data_ptr() % 16:
        t, sb, ss = t.clone(memory_format=torch.contiguous_format), S * D, D
    return t, B, S, D, sb, ss


_ROW_PIECE = {torch.bfloat16: 8, torch.float16: 8, torch.float32: 4}  # elements in 16 bytes


def _vector(what: str, name: str, v: Optional[torch.Tensor], shape: Tuple[int, ...]) -> None:
    if v is not None and (v.dtype != torch.float32 or v.shape != shape or not v.is_contiguous()):
        raise ValueError(f"{what}: {name} must be a contiguous fp32 {list(shape)} tensor, got {v.dtype} {list(v.shape)}")


def _grad_like(what: str, dy: torch.Tensor, x: torch.Tensor) -> None:
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"{what}: dy must be {list(x.shape)} of {x.dtype}, got {list(dy.shape)} of {dy.dtype}")


def _row_statistics(x: torch.Tensor, B: int, S: int) -> torch.Tensor:
    """One fp32 number for each row (``torch.empty`` costs twice as much on the host)."""
    size, strides = ((B, S), (S, 1)) if x.dim() == 3 else ((S,), (1,))
    return torch.empty_strided(size, strides, dtype=torch.float32, device=x.device)


@functools.lru_cache(maxsize=256)
def _norm_workspace_bytes(device: int, B: int, S: int, D: int) -> int:
    return load().dax_norm_backward_workspace_bytes(B, S, D)  # goes by the SM count of the current device, which is `device`


@functools.lru_cache(maxsize=256)
def _attention_plan(device: int, B: int, heads: int, Sq: int, Sk: int) -> Tuple[int, int]:
    """Workspace bytes and kernels of the forward pass on the current device, which is ``device``."""
    lib = load()
    return lib.dax_attn_lse_workspace_bytes(B, heads, Sq, Sk), lib.dax_attn_lse_kernels(B, heads, Sq, Sk)


@functools.lru_cache(maxsize=256)
def _attention_backward_plan(device: int, dtype: int, B: int, heads: int, Sq: int, Sk: int, keys: bool) -> Tuple[int, int]:
    lib = load()
    return lib.dax_attn_backward_workspace_bytes(B, heads, Sq, Sk), lib.dax_attn_backward_kernels(dtype, B, heads, Sq, Sk, keys)


@functools.lru_cache(maxsize=1024)
def _strides3(sample: int, head: int, token: int) -> I64x3:
    """Three strides as the C entries read them."""
    return I64x3(sample, head, token)


def _workspace(n: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty_strided((n,), (1,), dtype=torch.uint8, device=device) if n else None


def _dense_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


def layernorm_modulate(x: torch.Tensor, *, eps: float = 1e-6, ln_weight: Optional[torch.Tensor] = None,
                       ln_bias: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None,
                       scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``y = (n [* ln_weight + ln_bias]) [* (1 + scale) + shift]`` with ``n`` the LayerNorm of every token row of ``x [B, S, D]``
    (bf16, fp16 or fp32); ``ln_weight, ln_bias [D]`` and ``shift, scale [B, D]`` (one row for each sample) fp32.  ``x [S, D]``
    is one sample with ``shift, scale [D]``.  Returns ``(y, mean, rstd)``; the statistics (fp32, one for each row) are what
    ``layernorm_modulate_backward`` needs.  The inference step, which quantises ``y``, is ``layernorm_modulate_quant``."""
    what = "layernorm_modulate"
    rows, B, S, D, sb, ss = _rows(what, "x", x)
    modulation = (B, D) if x.dim() == 3 else (D,)
    _vector(what, "ln_weight", ln_weight, (D,))
    _vector(what, "ln_bias", ln_bias, (D,))
    _vector(what, "shift", shift, modulation)
    _vector(what, "scale", scale, modulation)
    dev = _on_one_device(what, x, ln_weight, ln_bias, shift, scale)
    y = _dense_like(x)
    mean = _row_statistics(x, B, S)
    rstd = torch.empty_like(mean)
    with _OnDevice(dev) as stream:
        tok = TRACE.begin(what, int(rows.numel() > 0))
        check(load().dax_layernorm_modulate(rows.data_ptr(), _dt(x.dtype), B, S, D, sb, ss, _ptr(ln_weight),
                                            _ptr(ln_bias), _ptr(shift), _ptr(scale), float(eps), y.data_ptr(), S * D, D,
                                            mean.data_ptr(), rstd.data_ptr(), stream))
        TRACE.end(tok, (B, S, D))
    return y, mean, rstd


def layernorm_modulate_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, *,
                                ln_weight: Optional[torch.Tensor] = None, ln_bias: Optional[torch.Tensor] = None,
                                scale: Optional[torch.Tensor] = None, need_params: bool = True):
    """Gradients of ``layernorm_modulate`` for the output gradient ``dy`` (shape and dtype of ``x``): ``(dx, dweight, dbias,
    dshift, dscale)``.  The parameter gradients are fp32 sums over the rows, in a fixed order (equal inputs give equal
    bits); those of vectors that were not given, and all of them with ``need_params=False``, are None."""
    what = "layernorm_modulate_backward"
    _grad_like(what, dy, x)
    rows, B, S, D, sb, ss = _rows(what, "x", x)
    grads, _, _, _, gb, gs = _rows(what, "dy", dy)
    statistics = x.shape[:-1]
    _vector(what, "mean", mean, statistics)
    _vector(what, "rstd", rstd, statistics)
    _vector(what, "ln_weight", ln_weight, (D,))
    _vector(what, "ln_bias", ln_bias, (D,))
    _vector(what, "scale", scale, (B, D) if x.dim() == 3 else (D,))
    dev = _on_one_device(what, dy, x, mean, rstd, ln_weight, ln_bias, scale)
    dx = _dense_like(x)
    dweight = torch.empty_like(ln_weight) if need_params and ln_weight is not None else None
    dbias = torch.empty_like(ln_bias) if need_params and ln_bias is not None else None
    dshift, dscale = (torch.empty_like(scale), torch.empty_like(scale)) if need_params and scale is not None else (None, None)
    with _OnDevice(dev) as stream:
        lib, dt = load(), _dt(x.dtype)
        sums = dweight is not None or dscale is not None
        n = _norm_workspace_bytes(dev, B, S, D) if sums else 0
        ws = _workspace(n, x.device)
        tok = TRACE.begin(what, (rows.numel() > 0) + sums)
        check(lib.dax_layernorm_modulate_backward(grads.data_ptr(), rows.data_ptr(), dt, B, S, D, gb, gs, sb, ss,
                                                  mean.data_ptr(), rstd.data_ptr(), _ptr(ln_weight), _ptr(ln_bias), _ptr(scale),
                                                  dx.data_ptr(), S * D, D, _ptr(dweight), _ptr(dbias), _ptr(dshift), _ptr(dscale),
                                                  _ptr(ws), n, stream))
        TRACE.end(tok, (B, S, D))
    return dx, dweight, dbias, dshift, dscale


def _rope_check(what: str, S: int, D: int, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor]) -> None:
    if (cos is None) != (sin is None):
        raise ValueError(f"{what}: rope_cos and rope_sin come together")
    for name, t in (("rope_cos", cos), ("rope_sin", sin)):
        if t is not None and (t.dtype != torch.float32 or t.dim() != 2 or t.shape[0] < S or t.shape[1] != 64 or not t.is_contiguous()):
            raise ValueError(f"{what}: {name} must be a contiguous fp32 [>= {S}, 64] table, got {t.dtype} {list(t.shape)}")
    if cos is not None and D % 128:
        raise ValueError(f"{what}: a rotation needs D={D} to be whole heads of 128 channels")


def rmsnorm_rope(x: torch.Tensor, norm_weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                 rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm over the whole row of ``x [B, S, D]`` (or ``[S, D]``; bf16, fp16 or fp32), times ``norm_weight [D]`` (fp32), then
    the rotation of every head's channel pairs by the angles of row ``s`` of the tables (fp32 ``[>= S, 64]``, the same for
    every sample).  Returns ``(y, rstd)``; ``rstd`` is what ``rmsnorm_rope_backward`` needs.  The inference step, which writes
    the exchange layout, is ``rmsnorm_rope_pack``."""
    what = "rmsnorm_rope"
    rows, B, S, D, sb, ss = _rows(what, "x", x)
    _vector(what, "norm_weight", norm_weight, (D,))
    _rope_check(what, S, D, rope_cos, rope_sin)
    dev = _on_one_device(what, x, norm_weight, rope_cos, rope_sin)
    y = _dense_like(x)
    rstd = _row_statistics(x, B, S)
    with _OnDevice(dev) as stream:
        tok = TRACE.begin(what, int(rows.numel() > 0))
        check(load().dax_rmsnorm_rope(rows.data_ptr(), _dt(x.dtype), B, S, D, sb, ss, _ptr(norm_weight), _ptr(rope_cos),
                                      _ptr(rope_sin), float(eps), y.data_ptr(), S * D, D, rstd.data_ptr(), stream))
        TRACE.end(tok, (B, S, D))
    return y, rstd


def rmsnorm_rope_backward(dy: torch.Tensor, x: torch.Tensor, rstd: torch.Tensor, norm_weight: Optional[torch.Tensor] = None, *,
                          rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
                          need_params: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Gradients of ``rmsnorm_rope``: ``(dx, dweight)``, ``dweight`` (fp32, summed in a fixed order) None without a weight
    or with ``need_params=False``."""
    what = "rmsnorm_rope_backward"
    _grad_like(what, dy, x)
    rows, B, S, D, sb, ss = _rows(what, "x", x)
    grads, _, _, _, gb, gs = _rows(what, "dy", dy)
    _vector(what, "rstd", rstd, x.shape[:-1])
    _vector(what, "norm_weight", norm_weight, (D,))
    _rope_check(what, S, D, rope_cos, rope_sin)
    dev = _on_one_device(what, dy, x, rstd, norm_weight, rope_cos, rope_sin)
    dx = _dense_like(x)
    dweight = torch.empty_like(norm_weight) if need_params and norm_weight is not None else None
    with _OnDevice(dev) as stream:
        lib, dt = load(), _dt(x.dtype)
        n = _norm_workspace_bytes(dev, B, S, D) if dweight is not None else 0
        ws = _workspace(n, x.device)
        tok = TRACE.begin(what, (rows.numel() > 0) + (dweight is not None))
        check(lib.dax_rmsnorm_rope_backward(grads.data_ptr(), rows.data_ptr(), dt, B, S, D, gb, gs, sb, ss,
                                            rstd.data_ptr(), _ptr(norm_weight), _ptr(rope_cos), _ptr(rope_sin), dx.data_ptr(), S * D, D,
                                            _ptr(dweight), _ptr(ws), n, stream))
        TRACE.end(tok, (B, S, D))
    return dx, dweight


def _heads_view(t: torch.Tensor) -> Tuple[torch.Tensor, I64x3]:
    """``t [B, heads, S, 128]`` and its strides for the kernels; a tensor they cannot address (channels not contiguous,
    broadcast dimensions, misaligned) is copied into token-major memory."""
    s0, s1, s2, s3 = t.stride()
    if s3 == 1 and s0 > 0 and s1 > 0 and s2 > 0 and (s0 | s1 | s2) % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, _strides3(s0, s1, s2)
    # a dimension of one may have any stride: the kernels get a valid one
    st = [st if n > 1 else 128 for n, st in zip(t.shape, (s0, s1, s2))]
    if s3 != 1 or t.data_ptr() % 16 or any(v <= 0 or v % 8 for v in st):
        t = _token_major(t).copy_(t)
        st = t.stride()[:3]
    return t, _strides3(*st)


def _attention_inputs(what: str, q, k, v, q_lens, k_lens, sm_scale) -> Tuple[int, int, int, int, float]:
    qs, ks, vs, dt = q.shape, k.shape, v.shape, q.dtype
    for name, shape in (("q", qs), ("k", ks), ("v", vs)):
        if len(shape) != 4 or shape[3] != 128:
            raise ValueError(f"{what}: {name} must be [B, heads, S, 128], got {list(shape)}")
    B, heads, Sq, _ = qs
    if ks != vs or ks[0] != B or ks[1] != heads:
        raise ValueError(f"{what}: q {list(qs)}, k {list(ks)} and v {list(vs)} do not belong together")
    if dt not in (torch.bfloat16, torch.float16) or k.dtype != dt or v.dtype != dt:
        raise NotImplementedError(f"{what}: q, k and v must all be bf16 or all fp16, got {dt}, {k.dtype}, {v.dtype}")
    for name, t in (("q_lens", q_lens), ("k_lens", k_lens)):
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (B,) or not t.is_contiguous()):
            raise ValueError(f"{what}: {name} must be a contiguous int32 [{B}] tensor, got {t.dtype} {list(t.shape)}")
    if sm_scale is None:
        sm_scale = _SM_SCALE
    elif not 0.0 < sm_scale < math.inf:
        raise ValueError(f"{what}: sm_scale must be positive and finite, got {sm_scale}")
    return B, heads, Sq, ks[2], float(sm_scale)


_SM_SCALE = 1.0 / math.sqrt(128)


def _token_major(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised ``[B, heads, S, 128]`` tensor like ``t`` whose memory is ``[B, S, heads, 128]``."""
    B, heads, S, d = t.shape
    return torch.empty_strided((B, heads, S, d), (S * heads * d, d, heads * d, 1), dtype=t.dtype, device=t.device)


def _token_major_strides(heads: int, S: int) -> I64x3:
    return _strides3(S * heads * 128, 128, heads * 128)


def attention_lse(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, q_lens: Optional[torch.Tensor] = None,
                  k_lens: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Non-causal attention over ``[B, heads, S, 128]`` (bf16 or fp16, any strides) that keeps what its gradient needs:
    ``(out, lse)``, ``out`` token-major like the result of ``attention``, ``lse [B, heads, Sq]`` fp32 (natural logarithm).
    ``q_lens`` / ``k_lens`` (int32 ``[B]`` on the device): the tokens of each sample of a padded batch that exist; the
    others may hold anything.  Queries that do not exist or see no key get ``out = 0``, ``lse = -inf``."""
    what = "attention_lse"
    B, heads, Sq, Sk, sm_scale = _attention_inputs(what, q, k, v, q_lens, k_lens, sm_scale)
    dev = _on_one_device(what, q, k, v, q_lens, k_lens)
    out = _token_major(q)
    lse = torch.empty_strided((B, heads, Sq), (heads * Sq, Sq, 1), dtype=torch.float32, device=q.device)
    if lse.numel() == 0:
        return out, lse
    if Sk == 0:
        return out.zero_(), lse.fill_(-math.inf)
    (q, qs), (k, ks), (v, vs) = _heads_view(q), _heads_view(k), _heads_view(v)
    with _OnDevice(dev) as stream:
        lib = load()
        n, kernels = _attention_plan(dev, B, heads, Sq, Sk)
        ws = _workspace(n, q.device)
        tok = TRACE.begin(what, kernels)
        check(lib.dax_attn_forward_lse(q.data_ptr(), k.data_ptr(), v.data_ptr(), _dt(q.dtype), B, heads, Sq, Sk, qs, ks, vs, sm_scale,
                                       _ptr(q_lens), _ptr(k_lens), out.data_ptr(), _token_major_strides(heads, Sq), lse.data_ptr(),
                                       _ptr(ws), n, stream))
        TRACE.end(tok, (B, heads, Sq, Sk))
    return out, lse


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, *,
                       q_lens: Optional[torch.Tensor] = None, k_lens: Optional[torch.Tensor] = None,
                       sm_scale: Optional[float] = None,
                       need_keys: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Gradients ``(dq, dk, dv)`` (token-major) of ``attention_lse`` for the output gradient ``dout``, from the same inputs
    and what it returned.  The probabilities are recomputed; sums are fp32 in a fixed order, so equal inputs give equal
    bits.  Tokens that do not exist get zero gradients and contribute to none.  With ``need_keys=False`` dk and dv are None
    and their kernel does not run."""
    what = "attention_backward"
    B, heads, Sq, Sk, sm_scale = _attention_inputs(what, q, k, v, q_lens, k_lens, sm_scale)
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != q.shape or t.dtype != q.dtype:
            raise ValueError(f"{what}: {name} must be {list(q.shape)} of {q.dtype}, got {list(t.shape)} of {t.dtype}")
    _vector(what, "lse", lse, (B, heads, Sq))
    dev = _on_one_device(what, dout, q, k, v, out, lse, q_lens, k_lens)
    dq = _token_major(q)
    dk = dv = None
    if need_keys:
        dk = _token_major(k)
        dv = torch.empty_like(dk)
    if lse.numel() == 0 or Sk == 0:
        return tuple(g if g is None else g.zero_() for g in (dq, dk, dv))
    (dout, dos), (q, qs), (k, ks), (v, vs), (out, os_) = map(_heads_view, (dout, q, k, v, out))
    kv = _token_major_strides(heads, Sk)
    with _OnDevice(dev) as stream:
        lib = load()
        dt = _dt(q.dtype)
        n, kernels = _attention_backward_plan(dev, dt, B, heads, Sq, Sk, need_keys)
        ws = _workspace(n, q.device)
        tok = TRACE.begin(what, kernels)
        check(lib.dax_attn_backward(dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), dt,
                                    B, heads, Sq, Sk, dos, qs, ks, vs, os_, sm_scale, _ptr(q_lens), _ptr(k_lens), dq.data_ptr(),
                                    _ptr(dk), _ptr(dv), _token_major_strides(heads, Sq), kv, kv, ws.data_ptr(), n, stream))
        TRACE.end(tok, (B, heads, Sq, Sk))
    return dq, dk, dv
