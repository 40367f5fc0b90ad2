"""Torch-facing wrappers of the libmi355attn entry points.

Each wrapper validates shapes/dtypes/devices on the host, allocates outputs with torch (the
library never allocates), and enqueues the kernel on torch's current stream of the tensors'
device. Nothing here synchronises the host, so the calls are hipGraph-capturable.
"""
from __future__ import annotations

import ctypes
import functools
import operator
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

# status of an entry point that cannot run the requested combination (nothing launched)
_E_UNSUPPORTED = -6


@dataclass
class KeyBoundTarget:
    """Where a QKV projection writes the attention's key-norm bounds (``mi355_*_kbound``).

    ``workspace`` is the attention workspace (uint8, ``attention_workspace``), whose bound
    section the projection fills for the K block: output columns ``[k_col0, k_col0 + heads *
    head_dim)`` of ``seq`` tokens per batch row, with ``key_valid`` ([B, seq] bool, optional)
    marking chunks that hold an invalid key. ``written`` tells whether the projection wrote
    them (the fused epilogue has shape requirements; otherwise the attention runs its own pass).
    """
    workspace: torch.Tensor
    k_col0: int
    heads: int
    head_dim: int
    seq: int
    key_valid: Optional[torch.Tensor] = None
    written: bool = False

    def _args(self, M: int):
        if self.workspace.dtype != torch.uint8 or self.workspace.dim() != 1:
            raise ValueError("the key-bound workspace is a 1-D uint8 tensor")
        kv = _mask_ptr(self.key_valid, (M // self.seq, self.seq)) if M % self.seq == 0 and \
            self.key_valid is not None else 0
        return (self.workspace.data_ptr(), self.k_col0, self.heads, self.head_dim, self.seq, kv)


def attention_workspace(B: int, S_q: int, S_k: int, H: int, head_dim: int, dtype: torch.dtype,
                        device: torch.device) -> torch.Tensor:
    """A workspace for ``attention(..., workspace=...)`` on ``[B, S, H, head_dim]`` problems of
    ``dtype``: the key-norm bounds and the redo flags (``mi355_attn_workspace_bytes_forced``);
    empty when the problem does not run on the matrix-core kernel."""
    n = _lib.lib().mi355_attn_workspace_bytes_forced(_lib.dtype_code(dtype), B, H, S_q, S_k,
                                                     head_dim)
    return torch.empty((max(int(n), 0),), device=device, dtype=torch.uint8)


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _on_gpu(*tensors: Optional[torch.Tensor]) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise ValueError(f"expected a GPU tensor, got one on {t.device}")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} vs {t.device}")
    if dev is None:
        raise ValueError("no tensor given")
    return dev


def _mask_ptr(mask: Optional[torch.Tensor], shape: Tuple[int, ...]) -> int:
    if mask is None:
        return 0
    if mask.dtype not in (torch.bool, torch.uint8):
        raise TypeError("masks must be bool or uint8")
    if tuple(mask.shape) != tuple(shape) or not mask.is_contiguous():
        raise ValueError(f"mask must be a contiguous tensor of shape {shape}")
    return mask.data_ptr()


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None, row_valid: Optional[torch.Tensor] = None,
           out_dtype: Optional[torch.dtype] = None,
           residual: Optional[torch.Tensor] = None, gelu: bool = False,
           zero_masked_rows: bool = False,
           key_bounds: Optional[KeyBoundTarget] = None) -> torch.Tensor:
    """``out[M, N] = x[M, K] @ weight[N, K]^T + bias[N]`` (nn.Linear), fp32 accumulate.

    ``x`` may be a row-strided 2-D view (unit column stride); ``weight`` must be contiguous and
    of x's dtype; ``bias`` is fp32. ``out_dtype`` (default x's dtype) may be any of fp32 /
    fp16 / bf16 for 16-bit inputs, and fp32 or fp16 for fp32 inputs. Rows whose ``row_valid`` entry is False are written as zeros.
    With ``residual`` ([M, N] of out_dtype, unit column stride; may be ``out`` itself) the result
    is ``residual + out_dtype(projection)``, masked rows giving ``residual`` -- or zeros with
    ``zero_masked_rows`` (the block's trailing masked_fill). ``gelu`` applies the exact GELU to
    the projection rounded to out_dtype (``F.gelu(nn.Linear(...)(x))``); it excludes
    ``residual`` and ``row_valid``. With ``key_bounds`` (a QKV projection; no residual, GELU
    or row mask) the epilogue also writes the attention's key-norm bounds when the shapes allow
    (``key_bounds.written``).
    """
    _on_gpu(x, weight, bias, out, row_valid, residual)
    if x.dim() != 2 or weight.dim() != 2:
        raise ValueError("linear expects 2-D x and weight")
    M, K = x.shape
    N, K2 = weight.shape
    if K2 != K:
        raise ValueError(f"inner sizes differ: x has K={K}, weight has K={K2}")
    dt = x.dtype
    odt = out_dtype or (out.dtype if out is not None else dt)
    if weight.dtype != dt:
        raise TypeError("x and weight must share one dtype")
    if x.stride(1) != 1 or not weight.is_contiguous():
        raise ValueError("x needs unit column stride and weight must be contiguous")
    if bias is not None and (bias.shape != (N,) or bias.dtype != torch.float32
                             or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous fp32 tensor of shape ({N},)")
    if out is None:
        out = torch.empty((M, N), device=x.device, dtype=odt)
    elif out.shape != (M, N) or out.dtype != odt or out.stride(1) != 1:
        raise ValueError("out must be [M, N] of out_dtype with unit column stride")
    if gelu:
        if residual is not None or row_valid is not None:
            raise ValueError("the GELU epilogue takes no residual or row mask")
        st = _lib.lib().mi355_gemm_bias_gelu(
            _lib.dtype_code(dt), _lib.dtype_code(odt), x.data_ptr(), x.stride(0),
            weight.data_ptr(), weight.stride(0), bias.data_ptr() if bias is not None else 0,
            out.data_ptr(), out.stride(0), M, N, K, _stream(x))
        _lib.check("mi355_gemm_bias_gelu", st)
        return out
    if zero_masked_rows and residual is None:
        raise ValueError("zero_masked_rows is a mode of the residual epilogue")
    if residual is not None:
        if residual.shape != (M, N) or residual.dtype != odt or residual.stride(1) != 1:
            raise ValueError("residual must be [M, N] of out_dtype with unit column stride")
        fn = "mi355_gemm_bias_residual_zero_masked" if zero_masked_rows else "mi355_gemm_bias_residual"
        st = getattr(_lib.lib(), fn)(
            _lib.dtype_code(dt), _lib.dtype_code(odt), x.data_ptr(), x.stride(0),
            weight.data_ptr(), weight.stride(0), bias.data_ptr() if bias is not None else 0,
            residual.data_ptr(), residual.stride(0), out.data_ptr(), out.stride(0), M, N, K,
            _mask_ptr(row_valid, (M,)), _stream(x))
        _lib.check(fn, st)
        return out
    if key_bounds is not None:
        if row_valid is not None:
            raise ValueError("the key-bound epilogue takes no row mask")
        _on_gpu(x, key_bounds.workspace, key_bounds.key_valid)
        st = _lib.lib().mi355_gemm_bias_kbound(
            _lib.dtype_code(dt), _lib.dtype_code(odt), x.data_ptr(), x.stride(0),
            weight.data_ptr(), weight.stride(0), bias.data_ptr() if bias is not None else 0,
            out.data_ptr(), out.stride(0), M, N, K, *key_bounds._args(M), _stream(x))
        key_bounds.written = st == 0
        if st != _E_UNSUPPORTED:
            _lib.check("mi355_gemm_bias_kbound", st)
            return out
    st = _lib.lib().mi355_gemm_bias(
        _lib.dtype_code(dt), _lib.dtype_code(odt), x.data_ptr(), x.stride(0), weight.data_ptr(),
        weight.stride(0), bias.data_ptr() if bias is not None else 0, out.data_ptr(),
        out.stride(0), M, N, K, _mask_ptr(row_valid, (M,)), _stream(x))
    _lib.check("mi355_gemm_bias", st)
    return out


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
               eps: float = 1e-5, out: Optional[torch.Tensor] = None,
               row_valid: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Row LayerNorm of a 2-D ``x`` (nn.LayerNorm over the last dimension): fp32 statistics,
    output rounded once to x's dtype, or to ``out_dtype`` (fp16 for an fp32 x: the fp16 operand
    of an fp32 model's projection). ``weight``/``bias`` are contiguous ``[K]`` of x's dtype.
    Rows whose ``row_valid`` entry is False are written as zeros."""
    _on_gpu(x, weight, bias, out, row_valid)
    if x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("layer_norm expects a 2-D x with unit column stride")
    M, K = x.shape
    for t in (weight, bias):
        if t is not None and (t.shape != (K,) or t.dtype != x.dtype or not t.is_contiguous()):
            raise ValueError(f"LayerNorm weight/bias must be contiguous [{K}] of x's dtype")
    odt = out_dtype or (out.dtype if out is not None else x.dtype)
    if out is None:
        out = torch.empty((M, K), device=x.device, dtype=odt)
    elif out.shape != (M, K) or out.dtype != odt or out.stride(1) != 1:
        raise ValueError("out must be [M, K] of the output dtype with unit column stride")
    if odt != x.dtype:
        if row_valid is not None:
            raise ValueError("a converting LayerNorm takes no row mask")
        st = _lib.lib().mi355_layernorm_cvt(
            _lib.dtype_code(x.dtype), _lib.dtype_code(odt), x.data_ptr(), x.stride(0),
            weight.data_ptr() if weight is not None else 0,
            bias.data_ptr() if bias is not None else 0, float(eps), out.data_ptr(), out.stride(0),
            M, K, _stream(x))
        _lib.check("mi355_layernorm_cvt", st)
        return out
    if row_valid is not None:
        st = _lib.lib().mi355_layernorm_masked(
            _lib.dtype_code(x.dtype), x.data_ptr(), x.stride(0),
            weight.data_ptr() if weight is not None else 0,
            bias.data_ptr() if bias is not None else 0, float(eps), out.data_ptr(), out.stride(0),
            M, K, _mask_ptr(row_valid, (M,)), _stream(x))
        _lib.check("mi355_layernorm_masked", st)
        return out
    st = _lib.lib().mi355_layernorm(
        _lib.dtype_code(x.dtype), x.data_ptr(), x.stride(0),
        weight.data_ptr() if weight is not None else 0, bias.data_ptr() if bias is not None else 0,
        float(eps), out.data_ptr(), out.stride(0), M, K, _stream(x))
    _lib.check("mi355_layernorm", st)
    return out


def fold_layernorm(weight: torch.Tensor, bias: Optional[torch.Tensor],
                   gamma: Optional[torch.Tensor], beta: Optional[torch.Tensor],
                   dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Host-side fold of a LayerNorm (gamma, beta) into the projection that consumes it, for
    ``layernorm_linear``: returns ``(Wf [N, K] of dtype, colsum [N] fp32, bias' [N] fp32)`` with
    ``Wf = dtype(W * gamma)``, ``colsum = sum_k Wf[:, k]`` (of the rounded Wf, so the epilogue's
    mean subtraction cancels exactly against the weights the GEMM uses) and
    ``bias' = b + W @ beta``; the sums are formed in fp64. Run once per weight version."""
    with torch.no_grad():
        w64 = weight.detach().to(torch.float64)
        g = gamma.detach().to(torch.float64) if gamma is not None else None
        wf = (w64 * g[None, :] if g is not None else w64).to(dtype).contiguous()
        colsum = wf.to(torch.float64).sum(dim=1).to(torch.float32).contiguous()
        b = (bias.detach().to(torch.float64) if bias is not None
             else torch.zeros(weight.shape[0], dtype=torch.float64, device=weight.device))
        if beta is not None:
            b = b + w64 @ beta.detach().to(torch.float64)
        return wf, colsum, b.to(torch.float32).contiguous()


def layernorm_linear(x: torch.Tensor, weight: torch.Tensor, colsum: torch.Tensor,
                     bias: Optional[torch.Tensor], eps: float = 1e-5,
                     out_dtype: Optional[torch.dtype] = None, gelu: bool = False,
                     out: Optional[torch.Tensor] = None,
                     stats: Optional[torch.Tensor] = None,
                     key_bounds: Optional[KeyBoundTarget] = None) -> torch.Tensor:
    """``nn.Linear(nn.LayerNorm(x))`` (optionally followed by the exact GELU) without writing the
    normalised rows: ``weight``, ``colsum`` and ``bias`` come from ``fold_layernorm``. ``x`` is a
    2-D row-strided tensor (unit column stride); the row statistics go to ``stats`` ([M, 2] fp32
    workspace, allocated when not given). ``out_dtype`` defaults to x's dtype (a bf16 or fp32
    input may give fp16). ``key_bounds`` as for ``linear`` (not with ``gelu``)."""
    _on_gpu(x, weight, colsum, bias, out, stats)
    if x.dim() != 2 or weight.dim() != 2 or x.stride(1) != 1:
        raise ValueError("layernorm_linear expects a 2-D x with unit column stride and 2-D weight")
    M, K = x.shape
    N, K2 = weight.shape
    if K2 != K:
        raise ValueError(f"inner sizes differ: x has K={K}, weight has K={K2}")
    if weight.dtype != x.dtype or not weight.is_contiguous():
        raise ValueError("weight must be contiguous and of x's dtype")
    if colsum.shape != (N,) or colsum.dtype != torch.float32 or not colsum.is_contiguous():
        raise ValueError(f"colsum must be a contiguous fp32 tensor of shape ({N},)")
    if bias is not None and (bias.shape != (N,) or bias.dtype != torch.float32
                             or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous fp32 tensor of shape ({N},)")
    odt = out_dtype or (out.dtype if out is not None else x.dtype)
    if out is None:
        out = torch.empty((M, N), device=x.device, dtype=odt)
    elif out.shape != (M, N) or out.dtype != odt or out.stride(1) != 1:
        raise ValueError("out must be [M, N] of out_dtype with unit column stride")
    if stats is None:
        stats = torch.empty((M, 2), device=x.device, dtype=torch.float32)
    elif stats.shape != (M, 2) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise ValueError(f"stats must be a contiguous fp32 tensor of shape ({M}, 2)")
    if key_bounds is not None:
        if gelu:
            raise ValueError("the key-bound epilogue takes no GELU")
        _on_gpu(x, key_bounds.workspace, key_bounds.key_valid)
        st = _lib.lib().mi355_layernorm_gemm_bias_kbound(
            _lib.dtype_code(x.dtype), _lib.dtype_code(odt), x.data_ptr(), x.stride(0),
            weight.data_ptr(), weight.stride(0), colsum.data_ptr(),
            bias.data_ptr() if bias is not None else 0, float(eps), stats.data_ptr(),
            out.data_ptr(), out.stride(0), M, N, K, *key_bounds._args(M), _stream(x))
        key_bounds.written = st == 0
        if st != _E_UNSUPPORTED:
            _lib.check("mi355_layernorm_gemm_bias_kbound", st)
            return out
    st = _lib.lib().mi355_layernorm_gemm_bias(
        _lib.dtype_code(x.dtype), _lib.dtype_code(odt), x.data_ptr(), x.stride(0),
        weight.data_ptr(), weight.stride(0), colsum.data_ptr(),
        bias.data_ptr() if bias is not None else 0, float(eps), stats.data_ptr(), out.data_ptr(),
        out.stride(0), M, N, K, _lib.EPI_GELU if gelu else 0, _stream(x))
    _lib.check("mi355_layernorm_gemm_bias", st)
    return out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: Optional[torch.Tensor] = None,
              scale: Optional[float] = None, causal: bool = False,
              key_valid: Optional[torch.Tensor] = None,
              key_bound: Optional[bool] = None,
              workspace: Optional[torch.Tensor] = None, bounds_ready: bool = False,
              causal_sweep_min_keys: Optional[int] = None) -> torch.Tensor:
    """Streamed softmax attention over ``[B, S, H, head_dim]`` views (unit head_dim stride).

    ``out`` defaults to a new contiguous ``[B, S_q, H, head_dim]`` tensor, whose
    ``view(B, S_q, H * head_dim)`` is the merged-head context of the reference block.
    ``key_valid`` is an optional ``[B, S_k]`` bool mask of keys to attend to.
    ``key_bound`` selects the key-norm bound pass of the matrix-core kernel (a workspace of
    per-chunk max |k| that lets waves skip the per-tile row maxima, and of the offset sweep's
    redo flags): None = the library's choice (``mi355_attn_workspace_bytes``: long key
    ranges), True = always (``mi355_attn_workspace_bytes_forced``), False = never. With the
    workspace, a key mask is resolved on the device: work-groups whose keys are all valid run
    the unmasked sweeps, the others a second, key-masked launch; nothing synchronises the host.
    ``workspace`` (``attention_workspace``) supplies the workspace instead, with
    ``bounds_ready`` when a QKV projection already wrote the bounds into it
    (``KeyBoundTarget``) and ``causal_sweep_min_keys`` the key range from which causal query
    tiles take the sweeps (``mi355_attn_fwd_kb``; default 32768, the library's choice).
    """
    _on_gpu(q, k, v, out, key_valid)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k, v must be 4-D [B, S, H, head_dim] views")
    B, Sq, H, D = q.shape
    Bk, Sk, Hk, Dk = k.shape
    if (Bk, Hk, Dk) != (B, H, D) or tuple(v.shape) != (B, Sk, H, D):
        raise ValueError(f"shape mismatch q={tuple(q.shape)} k={tuple(k.shape)} v={tuple(v.shape)}")
    dt = q.dtype
    if k.dtype != dt or v.dtype != dt:
        raise TypeError("q, k, v must share one dtype")
    if q.stride(3) != 1 or k.stride(3) != 1 or v.stride(3) != 1:
        raise ValueError("head_dim must be the unit-stride dimension")
    if out is None:
        out = torch.empty((B, Sq, H, D), device=q.device, dtype=dt)
    elif tuple(out.shape) != (B, Sq, H, D) or out.dtype != dt or out.stride(3) != 1:
        raise ValueError("out must be [B, S_q, H, head_dim] of q's dtype with unit head_dim stride")
    if scale is None:
        scale = D ** -0.5
    kv_ptr, kv_sb = 0, 0
    if key_valid is not None:
        kv_ptr = _mask_ptr(key_valid, (B, Sk))
        kv_sb = key_valid.stride(0)
    L = _lib
    code = L.dtype_code(dt)
    if workspace is not None or bounds_ready or causal_sweep_min_keys is not None:
        if workspace is None:
            raise ValueError("bounds_ready / causal_sweep_min_keys need a workspace")
        _on_gpu(q, workspace)
        if workspace.dtype != torch.uint8 or workspace.dim() != 1:
            raise ValueError("workspace must be a 1-D uint8 tensor")
        need = L.lib().mi355_attn_workspace_bytes_forced(code, B, H, Sq, Sk, D)
        if workspace.numel() < need:
            raise ValueError(f"workspace holds {workspace.numel()} bytes, {need} needed")
        gate = 32768 if causal_sweep_min_keys is None else int(causal_sweep_min_keys)
        st = L.lib().mi355_attn_fwd_kb(
            code, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), B, H, Sq, Sk, D,
            L.i64_array((q.stride(0), q.stride(1), q.stride(2))),
            L.i64_array((k.stride(0), k.stride(1), k.stride(2))),
            L.i64_array((v.stride(0), v.stride(1), v.stride(2))),
            L.i64_array((out.stride(0), out.stride(1), out.stride(2))),
            float(scale), 1 if causal else 0, kv_ptr, kv_sb,
            workspace.data_ptr() if need > 0 else 0, workspace.numel() if need > 0 else 0,
            1 if (bounds_ready and need > 0) else 0, gate, _stream(q))
        L.check("mi355_attn_fwd_kb", st)
        return out
    if key_bound is None:
        ws_bytes = L.lib().mi355_attn_workspace_bytes(code, B, H, Sq, Sk, D)
    elif key_bound:
        ws_bytes = L.lib().mi355_attn_workspace_bytes_forced(code, B, H, Sq, Sk, D)
    else:
        ws_bytes = 0
    args = (code, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), B, H, Sq, Sk, D,
            L.i64_array((q.stride(0), q.stride(1), q.stride(2))),
            L.i64_array((k.stride(0), k.stride(1), k.stride(2))),
            L.i64_array((v.stride(0), v.stride(1), v.stride(2))),
            L.i64_array((out.stride(0), out.stride(1), out.stride(2))),
            float(scale), 1 if causal else 0, kv_ptr, kv_sb)
    if ws_bytes > 0:
        ws = torch.empty((ws_bytes,), device=q.device, dtype=torch.uint8)
        st = L.lib().mi355_attn_fwd_ws(*args, ws.data_ptr(), ws_bytes, _stream(q))
        L.check("mi355_attn_fwd_ws", st)
    else:
        st = L.lib().mi355_attn_fwd(*args, _stream(q))
        L.check("mi355_attn_fwd", st)
    return out


# d_model that block_head takes: the packed QKV weight resident in LDS
BLOCK_HEAD_SIZES = frozenset((32, 64, 128))
# ... and the rows from which it pays: every CU's work-group stages the whole weight (96 KB at d
# 128) for its rows, which on 8192 rows cost more than the launch saved (4-layer model 162 -> 178 us);
# from 65536 rows on a work-group per CU walks them (a layer of d 128: 108 -> 73 us there)
BLOCK_HEAD_MIN_ROWS = 65536


def block_head(x: torch.Tensor, norm_w: Optional[torch.Tensor], norm_b: Optional[torch.Tensor],
               eps: float, w_qkv: torch.Tensor, b_qkv: Optional[torch.Tensor]) -> torch.Tensor:
    """``linear(layer_norm(x), w_qkv, b_qkv)`` with fp16 operands of a narrow block in one launch:
    ``x`` ([M, d], fp32 or fp16, unit column stride) gives fp16 [M, 3 d]; the normalised rows are
    rounded to fp16 as ``layer_norm`` with an fp16 output rounds them. ``w_qkv`` is contiguous fp16
    [3 d, d], ``b_qkv`` fp32, the norm's parameters of x's type; d must be in
    ``BLOCK_HEAD_SIZES``."""
    _on_gpu(x, norm_w, norm_b, w_qkv, b_qkv)
    if x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("block_head expects a 2-D x with unit column stride")
    M, d = x.shape
    if x.dtype not in (torch.float32, torch.float16):
        raise TypeError("x must be fp32 or fp16")
    if tuple(w_qkv.shape) != (3 * d, d) or w_qkv.dtype != torch.float16 or not w_qkv.is_contiguous():
        raise ValueError(f"w_qkv must be contiguous fp16 [{3 * d}, {d}]")
    for t, n, dt in ((b_qkv, 3 * d, torch.float32), (norm_w, d, x.dtype), (norm_b, d, x.dtype)):
        if t is not None and (tuple(t.shape) != (n,) or t.dtype != dt or not t.is_contiguous()):
            raise ValueError("b_qkv must be contiguous fp32 and the norm's parameters of x's dtype")
    y = torch.empty((M, 3 * d), device=x.device, dtype=torch.float16)

    def ptr(t):
        return t.data_ptr() if t is not None else 0

    st = _lib.lib().mi355_block_head(_lib.dtype_code(x.dtype), x.data_ptr(), x.stride(0), ptr(norm_w),
                                     ptr(norm_b), float(eps), w_qkv.data_ptr(), ptr(b_qkv),
                                     y.data_ptr(), y.stride(0), M, d, _stream(x))
    _lib.check("mi355_block_head", st)
    return y


# (d_model, ffn_dim) that block_tail takes: three fp16 weight matrices resident in LDS
BLOCK_TAIL_SIZES = frozenset(((32, 32), (32, 64), (32, 128), (64, 64), (64, 128), (128, 64),
                              (128, 128)))


def block_tail(ctx: torch.Tensor, x: torch.Tensor, w_o: torch.Tensor, b_o: Optional[torch.Tensor],
               norm_w: Optional[torch.Tensor], norm_b: Optional[torch.Tensor], eps: float,
               w_in: torch.Tensor, b_in: Optional[torch.Tensor], w_out: torch.Tensor,
               b_out: Optional[torch.Tensor],
               row_valid: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The row-local rest of a narrow block after its attention, in one launch: ``x1 = x +
    linear(ctx, w_o, b_o)`` (masked rows x), then ``x1 + linear(gelu(linear(layer_norm(x1), w_in,
    b_in)), w_out, b_out)`` with masked rows 0, rounded where ``linear`` / ``layer_norm`` with fp16
    operands round. ``ctx`` ([M, d] fp16, unit column stride) and the weights are fp16, the biases
    fp32, ``x`` ([M, d]), ``norm_w`` and ``norm_b`` of one type, fp32 or fp16. (d, ffn) must be in
    ``BLOCK_TAIL_SIZES``."""
    _on_gpu(ctx, x, w_o, b_o, norm_w, norm_b, w_in, b_in, w_out, b_out, row_valid)
    if ctx.dim() != 2 or x.dim() != 2 or ctx.shape != x.shape:
        raise ValueError("block_tail expects 2-D ctx and x of one shape")
    M, d = x.shape
    ffn = w_in.shape[0]
    for t, shape in ((w_o, (d, d)), (w_in, (ffn, d)), (w_out, (d, ffn))):
        if tuple(t.shape) != shape or t.dtype != torch.float16 or not t.is_contiguous():
            raise ValueError(f"weights must be contiguous fp16, [{d}, {d}], [ffn, {d}], [{d}, ffn]")
    if ctx.dtype != torch.float16 or x.dtype not in (torch.float32, torch.float16):
        raise TypeError("ctx must be fp16 and x fp32 or fp16")
    if ctx.stride(1) != 1 or x.stride(1) != 1:
        raise ValueError("ctx and x need unit column stride")
    for t, n, dt in ((b_o, d, torch.float32), (b_in, ffn, torch.float32), (b_out, d, torch.float32),
                     (norm_w, d, x.dtype), (norm_b, d, x.dtype)):
        if t is not None and (tuple(t.shape) != (n,) or t.dtype != dt or not t.is_contiguous()):
            raise ValueError("biases must be contiguous fp32 and the norm's parameters of x's dtype")
    y = torch.empty((M, d), device=x.device, dtype=x.dtype)

    def ptr(t):
        return t.data_ptr() if t is not None else 0

    st = _lib.lib().mi355_block_tail(
        _lib.dtype_code(x.dtype), ctx.data_ptr(), ctx.stride(0), x.data_ptr(), x.stride(0),
        y.data_ptr(), y.stride(0), w_o.data_ptr(), ptr(b_o), ptr(norm_w), ptr(norm_b), float(eps),
        w_in.data_ptr(), ptr(b_in), w_out.data_ptr(), ptr(b_out), M, d, ffn,
        _mask_ptr(row_valid, (M,)), _stream(x))
    _lib.check("mi355_block_tail", st)
    return y


def quant_rows_i8(x: torch.Tensor, mode: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-row symmetric int8 quantisation; returns ``(q [M, K] int8, scale [M] fp32)``.

    mode 0 is the activation recipe (scale = max(amax, 1e-6) / 127), mode 1 the weight recipe
    (scale = max(amax / 127, 1e-8)).
    """
    _on_gpu(x)
    if x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("quant_rows_i8 expects a 2-D tensor with unit column stride")
    M, K = x.shape
    q = torch.empty((M, K), device=x.device, dtype=torch.int8)
    s = torch.empty((M,), device=x.device, dtype=torch.float32)
    st = _lib.lib().mi355_quant_rows_i8(_lib.dtype_code(x.dtype), x.data_ptr(), x.stride(0),
                                        q.data_ptr(), s.data_ptr(), M, K, int(mode), _stream(x))
    _lib.check("mi355_quant_rows_i8", st)
    return q, s


def linear_i8(a: torch.Tensor, w: torch.Tensor, s_a: torch.Tensor, s_w: torch.Tensor,
              bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float16,
              out: Optional[torch.Tensor] = None, acc_out: Optional[torch.Tensor] = None,
              row_valid: Optional[torch.Tensor] = None, want_out: bool = True,
              residual: Optional[torch.Tensor] = None, gelu: bool = False,
              zero_masked_rows: bool = False) -> Optional[torch.Tensor]:
    """W8A8 projection: ``y = fp32(a @ w^T) * (s_a[:, None] * s_w[None, :]) + bias``.

    ``a`` is ``[M, K]`` int8, ``w`` is ``[N, K]`` int8 (K-major), scales fp32. ``acc_out``
    (``[M, N]`` int32) receives the raw int32 accumulators when given. Epilogues of the int8
    transformer block (k008_int8_gemm.py:221-233), each computed in fp32 from y rounded to
    ``out_dtype`` and rounded once: ``gelu`` gives gelu(y); ``residual`` ([M, N] of out_dtype,
    may be ``out``) gives residual + y with masked rows keeping the residual, or zeroed with
    ``zero_masked_rows``. The epilogues do not combine with ``acc_out``.
    """
    _on_gpu(a, w, s_a, s_w, bias, out, acc_out, row_valid, residual)
    if a.dtype != torch.int8 or w.dtype != torch.int8:
        raise TypeError("a and w must be int8")
    if not a.is_contiguous() or not w.is_contiguous():
        raise ValueError("a and w must be contiguous")
    M, K = a.shape
    N, K2 = w.shape
    if K2 != K:
        raise ValueError("inner sizes differ")
    if s_a.shape != (M,) or s_w.shape != (N,) or s_a.dtype != torch.float32 or s_w.dtype != torch.float32:
        raise ValueError("s_a [M] and s_w [N] must be fp32")
    if bias is not None and (bias.shape != (N,) or bias.dtype != torch.float32):
        raise ValueError("bias must be fp32 [N]")
    if acc_out is not None and (acc_out.shape != (M, N) or acc_out.dtype != torch.int32
                                or not acc_out.is_contiguous()):
        raise ValueError("acc_out must be a contiguous int32 [M, N] tensor")
    epilogue = gelu or residual is not None or zero_masked_rows
    if epilogue and acc_out is not None:
        raise ValueError("acc_out does not combine with the gelu / residual epilogues")
    if zero_masked_rows and residual is None:
        raise ValueError("zero_masked_rows needs a residual")
    if gelu and residual is not None:
        raise ValueError("gelu does not combine with a residual")
    if residual is not None and (residual.shape != (M, N) or residual.dtype != out_dtype
                                 or residual.stride(1) != 1):
        raise ValueError("residual must be [M, N] of out_dtype with unit column stride")
    if (want_out or epilogue) and out is None:
        out = torch.empty((M, N), device=a.device, dtype=out_dtype)
    if out is not None and (out.shape != (M, N) or out.dtype != out_dtype or out.stride(1) != 1):
        raise ValueError("out must be [M, N] of out_dtype with unit column stride")
    mask = _mask_ptr(row_valid, (M,))
    if epilogue:
        flags = (_lib.EPI_GELU if gelu else 0) | (_lib.EPI_ZERO_MASKED if zero_masked_rows else 0)
        st = _lib.lib().mi355_gemm_i8_epilogue(
            a.data_ptr(), w.data_ptr(), s_a.data_ptr(), s_w.data_ptr(),
            bias.data_ptr() if bias is not None else 0, _lib.dtype_code(out_dtype),
            out.data_ptr(), out.stride(0),
            residual.data_ptr() if residual is not None else 0,
            residual.stride(0) if residual is not None else N, M, N, K, mask, flags, _stream(a))
        _lib.check("mi355_gemm_i8_epilogue", st)
        return out
    st = _lib.lib().mi355_gemm_i8(
        a.data_ptr(), w.data_ptr(), s_a.data_ptr(), s_w.data_ptr(),
        bias.data_ptr() if bias is not None else 0, _lib.dtype_code(out_dtype),
        out.data_ptr() if out is not None else 0, out.stride(0) if out is not None else N,
        acc_out.data_ptr() if acc_out is not None else 0, M, N, K,
        mask, _stream(a))
    _lib.check("mi355_gemm_i8", st)
    return out


# head dims of attention_packed and attention_shared_prefix
GROUPED_HEAD_DIMS = (16, 32, 48, 64, 80, 96, 128, 192, 256)

# The operators below are called for single tokens, where a call's time is the host's. What their checks
# look at (shapes, strides, types) is checked once per combination: the checks are cached functions of
# those numbers alone, which also return the arguments made from them. Pointers, devices and gradients are
# looked at in every call.
_SIXTEEN_BIT = (torch.float16, torch.bfloat16)
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


class _Arrays(tuple):
    """int64 arrays of strides for the library."""
    def __new__(cls, *strides):
        return super().__new__(cls, [_lib.i64_array(st) for st in strides])


def _launch(device: int, fn, *args) -> int:
    """Calls a library entry point with ``device``'s current stream as the last argument and that
    device current."""
    if _current_device() == device:
        return fn(*args, _raw_stream(device))
    with torch.cuda.device(device):
        return fn(*args, _raw_stream(device))


def _capturing(device: int) -> bool:
    """Whether ``device``'s current stream is being captured."""
    if _current_device() == device:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _no_backward(*tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and t.requires_grad:
            raise ValueError("this operator has no backward pass: call it under torch.no_grad() "
                             "or with detached tensors")


def _no_tangent(*tensors: Optional[torch.Tensor]) -> None:
    """(called inside a forward-mode level, which no_grad does not turn off)"""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError("this operator has no forward-mode derivative: call it with unpacked tensors")


def _rows_strides(name: str, shape, stride, align: int, kv_axis: Optional[int] = None,
                  written: bool = False) -> Tuple[int, ...]:
    """Strides of a [..., token, head, head_dim] view but the last, checked: unit head_dim stride, whole
    vectors between rows, for K / V (kv_axis: the token axis) tokens that do not overlap, and for what is
    written no rows that do. Axes of one element get a stride that does not matter."""
    if 0 in shape:
        return tuple(shape[-1] if i == kv_axis else 0 for i in range(len(shape) - 1))
    if stride[-1] != 1:
        raise ValueError(f"head_dim must be the unit-stride dimension of {name}")
    out = []
    for i, (n, st) in enumerate(zip(shape[:-1], stride[:-1])):
        if n == 1:
            st = shape[-1] if i == kv_axis else 0
        elif st % align:
            raise ValueError(f"{name} needs strides that are multiples of {align} elements, got {tuple(stride)}")
        elif i == kv_axis and not shape[-1] <= st <= 1 << 24:
            raise ValueError(f"the tokens of {name} overlap or are too far apart (stride {st})")
        out.append(st)
    if written:  # no two elements in one place
        extent = shape[-1]
        for st, n in sorted((st, n) for n, st in zip(shape[:-1], stride[:-1]) if n > 1):
            if st < extent:
                raise ValueError(f"rows of {name} overlap (strides {tuple(stride)})")
            extent = st * n
    return tuple(out)


def _check_aligned(**pointers: int) -> None:
    for name, ptr in pointers.items():
        if ptr % (8 if name == "out" else 16):
            raise ValueError(f"{name} must start at a multiple of {8 if name == 'out' else 16} bytes")


def _scale(scale: Optional[float], head_dim: int) -> float:
    scale = head_dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale <= 1e30:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


@functools.lru_cache(maxsize=2048)
def _bytes(shape, stride, dtype) -> int:
    """From a view's first to behind its last byte."""
    if 0 in shape:
        return 0
    return (1 + sum((n - 1) * st for n, st in zip(shape, stride))) * dtype.itemsize


def _check_apart(out: torch.Tensor, *inputs: Optional[torch.Tensor]) -> None:
    """Refuses an ``out`` whose bytes (first to last) meet an input's."""
    lo = out.data_ptr()
    hi = lo + _bytes(out.shape, out.stride(), out.dtype)
    for t in inputs:
        if t is not None:
            start = t.data_ptr()
            if start < hi and lo < start + _bytes(t.shape, t.stride(), t.dtype):
                raise ValueError("out shares memory with an input")


@dataclass(frozen=True, eq=False)
class PackedPlan:
    """How ``attention_packed`` walks one batch of packed sequences (``packed_plan``). It holds for
    every call with these lengths (all layers of a model), on any stream of its device. It may be dropped
    while such calls are under way, but a captured graph reads ``tiles`` in every replay: like the graph's
    inputs, its plan has to be kept as long as the graph."""
    q_tokens: int
    k_tokens: int
    heads: int
    kv_heads: int
    head_dim: int
    causal: bool
    tile_rows: int
    counts: ctypes.Array  # tiles of tile_rows rows, of 32 rows, joins, partial rows
    tiles: torch.Tensor
    workspace_bytes: int
    stream: int = 0  # (raw) that tiles were allocated on

    def used_on(self, device: int) -> None:
        """Tells the allocator of a call on ``device``'s current stream where that is not the tiles' own: the
        block is not handed out again before what the stream holds by then is done. Not while capturing:
        the call's replays come at times that nobody knows here."""
        if _raw_stream(device) != self.stream and not _capturing(device):
            self.tiles.record_stream(torch.cuda.current_stream(device))


def packed_plan(q_lens: Sequence[int], k_lens: Optional[Sequence[int]] = None, *, heads: int,
                kv_heads: Optional[int] = None, head_dim: int, causal: bool = True,
                device="cuda") -> PackedPlan:
    """Plans ``attention_packed`` over sequences of ``q_lens`` new tokens against ``k_lens`` keys
    each (default: the same lengths). Lengths are host integers (0 included). Made once per batch,
    outside a graph capture: it lays the tiles out on the host and copies them to ``device``, and waits for the
    copy (30 us for a few sequences, 80 for hundreds). A captured graph's plan has to be kept as long as the graph."""
    kv_heads = heads if kv_heads is None else kv_heads
    q_lens = [operator.index(n) for n in q_lens]
    k_lens = q_lens if k_lens is None else [operator.index(n) for n in k_lens]
    if len(q_lens) != len(k_lens):
        raise ValueError(f"{len(q_lens)} query lengths and {len(k_lens)} key lengths")
    if any(not 0 <= n < 1 << 30 for n in q_lens + k_lens):
        raise ValueError("lengths must be between 0 and 2^30")
    if heads <= 0 or kv_heads <= 0 or heads % kv_heads:
        raise ValueError(f"{heads} query heads cannot share {kv_heads} K/V heads evenly")
    if head_dim not in GROUPED_HEAD_DIMS:
        raise ValueError(f"head_dim {head_dim} is not one of {GROUPED_HEAD_DIMS}")
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError(f"expected a GPU device, got {device}")
    n = len(q_lens)
    arr = ctypes.c_int32 * max(n, 1)
    ql, kl = arr(*q_lens), arr(*k_lens)
    counts, rows = _lib.i64_array((0, 0, 0, 0)), ctypes.c_int32(0)

    def plan(tiles: int, capacity: int) -> None:
        st = _lib.lib().mi355_attn_packed_plan(ql, kl, n, heads, kv_heads, head_dim, int(causal), tiles,
                                               capacity, counts, ctypes.byref(rows))
        _lib.check("mi355_attn_packed_plan", st)

    plan(0, 0)
    tiles = torch.empty((sum(counts[:3]), 8), dtype=torch.int32)
    if tiles.numel():
        plan(tiles.data_ptr(), tiles.shape[0])
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    on_gpu = tiles.to(device)  # (from pageable memory: there when this returns, for every stream)
    return PackedPlan(sum(q_lens), sum(k_lens), heads, kv_heads, head_dim, bool(causal), rows.value,
                      counts, on_gpu, counts[3] * kv_heads * (head_dim + 2) * 4, _raw_stream(device.index))


@functools.lru_cache(maxsize=512)
def _packed_views(q_tokens, k_tokens, heads, kv_heads, D, dtypes, qs, qst, ks, kst, vs, vst, os, ost):
    """(library type code, stride arrays) of attention_packed's tensors, checked."""
    if dtypes[0] not in _SIXTEEN_BIT:
        raise TypeError(f"q must be fp16 or bf16, got {dtypes[0]}")
    if len(set(dtypes)) > 1:
        raise TypeError(f"q, k, v and out must share one dtype, got {dtypes}")
    for name, shape, tokens, h in (("q", qs, q_tokens, heads), ("k", ks, k_tokens, kv_heads), ("v", vs, k_tokens, kv_heads)):
        if len(shape) != 3 or shape[0] < tokens or tuple(shape[1:]) != (h, D):
            raise ValueError(f"the plan needs {name} [{tokens} or more, {h}, {D}], got {tuple(shape)}")
    if os is not None and os != qs:
        raise ValueError(f"out must have q's shape {tuple(qs)}")
    arrays = _Arrays(_rows_strides("q", qs, qst, 8), _rows_strides("k", ks, kst, 8, 0), _rows_strides("v", vs, vst, 8, 0),
                     (heads * D, D) if os is None else _rows_strides("out", os, ost, 4, written=True))
    return _lib.dtype_code(dtypes[0]), arrays


def attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PackedPlan,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax attention of packed sequences with grouped heads: ``q`` ``[q_tokens, heads, head_dim]``,
    ``k`` and ``v`` ``[k_tokens, kv_heads, head_dim]`` (fp16 or bf16), sequence after sequence with
    the lengths of ``plan``; query head h reads K/V head ``h // (heads // kv_heads)``.

    With a causal plan, token i of a sequence's n sees its first ``k_len - n + i + 1`` keys (the last
    token sees them all); otherwise every token sees all keys of its sequence. A token that sees no
    key gives zeros, and a key that a token does not see never reaches it, NaN and infinities in its
    K or V included. ``out`` (default: a new contiguous tensor) must not share memory with the inputs;
    rows behind the plan's tokens (``q`` and ``out`` may have more) are left as they are, zeros in a new
    ``out``. fp32 statistics; probabilities are rounded to the input type in tiles of more than 32 rows, and held in
    twice its bits in smaller ones. No derivatives."""
    dev = q.get_device()
    if dev < 0 or k.get_device() != dev or v.get_device() != dev or plan.tiles.get_device() != dev or (
            out is not None and out.get_device() != dev):
        _on_gpu(q, k, v, plan.tiles, out)
    given = out is not None
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (given and out.requires_grad)):
        _no_backward(q, k, v, out)
    if forward_ad._current_level >= 0:
        _no_tangent(q, k, v, out)
    code, (qst, kst, vst, ost) = _packed_views(
        plan.q_tokens, plan.k_tokens, plan.heads, plan.kv_heads, plan.head_dim,
        (q.dtype, k.dtype, v.dtype, out.dtype) if given else (q.dtype, k.dtype, v.dtype),
        q.shape, q.stride(), k.shape, k.stride(), v.shape, v.stride(), out.shape if given else None,
        out.stride() if given else None)
    scale = _scale(scale, plan.head_dim)
    if given:
        _check_apart(out, q, k, v)
    else:  # (rows behind the last token have no value)
        out = q.new_empty(q.shape) if q.shape[0] == plan.q_tokens else q.new_zeros(q.shape)
    if plan.tiles.shape[0] == 0:
        return out
    qp, kp, vp, op = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    if (qp | kp | vp) & 15 or op & 7:
        _check_aligned(q=qp, k=kp, v=vp, out=op)
    plan.used_on(dev)
    need = plan.workspace_bytes
    ws = torch.empty((need,), device=q.device, dtype=torch.uint8) if need else None
    st = _launch(dev, _lib.lib().mi355_attn_packed, code, qp, kp, vp, op, plan.heads, plan.kv_heads,
                 plan.head_dim, qst, kst, vst, ost, scale, plan.causal, plan.tiles.data_ptr(), plan.counts,
                 plan.tile_rows, ws.data_ptr() if need else 0, need)
    if st:
        _lib.check("mi355_attn_packed", st)
    return out


@functools.lru_cache(maxsize=512)
def _prefix_views(dtypes, qs, qst, kps, kpst, vps, vpst, kos, kost, vos, vost, lens_dtype, lens_shape, os, ost):
    """(type code, sizes, stride arrays, workspace bytes) of attention_shared_prefix's tensors, checked."""
    if dtypes[0] not in _SIXTEEN_BIT:
        raise TypeError(f"q must be fp16 or bf16, got {dtypes[0]}")
    if len(set(dtypes)) > 1:
        raise TypeError(f"q, K, V and out must share one dtype, got {dtypes}")
    if len(qs) != 4 or len(kps) != 3 or len(kos) != 4:
        raise ValueError("q is [B, n, heads, head_dim], the prefix [P, kv_heads, head_dim], the caches "
                         "[B, room, kv_heads, head_dim]")
    B, n, H, D = qs
    P, Hkv = kps[:2]
    room = kos[1]
    if D not in GROUPED_HEAD_DIMS:
        raise ValueError(f"head_dim {D} is not one of {GROUPED_HEAD_DIMS}")
    if H == 0 or Hkv == 0 or H % Hkv:
        raise ValueError(f"{H} query heads cannot share {Hkv} K/V heads evenly")
    if tuple(kps) != (P, Hkv, D) or vps != kps or tuple(kos) != (B, room, Hkv, D) or vos != kos:
        raise ValueError(f"shape mismatch q={tuple(qs)} prefix={tuple(kps)}, {tuple(vps)} own={tuple(kos)}, {tuple(vos)}")
    if lens_dtype != torch.int32 or tuple(lens_shape) != (B,):
        raise ValueError(f"own_lens must be an int32 tensor of shape ({B},)")
    if os is not None and os != qs:
        raise ValueError(f"out must have q's shape {tuple(qs)}")
    arrays = _Arrays(_rows_strides("q", qs, qst, 8), _rows_strides("k_prefix", kps, kpst, 8, 0),
                     _rows_strides("v_prefix", vps, vpst, 8, 0), _rows_strides("k_own", kos, kost, 8, 1),
                     _rows_strides("v_own", vos, vost, 8, 1),
                     (n * H * D, H * D, D) if os is None else _rows_strides("out", os, ost, 4, written=True))
    need = _lib.lib().mi355_attn_shared_prefix_workspace_bytes(B, n, H, Hkv, D, P, room)
    if need < 0:
        _lib.check("mi355_attn_shared_prefix_workspace_bytes", need)
    return _lib.dtype_code(dtypes[0]), (B, n, H, Hkv, D, P, room), arrays, need


def attention_shared_prefix(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor,
                            k_own: torch.Tensor, v_own: torch.Tensor, own_lens: torch.Tensor,
                            scale: Optional[float] = None,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of a batch's newest tokens when all its sequences start with the same prefix, which
    is read once for all of them: ``q`` ``[B, n, heads, head_dim]`` (n = 1 when generating) against
    ``k_prefix`` / ``v_prefix`` ``[P, kv_heads, head_dim]`` and each sequence's own cache ``k_own`` /
    ``v_own`` ``[B, room, kv_heads, head_dim]``, of which the first ``own_lens[b]`` tokens (int32, on
    the GPU) are filled, the n newest at their end. Token i of the n sees the whole prefix and the
    first ``own_lens[b] - n + i + 1`` own keys; a token that sees no key gives zeros.

    Made for a few new tokens: a cache is read once for every 32 (token, head of a K/V head's group) rows; a prompt
    behind a prefix is ``attention_packed``'s.

    ``own_lens`` is read by the kernels, so a captured graph follows its values; it is clamped to
    [0, room], and what a cache holds behind it does not matter. Types, head dims and roundings as
    ``attention_packed``. ``out`` must not share memory with the inputs. No derivatives."""
    dev = q.get_device()
    given = out is not None
    if dev < 0 or k_prefix.get_device() != dev or v_prefix.get_device() != dev or k_own.get_device() != dev or (
            v_own.get_device() != dev or own_lens.get_device() != dev or (given and out.get_device() != dev)):
        _on_gpu(q, k_prefix, v_prefix, k_own, v_own, own_lens, out)
    if torch.is_grad_enabled():
        _no_backward(q, k_prefix, v_prefix, k_own, v_own, out)
    if forward_ad._current_level >= 0:
        _no_tangent(q, k_prefix, v_prefix, k_own, v_own, out)
    dt = q.dtype
    dtypes = (dt, k_prefix.dtype, v_prefix.dtype, k_own.dtype, v_own.dtype)
    code, sizes, strides, need = _prefix_views(
        dtypes + (out.dtype,) if given else dtypes, q.shape, q.stride(), k_prefix.shape, k_prefix.stride(),
        v_prefix.shape, v_prefix.stride(), k_own.shape, k_own.stride(), v_own.shape, v_own.stride(),
        own_lens.dtype, own_lens.shape, out.shape if given else None, out.stride() if given else None)
    if not own_lens.is_contiguous():
        raise ValueError("own_lens must be contiguous")
    scale = _scale(scale, sizes[4])
    if given:
        _check_apart(out, q, k_prefix, v_prefix, k_own, v_own, own_lens)
    else:
        out = q.new_empty(q.shape)
    if out.numel() == 0:
        return out
    qp, op = q.data_ptr(), out.data_ptr()
    kp, vp, ko, vo = k_prefix.data_ptr(), v_prefix.data_ptr(), k_own.data_ptr(), v_own.data_ptr()
    if (qp | kp | vp | ko | vo) & 15 or op & 7:
        _check_aligned(q=qp, k_prefix=kp, v_prefix=vp, k_own=ko, v_own=vo, out=op)
    ws = torch.empty((need,), device=q.device, dtype=torch.uint8) if need else None
    st = _launch(dev, _lib.lib().mi355_attn_shared_prefix, code, qp, kp, vp, ko, vo, own_lens.data_ptr(), op,
                 *sizes, *strides, scale, ws.data_ptr() if need else 0, need)
    if st:
        _lib.check("mi355_attn_shared_prefix", st)
    return out


# group sizes of linear_i4
I4_GROUPS = (32, 64, 128)


def _group_scale(step: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Scales for ``step``, rounded to ``dtype``: to the nearest, but upwards below its least normal number, where
    a step rounded down would leave a group's ends out of reach by whole steps, and at least its least number
    (groups of zeros)."""
    info = torch.finfo(dtype)
    least = info.tiny * info.eps
    up = ((step.double() / least).ceil().clamp_min(1) * least).float()
    return torch.where(step < info.tiny, up, step).to(dtype)


def quant_groups_i4(w: torch.Tensor, group: int = 128, symmetric: bool = False
                    ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """4-bit weights for ``linear_i4`` from ``w`` ``[N, K]`` (fp16 or bf16): ``(q, scale, zero)`` with
    ``w ~ scale[n, k / group] (q[n, k] - zero[n, k / group])``, q two to a byte (even k in the low
    half) ``[N, K / 2]`` uint8, scale of w's type. Each group's range (0 included) goes to 0 .. 15, or with
    ``symmetric`` its largest magnitude to +-7 around 8 (zero is None). Run once per weight: it waits for the GPU to see that
    all of it is finite."""
    if w.dim() != 2 or w.dtype not in _SIXTEEN_BIT:
        raise ValueError("quant_groups_i4 expects a 2-D fp16 or bf16 weight")
    if group not in I4_GROUPS or w.shape[1] % group or w.shape[1] == 0:
        raise ValueError(f"group must be one of {I4_GROUPS} and divide K = {w.shape[1]}")
    with torch.no_grad():
        x = w.detach().float().reshape(w.shape[0], w.shape[1] // group, group)
        if symmetric:
            scale = _group_scale(x.abs().amax(2) / 7, w.dtype)
        else:
            lo, hi = x.amin(2).clamp_max(0), x.amax(2).clamp_min(0)
            scale = _group_scale((hi - lo) / 15, w.dtype)
        if not bool(torch.isfinite(scale).all()):
            raise ValueError("quant_groups_i4 needs finite weights, of which a group's range is finite in fp32")
        if symmetric:
            zero, z = None, 8.0
        else:
            z = (-lo / scale.float()).round().clamp(0, 15)
            zero, z = z.to(torch.uint8), z[..., None]
        q = ((x / scale.float()[..., None]).round() + z).clamp(0, 15).to(torch.uint8).reshape(w.shape)
        return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), scale, zero


@functools.lru_cache(maxsize=512)
def _i4_views(xd, xs, xst, wd, ws, sd, ss, zd, zs, bd, bs, odt, os, ost):
    """(type codes, M, N, K, group, ldx, ldy) of linear_i4's tensors, checked."""
    if xd not in _SIXTEEN_BIT:
        raise TypeError(f"x must be fp16 or bf16, got {xd}")
    if len(xs) != 2 or len(ws) != 2 or len(ss) != 2:
        raise ValueError("linear_i4 expects 2-D x, w and scale")
    (M, K), N = xs, ws[0]
    if wd != torch.uint8 or ws[1] * 2 != K:
        raise ValueError(f"w must be a uint8 tensor of shape (N, {K // 2}) for K = {K}, got {tuple(ws)}")
    group = K // ss[1] if ss[1] else 0
    if group not in I4_GROUPS or tuple(ss) != (N, K // group) or K % group:
        raise ValueError(f"scale must be [N, K / group] with a group of {I4_GROUPS}, got {tuple(ss)}")
    if sd != xd:
        raise TypeError(f"scale is {sd}, x is {xd}")
    if zs is not None and (zd != torch.uint8 or zs != ss):
        raise ValueError("zero must be a uint8 tensor of scale's shape")
    if bs is not None and (tuple(bs) != (N,) or bd != torch.float32):
        raise ValueError(f"bias must be an fp32 tensor of shape ({N},)")
    ldx = xst[0] if M > 1 else (K + 7) // 8 * 8
    if M and (xst[1] != 1 or ldx < K or ldx % 8):
        raise ValueError("x needs unit column stride and a row stride that is a multiple of 8 and holds a row")
    if odt not in (xd, torch.float32):
        raise TypeError(f"out_dtype must be {xd} or float32, got {odt}")
    ldy = N
    if os is not None:
        if tuple(os) != (M, N) or (M and N > 1 and ost[1] != 1) or (M > 1 and ost[0] < N):
            raise ValueError("out must be [M, N] of out_dtype with unit column stride")
        ldy = ost[0] if M > 1 else N
    return _lib.dtype_code(xd), _lib.dtype_code(odt), M, N, K, group, ldx, ldy


def linear_i4(x: torch.Tensor, w: torch.Tensor, scale: torch.Tensor,
              zero: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
              out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Projection of a few rows with 4-bit weights: ``x @ W^T + bias`` with
    ``W[n, k] = scale[n, k / group] (q[n, k] - zero[n, k / group])``.

    ``x`` is ``[M, K]`` fp16 or bf16 (row-strided, unit column stride); ``w`` ``[N, K / 2]`` uint8 holds
    q two to a byte, the even k in the low half; ``scale`` ``[N, K / group]`` is of x's type, group 32,
    64 or 128; ``zero`` uint8 of scale's shape (None: 8); ``bias`` fp32 ``[N]``. Made for M of a few
    rows (the weights are read again for every 64). fp32 sums, the output (x's type, or fp32 with
    ``out_dtype``) rounded once. Infinities in x give NaN. ``out`` must not share memory with the
    inputs. No derivatives."""
    dev = x.get_device()
    if dev < 0 or w.get_device() != dev or scale.get_device() != dev or (zero is not None and zero.get_device() != dev) \
            or (bias is not None and bias.get_device() != dev) or (out is not None and out.get_device() != dev):
        _on_gpu(x, w, scale, zero, bias, out)
    if torch.is_grad_enabled() and (x.requires_grad or scale.requires_grad or (bias is not None and bias.requires_grad)
                                    or (out is not None and out.requires_grad)):
        _no_backward(x, scale, bias, out)
    if forward_ad._current_level >= 0:
        _no_tangent(x, scale, bias, out)
    odt = out_dtype or (out.dtype if out is not None else x.dtype)
    if out is not None and out.dtype != odt:
        raise ValueError("out must be [M, N] of out_dtype with unit column stride")
    code, ocode, M, N, K, group, ldx, ldy = _i4_views(
        x.dtype, x.shape, x.stride(), w.dtype, w.shape, scale.dtype, scale.shape,
        *((zero.dtype, zero.shape) if zero is not None else (None, None)),
        *((bias.dtype, bias.shape) if bias is not None else (None, None)), odt,
        *((out.shape, out.stride()) if out is not None else (None, None)))
    if not (w.is_contiguous() and scale.is_contiguous() and (zero is None or zero.is_contiguous())
            and (bias is None or bias.is_contiguous())):
        raise ValueError("w, scale, zero and bias must be contiguous")
    if out is None:
        out = x.new_empty((M, N)) if odt is x.dtype else x.new_empty((M, N), dtype=odt)
    else:
        _check_apart(out, x, w, scale, zero, bias)
    if M == 0 or N == 0:
        return out
    xp, wp = x.data_ptr(), w.data_ptr()
    if (xp | wp) & 15:
        _check_aligned(x=xp, w=wp)
    st = _launch(dev, _lib.lib().mi355_linear_i4, code, ocode, xp, ldx, wp, scale.data_ptr(),
                 0 if zero is None else zero.data_ptr(), 0 if bias is None else bias.data_ptr(),
                 out.data_ptr(), ldy, M, N, K, group)
    if st:
        _lib.check("mi355_linear_i4", st)
    return out
