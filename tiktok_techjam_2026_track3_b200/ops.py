"""Torch-facing wrappers over the C ABI: tensors in, tensors out, no fallback.

Every op checks device / dtype / contiguity, launches on the caller's current
CUDA stream through ``libttj_attn_sm100.so`` and raises ``RuntimeError`` on
any error code.  Nothing here computes on the CPU.
"""

from __future__ import annotations

import ctypes as C
import functools
from typing import Dict, NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _lib

_DTYPES = {torch.float16: _lib.TTJ_F16, torch.bfloat16: _lib.TTJ_BF16}
_status_words: Dict[int, torch.Tensor] = {}


def _dtype_code(t: torch.Tensor) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise RuntimeError(f"unsupported dtype {t.dtype}: the sm_100a kernels take float16 or bfloat16")
    return code


def _cuda(t: torch.Tensor, name: str) -> torch.Tensor:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (got {t.device}); there is no CPU path")
    if not t.is_contiguous():
        t = t.contiguous()
    return t


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def status_word(device: torch.device) -> torch.Tensor:
    """Per-device int32 status word the kernels write on a bounded-wait timeout."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    w = _status_words.get(idx)
    if w is None:
        with torch.inference_mode(False):
            w = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
        _status_words[idx] = w
    return w


def check_device_status(device: torch.device) -> None:
    """Synchronise and raise if any kernel on `device` reported a timeout."""
    lib = _lib.load()
    w = status_word(device)
    code = C.c_int(0)
    _lib.check(lib.ttj_read_status(w.data_ptr(), C.byref(code), _stream(device)), "device status")


def _workspace(workspace: Optional[torch.Tensor], need: int, device: torch.device) -> torch.Tensor:
    """The caller's workspace if it has `need` bytes, else a fresh one.  The kernels get
    its address alone, so one that would be used must be dense and on `device`."""
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        return torch.empty(need, dtype=torch.uint8, device=device)
    if workspace.device != device or not workspace.is_contiguous():
        raise RuntimeError(f"workspace must be a contiguous tensor on {device}, got one on {workspace.device} "
                           f"with strides {tuple(workspace.stride())}")
    return workspace


def _mask_u8(mask: Optional[torch.Tensor], b: int, s: int) -> Optional[torch.Tensor]:
    if mask is None:
        return None
    if mask.shape != (b, s):
        raise RuntimeError(f"valid_token_mask must be [B,S]=({b},{s}), got {tuple(mask.shape)}")
    mask = _cuda(mask, "valid_token_mask")
    if mask.dtype == torch.bool:
        return mask.view(torch.uint8)
    return (mask != 0).view(torch.uint8)


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor,
           residual: Optional[torch.Tensor] = None,
           row_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = x w^T + b (+ residual with masked rows keeping only the residual)."""
    lib = _lib.load()
    x, w, bias = _cuda(x, "x"), _cuda(w, "w"), _cuda(bias, "bias")
    dt = _dtype_code(x)
    if w.dtype != x.dtype or bias.dtype != x.dtype:
        raise RuntimeError("x, w and bias must share one dtype")
    k = x.shape[-1]
    m = x.numel() // k
    n = w.shape[0]
    if residual is not None:
        residual = _cuda(residual, "residual")
        if residual.dtype != x.dtype or residual.numel() != m * n:
            raise RuntimeError("residual must match the output's dtype and shape")
    rm = None
    if row_mask is not None:
        rm = _cuda(row_mask.reshape(-1), "row_mask")
        rm = rm.view(torch.uint8) if rm.dtype == torch.bool else (rm != 0).view(torch.uint8)
    y = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
    rc = lib.ttj_linear_fwd(x.data_ptr(), w.data_ptr(), bias.data_ptr(), _ptr(residual), _ptr(rm),
                            y.data_ptr(), m, n, k, dt, status_word(x.device).data_ptr(),
                            _stream(x.device))
    _lib.check(rc, "ttj_linear_fwd")
    return y


def linear_kchunked(x_chunks: torch.Tensor, w: torch.Tensor, bias: torch.Tensor,
                    residual: Optional[torch.Tensor] = None,
                    row_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[m, :] = sum_c x_chunks[c, m, :] . w[:, c*kc:(c+1)*kc]^T + bias (+ residual):
    the linear layer on an input stored K-chunk-major [K/kc, M, kc]."""
    lib = _lib.load()
    x_chunks, w, bias = _cuda(x_chunks, "x_chunks"), _cuda(w, "w"), _cuda(bias, "bias")
    dt = _dtype_code(x_chunks)
    nck, m, kc = x_chunks.shape
    n, k = w.shape
    if nck * kc != k:
        raise RuntimeError("x_chunks chunks * chunk width must equal w's input features")
    if residual is not None:
        residual = _cuda(residual, "residual")
    rm = None
    if row_mask is not None:
        rm = _cuda(row_mask.reshape(-1), "row_mask")
        rm = rm.view(torch.uint8) if rm.dtype == torch.bool else (rm != 0).view(torch.uint8)
    y = torch.empty(m, n, dtype=x_chunks.dtype, device=x_chunks.device)
    rc = lib.ttj_linear_kchunked_fwd(x_chunks.data_ptr(), kc, w.data_ptr(), bias.data_ptr(),
                                     _ptr(residual), _ptr(rm), y.data_ptr(), m, n, k, dt,
                                     status_word(x_chunks.device).data_ptr(), _stream(x_chunks.device))
    _lib.check(rc, "ttj_linear_kchunked_fwd")
    return y


def qkv_proj(x: torch.Tensor, w_qkv: torch.Tensor, b_qkv: torch.Tensor) -> torch.Tensor:
    """[B,S,D] -> packed [B,S,3D] (q | k | v)."""
    lib = _lib.load()
    x = _cuda(x, "x")
    dt = _dtype_code(x)
    B, S, D = x.shape
    qkv = torch.empty(B, S, 3 * D, dtype=x.dtype, device=x.device)
    rc = lib.ttj_qkv_proj_fwd(x.data_ptr(), _cuda(w_qkv, "w_qkv").data_ptr(),
                              _cuda(b_qkv, "b_qkv").data_ptr(), qkv.data_ptr(), B * S, D, dt,
                              status_word(x.device).data_ptr(), _stream(x.device))
    _lib.check(rc, "ttj_qkv_proj_fwd")
    return qkv


def flash_attn(qkv: torch.Tensor, num_heads: int, causal: bool,
               key_mask: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Packed [B,S,3D] -> context [B,S,D] (heads merged), optionally into ``out``."""
    lib = _lib.load()
    qkv = _cuda(qkv, "qkv")
    dt = _dtype_code(qkv)
    B, S, D3 = qkv.shape
    D = D3 // 3
    km = _mask_u8(key_mask, B, S)
    if out is None:
        ctx = torch.empty(B, S, D, dtype=qkv.dtype, device=qkv.device)
    else:
        if out.shape != (B, S, D) or out.dtype != qkv.dtype or not out.is_contiguous():
            raise RuntimeError("out must be a contiguous [B,S,D] tensor of qkv's dtype")
        ctx = out
    rc = lib.ttj_flash_attn_fwd(qkv.data_ptr(), _ptr(km), ctx.data_ptr(), B, S, num_heads,
                                D // num_heads, int(bool(causal)), dt,
                                status_word(qkv.device).data_ptr(), _stream(qkv.device))
    _lib.check(rc, "ttj_flash_attn_fwd")
    return ctx


def attn_layer(x: torch.Tensor, w_qkv: torch.Tensor, b_qkv: torch.Tensor, w_o: torch.Tensor,
               b_o: torch.Tensor, num_heads: int, causal: bool,
               valid_token_mask: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, add_residual: bool = True,
               out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = residual + attention(x); residual defaults to x (the attention
    layer); ``add_residual=False`` returns the attention output alone."""
    lib = _lib.load()
    x = _cuda(x, "x")
    dt = _dtype_code(x)
    B, S, D = x.shape
    for t, n in ((w_qkv, "w_qkv"), (b_qkv, "b_qkv"), (w_o, "w_o"), (b_o, "b_o")):
        if t.dtype != x.dtype or t.device != x.device:
            raise RuntimeError(f"{n} must be {x.dtype} on {x.device}")
    if add_residual:
        residual = x if residual is None else _cuda(residual, "residual")
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise RuntimeError("residual must match x's shape and dtype")
    else:
        residual = None
    km = _mask_u8(valid_token_mask, B, S)
    if out is None:
        out = torch.empty_like(x)
    need = lib.ttj_attn_layer_workspace_size(B, S, D, dt)
    workspace = _workspace(workspace, need, x.device)
    a = _lib.AttnLayerArgs(
        x=x.data_ptr(), w_qkv=_cuda(w_qkv, "w_qkv").data_ptr(), b_qkv=_cuda(b_qkv, "b_qkv").data_ptr(),
        w_o=_cuda(w_o, "w_o").data_ptr(), b_o=_cuda(b_o, "b_o").data_ptr(),
        valid_token_mask=_ptr(km), residual=_ptr(residual), out=out.data_ptr(),
        workspace=workspace.data_ptr(), workspace_bytes=workspace.numel() * workspace.element_size(),
        status=status_word(x.device).data_ptr(), batch=B, seq_len=S, d_model=D,
        num_heads=num_heads, causal=int(bool(causal)), dtype=dt)
    _lib.check(lib.ttj_attn_layer_fwd(C.byref(a), _stream(x.device)), "ttj_attn_layer_fwd")
    return out


# ------------------------------------------------------- transformer block

def layernorm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float,
              row_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """nn.LayerNorm over the last dimension (fp32 arithmetic); rows whose mask
    entry is False come out as zeros.  fp16, bf16 or fp32 (d <= 4096) rows."""
    lib = _lib.load()
    x = _cuda(x, "x")
    dt = _lib.TTJ_F32 if x.dtype == torch.float32 else _dtype_code(x)
    d = x.shape[-1]
    rows = x.numel() // d
    if weight.dtype != x.dtype or bias.dtype != x.dtype:
        raise RuntimeError("weight and bias must share x's dtype")
    rm = None
    if row_mask is not None:
        rm = _cuda(row_mask.reshape(-1), "row_mask")
        if rm.numel() != rows:
            raise RuntimeError("row_mask must have one entry per row")
        rm = rm.view(torch.uint8) if rm.dtype == torch.bool else (rm != 0).view(torch.uint8)
    y = torch.empty_like(x)
    rc = lib.ttj_layernorm_fwd(x.data_ptr(), _cuda(weight, "weight").data_ptr(),
                               _cuda(bias, "bias").data_ptr(), _ptr(rm), y.data_ptr(), rows, d,
                               float(eps), dt, _stream(x.device))
    _lib.check(rc, "ttj_layernorm_fwd")
    return y


def linear_gelu(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
    """gelu(x w^T + b) with the exact (erf) GELU, one GEMM launch."""
    lib = _lib.load()
    x, w, bias = _cuda(x, "x"), _cuda(w, "w"), _cuda(bias, "bias")
    dt = _dtype_code(x)
    if w.dtype != x.dtype or bias.dtype != x.dtype:
        raise RuntimeError("x, w and bias must share one dtype")
    k = x.shape[-1]
    m = x.numel() // k
    n = w.shape[0]
    y = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
    rc = lib.ttj_linear_gelu_fwd(x.data_ptr(), w.data_ptr(), bias.data_ptr(), y.data_ptr(), m, n, k, dt,
                                 status_word(x.device).data_ptr(), _stream(x.device))
    _lib.check(rc, "ttj_linear_gelu_fwd")
    return y


BLOCK_PARAMS = ("ln1_w", "ln1_b", "w_qkv", "b_qkv", "w_o", "b_o", "ln2_w", "ln2_b",
                "w_in", "b_in", "w_out", "b_out")
# An fp32 block (fp32 residual stream) keeps these in fp32 and the rest in fp16
# (ttj_transformer_block_fwd with TTJ_F32).
BLOCK_F32_STREAM_PARAMS = ("ln1_w", "ln1_b", "b_o", "ln2_w", "ln2_b", "b_out")


def block_param_dtype(name: str, x_dtype: torch.dtype) -> torch.dtype:
    """dtype the block kernels expect for parameter `name` given the input dtype."""
    if x_dtype == torch.float32:
        return torch.float32 if name in BLOCK_F32_STREAM_PARAMS else torch.float16
    return x_dtype


def transformer_block(x: torch.Tensor, params: Dict[str, torch.Tensor], num_heads: int,
                      causal: bool, eps1: float, eps2: float,
                      valid_token_mask: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None,
                      workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One pre-norm block (BaselineTransformerBlock.forward) in seven launches;
    ``params`` holds the tensors named in BLOCK_PARAMS (w_qkv packed q|k|v) in
    the dtypes of ``block_param_dtype``: x's dtype for fp16 / bf16 blocks; for
    fp32 x an fp32 residual stream with fp16 tensor-core operands."""
    lib = _lib.load()
    x = _cuda(x, "x")
    dt = _lib.TTJ_F32 if x.dtype == torch.float32 else _dtype_code(x)
    if x.dim() != 3:
        raise RuntimeError(f"x must be [B,S,D], got {tuple(x.shape)}")
    B, S, D = x.shape
    ptrs = {}
    for name in BLOCK_PARAMS:
        t = params[name]
        want = block_param_dtype(name, x.dtype)
        if t.dtype != want or t.device != x.device:
            raise RuntimeError(f"{name} must be {want} on {x.device}")
        ptrs[name] = _cuda(t, name).data_ptr()
    F = params["w_in"].shape[0]
    if params["w_in"].shape != (F, D) or params["w_out"].shape != (D, F) or params["w_qkv"].shape != (3 * D, D):
        raise RuntimeError("block weights do not match d_model / ffn_dim")
    km = _mask_u8(valid_token_mask, B, S)
    if out is None:
        out = torch.empty_like(x)
    need = lib.ttj_block_workspace_size(B, S, D, F, dt)
    workspace = _workspace(workspace, need, x.device)
    a = _lib.BlockArgs(x=x.data_ptr(), valid_token_mask=_ptr(km), out=out.data_ptr(),
                       workspace=workspace.data_ptr(), workspace_bytes=workspace.numel() * workspace.element_size(),
                       status=status_word(x.device).data_ptr(), batch=B, seq_len=S, d_model=D,
                       num_heads=num_heads, ffn_dim=F, eps1=float(eps1), eps2=float(eps2),
                       causal=int(bool(causal)), dtype=dt, **ptrs)
    _lib.check(lib.ttj_transformer_block_fwd(C.byref(a), _stream(x.device)), "ttj_transformer_block_fwd")
    return out


# ---------------------------------------------------------------------- int8

def int8_quant_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """[..., K] fp16/bf16 -> (int8 [..., K], fp32 scale [rows])."""
    lib = _lib.load()
    x = _cuda(x, "x")
    dt = _dtype_code(x)
    k = x.shape[-1]
    rows = x.numel() // k
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    s = torch.empty(rows, dtype=torch.float32, device=x.device)
    _lib.check(lib.ttj_int8_quant_rows(x.data_ptr(), q.data_ptr(), s.data_ptr(), rows, k, dt,
                                       _stream(x.device)), "ttj_int8_quant_rows")
    return q, s


def int8_gemm_s32(a: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """Raw int32 accumulators a[M,K] . w[N,K]^T."""
    lib = _lib.load()
    a, w = _cuda(a, "a"), _cuda(w, "w")
    if a.dtype != torch.int8 or w.dtype != torch.int8:
        raise RuntimeError("int8_gemm_s32 takes int8 operands")
    m, k = a.shape
    n = w.shape[0]
    acc = torch.empty(m, n, dtype=torch.int32, device=a.device)
    _lib.check(lib.ttj_int8_gemm_s32(a.data_ptr(), w.data_ptr(), acc.data_ptr(), m, n, k,
                                     status_word(a.device).data_ptr(), _stream(a.device)),
               "ttj_int8_gemm_s32")
    return acc


def int8_linear(a: torch.Tensor, s_a: torch.Tensor, w: torch.Tensor, s_w: torch.Tensor,
                bias: torch.Tensor, out_dtype: torch.dtype,
                residual: Optional[torch.Tensor] = None,
                row_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Dequantising int8 GEMM: acc * (s_a * s_w) + bias (+ residual)."""
    lib = _lib.load()
    a, w = _cuda(a, "a"), _cuda(w, "w")
    m, k = a.shape
    n = w.shape[0]
    dt = _DTYPES[out_dtype]
    y = torch.empty(m, n, dtype=out_dtype, device=a.device)
    rm = None
    if row_mask is not None:
        rm = _cuda(row_mask.reshape(-1), "row_mask")
        rm = rm.view(torch.uint8) if rm.dtype == torch.bool else (rm != 0).view(torch.uint8)
    if residual is not None:
        residual = _cuda(residual, "residual")
    _lib.check(lib.ttj_int8_linear_fwd(a.data_ptr(), _cuda(s_a, "s_a").data_ptr(), w.data_ptr(),
                                       _cuda(s_w, "s_w").data_ptr(), _cuda(bias, "bias").data_ptr(),
                                       _ptr(residual), _ptr(rm), y.data_ptr(), m, n, k, dt,
                                       status_word(a.device).data_ptr(), _stream(a.device)),
               "ttj_int8_linear_fwd")
    return y


def int8_attn_layer(x: torch.Tensor, w_qkv8: torch.Tensor, s_qkv: torch.Tensor,
                    b_qkv: torch.Tensor, w_o8: torch.Tensor, s_o: torch.Tensor,
                    b_o: torch.Tensor, num_heads: int, causal: bool,
                    valid_token_mask: Optional[torch.Tensor] = None,
                    residual: Optional[torch.Tensor] = None, add_residual: bool = True,
                    out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """W8A8 attention layer (benchmark configuration 3 recipe)."""
    lib = _lib.load()
    x = _cuda(x, "x")
    dt = _dtype_code(x)
    B, S, D = x.shape
    if add_residual:
        residual = x if residual is None else _cuda(residual, "residual")
    else:
        residual = None
    km = _mask_u8(valid_token_mask, B, S)
    if out is None:
        out = torch.empty_like(x)
    need = lib.ttj_int8_attn_layer_workspace_size(B, S, D, dt)
    workspace = _workspace(workspace, need, x.device)
    a = _lib.Int8AttnLayerArgs(
        x=x.data_ptr(), w_qkv=_cuda(w_qkv8, "w_qkv").data_ptr(), s_qkv=_cuda(s_qkv, "s_qkv").data_ptr(),
        b_qkv=_cuda(b_qkv, "b_qkv").data_ptr(), w_o=_cuda(w_o8, "w_o").data_ptr(),
        s_o=_cuda(s_o, "s_o").data_ptr(), b_o=_cuda(b_o, "b_o").data_ptr(),
        valid_token_mask=_ptr(km), residual=_ptr(residual), out=out.data_ptr(),
        workspace=workspace.data_ptr(), workspace_bytes=workspace.numel() * workspace.element_size(),
        status=status_word(x.device).data_ptr(), batch=B, seq_len=S, d_model=D,
        num_heads=num_heads, causal=int(bool(causal)), dtype=dt)
    _lib.check(lib.ttj_int8_attn_layer_fwd(C.byref(a), _stream(x.device)), "ttj_int8_attn_layer_fwd")
    return out


def quantize_weight(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-output-channel int8 weight packing (one-time, at weight load):
    s = max|w| / 127 clamped to >= 1e-8, q = round(w / s)
    (Project/kernels/k008_int8_gemm.py:154-158).  Runs as torch ops on the
    weights' device; it is set-up, not part of the timed forward."""
    wf = w.float()
    amax = wf.abs().amax(dim=1)
    # Divide by a tensor, not a Python scalar: CUDA torch turns a scalar
    # divisor into a reciprocal multiply, which is not the recipe's IEEE
    # division and can move the scale by one ulp.
    s = (amax / torch.full_like(amax, 127.0)).clamp(min=1e-8)
    q = torch.round(wf / s[:, None]).to(torch.int8)
    return q.contiguous(), s.contiguous()


# ------------------------------------------------------- serving: prompts, caches

def _strided(t: torch.Tensor) -> Tuple:
    """(t, address, element strides of all dimensions but the last): views whose rows
    are contiguous and 16-byte aligned are read in place, anything else is copied."""
    st, p = t.stride(), t.data_ptr()
    if len(st) == 3:
        a, b, c = st
        if c == 1 and a > 0 and b > 0 and not (a | b) & 7 and not p & 15:
            return t, p, a, b
    else:
        a, b, c, d = st
        if d == 1 and a > 0 and b > 0 and c > 0 and not (a | b | c) & 7 and not p & 15:
            return t, p, a, b, c
    lead = [s for n, s in zip(t.shape[:-1], st[:-1]) if n > 1]
    if st[-1] != 1 or p % 16 or any(s <= 0 or s % 8 for s in lead):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    # a dimension of one element has no stride of its own; give it a valid one
    return (t, t.data_ptr(), *(s if n > 1 else t.shape[-1] for n, s in zip(t.shape[:-1], t.stride()[:-1])))


def _same(ref: torch.Tensor, names: Tuple[str, ...], *tensors: torch.Tensor) -> None:
    """`ref` is on a GPU and `tensors` share its dtype and device."""
    dtype, device = ref.dtype, ref.get_device()
    for t in tensors:
        if t.dtype is not dtype or t.get_device() != device or device < 0:
            break
    else:
        return
    for name, t in zip(("the first operand",) + names, (ref,) + tensors):
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor (got {t.device}); there is no CPU path")
        if t.dtype != dtype or t.device != ref.device:
            raise RuntimeError(f"{name} must be {dtype} on {ref.device}, got {t.dtype} on {t.device}")


def _launch(call: _lib.PackedCall, index: int, *values) -> None:
    """Enqueue on device `index`'s current stream, with that device current."""
    if torch._C._cuda_getDevice() == index:
        call(torch._C._cuda_getCurrentRawStream(index), values)
    else:
        with torch.cuda.device(index):
            call(torch._C._cuda_getCurrentRawStream(index), values)


def _status(index: int) -> int:
    """Address of device `index`'s status word."""
    w = _status_words.get(index)
    return (status_word(torch.device("cuda", index)) if w is None else w).data_ptr()


def _group(num_heads: int, num_kv_heads: int) -> int:
    if num_kv_heads <= 0 or num_heads <= 0 or num_heads % num_kv_heads:
        raise RuntimeError(f"num_heads ({num_heads}) must be a positive multiple of num_kv_heads ({num_kv_heads})")
    return num_heads // num_kv_heads


class PromptPlan:
    """Work plan of a packed batch of prompts: built once from the prompts' lengths
    (on the host, zero lengths allowed) and read by every layer's ``prompt_attn``.
    Its table is on the device when the constructor returns, for any stream."""

    def __init__(self, seq_lens: Union[Sequence[int], torch.Tensor], num_heads: int, num_kv_heads: int,
                 head_dim: int, device: Union[torch.device, str, int]) -> None:
        lib = _lib.load()
        lens = [int(n) for n in (seq_lens.tolist() if isinstance(seq_lens, torch.Tensor) else seq_lens)]
        _group(num_heads, num_kv_heads)
        self.seq_lens = tuple(lens)
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, head_dim
        self.tokens = sum(lens)
        arr = (C.c_int64 * max(1, len(lens)))(*lens)
        n = lib.ttj_prompt_plan_entries(arr, len(lens), num_heads, num_kv_heads, head_dim)
        if n < 0:
            _lib.check(int(n), "ttj_prompt_plan_entries")
        host = torch.empty(max(1, n), 4, dtype=torch.int32)
        _lib.check(lib.ttj_prompt_plan_build(arr, len(lens), num_heads, num_kv_heads, head_dim,
                                             C.cast(host.data_ptr(), C.POINTER(C.c_int32)), n),
                   "ttj_prompt_plan_build")
        self.entries = int(n)
        self.q_shape = torch.Size((self.tokens, num_heads, head_dim))
        self.kv_shape = torch.Size((self.tokens, num_kv_heads, head_dim))
        self.table = host.to(device)

    @property
    def device(self) -> torch.device:
        return self.table.device


def prompt_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PromptPlan,
                scale: Optional[float] = None, return_lse: bool = False,
                out: Optional[torch.Tensor] = None):
    """Causal attention of packed prompts: q [T,Hq,hd] and k, v [T,Hkv,hd] hold the
    plan's prompts one after another; query head h reads key / value head
    h // (Hq / Hkv).  Returns [T,Hq,hd], and with ``return_lse`` also the log of
    each row's sum of exponentials, fp32 [T,Hq].  Views with strided rows (slices
    of a packed projection) are read in place.  scale defaults to hd ** -0.5."""
    dt = _dtype_code(q)
    if q.shape != plan.q_shape or k.shape != plan.kv_shape or v.shape != plan.kv_shape:
        for t, n, want in ((q, "q", plan.q_shape), (k, "k", plan.kv_shape), (v, "v", plan.kv_shape)):
            if t.shape != want:
                raise RuntimeError(f"{n} must be {list(want)} for this plan, got {list(t.shape)}")
    _same(q, ("k", "v"), k, v)
    q, qp, qt, qh = _strided(q)
    k, kp, kt, kh = _strided(k)
    v, vp, vt, vh = _strided(v)
    dev, index = q.device, q.get_device()
    if plan.table.get_device() != index:
        raise RuntimeError(f"the plan is on {plan.device}, q on {dev}")
    if out is None:
        out = q.new_empty(plan.q_shape)
    elif out.shape != plan.q_shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise RuntimeError("out must be a contiguous [T,Hq,hd] tensor of q's dtype on q's device")
    lse = torch.empty(plan.q_shape[:2], dtype=torch.float32, device=dev) if return_lse else None
    _launch(_lib.prompt_attn_fwd, index, qp, kp, vp, out.data_ptr(), _ptr(lse) or 0, plan.table.data_ptr(),
            plan.entries, _status(index), plan.tokens, plan.num_heads, plan.num_kv_heads,
            plan.head_dim, qt, qh, kt, kh, vt, vh, plan.head_dim ** -0.5 if scale is None else float(scale), dt)
    return (out, lse) if return_lse else out


def _dense(t: torch.Tensor, name: str, shape: Tuple[int, ...], dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise RuntimeError(f"{name} must be {str(dtype)[6:]} {list(shape)} on {device}, got {str(t.dtype)[6:]} "
                           f"{list(t.shape)} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


@functools.lru_cache(maxsize=256)
def _decode_workspace(B: int, P: int, Cap: int, Hq: int, Hkv: int, hd: int, weights: bool, index: int) -> int:
    """Bytes of workspace of a decode step of these sizes on device `index`."""
    with torch.cuda.device(index):
        return _lib.load().ttj_shared_prefix_attn_workspace_size(B, P, Cap, Hq, Hkv, hd, weights)


def shared_prefix_attn(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor,
                       k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor,
                       key_weights: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                       return_lse: bool = False, out: Optional[torch.Tensor] = None,
                       workspace: Optional[torch.Tensor] = None):
    """One decode step: each sequence's new token q [B,Hq,hd] attends the prefix rows
    prefix_k / prefix_v [P,Hkv,hd] that the whole batch shares, then the first
    ``lengths[b]`` rows of its own cache k_cache / v_cache [B,C,Hkv,hd] (P and C may
    be zero; a sequence without any key gets zeros).  Returns [B,Hq,hd], followed by
    whichever of these is asked for:

    ``key_weights`` (fp32 [B,Hkv,C]) gives new_key_weights, each cached key's weight
    plus this step's probabilities of that key summed over the group's heads, for
    ``cache_evict`` (the input is not written); ``return_lse`` gives the log of each
    row's sum of exponentials, fp32 [B,Hq], -inf for a row without any key.

    A key that scores -inf weighs nothing, and a row of such keys alone is as one
    without any.  ``workspace`` (contiguous, on q's device) is used if it is large
    enough."""
    dt = _dtype_code(q)
    if q.dim() != 3 or prefix_k.dim() != 3 or k_cache.dim() != 4:
        raise RuntimeError("q must be [B,Hq,hd], prefix_k and prefix_v [P,Hkv,hd], k_cache and v_cache [B,C,Hkv,hd]")
    B, Hq, hd = q.shape
    P, Hkv, _ = prefix_k.shape
    Cap = k_cache.shape[1]
    _group(Hq, Hkv)
    shared, own = (P, Hkv, hd), (B, Cap, Hkv, hd)
    if prefix_k.shape != shared or prefix_v.shape != shared or k_cache.shape != own or v_cache.shape != own:
        for t, n, want in ((prefix_k, "prefix_k", shared), (prefix_v, "prefix_v", shared),
                           (k_cache, "k_cache", own), (v_cache, "v_cache", own)):
            if t.shape != want:
                raise RuntimeError(f"{n} must be {list(want)}, got {list(t.shape)}")
    _same(q, ("prefix_k", "prefix_v", "k_cache", "v_cache"), prefix_k, prefix_v, k_cache, v_cache)
    q, qp, qs, qh = _strided(q)
    prefix_k, pkp, pkr, pkh = _strided(prefix_k)
    prefix_v, pvp, pvr, pvh = _strided(prefix_v)
    k_cache, kp, ks, kr, kh = _strided(k_cache)
    v_cache, vp, vs, vr, vh = _strided(v_cache)
    dev = q.device
    lengths = _dense(lengths, "lengths", (B,), torch.int32, dev)
    new_weights = None
    if key_weights is not None:
        key_weights = _dense(key_weights, "key_weights", (B, Hkv, Cap), torch.float32, dev)
        new_weights = torch.empty_like(key_weights)
    if out is None:
        out = q.new_empty((B, Hq, hd))
    elif out.shape != (B, Hq, hd) or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise RuntimeError("out must be a contiguous [B,Hq,hd] tensor of q's dtype on q's device")
    lse = torch.empty(B, Hq, dtype=torch.float32, device=dev) if return_lse else None
    index = dev.index
    need = _decode_workspace(B, P, Cap, Hq, Hkv, hd, key_weights is not None, index)
    workspace = _workspace(workspace, need, dev)
    _launch(_lib.shared_prefix_attn_fwd, index, qp, pkp, pvp, kp, vp, lengths.data_ptr(), _ptr(key_weights) or 0,
            _ptr(new_weights) or 0, out.data_ptr(), _ptr(lse) or 0, workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), _status(index), B, P, Cap, Hq, Hkv, hd, qs, qh, pkr, pkh,
            pvr, pvh, ks, kr, kh, vs, vr, vh,
            hd ** -0.5 if scale is None else float(scale), dt)
    if new_weights is None and lse is None:
        return out
    return (out,) + tuple(t for t in (new_weights, lse) if t is not None)


class EvictedCache(NamedTuple):
    """``cache_evict``'s result: the compacted cache and which rows it holds."""
    k: torch.Tensor            # [B, budget, Hkv, hd]
    v: torch.Tensor
    key_weights: torch.Tensor  # fp32 [B, Hkv, budget]
    lengths: torch.Tensor      # int32 [B]
    positions: torch.Tensor    # int32 [B, Hkv, budget], -1 past the kept rows


def cache_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, key_weights: torch.Tensor,
                lengths: torch.Tensor, budget: int, recent: int,
                out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> EvictedCache:
    """Cut each cache k_cache / v_cache [B,C,Hkv,hd] to ``budget`` rows per key / value
    head: the last ``recent`` of its ``lengths[b]`` rows and, of the others, those
    with the largest accumulated attention weight (key_weights, fp32 [B,Hkv,C];
    equal weights: the lowest row first; NaN counts as -infinity), in their order.
    Caches of at most ``budget`` rows are kept whole.  Rows past the kept ones are
    zeros.  ``out`` = (k, v) of at least ``budget`` rows takes the result in place
    of fresh caches (rows from ``budget`` on are left alone); it must not alias
    the input."""
    _dtype_code(k_cache)
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise RuntimeError(f"k_cache and v_cache must both be [B,C,Hkv,hd], got {list(k_cache.shape)} and {list(v_cache.shape)}")
    B, Cap, Hkv, hd = k_cache.shape
    budget, recent = int(budget), int(recent)
    if budget <= 0 or recent < 0 or recent > budget:
        raise RuntimeError(f"budget must be positive and recent in 0 .. budget, got {budget} and {recent}")
    _same(k_cache, ("v_cache",), v_cache)
    dev = k_cache.device
    k_cache, kp, ks, kr, kh = _strided(k_cache)
    v_cache, vp, vs, vr, vh = _strided(v_cache)
    lengths = _dense(lengths, "lengths", (B,), torch.int32, dev)
    key_weights = _dense(key_weights, "key_weights", (B, Hkv, Cap), torch.float32, dev)
    if out is None:
        k_out = k_cache.new_empty((B, budget, Hkv, hd))
        v_out = k_cache.new_empty((B, budget, Hkv, hd))
        kop, vop = k_out.data_ptr(), v_out.data_ptr()
        koh = voh = hd
        kor = vor = Hkv * hd
        kos = vos = budget * kor
    else:
        k_out, v_out = out
        _same(k_cache, ("k_out", "v_out"), k_out, v_out)
        for t, n in ((k_out, "k_out"), (v_out, "v_out")):
            if t.dim() != 4 or t.shape[0] != B or t.shape[1] < budget or t.shape[2:] != (Hkv, hd):
                raise RuntimeError(f"{n} must be [{B}, >={budget}, {Hkv}, {hd}], got {list(t.shape)}")
        ko, kop, kos, kor, koh = _strided(k_out)
        vo, vop, vos, vor, voh = _strided(v_out)
        if ko is not k_out or vo is not v_out:
            raise RuntimeError("out must have contiguous rows and 16-byte aligned strides")
    weights = key_weights.new_empty((B, Hkv, budget))
    new_lengths = lengths.new_empty((B,))
    positions = lengths.new_empty((B, Hkv, budget))
    _launch(_lib.cache_evict, dev.index, kp, vp, key_weights.data_ptr(), lengths.data_ptr(), kop, vop, weights.data_ptr(),
            new_lengths.data_ptr(), positions.data_ptr(), B, Cap, Hkv, hd, budget, recent, ks, kr, kh, vs, vr, vh,
            kos, kor, koh, vos, vor, voh)
    return EvictedCache(k_out, v_out, weights, new_lengths, positions)
