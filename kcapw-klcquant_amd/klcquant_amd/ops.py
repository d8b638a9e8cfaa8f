"""Tensor-level wrappers over the C ABI (device tensors in, device tensors out).

Every function validates shapes, dtypes, devices and contiguity on the host,
then enqueues HIP work on the current torch stream of the tensors' device and
returns without synchronising.  There is no CPU path: CPU tensors are
rejected.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
import operator
import struct
from typing import NamedTuple

import numpy as np
import torch

from . import _native as nat

_DTYPE_CODES = {torch.bfloat16: nat.DTYPE_BF16, torch.float16: nat.DTYPE_F16, torch.float32: nat.DTYPE_F32}
PRECISIONS = {"fp32": nat.PRECISION_FP32, "bf16": nat.PRECISION_BF16}


def _ptr(t: torch.Tensor | None) -> ctypes.c_void_p:
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _check_gpu(name: str, t: torch.Tensor, dtype: torch.dtype | None = None, ndim: int | None = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on a GPU device (the MoE path has no CPU implementation), got {t.device}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dims, got shape {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _same_device(*ts: torch.Tensor) -> torch.device:
    dev = ts[0].device
    for t in ts[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} vs {t.device}")
    return dev


# ---- MXFP4 -------------------------------------------------------------------

def _mxfp4_shapes(blocks: torch.Tensor, scales: torch.Tensor) -> tuple[int, int, int, bool]:
    if blocks.dim() < 3 or blocks.shape[:-1] != scales.shape:
        # same message as mxfp4_expert.py:368-369
        raise ValueError(f"MXFP4 block/scale shape mismatch: blocks.shape={blocks.shape} scales.shape={scales.shape}")
    if blocks.shape[-1] != 16:
        raise ValueError(f"MXFP4 blocks must pack 16 bytes per group, got shape {tuple(blocks.shape)}")
    single = blocks.dim() == 3
    n_mat = 1 if single else math.prod(blocks.shape[:-3])
    return n_mat, int(blocks.shape[-3]), int(blocks.shape[-2]), single


def mxfp4_dequant(blocks: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``[..., out, G, 16]`` + ``[..., out, G]`` -> ``[..., G * 32, out]`` in ``dtype``."""
    n_mat, out_dim, groups, single = _mxfp4_shapes(blocks, scales)
    if dtype not in _DTYPE_CODES:
        raise TypeError(f"unsupported dequant dtype {dtype}")
    blocks = blocks.contiguous() if blocks.dtype == torch.uint8 else blocks.to(torch.uint8).contiguous()
    scales = scales.contiguous() if scales.dtype == torch.uint8 else scales.to(torch.uint8).contiguous()
    _check_gpu("blocks", blocks, torch.uint8)
    _check_gpu("scales", scales, torch.uint8)
    dev = _same_device(blocks, scales)
    out = torch.empty((*blocks.shape[:-3], groups * 32, out_dim), dtype=dtype, device=dev)
    nat.call("klc_mxfp4_dequant", _ptr(blocks), _ptr(scales), _ptr(out), n_mat, out_dim, groups,
             _DTYPE_CODES[dtype], _stream(dev))
    return out


def packed_bytes(out_dim: int, groups: int) -> int:
    return nat.call("klc_mxfp4_packed_bytes", out_dim, groups)


def mxfp4_pack(blocks: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Checkpoint layout -> row-tile layout; returns uint8 ``[n, packed_bytes]``."""
    n_mat, out_dim, groups, _ = _mxfp4_shapes(blocks, scales)
    _check_gpu("blocks", blocks, torch.uint8)
    _check_gpu("scales", scales, torch.uint8)
    dev = _same_device(blocks, scales)
    nbytes = packed_bytes(out_dim, groups)
    if out is None:
        out = torch.empty((n_mat, nbytes), dtype=torch.uint8, device=dev)
    else:
        _check_gpu("out", out, torch.uint8)
        if out.numel() != n_mat * nbytes:
            raise ValueError(f"out holds {out.numel()} bytes, need {n_mat * nbytes}")
    nat.call("klc_mxfp4_pack", _ptr(blocks), _ptr(scales), _ptr(out), n_mat, out_dim, groups, _stream(dev))
    return out


def mxfp4_dequant_packed(packed: torch.Tensor, out_dim: int, groups: int,
                         dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Row-tile packed ``[n, bytes]`` (or ``[bytes]``) -> ``[n, G * 32, out]`` (or ``[G * 32, out]``)."""
    _check_gpu("packed", packed, torch.uint8)
    nbytes = packed_bytes(out_dim, groups)
    if packed.numel() % nbytes:
        raise ValueError(f"packed holds {packed.numel()} bytes, not a multiple of {nbytes}")
    n_mat = packed.numel() // nbytes
    shape = (groups * 32, out_dim) if packed.dim() == 1 else (n_mat, groups * 32, out_dim)
    out = torch.empty(shape, dtype=dtype, device=packed.device)
    nat.call("klc_mxfp4_dequant_packed", _ptr(packed), _ptr(out), n_mat, out_dim, groups, _DTYPE_CODES[dtype],
             _stream(packed.device))
    return out


# ---- Router --------------------------------------------------------------------

def router_logits(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, want_f32: bool = False):
    """bf16 ``x [B, H]``, ``weight [E, H]``, ``bias [E]`` -> bf16 logits ``[B, E]`` (and fp32 x)."""
    _check_gpu("hidden", x, torch.bfloat16, 2)
    _check_gpu("router weight", weight, torch.bfloat16, 2)
    _check_gpu("router bias", bias, torch.bfloat16, 1)
    dev = _same_device(x, weight, bias)
    n_tok, hidden = x.shape
    n_exp = weight.shape[0]
    if weight.shape[1] != hidden or bias.shape[0] != n_exp:
        raise ValueError(f"router shapes mismatch: x {tuple(x.shape)}, weight {tuple(weight.shape)}, bias {tuple(bias.shape)}")
    logits = torch.empty((n_tok, n_exp), dtype=torch.bfloat16, device=dev)
    x_f32 = torch.empty((n_tok, hidden), dtype=torch.float32, device=dev) if want_f32 else None
    nat.call("klc_moe_router_logits", _ptr(x), _ptr(weight), _ptr(bias), _ptr(logits), _ptr(x_f32), n_tok, hidden,
             n_exp, _stream(dev))
    return (logits, x_f32) if want_f32 else logits


def topk_softmax(logits: torch.Tensor, k: int):
    """bf16 logits ``[B, E]`` -> (int32 ids ``[B, k]``, fp32 values, bf16 weights)."""
    _check_gpu("logits", logits, torch.bfloat16, 2)
    n_tok, n_exp = logits.shape
    dev = logits.device
    ids = torch.empty((n_tok, k), dtype=torch.int32, device=dev)
    values = torch.empty((n_tok, k), dtype=torch.float32, device=dev)
    weights = torch.empty((n_tok, k), dtype=torch.bfloat16, device=dev)
    nat.call("klc_moe_topk_softmax", _ptr(logits), _ptr(ids), _ptr(values), _ptr(weights), n_tok, n_exp, k,
             _stream(dev))
    return ids, values, weights


def softmax_weights(values: torch.Tensor) -> torch.Tensor:
    """fp32 scores ``[B, k]`` -> bf16 softmax weights ``[B, k]``."""
    _check_gpu("values", values, torch.float32, 2)
    weights = torch.empty(values.shape, dtype=torch.bfloat16, device=values.device)
    nat.call("klc_moe_softmax_weights", _ptr(values), _ptr(weights), values.shape[0], values.shape[1],
             _stream(values.device))
    return weights


class Dispatch(NamedTuple):
    """klc_moe_dispatch outputs: expert offsets ``[E + 1]``, pairs sorted by expert
    ``[P]``, active experts ``[E]`` (-1 padded), their count ``[1]`` and the GEMV
    work units (``units[0]``/``units[1]`` = gate_up/down unit counts, then the lists)."""

    offsets: torch.Tensor
    sorted_pairs: torch.Tensor
    active: torch.Tensor
    n_active: torch.Tensor
    units: torch.Tensor
    n_experts: int


def max_tokens_per_call(k: int) -> int:
    """Tokens of top-``k`` routing that one dispatch / layer call takes."""
    return min(nat.LAYER_MAX_TOKENS, nat.DISPATCH_MAX_PAIRS // max(1, int(k)))


def dispatch(ids: torch.Tensor, n_experts: int) -> Dispatch:
    """int32 ids ``[B, k]`` -> :class:`Dispatch`."""
    _check_gpu("ids", ids, torch.int32)
    dev = ids.device
    n_pairs = ids.numel()
    offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=dev)
    sorted_pairs = torch.empty(n_pairs, dtype=torch.int32, device=dev)
    active = torch.empty(n_experts, dtype=torch.int32, device=dev)
    n_active = torch.empty(1, dtype=torch.int32, device=dev)
    units = torch.empty(nat.call("klc_moe_units_size", n_pairs, n_experts), dtype=torch.int32, device=dev)
    nat.call("klc_moe_dispatch", _ptr(ids), n_pairs, n_experts, _ptr(offsets), _ptr(sorted_pairs), _ptr(active),
             _ptr(n_active), _ptr(units), _stream(dev))
    return Dispatch(offsets, sorted_pairs, active, n_active, units, n_experts)


# ---- Experts --------------------------------------------------------------------

def pointer_table(mats: list[torch.Tensor] | torch.Tensor, device: torch.device) -> torch.Tensor:
    """Device int64 table of matrix base addresses (one per expert)."""
    if isinstance(mats, torch.Tensor):
        base = mats.data_ptr()
        stride = mats.stride(0) * mats.element_size()
        addrs = [base + i * stride for i in range(mats.shape[0])]
    else:
        addrs = [m.data_ptr() for m in mats]
    return torch.tensor(addrs, dtype=torch.int64).to(device)


def gate_up(table: torch.Tensor, bias: torch.Tensor, x: torch.Tensor, k: int, disp: Dispatch, hidden: int,
            inter: int, limit: float = 7.0, precision: str = "fp32", want_raw: bool = False, gemm: bool = False):
    """Returns the down input as bf16 hi/lo planes ``[2, B * k, I]`` (and the float32 SwiGLU output).

    ``gemm`` selects the grouped GEMM (klc_moe_gemm_gate_up) instead of the GEMV.
    """
    _check_gpu("hidden", x, torch.bfloat16, 2)
    dev = x.device
    n_tok = x.shape[0]
    split = torch.empty((2, n_tok * k, inter), dtype=torch.bfloat16, device=dev)
    raw = torch.empty((n_tok * k, inter), dtype=torch.float32, device=dev) if want_raw else None
    nat.call("klc_moe_gemm_gate_up" if gemm else "klc_moe_gate_up", _ptr(table), _ptr(bias), _ptr(x), n_tok, k,
             disp.n_experts, _ptr(disp.offsets), _ptr(disp.sorted_pairs), _ptr(disp.units), hidden, inter,
             float(limit), PRECISIONS[precision], _ptr(split), _ptr(raw), _stream(dev))
    return (split, raw) if want_raw else split


def down(table: torch.Tensor, bias: torch.Tensor, gated_split: torch.Tensor, disp: Dispatch, hidden: int, inter: int,
         precision: str = "fp32", gemm: bool = False) -> torch.Tensor:
    """float32 expert outputs ``[P, H]`` (``gemm``: klc_moe_gemm_down instead of the GEMV)."""
    _check_gpu("gated_split", gated_split, torch.bfloat16, 3)
    dev = gated_split.device
    n_pairs = gated_split.shape[1]
    eo = torch.empty((n_pairs, hidden), dtype=torch.float32, device=dev)
    nat.call("klc_moe_gemm_down" if gemm else "klc_moe_down", _ptr(table), _ptr(bias), _ptr(gated_split), n_pairs,
             disp.n_experts, _ptr(disp.offsets), _ptr(disp.sorted_pairs), _ptr(disp.units), hidden, inter,
             PRECISIONS[precision], _ptr(eo), _stream(dev))
    return eo


def combine(expert_out: torch.Tensor, weights: torch.Tensor, n_tokens: int, k: int,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 weighted sum of the k expert outputs per token (+ ``residual`` if given)."""
    _check_gpu("expert_out", expert_out, torch.float32)
    _check_gpu("weights", weights, torch.bfloat16)
    hidden = expert_out.shape[-1]
    if residual is not None:
        _check_gpu("residual", residual, torch.bfloat16, 2)
        if tuple(residual.shape) != (n_tokens, hidden):
            raise ValueError(f"residual shape {tuple(residual.shape)} != ({n_tokens}, {hidden})")
    out = torch.empty((n_tokens, hidden), dtype=torch.bfloat16, device=expert_out.device)
    nat.call("klc_moe_combine", _ptr(expert_out), _ptr(weights), _ptr(residual), n_tokens, k, hidden, _ptr(out),
             _stream(expert_out.device))
    return out


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, out: torch.Tensor | None = None):
    """bf16 ``x [B, H]`` -> ``x * rsqrt(mean(x^2) + eps).to(bf16) * weight`` (klc_rms_norm)."""
    _check_gpu("x", x, torch.bfloat16, 2)
    _check_gpu("weight", weight, torch.bfloat16, 1)
    if weight.shape[0] != x.shape[1]:
        raise ValueError(f"norm weight of {weight.shape[0]} for hidden {x.shape[1]}")
    if out is None:
        out = torch.empty_like(x)
    nat.call("klc_rms_norm", _ptr(x), _ptr(weight), _ptr(out), x.shape[0], x.shape[1], float(eps), _stream(x.device))
    return out


def bias_combine(down_bias: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
    _check_gpu("down_bias", down_bias, torch.bfloat16, 2)
    _check_gpu("ids", ids, torch.int32, 2)
    _check_gpu("weights", weights, torch.bfloat16, 2)
    n_tok, k = ids.shape
    hidden = down_bias.shape[1]
    out = torch.empty((n_tok, hidden), dtype=torch.bfloat16, device=ids.device)
    nat.call("klc_moe_bias_combine", _ptr(down_bias), _ptr(ids), _ptr(weights), n_tok, k, hidden, _ptr(out),
             _stream(ids.device))
    return out


def pair_norms(gated: torch.Tensor, expert_out: torch.Tensor) -> torch.Tensor:
    _check_gpu("gated", gated, torch.float32, 2)
    _check_gpu("expert_out", expert_out, torch.float32, 2)
    norms = torch.empty((gated.shape[0], 2), dtype=torch.float32, device=gated.device)
    nat.call("klc_moe_pair_norms", _ptr(gated), _ptr(expert_out), gated.shape[0], gated.shape[1],
             expert_out.shape[1], _ptr(norms), _stream(gated.device))
    return norms


def workspace_bytes(n_tokens: int, hidden: int, inter: int, n_experts: int, k: int) -> int:
    return nat.call("klc_moe_workspace_bytes", n_tokens, hidden, inter, n_experts, k)


# ---- Attention of many sequences ---------------------------------------------------

_KV_CODES = {torch.bfloat16: nat.DTYPE_BF16, torch.float16: nat.DTYPE_F16}
_TENSORS = (torch.Tensor, torch.nn.Parameter)
# klc_attn_prompt_args, klc_kv_append_args and klc_attn_batch_args: pointers, sizes, scale
_PROMPT_ARGS = struct.Struct("=6Q10qd")
_APPEND_ARGS = struct.Struct("=11Q10q")
_BATCH_ARGS = struct.Struct("=9Q12qd")
_batch_bytes: dict = {}  # sizes -> klc_attn_batch's workspace bytes


def _plain(t, dtype: torch.dtype, shape: tuple, index: int) -> bool:
    """A contiguous tensor of this type and shape on GPU ``index``, with nothing more to look at."""
    return (type(t) in _TENSORS and t.dtype is dtype and t.shape == shape and t.get_device() == index
            and t.is_contiguous())


def _row_stride(name: str, t: torch.Tensor, dtype: torch.dtype, dev: torch.device) -> int:
    """The token stride of ``[tokens, heads, head_dim]`` with contiguous heads, a view of wider rows allowed."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on a GPU device (there is no CPU implementation), got {t.device}")
    if t.device != dev:
        raise ValueError(f"tensors on different devices: {dev} vs {t.device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != 3 or 0 in t.shape[1:]:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got shape {tuple(t.shape)}")
    _, heads, dim = t.shape
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires grad: this operator has no backward pass")
    stride = t.stride(0) if t.shape[0] > 1 else heads * dim
    if t.stride(2) != 1 or (heads > 1 and t.stride(1) != dim) or stride < heads * dim or stride % 8:
        raise ValueError(f"{name} needs contiguous heads and a token stride that is a multiple of 8, got strides {t.stride()}")
    return stride


def _row_strides(rows: tuple, dtype: torch.dtype, dev: torch.device) -> list[int]:
    """Token strides of the named tensors; the checks in full where one is not a plain contiguous tensor."""
    index, grad = dev.index, torch.is_grad_enabled()
    strides = []
    for name, t in rows:
        if (type(t) in _TENSORS and t.dtype is dtype and t.get_device() == index and t.is_contiguous()
                and not (grad and t.requires_grad)):
            shape = t.shape
            if len(shape) == 3:
                _, heads, dim = shape
                if heads and dim:
                    strides.append(heads * dim)
                    continue
        strides.append(_row_stride(name, t, dtype, dev))
    return strides


def _check_index(name: str, t: torch.Tensor, shape: tuple, dev: torch.device) -> None:
    if (type(t) in _TENSORS and t.dtype is torch.int32 and t.shape == shape and t.get_device() == dev.index
            and t.is_contiguous()):
        return
    _check_gpu(name, t, torch.int32, len(shape))
    if t.device != dev:
        raise ValueError(f"tensors on different devices: {dev} vs {t.device}")
    raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}") if t.shape != shape else TypeError(
        f"{name} must be a torch.Tensor, got {type(t).__name__}")


def _check_heads(sinks: torch.Tensor | None, n_heads: int, n_kv: int, window: int | None, scale: float | None, dim: int,
                 dev: torch.device) -> tuple[int, int, float]:
    """The sinks' address, the window as the library takes it, and the scale."""
    if n_heads % n_kv:
        raise ValueError(f"{n_heads} query heads over {n_kv} KV heads")
    if sinks is not None:
        if not _plain(sinks, torch.bfloat16, (n_heads,), dev.index):
            _check_gpu("sinks", sinks, torch.bfloat16, 1)
            raise ValueError(f"sinks must be [{n_heads}] on {dev}, got {tuple(sinks.shape)} on {sinks.device}")
        if sinks.requires_grad and torch.is_grad_enabled():
            raise ValueError("sinks require grad: this operator has no backward pass")
    if window is not None and operator.index(window) <= 0:
        raise ValueError(f"window must be positive (None: no window), got {window}")
    return (0 if sinks is None else sinks.data_ptr(), min(operator.index(window), (1 << 30) - 1) if window else 0,
            dim ** -0.5 if scale is None else float(scale))


def _result(name: str, out: torch.Tensor | None, like: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """``out``, or a new contiguous tensor as ``like`` (a view of wider rows of contiguous heads, so empty_like is)."""
    if out is None:
        return torch.empty_like(like)
    shape, dtype = like.shape, like.dtype
    if not _plain(out, dtype, shape, dev.index):
        _check_gpu(name, out, dtype)
        raise ValueError(f"{name} must be {tuple(shape)} on {dev}, got {tuple(out.shape)} on {out.device}")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires grad: this operator has no backward pass")
    return out


def _call(name: str, args: bytes, dev: torch.device) -> None:
    """``name(args, current stream)`` with the tensors' device current."""
    index = dev.index
    fn = getattr(nat.load(), name)
    if torch._C._cuda_getDevice() == index:
        rc = fn(args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(args, torch._C._cuda_getCurrentRawStream(index))
    if rc < 0:
        raise nat.KlcError(name, int(rc), nat.last_error())


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor,
                     sinks: torch.Tensor | None = None, window: int | None = None, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed prompts (klc_attn_prompt): ``q [T, n_heads, D]``, ``k``, ``v [T, n_kv, D]``, all
    bfloat16 or all float16 (views with contiguous heads too, such as splits of one projection), sequence ``s`` =
    tokens ``starts[s]:starts[s + 1]`` (int32 ``[S + 1]`` on the device, ascending) -> ``[T, n_heads, D]``.  A token
    sees the last ``window`` tokens up to itself (None: all); ``sinks`` bf16 ``[n_heads]``; ``scale`` 1 / sqrt(D)
    unless given.  Rows outside every sequence are left as ``out`` had them; ``out`` shares no memory with the inputs."""
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"q must be a torch.Tensor, got {type(q).__name__}")
    dev, dtype = q.device, q.dtype
    if dtype not in _KV_CODES:
        raise TypeError(f"q must be bfloat16 or float16, got {dtype}")
    strides = _row_strides((("q", q), ("k", k), ("v", v)), dtype, dev)
    shape = q.shape
    tokens, n_heads, dim = shape
    n_kv = k.shape[1]
    if k.shape != (tokens, n_kv, dim) or v.shape != k.shape:
        raise ValueError(f"shapes mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    n_seq = (starts.shape[0] if isinstance(starts, torch.Tensor) and starts.dim() == 1 else 1) - 1
    _check_index("starts", starts, (n_seq + 1,), dev)
    if n_seq < 0:
        raise ValueError("starts must hold the sequences' starts and the end of the last one")
    sink_ptr, window, scale = _check_heads(sinks, n_heads, n_kv, window, scale, dim, dev)
    out = _result("out", out, q, dev)
    if tokens and n_seq:
        _call("klc_attn_prompt",
              _PROMPT_ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), starts.data_ptr(), sink_ptr, out.data_ptr(),
                                tokens, n_seq, n_heads, n_kv, dim, *strides, window, _KV_CODES[dtype], scale), dev)
    return out


def _check_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, dev: torch.device) -> tuple[int, int, int, int]:
    if not (type(k_pages) in _TENSORS and k_pages.dtype in _KV_CODES and k_pages.dim() == 4 and k_pages.is_contiguous()
            and k_pages.get_device() == dev.index and _plain(v_pages, k_pages.dtype, k_pages.shape, dev.index)):
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            _check_gpu(name, t, None, 4)
            if t.dtype not in _KV_CODES:
                raise TypeError(f"{name} must be bfloat16 or float16, got {t.dtype}")
        if k_pages.device != dev or v_pages.device != dev:
            raise ValueError(f"tensors on different devices: {dev} vs {k_pages.device}, {v_pages.device}")
        if k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
            raise ValueError(f"page pools mismatch: {k_pages.dtype} {tuple(k_pages.shape)}, {v_pages.dtype} {tuple(v_pages.shape)}")
    if (k_pages.requires_grad or v_pages.requires_grad) and torch.is_grad_enabled():
        raise ValueError("pages require grad: this operator has no backward pass")
    n_pages, page, n_kv, dim = k_pages.shape
    if n_pages == 0 or page < 16 or page > 4096 or page & (page - 1):
        raise ValueError(f"pages must hold a power of two of tokens, 16 to 4096, got {n_pages} of {page}")
    if n_kv == 0 or dim == 0:
        raise ValueError(f"pages of no heads: {tuple(k_pages.shape)}")
    return n_pages, page, n_kv, dim


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 positions: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 want_keys: bool = True):
    """Rotates bf16 ``q [T, n_heads, D]`` and ``k [T, n_kv, D]`` by rows ``positions`` of the bf16 tables ``cos`` and
    ``sin [n, D / 2]`` and stores the keys and ``v [T, n_kv, D]`` to ``slots`` (int32 ``[T]``, distinct; page * page
    size + offset, negative: stored nowhere) of the pools ``[n_pages, page, n_kv, D]`` (klc_kv_append).  Returns the
    rotated bf16 ``(q, k)``, ``k`` None unless ``want_keys``."""
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"q must be a torch.Tensor, got {type(q).__name__}")
    dev = q.device
    strides = _row_strides((("q", q), ("k", k), ("v", v)), torch.bfloat16, dev)
    tokens, n_heads, dim = q.shape
    n_pages, page, n_kv, page_dim = _check_pages(k_pages, v_pages, dev)
    if k.shape != (tokens, n_kv, dim) or v.shape != k.shape or page_dim != dim:
        raise ValueError(f"shapes mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}, pages {tuple(k_pages.shape)}")
    n_pos = cos.shape[0] if isinstance(cos, torch.Tensor) and cos.dim() == 2 else 0
    for name, t in (("cos", cos), ("sin", sin)):
        if not _plain(t, torch.bfloat16, (n_pos, dim // 2), dev.index) or not n_pos:
            _check_gpu(name, t, torch.bfloat16, 2)
            raise ValueError(f"{name} must be [positions, {dim // 2}] on {dev}, got {tuple(t.shape)} on {t.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires grad: this operator has no backward pass")
    _check_index("positions", positions, (tokens,), dev)
    _check_index("slots", slots, (tokens,), dev)
    q_out = _result("q", None, q, dev)
    k_out = _result("k", None, k, dev) if want_keys else None
    if tokens:
        _call("klc_kv_append",
              _APPEND_ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                                positions.data_ptr(), slots.data_ptr(), q_out.data_ptr(),
                                k_out.data_ptr() if want_keys else 0, k_pages.data_ptr(), v_pages.data_ptr(), tokens,
                                n_pos, n_pages * page, n_heads, n_kv, dim, *strides, _KV_CODES[k_pages.dtype]), dev)
    return q_out, k_out


def _page_numbers(x) -> np.ndarray:
    a = np.asarray(x)
    if a.dtype != np.int32:
        if a.size and a.dtype.kind not in "iu":
            raise TypeError(f"page numbers must be whole numbers, got {a.dtype}")
        if a.size and (a.min() < 0 or a.max() > 0x7FFFFFFF):
            raise ValueError("page numbers must be in [0, 2^31)")
        a = a.astype(np.int32)
    return np.ascontiguousarray(a)


def copy_pages(pools: torch.Tensor, src, dst) -> None:
    """``pools[:, dst[i]] = pools[:, src[i]]`` for every i (klc_kv_copy_pages), for contiguous ``pools [n, n_pages,
    ...]`` and page numbers on the host (sequences or int32 arrays).  The moves run at once: a destination is no other
    move's source or destination."""
    _check_gpu("pools", pools)
    if pools.requires_grad and torch.is_grad_enabled():
        raise ValueError("pools require grad: this operator has no backward pass")
    if pools.dim() < 3 or pools.numel() == 0:
        raise ValueError(f"pools must be [pools, pages, ...], got shape {tuple(pools.shape)}")
    src, dst = _page_numbers(src), _page_numbers(dst)
    if src.ndim != 1 or src.shape != dst.shape:
        raise ValueError(f"source and destination pages mismatch: {src.shape} and {dst.shape}")
    dev = pools.device
    n_pools, n_pages = pools.shape[:2]
    page_bytes = pools.stride(1) * pools.element_size() if n_pages > 1 else pools[0].numel() * pools.element_size()
    with torch.cuda.device(dev) if torch._C._cuda_getDevice() != dev.index else contextlib.nullcontext():
        rc = nat.load().klc_kv_copy_pages(pools.data_ptr(), n_pools, n_pages, page_bytes, src.ctypes.data, dst.ctypes.data,
                                          src.size, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc == nat.KLC_ERR_ARGUMENT:
        raise ValueError(nat.last_error())
    if rc < 0:
        raise nat.KlcError("klc_kv_copy_pages", int(rc), nat.last_error())


def batch_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor,
                    lengths: torch.Tensor, prefix_table: torch.Tensor | None = None, prefix_len: int = 0,
                    sinks: torch.Tensor | None = None, window: int | None = None, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one token of each of B sequences over pages (klc_attn_batch): bf16 ``q [B, n_heads, D]``; sequence
    b's keys are the first ``prefix_len`` tokens of the pages ``prefix_table`` (int32, shared by all sequences; without a
    window a long one is read once for all of them) and then ``lengths[b]`` of the pages ``tables[b]`` (int32 ``[B, width]``), the token's own last.  ``lengths[b]
    < 0``: no sequence, zeros.  Other arguments as :func:`prompt_attention`; returns bf16 ``[B, n_heads, D]``."""
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"q must be a torch.Tensor, got {type(q).__name__}")
    dev = q.device
    stride, = _row_strides((("q", q),), torch.bfloat16, dev)
    shape = q.shape
    count, n_heads, dim = shape
    n_pages, page, n_kv, page_dim = _check_pages(k_pages, v_pages, dev)
    if page_dim != dim:
        raise ValueError(f"shapes mismatch: q {tuple(q.shape)}, pages {tuple(k_pages.shape)}")
    width = tables.shape[1] if isinstance(tables, torch.Tensor) and tables.dim() == 2 else 0
    _check_index("tables", tables, (count, width), dev)
    _check_index("lengths", lengths, (count,), dev)
    prefix_len = operator.index(prefix_len)
    if prefix_len < 0:
        raise ValueError(f"prefix_len must not be negative, got {prefix_len}")
    if prefix_len:
        if prefix_table is None:
            raise ValueError("prefix_len without a prefix_table")
        held = prefix_table.shape[0] if isinstance(prefix_table, torch.Tensor) and prefix_table.dim() == 1 else 0
        _check_index("prefix_table", prefix_table, (held,), dev)
        if held * page < prefix_len:
            raise ValueError(f"prefix of {prefix_len} tokens in {held} pages of {page}")
    sink_ptr, window, scale = _check_heads(sinks, n_heads, n_kv, window, scale, dim, dev)
    out = _result("out", out, q, dev)
    if not count:
        return out
    sizes = (count, n_heads, n_kv, dim, prefix_len, width * page, window)
    nbytes = _batch_bytes.get(sizes)
    if nbytes is None:
        if len(_batch_bytes) > 4096:
            _batch_bytes.clear()
        nbytes = _batch_bytes[sizes] = nat.call("klc_attn_batch_workspace_bytes", *sizes)
    # of this call alone: calls on other streams and captured graphs have theirs
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _call("klc_attn_batch",
          _BATCH_ARGS.pack(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), tables.data_ptr() if width else 0,
                           lengths.data_ptr(), prefix_table.data_ptr() if prefix_len else 0, sink_ptr,
                           workspace.data_ptr() if nbytes else 0, out.data_ptr(), count, n_heads, n_kv, dim, stride,
                           n_pages, page, width, prefix_len, window, _KV_CODES[k_pages.dtype], nbytes, scale), dev)
    return out


def synth_fill(dst: torch.Tensor, seed: int, mode: int = 0, lo: int = 0, hi: int = 255) -> torch.Tensor:
    """Fills a uint8 device tensor from the SplitMix64 stream (see klcquant_amd.synth)."""
    _check_gpu("dst", dst, torch.uint8)
    nat.call("klc_synth_fill", _ptr(dst), dst.numel(), ctypes.c_uint64(seed & ((1 << 64) - 1)), mode, lo, hi,
             _stream(dst.device))
    return dst
