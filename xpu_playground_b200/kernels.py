"""torch-tensor wrappers over the C ABI (one function per entry point).

These pass device pointers and sizes straight through to libxpu_cuda; torch
only provides device memory and the current CUDA stream. Every tensor must be
a contiguous CUDA tensor; 16-bit tensors are passed by their bit patterns.

With ``stream`` a call is queued on that stream; outputs that are not given are
then allocated for it. As with any torch operation on another stream, inputs
have to be ready there and other streams have to wait for the results.
"""

from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _lib
from ._lib import XPU_BF16, XPU_FP16, call


def _ptr(t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise ValueError("libxpu_cuda entry points take CUDA tensors")
    if not t.is_contiguous():
        raise ValueError("tensor must be contiguous")
    return t.data_ptr()


def _stream(stream=None) -> int:
    if stream is not None:
        return stream.cuda_stream
    # torch.cuda.current_stream().cuda_stream without building a Stream object (3 us)
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _allocate(make, stream, *args, **kwargs) -> torch.Tensor:
    """make(*args, **kwargs) for a kernel on `stream`: memory of that stream, so that nothing
    still queued elsewhere uses it, and kept from reuse until the current stream's work is done too."""
    if stream is None or stream == torch.cuda.current_stream(stream.device):
        return make(*args, **kwargs)
    current = torch.cuda.current_stream(stream.device)
    with torch.cuda.stream(stream):
        t = make(*args, **kwargs)
    t.record_stream(current)
    return t


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return XPU_BF16
    if t.dtype == torch.float16:
        return XPU_FP16
    raise ValueError(f"unsupported dtype {t.dtype}")


def gemv(matrix: torch.Tensor, vector: torch.Tensor, out: torch.Tensor | None = None,
         stream=None) -> torch.Tensor:
    m, k = matrix.shape
    if out is None:
        out = _allocate(torch.empty, stream, m, dtype=matrix.dtype, device=matrix.device)
    call("xpu_gemv", _dtype_code(matrix), _ptr(matrix), _ptr(vector), _ptr(out), m, k,
         _stream(stream))
    return out


def gemm_bt(a: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """C[m,n] = A[m,k] . W^T for W [n,k] (row-major, contiguous, bf16 or fp16)."""
    m, k = a.shape
    n, k2 = w.shape
    if k2 != k or a.dtype != w.dtype:
        raise ValueError("gemm_bt: A is [m,k] and W is [n,k] of the same dtype")
    if out is None:
        out = _allocate(torch.empty, stream, m, n, dtype=a.dtype, device=a.device)
    call("xpu_gemm_bt", _dtype_code(a), _ptr(a), _ptr(w), _ptr(out), m, n, k, _stream(stream))
    return out


def gemm(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None,
         stream=None) -> torch.Tensor:
    """C[m,n] = A[m,k] . B[k,n] (row-major, contiguous, bf16 or fp16)."""
    m, k = a.shape
    k2, n = b.shape
    if k2 != k or a.dtype != b.dtype:
        raise ValueError("gemm: A is [m,k] and B is [k,n] of the same dtype")
    if out is None:
        out = _allocate(torch.empty, stream, m, n, dtype=a.dtype, device=a.device)
    call("xpu_gemm", _dtype_code(a), _ptr(a), _ptr(b), _ptr(out), m, n, k, _stream(stream))
    return out


def device_status() -> int:
    """Reads and clears the library's sticky device error word (synchronises)."""
    flags = ctypes.c_uint32(0)
    call("xpu_device_status", ctypes.byref(flags))
    return flags.value


def peak_mem_fill(surface: torch.Tensor, stream=None) -> None:
    """surface[i] = 1 + (hash(i) & 0xffff) / 65536 (float32 tensor)."""
    call("xpu_peak_mem_fill", _ptr(surface), surface.numel(), _stream(stream))


def peak_mem_read(surface: torch.Tensor, sink: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """One read of a [height, 1024] float32 surface; returns the per-unit
    checksums (one per 2 KiB unit: height * 2 of them)."""
    height = surface.numel() // 1024
    if sink is None:
        sink = _allocate(torch.zeros, stream, height * 2, dtype=torch.float32, device=surface.device)
    call("xpu_peak_mem_read", _ptr(surface), _ptr(sink), height, _stream(stream))
    return sink


def peak_compute(ctas: int, rounds: int, sink: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """ctas x rounds x 8 tensor-core MMAs; returns sink (1 + 32 rounds each)."""
    if sink is None:
        sink = _allocate(torch.zeros, stream, ctas, dtype=torch.float32, device="cuda")
    call("xpu_peak_compute", _ptr(sink), ctas, rounds, _stream(stream))
    return sink


def qwen_embedding(table, output, token: int, width: int, stream=None):
    call("xpu_qwen_embedding", _ptr(table), _ptr(output), token, width, _stream(stream))


def qwen_rms_norm(inp, weight, output, width: int, epsilon: float = 1e-6, stream=None):
    call("xpu_qwen_rms_norm", _ptr(inp), _ptr(weight), _ptr(output), width, epsilon, _stream(stream))


def qwen_gemv(matrix, vector, output, rows: int, columns: int, stream=None):
    call("xpu_qwen_gemv", _ptr(matrix), _ptr(vector), _ptr(output), rows, columns, _stream(stream))


def qwen_qkv_rope_cache(query, key, value, query_norm, key_norm, rope_cos, rope_sin, key_cache,
                        value_cache, position: int, maximum_sequence: int, query_heads: int,
                        key_value_heads: int, stream=None):
    call("xpu_qwen_qkv_rope_cache", _ptr(query), _ptr(key), _ptr(value), _ptr(query_norm),
         _ptr(key_norm), _ptr(rope_cos), _ptr(rope_sin), _ptr(key_cache), _ptr(value_cache),
         position, maximum_sequence, query_heads, key_value_heads, _stream(stream))


def qwen_attention_workspace_size(query_heads: int, maximum_positions: int) -> int:
    return int(_lib.load().xpu_qwen_attention_workspace_size(query_heads, maximum_positions))


def qwen_attention(query, key_cache, value_cache, output, position: int, query_heads: int,
                   key_value_heads: int, workspace: torch.Tensor, stream=None):
    call("xpu_qwen_attention", _ptr(query), _ptr(key_cache), _ptr(value_cache), _ptr(output),
         position, query_heads, key_value_heads, _ptr(workspace),
         workspace.numel() * workspace.element_size(), _stream(stream))


def qwen_add(left, right, width: int, stream=None):
    call("xpu_qwen_add", _ptr(left), _ptr(right), width, _stream(stream))


def qwen_silu_multiply(gate, up, width: int, stream=None):
    call("xpu_qwen_silu_multiply", _ptr(gate), _ptr(up), width, _stream(stream))


def qwen_argmax(values, token, width: int, stream=None):
    call("xpu_qwen_argmax", _ptr(values), _ptr(token), width, _stream(stream))


# ------------------------------------------------- attention for serving ----

def _packed(name: str, t: torch.Tensor, heads: int, head_dim: int) -> int:
    """Row stride of a packed [tokens, heads, head_dim] tensor whose rows may
    stand apart (a slice of a fused projection)."""
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != head_dim:
        raise ValueError(f"{name} must be [tokens, {heads}, {head_dim}], not {tuple(shape)}")
    if not t.is_cuda:
        raise ValueError("libxpu_cuda entry points take CUDA tensors")
    if t.is_contiguous():
        return heads * head_dim
    row, head, element = t.stride()
    if element != 1 or (head != head_dim and heads != 1):
        raise ValueError(f"{name}: the heads of a token must be contiguous")
    return row if shape[0] > 1 else max(row, heads * head_dim)


def _attention_args(q, k, v, kv_heads, head_dim, scale, out, lse, stream):
    dtype, shape, kv_shape = q.dtype, q.shape, k.shape
    if k.dtype != dtype or v.dtype != dtype:
        raise ValueError("q, k and v must have one dtype")
    if len(shape) != 3 or shape[2] != head_dim or kv_shape != (shape[0], kv_heads, head_dim) or v.shape != kv_shape:
        raise ValueError(f"q must be [tokens, q_heads, {head_dim}], k and v [tokens, {kv_heads}, {head_dim}]")
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise ValueError("libxpu_cuda entry points take CUDA tensors")
    tokens, q_heads = shape[0], shape[1]
    q_stride = out_stride = q_heads * head_dim
    kv_stride = kv_heads * head_dim
    whole = q.is_contiguous()
    if not (whole and k.is_contiguous() and v.is_contiguous()):
        q_stride, kv_stride = _packed("q", q, q_heads, head_dim), _packed("k", k, kv_heads, head_dim)
        if _packed("v", v, kv_heads, head_dim) != kv_stride:
            raise ValueError("k and v need one row stride")
    # (empty_like, and sizes one by one, take half the time of a torch.Size)
    if out is None:
        out = (_allocate(torch.empty_like, stream, q) if whole else
               _allocate(torch.empty, stream, tokens, q_heads, head_dim, dtype=dtype, device=q.device))
    elif out.dtype != dtype or out.shape != shape:
        raise ValueError("out must have q's shape and dtype")
    else:
        out_stride = _packed("out", out, q_heads, head_dim)
    if lse is None:
        lse = _allocate(torch.empty, stream, tokens, q_heads, dtype=torch.float32, device=q.device)
    elif lse.dtype != torch.float32 or lse.shape != shape[:2] or not lse.is_cuda or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous float32 CUDA tensor [tokens, q_heads]")
    return out, lse, q_stride, kv_stride, out_stride, head_dim ** -0.5 if scale is None else scale


_copy_streams: dict[int, torch.cuda.Stream] = {}


class PromptPlan:
    """Which thread block computes which tiles of a batch of packed prompts
    (xpu_prompt_plan). It depends on the lengths and heads alone: make it once
    per batch and use it for every layer. Making it waits for its own copy to
    the device and for nothing that is queued there; any stream may use it."""

    def __init__(self, lens, q_heads: int, kv_heads: int, head_dim: int, device=None):
        n = np.ascontiguousarray(lens, dtype=np.uint32)
        used = ctypes.c_size_t()
        lib = _lib.load()
        room = 2048 + 4 * kv_heads * (n.size + int(n.sum()) * max(1, q_heads // max(1, kv_heads)) // 128 + 1)
        plan = np.empty(room, np.int32)
        status = lib.xpu_prompt_plan(n.ctypes.data, n.size, q_heads, kv_heads, plan.ctypes.data, plan.size,
                                     ctypes.byref(used))
        if status == _lib.XPU_ERR_INVALID and used.value > plan.size:
            plan = np.empty(used.value, np.int32)
            status = lib.xpu_prompt_plan(n.ctypes.data, n.size, q_heads, kv_heads, plan.ctypes.data, plan.size,
                                         ctypes.byref(used))
        _lib.check(status)
        self.blocks, self.tokens = int(plan[0]), int(plan[1])
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        device = torch.device(device or "cuda")
        index = torch.cuda.current_device() if device.index is None else device.index
        stream = _copy_streams.get(index)
        if stream is None:
            stream = _copy_streams[index] = torch.cuda.Stream(index)
        with torch.cuda.stream(stream):
            self.device_plan = torch.from_numpy(plan[:used.value]).to(f"cuda:{index}")
        self._readers: set[int] = set()  # streams that the memory is kept for when the plan goes

    def _read_on(self, stream, raw: int) -> None:
        self._readers.add(raw)
        self.device_plan.record_stream(stream if stream is not None else torch.cuda.current_stream())


def prompt_attention(plan: PromptPlan, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None,
                     out: torch.Tensor | None = None, lse: torch.Tensor | None = None, stream=None):
    """Causal attention over packed prompts (xpu_prompt_attention): q [tokens,
    q_heads, head_dim], k and v [tokens, kv_heads, head_dim], bf16 or fp16;
    scale defaults to 1 / sqrt(head_dim). Returns (out, lse)."""
    if q.shape[0] != plan.tokens or q.dim() != 3 or q.shape[1] != plan.q_heads:
        raise ValueError(f"q must be [{plan.tokens}, {plan.q_heads}, {plan.head_dim}] for this plan")
    out, lse, q_stride, kv_stride, out_stride, scale = _attention_args(q, k, v, plan.kv_heads, plan.head_dim, scale, out, lse,
                                                                    stream)
    raw = _stream(stream)
    if raw not in plan._readers:
        plan._read_on(stream, raw)
    call("xpu_prompt_attention", _dtype_code(q), plan.device_plan.data_ptr(), plan.blocks, q.data_ptr(), k.data_ptr(),
         v.data_ptr(), out.data_ptr(), lse.data_ptr(), plan.tokens, plan.q_heads, plan.kv_heads, plan.head_dim, q_stride,
         kv_stride, out_stride, scale, raw)
    return out, lse


def tree_attention_workspace(count: int, nodes: int, q_heads: int, kv_heads: int, head_dim: int,
                             device=None) -> torch.Tensor:
    """Zeroed workspace for tree_attention calls of up to `count` sequences
    and `nodes` drafted tokens in all."""
    size = int(_lib.load().xpu_tree_attention_workspace_size(count, nodes, q_heads, kv_heads, head_dim))
    return torch.zeros(size, dtype=torch.uint8, device=device or "cuda")


def tree_attention(cache, layer: int, sequences: torch.Tensor, starts: torch.Tensor, ancestors: torch.Tensor,
                   q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, workspace: torch.Tensor,
                   scale: float | None = None, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                   stream=None):
    """Attention of trees of drafted tokens over a KvCache
    (xpu_tree_attention): tree i is nodes starts[i] .. starts[i+1] - 1 of the
    packed q, k, v and continues sequences[i]; bit j of ancestors[r] lets node
    r attend node j of its tree. int32 sequences and starts, int64 ancestors.
    Returns (out, lse)."""
    if q.dtype != cache.dtype:
        raise ValueError("q, k and v must have the cache's dtype")
    if sequences.dtype != torch.int32 or starts.dtype != torch.int32 or ancestors.dtype != torch.int64:
        raise ValueError("sequences and starts are int32, ancestors int64")
    if starts.numel() != sequences.numel() + 1 or ancestors.numel() != q.shape[0]:
        raise ValueError("starts needs one entry more than sequences, ancestors one per node")
    out, lse, q_stride, kv_stride, out_stride, scale = _attention_args(q, k, v, cache.kv_heads, cache.head_dim, scale, out, lse,
                                                                    stream)
    call("xpu_tree_attention", cache.handle, layer, _ptr(sequences), _ptr(starts), _ptr(ancestors), sequences.numel(),
         q.shape[0], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), q.shape[1], q_stride, kv_stride,
         out_stride, scale, _ptr(workspace), workspace.numel(), _stream(stream))
    return out, lse


# ------------------------------------- 8-bit rows, their products, sampling ----

FP8 = torch.float8_e4m3fn
FP8_BLOCK = 128  # columns of a row, and rows and columns of a weight, that share a scale
_CODES = {torch.bfloat16: XPU_BF16, torch.float16: XPU_FP16}


def _code(dtype: torch.dtype) -> int:
    code = _CODES.get(dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {dtype}")
    return code


def _here(first: torch.Tensor, *others) -> None:
    """Refuses tensors that are not on the current device."""
    device = first.get_device()
    for t in others:
        if t is not None and t.get_device() != device:
            raise ValueError("tensors must be on one device")
    if device < 0:
        raise ValueError("libxpu_cuda entry points take CUDA tensors")
    if device != torch._C._cuda_getDevice():
        raise ValueError("tensors must be on the current device")


def _row_stride(name: str, t: torch.Tensor, width: int) -> int:
    """Row stride of [rows, width] whose rows may stand apart."""
    if t.is_contiguous():
        return width
    row, column = t.stride()
    if column != 1:
        raise ValueError(f"{name}: a row must be contiguous")
    return row if t.shape[0] > 1 else max(width, row)


def _fp8_outputs(rows: int, width: int, x, q, scales, stream):
    if q is None:
        q = _allocate(torch.empty, stream, (rows, width), dtype=FP8, device=x.device)
    elif q.dtype != FP8 or q.shape != (rows, width) or not q.is_contiguous():
        raise ValueError(f"q must be a contiguous float8_e4m3fn tensor {(rows, width)}")
    blocks = -(-width // FP8_BLOCK)
    if scales is None:
        scales = _allocate(torch.empty, stream, (blocks, rows), dtype=torch.float32, device=x.device)
    elif scales.dtype != torch.float32 or scales.shape != (blocks, rows) or not scales.is_contiguous():
        raise ValueError(f"scales must be a contiguous float32 tensor {(blocks, rows)}")
    return q, scales


def fp8_quantize(x: torch.Tensor, q: torch.Tensor | None = None, scales: torch.Tensor | None = None, stream=None):
    """Rows x [rows, width] in 8 bits (xpu_fp8_quantize): q [rows, width] and a
    scale for each 128 columns, scales [blocks, rows]. Returns (q, scales)."""
    rows, width = x.shape
    code, stride = _code(x.dtype), _row_stride("x", x, width)
    q, scales = _fp8_outputs(rows, width, x, q, scales, stream)
    _here(x, q, scales)
    call("xpu_fp8_quantize", code, x.data_ptr(), stride, q.data_ptr(), scales.data_ptr(), rows, width, _stream(stream))
    return q, scales


def fp8_silu_multiply(gate_up: torch.Tensor, q: torch.Tensor | None = None, scales: torch.Tensor | None = None, stream=None):
    """silu(gate) * up of a fused projection's rows [gate | up] in 8 bits
    (xpu_fp8_silu_multiply). Returns (q, scales)."""
    rows, both = gate_up.shape
    if both % 2:
        raise ValueError("gate_up holds gate and up side by side")
    width = both // 2
    code, stride = _code(gate_up.dtype), _row_stride("gate_up", gate_up, both)
    q, scales = _fp8_outputs(rows, width, gate_up, q, scales, stream)
    _here(gate_up, q, scales)
    at = gate_up.data_ptr()
    call("xpu_fp8_silu_multiply", code, at, at + 2 * width, stride, q.data_ptr(), scales.data_ptr(), rows, width, _stream(stream))
    return q, scales


def fp8_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, epsilon: float = 1e-6,
                 total: torch.Tensor | None = None, q: torch.Tensor | None = None, scales: torch.Tensor | None = None,
                 stream=None):
    """The residual's addition and the root-mean-square norm of the sum, the
    norm's rows in 8 bits (xpu_fp8_rms_norm). Returns (total, q, scales) with
    total = x + residual; `total` may be x or residual, to be updated in place.
    Without a residual total is x."""
    shape, dtype = x.shape, x.dtype
    rows, width = shape
    code, stride = _code(dtype), _row_stride("x", x, width)
    if weight.dtype != dtype or weight.shape != (width,) or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous tensor [{width}] of x's dtype")
    residual_at = residual_stride = total_at = total_stride = 0
    if residual is not None:
        if residual.dtype != dtype or residual.shape != shape:
            raise ValueError("residual must have x's shape and dtype")
        residual_at, residual_stride = residual.data_ptr(), _row_stride("residual", residual, width)
        if total is None:
            total = _allocate(torch.empty, stream, rows, width, dtype=dtype, device=x.device)
    if total is not None:
        if total.dtype != dtype or total.shape != shape:
            raise ValueError("total must have x's shape and dtype")
        total_at, total_stride = total.data_ptr(), _row_stride("total", total, width)
    q, scales = _fp8_outputs(rows, width, x, q, scales, stream)
    _here(x, weight, residual, total, q, scales)
    call("xpu_fp8_rms_norm", code, x.data_ptr(), stride, residual_at, residual_stride, weight.data_ptr(), epsilon, total_at,
         total_stride, q.data_ptr(), scales.data_ptr(), rows, width, _stream(stream))
    return (x if total is None else total), q, scales


def fp8_gemm(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
             out: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16, stream=None) -> torch.Tensor:
    """C[m, n] = A[m, k] . W[n, k]^T of 8-bit rows (with scales [blocks of k, m])
    and 8-bit weights (scales [blocks of n, blocks of k]), in `dtype` or out's
    (xpu_fp8_gemm)."""
    m, k = a.shape
    n, k2 = w.shape
    blocks = -(-k // FP8_BLOCK)
    if k2 != k or a.dtype != FP8 or w.dtype != FP8:
        raise ValueError("fp8_gemm: a is [m, k] and w is [n, k], both float8_e4m3fn")
    if a_scales.shape != (blocks, m) or w_scales.shape != (-(-n // FP8_BLOCK), blocks):
        raise ValueError("fp8_gemm: a_scales is [blocks of k, m], w_scales [blocks of n, blocks of k]")
    if a_scales.dtype != torch.float32 or w_scales.dtype != torch.float32:
        raise ValueError("fp8_gemm: scales are float32")
    if not (a.is_contiguous() and w.is_contiguous() and a_scales.is_contiguous() and w_scales.is_contiguous()):
        raise ValueError("tensor must be contiguous")
    if out is None:
        out = _allocate(torch.empty, stream, m, n, dtype=dtype, device=a.device)
    elif out.shape != (m, n) or not out.is_contiguous():
        raise ValueError("fp8_gemm: out must be a contiguous tensor [m, n]")
    code = _code(out.dtype)
    _here(a, a_scales, w, w_scales, out)
    call("xpu_fp8_gemm", code, a.data_ptr(), a_scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(), out.data_ptr(), m, n, k,
         _stream(stream))
    return out


def _per_row(name: str, t: torch.Tensor | None, dtype: torch.dtype, rows: int) -> int:
    if t is None:
        return 0
    if t.dtype != dtype or t.shape != (rows,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor with an entry a row")
    return t.data_ptr()


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: torch.Tensor | None = None, top_k: torch.Tensor | None = None,
           top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None, tokens: torch.Tensor | None = None,
           logprobs: torch.Tensor | None = None, stream=None):
    """A token for each row of logits [rows, vocabulary] from random numbers u
    in [0, 1), with each row's settings (xpu_sample): float32 temperature, top_p,
    min_p and int32 top_k of one entry a row. Returns (tokens, logprobs)."""
    rows, vocabulary = logits.shape
    code, stride = _code(logits.dtype), _row_stride("logits", logits, vocabulary)
    if u is None:
        raise ValueError("u needs a random number a row")
    f, i = torch.float32, torch.int32
    settings = (_per_row("temperature", temperature, f, rows), _per_row("top_k", top_k, i, rows), _per_row("top_p", top_p, f, rows),
                _per_row("min_p", min_p, f, rows), _per_row("u", u, f, rows))
    if tokens is None:
        tokens = _allocate(torch.empty, stream, rows, dtype=i, device=logits.device)
    if logprobs is None:
        logprobs = _allocate(torch.empty, stream, rows, dtype=f, device=logits.device)
    outputs = _per_row("tokens", tokens, i, rows), _per_row("logprobs", logprobs, f, rows)
    _here(logits, u, temperature, top_k, top_p, min_p, tokens, logprobs)
    call("xpu_sample", code, logits.data_ptr(), stride, *settings, *outputs, rows, vocabulary, _stream(stream))
    return tokens, logprobs
