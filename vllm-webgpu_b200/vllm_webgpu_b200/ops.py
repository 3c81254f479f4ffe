"""PyTorch-facing operators over libggufmm (CUDA tensors in, CUDA tensors out).

These are the calls the model linear layers make in place of the reference's
``_dispatch("matmul_quant", [x, W, scales, out], {K, N, USE_QUANT}, ...)``
(vllm_webgpu/models/base.py:62-100, vllm_webgpu/models/llama.py:276-283).
Every function launches hand-written sm_100a kernels on the current CUDA
stream and returns without synchronizing. There is no CPU path: tensors must
live on a CUDA device and the native library must be present.
"""
from __future__ import annotations

import struct

import torch

from . import _lib
from .formats import GGUFQuantTensor

_DTYPE_CODE = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}

GEMV_MAX_M = 8


def _code(dtype: torch.dtype) -> int:
    if dtype not in _DTYPE_CODE:
        raise ValueError(f"unsupported dtype {dtype}; expected float32, float16 or bfloat16")
    return _DTYPE_CODE[dtype]


def _require_cuda(*ts: torch.Tensor) -> torch.device:
    dev = ts[0].device
    for t in ts:
        if t.device.type != "cuda":
            raise ValueError("libggufmm operates on CUDA tensors only (no CPU fallback)")
        if t.device != dev:
            raise ValueError(f"tensors on different devices: {t.device} vs {dev}")
    return dev


def _stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _as_2d(x: torch.Tensor, k: int) -> torch.Tensor:
    if x.shape[-1] != k:
        raise ValueError(f"activation last dim {x.shape[-1]} != K={k}")
    x2 = x.reshape(-1, k)
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    return x2


def _out(x2: torch.Tensor, n: int, out: torch.Tensor | None, out_dtype: torch.dtype | None) -> torch.Tensor:
    m = x2.shape[0]
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype or x2.dtype, device=x2.device)
    else:
        if out.dim() != 2 or out.shape[0] != m or out.shape[1] != n or out.stride(1) != 1:
            raise ValueError(f"out must be a row-major [{m}, {n}] tensor")
    return out


def dequantize(w: GGUFQuantTensor, out_dtype: torch.dtype = torch.float32,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """[N, K] dequantized weights; float32 output is bit-identical to
    gguf.quants.dequantize (the reference loader's decoder)."""
    dev = _require_cuda(w.data)
    n, k = w.shape
    if out is None:
        out = torch.empty((n, k), dtype=out_dtype, device=dev)
    elif out.shape != (n, k) or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous [{n}, {k}] tensor")
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_dequantize(w.data.data_ptr(), w.qtype, n, k, out.data_ptr(),
                                          _code(out.dtype), _stream(dev))
    _lib.check(st, "ggufmm_dequantize")
    return out


def embedding(ids: torch.Tensor, table: GGUFQuantTensor, out: torch.Tensor | None = None,
              out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Rows ``ids`` of a GGUF-quantized embedding table, dequantized: out[t, :] =
    table[ids[t], :]. Replaces the reference's ``embedding_lookup`` dispatch
    (vllm_webgpu/models/llama.py:170-178), which copied rows of an f16 table.
    float32 output is bit-identical to gguf.quants.dequantize of the row. An id
    outside the table gives a zero row and sets bit 2 of the device status word."""
    dev = _require_cuda(ids, table.data)
    ids32 = ids.reshape(-1)
    if ids32.dtype != torch.int32 or not ids32.is_contiguous():
        ids32 = ids32.to(torch.int32).contiguous()
    n_ids = ids32.numel()
    if out is None:
        out = torch.empty((n_ids, table.k), dtype=out_dtype, device=dev)
    elif out.dim() != 2 or out.shape != (n_ids, table.k) or out.stride(1) != 1:
        raise ValueError(f"out must be a row-major [{n_ids}, {table.k}] tensor")
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_embedding(table.data.data_ptr(), table.qtype, table.n, table.k, ids32.data_ptr(),
                                         n_ids, out.data_ptr(), _code(out.dtype), out.stride(0), _stream(dev))
    _lib.check(st, "ggufmm_embedding")
    return out


def stage_copy(dst: torch.Tensor, src: torch.Tensor) -> torch.Tensor:
    """dst <- src by a kernel, where one side is page-locked host memory and the other
    a CUDA tensor (both contiguous, same byte size, 16-byte aligned): the decode step's
    host <-> device staging on the SMs instead of a copy engine, chained with the
    projections by programmatic dependent launch. Replaces the reference's buffer
    upload / staging readback (vllm_webgpu/webgpu/buffer.py:34, :46-63). Ordered on
    the CUDA tensor's device's current stream."""
    dev = dst.device if dst.is_cuda else src.device
    if not dev.type == "cuda":
        raise ValueError("stage_copy needs a CUDA tensor on one side")
    host = src if dst.is_cuda else dst
    if host.device.type == "cpu" and not host.is_pinned():
        raise ValueError("the host side of stage_copy must be pinned")
    if not (dst.is_contiguous() and src.is_contiguous()):
        raise ValueError("stage_copy needs contiguous tensors")
    nbytes = dst.numel() * dst.element_size()
    if nbytes != src.numel() * src.element_size():
        raise ValueError("stage_copy: byte sizes differ")
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_stage_copy(dst.data_ptr(), src.data_ptr(), nbytes, _stream(dev))
    _lib.check(st, "ggufmm_stage_copy")
    return dst


def staged_copy(dst: torch.Tensor, src: torch.Tensor) -> None:
    """The serving graphs' host <-> device copy: ``stage_copy`` where its conditions
    hold (GGUFMM_STAGE_KERNEL=0 keeps the copy-engine memcpy), else ``dst.copy_``."""
    import os
    if (os.environ.get("GGUFMM_STAGE_KERNEL", "1") != "0" and dst.is_contiguous() and src.is_contiguous()
            and dst.data_ptr() % 16 == 0 and src.data_ptr() % 16 == 0 and dst.dtype == src.dtype
            and dst.numel() == src.numel() and (dst.is_cuda != src.is_cuda)):
        stage_copy(dst, src)
    else:
        dst.copy_(src, non_blocking=True)


def gemv(x: torch.Tensor, w: GGUFQuantTensor, out: torch.Tensor | None = None,
         out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Decode GEMV, M <= 8 tokens: out[m, n] = sum_k x[m, k] W[n, k]."""
    dev = _require_cuda(x, w.data)
    x2 = _as_2d(x, w.k)
    y = _out(x2, w.n, out, out_dtype)
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_gemv(w.data.data_ptr(), w.qtype, w.n, w.k, x2.data_ptr(), _code(x2.dtype),
                                    x2.shape[0], x2.stride(0), y.data_ptr(), _code(y.dtype), y.stride(0),
                                    _stream(dev))
    _lib.check(st, "ggufmm_gemv")
    return y


GEMV_STREAM, GEMV_F16, GEMV_INT8 = 0, 1, 2
_gemv_kernels: dict = {}


def gemv_kernel(m: int, w: GGUFQuantTensor, x_dtype: torch.dtype = torch.bfloat16) -> int:
    """Which decode GEMV kernel ``gemv`` launches for M tokens against ``w`` on the
    weight's device: GEMV_INT8, GEMV_F16 or GEMV_STREAM (the CUDA-core fallback), or
    ``_lib.ERR_ALIGN`` when no decode GEMV can stage the weight's rows."""
    dev = _require_cuda(w.data)
    key = (dev.index, w.qtype, w.n, w.k, m, x_dtype)
    kind = _gemv_kernels.get(key)
    if kind is None:
        with torch.cuda.device(dev):
            kind = int(_lib.lib().ggufmm_gemv_kernel(w.qtype, w.n, w.k, m, _code(x_dtype)))
        if kind != _lib.ERR_ALIGN:  # ERR_ALIGN: no decode GEMV can stage these rows
            _lib.check(min(kind, 0), "ggufmm_gemv_kernel")
        _gemv_kernels[key] = kind
    return kind


def gemv_preferred(m: int, w: GGUFQuantTensor, x_dtype: torch.dtype = torch.bfloat16) -> bool:
    """Whether the decode GEMV is the faster path for M tokens: M <= 8, and for
    Q4_K a tensor-core GEMV fits the shape (where only the streaming fallback
    does, as for M = 8 at K = 14336, the tcgen05 GEMM with fused dequantization
    is 2-4x faster)."""
    if not 1 <= m <= GEMV_MAX_M:
        return False
    kind = gemv_kernel(m, w, x_dtype)
    return kind >= 0 and (w.qtype != 12 or kind != GEMV_STREAM)


def gemv_grouped(x: torch.Tensor, ws: list[GGUFQuantTensor], outs: list[torch.Tensor] | None = None,
                 out_dtype: torch.dtype | None = None) -> list[torch.Tensor]:
    """Decode GEMV of up to 4 weights sharing the activations (fused q/k/v or
    gate/up) in one launch; returns one [M, N_i] output per weight."""
    if not 1 <= len(ws) <= 4:
        raise ValueError("gemv_grouped takes 1 to 4 weights")
    k, qt = ws[0].k, ws[0].qtype
    if any(w.k != k or w.qtype != qt for w in ws):
        raise ValueError("grouped weights must share K and the quantization type")
    dev = _require_cuda(x, *[w.data for w in ws])
    x2 = _as_2d(x, k)
    if outs is None:
        outs = [None] * len(ws)
    ys = [_out(x2, w.n, o, out_dtype) for w, o in zip(ws, outs)]
    if len({y.dtype for y in ys}) != 1:
        raise ValueError("grouped outputs must share a dtype")
    import ctypes
    nseg = len(ws)
    qs = (ctypes.c_void_p * nseg)(*[w.data.data_ptr() for w in ws])
    ns = (ctypes.c_int64 * nseg)(*[w.n for w in ws])
    yp = (ctypes.c_void_p * nseg)(*[y.data_ptr() for y in ys])
    ld = (ctypes.c_int64 * nseg)(*[y.stride(0) for y in ys])
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_gemv_grouped(nseg, qs, ns, qt, k, x2.data_ptr(), _code(x2.dtype), x2.shape[0],
                                            x2.stride(0), yp, _code(ys[0].dtype), ld, _stream(dev))
    _lib.check(st, "ggufmm_gemv_grouped")
    return ys


def swiglu_fusable(x: torch.Tensor, gate: GGUFQuantTensor, up: GGUFQuantTensor) -> bool:
    """Whether gemv_swiglu handles these operands (decode M, Q4_K / Q4_0, K % 256 == 0,
    and the activations fit the integer GEMV's shared memory)."""
    m = x.numel() // max(x.shape[-1], 1)
    return (x.is_cuda and 1 <= m <= GEMV_MAX_M and gate.qtype == up.qtype and gate.qtype in (2, 12)
            and gate.shape == up.shape and gate.k % 256 == 0 and x.shape[-1] == gate.k
            and gemv_kernel(m, gate, x.dtype) == GEMV_INT8)


def gemv_swiglu(x: torch.Tensor, gate: GGUFQuantTensor, up: GGUFQuantTensor, out: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Fused FFN input for decode (M <= 8): out = silu(x gate^T) * (x up^T), one launch
    (the gate and up GEMVs and the SwiGLU of the reference's three dispatches)."""
    if gate.shape != up.shape or gate.qtype != up.qtype:
        raise ValueError("gate and up must share shape and quantization type")
    dev = _require_cuda(x, gate.data, up.data)
    x2 = _as_2d(x, gate.k)
    y = _out(x2, gate.n, out, out_dtype)
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_gemv_swiglu(gate.data.data_ptr(), up.data.data_ptr(), gate.qtype, gate.n, gate.k,
                                           x2.data_ptr(), _code(x2.dtype), x2.shape[0], x2.stride(0),
                                           y.data_ptr(), _code(y.dtype), y.stride(0), _stream(dev))
    _lib.check(st, "ggufmm_gemv_swiglu")
    return y


def residual_fusable(x: torch.Tensor, w: GGUFQuantTensor) -> bool:
    """Whether gemv_residual handles these operands (decode M on the integer GEMV)."""
    m = x.numel() // max(x.shape[-1], 1)
    return (x.is_cuda and w.qtype in (2, 12) and w.k % 256 == 0 and x.shape[-1] == w.k
            and gemv_preferred(m, w, x.dtype) and gemv_kernel(m, w, x.dtype) == GEMV_INT8)


def gemv_residual(x: torch.Tensor, w: GGUFQuantTensor, residual: torch.Tensor,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Decode GEMV with the residual add fused: out = x W^T + residual, one launch,
    the sum rounded once into out's dtype (= residual's). ``out`` may be
    ``residual`` itself (in place)."""
    dev = _require_cuda(x, w.data, residual)
    x2 = _as_2d(x, w.k)
    r2 = residual.reshape(-1, w.n) if residual.dim() != 2 else residual
    if r2.shape != (x2.shape[0], w.n) or r2.stride(1) != 1:
        raise ValueError(f"residual must be [{x2.shape[0]}, {w.n}] with unit column stride")
    y = _out(x2, w.n, out, r2.dtype)
    if y.dtype != r2.dtype:
        raise ValueError("out and residual must share a dtype")
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_gemv_residual(w.data.data_ptr(), w.qtype, w.n, w.k, x2.data_ptr(), _code(x2.dtype),
                                             x2.shape[0], x2.stride(0), y.data_ptr(), _code(y.dtype), y.stride(0),
                                             r2.data_ptr(), r2.stride(0), _stream(dev))
    _lib.check(st, "ggufmm_gemv_residual")
    return y


_ffn_workspaces: dict = {}


def _ffn_workspace(w: GGUFQuantTensor, m: int, swiglu: bool) -> torch.Tensor:
    need = int(_lib.lib().ggufmm_gemm_ffn_workspace_size(w.qtype, m, w.n, w.k, int(swiglu)))
    idx = w.data.device.index
    ws = _ffn_workspaces.get(idx)
    if ws is None or ws.numel() < need:
        ws = torch.empty(max(need, 256), dtype=torch.uint8, device=w.data.device)
        _ffn_workspaces[idx] = ws
    return ws


def gemm_swiglu(x: torch.Tensor, gate: GGUFQuantTensor, up: GGUFQuantTensor, out: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """out = silu(x gate^T) * (x up^T) at any M through the tensor-core GEMM with the
    SwiGLU in its epilogue pass (ggufmm_gemm_swiglu), replacing the reference's gate and
    up dispatches and its gelu_mul shader (vllm_webgpu/models/llama.py:343-352)."""
    if gate.shape != up.shape or gate.qtype != up.qtype:
        raise ValueError("gate and up must share shape and quantization type")
    dev = _require_cuda(x, gate.data, up.data)
    x2 = _as_2d(x, gate.k)
    y = _out(x2, gate.n, out, out_dtype)
    ws = _ffn_workspace(gate, x2.shape[0], True)
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_gemm_swiglu(gate.data.data_ptr(), up.data.data_ptr(), gate.qtype, gate.n, gate.k,
                                           x2.data_ptr(), _code(x2.dtype), x2.shape[0], x2.stride(0), y.data_ptr(),
                                           _code(y.dtype), y.stride(0), ws.data_ptr(), ws.numel(), _stream(dev))
    _lib.check(st, "ggufmm_gemm_swiglu")
    return y


def gemm_residual(x: torch.Tensor, w: GGUFQuantTensor, residual: torch.Tensor,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """out = x W^T + residual at any M, the add in the GEMM's epilogue pass
    (ggufmm_gemm_residual); ``out`` may be ``residual`` (in place)."""
    dev = _require_cuda(x, w.data, residual)
    x2 = _as_2d(x, w.k)
    r2 = residual.reshape(-1, w.n) if residual.dim() != 2 else residual
    if r2.shape != (x2.shape[0], w.n) or r2.stride(1) != 1:
        raise ValueError(f"residual must be [{x2.shape[0]}, {w.n}] with unit column stride")
    y = _out(x2, w.n, out, r2.dtype)
    if y.dtype != r2.dtype:
        raise ValueError("out and residual must share a dtype")
    ws = _ffn_workspace(w, x2.shape[0], False)
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_gemm_residual(w.data.data_ptr(), w.qtype, w.n, w.k, x2.data_ptr(), _code(x2.dtype),
                                             x2.shape[0], x2.stride(0), y.data_ptr(), _code(y.dtype), y.stride(0),
                                             r2.data_ptr(), r2.stride(0), ws.data_ptr(), ws.numel(), _stream(dev))
    _lib.check(st, "ggufmm_gemm_residual")
    return y


def ffn_epilogue(sums: torch.Tensor, n: int, out: torch.Tensor, swiglu: bool,
                 residual: torch.Tensor | None = None) -> torch.Tensor:
    """The epilogue pass over fp32 sums (ggufmm_ffn_epilogue): swiglu, sums [M, 2n] (gate |
    up) -> out = silu(gate) * up; else sums [M, n] -> out = sums + residual."""
    dev = _require_cuda(sums, out)
    if sums.dtype != torch.float32 or not sums.is_contiguous():
        raise ValueError("sums must be contiguous float32")
    m = sums.shape[0]
    r = residual.reshape(m, n) if residual is not None else None
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_ffn_epilogue(sums.data_ptr(), m, n, int(swiglu), r.data_ptr() if r is not None else None,
                                            r.stride(0) if r is not None else 0, out.data_ptr(), _code(out.dtype),
                                            out.stride(0), _stream(dev))
    _lib.check(st, "ggufmm_ffn_epilogue")
    return out


def swiglu(x: torch.Tensor, gate: GGUFQuantTensor, up: GGUFQuantTensor, out: torch.Tensor | None = None,
           out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """silu(x gate^T) * (x up^T) on the fastest native path: the one-launch integer decode
    GEMV where it serves the shape; other decode shapes run the grouped decode GEMV into
    fp32 sums and the epilogue pass; above the GEMV the GEMM with the SwiGLU epilogue."""
    x2 = _as_2d(x, gate.k)
    m = x2.shape[0]
    if swiglu_fusable(x2, gate, up):
        try:
            return gemv_swiglu(x2, gate, up, out=out, out_dtype=out_dtype)
        except ValueError as exc:
            if not _lib.is_align_refusal(exc):
                raise
    if gemv_preferred(m, gate, x2.dtype) and gate.shape == up.shape and gate.qtype == up.qtype:
        sums = torch.empty((m, 2 * gate.n), dtype=torch.float32, device=x2.device)
        gemv_grouped(x2, [gate, up], outs=[sums[:, :gate.n], sums[:, gate.n:]])
        y = _out(x2, gate.n, out, out_dtype)
        return ffn_epilogue(sums, gate.n, y, swiglu=True)
    return gemm_swiglu(x2, gate, up, out=out, out_dtype=out_dtype)


def linear_residual(x: torch.Tensor, w: GGUFQuantTensor, residual: torch.Tensor,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """x W^T + residual on the fastest native path: the integer decode GEMV with the add in
    its epilogue, other decode shapes as a GEMV into fp32 plus the epilogue pass, above
    the GEMV the GEMM with the add in its epilogue pass."""
    x2 = _as_2d(x, w.k)
    m = x2.shape[0]
    if residual_fusable(x2, w):
        try:
            return gemv_residual(x2, w, residual, out=out)
        except ValueError as exc:
            if not _lib.is_align_refusal(exc):
                raise
    if gemv_preferred(m, w, x2.dtype):
        sums = gemv(x2, w, out_dtype=torch.float32)
        r2 = residual.reshape(m, w.n)
        y = _out(x2, w.n, out, r2.dtype)
        return ffn_epilogue(sums, w.n, y, swiglu=False, residual=r2)
    return gemm_residual(x2, w, residual, out=out)


class PeerExchange:
    """Exchange buffers for ``gemv_allreduce`` on every GPU of a process group:
    one symmetric-memory allocation per GPU (``torch.distributed._symmetric_memory``,
    CUDA IPC between the GPUs of one node), zero-filled, with the peer addresses
    and the epoch counter the kernel needs. Creating it is a collective."""

    def __init__(self, n: int, m_max: int, group=None, device: torch.device | None = None):
        import ctypes

        import torch.distributed as dist
        import torch.distributed._symmetric_memory as symm_mem
        group = group or dist.group.WORLD
        self.world, self.rank = dist.get_world_size(group), dist.get_rank(group)
        self.n, self.m_max = n, m_max
        nbytes = int(_lib.lib().ggufmm_gemv_allreduce_buffer_bytes(n, m_max, self.world))
        if nbytes == 0:
            raise ValueError(f"no peer exchange for n={n}, m_max={m_max}, world={self.world}")
        device = device or torch.device("cuda", torch.cuda.current_device())
        try:
            symm_mem.enable_symm_mem_for_group(group.group_name)
        except Exception:  # already enabled, or not needed by this torch
            pass
        self.buf = symm_mem.empty(nbytes, dtype=torch.uint8, device=device)
        self.buf.zero_()
        self.handle = symm_mem.rendezvous(self.buf, group.group_name)
        torch.cuda.synchronize(device)
        dist.barrier(group)  # every buffer is zero before any GPU publishes into it
        self.ptrs = (ctypes.c_void_p * self.world)(*self.handle.buffer_ptrs)
        self.epoch = 0


class PeerAllReduce:
    """One-shot fp32 all-reduce over NVLink peer memory (ggufmm_allreduce) for vectors of
    up to 65536 values: one symmetric-memory exchange buffer per GPU of the group
    (``torch.distributed._symmetric_memory``), zero-filled. Creating it is a collective;
    calls must be made by every rank in the same order, and may be captured in a CUDA
    graph (the call's generation counter lives in device memory)."""

    MAX_N = 1 << 16

    def __init__(self, n: int, group=None, device: torch.device | None = None):
        import ctypes

        import torch.distributed as dist
        import torch.distributed._symmetric_memory as symm_mem
        group = group or dist.group.WORLD
        self.world, self.rank, self.n = dist.get_world_size(group), dist.get_rank(group), n
        nbytes = int(_lib.lib().ggufmm_allreduce_buffer_bytes(n, self.world))
        if nbytes == 0:
            raise ValueError(f"no peer all-reduce for n={n} (a multiple of 4, at most {self.MAX_N} values)")
        device = device or torch.device("cuda", torch.cuda.current_device())
        try:
            symm_mem.enable_symm_mem_for_group(group.group_name)
        except Exception:  # already enabled, or not needed by this torch
            pass
        self.buf = symm_mem.empty(nbytes, dtype=torch.uint8, device=device)
        self.buf.zero_()
        self.handle = symm_mem.rendezvous(self.buf, group.group_name)
        torch.cuda.synchronize(device)
        dist.barrier(group)  # every buffer is zero before any GPU publishes into it
        self.ptrs = (ctypes.c_void_p * self.world)(*self.handle.buffer_ptrs)

    def __call__(self, x: torch.Tensor, out: torch.Tensor | None = None,
                 residual: torch.Tensor | None = None) -> torch.Tensor:
        """out = the sum of every rank's x (+ residual), identical on every rank; x, out
        and residual fp32, contiguous, n values; out may be x."""
        if x.dtype != torch.float32 or not x.is_contiguous() or x.numel() != self.n:
            raise ValueError(f"x must be a contiguous float32 tensor of {self.n} values")
        out = x if out is None else out
        dev = x.device
        with torch.cuda.device(dev):
            st = _lib.lib().ggufmm_allreduce(x.data_ptr(), out.data_ptr(), self.n, self.ptrs, self.world, self.rank,
                                             residual.data_ptr() if residual is not None else None, _stream(dev))
        _lib.check(st, "ggufmm_allreduce")
        return out


class PeerGather:
    """Output buffers for the N-split GEMM whose epilogue all-gathers over NVLink
    (``gemm_allgather``): on every GPU of the group one symmetric-memory buffer holding
    the device barrier's flags and the full [m, n_total] output. Creating it is a
    collective. ``y`` is this GPU's full output (valid after ``gemm_allgather``)."""

    def __init__(self, m: int, n_total: int, dtype: torch.dtype = torch.bfloat16, group=None,
                 device: torch.device | None = None):
        import ctypes

        import torch.distributed as dist
        import torch.distributed._symmetric_memory as symm_mem
        group = group or dist.group.WORLD
        self.world, self.rank, self.m, self.n_total, self.dtype = (dist.get_world_size(group),
                                                                   dist.get_rank(group), m, n_total, dtype)
        es = torch.empty((), dtype=dtype).element_size()
        device = device or torch.device("cuda", torch.cuda.current_device())
        try:
            symm_mem.enable_symm_mem_for_group(group.group_name)
        except Exception:  # already enabled, or not needed by this torch
            pass
        self.hdr = int(_lib.lib().ggufmm_allreduce_buffer_bytes(0, self.world))  # the barrier's flags
        self.buf = symm_mem.empty(self.hdr + m * n_total * es, dtype=torch.uint8, device=device)
        self.buf.zero_()
        self.handle = symm_mem.rendezvous(self.buf, group.group_name)
        torch.cuda.synchronize(device)
        dist.barrier(group)
        self.ptrs = (ctypes.c_void_p * self.world)(*self.handle.buffer_ptrs)
        self.y_ptrs = (ctypes.c_void_p * self.world)(*[p + self.hdr for p in self.handle.buffer_ptrs])
        self.y = self.buf[self.hdr:].view(dtype).view(m, n_total)


def gemm_allgather(x: torch.Tensor, w_local: GGUFQuantTensor, gather: PeerGather) -> torch.Tensor:
    """x @ W^T for a weight split by output rows over the gather's GPUs: this rank's slice
    ``w_local`` (n_total / world rows) is multiplied and every value is stored into every
    GPU's output at its column (the all-gather in the GEMM's epilogue); a device-side
    barrier then makes the full [M, n_total] output ``gather.y`` valid on every GPU."""
    dev = _require_cuda(x, w_local.data)
    x2 = _as_2d(x, w_local.k)
    m = x2.shape[0]
    if m != gather.m or w_local.n * gather.world != gather.n_total:
        raise ValueError("activations / weight slice do not match the gather buffers")
    ws = workspace_for(w_local, m)
    with torch.cuda.device(dev):
        lib = _lib.lib()
        st = lib.ggufmm_gemm_allgather(w_local.data.data_ptr(), w_local.qtype, w_local.n, w_local.k, x2.data_ptr(),
                                       _code(x2.dtype), m, x2.stride(0), gather.y_ptrs, gather.world,
                                       gather.rank * w_local.n, _code(gather.dtype), gather.n_total, ws.data_ptr(),
                                       ws.numel(), _stream(dev))
        _lib.check(st, "ggufmm_gemm_allgather")
        st = lib.ggufmm_peer_barrier(gather.ptrs, gather.world, gather.rank, _stream(dev))
    _lib.check(st, "ggufmm_peer_barrier")
    return gather.y


def gemv_allreduce(x: torch.Tensor, w: GGUFQuantTensor, exchange: PeerExchange, out: torch.Tensor | None = None,
                   out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Decode GEMV summed over the exchange's GPUs in the same kernel (NVLink peer
    memory): every GPU of the group calls it with its own W slice and receives
    the full sum. Replaces GEMV + NCCL all-reduce for the TP down projection."""
    dev = _require_cuda(x, w.data)
    x2 = _as_2d(x, w.k)
    if x2.shape[0] > exchange.m_max or w.n != exchange.n:
        raise ValueError("activations or output width do not match the exchange buffers")
    y = _out(x2, w.n, out, out_dtype)
    exchange.epoch += 1
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_gemv_allreduce(w.data.data_ptr(), w.qtype, w.n, w.k, x2.data_ptr(), _code(x2.dtype),
                                              x2.shape[0], x2.stride(0), y.data_ptr(), _code(y.dtype), y.stride(0),
                                              exchange.ptrs, exchange.world, exchange.rank, exchange.m_max,
                                              exchange.epoch, _stream(dev))
    if st != 0:
        exchange.epoch -= 1  # nothing was launched
    _lib.check(st, "ggufmm_gemv_allreduce")
    return y


_workspaces: dict[int, torch.Tensor] = {}


def workspace_for(w: GGUFQuantTensor, m: int) -> torch.Tensor:
    """A cached per-device scratch buffer large enough for ggufmm_gemm (and for
    ggufmm_gemm_grouped when w is the group's weight with the largest N)."""
    need = int(_lib.lib().ggufmm_gemm_workspace_size(w.qtype, m, w.n, w.k))
    idx = w.data.device.index
    ws = _workspaces.get(idx)
    if ws is None or ws.numel() < need:
        ws = torch.empty(max(need, 256), dtype=torch.uint8, device=w.data.device)
        _workspaces[idx] = ws
    return ws


def gemm(x: torch.Tensor, w: GGUFQuantTensor, out: torch.Tensor | None = None,
         out_dtype: torch.dtype | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Tensor-core (tcgen05) GEMM, any M: out[m, n] = sum_k x[m, k] W[n, k]."""
    dev = _require_cuda(x, w.data)
    x2 = _as_2d(x, w.k)
    y = _out(x2, w.n, out, out_dtype)
    ws = workspace if workspace is not None else workspace_for(w, x2.shape[0])
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_gemm(w.data.data_ptr(), w.qtype, w.n, w.k, x2.data_ptr(), _code(x2.dtype),
                                    x2.shape[0], x2.stride(0), y.data_ptr(), _code(y.dtype), y.stride(0),
                                    ws.data_ptr(), ws.numel(), _stream(dev))
    _lib.check(st, "ggufmm_gemm")
    return y


def gemm_grouped(x: torch.Tensor, ws: list[GGUFQuantTensor], outs: list[torch.Tensor] | None = None,
                 out_dtype: torch.dtype | None = None) -> list[torch.Tensor]:
    """GEMM of up to 4 weights sharing the activations (q/k/v or gate/up) at any M;
    Q4_K at M <= 1024 is one fused-dequant launch over all of them."""
    if not 1 <= len(ws) <= 4:
        raise ValueError("gemm_grouped takes 1 to 4 weights")
    k, qt = ws[0].k, ws[0].qtype
    if any(w.k != k or w.qtype != qt for w in ws):
        raise ValueError("grouped weights must share K and the quantization type")
    dev = _require_cuda(x, *[w.data for w in ws])
    x2 = _as_2d(x, k)
    if outs is None:
        outs = [None] * len(ws)
    ys = [_out(x2, w.n, o, out_dtype) for w, o in zip(ws, outs)]
    if len({y.dtype for y in ys}) != 1:
        raise ValueError("grouped outputs must share a dtype")
    import ctypes
    nseg = len(ws)
    wsp = workspace_for(max(ws, key=lambda w: w.n), x2.shape[0])
    qs = (ctypes.c_void_p * nseg)(*[w.data.data_ptr() for w in ws])
    ns = (ctypes.c_int64 * nseg)(*[w.n for w in ws])
    yp = (ctypes.c_void_p * nseg)(*[y.data_ptr() for y in ys])
    ld = (ctypes.c_int64 * nseg)(*[y.stride(0) for y in ys])
    with torch.cuda.device(dev):
        st = _lib.lib().ggufmm_gemm_grouped(nseg, qs, ns, qt, k, x2.data_ptr(), _code(x2.dtype), x2.shape[0],
                                            x2.stride(0), yp, _code(ys[0].dtype), ld, wsp.data_ptr(), wsp.numel(),
                                            _stream(dev))
    _lib.check(st, "ggufmm_gemm_grouped")
    return ys


def mul_mat(x: torch.Tensor, w: GGUFQuantTensor, out: torch.Tensor | None = None,
            out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y = x @ W^T: GEMV for M <= 8 where gemv_preferred holds, tensor-core GEMM otherwise.

    Same contract as vLLM's ``fused_mul_mat_gguf(x, qweight, qweight_type)``
    (vllm/model_executor/layers/quantization/gguf.py:198-230); the leading
    dimensions of ``x`` are preserved.
    """
    lead = x.shape[:-1]
    x2 = _as_2d(x, w.k)
    m = x2.shape[0]
    if x2.is_cuda and gemv_preferred(m, w, x2.dtype):
        try:
            y = gemv(x2, w, out=out, out_dtype=out_dtype)
        except ValueError as exc:
            if not _lib.is_align_refusal(exc):
                raise
            # unaligned operands: the GEMM path has no 16-byte alignment requirement
            y = gemm(x2, w, out=out, out_dtype=out_dtype)
    else:
        y = gemm(x2, w, out=out, out_dtype=out_dtype)
    return y.reshape(*lead, w.n)


# ---------------------------------------------------------------------------------------------
# what lies between a layer's projections: norm, rotary positions, key-value cache, attention
# (the reference's shaders of vllm_webgpu/models/llama.py:239-367)
# ---------------------------------------------------------------------------------------------
# These calls are short next to their launch, so their wrappers keep to few tensor attributes,
# look each up once and pass the arguments as one packed struct.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice  # the callers' tensors are on a GPU: CUDA is up
_native: dict = {}


def _on_device(index: int, name: str, *args) -> int:
    """The library's ``name``(*args) with CUDA device ``index`` current."""
    fn = _native.get(name)
    if fn is None:
        fn = _native[name] = getattr(_lib.lib(), name)
    if _current_device() == index:
        return fn(*args)
    with torch.cuda.device(index):
        return fn(*args)


def _call(index: int, name: str, *args) -> None:
    """The library's ``name``(*args, stream) with CUDA device ``index`` current, its status checked."""
    st = _on_device(index, name, *args, _raw_stream(index))
    if st:
        _lib.check(st, name)


def _norm_rows(t: torch.Tensor, shape, index: int, n: int, m: int, what: str | None) -> tuple[torch.Tensor, int]:
    """t as rows of n values, and the stride of a row: an input (what None: copied where its
    layout allows no rows) or an output."""
    if t.shape != shape or t.get_device() != index:
        raise ValueError(f"{what or 'residual'} must be a {tuple(shape)} tensor on cuda:{index}")
    if t.is_contiguous():
        return t, n
    if t.dim() == 2 and t.stride(1) == 1 and (m <= 1 or t.stride(0) >= n):
        return t, t.stride(0) if m > 1 else n
    if what is not None:
        raise ValueError(f"{what} must be contiguous, or two-dimensional with contiguous rows")
    return t.contiguous(), n


_NORM_ARGS = struct.Struct("5Q10q2d")


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-5,
             residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
             out_dtype: torch.dtype | None = None, residual_out: torch.Tensor | None = None,
             weight_add: float = 0.0):
    """Root-mean-square norm over the last dimension, s * (mean(s^2) + eps)^-1/2 *
    (weight + weight_add) of s = x, or s = x + residual: then (out, residual_out) is
    returned, residual_out holding s in the residual's dtype. The sum and the norm are
    computed in 32 bits and rounded once each; x, residual, weight and out may have
    different dtypes. ``residual_out`` may be ``residual`` and ``out`` may be ``x`` (in
    place). Replaces the reference's add and rms_norm dispatches
    (vllm_webgpu/models/llama.py:239-367)."""
    shape, index = x.shape, x.get_device()
    if index < 0:
        _require_cuda(x)
    count = x.numel()
    n = shape[-1] if shape else 0
    if n == 0:
        raise ValueError("rms_norm needs at least one value in a row")
    m = count // n
    x2, ldx = (x, n) if x.is_contiguous() else _norm_rows(x, shape, index, n, m, None)
    r_ptr = r_code = ldr = ro_ptr = ldro = w_ptr = w_code = 0
    like = x2
    try:
        if residual is not None:
            r2, ldr = _norm_rows(residual, shape, index, n, m, None)
            r_dtype = r2.dtype
            r_ptr, r_code = r2.data_ptr(), _DTYPE_CODE[r_dtype]
            if residual_out is None:
                residual_out, ldro = torch.empty_like(r2, memory_format=torch.contiguous_format), n
                like = residual_out
            else:
                if residual_out.dtype is not r_dtype:
                    raise ValueError("residual_out must have the residual's dtype")
                _, ldro = _norm_rows(residual_out, shape, index, n, m, "residual_out")
            ro_ptr = residual_out.data_ptr()
        elif residual_out is not None:
            raise ValueError("residual_out needs a residual")
        if out is None:
            dtype = out_dtype or x2.dtype
            if like.is_contiguous():
                out = torch.empty_like(like) if like.dtype is dtype else torch.empty_like(like, dtype=dtype)
            else:
                out = torch.empty(shape, dtype=dtype, device=like.device)
            ldy = n
        else:
            _, ldy = _norm_rows(out, shape, index, n, m, "out")
            dtype = out.dtype
        if weight is not None:
            if weight.numel() != n or weight.dim() != 1 or weight.get_device() != index or not weight.is_contiguous():
                raise ValueError(f"weight must be a contiguous [{n}] tensor on {x.device}")
            w_ptr, w_code = weight.data_ptr(), _DTYPE_CODE[weight.dtype]
        args = _NORM_ARGS.pack(x2.data_ptr(), r_ptr, ro_ptr, w_ptr, out.data_ptr(), ldx, ldr, ldro, ldy, m, n,
                               _DTYPE_CODE[x2.dtype], r_code, w_code, _DTYPE_CODE[dtype], weight_add, eps)
    except KeyError as e:
        raise ValueError(f"unsupported dtype {e.args[0]}; expected float32, float16 or bfloat16") from None
    _call(index, "ggufmm_rms_norm", args)
    return out if residual is None else (out, residual_out)


def rope_steps(rot_dim: int, theta: float = 10000.0, scaling: dict | None = None,
               freq_factors=None, device=None) -> tuple[torch.Tensor, float]:
    """The rotary frequencies as ``rope`` and ``rope_append`` take them, computed in 64
    bits: (steps, factor), steps int64 [rot_dim / 2] the turn per position of each pair in
    units of 2^-64 turns, factor the multiplier of the turned values.

    ``scaling`` stretches them to long contexts, by its ``rope_type`` (the keys of Hugging
    Face's ``rope_scaling``): "linear" (factor), "llama3" (factor, low_freq_factor,
    high_freq_factor, original_max_position_embeddings) or "yarn" (factor,
    original_max_position_embeddings, beta_fast, beta_slow, attention_factor).
    ``freq_factors`` [rot_dim / 2] divides each frequency (GGUF's ``rope_freqs.weight``)."""
    import math

    import numpy as np
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim must be a positive even number, not {rot_dim}")
    if not theta > 0:
        raise ValueError(f"theta must be positive, not {theta}")
    half = rot_dim // 2
    f = np.float64(theta) ** (-np.arange(half, dtype=np.float64) * 2 / rot_dim)  # radians per position
    factor = 1.0
    kind = (scaling or {}).get("rope_type", (scaling or {}).get("type", "default"))
    if kind == "linear":
        f = f / float(scaling["factor"])
    elif kind == "llama3":
        turns = float(scaling["original_max_position_embeddings"]) * f / (2 * math.pi)
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not high > low:
            raise ValueError("llama3 scaling needs high_freq_factor > low_freq_factor")
        keep = np.clip((turns - low) / (high - low), 0.0, 1.0)
        f = keep * f + (1.0 - keep) * f / float(scaling["factor"])
    elif kind == "yarn":
        for name, plain in (("mscale", None), ("mscale_all_dim", None), ("truncate", True)):
            if scaling.get(name, plain) not in (None, plain):
                raise ValueError(f"yarn scaling with {name} = {scaling[name]} is not supported")
        old, by = float(scaling["original_max_position_embeddings"]), float(scaling["factor"])

        def pair_with(turns):  # the pair that makes so many turns over the original context
            return rot_dim * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low = max(math.floor(pair_with(float(scaling.get("beta_fast", 32.0)))), 0)
        high = min(math.ceil(pair_with(float(scaling.get("beta_slow", 1.0)))), rot_dim - 1)
        ramp = np.clip((np.arange(half) - low) / max(high - low, 0.001), 0.0, 1.0)
        f = f * (1.0 - ramp) + f / by * ramp
        given = scaling.get("attention_factor")
        factor = float(given) if given is not None else (0.1 * math.log(by) + 1.0 if by > 1 else 1.0)
    elif kind != "default":
        raise ValueError(f"rope scaling {kind!r} is not supported (supported: default, linear, llama3, yarn)")
    if freq_factors is not None:
        ff = np.asarray(torch.as_tensor(freq_factors).cpu(), dtype=np.float64)
        if ff.shape != (half,):
            raise ValueError(f"freq_factors must hold {half} values")
        if not (np.isfinite(ff) & (ff != 0)).all():
            raise ValueError("freq_factors must be finite and not zero")
        f = f / ff
    turns = np.remainder(f / (2 * math.pi), 1.0)  # whole turns change nothing at whole positions
    steps = np.array([int(round(float(t) * 2.0 ** 64)) % 2 ** 64 for t in turns], dtype=np.uint64).view(np.int64)
    return torch.from_numpy(steps.copy()).to(device if device is not None else "cuda"), factor


def _heads(t: torch.Tensor, what: str, index: int) -> tuple[torch.Tensor, tuple, tuple]:
    """t as [tokens, heads, head_dim] with a unit stride in the last dimension, on device
    ``index``; its shape and strides."""
    shape = t.shape
    if len(shape) != 3 or t.get_device() != index:
        raise ValueError(f"{what} must be a [tokens, heads, head_dim] tensor on cuda:{index}")
    st = t.stride()
    if st[2] != 1:
        t = t.contiguous()
        st = t.stride()
    return t, shape, st


def _index(t: torch.Tensor, dtype: torch.dtype, length: int, what: str, index: int) -> torch.Tensor:
    if t.numel() != length or t.dim() != 1 or t.get_device() != index:
        raise ValueError(f"{what} must be a [{length}] tensor on cuda:{index}")
    return t if t.dtype is dtype and t.is_contiguous() else t.to(dtype).contiguous()


def _cache_strides(k_cache: torch.Tensor, v_cache: torch.Tensor, index: int) -> tuple:
    """(shape, dtype, strides of k, of v) of caches [pages, kv heads, page size, head_dim]."""
    shape, dtype = k_cache.shape, k_cache.dtype
    if len(shape) != 4 or shape != v_cache.shape or dtype is not v_cache.dtype:
        raise ValueError("k_cache and v_cache must be [pages, kv heads, page size, head_dim] tensors of one shape and dtype")
    if k_cache.get_device() != index or v_cache.get_device() != index:
        raise ValueError(f"the cache must lie on cuda:{index}")
    ks, vs = k_cache.stride(), v_cache.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("the caches' last dimension must have unit stride")
    if 1 in shape:  # the stride of a dimension of one says nothing: any valid one does
        d = shape[3]
        ks, vs = ([d if shape[i] == 1 else st[i] for i in range(3)] for st in (ks, vs))
    return shape, dtype, ks, vs


_ROPE_ARGS = struct.Struct("Q2qQ2qQ2qQ2qQ3qQ3q3Q11qd")


def _rope(q, k, v, positions, steps, slots, k_cache, v_cache, interleaved, factor, q_out):
    index = q.get_device()
    if index < 0:
        _require_cuda(q)
    q, shape, qs = _heads(q, "q", index)
    t, hq, d = shape
    dtype = q.dtype
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif q_out.shape != shape or q_out.get_device() != index or q_out.stride(2) != 1:
        raise ValueError(f"q_out must be a {tuple(shape)} tensor with unit stride in its last dimension")
    positions = _index(positions, torch.int64, t, "positions", index)
    if steps.get_device() != index or steps.dtype is not torch.int64 or steps.dim() != 1 or not steps.is_contiguous():
        raise ValueError(f"steps must be the int64 tensor of rope_steps on cuda:{index}")
    os = q_out.stride()
    try:
        if k is None:
            kv = (0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
            hkv, cache_code, page, pages, slot_ptr = 0, 0, 0, 0, 0
        else:
            (k, k_shape, s), (v, v_shape, u) = _heads(k, "k", index), _heads(v, "v", index)
            hkv = k_shape[1]
            if k_shape[0] != t or k_shape[2] != d or v_shape != k_shape or k.dtype is not dtype or v.dtype is not dtype:
                raise ValueError(f"k and v must be [{t}, kv heads, {d}] tensors of q's dtype")
            (pages, heads, page, dk), cache_dtype, ks, vs = _cache_strides(k_cache, v_cache, index)
            if heads != hkv or dk != d:
                raise ValueError(f"the cache holds {heads} heads of {dk}, k has {hkv} of {d}")
            slots = _index(slots, torch.int64, t, "slots", index)
            slot_ptr, cache_code = slots.data_ptr(), _DTYPE_CODE[cache_dtype]
            kv = (k.data_ptr(), s[0], s[1], v.data_ptr(), u[0], u[1], k_cache.data_ptr(), ks[0], ks[1], ks[2],
                  v_cache.data_ptr(), vs[0], vs[1], vs[2])
        args = _ROPE_ARGS.pack(q.data_ptr(), qs[0], qs[1], q_out.data_ptr(), os[0], os[1], *kv, positions.data_ptr(),
                               slot_ptr, steps.data_ptr(), t, hq, hkv, d, 2 * steps.numel(), 1 if interleaved else 0,
                               _DTYPE_CODE[dtype], _DTYPE_CODE[q_out.dtype], cache_code, page, pages, factor)
    except KeyError as e:
        raise ValueError(f"unsupported dtype {e.args[0]}; expected float32, float16 or bfloat16") from None
    _call(index, "ggufmm_rope_append", args)
    return q_out


def rope(x: torch.Tensor, positions: torch.Tensor, steps: torch.Tensor, interleaved: bool = False,
         factor: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions on x [tokens, heads, head_dim]: the first 2 * len(steps) values of
    each head turn in pairs (i, i + half) or, ``interleaved`` (as GGUF files of the Llama
    family order them), (2i, 2i + 1), by positions[t] times the step of ``rope_steps``;
    the rest passes. ``out`` may be x. Replaces the reference's rope dispatch
    (vllm_webgpu/models/llama.py:239-367)."""
    return _rope(x, None, None, positions, steps, None, None, None, interleaved, factor, out)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, steps: torch.Tensor,
                slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, interleaved: bool = False,
                factor: float = 1.0, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """``rope`` on q and on k, with k and v appended to the paged cache, in one launch:
    returns the turned q [tokens, q heads, head_dim] (in q's dtype, or into ``q_out``,
    which may be q) and writes the turned k and v to slot slots[t] (offset s % page size of
    page s // page size) of ``k_cache`` / ``v_cache`` [pages, kv heads, page size,
    head_dim], f16 or bf16. A negative slot stores nothing; one past the last page too, and
    sets bit 2 of the device status word. Replaces the reference's rope and kv_cache_store
    dispatches (vllm_webgpu/models/llama.py:239-367)."""
    if k is None or v is None or slots is None or k_cache is None or v_cache is None:
        raise ValueError("rope_append needs k, v, slots and the caches (rope turns q alone)")
    return _rope(q, k, v, positions, steps, slots, k_cache, v_cache, interleaved, factor, q_out)


_ATTENTION_ARGS = struct.Struct("Q2qQ2qQ3qQ3qQ2q2Q10qd")
_attention_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def attention_workspace(batch: int, q_heads: int, kv_heads: int, head_dim: int, device) -> torch.Tensor:
    """A zero-filled workspace for ``paged_attention`` calls of up to this size, which a
    program that captures CUDA graphs keeps for them (calls that may run at the same time
    need one each)."""
    need = int(_lib.lib().ggufmm_paged_attention_workspace_size(batch, q_heads, kv_heads, head_dim))
    return torch.zeros(max(need, 256), dtype=torch.uint8, device=device)


_attention_workspace_bytes: dict[tuple, int] = {}


def _attention_workspace(batch: int, hq: int, hkv: int, d: int, index: int) -> torch.Tensor:
    """The workspace of the current stream: one per stream, since calls on different streams
    may overlap; inside a graph capture one of the capture's own, zeroed in the graph."""
    if torch.cuda.is_current_stream_capturing():
        return attention_workspace(batch, hq, hkv, d, torch.device("cuda", index))
    size = (batch, hq, hkv, d)
    need = _attention_workspace_bytes.get(size)
    if need is None:
        need = _attention_workspace_bytes[size] = int(_lib.lib().ggufmm_paged_attention_workspace_size(*size))
    key = (index, _raw_stream(index))
    ws = _attention_workspaces.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.zeros(max(need, 256), dtype=torch.uint8, device=torch.device("cuda", index))
        _attention_workspaces[key] = ws
    return ws


def _attention_args(q, k_cache, v_cache, tables, lens, scale, window, out, q_starts, max_q):
    """(device index, packed arguments, out, sizes, the tensors the arguments point to)."""
    index = q.get_device()
    if index < 0:
        _require_cuda(q)
    q, shape, qs = _heads(q, "q", index)
    t, hq, d = shape
    if (t > 1 and qs[0] < d) or (hq > 1 and qs[1] < d):  # rows that lie over one another
        q = q.contiguous()
        qs = q.stride()
    (pages, hkv, page, dk), cache_dtype, ks, vs = _cache_strides(k_cache, v_cache, index)
    dtype = q.dtype
    if dk != d or cache_dtype is not dtype:
        raise ValueError(f"q and the cache must share head_dim and dtype: {d} {dtype}, {dk} {cache_dtype}")
    if hkv == 0 or hq % hkv:
        raise ValueError(f"{hq} query heads are no multiple of {hkv} kv heads")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        os = (hq * d, d)
    else:
        if out.shape != shape or out.dtype is not dtype or out.get_device() != index or out.stride(2) != 1:
            raise ValueError(f"out must be a {tuple(shape)} {dtype} tensor with unit stride in its last dimension")
        os = out.stride()
    if tables.dim() != 2 or tables.get_device() != index:
        raise ValueError(f"block_tables must be a [batch, pages] tensor on cuda:{index}")
    b, width = tables.shape
    if tables.dtype is not torch.int32 or (width > 1 and tables.stride(1) != 1) or (b > 1 and tables.stride(0) < width):
        tables = tables.to(torch.int32).contiguous()
    lens = _index(lens, torch.int32, b, "lens", index)
    starts = 0
    if q_starts is not None:
        q_starts = _index(q_starts, torch.int32, b + 1, "q_starts", index)
        starts = q_starts.data_ptr()
    elif t != b:
        raise ValueError(f"q holds {t} tokens for {b} sequences")
    if t == 1 or hq == 1:  # the stride of a dimension of one says nothing: any valid one does
        qs, os = ((st[0] if t > 1 else hq * d, st[1] if hq > 1 else d) for st in (qs, os))
    code = _DTYPE_CODE.get(dtype, -1)  # the library refuses what the cache cannot hold
    args = _ATTENTION_ARGS.pack(
        q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1], k_cache.data_ptr(), ks[0], ks[1], ks[2],
        v_cache.data_ptr(), vs[0], vs[1], vs[2], tables.data_ptr(), tables.stride(0) if b > 1 else width, width,
        lens.data_ptr(), starts, b, t, max_q, hq, hkv, d, page, pages, code, window, d ** -0.5 if scale is None else scale)
    return index, args, out, (b, hq, hkv, d), (q, tables, lens, q_starts)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                    lens: torch.Tensor, scale: float | None = None, window: int = 0, out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over a paged cache: q and out [batch, q heads,
    head_dim] in the cache's dtype (f16 / bf16), caches [pages, kv heads, page size,
    head_dim], block_tables int32 [batch, pages of the longest], lens int32 [batch] (the new
    token included). ``scale`` defaults to head_dim^-1/2; ``window`` > 0 lets a token see
    the last ``window`` positions only. A sequence of length 0 gives zeros. ``workspace``
    (``attention_workspace``) defaults to one kept per stream. Replaces the reference's
    score, softmax and output dispatches (vllm_webgpu/models/llama.py:239-367)."""
    index, args, out, sizes, keep = _attention_args(q, k_cache, v_cache, block_tables, lens, scale, window, out, None, 0)
    if workspace is None:
        workspace = _attention_workspace(*sizes, index)
    elif workspace.get_device() != index or workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous uint8 tensor on cuda:{index} (attention_workspace makes it)")
    _call(index, "ggufmm_paged_attention", args, workspace.data_ptr(), workspace.numel())
    return out


def paged_prompt_attention(q: torch.Tensor, q_starts: torch.Tensor, max_q: int, k_cache: torch.Tensor,
                           v_cache: torch.Tensor, block_tables: torch.Tensor, lens: torch.Tensor,
                           scale: float | None = None, window: int = 0,
                           out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of several new tokens per sequence over a paged cache that holds them
    already: q and out [tokens, q heads, head_dim], sequence b's new tokens in rows
    q_starts[b] to q_starts[b + 1] (int32 [batch + 1]), at the last positions of its
    lens[b]; ``max_q`` is at least the longest run. Otherwise as ``paged_attention``. The
    reference feeds a prompt token by token (run_inference.py:323-350)."""
    index, args, out, _, keep = _attention_args(q, k_cache, v_cache, block_tables, lens, scale, window, out, q_starts,
                                                max_q)
    # few new tokens may share the keys of a long cache out: scratch for this call alone
    need = _on_device(index, "ggufmm_paged_prompt_attention_workspace_size", args)
    ws = torch.empty(need, dtype=torch.uint8, device=out.device) if need else None
    _call(index, "ggufmm_paged_prompt_attention", args, None if ws is None else ws.data_ptr(),
          0 if ws is None else ws.numel())
    return out
