"""Torch-facing wrappers of the hq4 kernels.

PyTorch provides device memory and the current CUDA stream; the arithmetic is
all in ``libhq4.so``.  Every op checks that its tensors are CUDA, contiguous and
of the dtype the C ABI expects, and raises instead of computing anything on the
CPU.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib


def _stream_ptr(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _need_cuda(t: torch.Tensor, name: str, dtype=None) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (no CPU fallback)")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")


def q4_gemv(w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, x: torch.Tensor,
            group_size: int = 64, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[m, n_out] = x[m, n_in] @ dequant(w).T`` on the GPU (hq4_gemv).

    w: uint32/int32 [n_out, n_in/8]; scales, biases: fp16 [n_out, n_in/gs];
    x: fp32 [..., n_in]."""
    lib = _lib.load()
    _need_cuda(w, "w")
    if w.dtype not in (torch.int32, torch.uint32):
        raise RuntimeError("w must hold packed uint32 words")
    _need_cuda(scales, "scales", torch.float16)
    _need_cuda(biases, "biases", torch.float16)
    n_out, n_in = w.shape[0], w.shape[1] * 8
    xf = x.reshape(-1, n_in)
    _need_cuda(xf, "x", torch.float32)
    m = xf.shape[0]
    if out is None:
        out = torch.empty((m, n_out), dtype=torch.float32, device=x.device)
    _need_cuda(out, "out", torch.float32)
    rc = lib.hq4_gemv(w.data_ptr(), scales.data_ptr(), biases.data_ptr(), xf.data_ptr(),
                      out.data_ptr(), n_out, n_in, group_size, m, _stream_ptr(x.device))
    _lib.check(rc, "hq4_gemv")
    return out.reshape(*x.shape[:-1], n_out)


def q4_gemv_fused(w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, x: torch.Tensor,
                  group_size: int = 64, row_add: Optional[torch.Tensor] = None,
                  residual: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """GEMV with the bias / residual add fused into its store (hq4_gemv_fused).

    ``out`` may alias ``residual`` (in-place residual update) but not ``x``."""
    lib = _lib.load()
    _need_cuda(w, "w")
    _need_cuda(scales, "scales", torch.float16)
    _need_cuda(biases, "biases", torch.float16)
    n_out, n_in = w.shape[0], w.shape[1] * 8
    xf = x.reshape(-1, n_in)
    _need_cuda(xf, "x", torch.float32)
    m = xf.shape[0]
    if out is None:
        out = torch.empty((m, n_out), dtype=torch.float32, device=x.device)
    _need_cuda(out, "out", torch.float32)
    ra = 0
    if row_add is not None:
        _need_cuda(row_add, "row_add", torch.float32)
        ra = row_add.data_ptr()
    rs = 0
    if residual is not None:
        _need_cuda(residual, "residual", torch.float32)
        rs = residual.data_ptr()
    rc = lib.hq4_gemv_fused(w.data_ptr(), scales.data_ptr(), biases.data_ptr(), xf.data_ptr(),
                            out.data_ptr(), n_out, n_in, group_size, m, ra or None, rs or None,
                            _stream_ptr(x.device))
    _lib.check(rc, "hq4_gemv_fused")
    return out.reshape(*x.shape[:-1], n_out)


def q4_dequant(w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, row0: int, row1: int,
               group_size: int = 64, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fp32 expansion of rows [row0, row1) (hq4_dequant)."""
    lib = _lib.load()
    _need_cuda(w, "w")
    _need_cuda(scales, "scales", torch.float16)
    _need_cuda(biases, "biases", torch.float16)
    n_in = w.shape[1] * 8
    rows = max(row1 - row0, 0)
    if out is None:
        out = torch.empty((rows, n_in), dtype=torch.float32, device=w.device)
    _need_cuda(out, "out", torch.float32)
    rc = lib.hq4_dequant(w.data_ptr(), scales.data_ptr(), biases.data_ptr(), out.data_ptr(),
                         row0, row1, n_in, group_size, _stream_ptr(w.device))
    _lib.check(rc, "hq4_dequant")
    return out


_WORKSPACES = {}


def gemm_workspace(n_out: int, n_in: int, m: int, device: torch.device) -> torch.Tensor:
    """A grow-only per-device workspace large enough for hq4_gemm_w4a16 on
    this shape.  Callers that capture CUDA graphs should take it before
    capturing and pass it explicitly."""
    lib = _lib.load()
    need = int(lib.hq4_gemm_workspace_bytes(n_out, n_in, m))
    if need < 0:
        raise RuntimeError(f"hq4_gemm_workspace_bytes({n_out}, {n_in}, {m}) = {need}")
    key = torch.device(device).index if torch.device(device).index is not None else torch.cuda.current_device()
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.empty(max(need, 1 << 20), dtype=torch.uint8, device=torch.device("cuda", key))
        _WORKSPACES[key] = ws
    return ws


def q4_gemm(w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, x: torch.Tensor,
            group_size: int = 64, row_add: Optional[torch.Tensor] = None,
            residual: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None,
            workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """W4A16 GEMM on the tcgen05 tensor cores (hq4_gemm_w4a16):
    ``out[m, n_out] = x[m, n_in] @ dequant(w).T`` with x bf16 or fp32 and an
    fp32 result, for token counts where the product is a dense contraction."""
    lib = _lib.load()
    _need_cuda(w, "w")
    if w.dtype not in (torch.int32, torch.uint32):
        raise RuntimeError("w must hold packed uint32 words")
    _need_cuda(scales, "scales", torch.float16)
    _need_cuda(biases, "biases", torch.float16)
    n_out, n_in = w.shape[0], w.shape[1] * 8
    xf = x.reshape(-1, n_in)
    _need_cuda(xf, "x")
    if xf.dtype not in (torch.bfloat16, torch.float32):
        raise RuntimeError(f"x must be bfloat16 or float32, got {xf.dtype}")
    m = xf.shape[0]
    if out is None:
        out = torch.empty((m, n_out), dtype=torch.float32, device=x.device)
    _need_cuda(out, "out", torch.float32)
    ra = 0
    if row_add is not None:
        _need_cuda(row_add, "row_add", torch.float32)
        ra = row_add.data_ptr()
    rs = 0
    if residual is not None:
        _need_cuda(residual, "residual", torch.float32)
        rs = residual.data_ptr()
    if workspace is None:
        workspace = gemm_workspace(n_out, n_in, m, x.device)
    _need_cuda(workspace, "workspace", torch.uint8)
    rc = lib.hq4_gemm_w4a16(w.data_ptr(), scales.data_ptr(), biases.data_ptr(), xf.data_ptr(),
                            1 if xf.dtype == torch.float32 else 0, out.data_ptr(), n_out, n_in,
                            group_size, m, ra or None, rs or None, workspace.data_ptr(), workspace.numel(),
                            _stream_ptr(x.device))
    _lib.check(rc, "hq4_gemm_w4a16")
    return out.reshape(*x.shape[:-1], n_out)


def gemm_plan(n_out: int, n_in: int, m: int, x_is_f32: bool = False) -> dict:
    """The launch plan hq4_gemm_w4a16 uses for a shape (host only)."""
    import ctypes
    lib = _lib.load()
    info = (ctypes.c_int * 8)()
    _lib.check(lib.hq4_gemm_plan(n_out, n_in, m, 1 if x_is_f32 else 0, info), "hq4_gemm_plan")
    keys = ("row_tiles", "ksplit", "token_tiles", "tile_tokens", "stages", "smem", "weight_slots", "kernel")
    d = dict(zip(keys, list(info)))
    d["kernel"] = {0: "tcgen05", 1: "mma.sync", 2: "gemv", 3: "gemv_mt"}[d["kernel"]]
    return d


def act_encode_i8(x: torch.Tensor, payload: Optional[torch.Tensor] = None, wire: bool = False) -> torch.Tensor:
    """int8 wire payload of fp32 activations [..., cols] (hetero/transport.py:198-211):
    the rows' fp32 scales then the int8 rows, as a uint8 tensor.  wire=True
    rounds every value to fp16 first, as the reference's engine encodes the
    fp16 array its backend's to_wire made (hetero/engine.py:97)."""
    xs = x.contiguous()
    cols = int(xs.shape[-1])
    rows = xs.numel() // cols
    if payload is None:
        payload = torch.empty(rows * (4 + cols), dtype=torch.uint8, device=xs.device)
    lib = _lib.load()
    fn, name = (lib.hq4_act_encode_i8_wire, "hq4_act_encode_i8_wire") if wire else \
        (lib.hq4_act_encode_i8, "hq4_act_encode_i8")
    _lib.check(fn(xs.data_ptr(), rows, cols, payload.data_ptr(), torch.cuda.current_stream(xs.device).cuda_stream),
               name)
    return payload


def act_decode_i8(payload: torch.Tensor, rows: int, cols: int, dtype=torch.float16,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Activations [rows, cols] from an int8 wire payload (hetero/transport.py:214-225):
    fp16(q * scale), or that value widened to fp32 when dtype is float32."""
    if out is None:
        out = torch.empty((rows, cols), dtype=dtype, device=payload.device)
    lib = _lib.load()
    f16 = out.data_ptr() if out.dtype == torch.float16 else None
    f32 = out.data_ptr() if out.dtype == torch.float32 else None
    _lib.check(lib.hq4_act_decode_i8(payload.data_ptr(), rows, cols, f16, f32,
                                     torch.cuda.current_stream(payload.device).cuda_stream), "hq4_act_decode_i8")
    return out


# ---------------------------------------------------------------------------
# Many streams over a paged cache
# ---------------------------------------------------------------------------
#
# A batch is n_seqs sequences over caches [n_pages, n_kv, page_size, head_dim]
# (bf16 or fp16).  Sequence s owns rows cu_rows[s] to cu_rows[s + 1] of q, k and
# v, its cache holds lens[s] entries before them, and entry e lies at place
# e % page_size of page pages[s, e // page_size].  cu_rows, lens and pages are
# int32 CUDA tensors that the kernels read when they run, so a captured step can
# be replayed while the sequences grow.  A step appends first, then attends.

# The calls are checked and made in native code (csrc/hq4_torch.cpp): in Python
# that takes longer than the kernels of a small step.


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 pages: torch.Tensor, cu_rows: torch.Tensor, lens: torch.Tensor, rope_cos: torch.Tensor,
                 rope_sin: torch.Tensor, positions: Optional[torch.Tensor] = None,
                 q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Append a step's rotated keys and its values to their pages; returns the
    rotated queries [rows, n_heads, head_dim] (hq4_paged_append).

    q: [rows, n_heads, head_dim], k, v: [rows, n_kv, head_dim], float32 or the
    caches' type, views of one projection if need be; rope_cos, rope_sin:
    float32 [max_pos, head_dim / 2].  A row's position is its entry's number or
    positions[row] (int32); q_norm, k_norm: float32 [head_dim], an RMS norm of
    each head before the rotation.  out must not overlap q, k, v or the caches,
    nor the caches q, k or v."""
    return _lib.torch_calls().paged_append(q, k, v, k_cache, v_cache, pages, cu_rows, lens, rope_cos, rope_sin,
                                           positions, q_norm, k_norm, eps, out)


def paged_attention_workspace(q: torch.Tensor, k_cache: torch.Tensor, pages: torch.Tensor) -> torch.Tensor:
    """A workspace for paged_attention / tree_attention calls of these shapes
    (one to a stream; the calls take a fresh one where none is given)."""
    return _lib.torch_calls().workspace(q, k_cache, pages)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pages: torch.Tensor,
                    cu_rows: torch.Tensor, lens: torch.Tensor, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal grouped-query attention of a ragged batch over the paged cache
    (hq4_paged_attention): row i of sequence s sees entries 0 .. lens[s] + i.
    q: [rows, n_heads, head_dim] as paged_append returns it; scale defaults to
    head_dim ** -0.5, out must not overlap q or the caches.  Decode, prompt chunks and
    mixtures of them alike."""
    return _lib.torch_calls().attend(q, k_cache, v_cache, pages, cu_rows, lens, None, scale, out, workspace)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pages: torch.Tensor,
                   cu_rows: torch.Tensor, lens: torch.Tensor, tree_mask: torch.Tensor, scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """paged_attention for trees of drafted tokens (hq4_tree_attention): row i
    of sequence s sees the entries before lens[s], and entry lens[s] + j where
    bit j % 32 of tree_mask[row, j // 32] is set (int32 words)."""
    if tree_mask is None:
        raise RuntimeError("tree_mask must be int32 [rows, words]")
    return _lib.torch_calls().attend(q, k_cache, v_cache, pages, cu_rows, lens, tree_mask, scale, out, workspace)


def sample_rows(logits: torch.Tensor, u: torch.Tensor, temperature: Optional[torch.Tensor] = None,
                top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
                min_p: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, logprob: bool = False):
    """A token for each row of logits [rows, vocab] (hq4_sample_rows); int32
    [rows], with logprob also the float32 log probabilities of the tokens.

    u: float64 [rows], uniform in [0, 1); temperature, top_p, min_p: float32
    [rows], top_k: int32 [rows], None for off.  temperature <= 0 is greedy."""
    return _lib.torch_calls().sample_rows(logits, u, temperature, top_k, top_p, min_p, out, logprob)
