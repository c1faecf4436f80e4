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

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _stream_of(t: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _need_rows(t: torch.Tensor, name: str, heads, head_dim, like: Optional[torch.Tensor] = None) -> None:
    """[rows, heads, head_dim] whose rows may be apart (a view of a fused projection)."""
    if t.dim() != 3 or (heads is not None and t.shape[1] != heads) or (head_dim is not None and t.shape[2] != head_dim):
        raise RuntimeError(f"{name} must be [rows, heads, head_dim], got {tuple(t.shape)}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (no CPU fallback)")
    if t.dtype not in _TYPES:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != t.shape[2]):
        raise RuntimeError(f"{name}'s heads must lie one after another within a row")
    if like is not None and (t.dtype != like.dtype or t.shape[0] != like.shape[0] or t.device != like.device):
        raise RuntimeError(f"{name} must have q's rows, type and device")


def _need_ints(t: torch.Tensor, name: str, device, shape) -> None:
    if not t.is_cuda or t.device != device or t.dtype != torch.int32 or not t.is_contiguous() or t.shape != shape:
        raise RuntimeError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)} on {device}, "
                           f"got {t.dtype} {tuple(t.shape)} on {t.device}")


def _row_stride(t: torch.Tensor) -> int:
    """Elements from a row to the next (a lone row has none of its own)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]


def _need_caches(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor):
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if t.dim() != 4 or not t.is_cuda or t.device != q.device:
            raise RuntimeError(f"{name} must be [n_pages, n_kv, page_size, head_dim] on {q.device}")
        if t.dtype not in (torch.bfloat16, torch.float16) or t.dtype != k_cache.dtype:
            raise RuntimeError("the caches must be both bfloat16 or both float16")
        _, _, ps, hd = t.shape
        if t.stride()[1:] != (ps * hd, hd, 1):
            raise RuntimeError(f"{name}'s pages must each be contiguous")
    if v_cache.shape != k_cache.shape or v_cache.stride(0) != k_cache.stride(0):
        raise RuntimeError("k_cache and v_cache must have the same shape and strides")
    if q.dtype != torch.float32 and q.dtype != k_cache.dtype:
        raise RuntimeError(f"activations must be float32 or the caches' {k_cache.dtype}, got {q.dtype}")
    if q.device.index != torch.cuda.current_device():
        raise RuntimeError(f"tensors on {q.device}, current device {torch.cuda.current_device()}")


def _need_batch(q, pages, cu_rows, lens):
    n_seqs = lens.numel()
    _need_ints(lens, "lens", q.device, (n_seqs,))
    _need_ints(cu_rows, "cu_rows", q.device, (n_seqs + 1,))
    if pages.dim() != 2:
        raise RuntimeError("pages must be [n_seqs, pages_per_seq]")
    _need_ints(pages, "pages", q.device, (n_seqs, pages.shape[1]))
    return n_seqs


def _page_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2] * t.shape[3]


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
    each head before the rotation."""
    hd = k_cache.shape[-1] if k_cache.dim() == 4 else None
    _need_rows(q, "q", None, hd)
    _need_caches(q, k_cache, v_cache)
    n_pages, n_kv, ps, hd = k_cache.shape
    _need_rows(k, "k", n_kv, hd, q)
    _need_rows(v, "v", n_kv, hd, q)
    n_seqs = _need_batch(q, pages, cu_rows, lens)
    rows, nh = q.shape[0], q.shape[1]
    for t, name in ((rope_cos, "rope_cos"), (rope_sin, "rope_sin")):
        _need_cuda(t, name, torch.float32)
        if t.dim() != 2 or t.shape[1] * 2 != hd or t.shape != rope_cos.shape or t.device != q.device:
            raise RuntimeError(f"{name} must be [max_pos, head_dim / 2] on {q.device}")
    for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            _need_cuda(t, name, torch.float32)
            if t.shape != (hd,) or t.device != q.device:
                raise RuntimeError(f"{name} must be [head_dim] on {q.device}")
    if positions is not None:
        _need_ints(positions, "positions", q.device, (rows,))
    if out is None:
        out = torch.empty((rows, nh, hd), dtype=q.dtype, device=q.device)
    else:
        _need_cuda(out, "out", q.dtype)
        if out.shape != q.shape or out.device != q.device:
            raise RuntimeError("out must have q's shape and device")
    if rows == 0:
        return out
    rc = _lib.load().hq4_paged_append(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _TYPES[q.dtype], rows, nh, n_kv, hd, _row_stride(q), _row_stride(k),
        _row_stride(v), None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(),
        eps, cu_rows.data_ptr(), lens.data_ptr(), n_seqs, None if positions is None else positions.data_ptr(),
        rope_cos.data_ptr(), rope_sin.data_ptr(), rope_cos.shape[0], pages.data_ptr(), pages.shape[1],
        k_cache.data_ptr(), v_cache.data_ptr(), _TYPES[k_cache.dtype], n_pages, ps, _page_stride(k_cache),
        out.data_ptr(), _stream_of(q))
    if rc:
        _lib.check(rc, "hq4_paged_append")
    return out


def paged_attention_workspace(q: torch.Tensor, k_cache: torch.Tensor, pages: torch.Tensor) -> torch.Tensor:
    """A workspace for paged_attention / tree_attention calls of these shapes
    (one to a stream; the calls take a fresh one where none is given)."""
    n = int(_lib.load().hq4_paged_attention_workspace_bytes(
        _TYPES[q.dtype], q.shape[0], q.shape[1], k_cache.shape[1], q.shape[2], pages.shape[0], pages.shape[1],
        k_cache.shape[2]))
    if n < 0:
        raise RuntimeError(f"hq4_paged_attention_workspace_bytes = {n} for q {tuple(q.shape)}, "
                           f"cache {tuple(k_cache.shape)}")
    return torch.empty(n, dtype=torch.uint8, device=q.device)


def _attend(q, k_cache, v_cache, pages, cu_rows, lens, tree_mask, scale, out, workspace):
    hd = k_cache.shape[-1] if k_cache.dim() == 4 else None
    _need_rows(q, "q", None, hd)
    _need_caches(q, k_cache, v_cache)
    n_seqs = _need_batch(q, pages, cu_rows, lens)
    n_pages, n_kv, ps, hd = k_cache.shape
    rows, nh = q.shape[0], q.shape[1]
    if scale is None:
        scale = hd ** -0.5
    if out is None:
        out = torch.empty((rows, nh, hd), dtype=q.dtype, device=q.device)
    else:
        _need_cuda(out, "out", q.dtype)
        if out.shape != q.shape or out.device != q.device:
            raise RuntimeError("out must have q's shape and device")
    if rows == 0:
        return out
    if workspace is None:
        workspace = paged_attention_workspace(q, k_cache, pages)
    else:
        _need_cuda(workspace, "workspace", torch.uint8)
        if workspace.device != q.device:
            raise RuntimeError(f"workspace must be on {q.device}")
    lib = _lib.load()
    head = (q.data_ptr(), _TYPES[q.dtype], rows, nh, n_kv, hd, _row_stride(q), cu_rows.data_ptr(), lens.data_ptr(),
            n_seqs, pages.data_ptr(), pages.shape[1], k_cache.data_ptr(), v_cache.data_ptr(), _TYPES[k_cache.dtype],
            n_pages, ps, _page_stride(k_cache))
    tail = (scale, out.data_ptr(), workspace.data_ptr(), workspace.numel(), _stream_of(q))
    if tree_mask is None:
        rc = lib.hq4_paged_attention(*head, *tail)
    else:
        rc = lib.hq4_tree_attention(*head, tree_mask.data_ptr(), tree_mask.shape[1], *tail)
    if rc:
        _lib.check(rc, "hq4_paged_attention" if tree_mask is None else "hq4_tree_attention")
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pages: torch.Tensor,
                    cu_rows: torch.Tensor, lens: torch.Tensor, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal grouped-query attention of a ragged batch over the paged cache
    (hq4_paged_attention): row i of sequence s sees entries 0 .. lens[s] + i.
    q: [rows, n_heads, head_dim] as paged_append returns it; scale defaults to
    head_dim ** -0.5.  Decode, prompt chunks and mixtures of them alike."""
    return _attend(q, k_cache, v_cache, pages, cu_rows, lens, None, scale, out, workspace)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pages: torch.Tensor,
                   cu_rows: torch.Tensor, lens: torch.Tensor, tree_mask: torch.Tensor, scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """paged_attention for trees of drafted tokens (hq4_tree_attention): row i
    of sequence s sees the entries before lens[s], and entry lens[s] + j where
    bit j % 32 of tree_mask[row, j // 32] is set (int32 words)."""
    _need_cuda(tree_mask, "tree_mask", torch.int32)
    if tree_mask.dim() != 2 or tree_mask.shape[0] != q.shape[0] or tree_mask.shape[1] < 1 \
            or tree_mask.device != q.device:
        raise RuntimeError(f"tree_mask must be int32 [rows, words] on {q.device}")
    return _attend(q, k_cache, v_cache, pages, cu_rows, lens, tree_mask, scale, out, workspace)


def sample_rows(logits: torch.Tensor, u: torch.Tensor, temperature: Optional[torch.Tensor] = None,
                top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
                min_p: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, logprob: bool = False):
    """A token for each row of logits [rows, vocab] (hq4_sample_rows); int32
    [rows], with logprob also the float32 log probabilities of the tokens.

    u: float64 [rows], uniform in [0, 1); temperature, top_p, min_p: float32
    [rows], top_k: int32 [rows], None for off.  temperature <= 0 is greedy."""
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in _TYPES:
        raise RuntimeError("logits must be a CUDA float32, bfloat16 or float16 tensor [rows, vocab]")
    rows, n = logits.shape
    if n > 1 and logits.stride(1) != 1:
        raise RuntimeError("logits' rows must each be contiguous")
    if logits.device.index != torch.cuda.current_device():
        raise RuntimeError(f"tensors on {logits.device}, current device {torch.cuda.current_device()}")
    ptrs = []
    for t, name, dt in ((u, "u", torch.float64), (temperature, "temperature", torch.float32),
                        (top_k, "top_k", torch.int32), (top_p, "top_p", torch.float32),
                        (min_p, "min_p", torch.float32), (out, "out", torch.int32)):
        if t is None:
            ptrs.append(None)
            continue
        if not t.is_cuda or t.dtype != dt or t.shape != (rows,) or not t.is_contiguous() or t.device != logits.device:
            raise RuntimeError(f"{name} must be a contiguous {dt} tensor of {rows} values on {logits.device}")
        ptrs.append(t.data_ptr())
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=logits.device)
        ptrs[5] = out.data_ptr()
    lp = torch.empty(rows, dtype=torch.float32, device=logits.device) if logprob else None
    if rows:
        rc = _lib.load().hq4_sample_rows(
            logits.data_ptr(), _TYPES[logits.dtype], rows, n, logits.stride(0) if rows > 1 else n, ptrs[1], ptrs[2],
            ptrs[3], ptrs[4], ptrs[0], ptrs[5], None if lp is None else lp.data_ptr(), _stream_of(logits))
        if rc:
            _lib.check(rc, "hq4_sample_rows")
    return (out, lp) if logprob else out
