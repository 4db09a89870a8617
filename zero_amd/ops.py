"""Tensor-level wrappers over the C ABI (include/zero_hip.h).

PyTorch is used here for device memory and streams only; every arithmetic op below is a
hand-written gfx950 kernel in libzero_hip.so.  All tensors are bf16 on a ROCm device unless
stated; 2-D operands may be row-strided views (stride(1) == 1), so column slices of packed
buffers are passed without copies.
"""
from __future__ import annotations

from typing import Optional

import torch

import ctypes
import functools

from ._lib import GemmPlan, check, lib

EPI_NONE, EPI_QUICK_GELU, EPI_GELU_ERF, EPI_MUL_DQUICK_GELU, EPI_MUL_DGELU_ERF = 0, 1, 2, 3, 4
EPI_SWIGLU, EPI_SWIGLU_BWD = 5, 6
BF16 = torch.bfloat16


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    """hipStream_t of torch's current stream on the current device (the raw getter is ~20x cheaper than building a
    torch.cuda.Stream object per launch: 500 launches per step)."""
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _chk2d(t: torch.Tensor, name: str, dtype=BF16):
    if not t.is_cuda:
        raise ValueError(f"{name}: zero_amd kernels need a ROCm device tensor (no CPU path exists)")
    if t.dtype != dtype:
        raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name}: expected a 2-D row-major view, got shape {tuple(t.shape)} strides {t.stride()}")


def _ld(t: torch.Tensor) -> int:
    """Leading dimension of a 2-D row-major view; a single row may carry any stride (torch keeps the
    parent's), so its own width is reported instead."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _chk_flat(t: torch.Tensor, name: str, dtype=BF16):
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {dtype} ROCm tensor")


GEMV_MAX_ROWS = 4        # products with at most this many rows go to the weight-streaming kernel
_WORKSPACE = {}
WORKSPACE_BYTES = 160 << 20


def _workspace(device) -> torch.Tensor:
    """fp32 scratch for split-K GEMMs, one per (device, stream) — two streams that each run a split-K product
    must not share partial slabs — allocated on first use (the C ABI never allocates)."""
    key = (device, _stream())
    ws = _WORKSPACE.get(key)
    if ws is None:
        ws = _WORKSPACE[key] = torch.empty(WORKSPACE_BYTES // 4, dtype=torch.float32, device=device)
    return ws


# Kernel plan forced by tests / tools (None = the library's cost model).  This is state of the PYTHON harness,
# passed per call through zk_gemm_bf16_plan: libzero_hip.so itself holds no mutable tuning state.
_PLAN = None


def _gemm_call(*args):
    """args = the zk_gemm_bf16 argument list without the trailing stream."""
    if _PLAN is None:
        return lib.zk_gemm_bf16(*args, _stream())
    return lib.zk_gemm_bf16_plan(*args, ctypes.addressof(_PLAN), _stream())


def gemm(a: torch.Tensor, b: torch.Tensor, *, trans_a: bool = False, trans_b: bool = False,
         out: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
         residual: Optional[torch.Tensor] = None, epilogue: int = EPI_NONE,
         aux_out: Optional[torch.Tensor] = None, aux_in: Optional[torch.Tensor] = None,
         alpha: float = 1.0, alpha_dev: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """C[m,n] = epi(alpha * sum_k A(m,k) B(n,k)).  a: [M,K] (or [K,M] if trans_a); b: [N,K] (or [K,N] if trans_b)."""
    _chk2d(a, "a"); _chk2d(b, "b")
    M, K = (a.shape[1], a.shape[0]) if trans_a else (a.shape[0], a.shape[1])
    N, Kb = (b.shape[1], b.shape[0]) if trans_b else (b.shape[0], b.shape[1])
    if K != Kb:
        raise ValueError(f"gemm: contraction mismatch {K} vs {Kb}")
    if out is None:
        out = torch.empty((M, N), dtype=BF16, device=a.device)
    _chk2d(out, "out")
    if out.shape != (M, N):
        raise ValueError(f"gemm: out shape {tuple(out.shape)} != {(M, N)}")
    if bias is not None:
        _chk_flat(bias, "bias")
        if bias.numel() != N:
            raise ValueError("gemm: bias size")
    ldr = 0
    if residual is not None:
        _chk2d(residual, "residual")
        if residual.shape != (M, N):
            raise ValueError("gemm: residual shape")
        ldr = _ld(residual)
    if aux_out is not None:
        _chk2d(aux_out, "aux_out")
        if aux_out.shape != (M, N) or _ld(aux_out) != _ld(out):
            raise ValueError("gemm: aux_out must match out's shape and row stride")
    ldaux = 0
    if aux_in is not None:
        _chk2d(aux_in, "aux_in")
        if aux_in.shape != (M, N):
            raise ValueError("gemm: aux_in shape")
        ldaux = _ld(aux_in)
    if alpha_dev is not None:
        _chk_flat(alpha_dev, "alpha_dev", torch.float32)
    if (M <= GEMV_MAX_ROWS and not trans_a and not trans_b and epilogue == EPI_NONE and bias is None and aux_out is None
            and alpha_dev is None and alpha == 1.0 and not accumulate):
        # decode-time product: stream the weight once (zk_gemv_bf16) instead of a 128-row MFMA tile
        rc = lib.zk_gemv_bf16(_p(a), _p(b), _p(out), M, N, K, _ld(a), _ld(b), _ld(out), _p(residual), ldr, _stream())
        check(rc, f"zk_gemv_bf16 M={M} N={N} K={K}")
        return out
    rc = _gemm_call(_p(a), _p(b), _p(out), M, N, K, _ld(a), _ld(b), _ld(out),
                    int(trans_a), int(trans_b), epilogue, _p(bias), _p(residual), ldr, _p(aux_out),
                    _p(aux_in), ldaux, float(alpha), _p(alpha_dev), int(accumulate),
                    _workspace(a.device).data_ptr(), WORKSPACE_BYTES)
    check(rc, f"zk_gemm_bf16 M={M} N={N} K={K} tA={trans_a} tB={trans_b}")
    return out


def gemv_fused(x, w, *, xmode: int, ln_w=None, eps: float = 0.0, residual=None, out=None):
    """Decode-time product with the x operand made on the fly: xmode 1 = RMSNorm(x; ln_w, eps),
    xmode 2 = SwiGLU of the packed gate|up rows x [M, 2K].  M <= 4."""
    _chk2d(x, "x"); _chk2d(w, "w")
    M = x.shape[0]
    N, K = w.shape
    if (xmode == 2 and x.shape[1] != 2 * K) or (xmode != 2 and x.shape[1] != K):
        raise ValueError("gemv_fused: operand widths")
    if out is None:
        out = torch.empty((M, N), dtype=BF16, device=x.device)
    ldr = _ld(residual) if residual is not None else 0
    check(lib.zk_gemv_fused_bf16(_p(x), _p(w), _p(out), M, N, K, _ld(x), _ld(w), _ld(out), _p(residual), ldr, xmode,
                                 _p(ln_w), float(eps), _stream()), "zk_gemv_fused_bf16")
    return out


def interleave_gate_up(gate_w: torch.Tensor, up_w: torch.Tensor) -> torch.Tensor:
    """[2F, in] weight whose row blocks of 64 are [32 gate rows | the matching 32 up rows]: the layout
    the fused SwiGLU epilogues expect (include/zero_hip.h, ZK_EPI_SWIGLU).  One-time preparation."""
    F, K = gate_w.shape
    if F % 32 or up_w.shape != gate_w.shape:
        raise ValueError("interleave_gate_up: F must be a multiple of 32")
    return torch.stack((gate_w.reshape(F // 32, 32, K), up_w.reshape(F // 32, 32, K)), dim=1).reshape(2 * F, K).contiguous()


def gemm_swiglu(x: torch.Tensor, wgu_i: torch.Tensor, keep_gu: bool = True):
    """gu_i[M, 2F] = x @ wgu_i^T (interleaved gate|up, kept for backward) and h[M, F] = silu(gate) * up,
    in one launch (ZK_EPI_SWIGLU).  keep_gu=False (no backward will run): gu_i is neither allocated nor written
    (returned as None)."""
    _chk2d(x, "x"); _chk2d(wgu_i, "wgu_i")
    M, K = x.shape
    N = wgu_i.shape[0]
    if wgu_i.shape[1] != K or N % 64:
        raise ValueError("gemm_swiglu: shapes")
    gu = torch.empty((M, N), dtype=BF16, device=x.device) if keep_gu else None
    h = torch.empty((M, N // 2), dtype=BF16, device=x.device)
    rc = _gemm_call(_p(x), _p(wgu_i), _p(gu) if keep_gu else None, M, N, K, _ld(x), _ld(wgu_i), N, 0, 0,
                    EPI_SWIGLU, None, None, 0, _p(h), None, _ld(h), 1.0, None, 0,
                    _workspace(x.device).data_ptr(), WORKSPACE_BYTES)
    check(rc, f"zk_gemm_bf16(SWIGLU) M={M} N={N} K={K}")
    return gu, h


def gemm_swiglu_bwd(dy: torch.Tensor, w_down_t: torch.Tensor, gu_i: torch.Tensor) -> torch.Tensor:
    """d_gu_i[M, 2F] (interleaved) from dh = dy @ w_down_t^T (w_down_t: [F, d] = down_proj.weight^T) and the
    saved interleaved gate|up, in one launch (ZK_EPI_SWIGLU_BWD)."""
    _chk2d(dy, "dy"); _chk2d(w_down_t, "w_down_t"); _chk2d(gu_i, "gu_i")
    M, K = dy.shape
    F = w_down_t.shape[0]
    if w_down_t.shape[1] != K or gu_i.shape != (M, 2 * F) or F % 32:
        raise ValueError("gemm_swiglu_bwd: shapes")
    dgu = torch.empty((M, 2 * F), dtype=BF16, device=dy.device)
    rc = _gemm_call(_p(dy), _p(w_down_t), _p(dgu), M, F, K, dy.stride(0), w_down_t.stride(0), dgu.stride(0), 0, 0,
                    EPI_SWIGLU_BWD, None, None, 0, None, _p(gu_i), gu_i.stride(0), 1.0, None, 0,
                    _workspace(dy.device).data_ptr(), WORKSPACE_BYTES)
    check(rc, f"zk_gemm_bf16(SWIGLU_BWD) M={M} N={F} K={K}")
    return dgu


def attn_fwd(q, k, v, B: int, S: int, Hq: int, Hkv: int, hd: int, scale: float, causal: bool,
             out: Optional[torch.Tensor] = None, need_lse: bool = True, variant: str = "default"):
    """q/k/v: [B*S, H*hd] row-strided views.  Returns (o [B*S, Hq*hd], lse [B,Hq,S] fp32 or None).
    variant "w64" = the 64-rows-per-wave kernel (zk_attn_fwd_w64: tests / benchmarks)."""
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _chk2d(t, n)
    if q.shape != (B * S, Hq * hd) or k.shape != (B * S, Hkv * hd) or v.shape != (B * S, Hkv * hd):
        raise ValueError("attn_fwd: q/k/v shapes")
    if out is None:
        out = torch.empty((B * S, Hq * hd), dtype=BF16, device=q.device)
    _chk2d(out, "out")
    lse = torch.empty((B, Hq, S), dtype=torch.float32, device=q.device) if need_lse else None
    fn = {"default": lib.zk_attn_fwd, "w64": lib.zk_attn_fwd_w64}[variant]
    rc = fn(_p(q), _p(k), _p(v), _p(out), _p(lse), B, S, Hq, Hkv, hd, q.stride(0), k.stride(0),
            v.stride(0), out.stride(0), float(scale), int(causal), _stream())
    check(rc, "zk_attn_fwd")
    return out, lse


def attn_bwd(q, k, v, o, d_o, lse, dq, dk, dv, B: int, S: int, Hq: int, Hkv: int, hd: int, scale: float,
             causal: bool, rope=None):
    """Writes dq/dk/dv (row-strided views, may be slices of one packed d_qkv buffer).  rope = (cos, sin)
    fp32 [S, hd/2] tables: dq / dk then leave with the inverse rotary applied (= rope_(inverse=True) after)."""
    for t, n in ((q, "q"), (k, "k"), (v, "v"), (o, "o"), (d_o, "d_o"), (dq, "dq"), (dk, "dk"), (dv, "dv")):
        _chk2d(t, n)
    if o.stride(0) != d_o.stride(0):
        raise ValueError("attn_bwd: o and d_o must share a row stride")
    _chk_flat(lse, "lse", torch.float32)
    delta = torch.empty_like(lse)
    cos_t = sin_t = None
    if rope is not None:
        cos_t, sin_t = rope
        for t, n in ((cos_t, "cos"), (sin_t, "sin")):
            _chk_flat(t, n, torch.float32)
            if t.dim() != 2 or t.shape[0] < S or t.shape[1] != hd // 2:
                raise ValueError(f"attn_bwd: {n} table must be [>=S, hd/2]")
    rc = lib.zk_attn_bwd_rope(_p(q), _p(k), _p(v), _p(o), _p(d_o), _p(lse), _p(delta), _p(dq), _p(dk), _p(dv), B, S,
                              Hq, Hkv, hd, q.stride(0), k.stride(0), v.stride(0), o.stride(0), dq.stride(0),
                              dk.stride(0), dv.stride(0), float(scale), int(causal), _p(cos_t), _p(sin_t), _stream())
    check(rc, "zk_attn_bwd_rope")


def attn_decode(q, k_cache, v_cache, lens_i32, max_len: int, Hq: int, Hkv: int, hd: int, scale: float, out=None):
    """One query per sequence over a KV cache.  q: [B, Hq*hd]; caches: [B, rows, Hkv*hd] (contiguous
    last dim); lens_i32: int32 [B] valid rows per sequence (<= max_len <= rows)."""
    _chk2d(q, "q")
    B = q.shape[0]
    for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if t.dtype != BF16 or t.dim() != 3 or t.stride(2) != 1 or t.shape[0] != B or t.shape[2] != Hkv * hd:
            raise ValueError(f"attn_decode: {n} must be bf16 [B, rows, Hkv*hd]")
    if lens_i32.dtype != torch.int32 or lens_i32.numel() != B or max_len > k_cache.shape[1]:
        raise ValueError("attn_decode: lens must be int32 [B] and max_len within the cache")
    if out is None:
        out = torch.empty((B, Hq * hd), dtype=BF16, device=q.device)
    check(lib.zk_attn_decode(_p(q), _p(k_cache), _p(v_cache), _p(out), _p(lens_i32), B, Hq, Hkv, hd, q.stride(0),
                             k_cache.stride(1), v_cache.stride(1), out.stride(0), k_cache.stride(0), v_cache.stride(0),
                             int(max_len), float(scale), _stream()), "zk_attn_decode")
    return out


def attn_decode_fused(qkv, cos_t, sin_t, k_cache, v_cache, pos: int, Hq: int, Hkv: int, hd: int, scale: float,
                      ws: Optional[torch.Tensor] = None, out=None):
    """Single-token decoding step of the attention: RoPE of the new q / k (table rows of ``pos``), k / v
    appended to cache row ``pos``, attention over rows 0..pos split over 64-key chunks + merge.
    qkv: [B, (Hq + 2 Hkv) * hd] packed, BEFORE RoPE (left untouched); caches [B, rows, Hkv*hd] contiguous."""
    _chk2d(qkv, "qkv")
    B = qkv.shape[0]
    for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if t.dtype != BF16 or t.dim() != 3 or not t.is_contiguous() or t.shape[0] != B or t.shape[2] != Hkv * hd:
            raise ValueError(f"attn_decode_fused: {n} must be contiguous bf16 [B, rows, Hkv*hd]")
    rows = k_cache.shape[1]
    if v_cache.shape[1] != rows or not 0 <= pos < rows or qkv.shape[1] != (Hq + 2 * Hkv) * hd:
        raise ValueError("attn_decode_fused: position / shapes")
    for t in (cos_t, sin_t):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != hd // 2 or t.shape[0] <= pos or not t.is_contiguous():
            raise ValueError("attn_decode_fused: cos / sin tables must be fp32 [positions, hd / 2]")
    need = B * Hq * (pos // 64 + 1) * (hd + 2)
    if ws is None:
        ws = torch.empty(need, dtype=torch.float32, device=qkv.device)
    if ws.dtype != torch.float32 or ws.numel() < need or not ws.is_contiguous():
        raise ValueError("attn_decode_fused: workspace too small")
    if out is None:
        out = torch.empty((B, Hq * hd), dtype=BF16, device=qkv.device)
    check(lib.zk_attn_decode_fused(_p(qkv), cos_t[pos].data_ptr(), sin_t[pos].data_ptr(), _p(k_cache), _p(v_cache),
                                   _p(out), _p(ws), ws.numel(), B, Hq, Hkv, hd, qkv.stride(0), out.stride(0), rows,
                                   int(pos), float(scale), _stream()), "zk_attn_decode_fused")
    return out


def _here(name: str, *tensors):
    """The call's tensors are on the current device, where the kernel is launched (None passes)."""
    dev = -2
    for t in tensors:
        if t is not None:
            at = t.get_device()
            if dev == -2:
                dev = torch.cuda.current_device() if at >= 0 else -1
            if at != dev or at < 0:
                if at < 0:
                    raise ValueError(f"{name}: zero_amd kernels need ROCm device tensors (no CPU path exists)")
                raise ValueError(f"{name}: a tensor on cuda:{at}, but the current device is cuda:{dev}")


def _rows2d(name: str, what: str, t, rows: int, width: int) -> int:
    """Row stride of a bf16 row-major view [rows, width] (its device is checked by _here)."""
    if t.dtype != BF16 or t.shape != (rows, width) or (t.stride(1) != 1 and width > 1):
        raise ValueError(f"{name}: {what} must be a row-major bf16 view [{rows}, {width}], got {t.dtype} "
                         f"{tuple(t.shape)} strides {t.stride()}")
    return t.stride(0) if rows > 1 else (width + 7) // 8 * 8


def _chk_paged_cache(name: str, k_cache, v_cache, width: int):
    shape = k_cache.shape
    if (k_cache.dtype != BF16 or v_cache.dtype != BF16 or len(shape) != 3 or shape[2] != width or v_cache.shape != shape
            or not k_cache.is_contiguous() or not v_cache.is_contiguous()):
        raise ValueError(f"{name}: key and value caches must be contiguous bf16 [pages, page_size, {width}] of one shape")
    return shape


def _chk_vec(name: str, t, n: int, dtype, what: str):
    if t.dtype != dtype or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name}: {what} must be contiguous {dtype} [{n}]")


def kv_append_paged(qkv, cos_t, sin_t, k_cache, v_cache, positions, slots, Hq: int, Hkv: int, hd: int,
                    interleaved: bool = False, q_out=None):
    """T new tokens into a paged cache: rotated keys and values go to the flat cache rows ``slots`` (int32 [T]; outside
    the cache, e.g. -1: nothing is appended), the rotated queries are returned [T, Hq*hd].
    qkv: [T, (Hq + 2 Hkv) * hd] packed, before the rotation (left untouched); cos_t / sin_t fp32 [P, rot/2], rot <= hd a
    multiple of 16: the first rot values of a head turn by row ``positions[t]`` (int32 [T]; outside the table: a padding
    token, q row of zeros and nothing appended), value i with i + rot/2, or 2i with 2i + 1 (``interleaved``).
    Caches: contiguous [pages, page_size, Hkv*hd]; the live slots of one call are distinct."""
    name = "kv_append_paged"
    _here(name, qkv, cos_t, sin_t, k_cache, v_cache, positions, slots, q_out)
    T = qkv.shape[0]
    if Hq <= 0 or Hkv <= 0 or Hq % Hkv:
        raise ValueError(f"{name}: Hq must be a multiple of Hkv")
    ldqkv = _rows2d(name, "qkv", qkv, T, (Hq + 2 * Hkv) * hd)
    pages, page, _ = _chk_paged_cache(name, k_cache, v_cache, Hkv * hd)
    table = cos_t.shape
    if (cos_t.dtype != torch.float32 or len(table) != 2 or not cos_t.is_contiguous() or sin_t.dtype != torch.float32
            or sin_t.shape != table or not sin_t.is_contiguous()):
        raise ValueError(f"{name}: cos / sin tables must be contiguous fp32 [positions, rot / 2]")
    _chk_vec(name, positions, T, torch.int32, "positions")
    _chk_vec(name, slots, T, torch.int32, "slots")
    if q_out is None:
        q_out = qkv.new_empty((T, Hq * hd))
    ldq = _rows2d(name, "q_out", q_out, T, Hq * hd)
    if T == 0:
        return q_out
    rc = lib.zk_kv_append_paged(qkv.data_ptr(), cos_t.data_ptr(), sin_t.data_ptr(), q_out.data_ptr(), k_cache.data_ptr(),
                                v_cache.data_ptr(), positions.data_ptr(), slots.data_ptr(), T, Hq, Hkv, hd, 2 * table[1],
                                table[0], ldqkv, ldq, pages * page, 1 if interleaved else 0, _stream())
    if rc:
        check(rc, name)
    return q_out


@functools.lru_cache(maxsize=256)
def attn_paged_ws_floats(B: int, T: int, max_q: int, max_ctx: int, Hq: int, Hkv: int, hd: int) -> int:
    """fp32 values of workspace that attn_paged needs for such a call."""
    n = ctypes.c_int64()
    check(lib.zk_attn_paged_ws(B, T, max_q, max_ctx, Hq, Hkv, hd, ctypes.addressof(n)), "zk_attn_paged_ws")
    return n.value


def attn_paged(q, k_cache, v_cache, page_table, ctx_lens, cu_q, max_q: int, max_ctx: int, Hq: int, Hkv: int, hd: int,
               scale: float, tree_mask=None, out=None, ws=None):
    """Attention of the new tokens of B sequences over a paged cache that holds them already.  q [T, Hq*hd]: rows
    cu_q[b] .. cu_q[b+1]-1 (int32 [B+1]) are the n_b new tokens of sequence b, the last n_b of its ctx_lens[b]
    (int32 [B]) cached rows; row r is row r % page_size of page page_table[b, r // page_size] (int32 [B, cols]).
    A new token sees all rows before the new ones and, of those, the ones up to its own (tree_mask None) or the ones its
    bits name (tree_mask int64 [T, words], bit j % 64 of word j // 64 = new token j of the sequence; see
    inference.paged.tree_mask).  A token that sees nothing gets zeros.  max_q >= every n_b; max_ctx: an upper bound of
    ctx_lens that only shapes the launch.  Rows of q past cu_q[B] are left as they are in ``out``.
    ws: fp32 workspace of at least attn_paged_ws_floats(...) values (allocated when not given)."""
    name = "attn_paged"
    _here(name, q, k_cache, v_cache, page_table, ctx_lens, cu_q, tree_mask, out, ws)
    T = q.shape[0]
    if Hq <= 0 or Hkv <= 0 or Hq % Hkv:
        raise ValueError(f"{name}: Hq must be a multiple of Hkv")
    ldq = _rows2d(name, "q", q, T, Hq * hd)
    pages, page, _ = _chk_paged_cache(name, k_cache, v_cache, Hkv * hd)
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or (page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError(f"{name}: page_table must be int32 [B, columns]")
    B, cols = page_table.shape
    _chk_vec(name, ctx_lens, B, torch.int32, "ctx_lens")
    _chk_vec(name, cu_q, B + 1, torch.int32, "cu_q")
    words, mask = 0, None
    if tree_mask is not None:
        if tree_mask.dtype != torch.int64 or tree_mask.dim() != 2 or tree_mask.shape[0] != T or not tree_mask.is_contiguous():
            raise ValueError(f"{name}: tree_mask must be contiguous int64 [T, words]")
        words, mask = tree_mask.shape[1], tree_mask.data_ptr()
    if out is None:
        out = q.new_empty((T, Hq * hd))
    ldo = _rows2d(name, "out", out, T, Hq * hd)
    need = attn_paged_ws_floats(B, T, max_q, max_ctx, Hq, Hkv, hd)
    if ws is None:
        if need:
            ws = torch.empty(need, dtype=torch.float32, device=q.device)
    elif ws.dtype != torch.float32 or not ws.is_contiguous() or ws.numel() < need:
        raise ValueError(f"{name}: ws must be contiguous fp32 with at least {need} values")
    if T == 0:
        return out
    rc = lib.zk_attn_paged(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), page_table.data_ptr(),
                           ctx_lens.data_ptr(), cu_q.data_ptr(), mask, ws.data_ptr() if need else None, need, T, B, max_q,
                           max_ctx, Hq, Hkv, hd, page, pages, cols, page_table.stride(0) if B > 1 else cols, words, ldq, ldo,
                           scale, _stream())
    if rc:
        check(rc, name)
    return out


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Draws a token per row of bf16 logits [rows, V] with the numbers u (fp32 [rows], in [0, 1)); returns (tokens int64
    [rows], log-probabilities fp32 [rows] of the drawn tokens among the kept ones).  Settings are numbers for the call or
    tensors [rows] (fp32; top_k int32): temperature 0 = the largest logit; top_k 0, top_p 1 and min_p 0 keep everything.
    Tokens stand in falling order of their logit, equal ones by the lower index: top_k keeps the first, top_p the shortest
    prefix that reaches its share of what top_k kept, min_p those with at least that share of the largest's probability;
    the token drawn is the first whose running sum exceeds u times the kept sum (64-bit sums).  -inf is never drawn; a row
    of -inf gives token -1 with -inf, a row with a NaN -1 with NaN."""
    name = "sample"
    t, k, p, mp = temperature, top_k, top_p, min_p
    tt, kt, pt, mt = (v if torch.is_tensor(v) else None for v in (t, k, p, mp))
    _here(name, logits, u, tt, kt, pt, mt)
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"{name}: logits must be [rows, vocabulary]")
    rows, V = logits.shape
    if logits.dtype != BF16 or (logits.stride(1) != 1 and V > 1):
        raise ValueError(f"{name}: logits must be a row-major bf16 view")
    _chk_vec(name, u, rows, torch.float32, "u")
    if tt is not None:
        t = 0.0
        _chk_vec(name, tt, rows, torch.float32, "temperature")
    if kt is not None:
        k = 0
        _chk_vec(name, kt, rows, torch.int32, "top_k")
    if pt is not None:
        p = 1.0
        _chk_vec(name, pt, rows, torch.float32, "top_p")
    if mt is not None:
        mp = 0.0
        _chk_vec(name, mt, rows, torch.float32, "min_p")
    if not (0 <= t <= 2 ** 20 and 0 <= k < 2 ** 31 and k == int(k) and 0 < p <= 1 and 0 <= mp <= 1):
        raise ValueError(f"{name}: temperature in [0, 2^20], top_k a whole number >= 0, top_p in (0, 1], min_p in [0, 1]")
    tokens = torch.empty(rows, dtype=torch.int64, device=logits.device)
    logp = u.new_empty((rows,))
    if rows == 0:
        return tokens, logp
    rc = lib.zk_sample(logits.data_ptr(), u.data_ptr(), _p(tt), _p(kt), _p(pt), _p(mt), t, int(k), p, mp, tokens.data_ptr(),
                       logp.data_ptr(), rows, V, logits.stride(0) if rows > 1 else V, _stream())
    if rc:
        check(rc, name)
    return tokens, logp


def layernorm_fwd(x, gamma, beta, eps: float, save_stats: bool = True):
    _chk2d(x, "x"); _chk_flat(gamma, "gamma"); _chk_flat(beta, "beta")
    if not x.is_contiguous():
        raise ValueError("layernorm: x must be contiguous")
    rows, D = x.shape
    y = torch.empty_like(x)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device) if save_stats else None
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if save_stats else None
    check(lib.zk_layernorm_fwd(_p(x), _p(gamma), _p(beta), _p(y), _p(mean), _p(rstd), rows, D, float(eps), _stream()),
          "zk_layernorm_fwd")
    return y, mean, rstd


NORM_MAX_PARTS = 512


def norm_parts(rows: int) -> int:
    """Partial-sum count for the norm weight gradients: about 16 rows per workgroup."""
    return max(1, min(NORM_MAX_PARTS, (rows + 15) // 16))


def layernorm_bwd(dy, x, gamma, mean, rstd, dres=None, dgamma=None, dbeta=None, need_dx: bool = True):
    """dx = dres + LN'(dy).  dgamma / dbeta: fp32 [nparts, D] buffers that are OVERWRITTEN with partial sums
    (deterministic; add the parts in order — f32_to_bf16_multi_ does)."""
    _chk2d(dy, "dy"); _chk2d(x, "x")
    if not (dy.is_contiguous() and x.is_contiguous()):
        raise ValueError("layernorm_bwd: contiguous inputs required")
    rows, D = x.shape
    dx = torch.empty_like(x) if need_dx else None
    if dres is not None and not dres.is_contiguous():
        raise ValueError("layernorm_bwd: dres must be contiguous")
    nparts = 0
    if dgamma is not None:
        if (dbeta is None or dgamma.shape != dbeta.shape or dgamma.dim() != 2 or dgamma.shape[1] != D
                or dgamma.dtype != torch.float32 or not (dgamma.is_contiguous() and dbeta.is_contiguous())):
            raise ValueError("layernorm_bwd: dgamma / dbeta must be contiguous fp32 [nparts, D]")
        nparts = dgamma.shape[0]
    check(lib.zk_layernorm_bwd(_p(dy), _p(x), _p(gamma), _p(mean), _p(rstd), _p(dres), _p(dx), _p(dgamma), _p(dbeta),
                               nparts, rows, D, _stream()), "zk_layernorm_bwd")
    return dx


def rmsnorm_fwd(x, w, eps: float, save_stats: bool = True):
    _chk2d(x, "x"); _chk_flat(w, "w")
    if not x.is_contiguous():
        raise ValueError("rmsnorm: x must be contiguous")
    rows, D = x.shape
    y = torch.empty_like(x)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if save_stats else None
    check(lib.zk_rmsnorm_fwd(_p(x), _p(w), _p(y), _p(rstd), rows, D, float(eps), _stream()), "zk_rmsnorm_fwd")
    return y, rstd


def rmsnorm_bwd(dy, x, w, rstd, dres=None):
    _chk2d(dy, "dy"); _chk2d(x, "x")
    if not (dy.is_contiguous() and x.is_contiguous()) or (dres is not None and not dres.is_contiguous()):
        raise ValueError("rmsnorm_bwd: contiguous inputs required")
    rows, D = x.shape
    dx = torch.empty_like(x)
    check(lib.zk_rmsnorm_bwd(_p(dy), _p(x), _p(w), _p(rstd), _p(dres), _p(dx), rows, D, _stream()), "zk_rmsnorm_bwd")
    return dx


def rmsnorm_dweight_(dy, x, rstd, dw_parts):
    """dw_parts (fp32 [nparts, D], overwritten) = partial sums over rows of dy * bf16(x * rstd)."""
    _chk2d(dy, "dy"); _chk2d(x, "x"); _chk_flat(rstd, "rstd", torch.float32)
    if (not (dy.is_contiguous() and x.is_contiguous()) or dy.shape != x.shape or dw_parts.dim() != 2
            or dw_parts.shape[1] != x.shape[1] or dw_parts.dtype != torch.float32 or not dw_parts.is_contiguous()):
        raise ValueError("rmsnorm_dweight: contiguous [rows, D] inputs and an fp32 [nparts, D] buffer required")
    check(lib.zk_rmsnorm_dweight(_p(dy), _p(x), _p(rstd), _p(dw_parts), dw_parts.shape[0], x.shape[0], x.shape[1],
                                 _stream()), "zk_rmsnorm_dweight")
    return dw_parts


def rope_(x2d, cos_t, sin_t, S: int, heads: int, hd: int, inverse: bool = False):
    """In place on the first `heads*hd` columns of the row-strided view x2d."""
    _chk2d(x2d, "x")
    _chk_flat(cos_t, "cos", torch.float32); _chk_flat(sin_t, "sin", torch.float32)
    if cos_t.shape[0] < S or cos_t.shape[1] != hd // 2:
        raise ValueError("rope: table shape")
    check(lib.zk_rope(_p(x2d), _p(cos_t), _p(sin_t), x2d.shape[0], S, heads, hd, x2d.stride(0), int(inverse),
                      _stream()), "zk_rope")
    return x2d


def swiglu_fwd(gu, F: int):
    _chk2d(gu, "gu")
    if not gu.is_contiguous() or gu.shape[1] != 2 * F:
        raise ValueError("swiglu_fwd: gu must be contiguous [rows, 2F]")
    h = torch.empty((gu.shape[0], F), dtype=BF16, device=gu.device)
    check(lib.zk_swiglu_fwd(_p(gu), _p(h), gu.shape[0], F, _stream()), "zk_swiglu_fwd")
    return h


def swiglu_bwd(dh, gu, F: int):
    _chk2d(dh, "dh"); _chk2d(gu, "gu")
    if not (dh.is_contiguous() and gu.is_contiguous()):
        raise ValueError("swiglu_bwd: contiguous inputs required")
    dgu = torch.empty_like(gu)
    check(lib.zk_swiglu_bwd(_p(dh), _p(gu), _p(dgu), gu.shape[0], F, _stream()), "zk_swiglu_bwd")
    return dgu


def colsum_parts(rows: int) -> int:
    return max(1, min(128, rows // 64))


def colsum_(dy, out_parts):
    """out_parts (fp32 [nparts, N], overwritten) = partial column sums of dy (deterministic; add the parts in order)."""
    _chk2d(dy, "dy")
    if (out_parts.dim() != 2 or out_parts.shape[1] != dy.shape[1] or out_parts.dtype != torch.float32
            or not out_parts.is_contiguous()):
        raise ValueError("colsum: out must be a contiguous fp32 [nparts, N] buffer")
    check(lib.zk_colsum(_p(dy), _p(out_parts), dy.shape[0], dy.shape[1], dy.stride(0), out_parts.shape[0], _stream()),
          "zk_colsum")
    return out_parts


def act_bwd(dy, pre, kind: int, out=None):
    if not (dy.is_contiguous() and pre.is_contiguous()):
        raise ValueError("act_bwd: contiguous inputs required")
    if out is None:
        out = torch.empty_like(dy)
    check(lib.zk_act_bwd(_p(dy), _p(pre), _p(out), dy.numel(), kind, _stream()), "zk_act_bwd")
    return out


def patch_im2col(pixels, P: int, Kpad: int):
    if pixels.dtype != BF16 or not pixels.is_contiguous() or pixels.dim() != 4 or pixels.shape[1] != 3:
        raise ValueError("patch_im2col: pixels must be contiguous bf16 [B,3,H,W]")
    B, _, H, W = pixels.shape
    cols = torch.empty((B * (H // P) * (W // P), Kpad), dtype=BF16, device=pixels.device)
    check(lib.zk_patch_im2col(_p(pixels), _p(cols), B, H, W, P, Kpad, _stream()), "zk_patch_im2col")
    return cols


def embed_finish(patch, cls, pos, B: int, T: int, D: int):
    out = torch.empty((B, T, D), dtype=BF16, device=patch.device)
    check(lib.zk_embed_finish(_p(patch), _p(cls), _p(pos), _p(out), B, T, D, _stream()), "zk_embed_finish")
    return out


def transpose(w: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[C, R] = w[R, C]^T (bf16, rows of w may be strided; R and C multiples of 8)."""
    _chk2d(w, "w")
    R, C = w.shape
    if out is None:
        out = torch.empty((C, R), dtype=BF16, device=w.device)
    check(lib.zk_transpose_bf16(_p(w), _p(out), R, C, w.stride(0), out.stride(0), _stream()), "zk_transpose_bf16")
    return out


def gather_rows(table0, table1, codes, D: int, out=None, accumulate: bool = False):
    """out[r] = table0[code] (code>=0) | 0 (code==-1) | table1[-2-code] (code<=-2)."""
    if codes.dtype != torch.int32 or not codes.is_contiguous():
        raise ValueError("gather_rows: codes must be contiguous int32")
    rows = codes.numel()
    if out is None:
        out = torch.empty((rows, D), dtype=BF16, device=codes.device)
    check(lib.zk_gather_rows(_p(table0), _p(table1), _p(codes), _p(out), rows, D, int(accumulate), _stream()),
          "zk_gather_rows")
    return out


def cross_entropy(logits, targets_i32, loss_acc, dlogits=None):
    """loss_acc (fp32[2]) += [sum of row losses, number of non-ignored rows]."""
    _chk2d(logits, "logits")
    rows, V = logits.shape
    row_loss = torch.empty(rows, dtype=torch.float32, device=logits.device)      # ordered (reproducible) loss sum
    check(lib.zk_cross_entropy(_p(logits), _p(targets_i32), _p(loss_acc), _p(row_loss), _p(dlogits), rows, V,
                               logits.stride(0), _stream()), "zk_cross_entropy")
    return loss_acc


def sumsq_(g_flat, out_f32, scale: float = 1.0):
    parts = torch.empty(1024, dtype=torch.float32, device=g_flat.device)          # ZK_SUMSQ_PARTS: ordered block sums
    check(lib.zk_sumsq(_p(g_flat), _p(out_f32), _p(parts), g_flat.numel(), float(scale), _stream()), "zk_sumsq")
    return out_f32


def adamw_step_(p, g, m, v, *, lr, beta1, beta2, eps, weight_decay, step, max_norm, sumsq, grad_scale=1.0):
    check(lib.zk_adamw_step(_p(p), _p(g), _p(m), _p(v), p.numel(), float(lr), float(beta1), float(beta2), float(eps),
                            float(weight_decay), int(step), float(max_norm), _p(sumsq), float(grad_scale), _stream()),
          "zk_adamw_step")


def f32_to_bf16_(src, dst, scale: float = 1.0, accumulate: bool = False):
    check(lib.zk_f32_to_bf16(_p(src), _p(dst), src.numel(), float(scale), int(accumulate), _stream()),
          "zk_f32_to_bf16")
    return dst


def f32_to_bf16_multi_(pairs, scale: float = 1.0):
    """pairs: list of (src fp32 [nparts, n] partial sums (or flat [n]), dst bf16 flat [n], accumulate) — the parts
    are added in index order; ONE launch per 16 segments.  src rows may be strided column slices."""
    for i in range(0, len(pairs), 16):
        chunk = pairs[i:i + 16]
        k = len(chunk)
        np_, st_ = [], []
        for s_, d_, _ in chunk:
            if s_.dim() == 1:
                s_parts, s_n, s_stride = 1, s_.numel(), s_.numel()
                ok = s_.is_contiguous()
            else:
                s_parts, s_n = s_.shape
                s_stride = s_.stride(0) if s_parts > 1 else s_n
                ok = s_.dim() == 2 and s_.stride(1) == 1
            if s_.dtype != torch.float32 or d_.dtype != BF16 or s_n != d_.numel() or not ok or not d_.is_contiguous():
                raise ValueError("f32_to_bf16_multi: (fp32 [nparts, n], bf16 [n]) pairs required")
            np_.append(s_parts); st_.append(s_stride)
        srcs = (ctypes.c_void_p * k)(*[s_.data_ptr() for s_, _, _ in chunk])
        dsts = (ctypes.c_void_p * k)(*[d_.data_ptr() for _, d_, _ in chunk])
        ns = (ctypes.c_int64 * k)(*[d_.numel() for _, d_, _ in chunk])
        accs = (ctypes.c_int * k)(*[int(a_) for _, _, a_ in chunk])
        nps = (ctypes.c_int * k)(*np_)
        sts = (ctypes.c_int64 * k)(*st_)
        check(lib.zk_f32_to_bf16_multi(ctypes.cast(srcs, ctypes.c_void_p), ctypes.cast(dsts, ctypes.c_void_p),
                                       ctypes.cast(ns, ctypes.c_void_p), ctypes.cast(accs, ctypes.c_void_p),
                                       ctypes.cast(nps, ctypes.c_void_p), ctypes.cast(sts, ctypes.c_void_p), k,
                                       float(scale), _stream()), "zk_f32_to_bf16_multi")


def set_gemm_tile(cfg: int = -1):
    """Test / tool hook: edit the per-call kernel plan that ops.gemm passes to zk_gemm_bf16_plan (the numeric
    codes are kept from the round-1 tools).  -1 / 0..5 tile (cost model, 128x128, 256x128, 256x256, 128x96,
    384x192); 10 / 11 staging mode; 20 / 21 256x128 ring off / on; 30..33 ablation mode (needs a -DZK_ABLATION
    build); 40 / 41 lean addressing; 50 / 51 persistent ring off / on; 60 + b band; 100 split-K heuristic,
    101 no split-K, 102..116 forced splits; 100000 + t start stagger, 99999 built-in stagger.  When every field
    is back at its default the plan is dropped and the plain zk_gemm_bf16 entry is called again."""
    global _PLAN
    cfg = int(cfg)
    pl = _PLAN if _PLAN is not None else GemmPlan.default()
    if cfg in (10, 11):
        pl.stage_mode = cfg - 10
    elif cfg in (20, 21):
        pl.ring = cfg - 20
    elif 30 <= cfg <= 33:
        pl.ablation = cfg - 30
    elif cfg in (40, 41):
        pl.lean = cfg - 40
    elif cfg in (50, 51):
        pl.pring = cfg - 50
    elif 60 <= cfg <= 76:
        pl.band = cfg - 60
    elif cfg >= 100000:
        pl.phase_delay = cfg - 100000
    elif cfg == 99999:
        pl.phase_delay = -1
    elif 100 <= cfg <= 116:
        pl.splits = cfg - 100
    elif -1 <= cfg <= 5:
        pl.tile = cfg
    else:
        raise ValueError(f"set_gemm_tile: unknown code {cfg}")
    d = GemmPlan.default()
    builtin = {"stage_mode": 0, "ring": 1, "lean": 1, "pring": 1}          # what -1 means inside the library
    same = all(getattr(pl, n) == getattr(d, n) or builtin.get(n) == getattr(pl, n) for n, _ in GemmPlan._fields_)
    _PLAN = None if same else pl
