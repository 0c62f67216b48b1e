"""
Latent attention on the GPU: the attention of a layer whose keys and values come from one shared
latent vector per token (d_c values) and one rotary key per token (d_r values, shared by the heads).

  * append_latent            new tokens' latent rows into a paged cache, their rotary keys (and the
                             queries' rotary parts) turned on the way
  * paged_latent_attention   the absorbed form over that cache, for decoding: a cache row is the key
                             of every head and, its first d_c entries, the value
  * head_linear              one product per head: queries into the latent space, outputs back
  * latent_attention_forward / _backward
                             the expanded form on packed sequences: per-head keys and values, the
                             rotary key shared by the heads; with its gradients, for training
  * rotate_positions         the rotation alone, and its inverse (its gradient)

bf16 or fp16 tensors, fp32 softmax statistics and sums; CUDA tensors only, no fallback. Calls run on
the current stream and synchronise nothing; check_status() raises for what only the device can see (a
position, slot or page out of range). Tensors may be strided: the last dimension contiguous, strides
multiples of 8 elements and 16-byte aligned starts; others are copied once.
"""
import ctypes
from typing import Optional, Tuple

import torch

from .. import _lib as L

_DTYPES = {torch.bfloat16: 1, torch.float16: 2}


def _code(*tensors) -> int:
    dt = tensors[0].dtype
    if dt not in _DTYPES or any(t is not None and t.dtype != dt for t in tensors):
        raise ValueError("latent attention takes bf16 or fp16 tensors of one type")
    return _DTYPES[dt]


def _fits(t: torch.Tensor) -> bool:
    if t.data_ptr() % 16 or (t.shape[-1] > 1 and t.stride(-1) != 1):
        return False
    return all(st % 8 == 0 and st >= 8 for st, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)


def _in(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself when the kernels can read it in place, else a contiguous copy."""
    return t if _fits(t) else t.clone(memory_format=torch.contiguous_format)


def _st(t: torch.Tensor, d: int) -> int:
    """A stride the library accepts (of a dimension of one entry, whose stride is never used, the
    extent of what lies inside it)."""
    if t.shape[d] > 1:
        return t.stride(d)
    inner = 1
    for i in range(d + 1 if d >= 0 else t.dim() + d + 1, t.dim()):
        inner = max(inner, t.stride(i) * t.shape[i])
    return (inner + 7) // 8 * 8


def _ints(t: torch.Tensor, dtype, shape, what: str) -> torch.Tensor:
    if t.dtype != dtype or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: {dtype} {tuple(shape)}")
    return t.contiguous()


def _table(table: torch.Tensor, d_r: int) -> torch.Tensor:
    if table.dim() != 2 or table.shape[1] != d_r or table.shape[0] == 0 or table.dtype != torch.float32:
        raise ValueError(f"table: fp32 [positions, {d_r}], cosines then sines")
    return _in(table.contiguous())


def append_latent(cache: torch.Tensor, kv: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
                  table: torch.Tensor, q_pe: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
                  interleaved: bool = False) -> Optional[torch.Tensor]:
    """Write tokens into the paged cache [pages, page_size, d_c + d_r] in place.

    kv [T, d_c + d_r]: each token's latent row and its rotary key, not yet rotated; slots int64 [T]
    (page * page_size + offset, distinct; negative: not written); positions int64 [T]; table fp32
    [positions, d_r]: d_r / 2 cosines, then sines (d_r = its width). q_pe [T, H, d_r], the queries'
    rotary parts, come back rotated: in q_out when given (it may be q_pe itself, or a slice of the
    query buffer), else in a new tensor."""
    L.require_cuda(cache, kv, slots, positions, table, q_pe, q_out)
    dt = _code(cache, kv, q_pe, q_out)
    if cache.dim() != 3 or kv.dim() != 2 or kv.shape[1] != cache.shape[2]:
        raise ValueError("cache [pages, page_size, d_c + d_r] and kv [T, d_c + d_r]")
    T, d_r = kv.shape[0], table.shape[-1]
    d_c = kv.shape[1] - d_r
    if d_c <= 0 or d_c % 16 or d_r % 16 or d_r == 0:
        raise ValueError("d_c and d_r must be positive multiples of 16")
    if not _fits(cache) or cache.numel() == 0:
        raise ValueError("cache: contiguous rows, strides multiples of 8, 16-byte aligned")
    table = _table(table, d_r)
    slots, positions = _ints(slots, torch.int64, (T,), "slots"), _ints(positions, torch.int64, (T,), "positions")
    kv = _in(kv)
    H, qs, os_, qp, op = 0, (0, 0), (0, 0), None, None
    if q_pe is not None:
        if q_pe.dim() != 3 or q_pe.shape[0] != T or q_pe.shape[2] != d_r:
            raise ValueError(f"q_pe [T, H, {d_r}]")
        src = _in(q_pe)
        if q_out is None:
            q_out = torch.empty(q_pe.shape, dtype=q_pe.dtype, device=q_pe.device)
        elif q_out.shape != q_pe.shape or not _fits(q_out):
            raise ValueError("q_out: q_pe's shape, contiguous rows, strides multiples of 8, 16-byte aligned")
        H, qs, os_ = q_pe.shape[1], (_st(src, 0), _st(src, 1)), (_st(q_out, 0), _st(q_out, 1))
        qp, op = src.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q_pe")
    page_stride, row_stride = _st(cache, 0), _st(cache, 1)
    L.check(L.load().ll_latent_append(kv.data_ptr(), _st(kv, 0), slots.data_ptr(), positions.data_ptr(),
                                      table.data_ptr(), table.shape[0], T, d_c, d_r, dt, int(interleaved),
                                      cache.data_ptr(), page_stride, row_stride, cache.shape[0], cache.shape[1], qp,
                                      qs[0], qs[1], H, op, os_[0], os_[1], L.stream_ptr()), "ll_latent_append")
    return q_out


def rotate_positions(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, inverse: bool = False,
                     interleaved: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [T, H, d_r] turned by its tokens' positions (inverse: turned back, the gradient), into out
    (may be x) or a new tensor. table as for append_latent."""
    L.require_cuda(x, positions, table, out)
    dt = _code(x, out)
    if x.dim() != 3 or x.shape[2] % 16 or x.shape[2] == 0:
        raise ValueError("x [T, H, d_r] with d_r a multiple of 16")
    T, H, d_r = x.shape
    table, positions = _table(table, d_r), _ints(positions, torch.int64, (T,), "positions")
    src = _in(x)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or not _fits(out):
        raise ValueError("out: x's shape, contiguous rows, strides multiples of 8, 16-byte aligned")
    L.check(L.load().ll_latent_rotate(src.data_ptr(), _st(src, 0), _st(src, 1), positions.data_ptr(), table.data_ptr(),
                                      table.shape[0], T, H, d_r, dt, int(interleaved), int(inverse), out.data_ptr(),
                                      _st(out, 0), _st(out, 1), L.stream_ptr()), "ll_latent_rotate")
    return out


def paged_latent_attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                           d_c: int, scale: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out [B, Tq, H, d_c], lse fp32 [B, Tq, H]) of the absorbed form.

    q [B, Tq, H, d_c + d_r]; cache [pages, page_size, d_c + d_r] (page_size a multiple of 8);
    block_table int32 [B, max_pages]; seq_lens int32 [B], the cached rows of each sequence with the
    Tq queries' own tokens last. Query t of sequence b sees its first seq_lens[b] - Tq + t + 1 rows;
    one that sees none gets zeros and lse = -inf. d_c 128, 256, 384 or 512; d_r 0 or 64."""
    L.require_cuda(q, cache, block_table, seq_lens)
    dt = _code(q, cache)
    if q.dim() != 4 or cache.dim() != 3 or q.shape[3] != cache.shape[2]:
        raise ValueError("q [B, Tq, H, d_c + d_r] and cache [pages, page_size, d_c + d_r]")
    B, Tq, H, D = q.shape
    d_r = D - d_c
    if d_c not in (128, 256, 384, 512) or d_r not in (0, 64):
        raise ValueError("d_c 128, 256, 384 or 512; d_r 0 or 64")
    if cache.shape[1] % 8 or cache.numel() == 0 or not _fits(cache):
        raise ValueError("cache: page_size a multiple of 8, contiguous rows, strides multiples of 8, 16-byte aligned")
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.shape[0] != B or \
            block_table.shape[1] == 0 or block_table.stride(1) != 1:
        raise ValueError("block_table: int32 [B, max_pages]")
    seq_lens = _ints(seq_lens, torch.int32, (B,), "seq_lens")
    lib, src = L.load(), _in(q)
    if Tq > 1 and H > 1 and src.stride(1) != H * src.stride(2):     # the rows (t, h) must be evenly spaced
        src = src.contiguous()
    out = torch.empty((B, Tq, H, d_c), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, Tq, H), dtype=torch.float32, device=q.device)
    if out.numel() == 0:
        return out, lse
    n = lib.ll_paged_latent_workspace_bytes(B, Tq, H, d_c)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device)
    L.check(lib.ll_paged_latent_attention(src.data_ptr(), _st(src, 0), _st(src, 2) if H > 1 else _st(src, 1),
                                          cache.data_ptr(), _st(cache, 0), _st(cache, 1), cache.shape[0], cache.shape[1],
                                          block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
                                          seq_lens.data_ptr(), B, Tq, H, d_c, d_r, float(scale), dt, out.data_ptr(),
                                          lse.data_ptr(), ws.data_ptr(), n, L.stream_ptr()),
            "ll_paged_latent_attention")
    return out, lse


def head_linear(x: torch.Tensor, w: torch.Tensor, w_nk: bool = True, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [T, H, N] bf16: x [T, H, K] times each head's weight, w [H, N, K] (w_nk, y = x w^T) or
    [H, K, N] (y = x w). out, when given, may be a slice of a wider buffer."""
    L.require_cuda(x, w, out)
    if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16 or (out is not None and out.dtype != torch.bfloat16):
        raise ValueError("head_linear takes bf16 tensors")
    if x.dim() != 3 or w.dim() != 3:
        raise ValueError("x [T, H, K] and w [H, N, K] or [H, K, N]")
    T, H, K = x.shape
    N = w.shape[1] if w_nk else w.shape[2]
    if w.shape[0] != H or w.shape[2 if w_nk else 1] != K:
        raise ValueError(f"head_linear: x {tuple(x.shape)} and w {tuple(w.shape)} do not match")
    if K % 8 or N % 8:
        raise ValueError("head_linear: K and N multiples of 8")
    a, b = _in(x), _in(w)
    if out is None:
        out = torch.empty((T, H, N), dtype=x.dtype, device=x.device)
    elif tuple(out.shape) != (T, H, N) or not _fits(out):
        raise ValueError("out [T, H, N]: contiguous rows, strides multiples of 8, 16-byte aligned")
    L.check(L.load().ll_gemm_bf16_heads(T, H, N, K, a.data_ptr(), max(_st(a, 0), K), _st(a, 1), b.data_ptr(), _st(b, 0),
                                        _st(b, 1), int(w_nk), out.data_ptr(), max(_st(out, 0), N), _st(out, 1),
                                        L.stream_ptr()), "ll_gemm_bf16_heads")
    return out


def _packed(q, k_nope, k_pe, v, cu_q, cu_k, scale, causal):
    L.require_cuda(q, k_nope, k_pe, v, cu_q, cu_k)
    dt = _code(q, k_nope, k_pe, v)
    if q.dim() != 3 or k_nope.dim() != 3 or v.dim() != 3 or (k_pe is not None and k_pe.dim() != 2):
        raise ValueError("q [Tq, H, d_n + d_r], k_nope [Tk, H, d_n], k_pe [Tk, d_r] or None, v [Tk, H, d_v]")
    Tq, H, D = q.shape
    Tk, d_n, d_v = k_nope.shape[0], k_nope.shape[2], v.shape[2]
    d_r = 0 if k_pe is None else k_pe.shape[1]
    if k_nope.shape[1] != H or tuple(v.shape[:2]) != (Tk, H) or D != d_n + d_r or (k_pe is not None and k_pe.shape[0] != Tk):
        raise ValueError("q [Tq, H, d_n + d_r], k_nope [Tk, H, d_n], k_pe [Tk, d_r] or None, v [Tk, H, d_v]")
    if d_n not in (64, 128) or d_v not in (64, 128) or d_r not in (0, 64) or H == 0:
        raise ValueError("d_n and d_v 64 or 128, d_r 0 (k_pe None) or 64, at least one head")
    if cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise ValueError("cu_q and cu_k: int32 [sequences + 1]")
    B = cu_q.shape[0] - 1
    cu_q, cu_k = _ints(cu_q, torch.int32, (B + 1,), "cu_q"), _ints(cu_k, torch.int32, (B + 1,), "cu_k")
    q, k_nope, v = _in(q), _in(k_nope), _in(v)
    k_pe = None if k_pe is None else _in(k_pe)
    p = L.LatentPacked(B, Tq, Tk, H, d_n, d_r, d_v, int(bool(causal)), dt, float(scale), q.data_ptr(), _st(q, 0), _st(q, 1),
                       k_nope.data_ptr(), _st(k_nope, 0), _st(k_nope, 1), L.ptr(k_pe), 0 if k_pe is None else _st(k_pe, 0),
                       v.data_ptr(), _st(v, 0), _st(v, 1), cu_q.data_ptr(), cu_k.data_ptr())
    return p, (q, k_nope, k_pe, v, cu_q, cu_k)


def latent_attention_forward(q: torch.Tensor, k_nope: torch.Tensor, k_pe: Optional[torch.Tensor], v: torch.Tensor,
                             cu_q: torch.Tensor, cu_k: torch.Tensor, scale: float,
                             causal: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out [Tq, H, d_v], lse fp32 [H, Tq]) on packed sequences.

    q [Tq, H, d_n + d_r], k_nope [Tk, H, d_n], k_pe [Tk, d_r] shared by the heads (None: d_r = 0),
    v [Tk, H, d_v]; sequence b is rows cu_q[b] .. cu_q[b + 1] of the queries and cu_k[b] .. cu_k[b + 1]
    of the keys (int32; the first is 0 and the last the number of rows). causal: query i of a sequence
    sees keys j <= i + keys - queries, so its last query sees them all; a query that sees none gets
    zeros and lse = -inf."""
    p, keep = _packed(q, k_nope, k_pe, v, cu_q, cu_k, scale, causal)
    out = torch.empty((p.Tq, p.H, p.d_v), dtype=q.dtype, device=q.device)
    lse = torch.empty((p.H, p.Tq), dtype=torch.float32, device=q.device)
    L.check(L.load().ll_latent_forward(ctypes.byref(p), out.data_ptr(), lse.data_ptr(), L.stream_ptr()),
            "ll_latent_forward")
    return out, lse


def latent_attention_backward(g: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, q: torch.Tensor,
                              k_nope: torch.Tensor, k_pe: Optional[torch.Tensor], v: torch.Tensor, cu_q: torch.Tensor,
                              cu_k: torch.Tensor, scale: float, causal: bool = True):
    """(dq, dk_nope, dk_pe, dv) for the gradient g of out, from the forward's out and lse; dk_pe [Tk,
    d_r] is summed over the heads (None when k_pe is). Bitwise reproducible."""
    p, keep = _packed(q, k_nope, k_pe, v, cu_q, cu_k, scale, causal)
    L.require_cuda(g, out, lse)
    _code(keep[0], g, out)
    if tuple(g.shape) != (p.Tq, p.H, p.d_v) or tuple(out.shape) != (p.Tq, p.H, p.d_v) or \
            tuple(lse.shape) != (p.H, p.Tq) or lse.dtype != torch.float32:
        raise ValueError("g and out [Tq, H, d_v], lse fp32 [H, Tq]")
    g, out, lse = _in(g), out.contiguous(), lse.contiguous()
    lib, dev = L.load(), q.device
    new = lambda *shape: torch.empty(shape, dtype=q.dtype, device=dev)  # noqa: E731
    dq, dk, dv = new(p.Tq, p.H, p.d_n + p.d_r), new(p.Tk, p.H, p.d_n), new(p.Tk, p.H, p.d_v)
    dkpe = new(p.Tk, p.d_r) if p.d_r else None
    n = lib.ll_latent_backward_workspace_bytes(ctypes.byref(p))
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device=dev)
    L.check(lib.ll_latent_backward(ctypes.byref(p), g.data_ptr(), _st(g, 0), _st(g, 1), out.data_ptr(), lse.data_ptr(),
                                   dq.data_ptr(), dk.data_ptr(), L.ptr(dkpe), dv.data_ptr(), ws.data_ptr(), n,
                                   L.stream_ptr()), "ll_latent_backward")
    return dq, dk, dkpe, dv


def check_status():
    """Synchronise and raise if a call since the last check met a position, slot or page out of range
    (it was skipped) or a bounded wait that ran out."""
    L.check(L.load().ll_latent_status(L.stream_ptr()), "latent attention")
