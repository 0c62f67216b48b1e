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
position, slot, page or length out of range). Tensors may be strided: the last dimension contiguous, strides
multiples of 8 elements and 16-byte aligned starts; others are copied once. The functions record nothing
for autograd: what they return has no graph, also for inputs that require one, and the expanded form's
gradients are a call of their own.
"""
import ctypes
import functools
from typing import Optional, Tuple

import torch

from .. import _lib as L
from . import dense

_DTYPES = {torch.bfloat16: 1, torch.float16: 2}


def _code(t: torch.Tensor, *others) -> int:
    """The library's type code of tensors on the current device that share a 16-bit type."""
    dt = t.dtype
    if dt not in _DTYPES:
        raise ValueError("latent attention takes bf16 or fp16 tensors")
    for o in others:
        if o is not None and o.dtype is not dt:
            raise ValueError("latent attention takes tensors of one type")
    return _DTYPES[dt]


_library = None
_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _lib():
    global _library
    if _library is None:
        _library = L.load()
    return _library


def _stream(*tensors) -> int:
    """The current stream, for CUDA tensors that all lie on the current device."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError("latent attention takes tensors of one CUDA device (no CPU fallback)")
    if dev < 0:
        raise ValueError("lazylora_b200 works on CUDA tensors only (no CPU fallback)")
    if dev != _device():
        raise ValueError(f"tensors on cuda:{dev}, while the current device is another")
    return _raw_stream(dev)


def _view(t: torch.Tensor, copy: bool = True):
    """(tensor, strides) as the kernels take them: the last dimension contiguous, the other strides
    positive multiples of 8, the start 16-byte aligned. A tensor that is not laid out so is copied once
    (copy), or None comes back; the stride of a dimension of one entry, which nothing uses, is replaced."""
    st = t.stride()
    fine = not t.data_ptr() & 15 and st[-1] == 1
    for s in st[:-1]:
        if s & 7 or s <= 0:
            fine = False
    if fine:
        return t, st
    st, inner, fine = list(st), t.shape[-1], not t.data_ptr() & 15 and (st[-1] == 1 or t.shape[-1] <= 1)
    for d in range(t.dim() - 2, -1, -1):
        if t.shape[d] <= 1:
            st[d] = max(8, (inner + 7) // 8 * 8)
        fine = fine and st[d] > 0 and st[d] % 8 == 0
        inner = max(inner, st[d] * t.shape[d])
    if fine or t.numel() == 0:
        return t, st
    if not copy:
        return None
    t = t.clone(memory_format=torch.contiguous_format)
    if all(s % 8 == 0 for s in t.stride()[:-1]):
        return t, t.stride()
    raise ValueError("latent attention: last dimensions must be multiples of 8")


def _ints(t: torch.Tensor, dtype, n: int, what: str) -> torch.Tensor:
    if t.dtype is not dtype or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{what}: {dtype} [{n}]")
    return t.contiguous()


def _table(table: torch.Tensor, d_r: int) -> torch.Tensor:
    if table.dim() != 2 or table.shape[1] != d_r or table.shape[0] == 0 or table.dtype is not torch.float32:
        raise ValueError(f"table: fp32 [positions, {d_r}], cosines then sines")
    table = table.contiguous()
    return table.clone() if table.data_ptr() & 15 else table


_NO_STRIDES = (8, 8)


def append_latent(cache: torch.Tensor, kv: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
                  table: torch.Tensor, q_pe: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
                  interleaved: bool = False) -> Optional[torch.Tensor]:
    """Write tokens into the paged cache [pages, page_size, d_c + d_r] in place.

    kv [T, d_c + d_r]: each token's latent row and its rotary key, not yet rotated; slots int64 [T]
    (page * page_size + offset, distinct; negative: not written); positions int64 [T]; table fp32
    [positions, d_r]: d_r / 2 cosines, then sines (d_r = its width). q_pe [T, H, d_r], the queries'
    rotary parts, come back rotated: in q_out when given (it may be q_pe itself, or a slice of the
    query buffer), else in a new tensor."""
    stream = _stream(cache, kv, slots, positions, table, q_pe, q_out)
    dt = _code(cache, kv, q_pe, q_out)
    if cache.dim() != 3 or kv.dim() != 2 or kv.shape[1] != cache.shape[2]:
        raise ValueError("cache [pages, page_size, d_c + d_r] and kv [T, d_c + d_r]")
    (T, D), d_r = kv.shape, table.shape[-1]
    d_c = D - d_r
    if d_c <= 0 or d_c % 16 or d_r % 16 or d_r == 0:
        raise ValueError("d_c and d_r must be positive multiples of 16")
    cv = _view(cache, copy=False)
    if cv is None or cache.numel() == 0:
        raise ValueError("cache: contiguous rows, strides multiples of 8, 16-byte aligned")
    cs, table = cv[1], _table(table, d_r)
    slots, positions = _ints(slots, torch.int64, T, "slots"), _ints(positions, torch.int64, T, "positions")
    kv, ks = _view(kv)
    H, qs, os_, qp, op = 0, _NO_STRIDES, _NO_STRIDES, None, None
    if q_pe is not None:
        if q_pe.dim() != 3 or q_pe.shape[0] != T or q_pe.shape[2] != d_r:
            raise ValueError(f"q_pe [T, H, {d_r}]")
        src, qs = _view(q_pe)
        if q_out is None:
            q_out = src.new_empty(q_pe.shape)
        ov = _view(q_out, copy=False)
        if q_out.shape != q_pe.shape or ov is None:
            raise ValueError("q_out: q_pe's shape, contiguous rows, strides multiples of 8, 16-byte aligned")
        H, os_, qp, op = q_pe.shape[1], ov[1], src.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q_pe")
    rc = _lib().ll_latent_append(kv.data_ptr(), ks[0], slots.data_ptr(), positions.data_ptr(), table.data_ptr(),
                                   table.shape[0], T, d_c, d_r, dt, interleaved, cache.data_ptr(), cs[0], cs[1],
                                   cache.shape[0], cache.shape[1], qp, qs[0], qs[1], H, op, os_[0], os_[1], stream)
    if rc:
        L.check(rc, "ll_latent_append")
    return q_out


def rotate_positions(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, inverse: bool = False,
                     interleaved: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [T, H, d_r] turned by its tokens' positions (inverse: turned back, the gradient), into out
    (may be x) or a new tensor. table as for append_latent."""
    stream = _stream(x, positions, table, out)
    dt = _code(x, out)
    if x.dim() != 3 or x.shape[2] % 16 or x.shape[2] == 0:
        raise ValueError("x [T, H, d_r] with d_r a multiple of 16")
    T, H, d_r = x.shape
    table, positions = _table(table, d_r), _ints(positions, torch.int64, T, "positions")
    src, xs = _view(x)
    if out is None:
        out = src.new_empty(x.shape)
    ov = _view(out, copy=False)
    if out.shape != x.shape or ov is None:
        raise ValueError("out: x's shape, contiguous rows, strides multiples of 8, 16-byte aligned")
    rc = _lib().ll_latent_rotate(src.data_ptr(), xs[0], xs[1], positions.data_ptr(), table.data_ptr(),
                                   table.shape[0], T, H, d_r, dt, interleaved, inverse, out.data_ptr(), ov[1][0],
                                   ov[1][1], stream)
    if rc:
        L.check(rc, "ll_latent_rotate")
    return out


@functools.lru_cache(maxsize=256)
def _paged_workspace(device: int, B: int, Tq: int, H: int, d_c: int) -> int:
    """Bytes on the current device, which is `device` (they go by its SMs)."""
    return _lib().ll_paged_latent_workspace_bytes(B, Tq, H, d_c)


def paged_latent_attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                           d_c: int, scale: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out [B, Tq, H, d_c], lse fp32 [B, Tq, H]) of the absorbed form.

    q [B, Tq, H, d_c + d_r]; cache [pages, page_size, d_c + d_r] (page_size a multiple of 8);
    block_table int32 [B, max_pages] (a page outside the cache is recorded for check_status(), its keys count as
    rows of zeros); seq_lens int32 [B], the cached rows of each sequence with the
    Tq queries' own tokens last (0 to max_pages * page_size; others are recorded for check_status()).
    Query t of sequence b sees its first seq_lens[b] - Tq + t + 1 rows; one that sees none gets zeros and
    lse = -inf. d_c 128, 256, 384 or 512; d_r 0 or 64 (append_latent takes 16 and more: without rotary values
    the rows are the program's own to write); scale > 0."""
    stream = _stream(q, cache, block_table, seq_lens)
    dt = _code(q, cache)
    if q.dim() != 4 or cache.dim() != 3 or q.shape[3] != cache.shape[2]:
        raise ValueError("q [B, Tq, H, d_c + d_r] and cache [pages, page_size, d_c + d_r]")
    B, Tq, H, D = q.shape
    pages, page_size, _ = cache.shape
    if d_c not in (128, 256, 384, 512) or D - d_c not in (0, 64):
        raise ValueError("d_c 128, 256, 384 or 512; d_r 0 or 64")
    cv = _view(cache, copy=False)
    if cv is None or page_size % 8 or cache.numel() == 0:
        raise ValueError("cache: page_size a multiple of 8, contiguous rows, strides multiples of 8, 16-byte aligned")
    if block_table.dim() != 2 or block_table.dtype is not torch.int32 or block_table.shape[0] != B or \
            block_table.shape[1] == 0:
        raise ValueError("block_table: int32 [B, max_pages]")
    if block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    seq_lens = _ints(seq_lens, torch.int32, B, "seq_lens")
    src, qs = _view(q)
    if Tq > 1 and H > 1 and qs[1] != H * qs[2]:                     # the rows (t, h) must be evenly spaced
        src = src.contiguous()
        qs = src.stride()
    out, lse = src.new_empty((B, Tq, H, d_c)), src.new_empty((B, Tq, H), dtype=torch.float32)
    if B == 0 or Tq == 0 or H == 0:
        return out, lse
    lib, cs = _lib(), cv[1]
    n = _paged_workspace(_device(), B, Tq, H, d_c)
    ws = src.new_empty(n, dtype=torch.uint8)
    rc = lib.ll_paged_latent_attention(src.data_ptr(), qs[0], qs[2] if H > 1 else qs[1], cache.data_ptr(), cs[0], cs[1],
                                       pages, page_size, block_table.data_ptr(), block_table.stride(0),
                                       block_table.shape[1], seq_lens.data_ptr(), B, Tq, H, d_c, D - d_c, scale, dt,
                                       out.data_ptr(), lse.data_ptr(), ws.data_ptr(), n, stream)
    if rc:
        L.check(rc, "ll_paged_latent_attention")
    return out, lse


def head_linear(x: torch.Tensor, w: torch.Tensor, w_nk: bool = True, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [T, H, N] bf16: x [T, H, K] times each head's weight, w [H, N, K] (w_nk, y = x w^T) or
    [H, K, N] (y = x w). K and N multiples of 8. out, when given, may be a slice of a wider buffer."""
    stream = _stream(x, w, out)
    if x.dtype is not torch.bfloat16 or w.dtype is not torch.bfloat16 or (out is not None and out.dtype is not torch.bfloat16):
        raise ValueError("head_linear takes bf16 tensors")
    if x.dim() != 3 or w.dim() != 3:
        raise ValueError("x [T, H, K] and w [H, N, K] or [H, K, N]")
    T, H, K = x.shape
    N, wk = (w.shape[1], w.shape[2]) if w_nk else (w.shape[2], w.shape[1])
    if w.shape[0] != H or wk != K:
        raise ValueError(f"head_linear: x {tuple(x.shape)} and w {tuple(w.shape)} do not match")
    if K % 8 or N % 8:
        raise ValueError("head_linear: K and N multiples of 8")
    (x, xs), (w, ws) = _view(x), _view(w)
    if out is None:
        out = x.new_empty((T, H, N))
    ov = _view(out, copy=False)
    if out.shape != (T, H, N) or ov is None:
        raise ValueError("out [T, H, N]: contiguous rows, strides multiples of 8, 16-byte aligned")
    os_ = ov[1]
    rc = _lib().ll_gemm_bf16_heads(T, H, N, K, x.data_ptr(), xs[0], xs[1], w.data_ptr(), ws[0], ws[1], w_nk,
                                     out.data_ptr(), os_[0], os_[1], stream)
    if rc:
        L.check(rc, "ll_gemm_bf16_heads")
    return out


def _packed(q, k_nope, k_pe, v, cu_q, cu_k, scale, causal):
    dt = _code(q, k_nope, k_pe, v)
    if q.dim() != 3 or k_nope.dim() != 3 or v.dim() != 3 or (k_pe is not None and k_pe.dim() != 2):
        raise ValueError("q [Tq, H, d_n + d_r], k_nope [Tk, H, d_n], k_pe [Tk, d_r] or None, v [Tk, H, d_v]")
    Tq, H, D = q.shape
    Tk, kh, d_n = k_nope.shape
    vt, vh, d_v = v.shape
    pt, d_r = (Tk, 0) if k_pe is None else k_pe.shape
    if kh != H or vh != H or vt != Tk or pt != Tk or D != d_n + d_r:
        raise ValueError("q [Tq, H, d_n + d_r], k_nope [Tk, H, d_n], k_pe [Tk, d_r] or None, v [Tk, H, d_v]")
    if d_n not in (64, 128) or d_v not in (64, 128) or d_r not in (0, 64) or H == 0:
        raise ValueError("d_n and d_v 64 or 128, d_r 0 (k_pe None) or 64, at least one head")
    if cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise ValueError("cu_q and cu_k: int32 [sequences + 1]")
    B = cu_q.shape[0] - 1
    if B == 0 and (Tq or Tk):
        raise ValueError("cu_q and cu_k: rows without a sequence")
    cu_q, cu_k = _ints(cu_q, torch.int32, B + 1, "cu_q"), _ints(cu_k, torch.int32, B + 1, "cu_k")
    (q, qs), (k_nope, ks), (v, vs) = _view(q), _view(k_nope), _view(v)
    k_pe, ps = (None, _NO_STRIDES) if k_pe is None else _view(k_pe)
    p = L.LatentPacked(B, Tq, Tk, H, d_n, d_r, d_v, causal, dt, scale, q.data_ptr(), qs[0], qs[1], k_nope.data_ptr(),
                       ks[0], ks[1], None if k_pe is None else k_pe.data_ptr(), ps[0], v.data_ptr(), vs[0], vs[1],
                       cu_q.data_ptr(), cu_k.data_ptr())
    return p, (q, k_nope, k_pe, v, cu_q, cu_k)


def latent_attention_forward(q: torch.Tensor, k_nope: torch.Tensor, k_pe: Optional[torch.Tensor], v: torch.Tensor,
                             cu_q: torch.Tensor, cu_k: torch.Tensor, scale: float,
                             causal: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out [Tq, H, d_v], lse fp32 [H, Tq]) on packed sequences.

    q [Tq, H, d_n + d_r], k_nope [Tk, H, d_n], k_pe [Tk, d_r] shared by the heads (None: d_r = 0),
    v [Tk, H, d_v]; sequence b is rows cu_q[b] .. cu_q[b + 1] of the queries and cu_k[b] .. cu_k[b + 1]
    of the keys (int32; the first is 0 and the last the number of rows, which check_status() holds them to: rows
    outside every sequence are not written). causal: query i of a sequence
    sees keys j <= i + keys - queries, so its last query sees them all; a query that sees none gets
    zeros and lse = -inf. d_n and d_v 64 or 128, d_r 0 or 64; scale > 0."""
    stream = _stream(q, k_nope, k_pe, v, cu_q, cu_k)
    p, keep = _packed(q, k_nope, k_pe, v, cu_q, cu_k, scale, causal)
    out, lse = q.new_empty((p.Tq, p.H, p.d_v)), q.new_empty((p.H, p.Tq), dtype=torch.float32)
    rc = _lib().ll_latent_forward(ctypes.byref(p), out.data_ptr(), lse.data_ptr(), stream)
    if rc:
        L.check(rc, "ll_latent_forward")
    return out, lse


def latent_attention_backward(g: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, q: torch.Tensor,
                              k_nope: torch.Tensor, k_pe: Optional[torch.Tensor], v: torch.Tensor, cu_q: torch.Tensor,
                              cu_k: torch.Tensor, scale: float, causal: bool = True):
    """(dq, dk_nope, dk_pe, dv) for the gradient g of out, from the forward's out and lse; dk_pe [Tk,
    d_r] is summed over the heads (None when k_pe is). Bitwise reproducible."""
    stream = _stream(g, out, lse, q, k_nope, k_pe, v, cu_q, cu_k)
    p, keep = _packed(q, k_nope, k_pe, v, cu_q, cu_k, scale, causal)
    _code(q, g, out)
    Tq, Tk, H, d_r, d_v = p.Tq, p.Tk, p.H, p.d_r, p.d_v
    if g.shape != (Tq, H, d_v) or out.shape != (Tq, H, d_v) or lse.shape != (H, Tq) or lse.dtype is not torch.float32:
        raise ValueError("g and out [Tq, H, d_v], lse fp32 [H, Tq]")
    (g, gs), out, lse = _view(g), _view(out.contiguous())[0], lse.contiguous()
    lib = _lib()
    dq, dk, dv = q.new_empty((Tq, H, p.d_n + d_r)), q.new_empty((Tk, H, p.d_n)), q.new_empty((Tk, H, d_v))
    dkpe = q.new_empty((Tk, d_r)) if d_r else None
    n = lib.ll_latent_backward_workspace_bytes(ctypes.byref(p))
    ws = q.new_empty(n, dtype=torch.uint8)
    rc = lib.ll_latent_backward(ctypes.byref(p), g.data_ptr(), gs[0], gs[1], out.data_ptr(), lse.data_ptr(),
                                dq.data_ptr(), dk.data_ptr(), L.ptr(dkpe), dv.data_ptr(), ws.data_ptr(), n, stream)
    if rc:
        L.check(rc, "ll_latent_backward")
    return dq, dk, dkpe, dv


def check_status():
    """Synchronise and raise if a call since the last check met a position, slot, page or length out of range
    (nothing is read or written outside, but the attention of such a sequence is not its formula's) or a
    bounded wait that ran out, head_linear's included (they are recorded with those of core.dense, whose
    check_status() this calls too)."""
    try:
        L.check(L.load().ll_latent_status(L.stream_ptr()), "latent attention")
    finally:
        dense.check_status()
