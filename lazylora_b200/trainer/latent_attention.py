"""
A latent-attention layer on the GPU: the attention half beside the MoE half that latent_moe.py,
routed_experts.py and shared_expert.py run. Keys and values come from one shared latent vector per
token (d_c values, RMS-normed when a norm weight is given) and one rotary key per token shared by the
heads:

    q            = x W_q^T                        [N, H, d_n + d_r], its last d_r values rotated
    (c, k_pe)    = x W_kva^T                      [N, d_c], [N, d_r]; c normed, k_pe rotated
    (k_nope, v)  = c W_kvb^T                      [N, H, d_n], [N, H, d_v]
    y            = (softmax(scale q . (k_nope | k_pe)) v) W_o^T

  * forward / backward: the expanded form on packed sequences, for training (frozen bf16 weights, as the
    rest of the layer: the backward returns dL/dx);
  * decode: the absorbed form over a paged cache of (c | k_pe) rows. k_nope's product moves to the
    query, q_nope W_k, and v's to the output, so a token costs d_c + d_r cached values instead of
    H (d_n + d_r + d_v). It takes d_c 128, 256, 384 or 512 (the expanded form is not bound to them).

The projections run on the library's tcgen05 GEMM (core.dense), the rest on core.latent_attention.
"""
from typing import Optional

import torch

from .. import _lib as L
from ..core import dense
from ..core import latent_attention as A


class LatentAttention:
    """W_q [H (d_n + d_r), d], W_kva [d_c + d_r, d], W_kvb [H, d_n + d_v, d_c], W_o [d, H d_v] (bf16, frozen);
    norm_w [d_c] or None; table fp32 [positions, d_r]: cosines, then sines."""

    def __init__(self, W_q: torch.Tensor, W_kva: torch.Tensor, W_kvb: torch.Tensor, W_o: torch.Tensor, table: torch.Tensor,
                 d_v: int, norm_w: Optional[torch.Tensor] = None, scale: Optional[float] = None, eps: float = 1e-5,
                 interleaved: bool = False):
        L.require_cuda(W_q, W_kva, W_kvb, W_o, table, norm_w)
        self.H, nv, self.d_c = W_kvb.shape
        self.d_v, self.d_n, self.d_r = d_v, nv - d_v, table.shape[1]
        self.d = W_q.shape[1]
        if tuple(W_q.shape) != (self.H * (self.d_n + self.d_r), self.d) or \
                tuple(W_kva.shape) != (self.d_c + self.d_r, self.d) or tuple(W_o.shape) != (self.d, self.H * d_v):
            raise ValueError("W_q [H (d_n + d_r), d], W_kva [d_c + d_r, d], W_kvb [H, d_n + d_v, d_c], W_o [d, H d_v]")
        bf = lambda t: t.to(torch.bfloat16).contiguous()  # noqa: E731
        self.W_q, self.W_kva, self.W_kvb, self.W_o = bf(W_q), bf(W_kva), bf(W_kvb), bf(W_o)
        self.W_k, self.W_v = self.W_kvb[:, :self.d_n], self.W_kvb[:, self.d_n:]        # views, per head
        self.norm_w = None if norm_w is None else norm_w.to(torch.float32).contiguous()
        self.table, self.eps, self.interleaved = table, float(eps), bool(interleaved)
        self.scale = float(scale) if scale is not None else (self.d_n + self.d_r) ** -0.5
        self.lib = L.load()
        self._saved = None

    def _norm(self, c: torch.Tensor):
        """(normed latent rows bf16, what the norm's backward needs)."""
        if self.norm_w is None:
            return c, None
        x = c.float().contiguous()
        y = torch.empty(c.shape, dtype=torch.bfloat16, device=c.device)
        rstd = torch.empty(c.shape[0], dtype=torch.float32, device=c.device)
        L.check(self.lib.ll_rmsnorm_forward(x.data_ptr(), self.norm_w.data_ptr(), x.shape[0], self.d_c, self.eps,
                                            y.data_ptr(), 1, rstd.data_ptr(), L.stream_ptr()), "ll_rmsnorm_forward")
        return y, (x, rstd)

    def forward(self, x: torch.Tensor, cu: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """y [N, d] bf16 for packed tokens x [N, d]; cu int32 [sequences + 1], positions int64 [N]."""
        L.require_cuda(x, cu, positions)
        xb = x.reshape(-1, self.d).to(torch.bfloat16).contiguous()
        N, H = xb.shape[0], self.H
        if N == 0:
            self._saved = ()
            return torch.empty((0, self.d), dtype=torch.bfloat16, device=x.device)
        q = dense.linear(xb, self.W_q).contiguous().view(N, H, self.d_n + self.d_r)
        A.rotate_positions(q[..., self.d_n:], positions, self.table, interleaved=self.interleaved, out=q[..., self.d_n:])
        kva = dense.linear(xb, self.W_kva)
        c, norm = self._norm(kva[:, :self.d_c])
        k_pe = A.rotate_positions(kva[:, None, self.d_c:], positions, self.table, interleaved=self.interleaved)[:, 0]
        kv = dense.linear(c, self.W_kvb.view(-1, self.d_c)).contiguous().view(N, H, -1)
        k_nope, v = kv[..., :self.d_n], kv[..., self.d_n:]
        out, lse = A.latent_attention_forward(q, k_nope, k_pe, v, cu, cu, self.scale)
        self._saved = (q, k_nope, k_pe, v, out, lse, norm, cu, positions)
        return dense.linear(out.view(N, -1), self.W_o).contiguous()

    def backward(self, g: torch.Tensor) -> torch.Tensor:
        """dL/dx [N, d] bf16 of the last forward."""
        if self._saved is None:
            raise RuntimeError("backward before forward")
        if not self._saved:                       # a forward without tokens
            return torch.empty_like(g.reshape(0, self.d), dtype=torch.bfloat16)
        q, k_nope, k_pe, v, out, lse, norm, cu, positions = self._saved
        N, H = q.shape[:2]
        g_out = dense.matmul(g.reshape(N, self.d).to(torch.bfloat16), self.W_o).contiguous().view(N, H, self.d_v)
        dq, dk, dk_pe, dv = A.latent_attention_backward(g_out, out, lse, q, k_nope, k_pe, v, cu, cu, self.scale)
        turn = dict(inverse=True, interleaved=self.interleaved)
        A.rotate_positions(dq[..., self.d_n:], positions, self.table, out=dq[..., self.d_n:], **turn)
        dk_pe = A.rotate_positions(dk_pe[:, None], positions, self.table, **turn)[:, 0]
        dc = dense.matmul(torch.cat([dk, dv], -1).view(N, -1), self.W_kvb.view(-1, self.d_c)).contiguous()
        if norm is not None:
            x32, rstd = norm
            gx = torch.empty_like(x32)
            L.check(self.lib.ll_rmsnorm_backward(x32.data_ptr(), self.norm_w.data_ptr(), rstd.data_ptr(), dc.data_ptr(), 1,
                                                 N, self.d_c, gx.data_ptr(), L.stream_ptr()), "ll_rmsnorm_backward")
            dc = gx.to(torch.bfloat16)
        return dense.matmul_sum2(dq.view(N, -1), self.W_q, torch.cat([dc, dk_pe], 1), self.W_kva).contiguous()

    def decode(self, x: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
               block_table: torch.Tensor, seq_lens: torch.Tensor) -> torch.Tensor:
        """y [B, Tq, d] for the last Tq tokens x [B, Tq, d] of B sequences, which are appended to the cache
        [pages, page_size, d_c + d_r] at slots [B Tq] first; seq_lens int32 [B] counts them in."""
        L.require_cuda(x, cache)
        if self.d_c not in (128, 256, 384, 512):  # (before anything is written to the cache)
            raise ValueError("decode: d_c 128, 256, 384 or 512")
        B, Tq, _ = x.shape
        N, H = B * Tq, self.H
        xb = x.reshape(N, self.d).to(torch.bfloat16).contiguous()
        if N == 0:
            return torch.empty((B, Tq, self.d), dtype=torch.bfloat16, device=x.device)
        q = dense.linear(xb, self.W_q).contiguous().view(N, H, self.d_n + self.d_r)
        kva = dense.linear(xb, self.W_kva)
        if self.norm_w is not None:
            kva[:, :self.d_c] = self._norm(kva[:, :self.d_c])[0]
        q_lat = torch.empty((N, H, self.d_c + self.d_r), dtype=torch.bfloat16, device=x.device)
        A.head_linear(q[..., :self.d_n], self.W_k, w_nk=False, out=q_lat[..., :self.d_c])
        A.append_latent(cache, kva, slots, positions, self.table, q[..., self.d_n:], q_lat[..., self.d_c:],
                        interleaved=self.interleaved)
        o, _ = A.paged_latent_attention(q_lat.view(B, Tq, H, -1), cache, block_table, seq_lens, self.d_c, self.scale)
        o = A.head_linear(o.view(N, H, self.d_c), self.W_v)
        return dense.linear(o.view(N, -1), self.W_o).contiguous().view(B, Tq, self.d)
