"""
The latent-attention layer (trainer.latent_attention.LatentAttention): forward and input gradient against
the same layer in 64 bits with autograd, and decoding through the paged cache against the forward.

Tolerance: each of the layer's bf16 tensors is rounded once (2^-8 of a value at most, 2^-9 / sqrt(3) = 1.1e-3
rms); a forward has at most seven such tensors between x and y and a backward nine, so the relative L2 error
stays within sqrt(16) * 1.1e-3 = 4.5e-3 rms; 1e-2 leaves a factor of two.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TOL = 1e-2


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _layer(g, H, d, d_c, d_r, d_n, d_v, norm, interleaved):
    from lazylora_b200.trainer.latent_attention import LatentAttention
    w = lambda o, i: (torch.randn(o, i, generator=g, device="cuda") * i ** -0.5).to(torch.bfloat16)  # noqa: E731
    inv = 10000.0 ** (-torch.arange(0, d_r, 2, device="cuda", dtype=torch.float64) / d_r)
    ang = torch.arange(400, device="cuda", dtype=torch.float64)[:, None] * inv
    table = torch.cat([ang.cos(), ang.sin()], 1).float()
    W = dict(W_q=w(H * (d_n + d_r), d), W_kva=w(d_c + d_r, d), W_kvb=w(H * (d_n + d_v), d_c).view(H, d_n + d_v, d_c),
             W_o=w(d, H * d_v))
    norm_w = 1 + 0.1 * torch.randn(d_c, generator=g, device="cuda") if norm else None
    return LatentAttention(**W, table=table, d_v=d_v, norm_w=norm_w, interleaved=interleaved), W, table, norm_w


def _exact(x, W, table, norm_w, lens, pos, H, d_c, d_n, d_r, interleaved):
    W = {k: t.double() for k, t in W.items()}
    cs = table.double()[pos]
    c, s = cs[:, :d_r // 2], cs[:, d_r // 2:]

    def turn(t):
        cc, ss = (c, s) if t.dim() == 2 else (c[:, None], s[:, None])
        a, b = (t[..., ::2], t[..., 1::2]) if interleaved else (t[..., :d_r // 2], t[..., d_r // 2:])
        u, v = a * cc - b * ss, a * ss + b * cc
        return torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)

    N = x.shape[0]
    q = (x @ W["W_q"].T).view(N, H, -1)
    q = torch.cat([q[..., :d_n], turn(q[..., d_n:])], -1)
    kva = x @ W["W_kva"].T
    lat = kva[:, :d_c]
    if norm_w is not None:
        lat = lat * torch.rsqrt(lat.pow(2).mean(1, keepdim=True) + 1e-5) * norm_w.double()
    kv = torch.einsum("nc,hkc->nhk", lat, W["W_kvb"])
    k = torch.cat([kv[..., :d_n], turn(kva[:, d_c:])[:, None].expand(-1, H, -1)], -1)
    outs, at = [], 0
    for n in lens:
        a = slice(at, at + n)
        at += n
        sc = torch.einsum("ihd,jhd->hij", q[a], k[a]) / math.sqrt(d_n + d_r)
        sc = sc.masked_fill(~torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), -math.inf)
        outs.append(torch.einsum("hij,jhd->ihd", torch.softmax(sc, -1), kv[a][..., d_n:]))
    return torch.cat(outs).reshape(N, -1) @ W["W_o"].T


@pytest.mark.parametrize("norm,interleaved", [(True, False), (False, True)])
def test_layer_against_64_bits(norm, interleaved):
    g = torch.Generator(device="cuda").manual_seed(5)
    H, d, d_c, d_r, d_n, d_v, lens = 6, 256, 256, 64, 128, 128, [150, 1, 77]
    layer, W, table, norm_w = _layer(g, H, d, d_c, d_r, d_n, d_v, norm, interleaved)
    N = sum(lens)
    x = torch.randn(N, d, generator=g, device="cuda").to(torch.bfloat16)
    go = torch.randn(N, d, generator=g, device="cuda").to(torch.bfloat16)
    cu = torch.tensor([0, 150, 151, 228], dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(n, device="cuda") for n in lens])
    y = layer.forward(x, cu, pos)
    dx = layer.backward(go)
    xr = x.double().requires_grad_()
    want = _exact(xr, W, table, norm_w, lens, pos, H, d_c, d_n, d_r, interleaved)
    want.backward(go.double())
    assert _rel(y, want.detach()) < TOL
    assert _rel(dx, xr.grad) < TOL


@pytest.mark.parametrize("Tq", [1, 3])
def test_decode_matches_forward(Tq):
    """Tokens decoded Tq at a time through the cache against the packed forward of the same tokens."""
    from lazylora_b200.core import latent_attention as A
    g = torch.Generator(device="cuda").manual_seed(6)
    H, d, d_c, d_r, d_n, d_v = 5, 192, 256, 64, 64, 128
    layer, *_ = _layer(g, H, d, d_c, d_r, d_n, d_v, True, False)
    B, n, page = 2, 24, 8
    x = torch.randn(B, n, d, generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.arange(n, device="cuda")
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
    want = layer.forward(x.view(-1, d), cu, pos.repeat(B)).view(B, n, d)
    cache = torch.full((8, page, d_c + d_r), float("nan"), dtype=torch.bfloat16, device="cuda")
    bt = torch.tensor([[5, 0, 3], [1, 7, 2]], dtype=torch.int32, device="cuda")
    got = []
    for t in range(0, n, Tq):
        p = pos[t:t + Tq]
        slots = (bt[:, (p // page)].long() * page + p % page).reshape(-1)
        sl = torch.full((B,), t + Tq, dtype=torch.int32, device="cuda")
        got.append(layer.decode(x[:, t:t + Tq], cache, slots, p.repeat(B), bt, sl))
    assert _rel(torch.cat(got, 1), want) < TOL
    A.check_status()
