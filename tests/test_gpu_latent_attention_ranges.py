"""
The latent-attention operators at the ends of their ranges: lengths and pages that only the device can see
to be wrong, gradients past fp16's range, empty batches. Each is recorded or computed, never passed over.
"""
import math

import pytest
import torch

from test_gpu_latent_attention import BF, HF, U, _check_paged, _expand_case, _gen, _paged_case, _rand, _within

pytestmark = pytest.mark.gpu


def _raises_once():
    from lazylora_b200 import _lib as L
    from lazylora_b200.core import latent_attention as A
    with pytest.raises(L.LLError, match="out of range"):
        A.check_status()
    A.check_status()


# ---------------------------------------------------------------------------------------------- paged
@pytest.mark.parametrize("at,n", [(0, 33), (1, 1000), (2, -1), (0, 2 ** 31 - 1), (1, -2 ** 31)])
def test_paged_reports_lengths_outside_the_block_table(at, n):
    """Four pages of eight rows hold 32 keys; one length is past them or negative. The other sequences'
    outputs are those of the call without it."""
    from lazylora_b200.core import latent_attention as A
    q, cache, bt, sl, rows = _paged_case(BF, [20, 24, 9], 1, 4, 128, 64, 8, 2, garbage=0.0)
    bt = bt.clamp(0, cache.shape[0] - 1)
    assert bt.shape[1] == 4
    out, lse = A.paged_latent_attention(q, cache, bt, sl, 128, 0.1)
    A.check_status()
    sl[at] = n
    got, got_lse = A.paged_latent_attention(q, cache, bt, sl, 128, 0.1)
    _raises_once()
    others = [b for b in range(3) if b != at]
    assert torch.equal(got[others], out[others]) and torch.equal(got_lse[others], lse[others])


def test_paged_lengths_that_fill_the_block_table_are_fine():
    from lazylora_b200.core import latent_attention as A
    q, cache, bt, sl, rows = _paged_case(BF, [32, 0, 31], 2, 4, 128, 64, 8, 3)
    out, lse = A.paged_latent_attention(q, cache, bt[:, :4].contiguous(), sl, 128, 0.1)
    A.check_status()
    _check_paged(out, lse, q, rows, 128, 0.1)


@pytest.mark.parametrize("page", [-1, 10 ** 6])
def test_paged_page_out_of_range_reads_zeros(page):
    """A page outside the cache is recorded, and its keys are rows of zeros (scores of 0, values of 0)."""
    from lazylora_b200.core import latent_attention as A
    q, cache, bt, sl, rows = _paged_case(BF, [30, 90], 1, 4, 128, 64, 8, 4)
    bt[1, 3] = page
    rows[1][24:32] = 0
    out, lse = A.paged_latent_attention(q, cache, bt, sl, 128, 0.1)
    _raises_once()
    _check_paged(out, lse, q, rows, 128, 0.1)


# ------------------------------------------------------------------------------------------- expanded
@pytest.mark.parametrize("which", ["cu_q", "cu_k"])
@pytest.mark.parametrize("cu", [[1, 70, 100], [0, 70, 99], [0, 70, 101], [0, 101, 100], [0, -1, 100], [-5, 70, 100]])
def test_expanded_reports_cumulative_lengths_that_do_not_cover_the_rows(which, cu):
    """100 rows in two sequences: cumulative lengths that start past 0, fall, or end elsewhere are recorded
    by the forward and by the backward."""
    from lazylora_b200.core import latent_attention as A
    q, kn, kp, v, cq, ck, go = _expand_case(BF, [70, 30], [70, 30], 2, 128, 64, 128, 1)
    out, lse = A.latent_attention_forward(q, kn, kp, v, cq, ck, 0.1)
    A.latent_attention_backward(go, out, lse, q, kn, kp, v, cq, ck, 0.1)
    A.check_status()
    bad = torch.tensor(cu, dtype=torch.int32, device="cuda")
    cq, ck = (bad, ck) if which == "cu_q" else (cq, bad)
    A.latent_attention_forward(q, kn, kp, v, cq, ck, 0.1)
    _raises_once()
    A.latent_attention_backward(go, out, lse, q, kn, kp, v, cq, ck, 0.1)
    _raises_once()


def test_expanded_backward_reports_cumulative_lengths_without_queries():
    """No query rows at all: the gradients of the keys are zeros, and bad lengths of theirs are recorded too."""
    from lazylora_b200.core import latent_attention as A
    q, kn, kp, v, cq, ck, go = _expand_case(BF, [0, 0], [40, 30], 2, 128, 64, 128, 1)
    lse = torch.zeros(2, 0, device="cuda")
    d = A.latent_attention_backward(go, go, lse, q, kn, kp, v, cq, ck, 0.1)
    A.check_status()
    assert all(bool((t == 0).all()) for t in d[1:])
    ck[2] = 69
    A.latent_attention_backward(go, go, lse, q, kn, kp, v, cq, ck, 0.1)
    _raises_once()


def test_expanded_refuses_rows_without_sequences():
    from lazylora_b200.core import latent_attention as A
    z = lambda *s: torch.zeros(*s, dtype=BF, device="cuda")  # noqa: E731
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    for tq, tk in ((4, 4), (4, 0), (0, 4)):
        x = (z(tq, 2, 192), z(tk, 2, 128), z(tk, 64), z(tk, 2, 128), none, none, 0.1)
        with pytest.raises(ValueError):
            A.latent_attention_forward(*x)
        with pytest.raises(ValueError):
            A.latent_attention_backward(z(tq, 2, 128), z(tq, 2, 128), torch.zeros(2, tq, device="cuda"), *x)


def _wide(seed, ql, kl, grow):
    """fp16 operands whose P (dP - delta) passes 65504 while the gradients, which carry the scale and small
    queries and keys, do not: |g| about 4000 and |v| about 32, or |g| about 1500, both growing along the rows
    (later steps raise the largest value again); |q| and |k| about 1/256; every third query's gradient is
    a thousandth of that."""
    gen, H = torch.Generator().manual_seed(seed), 2
    new = lambda n, std, *s: torch.randn(n, *s, generator=gen) * std  # noqa: E731
    up = lambda n: 1 + torch.arange(n)[:, None, None] / 40 if grow else 1.0  # noqa: E731
    n, m = sum(ql), sum(kl)
    small = torch.where(torch.arange(n) % 3 == 1, 1e-3, 1.0)[:, None, None]
    q, k = new(n, 1 / 256, H, 192), new(m, 1 / 256, H, 128)
    go = new(n, 1500 if grow else 4000, H, 128) * up(n) * small
    x = (q, k, new(m, 1 / 256, 64), new(m, 32, H, 128) * up(m), go)
    q, kn, kp, v, go = (t.to("cuda", HF) for t in x)
    cum = lambda ls: torch.tensor([sum(ls[:i]) for i in range(len(ls) + 1)], dtype=torch.int32, device="cuda")  # noqa: E731
    return q, kn, kp, v, cum(ql), cum(kl), go


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("ql,kl,grow", [([40, 3], [40, 3], False), ([300, 70], [300, 70], True), ([65], [400], True)])
def test_fp16_gradients_whose_unscaled_scores_pass_the_type(ql, kl, grow, causal):
    """The formula's gradients are finite in fp16 although P (dP - delta), before the scale and the sums,
    is not. Bound: as derived for ordinary values (dS and P rounded to the type, fp32 scores and sums), where
    dS is held times a power of two f of its row that brings the row's largest value m to 2^14 .. 2^15
    when it passes the type: what falls below the type's smallest step is at most 2^-25 / f <= m 2^-39 in
    dS, twice that beside 2^-24 for the rows that need no factor. The fp32 sums of dP and delta, whose terms
    cancel where they are large, are off by at most 2^-20 of the sums of their terms' sizes (8 additions of
    2^-23 each)."""
    from lazylora_b200.core import latent_attention as A
    q, kn, kp, v, cq, ck, go = _wide(7, ql, kl, grow)
    scale, u = 192 ** -0.5, U[HF]
    out, lse = A.latent_attention_forward(q, kn, kp, v, cq, ck, scale, causal=causal)
    dq, dkn, dkp, dv = A.latent_attention_backward(go, out, lse, q, kn, kp, v, cq, ck, scale, causal=causal)
    A.check_status()
    k = torch.cat([kn, kp[:, None].expand(-1, 2, -1)], -1)
    Q, K, V, G, O = (t.double().transpose(0, 1) for t in (q, k, v, go, out))
    want = {n: torch.zeros_like(t) for n, t in (("q", Q), ("k", K), ("v", V))}
    bound = {n: torch.zeros_like(t) for n, t in want.items()}
    largest, q0, k0 = 0.0, 0, 0
    for n, m in zip(ql, kl):
        a, b = slice(q0, q0 + n), slice(k0, k0 + m)
        q0, k0 = q0 + n, k0 + m
        seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
        seen = seen.tril(m - n) if causal else seen
        s = (Q[:, a] @ K[:, b].transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
        p = torch.softmax(s, -1)
        dp, delta = G[:, a] @ V[:, b].transpose(1, 2), (G[:, a] * O[:, a]).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        largest = max(largest, float(ds.abs().max()))
        terms = G[:, a].abs() @ V[:, b].abs().transpose(1, 2) + (G[:, a] * O[:, a]).abs().sum(-1, keepdim=True)
        size = p * ((u + 1e-4) * (dp.abs() + delta.abs()) + 2.0 ** -20 * terms)
        tiny = lambda d: (2.0 ** -24 + ds.abs().amax(d, keepdim=True) * 2.0 ** -38) * seen  # noqa: E731
        for name, at, x, e, y in (("q", a, ds, size + tiny(2), K[:, b]),
                                  ("k", b, ds.transpose(1, 2), (size + tiny(1)).transpose(1, 2), Q[:, a])):
            w = x @ y * scale
            want[name][:, at] = w
            bound[name][:, at] = u * w.abs() + scale * (e @ y.abs()) + 2.0 ** -24
        w = p.transpose(1, 2) @ G[:, a]
        want["v"][:, b] = w
        bound["v"][:, b] = u * w.abs() + ((u + 1e-4) * p + 2.0 ** -24 * seen).transpose(1, 2) @ G[:, a].abs() + 2.0 ** -24
    assert largest > 65504, "the case is about values past the type"
    w, e = want["k"].transpose(0, 1), bound["k"].transpose(0, 1)
    kpe = w[..., 128:].sum(1)
    for got, x, y in ((dq, want["q"].transpose(0, 1), bound["q"].transpose(0, 1)),
                      (dv, want["v"].transpose(0, 1), bound["v"].transpose(0, 1)), (dkn, w[..., :128], e[..., :128]),
                      (dkp, kpe, e[..., 128:].sum(1) + u * kpe.abs())):
        assert float(x.abs().max()) < 65504, "and gradients within it"
        _within(got, x, y)


def test_fp16_gradient_of_one_bad_row_stays_in_it():
    """An infinite gradient in one query row leaves the other rows' dq as they are without it."""
    from lazylora_b200.core import latent_attention as A
    q, kn, kp, v, cq, ck, go = _expand_case(HF, [200], [200], 2, 128, 64, 128, 11)
    out, lse = A.latent_attention_forward(q, kn, kp, v, cq, ck, 0.07)
    want = A.latent_attention_backward(go, out, lse, q, kn, kp, v, cq, ck, 0.07)[0]
    go[37] = float("inf")
    got = A.latent_attention_backward(go, out, lse, q, kn, kp, v, cq, ck, 0.07)[0]
    keep = torch.arange(200, device="cuda") != 37
    assert torch.equal(got[keep], want[keep])


# ------------------------------------------------------------------------------------------------ layer
def test_layer_without_tokens():
    from test_gpu_latent_attention_layer import _layer
    layer, *_ = _layer(_gen(1), 2, 128, 128, 64, 64, 64, True, False)
    x = torch.zeros(0, 128, dtype=BF, device="cuda")
    cu, pos = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    assert layer.forward(x, cu, pos).shape == (0, 128)
    dx = layer.backward(x)
    assert dx.shape == (0, 128) and dx.dtype is BF
    # and with tokens again afterwards, and none after those
    x = _rand(_gen(2), BF, 5, 128)
    cu, pos = torch.tensor([0, 5], dtype=torch.int32, device="cuda"), torch.arange(5, device="cuda")
    layer.forward(x, cu, pos)
    assert layer.backward(x).shape == (5, 128)
    layer.forward(x[:0], cu[:1], pos[:0])
    assert layer.backward(x[:0]).shape == (0, 128)


def test_layer_decode_refuses_other_latents_before_it_writes():
    """A latent of 192 values trains; decode, whose absorbed form does not take it, leaves the cache alone."""
    from test_gpu_latent_attention_layer import _layer
    layer, *_ = _layer(_gen(3), 2, 128, 192, 64, 64, 64, False, False)
    x = _rand(_gen(4), BF, 5, 128)
    cu, pos = torch.tensor([0, 5], dtype=torch.int32, device="cuda"), torch.arange(5, device="cuda")
    assert layer.forward(x, cu, pos).shape == layer.backward(x).shape == (5, 128)
    cache = torch.full((2, 8, 256), 7.0, dtype=BF, device="cuda")
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        layer.decode(x[:1, None], cache, pos[:1], pos[:1], one[:, None], one)
    assert bool((cache == 7.0).all())


# ------------------------------------------------------------------------------------------ large scores
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_of_large_magnitude(dt, sign):
    """Scores of 2^25 to 2^26, each one exact product, so far apart that a row's largest ones (2 or 46 equal
    ones) share its softmax: out is the mean of their values (the shares carry one common factor and are
    rounded to the type: u, and the output once more), lse their score plus the log of their number (fp32 of
    that size: 2^-22 relative)."""
    from lazylora_b200.core import latent_attention as A
    n, H, scale = 300, 3, 0.5
    g = _gen(12)
    steps = 1 + (torch.arange(n, device="cuda") % 150).clamp_max(127) / 128
    key = (sign * 16384 * steps).to(dt)
    assert bool((key.double() == sign * 16384 * steps.double()).all())
    score = key.double() * 4096 * scale
    top = (score == score.max()).double()
    top /= top.sum()
    lse_want = score.max() - torch.log(top.max())
    # absorbed
    rows = _rand(g, dt, n, 192)
    rows[:, 0] = key
    q = torch.zeros(1, 1, H, 192, dtype=dt, device="cuda")
    q[..., 0] = 4096
    pages = (n + 7) // 8
    cache = torch.zeros(pages, 8, 192, dtype=dt, device="cuda")
    cache.view(-1, 192)[:n] = rows
    bt = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    out, lse = A.paged_latent_attention(q, cache, bt, torch.tensor([n], dtype=torch.int32, device="cuda"), 128, scale)
    want = (top @ rows[:, :128].double()).expand(1, 1, H, 128)
    _within(out, want, 2 * U[dt] * (top @ rows[:, :128].double().abs()))
    _within(lse, lse_want.expand(1, 1, H), lse_want.abs() * 2.0 ** -22)
    # expanded: as many queries as there are row tiles for, not causal
    k, v = _rand(g, dt, n, H, 128), _rand(g, dt, n, H, 128)
    k[..., 0] = key[:, None]
    qe = torch.zeros(260, H, 128, dtype=dt, device="cuda")
    qe[..., 0] = 4096
    cq, ck = (torch.tensor([0, m], dtype=torch.int32, device="cuda") for m in (260, n))
    out, lse = A.latent_attention_forward(qe, k, None, v, cq, ck, scale, causal=False)
    want = torch.einsum("j,jhd->hd", top, v.double()).expand(260, H, 128)
    _within(out, want, 2 * U[dt] * torch.einsum("j,jhd->hd", top, v.double().abs()))
    _within(lse, lse_want.expand(H, 260), lse_want.abs() * 2.0 ** -22)
    A.check_status()
