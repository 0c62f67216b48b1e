"""
The latent-attention operators against plain implementations in 64 bits on the same 16-bit inputs.

Tolerances, from the kernels' roundings (u: half a unit in the last place of the type, 2^-8 for bf16,
2^-11 for fp16):
  * outputs: P is rounded to the type (u P relative, and in fp16 at most 2^-25 absolute below the normal
    range), products are exact and summed in fp32, the result is rounded once (u relative). The scores are
    fp32 sums of at most 576 products, the tensor cores adding 16 at a time: 36 additions of relative error
    2^-23 on sums of about 10 give 5e-5 absolute in a score, 1e-4 relative in a P with the exponential's
    own error. So |out - exact| <= u |out| + sum_j P_j |v_j| (u + 1e-4) + tiny sum_j |v_j|.
  * lse: 1e-4 absolute by the same count.
  * gradients: |dS| <= P (|dP| + |delta|), each of its parts within 1e-4, dS and P rounded (u); the bound
    is the sum of these over the products that make up the gradient, plus one rounding.
  * the append's rotation: fp32 products and one rounding: u + 2^-22 relative to |a| + |b|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24}
BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(g, dt, *shape):
    return torch.randn(*shape, generator=g, device="cuda").to(dt)


def _within(got, want, bound):
    err = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all()) and bool((err <= bound).all()), \
        f"worst {float((err - bound).max()):.3e} over the bound, error {float(err.max()):.3e}"


# ------------------------------------------------------------------------------------ append, rotate
def _table(n, d_r):
    inv = 10000.0 ** (-torch.arange(0, d_r, 2, device="cuda", dtype=torch.float64) / d_r)
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def _turn(x, pos, table, interleaved, inverse=False):
    """(turned, |a| + |b| of each value's pair) in 64 bits; x [T, ..., d_r]."""
    h = x.shape[-1] // 2
    cs = table[pos].double()
    shape = (x.shape[0],) + (1,) * (x.dim() - 2) + (h,)
    c, s = cs[:, :h].reshape(shape), cs[:, h:].reshape(shape) * (-1 if inverse else 1)
    x = x.double()
    a, b = (x[..., ::2], x[..., 1::2]) if interleaved else (x[..., :h], x[..., h:])
    join = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if interleaved else (lambda u, v: torch.cat([u, v], -1))
    return join(a * c - b * s, a * s + b * c), join(a.abs() + b.abs(), a.abs() + b.abs())


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("T,H,d_c,d_r,page,interleaved", [(1, 1, 128, 64, 8, False), (37, 5, 512, 64, 24, True),
                                                         (130, 64, 256, 32, 48, False), (3, 0, 144, 16, 1, True), (9, 7, 128, 16, 8, False),
                                                         (5, 3, 128, 48, 8, True)])
def test_append(dt, T, H, d_c, d_r, page, interleaved):
    from lazylora_b200.core import latent_attention as A
    g = _gen(T + H)
    D, pages = d_c + d_r, T // page + 3
    cache = _rand(g, dt, pages, page, D + 8)[:, :, :D]             # rows with a gap behind them
    kv = _rand(g, dt, T, D + 16)[:, :D]                            # and strided tokens
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T]
    if T > 2:
        slots[1] = -1
    pos = torch.randint(0, 500, (T,), generator=g, device="cuda")
    table = _table(500, d_r)
    before = cache.clone()
    buf = torch.full((T, max(H, 1), d_c + d_r), 7.0, dtype=dt, device="cuda")
    q = _rand(g, dt, T, H, d_r + 8)[..., 8:] if H else None
    out = A.append_latent(cache, kv, slots, pos, table, q, buf[..., d_c:] if H else None, interleaved=interleaved)
    want = before.double().reshape(-1, D)
    bound = torch.zeros_like(want)
    on = (slots >= 0).nonzero()[:, 0]
    turned, size = _turn(kv[:, d_c:], pos, table, interleaved)
    want[slots[on]] = torch.cat([kv[:, :d_c].double(), turned], 1)[on]
    bound[slots[on], d_c:] = (turned.abs() * U[dt] + size * 2.0 ** -22 + TINY[dt])[on]
    _within(cache, want.view(pages, page, D), bound.view(pages, page, D))
    if H:
        turned, size = _turn(q, pos, table, interleaved)
        _within(out, turned, turned.abs() * U[dt] + size * 2.0 ** -22 + TINY[dt])
        assert bool((buf[..., :d_c] == 7.0).all()), "nothing beside the slice is written"
    else:
        assert out is None
    A.check_status()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotate_and_back_in_place(interleaved):
    from lazylora_b200.core import latent_attention as A
    g = _gen(5)
    x = _rand(g, BF, 50, 3, 192)
    keep = x.clone()
    pos, table = torch.randint(0, 99, (50,), generator=g, device="cuda"), _table(99, 64)
    y = A.rotate_positions(x[..., 128:], pos, table, interleaved=interleaved, out=x[..., 128:])
    assert y.data_ptr() == x[..., 128:].data_ptr() and torch.equal(x[..., :128], keep[..., :128])
    want, size = _turn(keep[..., 128:], pos, table, interleaved)
    _within(y, want, want.abs() * U[BF] + size * 2.0 ** -22)
    back = A.rotate_positions(y, pos, table, inverse=True, interleaved=interleaved)
    want, size = _turn(y, pos, table, interleaved, inverse=True)
    _within(back, want, want.abs() * U[BF] + size * 2.0 ** -22)


def test_append_reports_what_is_out_of_range():
    from lazylora_b200 import _lib as L
    from lazylora_b200.core import latent_attention as A
    g = _gen(6)
    cache = _rand(g, BF, 4, 8, 192)
    before = cache.clone()
    kv, table = _rand(g, BF, 2, 192), _table(10, 64)
    slots = torch.tensor([32, 3], device="cuda")                   # one past the cache; a good one
    A.append_latent(cache, kv, slots, torch.tensor([1, 2], device="cuda"), table)
    with pytest.raises(L.LLError):
        A.check_status()
    A.check_status()                                                # reported once
    assert torch.equal(cache.view(32, 192)[torch.arange(32, device="cuda") != 3],
                       before.view(32, 192)[torch.arange(32, device="cuda") != 3])
    A.append_latent(cache, kv, torch.tensor([1, 2], device="cuda"), torch.tensor([10, -1], device="cuda"), table)
    with pytest.raises(L.LLError):
        A.check_status()
    assert torch.equal(cache.view(32, 192)[1:3], before.view(32, 192)[1:3]), "a bad position writes nothing"


# ---------------------------------------------------------------------------------------------- paged
def _paged_case(dt, lens, Tq, H, d_c, d_r, page, seed, garbage=float("nan")):
    g = _gen(seed)
    D, need = d_c + d_r, [(n + page - 1) // page for n in lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    bt = torch.full((len(lens), max(1, max(need)) + 1), -7, dtype=torch.int32, device="cuda")
    cache = torch.full((pages, page, D), garbage, dtype=dt, device="cuda")
    rows, at = [], 0
    for b, n in enumerate(lens):
        bt[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        r = _rand(g, dt, n, D)
        rows.append(r)
        for i in range(need[b]):
            piece = r[i * page:(i + 1) * page]
            cache[int(bt[b, i]), :len(piece)] = piece
    q = _rand(g, dt, len(lens), Tq, H, D)
    return q, cache, bt, torch.tensor(lens, dtype=torch.int32, device="cuda"), rows


def _check_paged(out, lse, q, rows, d_c, scale):
    dt = q.dtype
    B, Tq, H, _ = q.shape
    for b in range(B):
        n = rows[b].shape[0]
        for t in range(Tq):
            m = n - Tq + t + 1
            if m <= 0:
                assert bool((out[b, t] == 0).all()) and bool((lse[b, t] == -math.inf).all())
                continue
            k = rows[b][:m].double()
            s = q[b, t].double() @ k.T * scale
            want_l = torch.logsumexp(s, -1)
            p = torch.exp(s - want_l[:, None])
            v = k[:, :d_c]
            want = p @ v
            _within(lse[b, t], want_l, 1e-4)
            _within(out[b, t], want, U[dt] * want.abs() + (U[dt] + 1e-4) * (p @ v.abs()) + TINY[dt] * v.abs().sum(0))


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("lens,Tq,H,d_c,d_r,page", [
    ([1], 1, 1, 512, 64, 8),
    ([0, 1, 7, 8, 63, 64, 65, 129], 1, 5, 512, 64, 24),           # ends inside a tile, a page, a box
    ([700, 0, 2], 1, 64, 512, 0, 64),
    ([200, 1, 3, 65, 2], 3, 40, 512, 64, 16),                     # queries that see nothing, rows split 64 + 56
    ([90, 300], 2, 128, 256, 64, 48),                             # 256 rows: four row tiles
    ([130], 1, 20, 384, 64, 128), ([64] * 70, 1, 16, 128, 64, 8),
    ([5000], 1, 33, 512, 64, 32),                                 # split over many CTAs
    ([1500] * 3 + [1] * 200, 1, 10, 128, 0, 8),                   # many sequences a CTA
    ([40], 70, 64, 128, 64, 8),                                   # more row tiles than SMs would split, most rows empty
])
def test_paged(dt, lens, Tq, H, d_c, d_r, page):
    from lazylora_b200.core import latent_attention as A
    q, cache, bt, sl, rows = _paged_case(dt, lens, Tq, H, d_c, d_r, page, len(lens) * 31 + H)
    scale = 1 / math.sqrt(d_c / 4 + d_r)
    out, lse = A.paged_latent_attention(q, cache, bt, sl, d_c, scale)
    _check_paged(out, lse, q, rows, d_c, scale)
    again = A.paged_latent_attention(q, cache, bt, sl, d_c, scale)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    A.check_status()


def test_paged_large_scores_move_the_reference():
    """Scores that grow along the keys by far more than the slack, and some very negative ones."""
    from lazylora_b200.core import latent_attention as A
    q, cache, bt, sl, rows = _paged_case(BF, [1000, 300], 1, 20, 256, 64, 16, 3)
    grow = torch.linspace(-30, 30, 1000, device="cuda")
    for b, n in enumerate((1000, 300)):
        rows[b][:, 0] = grow[:n].to(BF)
        for i in range((n + 15) // 16):
            piece = rows[b][i * 16:(i + 1) * 16]
            cache[int(bt[b, i]), :len(piece)] = piece
    q[..., 0] = 40.0
    q[0, 0, 3, 0] = -40.0
    out, lse = A.paged_latent_attention(q, cache, bt, sl, 256, 0.1)
    # scores reach 120 here: their fp32 sums carry 36 * 2^-23 * 120 = 5e-4, so the bounds are ten times wider
    for b in range(2):
        k = rows[b].double()
        s = q[b, 0].double() @ k.T * 0.1
        want_l = torch.logsumexp(s, -1)
        p = torch.exp(s - want_l[:, None])
        want, size = p @ k[:, :256], p @ k[:, :256].abs()
        _within(lse[b, 0], want_l, 1e-3)
        _within(out[b, 0], want, U[BF] * want.abs() + (U[BF] + 1e-3) * size)


def test_paged_strides_stream_and_far_pages():
    """A strided query, a cache of more than 2^32 bytes used at its end, another stream than the default."""
    from lazylora_b200.core import latent_attention as A
    g = _gen(9)
    pages, page, D = 62000, 64, 576                                # 4.57e9 bytes
    cache = torch.empty((pages, page, D), dtype=BF, device="cuda")
    rows = _rand(g, BF, 100, D)
    bt = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    cache[pages - 1] = rows[:64]
    cache[pages - 3, :36] = rows[64:]
    cache[pages - 3, 36:] = float("inf")
    wide = _rand(g, BF, 1, 2, 24, D + 40)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out, lse = A.paged_latent_attention(wide[..., :D], cache, bt, torch.tensor([100], dtype=torch.int32, device="cuda"),
                                            512, 0.07)
    torch.cuda.current_stream().wait_stream(s)
    _check_paged(out, lse, wide[..., :D], [rows], 512, 0.07)


def test_paged_graph_replay_with_other_lengths():
    from lazylora_b200.core import latent_attention as A
    q, cache, bt, sl, rows = _paged_case(BF, [400, 90, 33], 1, 12, 128, 64, 8, 12)
    A.paged_latent_attention(q, cache, bt, sl, 128, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = A.paged_latent_attention(q, cache, bt, sl, 128, 0.1)
    for lens in ([400, 90, 33], [17, 0, 33], [1, 64, 8]):
        sl.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        _check_paged(out, lse, q, [r[:n] for r, n in zip(rows, lens)], 128, 0.1)


def test_paged_reports_a_page_out_of_range():
    from lazylora_b200 import _lib as L
    from lazylora_b200.core import latent_attention as A
    q, cache, bt, sl, _ = _paged_case(BF, [30], 1, 4, 128, 64, 8, 1)
    bt[0, 2] = cache.shape[0]
    A.paged_latent_attention(q, cache, bt, sl, 128, 0.1)
    with pytest.raises(L.LLError):
        A.check_status()


# ------------------------------------------------------------------------------------------- expanded
def _expand_case(dt, ql, kl, H, d_n, d_r, d_v, seed):
    g = _gen(seed)
    cum = lambda ls: torch.tensor([sum(ls[:i]) for i in range(len(ls) + 1)], dtype=torch.int32, device="cuda")  # noqa: E731
    q = _rand(g, dt, sum(ql), H, d_n + d_r)
    kv = _rand(g, dt, sum(kl), H, d_n + d_v)
    k_pe = _rand(g, dt, sum(kl), d_r + 8)[:, :d_r] if d_r else None
    go = _rand(g, dt, sum(ql), H, d_v)
    return q, kv[..., :d_n], k_pe, kv[..., d_n:], cum(ql), cum(kl), go


def _expand_exact(q, kn, kp, v, go, out, ql, kl, scale, causal):
    """The definitions in 64 bits (gradients with delta from `out` as stored) and the bounds."""
    dt, H = q.dtype, q.shape[1]
    u, tiny = U[dt], TINY[dt]
    k = kn if kp is None else torch.cat([kn, kp[:, None].expand(-1, H, -1)], -1)
    q, k, v, go, o = (t.double().transpose(0, 1) for t in (q, k, v, go, out))       # [H, T, d]
    new = lambda t: torch.zeros_like(t)  # noqa: E731
    r = {n: (new(t), new(t)) for n, t in (("out", o), ("dq", q), ("dk", k), ("dv", v))}
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for n, m in zip(ql, kl):
        a, b = slice(q0, q0 + n), slice(k0, k0 + m)
        q0, k0 = q0 + n, k0 + m
        if n == 0 or m == 0:
            continue
        seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
        if causal:
            seen = seen.tril(m - n)
        s = (q[:, a] @ k[:, b].transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
        L = torch.logsumexp(s, -1)
        lse[:, a] = L
        p = torch.exp(s - L.masked_fill(L == -math.inf, 0.0)[..., None])
        want = p @ v[:, b]
        r["out"][0][:, a] = want
        r["out"][1][:, a] = u * want.abs() + (u + 1e-4) * (p @ v[:, b].abs()) + tiny * v[:, b].abs().sum(1, keepdim=True)
        dp, delta = go[:, a] @ v[:, b].transpose(1, 2), (go[:, a] * o[:, a]).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        size = (u + 1e-4) * p * (dp.abs() + delta.abs()) + tiny * seen
        for name, at, x, y in (("dq", a, ds, k[:, b]), ("dk", b, ds.transpose(1, 2), q[:, a])):
            w = x @ y * scale
            r[name][0][:, at] = w
            r[name][1][:, at] = u * w.abs() + scale * ((size if name == "dq" else size.transpose(1, 2)) @ y.abs()) + tiny
        w = p.transpose(1, 2) @ go[:, a]
        r["dv"][0][:, b] = w
        r["dv"][1][:, b] = u * w.abs() + ((u + 1e-4) * p + tiny * seen).transpose(1, 2) @ go[:, a].abs() + tiny
    return lse, {n: (x.transpose(0, 1), y.transpose(0, 1)) for n, (x, y) in r.items()}


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("ql,kl,H,d_n,d_r,d_v,causal", [
    ([1], [1], 1, 128, 64, 128, True),
    ([1, 127, 128, 129, 5], None, 3, 128, 64, 128, True),
    ([300, 0, 257], None, 2, 128, 64, 128, False),
    ([100, 3], [350, 3], 2, 128, 64, 128, True),                  # queries at the end of longer keys
    ([200, 65], [70, 0], 2, 128, 64, 128, True),                  # queries that see nothing, a sequence without keys
    ([130, 0], [140, 60], 2, 64, 64, 64, True),                   # keys without queries
    ([70, 260], None, 2, 64, 0, 128, True), ([257], None, 1, 128, 0, 64, False),
    ([600], None, 5, 128, 64, 128, True),
    ([3] * 70 + [200], None, 1, 128, 64, 128, True),              # more sequences than a warp scans at once
    ([2880, 2305], None, 2, 128, 64, 128, True),                  # long rows of tiles whose last half is empty, or one row
    ([20, 1], [2500, 1300], 2, 128, 64, 128, True), ([1500], None, 2, 64, 0, 128, False),
])
def test_expanded_forward_and_gradients(dt, ql, kl, H, d_n, d_r, d_v, causal):
    from lazylora_b200.core import latent_attention as A
    kl = kl or ql
    q, kn, kp, v, cq, ck, go = _expand_case(dt, ql, kl, H, d_n, d_r, d_v, sum(ql) + H)
    scale = 1 / math.sqrt(d_n + d_r)
    out, lse = A.latent_attention_forward(q, kn, kp, v, cq, ck, scale, causal=causal)
    want_l, r = _expand_exact(q, kn, kp, v, go, out, ql, kl, scale, causal)
    none = want_l == -math.inf
    assert bool((lse[none] == -math.inf).all())
    _within(lse[~none], want_l[~none], 1e-4)
    _within(out, *r["out"])
    grads = A.latent_attention_backward(go, out, lse, q, kn, kp, v, cq, ck, scale, causal=causal)
    dq, dkn, dkp, dv = grads
    _within(dq, *r["dq"])
    _within(dv, *r["dv"])
    dk, bound = r["dk"]
    _within(dkn, dk[..., :d_n], bound[..., :d_n])
    if d_r:
        _within(dkp, dk[..., d_n:].sum(1), bound[..., d_n:].sum(1) + U[dt] * dk[..., d_n:].sum(1).abs())
    else:
        assert dkp is None
    again = A.latent_attention_backward(go, out, lse, q, kn, kp, v, cq, ck, scale, causal=causal)
    assert all(x is y or torch.equal(x, y) for x, y in zip(grads, again)), "bitwise reproducible"
    A.check_status()


def test_expanded_gradients_against_differences():
    """sum(out * g) along random directions: central differences of the 64-bit forward against the
    kernels' gradients. The differences are exact to 1e-6 here; each gradient is within the bound that the
    test above derives, so its product with the direction is within the sum of the bounds."""
    from lazylora_b200.core import latent_attention as A
    ql = [70, 33]
    q, kn, kp, v, cq, ck, go = _expand_case(HF, ql, ql, 2, 128, 64, 128, 4)
    scale, eps = 192 ** -0.5, 1e-4

    def loss(q, kn, kp, v):
        total, at = 0.0, 0
        for n in ql:
            a = slice(at, at + n)
            at += n
            k = torch.cat([kn[a], kp[a][:, None].expand(-1, 2, -1)], -1)
            s = torch.einsum("ihd,jhd->hij", q[a], k) * scale
            s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), -math.inf)
            total += (torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v[a]) * go[a].double()).sum()
        return float(total)

    out, lse = A.latent_attention_forward(q, kn, kp, v, cq, ck, scale)
    grads = A.latent_attention_backward(go, out, lse, q, kn, kp, v, cq, ck, scale)
    _, r = _expand_exact(q, kn, kp, v, go, out, ql, ql, scale, True)
    bounds = (r["dq"][1], r["dk"][1][..., :128], r["dk"][1][..., 128:].sum(1) * 2, r["dv"][1])
    x = [t.double() for t in (q, kn, kp, v)]
    g = _gen(8)
    for i in range(4):
        d = torch.randn(x[i].shape, generator=g, device="cuda", dtype=torch.float64)
        plus, minus = ([t + s * eps * d if j == i else t for j, t in enumerate(x)] for s in (1, -1))
        want = (loss(*plus) - loss(*minus)) / (2 * eps)
        got = float((grads[i].double() * d).sum())
        # delta comes from the stored output: its rounding (u |o|) moves dS by P |g| . u |o|
        extra = float((out.double().abs() * go.double().abs()).sum()) * U[HF] if i != 3 else 0.0
        assert abs(got - want) <= float((bounds[i] * d.abs()).sum()) + extra + 1e-4, i


def test_expanded_neighbours_do_not_leak():
    """A sequence full of NaN and infinities between two others leaves them as they are without it."""
    from lazylora_b200.core import latent_attention as A
    ql = [77, 50, 130]
    q, kn, kp, v, cq, ck, go = _expand_case(BF, ql, ql, 2, 128, 64, 128, 21)
    bad = slice(77, 127)
    for i, t in enumerate((q, kn, kp, v, go)):
        t[bad] = (float("nan"), float("inf"))[i % 2]
    keep = torch.cat([torch.arange(0, 77), torch.arange(127, 257)]).cuda()
    cut = lambda t: t[keep].contiguous()  # noqa: E731
    c2 = torch.tensor([0, 77, 207], dtype=torch.int32, device="cuda")
    out, lse = A.latent_attention_forward(q, kn, kp, v, cq, ck, 0.07)
    out2, lse2 = A.latent_attention_forward(cut(q), cut(kn), cut(kp), cut(v), c2, c2, 0.07)
    assert torch.equal(out[keep], out2) and torch.equal(lse[:, keep], lse2)
    got = A.latent_attention_backward(go, out, lse, q, kn, kp, v, cq, ck, 0.07)
    want = A.latent_attention_backward(cut(go), out2, lse2, cut(q), cut(kn), cut(kp), cut(v), c2, c2, 0.07)
    for x, y in zip(got, want):
        assert torch.equal(x[keep], y) and bool(torch.isfinite(y).all())


# -------------------------------------------------------------------------------------------- per head
@pytest.mark.parametrize("T,H,K,N,nk", [(1, 1, 64, 64, True), (5, 3, 128, 512, False), (130, 7, 512, 128, True),
                                        (64, 20, 72, 200, True), (300, 2, 256, 64, False)])
def test_head_linear(T, H, K, N, nk):
    """Exact products summed in fp32, one rounding: u relative, and the sums' 1e-4 of their size at most."""
    from lazylora_b200.core import dense
    from lazylora_b200.core import latent_attention as A
    g = _gen(T + N)
    x = _rand(g, BF, T, H, K + 8)[..., :K]
    w = _rand(g, BF, H, *((N, K) if nk else (K, N)))
    buf = torch.full((T, H, N + 64), 3.0, dtype=BF, device="cuda")
    y = A.head_linear(x, w, w_nk=nk, out=buf[..., :N])
    eq = "thk,hnk->thn" if nk else "thk,hkn->thn"
    want, size = torch.einsum(eq, x.double(), w.double()), torch.einsum(eq, x.double().abs(), w.double().abs())
    _within(y, want, U[BF] * want.abs() + 1e-6 * size + 1e-4 * want.pow(2).mean().sqrt())
    assert bool((buf[..., N:] == 3.0).all())
    assert torch.equal(A.head_linear(x, w, w_nk=nk), y)
    dense.check_status()


# -------------------------------------------------------------------------------------------- refusals
def test_refusals():
    from lazylora_b200.core import latent_attention as A
    z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    i64 = lambda *s: torch.zeros(*s, dtype=torch.int64, device="cuda")  # noqa: E731
    tab = torch.zeros(4, 64, device="cuda")
    for bad in (
        lambda: A.append_latent(z(2, 8, 192), z(1, 192, dt=HF), i64(1), i64(1), tab),
        lambda: A.append_latent(z(2, 8, 192), z(1, 200), i64(1), i64(1), tab),
        lambda: A.append_latent(z(2, 8, 192), z(1, 192), i32(1), i64(1), tab),
        lambda: A.append_latent(z(2, 8, 192), z(1, 192), i64(1), i64(2), tab),
        lambda: A.append_latent(z(2, 8, 192), z(1, 192), i64(1), i64(1), tab.to(BF)),
        lambda: A.append_latent(z(2, 8, 192), z(1, 192), i64(1), i64(1), tab, z(1, 2, 32)),
        lambda: A.append_latent(z(2, 8, 192).float(), z(1, 192).float(), i64(1), i64(1), tab),
        lambda: A.rotate_positions(z(2, 3, 24), i64(2), torch.zeros(4, 24, device="cuda")),
        lambda: A.paged_latent_attention(z(1, 1, 2, 192), z(2, 12, 192), i32(1, 1), i32(1), 128, 0.1),
        lambda: A.paged_latent_attention(z(1, 1, 2, 192), z(2, 8, 192), i32(1, 1), i32(1), 192, 0.1),
        lambda: A.paged_latent_attention(z(1, 1, 2, 192), z(2, 8, 192), i64(1, 1), i32(1), 128, 0.1),
        lambda: A.paged_latent_attention(z(1, 1, 2, 192), z(2, 8, 192), i32(2, 1), i32(1), 128, 0.1),
        lambda: A.paged_latent_attention(z(1, 1, 2, 192), z(2, 8, 192), i32(1, 1), i32(1), 128, 0.0),
        lambda: A.latent_attention_forward(z(4, 2, 192), z(4, 2, 128), z(4, 32), z(4, 2, 128), i32(2), i32(2), 0.1),
        lambda: A.latent_attention_forward(z(4, 2, 192), z(4, 2, 128), z(4, 64), z(4, 3, 128), i32(2), i32(2), 0.1),
        lambda: A.latent_attention_forward(z(4, 2, 192), z(4, 2, 128), z(4, 64), z(4, 2, 128), i32(2), i32(3), 0.1),
        lambda: A.latent_attention_forward(z(4, 2, 192), z(4, 2, 128), z(4, 64), z(4, 2, 128), i32(2), i32(2), -1.0),
        lambda: A.head_linear(z(2, 2, 64), z(3, 64, 64)),
        lambda: A.head_linear(z(2, 2, 60), z(2, 64, 60)),
        lambda: A.head_linear(z(2, 2, 64, dt=HF), z(2, 64, 64, dt=HF)),
        lambda: A.rotate_positions(torch.zeros(2, 3, 64), i64(2), tab),          # a CPU tensor
    ):
        with pytest.raises((ValueError, RuntimeError)):
            bad()


def test_empty_calls():
    from lazylora_b200.core import latent_attention as A
    z = lambda *s: torch.zeros(*s, dtype=BF, device="cuda")  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    i64 = torch.zeros(0, dtype=torch.int64, device="cuda")
    tab = torch.zeros(4, 64, device="cuda")
    assert A.append_latent(z(2, 8, 192), z(0, 192), i64, i64, tab, z(0, 3, 64)).shape == (0, 3, 64)
    assert A.rotate_positions(z(0, 3, 64), i64, tab).shape == (0, 3, 64)
    out, lse = A.paged_latent_attention(z(0, 1, 2, 192), z(2, 8, 192), i32(0, 1), i32(0), 128, 0.1)
    assert out.shape == (0, 1, 2, 128) and lse.shape == (0, 1, 2)
    x = (z(0, 2, 192), z(0, 2, 128), z(0, 64), z(0, 2, 128), i32(1), i32(1))
    out, lse = A.latent_attention_forward(*x, 0.1)
    assert out.shape == (0, 2, 128) and lse.shape == (2, 0)
    d = A.latent_attention_backward(z(0, 2, 128), out, lse, *x, 0.1)
    assert [tuple(t.shape) for t in d] == [(0, 2, 192), (0, 2, 128), (0, 64), (0, 2, 128)]
    assert A.head_linear(z(0, 2, 64), z(2, 128, 64)).shape == (0, 2, 128)
    A.check_status()
