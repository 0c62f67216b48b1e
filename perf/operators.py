"""
The latent-attention operators (lazylora_b200.core.latent_attention) as measured cases: what each
stands for in use, its inputs, one pass through it, its unavoidable bytes and operations, and its
definition in 64 bits.

Four operators, of an attention layer whose keys and values come from one shared latent vector per
token (d_c values) and one rotary key per token (d_r values):

  append   new tokens' latent rows and rotated keys written into a paged cache, their queries'
           rotary part rotated on the way
  paged    the absorbed form over that cache: every head's query has d_c + d_r values, a token's key
           is its cache row and its value the row's first d_c entries
  heads    one product per head (absorbing the queries into the latent space, expanding the outputs)
  expand   the expanded form: per-head keys and values, one rotary key shared by the heads, packed
           sequences, causal; forward alone (prompts) or with its backward pass (training)
"""
import math

import torch

#: The tools set this: False computes the plain form, True calls the framework's operators.
own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a decode step of 40 sequences: the smallest call, bound by latency
        {"name": "append_step", "kind": "append", "T": 40, "H": 64, "d_c": 512, "d_r": 64, "page": 32, "pages": 600,
         "interleaved": False, "type": "bf16"},
        # the prompts of a serving step written at once, in pages that are no power of two
        {"name": "append_prompt", "kind": "append", "T": 9001, "H": 64, "d_c": 512, "d_r": 64, "page": 48, "pages": 300,
         "interleaved": True, "type": "bf16"},
        # one user, a short context
        {"name": "paged_one", "kind": "paged", "B": 1, "Tq": 1, "H": 32, "d_c": 512, "d_r": 64, "page": 16,
         "shortest": 700, "longest": 700, "type": "bf16"},
        # a batch of ragged contexts, as a server decodes it
        {"name": "paged_batch", "kind": "paged", "B": 44, "Tq": 1, "H": 64, "d_c": 512, "d_r": 64, "page": 64,
         "shortest": 1, "longest": 6000, "type": "bf16"},
        # a few very long contexts: the split along the keys
        {"name": "paged_long", "kind": "paged", "B": 4, "Tq": 1, "H": 64, "d_c": 512, "d_r": 64, "page": 64,
         "shortest": 50000, "longest": 70000, "type": "bf16"},
        # drafted tokens verified together, many heads: 256 query rows a sequence
        {"name": "paged_verify", "kind": "paged", "B": 24, "Tq": 2, "H": 128, "d_c": 512, "d_r": 64, "page": 24,
         "shortest": 1500, "longest": 5000, "type": "fp16"},
        # queries into the latent space for a decode batch
        {"name": "heads_absorb", "kind": "heads", "T": 40, "H": 64, "K": 128, "N": 512, "nk": False},
        # outputs back from it for a longer step
        {"name": "heads_expand", "kind": "heads", "T": 900, "H": 64, "K": 512, "N": 128, "nk": True},
        # a few short prompts
        {"name": "prompt_short", "kind": "expand", "train": False, "B": 5, "shortest": 1, "longest": 150, "H": 20,
         "earlier": 0, "type": "fp16"},
        # one long prompt
        {"name": "prompt_long", "kind": "expand", "train": False, "B": 1, "shortest": 8000, "longest": 8000, "H": 32,
         "earlier": 0, "type": "bf16"},
        # packed documents of a fine-tuning step: sequences of at most 1024 tokens
        {"name": "train_packed", "kind": "expand", "train": True, "B": 7, "shortest": 150, "longest": 1024, "H": 64,
         "earlier": 0, "type": "bf16"},
        # one long training sequence
        {"name": "train_long", "kind": "expand", "train": True, "B": 1, "shortest": 4100, "longest": 4100, "H": 64,
         "earlier": 0, "type": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of its range; the one size kept out of every case is drawn again."""
    while True:
        n = min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.999)))))))
        if n != 3072:
            return n


def _draw_once(rng):
    kind = rng.choice(["append", "paged", "paged", "heads", "expand", "expand"])
    if kind == "append":
        page = rng.choice([8, 16, 24, 32, 48, 64, 128])
        T = _spread(rng, 1, 9001)
        return {"kind": kind, "T": T, "H": rng.choice([8, 20, 32, 64, 128]), "d_c": rng.choice([128, 256, 384, 512]),
                "d_r": 64, "page": page, "pages": T // page + rng.randint(1, 200), "interleaved": rng.random() < 0.5,
                "type": rng.choice(["bf16", "fp16"])}
    if kind == "paged":
        longest = _spread(rng, 1, 70000)
        return {"kind": kind, "B": _spread(rng, 1, 96), "Tq": rng.choice([1, 1, 1, 2, 3, 5]),
                "H": rng.choice([10, 20, 32, 64, 96, 128]), "d_c": rng.choice([128, 256, 384, 512, 512, 512]),
                "d_r": rng.choice([0, 64, 64, 64]), "page": rng.choice([8, 16, 24, 32, 64, 128]),
                "shortest": rng.choice([0, 1, longest // 2, longest]), "longest": longest,
                "type": rng.choice(["bf16", "fp16"])}
    if kind == "heads":
        K, N, nk = rng.choice([(128, 512, False), (512, 128, True), (64, 256, False), (256, 64, True)])
        return {"kind": kind, "T": _spread(rng, 1, 900), "H": rng.choice([8, 20, 32, 64]), "K": K, "N": N, "nk": nk}
    train = rng.random() < 0.5
    longest = _spread(rng, 1, 4100 if train else 8000)
    return {"kind": kind, "train": train, "B": _spread(rng, 1, 24),
            "shortest": rng.choice([1, max(1, longest // 2), longest]), "longest": longest, "H": rng.choice([4, 10, 20, 32, 64]),
            "earlier": 0 if train else rng.choice([0, 0, 1, longest // 2]), "type": rng.choice(["bf16", "fp16"])}


def draw(rng):
    """One more case of the listed ranges, none dearer than the largest listed one."""
    most = {}
    for c in listed():
        w = work(c)
        for k in ("bytes", "flops"):
            most[k] = max(most.get(k, 0), w[k])
    while True:
        c = _draw_once(rng)
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and _plain_cells(c) <= 1.1e9:
            return c


def _plain_cells(c):
    """Scores that the padded plain form holds at a time."""
    if c["kind"] == "expand":
        return c["B"] * c["H"] * c["longest"] * (c["longest"] + c["earlier"])
    if c["kind"] == "paged":
        return c["B"] * c["Tq"] * c["H"] * c["longest"]
    return 0


def _lengths(c):
    """A case's sequence lengths, the same for every seed: spread evenly from the shortest to the
    longest, in an order that mixes them."""
    B, lo, hi = c["B"], c["shortest"], c["longest"]
    even = [hi if B == 1 else lo + (hi - lo) * i // (B - 1) for i in range(B)]
    return [even[(i * 7 + 3) % B] if B % 7 else even[(i * 5 + 3) % B if B % 5 else i] for i in range(B)]


# ------------------------------------------------------------------------------------------- work
def work(case):
    """What one pass cannot do without: inputs read once, outputs written once, products over the
    visible pairs alone."""
    c = case
    if c["kind"] == "append":
        row = c["d_c"] + c["d_r"]
        n = c["T"] * (2 * row + 2 * c["H"] * c["d_r"]) * 2 + c["T"] * (16 + 4 * c["d_r"])
        return {"bytes": n, "flops": 3 * c["T"] * (c["H"] + 1) * c["d_r"]}
    if c["kind"] == "heads":
        return {"bytes": 2 * c["H"] * (c["T"] * (c["K"] + c["N"]) + c["K"] * c["N"]),
                "flops": 2 * c["H"] * c["T"] * c["K"] * c["N"]}
    lens = _lengths(c)
    if c["kind"] == "paged":
        row, rows = c["d_c"] + c["d_r"], c["Tq"] * c["H"]
        pairs = sum(max(0, n - c["Tq"] + 1 + t) for n in lens for t in range(c["Tq"])) * c["H"]
        return {"bytes": 2 * row * sum(lens) + c["B"] * rows * (2 * row + 2 * c["d_c"] + 4),
                "flops": 2 * pairs * (row + c["d_c"])}
    tq, tk, H = sum(lens), sum(lens) + c["earlier"] * len(lens), c["H"]
    pairs = H * sum(n * c["earlier"] + n * (n + 1) // 2 for n in lens)
    ins = 2 * (tq * H * 192 + tk * H * 256 + tk * 64)
    outs = 2 * tq * H * 128 + 4 * tq * H
    if not c["train"]:
        return {"bytes": ins + outs, "flops": 2 * pairs * (192 + 128)}
    # the backward pass reads the inputs, the output and its gradient, and writes four gradients;
    # its five products are the scores again (192), dP (128), dV (128), dQ (192) and dK (192)
    return {"bytes": 3 * ins + 2 * outs + 2 * tq * H * 128, "flops": 2 * pairs * (192 + 128 + 192 + 128 + 128 + 192 + 192)}


# ----------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[c.get("type", "bf16")]
    rand = lambda *shape, std=1.0: (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)  # noqa: E731
    s = {"case": c}
    if c["kind"] == "append":
        T, rows = c["T"], c["page"] * c["pages"]
        s["cache"] = rand(c["pages"], c["page"], c["d_c"] + c["d_r"])
        s["kv"] = rand(T, c["d_c"] + c["d_r"])
        s["q_pe"] = rand(T, c["H"], c["d_r"])
        s["slots"] = torch.randperm(rows, generator=g, device="cuda")[:T]
        s["slots"][T // 2] = -1 if T > 3 else s["slots"][T // 2]         # a padding token is not written
        s["positions"] = torch.randint(0, 16384, (T,), generator=g, device="cuda")
        inv = 10000.0 ** (-torch.arange(0, c["d_r"], 2, device="cuda", dtype=torch.float64) / c["d_r"])
        angle = torch.arange(16384, device="cuda", dtype=torch.float64)[:, None] * inv
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        return s
    if c["kind"] == "heads":
        s["x"] = rand(c["T"], c["H"], c["K"])
        s["w"] = rand(c["H"], *((c["N"], c["K"]) if c["nk"] else (c["K"], c["N"])), std=c["K"] ** -0.5)
        return s
    lens = _lengths(c)
    if c["kind"] == "paged":
        row, page = c["d_c"] + c["d_r"], c["page"]
        need = [(n + page - 1) // page for n in lens]
        order = torch.randperm(sum(need) + 3, generator=g, device="cuda").to(torch.int32)
        at = torch.zeros((c["B"], max(1, max(need))), dtype=torch.int32)
        first = 0
        host = order.cpu()
        for b, n in enumerate(need):
            at[b, :n] = host[first:first + n]
            first += n
        s["cache"] = rand(sum(need) + 3, page, row)
        s["block_table"] = at.cuda()
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["longest"] = max(lens)
        s["q"] = rand(c["B"], c["Tq"], c["H"], row)
        s["scale"] = 192 ** -0.5
        return s
    H = c["H"]
    kl = [n + c["earlier"] for n in lens]
    cum = lambda ls: torch.tensor([sum(ls[:i]) for i in range(len(ls) + 1)], dtype=torch.int32, device="cuda")  # noqa: E731
    s["cu_q"], s["cu_k"] = cum(lens), cum(kl)
    s["longest"] = (max(lens), max(kl))
    s["q"] = rand(sum(lens), H, 192)
    kv = rand(sum(kl), H, 256)                          # the up-projection's output: keys and values side by side
    s["k_nope"], s["v"] = kv[..., :128], kv[..., 128:]
    s["k_pe"] = rand(sum(kl), 64)
    s["scale"] = 192 ** -0.5
    if c["train"]:
        s["g"] = rand(sum(lens), H, 128)
    return s


# ------------------------------------------------------------------------------------------- runs
def run(state):
    kind = state["case"]["kind"]
    if own:
        from lazylora_b200.core import latent_attention as A
        s, c = state, state["case"]
        if kind == "append":
            q_pe = A.append_latent(s["cache"], s["kv"], s["slots"], s["positions"], s["table"], s["q_pe"],
                                   interleaved=c["interleaved"])
            return {"cache": s["cache"], "q_pe": q_pe}
        if kind == "heads":
            return A.head_linear(s["x"], s["w"], w_nk=c["nk"])
        if kind == "paged":
            out, lse = A.paged_latent_attention(s["q"], s["cache"], s["block_table"], s["seq_lens"], c["d_c"], s["scale"])
            return {"out": out, "lse": lse}
        x = (s["q"], s["k_nope"], s["k_pe"], s["v"])
        out, lse = A.latent_attention_forward(*x, s["cu_q"], s["cu_k"], s["scale"])
        res = {"out": out, "lse": lse}
        if c["train"]:
            d = A.latent_attention_backward(s["g"], out, lse, *x, s["cu_q"], s["cu_k"], s["scale"])
            res.update(zip(("dq", "dk_nope", "dk_pe", "dv"), d))
        return res
    return {"append": _append, "heads": _heads, "paged": _paged, "expand": _expand}[kind](state)


def _turn(x, cos, sin, interleaved):
    """x [..., d_r] turned by the angles whose cosines and sines are given [..., d_r / 2]."""
    h = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :h], x[..., h:])
    u, v = a * cos - b * sin, a * sin + b * cos
    return torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)


def _append(s):
    c, dt = s["case"], s["kv"].dtype
    cs = s["table"][s["positions"]]
    cos, sin = cs[:, :c["d_r"] // 2], cs[:, c["d_r"] // 2:]
    k_pe = _turn(s["kv"][:, c["d_c"]:].float(), cos, sin, c["interleaved"]).to(dt)
    rows = torch.cat([s["kv"][:, :c["d_c"]], k_pe], 1)
    flat, keep = s["cache"].view(-1, rows.shape[1]), s["slots"] >= 0
    # a token without a slot writes one row past a copy of the cache
    padded = torch.cat([flat, flat[:1]])
    padded[torch.where(keep, s["slots"], flat.shape[0])] = rows
    flat.copy_(padded[:-1])
    q = _turn(s["q_pe"].float(), cos[:, None], sin[:, None], c["interleaved"]).to(dt)
    return {"cache": s["cache"], "q_pe": q}


def _heads(s):
    w = s["w"].float()
    return torch.matmul(s["x"].float().transpose(0, 1), w.transpose(1, 2) if s["case"]["nk"] else w).transpose(0, 1).to(s["x"].dtype).contiguous()


def _softmax(scores, seen):
    """(probabilities, log of the sum of exponentials) over the last axis where `seen`; a row that
    sees nothing has zeros and minus infinity."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    return e / total.clamp_min(1e-38), (top + torch.log(total)).squeeze(-1)


def _paged(s):
    c = s["case"]
    B, Tq, H, d_c, n = c["B"], c["Tq"], c["H"], c["d_c"], s["longest"]
    if n == 0:
        return {"out": torch.zeros_like(s["q"][..., :d_c]).contiguous(), "lse": torch.full((B, Tq, H), -math.inf, device="cuda")}
    rows = s["cache"][s["block_table"].long()].flatten(1, 2)[:, :n].float()
    scores = torch.matmul(s["q"].float().flatten(1, 2), rows.transpose(1, 2)).view(B, Tq, H, n) * s["scale"]
    last = s["seq_lens"].long()[:, None] - Tq + torch.arange(Tq, device="cuda")        # the last key that a query sees
    p, lse = _softmax(scores, (torch.arange(n, device="cuda") <= last[:, :, None])[:, :, None])
    out = torch.matmul(p.flatten(1, 2), rows[..., :d_c]).view(B, Tq, H, d_c)
    return {"out": out.to(s["q"].dtype), "lse": lse}


def _expand(s):
    c, dt = s["case"], s["q"].dtype
    nq, nk = s["longest"]
    lens = lambda cu: (cu[1:] - cu[:-1]).long()[:, None]  # noqa: E731
    iq, ik = torch.arange(nq, device="cuda")[None], torch.arange(nk, device="cuda")[None]
    has_q, has_k = iq < lens(s["cu_q"]), ik < lens(s["cu_k"])
    at_q = (s["cu_q"][:-1].long()[:, None] + iq).clamp_max(s["q"].shape[0] - 1)
    at_k = (s["cu_k"][:-1].long()[:, None] + ik).clamp_max(s["k_pe"].shape[0] - 1)
    H = c["H"]
    q = s["q"].float()[at_q].transpose(1, 2)                                            # [B, H, nq, 192]
    k = torch.cat([s["k_nope"].float(), s["k_pe"].float()[:, None].expand(-1, H, -1)], -1)[at_k].transpose(1, 2)
    v = s["v"].float()[at_k].transpose(1, 2)
    shift = lens(s["cu_k"]) - lens(s["cu_q"])
    seen = has_q[:, :, None] & has_k[:, None] & (ik[:, None] <= (iq + shift)[:, :, None])
    p, lse = _softmax(torch.matmul(q, k.transpose(2, 3)) * s["scale"], seen[:, None])
    out = torch.matmul(p, v)
    pack_q = lambda t: t.transpose(1, 2)[has_q]  # noqa: E731  (the rows of real queries, in their order)
    pack_k = lambda t: t.transpose(1, 2)[has_k]  # noqa: E731
    packed = pack_q(out)
    res = {"out": packed.to(dt), "lse": pack_q(lse[..., None])[..., 0].t().contiguous()}
    if c["train"]:
        g = s["g"].float()[at_q].transpose(1, 2) * has_q[:, None, :, None]
        # the backward pass is handed the output as it was stored
        o = res["out"].float()[at_q].transpose(1, 2)
        ds = p * (torch.matmul(g, v.transpose(2, 3)) - (g * o).sum(-1, keepdim=True)) * s["scale"]
        res["dq"] = pack_q(torch.matmul(ds, k)).to(dt)
        dk = pack_k(torch.matmul(ds.transpose(2, 3), q))
        res["dk_nope"], res["dk_pe"] = dk[..., :128].to(dt), dk[..., 128:].sum(1).to(dt)
        res["dv"] = pack_k(torch.matmul(p.transpose(2, 3), g)).to(dt)
    return res


# ------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """What run() returns, from the definitions in 64 bits, sequence by sequence and head by head."""
    c, s = case, prepare(case, seed)
    f = lambda t: t.to(torch.float64)  # noqa: E731
    if c["kind"] == "append":
        d_c, h = c["d_c"], c["d_r"] // 2
        ang = f(s["table"])[s["positions"]]
        z = torch.complex(ang[:, :h].contiguous(), ang[:, h:].contiguous())

        def turned(x, z):
            x = f(x)
            w = (torch.complex(x[..., ::2].contiguous(), x[..., 1::2].contiguous()) if c["interleaved"]
                 else torch.complex(x[..., :h].contiguous(), x[..., h:].contiguous())) * z
            if c["interleaved"]:
                return torch.view_as_real(w).reshape(x.shape)
            return torch.cat([w.real, w.imag], -1)

        cache = f(s["cache"]).view(-1, d_c + c["d_r"])
        on = (s["slots"] >= 0).nonzero()[:, 0]
        cache[s["slots"][on], :d_c] = f(s["kv"])[on, :d_c]
        cache[s["slots"][on], d_c:] = turned(s["kv"][:, d_c:], z)[on]
        return {"cache": cache.view(s["cache"].shape), "q_pe": turned(s["q_pe"], z[:, None])}
    if c["kind"] == "heads":
        return torch.einsum("thk,hnk->thn" if c["nk"] else "thk,hkn->thn", f(s["x"]), f(s["w"]))
    lens = _lengths(c)
    if c["kind"] == "paged":
        out = torch.zeros(*s["q"].shape[:3], c["d_c"], dtype=torch.float64, device="cuda")
        lse = torch.full(s["q"].shape[:3], -math.inf, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            for t in range(c["Tq"]):
                m = n - c["Tq"] + t + 1
                if m <= 0:
                    continue
                used = (m + c["page"] - 1) // c["page"]
                rows = f(s["cache"][s["block_table"][b, :used].long()]).reshape(-1, c["d_c"] + c["d_r"])[:m]
                z = f(s["q"][b, t]) @ rows.T * s["scale"]
                lse[b, t] = torch.logsumexp(z, -1)
                out[b, t] = torch.exp(z - lse[b, t][:, None]) @ rows[:, :c["d_c"]]
        return {"out": out, "lse": lse}
    H = c["H"]
    new = lambda t: torch.zeros(t.shape, dtype=torch.float64, device="cuda")  # noqa: E731
    res = {"out": torch.zeros(s["q"].shape[0], H, 128, dtype=torch.float64, device="cuda"),
           "lse": torch.zeros(H, s["q"].shape[0], dtype=torch.float64, device="cuda")}
    if c["train"]:
        res.update(dq=new(s["q"]), dk_nope=new(s["k_nope"]), dk_pe=new(s["k_pe"]), dv=new(s["v"]))
    q0 = k0 = 0
    for n in lens:
        m = n + c["earlier"]
        qs, ks = slice(q0, q0 + n), slice(k0, k0 + m)
        q0, k0 = q0 + n, k0 + m
        hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
        for h in range(H):
            q, v = f(s["q"][qs, h]), f(s["v"][ks, h])
            k = torch.cat([f(s["k_nope"][ks, h]), f(s["k_pe"][ks])], 1)
            z = (q @ k.T * s["scale"]).masked_fill(hidden, -math.inf)
            lse = torch.logsumexp(z, 1)
            p = torch.exp(z - lse[:, None])
            o = p @ v
            res["out"][qs, h], res["lse"][h, qs] = o, lse
            if c["train"]:
                g = f(s["g"][qs, h])
                ds = p * (g @ v.T - (g * o).sum(1)[:, None]) * s["scale"]
                res["dq"][qs, h] = ds @ k
                dk = ds.T @ q
                res["dk_nope"][ks, h] = dk[:, :128]
                res["dk_pe"][ks] += dk[:, 128:]
                res["dv"][ks, h] = p.T @ g
    return res
