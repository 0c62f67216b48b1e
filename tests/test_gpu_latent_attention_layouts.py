"""
The latent-attention operators in layouts, sizes and orders of calls beside the usual ones: caches whose
pages are interleaved, queries whose rows are unevenly spaced, block tables of other strides, more row
tiles than SMs, one long sequence among short ones, calls on two streams at once, a decode step captured in
a graph. Bounds: those of the tests that they take their checks from.
"""
import pytest
import torch

from test_gpu_latent_attention import BF, HF, _check_paged, _gen, _paged_case, _rand, _table, _turn, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,Tq,H", [
    ([100, 0, 130], 76, 64),          # 76 row tiles: one range of keys, no pieces, no join
    ([200, 0, 170, 3], 160, 64),      # 160 row tiles: more blocks than SMs
    ([70, 9], 74, 64),                # 74 row tiles: two ranges, the last count that is split
])
@pytest.mark.parametrize("d_c", [128, 512])
def test_paged_with_many_row_tiles(lens, Tq, H, d_c):
    from lazylora_b200.core import latent_attention as A
    q, cache, bt, sl, rows = _paged_case(BF, lens, Tq, H, d_c, 64, 8, Tq)
    out, lse = A.paged_latent_attention(q, cache, bt, sl, d_c, 0.06)
    _check_paged(out, lse, q, rows, d_c, 0.06)
    A.check_status()


@pytest.mark.parametrize("dt", [BF, HF])
def test_cache_with_interleaved_pages(dt):
    """[page_size][pages][D] in memory: a page's rows lie further apart than the pages do."""
    from lazylora_b200.core import latent_attention as A
    q, cache, bt, sl, rows = _paged_case(dt, [150, 3, 64], 2, 10, 128, 64, 16, 5)
    mixed = torch.empty(16, cache.shape[0], 192, dtype=dt, device="cuda").transpose(0, 1)
    mixed.copy_(cache)
    assert mixed.stride(0) < mixed.stride(1)
    out, lse = A.paged_latent_attention(q, mixed, bt, sl, 128, 0.1)
    _check_paged(out, lse, q, rows, 128, 0.1)
    plain = A.paged_latent_attention(q, cache, bt, sl, 128, 0.1)
    assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])
    g = _gen(6)
    kv, table = _rand(g, dt, 9, 192), _table(50, 64)
    slots = torch.randperm(cache.shape[0] * 16, generator=g, device="cuda")[:9]
    pos = torch.randint(0, 50, (9,), generator=g, device="cuda")
    cache.nan_to_num_(0.0)
    mixed.copy_(cache)
    A.append_latent(cache, kv, slots, pos, table)
    A.append_latent(mixed, kv, slots, pos, table)
    assert torch.equal(cache, mixed)
    turned, size = _turn(kv[:, 128:], pos, table, False)
    got = mixed[slots // 16, slots % 16]
    assert torch.equal(got[:, :128], kv[:, :128])
    _within(got[:, 128:], turned, turned.abs() * 2.0 ** -8 + size * 2.0 ** -22 + 2.0 ** -24)
    A.check_status()


def test_queries_with_unevenly_spaced_rows():
    """A slice of the heads of a wider buffer: rows (t, h) at no single distance, copied once."""
    from lazylora_b200.core import latent_attention as A
    q, cache, bt, sl, rows = _paged_case(BF, [90, 31], 3, 24, 128, 64, 8, 7)
    part = q[:, :, 5:12]
    out, lse = A.paged_latent_attention(part, cache, bt, sl, 128, 0.1)
    _check_paged(out, lse, part, rows, 128, 0.1)
    whole = A.paged_latent_attention(part.contiguous(), cache, bt, sl, 128, 0.1)
    assert torch.equal(out, whole[0]) and torch.equal(lse, whole[1])


@pytest.mark.parametrize("lens", [[90, 31, 64], [5, 8, 1]])
def test_block_tables_in_other_layouts(lens):
    """Columns first, and a slice of a wider table; the one-page tables' columns have any stride."""
    from lazylora_b200.core import latent_attention as A
    q, cache, bt, sl, rows = _paged_case(BF, lens, 1, 4, 128, 64, 8, 13)
    bt = bt[:, :(max(lens) + 7) // 8]
    want = A.paged_latent_attention(q, cache, bt.contiguous(), sl, 128, 0.1)
    _check_paged(*want, q, rows, 128, 0.1)
    for other in (bt, bt.t().contiguous().t(), torch.cat([bt, bt], 1)[:, bt.shape[1]:], bt.repeat_interleave(2, 1)[:, ::2]):
        got = A.paged_latent_attention(q, cache, other, sl, 128, 0.1)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    A.check_status()


def test_one_long_sequence_among_short_ones():
    """The long one is cut into more than a hundred pieces, the short ones into none."""
    from lazylora_b200.core import latent_attention as A
    lens = [40 + 19 * i for i in range(23)]
    lens.insert(11, 20000)
    q, cache, bt, sl, rows = _paged_case(BF, lens, 1, 16, 256, 64, 64, 8)
    out, lse = A.paged_latent_attention(q, cache, bt, sl, 256, 0.1)
    _check_paged(out, lse, q, rows, 256, 0.1)
    A.check_status()


def test_two_streams_at_once():
    """Two series of calls that run beside each other give what each gives alone."""
    from lazylora_b200.core import latent_attention as A
    cases = [_paged_case(BF, lens, 1, 32, 256, 64, 16, 9 + i) for i, lens in enumerate(([3000, 70, 900], [50] * 40))]
    xs = [(_rand(_gen(i), BF, 60, 8, 128), _rand(_gen(i + 2), BF, 8, 128, 256)) for i in range(2)]
    alone = [A.paged_latent_attention(*c[:4], 256, 0.1) + (A.head_linear(*x, w_nk=False),) for c, x in zip(cases, xs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(A.paged_latent_attention(*cases[i][:4], 256, 0.1) + (A.head_linear(*xs[i], w_nk=False),))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, alone[i]))
    A.check_status()


def test_decode_step_in_a_graph():
    """A captured decode step replayed with other tokens, slots, positions and lengths."""
    from test_gpu_latent_attention_layer import _layer
    from lazylora_b200.core import latent_attention as A
    g = _gen(10)
    B, d, page = 3, 192, 8
    layer, *_ = _layer(g, 5, d, 256, 64, 64, 128, True, False)
    bt = torch.randperm(12, generator=g, device="cuda").to(torch.int32).view(B, 4)
    caches = [torch.zeros(12, page, 320, dtype=BF, device="cuda") for _ in range(2)]
    x = torch.zeros(B, 1, d, dtype=BF, device="cuda")
    pos, slots = (torch.zeros(B, dtype=torch.int64, device="cuda") for _ in range(2))
    sl = torch.ones(B, dtype=torch.int32, device="cuda")
    step = lambda c: layer.decode(x, c, slots, pos, bt, sl)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    slots.fill_(-1)                                               # the step before the capture writes nothing
    with torch.cuda.stream(s):
        step(caches[0])
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(caches[0])
    caches[0].zero_()
    for t in range(20):
        x.copy_(_rand(g, BF, B, 1, d))
        p = torch.tensor([t, (t + 3) % 20, 5 + t // 2], device="cuda")
        pos.copy_(p)
        slots.copy_(bt[torch.arange(B, device="cuda"), p // page].long() * page + p % page)
        sl.copy_(p + 1)
        graph.replay()
        assert torch.equal(y, step(caches[1]))
    assert torch.equal(caches[0], caches[1])
    A.check_status()


def test_two_host_threads():
    """Calls of different widths from two threads, whose kernels take different amounts of shared memory."""
    import threading
    from lazylora_b200.core import latent_attention as A
    paged = [_paged_case(BF, [300, 40], 1, 64, d_c, 64, 8, d_c) for d_c in (512, 128)]
    g = _gen(14)
    cu = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    packed = [(_rand(g, BF, 200, 2, d), _rand(g, BF, 200, 2, 64 if i else 128), None if i else _rand(g, BF, 200, 64),
               _rand(g, BF, 200, 2, 64), cu, cu, 0.1) for i, d in enumerate((192, 64))]
    heads = [(_rand(g, BF, 40, 8, 128), _rand(g, BF, 8, 64 + 448 * i, 128)) for i in range(2)]

    def step(i):
        out = A.paged_latent_attention(*paged[i][:4], (512, 128)[i], 0.1)
        o, lse = A.latent_attention_forward(*packed[i])
        return (*out, o, *A.latent_attention_backward(o, o, lse, *packed[i]), A.head_linear(*heads[i]))
    alone = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    faults = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(400):
                    got = step(i)
                torch.cuda.current_stream().synchronize()
                if not all(x is y or torch.equal(x, y) for x, y in zip(got, alone[i])):
                    faults.append("other results")
        except Exception as e:  # noqa: BLE001
            faults.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not faults, faults
    A.check_status()
