"""The paged cache on the GPU: append, decode, prefill and evict against 64-bit
references (paged_util), with NaN in every place that no query may see."""
import numpy as np
import pytest

import obsmoe

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_(cuda):
    return cuda


def make_ctx(heads, kv, hd, page, dtype="bf16", seqs=16, max_len=4096, weights=False):
    ctx = obsmoe.MoeContext(obsmoe.MoeShape(2048, 256, 16, 4, n_layers=1, max_tokens=1), 0)
    ctx.paged_init(n_heads=heads, n_kv_heads=kv, head_dim=hd, page_size=page, max_seqs=seqs, max_kv_len=max_len,
                   dtype=dtype, weights=weights)
    return ctx


def view(c):
    return obsmoe.PagedKV(c.k, c.v, c.table, c.len)


def queries(torch, rows, heads, hd, dtype, seed, amp=1.0):
    gen = torch.Generator(device="cuda").manual_seed(1000 + seed)
    return (amp * torch.randn((rows, heads, hd), generator=gen, device="cuda")).to(dtype)


# ------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("kv,hd,page,order,rows", [
    (4, 128, 64, "slots", 1), (4, 128, 64, "heads", 97), (1, 8, 1, "slots", 33), (3, 80, 3, "heads", 50),
    (8, 64, 16, "slots", 700), (2, 120, 1000, "slots", 1300)])
def test_append(torch_, dtype, kv, hd, page, order, rows):
    from paged_util import Cache

    torch = torch_
    c = Cache([rows, 5, rows // 2 + 1], kv, hd, page, dtype, order=order)
    ctx = make_ctx(4 * kv, kv, hd, page, dtype)
    want_k, want_v = c.k.clone(), c.v.clone()
    gen = torch.Generator(device="cuda").manual_seed(5)
    # rows cut out of a wider projection, in a mixed order of sequences and positions
    wide = torch.randn((rows, 2 * kv * hd + 8), generator=gen, device="cuda").to(c.dtype)
    k, v = (wide[:, i * kv * hd:(i + 1) * kv * hd].unflatten(1, (kv, hd)) for i in (0, 1))
    seq = torch.tensor([(0 if t % 3 else 2) if t < len(range(rows)) else 0 for t in range(rows)], dtype=torch.int32)
    slot = torch.zeros(rows, dtype=torch.int32)
    for s in (0, 2):
        at = (seq == s).nonzero()[:, 0]
        slot[at] = torch.randperm(c.lens[s])[: len(at)].to(torch.int32)
    seq, slot = seq.cuda(), slot.cuda()
    for s in (0, 2):
        at = (seq == s).nonzero()[:, 0]
        if len(at):
            p, o = c.places(s, slot[at].long())
            want_k[p, o], want_v[p, o] = k[at], v[at]
    ctx.paged_append(view(c), k, v, seq, slot, rows)
    ctx.check_device()
    for got, want in ((c.k, want_k), (c.v, want_v)):
        assert torch.equal(got.contiguous().view(torch.int16), want.contiguous().view(torch.int16))
    ctx.close()


# ------------------------------------------------------------------- decode
DECODE = [
    # heads, kv, hd, page, lens, window, sinks
    (32, 4, 128, 64, [1], 0, 0),
    (32, 4, 128, 64, [2049], 0, 0),
    (32, 4, 128, 16, [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 700, 0, 1031, 3], 0, 0),
    (8, 1, 128, 64, [3000, 1], 0, 0),
    (16, 16, 64, 16, [5, 333, 64], 0, 0),
    (12, 4, 80, 32, [100, 31], 0, 0),
    (5, 1, 8, 1, [1, 2, 77], 0, 0),
    (32, 2, 120, 128, [260, 511], 0, 0),
    (15, 1, 64, 3, [400], 0, 0),
    (26, 2, 128, 1000, [1999, 7], 0, 0),
    (32, 4, 128, 64, [1, 100, 128, 129, 1000, 4000], 128, 4),
    (32, 4, 128, 64, [1000, 65, 0, 2048], 1, 0),
    (32, 4, 128, 16, [1000, 65, 0, 333], 1, 1),
    (12, 4, 64, 32, [900, 50], 37, 13),
    (8, 1, 128, 64, [700, 300], 100, 650),  # more sinks than the window leaves out
    (4, 4, 128, 64, [500], 10000, 3),       # a window wider than the cache
]


def check_decode(torch, c, ctx, heads, window, sinks, seed, weights=False, q=None, scale=0.0, stream=None):
    from paged_util import attend, check_out, visible

    n, group = len(c.lens), heads // c.kv
    if q is None:
        q = queries(torch, n, heads, c.hd, c.dtype, seed)
    out = torch.full((n, heads, c.hd), float("nan"), dtype=c.dtype, device="cuda")
    w0 = w = None
    if weights:
        w0 = torch.rand((n, c.kv, max(c.lens) + 3), device="cuda")
        w = w0.clone()
    ctx.paged_decode(view(c), q, out, window=window, n_sink=sinks, scale=scale, weights=w, stream=stream)
    ctx.check_device(stream)
    for s, ln in enumerate(c.lens):
        ok = visible(torch.tensor([ln - 1], device="cuda"), ln, window, sinks)
        k, v = c.rows(s, ln)
        if w is not None:
            assert torch.equal(w[s, :, ln:], w0[s, :, ln:])
        for h in range(c.kv):
            o, a, sv, p = attend(q[s:s + 1, h * group:(h + 1) * group], k[:, h], v[:, h], ok, scale or c.hd ** -0.5)
            check_out(out[s:s + 1, h * group:(h + 1) * group], o, a, sv, c.dtype)
            if w is not None and ln:
                add = p[0].sum(0)
                want = w0[s, h, :ln].double() + add
                bound = 1e-4 * add + 2.0 ** -22 * want
                assert bool(((w[s, h, :ln].double() - want).abs() <= bound).all()), (s, h)
                assert torch.equal(w[s, h, :ln][~ok[0]], w0[s, h, :ln][~ok[0]])
    return q, out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode(torch_, dtype, case):
    from paged_util import Cache

    heads, kv, hd, page, lens, window, sinks = DECODE[case]
    c = Cache(lens, kv, hd, page, dtype, seed=case, order="heads" if case % 2 else "slots", table_extra=case % 3)
    blank(torch_, c, window, sinks, [1] * len(lens))
    ctx = make_ctx(heads, kv, hd, page, dtype, weights=True)
    check_decode(torch_, c, ctx, heads, window, sinks, case)
    check_decode(torch_, c, ctx, heads, window, sinks, case, weights=True)
    ctx.close()


def blank(torch, c, window, sinks, rows):
    """NaN, infinities and the type's extremes in every held position that no query of the last `rows` sees."""
    if not window:
        return
    bad = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(c.dtype).min], dtype=c.dtype, device="cuda")
    for s, n in enumerate(c.lens):
        lo = max(0, n - rows[s] + 1 - window)
        j = torch.arange(min(sinks, lo), lo, device="cuda")
        if len(j):
            x = bad[j % 4][:, None, None].expand(len(j), c.kv, c.hd)
            c.put(s, j, x, x)


def test_decode_long_and_batched(torch_):
    """A long axis split many ways next to short sequences; the same call twice gives the same bits."""
    from paged_util import Cache

    torch = torch_
    c = Cache([40000, 1, 700, 0, 129], 4, 128, 64, "bf16", seed=3)
    ctx = make_ctx(32, 4, 128, 64, "bf16", seqs=5, max_len=40000, weights=True)
    q, one = check_decode(torch, c, ctx, 32, 0, 0, 3)
    _, two = check_decode(torch, c, ctx, 32, 0, 0, 3, q=q)
    assert torch.equal(one, two)
    check_decode(torch, c, ctx, 32, 0, 0, 3, weights=True)
    check_decode(torch, c, ctx, 32, 20000, 5, 3, weights=True)
    ctx.close()
    many = Cache([(i * 37) % 300 for i in range(600)], 2, 64, 16, "f16", seed=4)
    ctx = make_ctx(4, 2, 64, 16, "f16", seqs=600, max_len=512)
    check_decode(torch, many, ctx, 4, 0, 0, 4)
    check_decode(torch, many, ctx, 4, 33, 2, 4)
    ctx.close()


def test_decode_extreme_scores(torch_):
    """Scores of hundreds in size (one position takes all), -inf scores, a sequence whose scores are all -inf
    (0/0, as the formula), and a NaN query: each stays in its own row."""
    from paged_util import Cache

    torch = torch_
    c = Cache([300, 300, 300, 300], 2, 128, 16, "bf16", seed=6, amp=30.0)
    ctx = make_ctx(16, 2, 128, 16, "bf16")
    check_decode(torch, c, ctx, 16, 0, 0, 6, q=queries(torch, 4, 16, 128, c.dtype, 6, amp=1.0))
    q = queries(torch, 4, 16, 128, c.dtype, 7).abs() + 0.25
    c.k[c.table[0].long()[2], 5] = -float("inf")           # one -inf score: that position gets nothing
    for p in c.table[1].long()[: -(-300 // 16)].tolist():  # every score -inf
        c.k[p] = -float("inf")
    q[2, 3] = float("nan")
    out = torch.empty_like(q)
    ctx.paged_decode(view(c), q, out)
    ctx.check_device()
    assert torch.isnan(out[1]).all()
    assert torch.isnan(out[2, 3]).all() and not torch.isnan(out[2, :3]).any() and not torch.isnan(out[2, 4:]).any()
    assert not torch.isnan(out[0]).any() and not torch.isnan(out[3]).any()
    ctx.close()


# ------------------------------------------------------------------ prefill
PREFILL = [
    # heads, kv, hd, page, lens, rows, window, sinks
    (32, 4, 128, 64, [1], [1], 0, 0),
    (32, 4, 128, 64, [300], [300], 0, 0),
    (32, 4, 128, 16, [700, 129, 1, 0, 256, 40], [33, 129, 1, 0, 1, 0], 0, 0),
    (8, 1, 128, 64, [1031, 17], [700, 17], 0, 0),
    (16, 16, 64, 16, [5, 333, 64, 128], [5, 333, 10, 128], 0, 0),
    (12, 4, 80, 32, [400, 31], [100, 31], 0, 0),
    (5, 1, 8, 1, [130, 2], [130, 1], 0, 0),
    (32, 2, 120, 128, [260, 511], [260, 3], 0, 0),
    (15, 1, 64, 3, [400], [399], 0, 0),
    (13, 1, 128, 1000, [900], [300], 0, 0),
    (32, 4, 128, 64, [1500, 700], [1500, 64], 128, 4),
    (32, 4, 128, 64, [400, 300], [400, 20], 1, 0),
    (32, 4, 128, 16, [400, 300], [400, 20], 1, 1),
    (12, 4, 64, 32, [900, 50], [333, 50], 37, 13),
    (8, 1, 128, 64, [700, 300], [500, 300], 100, 650),
    (4, 4, 128, 64, [500], [500], 10000, 3),
    (8, 2, 128, 64, [5, 200], [9, 201], 0, 0),      # more rows than positions: the first ones see nothing
    (8, 2, 64, 64, [3000], [20], 0, 0),             # few rows, long axis
]


def check_prefill(torch, c, ctx, heads, rows, window, sinks, seed, q=None, scale=0.0, stream=None):
    from paged_util import attend, check_out, visible

    T, group = sum(rows), heads // c.kv
    start = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda")
    if q is None:
        q = queries(torch, T, heads, c.hd, c.dtype, seed)
    out = torch.full((T, heads, c.hd), float("nan"), dtype=c.dtype, device="cuda")
    ctx.paged_prefill(view(c), q, out, start, T, window=window, n_sink=sinks, scale=scale, stream=stream)
    ctx.check_device(stream)
    at = 0
    for s, (ln, r) in enumerate(zip(c.lens, rows)):
        ok = visible(torch.arange(ln - r, ln, device="cuda"), ln, window, sinks)
        k, v = c.rows(s, ln)
        for h in range(c.kv):
            o, a, sv, _ = attend(q[at:at + r, h * group:(h + 1) * group], k[:, h], v[:, h], ok, scale or c.hd ** -0.5)
            check_out(out[at:at + r, h * group:(h + 1) * group], o, a, sv, c.dtype)
        at += r
    return q, out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(PREFILL)))
def test_prefill(torch_, dtype, case):
    from paged_util import Cache

    heads, kv, hd, page, lens, rows, window, sinks = PREFILL[case]
    c = Cache(lens, kv, hd, page, dtype, seed=50 + case, order="heads" if case % 2 else "slots", table_extra=case % 3)
    blank(torch_, c, window, sinks, rows)
    ctx = make_ctx(heads, kv, hd, page, dtype)
    q, one = check_prefill(torch_, c, ctx, heads, rows, window, sinks, case)
    _, two = check_prefill(torch_, c, ctx, heads, rows, window, sinks, case, q=q)
    assert torch_.equal(one, two)
    ctx.close()


def test_prefill_rows_are_decodes(torch_):
    """Row r of a prefill sees what a decode at its position sees: the two kernels agree within both bounds."""
    from paged_util import Cache

    torch = torch_
    c = Cache([600], 4, 128, 16, "bf16", seed=70)
    ctx = make_ctx(32, 4, 128, 16)
    q, out = check_prefill(torch, c, ctx, 32, [600], 200, 4, 70)
    for r in (0, 1, 127, 128, 300, 599):
        c.len.fill_(r + 1)
        one = torch.empty((1, 32, 128), dtype=c.dtype, device="cuda")
        ctx.paged_decode(view(c), q[r:r + 1], one, window=200, n_sink=4)
        ctx.check_device()
        assert float((one[0].float() - out[r].float()).abs().max()) <= 2.0 ** -6
    ctx.close()


@pytest.mark.parametrize("window,sinks", [(0, 0), (64, 2)])
def test_prefill_nan_stays_with_the_rows_that_see_it(torch_, window, sinks):
    """A NaN or infinity in a key or value reaches the rows that see its position and no other."""
    from paged_util import Cache

    torch = torch_
    c = Cache([400, 200], 2, 128, 16, "bf16", seed=80)
    ctx = make_ctx(16, 2, 128, 16)
    rows = [400, 150]
    q, clean = check_prefill(torch, c, ctx, 16, rows, window, sinks, 80)
    start = torch.tensor([0, 400, 550], dtype=torch.int32, device="cuda")
    for pool, bad in ((c.v, float("nan")), (c.v, float("inf")), (c.k, float("nan"))):
        p, o = c.places(0, torch.tensor([250], device="cuda"))
        keep = pool[p, o].clone()
        pool[p, o] = bad
        out = torch.empty_like(clean)
        ctx.paged_prefill(view(c), q, out, start, 550, window=window, n_sink=sinks)
        ctx.check_device()
        sees = torch.zeros(550, dtype=torch.bool, device="cuda")
        sees[250:(250 + window if window else 400)] = True
        assert torch.equal(out[~sees], clean[~sees]) or \
            float((out[~sees].float() - clean[~sees].float()).abs().max()) <= 2.0 ** -6
        assert not torch.isfinite(out[sees].float()).all(dim=-1).any()
        pool[p, o] = keep
    ctx.close()


# ------------------------------------------------------------------ eviction
EVICT = [
    # kv, hd, page, lens, budget, sinks, recent
    (4, 128, 64, [4096], 1024, 4, 256),
    (4, 128, 16, [1, 0, 17, 300, 301, 1000, 299], 300, 4, 64),
    (1, 8, 1, [50, 3], 7, 1, 2),
    (2, 80, 3, [500, 100], 101, 0, 0),
    (3, 64, 32, [700], 20, 13, 7),         # sinks and recent are the whole budget
    (2, 128, 64, [3000, 2500], 2000, 0, 2000),
    (2, 64, 64, [900], 1, 0, 0),
    (8, 128, 128, [20000], 5000, 4, 512),
]


def weights_of(torch, kind, shape, seed):
    gen = torch.Generator(device="cuda").manual_seed(200 + seed)
    w = torch.exp(2 * torch.randn(shape, generator=gen, device="cuda"))
    if kind == "ties":
        w = torch.round(w * 2) / 2
    elif kind == "odd":  # NaN, zeros of both signs, infinities, negative values, subnormals
        pick = torch.randint(0, 8, shape, generator=gen, device="cuda")
        for i, x in enumerate((float("nan"), 0.0, -0.0, float("inf"), -float("inf"), -1.5, 1e-42)):
            w = torch.where(pick == i, torch.tensor(x, device="cuda"), w)
    elif kind == "same":
        w = torch.ones(shape, device="cuda")
    return w


def check_evicted(torch, c, before, w, kept, new_len, budget, sinks, recent, k, v, table, w_dst):
    from paged_util import evict_ref

    for s, n in enumerate(c.lens):
        m = min(n, budget)
        assert int(new_len[s]) == m
        for h in range(c.kv):
            want = evict_ref(w[s, h, :n], n, budget, sinks, recent)
            assert kept[s, h].tolist() == want + [-1] * (budget - m), (s, h)
            if m:
                j = torch.arange(m, device="cuda")
                p, o = table[s].long()[j // c.page], j % c.page
                src = torch.tensor(want, device="cuda")
                bk, bv = before[s]
                assert torch.equal(k[p, o, h], bk[src, h]) and torch.equal(v[p, o, h], bv[src, h])
            if w_dst is not None:
                got = w_dst[s, h].clone()
                assert torch.equal(got[:m].view(torch.int32), w[s, h, want].view(torch.int32))
                assert not got[m:].any()


@pytest.mark.parametrize("kind", ["plain", "ties", "odd", "same"])
@pytest.mark.parametrize("case", range(len(EVICT)))
def test_evict(torch_, kind, case):
    from paged_util import Cache

    torch = torch_
    kv, hd, page, lens, budget, sinks, recent = EVICT[case]
    c = Cache(lens, kv, hd, page, "bf16" if case % 2 else "f16", seed=case, order="heads" if case % 2 else "slots")
    ctx = make_ctx(4 * kv, kv, hd, page, "bf16" if case % 2 else "f16", max_len=max(lens))
    n = len(lens)
    w = weights_of(torch, kind, (n, kv, max(lens + [budget]) + 5), case)
    before = [tuple(x.clone() for x in c.rows(s, ln)) for s, ln in enumerate(lens)]
    per = -(-budget // page)
    to_table = torch.randperm(n * per, device="cuda").to(torch.int32).reshape(n, per)
    to_k, to_v = (torch.zeros((n * per, page, kv, hd), dtype=c.dtype, device="cuda") for _ in range(2))
    kept = torch.full((n, kv, budget), 77, dtype=torch.int32, device="cuda")
    new_len = torch.full((n,), 77, dtype=torch.int32, device="cuda")
    w_dst = torch.full_like(w, 9.0)
    dst = obsmoe.PagedKV(to_k, to_v, to_table, new_len)
    ctx.paged_evict(view(c), dst, w, w_dst, budget, n_sink=sinks, n_recent=recent, kept=kept, new_len=new_len)
    ctx.check_device()
    check_evicted(torch, c, before, w, kept, new_len, budget, sinks, recent, to_k, to_v, to_table, w_dst)
    # in place, the weights too: the same outcome
    if all(-(-min(ln, budget) // page) <= c.table.shape[1] for ln in lens) and c.table.shape[1] * page >= budget:
        w2, kept2, len2 = w.clone(), torch.empty_like(kept), torch.empty_like(new_len)
        ctx.paged_evict(view(c), view(c), w2, w2, budget, n_sink=sinks, n_recent=recent, kept=kept2, new_len=len2)
        ctx.check_device()
        assert torch.equal(kept, kept2) and torch.equal(new_len, len2)
        check_evicted(torch, c, before, w, kept2, len2, budget, sinks, recent, c.k, c.v, c.table, w2)
    ctx.close()


# -------------------------------------------------- streams, graphs, layouts
def test_other_stream_and_graph(torch_):
    """Calls on a side stream, and a captured decode whose lengths grow between replays."""
    from paged_util import Cache

    torch = torch_
    c = Cache([500, 260], 4, 128, 64, "bf16", seed=90)
    ctx = make_ctx(32, 4, 128, 64, weights=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check_decode(torch, c, ctx, 32, 0, 0, 90, stream=side)
        check_decode(torch, c, ctx, 32, 100, 4, 90, weights=True, stream=side)
        check_prefill(torch, c, ctx, 32, [100, 200], 0, 0, 90, stream=side)
    torch.cuda.synchronize()
    q = queries(torch, 2, 32, 128, c.dtype, 91)
    out = torch.empty_like(q)
    kv = view(c)
    c.len.copy_(torch.tensor([400, 7], dtype=torch.int32))
    ctx.paged_decode(kv, q, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        ctx.paged_decode(kv, q, out, stream=side)
    for lens in ([400, 7], [401, 8], [500, 260], [0, 1]):
        c.len.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        ctx.paged_decode(kv, q, out)
        ctx.check_device()
        assert torch.equal(got, out)
    ctx.close()


def test_query_rows_with_a_stride_and_table_slices(torch_):
    from paged_util import Cache, attend, check_out, visible

    torch = torch_
    c = Cache([300, 45, 130], 2, 64, 16, "f16", seed=95)
    ctx = make_ctx(8, 2, 64, 16, "f16")
    wide = queries(torch, 3, 12, 64, c.dtype, 95)     # q | k | v of a fused projection
    q = wide[:, :8]
    out = torch.empty((3, 8, 64), dtype=c.dtype, device="cuda")
    table = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
    table[:, : c.table.shape[1]] = c.table
    kv = obsmoe.PagedKV(c.k, c.v, table[:, : c.table.shape[1]], c.len)
    ctx.paged_decode(kv, q, out, scale=0.3)
    ctx.check_device()
    for s, n in enumerate(c.lens):
        k, v = c.rows(s, n)
        for h in range(2):
            o, a, sv, _ = attend(q[s:s + 1, 4 * h:4 * h + 4], k[:, h], v[:, h], visible(torch.tensor([n - 1], device="cuda"), n, 0, 0), 0.3)
            check_out(out[s:s + 1, 4 * h:4 * h + 4], o, a, sv, c.dtype)
    ctx.close()


def test_offsets_beyond_32_bits(torch_):
    """Pages whose elements lie past 2^32 in the pool (decode, prefill, append, evict)."""
    from paged_util import Cache

    torch = torch_
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    page, kv, hd = 64, 4, 128
    pages = (1 << 32) // (page * kv * hd) + 8
    big_k = torch.empty((pages, page, kv, hd), dtype=torch.bfloat16, device="cuda")
    big_v = torch.empty_like(big_k)
    c = Cache([200, 70], kv, hd, page, "bf16", seed=97)
    n = c.k.shape[0]
    assert n <= 8
    big_k[-n:], big_v[-n:] = c.k, c.v
    c.table += pages - n
    c.k, c.v = big_k, big_v
    ctx = make_ctx(32, kv, hd, page)
    check_decode(torch, c, ctx, 32, 0, 0, 97)
    check_prefill(torch, c, ctx, 32, [200, 9], 0, 0, 97)
    rows = queries(torch, 2, 2 * kv, hd, c.dtype, 98)
    ctx.paged_append(view(c), rows[:, :kv], rows[:, kv:], torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                     torch.tensor([199, 3], dtype=torch.int32, device="cuda"), 2)
    check_decode(torch, c, ctx, 32, 50, 4, 97)
    before = [tuple(x.clone() for x in c.rows(s, ln)) for s, ln in enumerate(c.lens)]
    w = weights_of(torch, "plain", (2, kv, 200), 97)
    kept = torch.empty((2, kv, 90), dtype=torch.int32, device="cuda")
    new_len = torch.empty((2,), dtype=torch.int32, device="cuda")
    w2 = w.clone()
    ctx.paged_evict(view(c), view(c), w2, w2, 90, n_sink=4, n_recent=20, kept=kept, new_len=new_len)
    ctx.check_device()
    check_evicted(torch, c, before, w, kept, new_len, 90, 4, 20, c.k, c.v, c.table, w2)
    ctx.close()
    del big_k, big_v, c
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ refusals
def test_device_refuses_bad_tables_and_lengths(torch_):
    """A page id outside the pool, a length beyond the table and a row outside the cache are refused by the
    kernels' bounds checks and reported; the context stays usable."""
    from paged_util import Cache

    torch = torch_
    c = Cache([200, 70], 2, 64, 16, "bf16", seed=99)
    ctx = make_ctx(8, 2, 64, 16, weights=True, max_len=400)
    q, out = queries(torch, 2, 8, 64, c.dtype, 99), torch.empty((2, 8, 64), dtype=c.dtype, device="cuda")
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    w = torch.zeros((2, 2, 300), device="cuda")
    kept = torch.empty((2, 2, 50), dtype=torch.int32, device="cuda")
    new_len = torch.empty((2,), dtype=torch.int32, device="cuda")
    good = c.table.clone()

    def calls():
        yield lambda: ctx.paged_decode(view(c), q, out)
        yield lambda: ctx.paged_decode(view(c), q, out, weights=w)
        yield lambda: ctx.paged_prefill(view(c), q, out, start, 2)
        yield lambda: ctx.paged_evict(view(c), view(c), w.clone(), None, 50, kept=kept, new_len=new_len)

    for bad in (-1, c.k.shape[0], 1 << 30, -(1 << 31)):
        c.table.copy_(good)
        c.table[0, 0] = bad
        for call in calls():
            call()
            with pytest.raises(obsmoe.ObsError, match="page id"):
                ctx.check_device()
    c.table.copy_(good)
    for bad in (c.table.shape[1] * 16 + 1, 401, 1 << 30, -3):
        c.len[0] = bad
        for call in calls():
            call()
            with pytest.raises(obsmoe.ObsError, match="length"):
                ctx.check_device()
    c.len[0] = 200
    rows = queries(torch, 1, 4, 64, c.dtype, 1)
    for s, j in ((2, 0), (-1, 0), (0, -1), (0, c.table.shape[1] * 16)):
        ctx.paged_append(view(c), rows[:, :2], rows[:, 2:], torch.tensor([s], dtype=torch.int32, device="cuda"),
                         torch.tensor([j], dtype=torch.int32, device="cuda"), 1)
        with pytest.raises(obsmoe.ObsError, match="outside the KV caches"):
            ctx.check_device()
    for bad in ([0, 1, 1], [0, 3, 2], [1, 1, 2]):  # rows of no sequence
        ctx.paged_prefill(view(c), q, out, torch.tensor(bad, dtype=torch.int32, device="cuda"), 2)
        with pytest.raises(obsmoe.ObsError, match="outside the KV caches"):
            ctx.check_device()
    check_decode(torch, c, ctx, 8, 0, 0, 99)
    ctx.close()


def test_host_refusals(torch_):
    from paged_util import Cache

    torch = torch_
    c = Cache([200, 70], 2, 64, 16, "bf16", seed=99)
    ctx = obsmoe.MoeContext(obsmoe.MoeShape(2048, 256, 16, 4, n_layers=1, max_tokens=1), 0)
    q, out = queries(torch, 2, 8, 64, c.dtype, 99), torch.empty((2, 8, 64), dtype=c.dtype, device="cuda")
    kv = view(c)
    lib = obsmoe.lib()

    def decode(view_=kv, q_=None, stride=512, out_=None, window=0, sinks=0, scale=0.0, w=None, ws=0):
        ctx._chk(lib.obs_paged_decode(ctx._h, view_.ref if view_ else None, q.data_ptr() if q_ is None else q_, stride,
                                      out.data_ptr() if out_ is None else out_, window, sinks, scale, w, ws, None))

    with pytest.raises(obsmoe.ObsError, match="not initialised"):
        decode()
    for bad in (dict(n_kv_heads=3), dict(n_heads=34), dict(head_dim=136), dict(head_dim=12), dict(head_dim=0),
                dict(page_size=0), dict(page_size=1025), dict(max_seqs=0), dict(max_kv_len=0),
                dict(max_kv_len=(1 << 20) + 1)):
        with pytest.raises(obsmoe.ObsError, match="bad paged config"):
            ctx.paged_init(**{**dict(n_heads=8, n_kv_heads=2, head_dim=64, page_size=16), **bad})
    ctx.paged_init(n_heads=8, n_kv_heads=2, head_dim=64, page_size=16, max_seqs=2, max_kv_len=400)
    with pytest.raises(obsmoe.ObsError, match="already initialised"):
        ctx.paged_init(n_heads=8, n_kv_heads=2, head_dim=64, page_size=16)
    with pytest.raises(obsmoe.ObsError, match="null cache"):
        decode(view_=None)
    for kw, msg in ((dict(q_=0), "null"), (dict(out_=0), "null"), (dict(q_=q.data_ptr() + 2), "aligned"),
                    (dict(stride=516), "q_stride"), (dict(stride=504), "smaller than a row"), (dict(window=-1), "window"),
                    (dict(sinks=-1), "n_sink"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
                    (dict(scale=float("inf")), "scale"), (dict(w=out.data_ptr(), ws=400), "without room for weights")):
        with pytest.raises(obsmoe.ObsError, match=msg):
            decode(**kw)
    for field, value, msg in (("k", c.k.data_ptr() + 2, "aligned"), ("v", None, "null cache"), ("slot_stride", 65, "multiples"),
                              ("page_stride", -8, "negative"), ("n_seqs", 3, "n_seqs"), ("n_seqs", -1, "n_seqs"),
                              ("n_pages", 0, "n_pages"), ("table_pages", 0, "table_pages"), ("table_stride", 1, "table_stride")):
        bad = view(c)
        setattr(bad.view, field, value)
        with pytest.raises(obsmoe.ObsError, match=msg):
            decode(view_=bad)
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    with pytest.raises(obsmoe.ObsError, match="T out of range"):
        ctx._chk(lib.obs_paged_prefill(ctx._h, kv.ref, q.data_ptr(), 512, out.data_ptr(), start.data_ptr(), -1, 0, 0, 0.0, None))
    with pytest.raises(obsmoe.ObsError, match="null"):
        ctx._chk(lib.obs_paged_prefill(ctx._h, kv.ref, q.data_ptr(), 512, out.data_ptr(), None, 2, 0, 0, 0.0, None))
    w = torch.zeros((2, 2, 208), device="cuda")
    kept, new_len = torch.empty((2, 2, 500), dtype=torch.int32, device="cuda"), torch.empty((2,), dtype=torch.int32, device="cuda")
    for kw, msg in ((dict(budget=0), "budget"), (dict(n_sink=40, n_recent=30), "budget"), (dict(n_sink=-1), "budget"),
                    (dict(budget=209), "no room"), (dict(new_len=c.len), "alias"), (dict(kept=None), "null"),
                    (dict(weights_dst=torch.zeros((2, 2, 40), device="cuda"), weights=torch.zeros((2, 2, 40), device="cuda")), "w_stride")):
        args = {**dict(weights=w, weights_dst=None, budget=50, n_sink=0, n_recent=0, kept=kept, new_len=new_len), **kw}
        with pytest.raises(obsmoe.ObsError, match=msg):
            ctx.paged_evict(kv, kv, args["weights"], args["weights_dst"], args["budget"], n_sink=args["n_sink"],
                            n_recent=args["n_recent"], kept=args["kept"], new_len=args["new_len"])
    for bad_q in (q.float(), q[:1], q.transpose(1, 2)):
        with pytest.raises(ValueError):
            ctx.paged_decode(kv, bad_q, out)
    with pytest.raises(ValueError):
        ctx.paged_decode(obsmoe.PagedKV(c.k[:, :8], c.v[:, :8], c.table, c.len), q, out)
    with pytest.raises(ValueError):
        obsmoe.PagedKV(c.k, c.v.transpose(1, 2), c.table, c.len)
    ctx.paged_decode(kv, q, out)
    ctx.check_device()
    ctx.close()


# ------------------------------------------------- values at the types' ends
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd,ln", [(8, 1, 128, 20), (8, 1, 128, 9000), (6, 2, 64, 700), (32, 2, 120, 300)])
def test_infinite_values_stay_in_their_dimension(torch_, dtype, heads, kv, hd, ln):
    """p v_j of a visible infinity is that infinity, of a NaN NaN, for the queries that see it and in its dimension
    alone; both infinities in one dimension give NaN."""
    from paged_util import Cache, attend, check_out, visible

    torch = torch_
    group, inf = heads // kv, float("inf")
    c = Cache([ln, 40], kv, hd, 16, dtype, seed=90)
    ctx = make_ctx(heads, kv, hd, 16, dtype, max_len=9000)
    rows = 3
    q = queries(torch, 2 * rows, heads, hd, c.dtype, 90)
    start = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device="cuda")
    bad = {(5, 0): inf, (6, 3): -inf, (7, 4): float("nan"), (8, 7): inf, (9, 7): -inf}
    want = {0: inf, 3: -inf, 4: float("nan"), 7: float("nan")}
    for (j, d), x in bad.items():
        p, o = c.places(0, torch.tensor([j], device="cuda"))
        c.v[p, o, kv - 1, d] = x
    out = torch.zeros((2 * rows, heads, hd), dtype=c.dtype, device="cuda")
    ctx.paged_prefill(view(c), q, out, start, 2 * rows)
    last = torch.zeros((2, heads, hd), dtype=c.dtype, device="cuda")
    ctx.paged_decode(view(c), q[rows - 1::rows].contiguous(), last)
    ctx.check_device()
    for got, at in ((out, (0, rows)), (last, (0, 1))):
        n = rows if got is out else 1
        for s, length in enumerate(c.lens):
            ok = visible(torch.arange(length - n, length, device="cuda"), length, 0, 0)
            k, v = c.rows(s, length)
            for h in range(kv):
                sees = s == 0 and h == kv - 1
                mine = got[at[s]:at[s] + n, h * group:(h + 1) * group].clone()
                qs = q[rows * s + rows - n:rows * (s + 1), h * group:(h + 1) * group]
                vv = v[:, h].clone()
                if sees:
                    for d, x in want.items():
                        assert torch.equal(mine[..., d].float().nan_to_num(nan=7.0, posinf=8.0, neginf=9.0),
                                           torch.full_like(mine[..., d], 7.0 if x != x else 8.0 if x > 0 else 9.0).float()), d
                        mine[..., d], vv[:, d] = 0.0, 0.0
                o, a, sv, _ = attend(qs, k[:, h], vv, ok, hd ** -0.5)
                check_out(mine, o, a, sv, c.dtype)
    ctx.close()


def test_f16_many_small_probabilities(torch_):
    """A first position whose score lies 26 powers of two above 65535 equal ones, in heads enough that no CTA sees
    few of them: what the small ones add up to is there.  The bound of paged_util with its term for p below the
    smallest normal f16, 2^-24 S, as it is for p multiplied by 2^15 (decode) and 2^7 (prefill)."""
    from paged_util import Cache, attend, visible, U

    torch = torch_
    ln, kv, hd = 65536, 160, 8
    c = Cache([ln], kv, hd, 64, "f16", seed=91)
    j = torch.arange(ln, device="cuda")
    k, v = torch.zeros_like(c.kd[0]), c.vd[0].abs()
    k[0], v[0] = 18.0 / hd, 0.0
    c.put(0, j, k, v)
    ctx = make_ctx(kv, kv, hd, 64, "f16", max_len=ln)
    q = torch.ones((1, kv, hd), dtype=c.dtype, device="cuda")
    start = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    one, two = torch.zeros_like(q), torch.zeros_like(q)
    ctx.paged_decode(view(c), q, one, scale=1.0)
    ctx.paged_prefill(view(c), q, two, start, 1, scale=1.0)
    ctx.check_device()
    ok, u = visible(j[-1:], ln, 0, 0), U[c.dtype]
    for h in range(kv):
        o, a, sv, _ = attend(q[:, h:h + 1], k[:, h], v[:, h], ok, 1.0)
        for got, shift in ((one, 15), (two, 7)):
            # (the output itself may lie below the smallest normal f16: 2^-25)
            bound = u * o.abs() + (u + 1e-4) * a + 2.0 ** (-24 - shift) * sv + 2.0 ** -25
            worst = float(((got[:, h:h + 1].double() - o).abs() / bound).max())
            assert worst <= 1.0, f"head {h}, shift {shift}: {worst:.3f} times the bound"
    ctx.close()
