"""The paged cache where a value, a position or a size is out of the ordinary: infinities among
many rows, refused tokens, more sequences than a warp has lanes, caches longer than a cluster
holds.  References and bounds are paged_util's."""
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


def coded(x):
    """Finite values to 0, the others to a number for each kind: comparable."""
    return x.float().nan_to_num(nan=7.0, posinf=8.0, neginf=9.0).where(~x.float().isfinite(), 0.0)


# ------------------------------------------------------ infinities among many rows
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd,rows,window", [(32, 4, 128, 700, 0), (32, 4, 128, 700, 100), (12, 12, 64, 1800, 0),
                                                     (24, 8, 80, 900, 200)])
def test_infinities_of_a_prompt_reach_the_rows_that_see_them(torch_, dtype, heads, kv, hd, rows, window):
    """Whole prompts (no split): infinities and a NaN in single dimensions of V.  In every row the dimensions that
    see one hold it, whichever lane stored the row first; all the others hold what the formula gives."""
    from paged_util import Cache, attend, check_out, visible

    torch = torch_
    group, inf, nan = heads // kv, float("inf"), float("nan")
    c = Cache([rows], kv, hd, 16, dtype, seed=110)
    ctx = make_ctx(heads, kv, hd, 16, dtype)
    q = queries(torch, rows, heads, hd, c.dtype, 110)
    bad = {(0, 1): inf, (130, 1): inf, (250, 2): -inf, (251, 6): inf, (333, 6): -inf, (500, 7): nan, (500, hd - 1): inf}
    for (j, d), x in bad.items():
        p, o = c.places(0, torch.tensor([j], device="cuda"))
        c.v[p, o, kv - 1, d] = x
    out = torch.full((rows, heads, hd), 3.0, dtype=c.dtype, device="cuda")
    start = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    ctx.paged_prefill(view(c), q, out, start, rows, window=window)
    ctx.check_device()
    pos = torch.arange(rows, device="cuda")
    ok = visible(pos, rows, window, 0)
    k, v = c.rows(0, rows)
    for h in range(kv):
        mine, vv = out[:, h * group:(h + 1) * group].clone(), v[:, h].clone()
        if h == kv - 1:
            plus, minus = (torch.zeros((rows, hd), dtype=torch.bool, device="cuda") for _ in "pm")
            for (j, d), x in bad.items():
                if x != -inf:
                    plus[:, d] |= ok[:, j]
                if x != inf:
                    minus[:, d] |= ok[:, j]
                vv[j, d] = 0.0
            code = torch.where(plus & minus, 7.0, torch.where(plus, 8.0, torch.where(minus, 9.0, 0.0)))
            want = code[:, None].expand_as(mine)
            assert torch.equal(coded(mine), want)
            mine = mine.where(want == 0, 0.0)
        o, a, sv, _ = attend(q[:, h * group:(h + 1) * group], k[:, h], vv, ok, hd ** -0.5)
        if h == kv - 1:
            o, a = o.where(want == 0, 0.0), a.where(want == 0, 0.0)
        check_out(mine, o, a, sv, c.dtype)
    ctx.close()


# ------------------------------------------------------------------ refused tokens
@pytest.mark.parametrize("prefill", [False, True])
def test_a_refused_token_leaves_the_cache_as_it_was(torch_, prefill):
    """A token whose position lies past the RoPE table, with a slot that the cache has: nothing is appended for it,
    and what the call gives does not depend on what an earlier call left in the context."""
    import oracle as O
    from parity_util import dev

    torch = torch_
    H, nq, nkv, hd, max_seq, page = 2048, 32, 4, 128, 32, 16
    ctx = obsmoe.MoeContext(obsmoe.MoeShape(H, 256, 16, 4, n_layers=1, max_tokens=8), 0)
    ctx.attn_init(nq, nkv, hd, max_seq, 1, 1e7)
    ctx.load_attn(0, O.synth_attn(seed=9, layer=0, H=H, nq=nq, nkv=nkv, hd=hd))
    ctx.paged_init(nq, nkv, hd, page, max_seqs=2, max_kv_len=64)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.arange(8, dtype=torch.int32, device="cuda").reshape(2, 4)
    k, v = (torch.full((8, page, nkv, hd), 0.5, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    kv = obsmoe.PagedKV(k, v, table, i32(4, 4))
    start = i32(0, 1, 2) if prefill else None
    x = dev(torch, O.synth_x(70, 0, 2, H))
    for bad in (max_seq, max_seq + 5, -1, 1 << 30):
        outs = []
        for before in (71, 72):  # what the context's scratch holds
            y = torch.empty((2, H), dtype=torch.int16, device="cuda")
            ctx.paged_attn_forward(0, kv, dev(torch, O.synth_x(before, 0, 2, H)), y, 2, i32(0, 1), i32(3, 3), i32(3, 3), start)
            ctx.check_device()
            k[:, 3], v[:, 3] = 0.25, 0.75
            ctx.paged_attn_forward(0, kv, x, y, 2, i32(0, 1), i32(3, bad), i32(3, 3), start)
            with pytest.raises(obsmoe.ObsError, match="outside the KV caches"):
                ctx.check_device()
            # sequence 1's slot (page 4) as it was, sequence 0's written
            assert bool((k[4, 3] == 0.25).all()) and bool((v[4, 3] == 0.75).all())
            assert not bool((k[0, 3] == 0.25).all()) and not bool((v[0, 3] == 0.75).all())
            outs.append(y)
        assert torch.equal(*outs)
    ctx.close()


# ------------------------------------------- more sequences than a warp has lanes
MANY = [
    # heads, kv, hd, page, sequences, window, sinks
    (8, 2, 64, 16, 33, 0, 0),
    (32, 4, 128, 64, 40, 0, 0),
    (6, 2, 128, 16, 600, 0, 0),       # several sequences per thread of the search
    (8, 1, 64, 16, 1100, 20, 3),
]


def many(torch, case):
    """Lengths and new rows of many short sequences: some without rows, some without positions, some with a history."""
    rng = np.random.default_rng(case)
    n = MANY[case][4]
    rows = rng.integers(0, 40, n)
    rows[::7] = 0
    rows[n // 2] = 90
    lens = rows + rng.integers(0, 60, n) * (rng.random(n) < 0.5)
    lens[3] = 0 if rows[3] == 0 else lens[3]
    return [int(x) for x in lens], [int(x) for x in rows]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(MANY)))
def test_prefill_of_many_sequences(torch_, dtype, case):
    from paged_util import Cache
    from test_gpu_paged import check_prefill

    heads, kv, hd, page, n, window, sinks = MANY[case]
    lens, rows = many(torch_, case)
    c = Cache(lens, kv, hd, page, dtype, seed=120 + case)
    ctx = make_ctx(heads, kv, hd, page, dtype, seqs=n)
    check_prefill(torch_, c, ctx, heads, rows, window, sinks, 120 + case)
    ctx.close()


def test_prefill_of_many_sequences_with_one_row_each(torch_):
    """As many rows as sequences and few of them: the split form, 40 sequences."""
    from paged_util import Cache
    from test_gpu_paged import check_prefill

    c = Cache([1 + 37 * i for i in range(40)], 1, 128, 16, "bf16", seed=130)
    ctx = make_ctx(8, 1, 128, 16, seqs=40)
    check_prefill(torch_, c, ctx, 8, [1] * 40, 0, 0, 130)
    ctx.close()


def test_prefill_of_many_sequences_refuses_bad_row_ranges(torch_):
    from paged_util import Cache
    from test_gpu_paged import check_prefill

    torch = torch_
    n = 40
    c = Cache([9] * n, 2, 64, 16, "bf16", seed=131)
    ctx = make_ctx(8, 2, 64, 16, seqs=n)
    q = queries(torch, 2 * n, 8, 64, c.dtype, 131)
    out = torch.empty_like(q)
    good = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32)
    for at, x in ((0, 1), (0, -2), (n, 2 * n - 1), (n, 2 * n + 3), (n // 2, 0), (n // 2, 1 << 30), (35, -5)):
        bad = good.clone()
        bad[at] = x
        ctx.paged_prefill(view(c), q, out, bad.cuda(), 2 * n)
        with pytest.raises(obsmoe.ObsError, match="outside the KV caches"):
            ctx.check_device()
    check_prefill(torch, c, ctx, 8, [2] * n, 0, 0, 131)
    ctx.close()


# ----------------------------------- eviction past what a cluster's shared memory holds
@pytest.mark.parametrize("kind", ["plain", "ties", "odd", "same"])
@pytest.mark.parametrize("lens,budget,sinks,recent", [([70000, 65540, 66000], 30000, 4, 500), ([140000, 9000], 20001, 0, 0),
                                                      ([300001], 299990, 3, 1000)])
def test_evict_long_caches(torch_, kind, lens, budget, sinks, recent):
    from paged_util import Cache
    from test_gpu_paged import check_evicted, weights_of

    torch = torch_
    kv, hd, page, n = 1, 8, 64, len(lens)
    c = Cache(lens, kv, hd, page, "bf16", seed=140)
    ctx = make_ctx(4, kv, hd, page, max_len=max(lens))
    w = weights_of(torch, kind, (n, kv, max(lens)), 140)
    before = [tuple(x.clone() for x in c.rows(s, ln)) for s, ln in enumerate(lens)]
    per = -(-budget // page)
    to_table = torch.randperm(n * per, device="cuda").to(torch.int32).reshape(n, per)
    to_k, to_v = (torch.zeros((n * per, page, kv, hd), dtype=c.dtype, device="cuda") for _ in range(2))
    kept, kept2 = (torch.full((n, kv, budget), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    new_len, len2 = (torch.full((n,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    w_dst = torch.full_like(w, 9.0)
    ctx.paged_evict(view(c), obsmoe.PagedKV(to_k, to_v, to_table, new_len), w, w_dst, budget, n_sink=sinks, n_recent=recent,
                    kept=kept, new_len=new_len)
    ctx.check_device()
    check_evicted(torch, c, before, w, kept, new_len, budget, sinks, recent, to_k, to_v, to_table, w_dst)
    w2 = w.clone()
    ctx.paged_evict(view(c), view(c), w2, w2, budget, n_sink=sinks, n_recent=recent, kept=kept2, new_len=len2)
    ctx.check_device()
    assert torch.equal(kept, kept2) and torch.equal(new_len, len2)
    check_evicted(torch, c, before, w, kept2, len2, budget, sinks, recent, c.k, c.v, c.table, w2)
    ctx.close()


def test_infinities_cost_a_bounded_time(torch_):
    """A prompt of 4096 with an infinity at its front, and with nothing but infinities in V: some milliseconds
    (2 and 9 when this was written, 0.16 without; row by row a prompt of 2048 took 25), and the values are right."""
    torch = torch_
    from paged_util import Cache

    inf, n = float("inf"), 4096
    c = Cache([n], 4, 128, 64, "bf16", seed=111)
    ctx = make_ctx(32, 4, 128, 64)
    q = queries(torch, n, 32, 128, c.dtype, 111)
    out = torch.empty_like(q)
    start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    p, o = c.places(0, torch.tensor([0], device="cuda"))
    c.v[p, o, :, 9] = inf
    for every in (False, True):
        if every:
            c.v.fill_(inf)
        ms = []
        for _ in range(3):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in "ab")
            a.record()
            ctx.paged_prefill(view(c), q, out, start, n)
            b.record()
            ctx.check_device()
            ms.append(a.elapsed_time(b))
        assert min(ms) < 40, ms
        assert bool((out[..., 9] == inf).all())
        assert bool((out == inf).all()) if every else bool(out[..., :9].isfinite().all() and out[..., 10:].isfinite().all())
    ctx.close()


# ------------------------------------------------------- values near bf16's largest
@pytest.mark.parametrize("heads,kv,hd,ln", [(8, 1, 128, 2), (32, 4, 128, 700), (8, 1, 64, 9000), (4, 2, 80, 130)])
@pytest.mark.parametrize("signs", [False, True])
def test_sums_past_fp32_of_values_that_are_not(torch_, heads, kv, hd, ln, signs):
    """Values of 1e38 to bf16's largest: a sum of p v over some positions lies past fp32's largest number before it
    is divided by the sum of p; the output does not."""
    from paged_util import Cache
    from test_gpu_paged import check_decode, check_prefill

    torch = torch_
    c = Cache([ln, 40], kv, hd, 16, "bf16", seed=112)
    big = torch.finfo(torch.bfloat16).max
    gen = torch.Generator(device="cuda").manual_seed(113)
    for s, n in enumerate(c.lens):
        j = torch.arange(n, device="cuda")
        x = big * (0.3 + 0.7 * torch.rand((n, kv, hd), generator=gen, device="cuda"))
        if signs:
            x = torch.where(torch.rand(x.shape, generator=gen, device="cuda") < 0.5, -x, x)
        x[:, :, 0] = big
        x[:, :, 1] = 1.0 + torch.rand((n, kv), generator=gen, device="cuda")  # and an ordinary dimension
        c.put(s, j, c.kd[s], x.to(c.dtype))
    ctx = make_ctx(heads, kv, hd, 16, max_len=9000, weights=True)
    check_decode(torch, c, ctx, heads, 0, 0, 112)
    check_decode(torch, c, ctx, heads, 0, 0, 112, weights=True)
    check_prefill(torch, c, ctx, heads, [min(ln, 3), 40], 0, 0, 112)
    check_prefill(torch, c, ctx, heads, [min(ln, 700), 1], 0, 0, 112)
    ctx.close()


# ------------------------------------------------------------------ messages
def test_a_timeout_names_the_kernel_that_waited(torch_):
    """A wait that ran out outside the expert GEMM (obs_probe_wait: one wait on a stamp that nothing writes, 10 ms)
    is not reported as one of the GEMM's."""
    ctx = obsmoe.MoeContext(obsmoe.MoeShape(2048, 256, 16, 4, n_layers=1, max_tokens=1), 0)
    ctx.set_wait_limit(10_000_000)
    ctx.probe_wait()
    with pytest.raises(obsmoe.ObsError, match="gave up") as e:
        ctx.check_device()
    assert e.value.status == 5 and "GEMM" not in str(e.value)
    ctx.check_device()
    ctx.close()


def test_out_may_not_overlap_q(torch_):
    """Rows with an infinity among their values are computed again from q, which must still be there."""
    from paged_util import Cache

    torch = torch_
    c = Cache([30, 40, 50], 2, 64, 16, "bf16", seed=150)
    ctx = make_ctx(8, 2, 64, 16, seqs=3, max_len=64)
    start = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    pool = queries(torch, 12, 8, 64, c.dtype, 150)
    for q, out in ((pool[:3], pool[:3]), (pool[:3], pool[2:5]), (pool[4:7], pool[2:5]), (pool[::4], pool[6:9])):
        with pytest.raises(obsmoe.ObsError, match="overlap"):
            ctx.paged_decode(view(c), q, out)
        with pytest.raises(obsmoe.ObsError, match="overlap"):
            ctx.paged_prefill(view(c), q, out, start, 3)
    want = torch.empty_like(pool[:3])
    for q, out in ((pool[:3], pool[3:6]), (pool[9:], pool[6:9])):
        ctx.paged_decode(view(c), q, out)
        ctx.paged_decode(view(c), q, want)
        ctx.check_device()
        assert torch.equal(out, want)
    ctx.close()


def test_no_sequences(torch_):
    """A batch of no sequences: tensors of no elements (no address), nothing to do."""
    torch = torch_
    ctx = make_ctx(8, 2, 64, 16, seqs=3, max_len=64, weights=True)
    k, v = (torch.full((4, 16, 2, 64), 0.5, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    i32 = dict(dtype=torch.int32, device="cuda")
    for pages in (4, 0):
        kv = obsmoe.PagedKV(k, v, torch.empty((0, pages), **i32), torch.empty(0, **i32))
        q, rows, w = torch.empty((0, 8, 64), dtype=k.dtype, device="cuda"), k[:0, 0], torch.empty((0, 2, 64), device="cuda")
        none = torch.empty(0, **i32)
        ctx.paged_append(kv, rows, rows, none, none, 0)
        ctx.paged_decode(kv, q, q.clone())
        ctx.paged_decode(kv, q, q.clone(), weights=w)
        ctx.paged_prefill(kv, q, q.clone(), torch.zeros(1, **i32), 0)
        ctx.paged_evict(kv, kv, w, w, 32, kept=torch.empty((0, 2, 32), **i32), new_len=torch.empty(0, **i32))
        ctx.check_device()
    assert bool((k == 0.5).all()) and bool((v == 0.5).all())
    ctx.close()


# --------------------------------------------------- the attention block without dense caches
def test_attention_block_without_dense_caches(torch_):
    """obs_attn_init with n_seqs 0: the paged block gives the same bits, the dense entry points refuse, and the
    caches' memory is not taken."""
    import oracle as O
    from parity_util import dev

    torch = torch_
    H, nq, nkv, hd, page, max_seq = 2048, 32, 4, 128, 16, 40960
    A = O.synth_attn(seed=9, layer=0, H=H, nq=nq, nkv=nkv, hd=hd)
    x = dev(torch, O.synth_x(80, 0, 5, H))
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    got, taken = [], []
    for n_seqs in (2, 0):
        before = torch.cuda.mem_get_info()[0]
        ctx = obsmoe.MoeContext(obsmoe.MoeShape(H, 256, 16, 4, n_layers=1, max_tokens=8), 0)
        ctx.attn_init(nq, nkv, hd, max_seq, n_seqs, 1e7)
        ctx.load_attn(0, A)
        ctx.paged_init(nq, nkv, hd, page, max_seqs=2, max_kv_len=64)
        taken.append(before - torch.cuda.mem_get_info()[0])
        k, v = (torch.zeros((8, page, nkv, hd), dtype=torch.bfloat16, device="cuda") for _ in "kv")
        kv = obsmoe.PagedKV(k, v, torch.arange(8, dtype=torch.int32, device="cuda").reshape(2, 4), i32(3, 2))
        y = torch.empty_like(x)
        ctx.paged_attn_forward(0, kv, x, y, 5, i32(0, 0, 0, 1, 1), i32(0, 1, 2, 7, 40959), i32(0, 1, 2, 0, 1), i32(0, 3, 5))
        ctx.check_device()
        got.append((y, k.view(torch.int16), v.view(torch.int16)))
        if n_seqs == 0:
            with pytest.raises(obsmoe.ObsError, match="no dense caches"):
                ctx.attn_forward(0, x, torch.empty_like(x), 1, i32(0), i32(0))
            with pytest.raises(obsmoe.ObsError, match="out of bounds"):
                ctx.kv_read(0, 0, 0, 1, k)
        ctx.close()
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert taken[0] - taken[1] >= 2 * 2 * nkv * max_seq * hd * 2
    with pytest.raises(obsmoe.ObsError, match="bad attention config"):
        ctx = obsmoe.MoeContext(obsmoe.MoeShape(H, 256, 16, 4, n_layers=1, max_tokens=8), 0)
        ctx.attn_init(nq, nkv, hd, 64, -1, 1e7)


# ----------------------------------------------------------- pages at every position
@pytest.mark.parametrize("page", [1, 3, 16, 63, 64, 1000, 1023, 1024])
def test_every_position_of_the_longest_sequence_lies_in_its_page(torch_, page):
    """append to each of 2^20 positions, in a mixed order; each row is where j / page and j % page say.  A decode
    over a window of one reads the last back."""
    torch = torch_
    n, hd = 1 << 20, 8
    pages = -(-n // page)
    gen = torch.Generator(device="cuda").manual_seed(page)
    table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)[None]
    k, v = (torch.zeros((pages, page, 1, hd), dtype=torch.bfloat16, device="cuda") for _ in "kv")
    slot = torch.randperm(n, generator=gen, device="cuda").to(torch.int32)
    # the position in three digits of 7 bits, which bf16 holds
    digits = torch.stack([slot >> s & 127 for s in (0, 7, 14)] + [slot * 0 + 1] * 5, dim=1).to(torch.bfloat16)
    ctx = make_ctx(1, 1, hd, page, seqs=1, max_len=n)
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    kv = obsmoe.PagedKV(k, v, table, length)
    ctx.paged_append(kv, digits.view(n, 1, hd), (-digits).view(n, 1, hd), torch.zeros_like(slot), slot, n)
    ctx.check_device()
    j = torch.arange(n, device="cuda")
    want = torch.stack([j >> s & 127 for s in (0, 7, 14)] + [j * 0 + 1] * 5, dim=1).to(torch.bfloat16)
    p, o = table[0].long()[j // page], j % page
    assert torch.equal(k[p, o, 0], want) and torch.equal(v[p, o, 0], -want)
    q = torch.ones((1, 1, hd), dtype=torch.bfloat16, device="cuda")
    for last in (n, n - 1, page, page + 1, 1, n // 2 + 1):
        length.fill_(last)
        out = torch.empty_like(q)
        ctx.paged_decode(kv, q, out, window=1)
        ctx.check_device()
        assert torch.equal(out[0, 0], -want[last - 1]), last
    ctx.close()


# ------------------------------------------------------------- eviction's mixed forms
@pytest.mark.parametrize("form", ["other pages of the same pools", "weights in place", "weights elsewhere", "no weights"])
def test_evict_mixed_forms(torch_, form):
    """Other pages of the same pools; rows to other pages with the weights in place; rows in place with the weights
    to another tensor or nowhere."""
    from paged_util import Cache
    from test_gpu_paged import check_evicted, weights_of

    torch = torch_
    kv, hd, page, lens, budget, sinks, recent = 2, 64, 16, [700, 90, 33], 65, 3, 20
    per = -(-budget // page)
    c = Cache(lens, kv, hd, page, "bf16", seed=160, pages_extra=len(lens) * per)
    ctx = make_ctx(4 * kv, kv, hd, page, max_len=max(lens))
    w = weights_of(torch, "ties", (len(lens), kv, max(lens)), 160)
    before = [tuple(x.clone() for x in c.rows(s, ln)) for s, ln in enumerate(lens)]
    i32 = dict(dtype=torch.int32, device="cuda")
    kept, new_len = torch.empty((len(lens), kv, budget), **i32), torch.empty(len(lens), **i32)
    held = {int(p) for s, ln in enumerate(lens) for p in c.table[s, :-(-ln // page)].tolist()}
    spare = torch.tensor([p for p in range(c.k.shape[0]) if p not in held], **i32)
    k, v, table, w_src, w_dst = c.k, c.v, c.table, w.clone(), torch.full_like(w, 9.0)
    if form == "other pages of the same pools":
        table = spare[:len(lens) * per].view(len(lens), per)
    elif form == "weights in place":
        k, v = torch.zeros_like(c.k), torch.zeros_like(c.v)
        w_dst = w_src
    elif form == "no weights":
        w_dst = None
    ctx.paged_evict(view(c), obsmoe.PagedKV(k, v, table, new_len), w_src, w_dst, budget, n_sink=sinks, n_recent=recent, kept=kept,
                    new_len=new_len)
    ctx.check_device()
    check_evicted(torch, c, before, w, kept, new_len, budget, sinks, recent, k, v, table, w_dst)
    if form in ("other pages of the same pools", "weights in place"):  # the source stays
        for s, ln in enumerate(lens):
            assert all(torch.equal(a, b) for a, b in zip(before[s], c.rows(s, ln)))
    if w_dst is not w_src:
        assert torch.equal(w_src.view(torch.int32), w.view(torch.int32))
    ctx.close()


def test_a_captured_step_serves_other_lengths(torch_):
    """append, prefill and evict in one graph on a side stream; replayed with other rows, lengths and row ranges."""
    from paged_util import Cache
    from test_gpu_paged import weights_of

    torch = torch_
    T, heads, kv, hd, page, budget = 60, 8, 2, 64, 16, 40
    c = Cache([200, 90, 130], kv, hd, page, "bf16", seed=170)
    ctx = make_ctx(heads, kv, hd, page)
    i32 = dict(dtype=torch.int32, device="cuda")
    w = weights_of(torch, "plain", (3, kv, 200), 170)
    rows, q = queries(torch, T, 2 * kv, hd, c.dtype, 170), queries(torch, T, heads, hd, c.dtype, 171)
    k, v = rows[:, :kv].contiguous(), rows[:, kv:].contiguous()
    seq, slot, start = torch.zeros(T, **i32), torch.zeros(T, **i32), torch.zeros(4, **i32)
    out, kept, new_len = torch.empty_like(q), torch.empty((3, kv, budget), **i32), torch.empty(3, **i32)
    per = -(-budget // page)
    to = [torch.zeros((3 * per, page, kv, hd), dtype=c.dtype, device="cuda") for _ in "kv"]
    w2, kv_ = torch.empty_like(w), view(c)
    dst = obsmoe.PagedKV(*to, torch.arange(3 * per, **i32).view(3, per), new_len)

    def step(stream=None):
        ctx.paged_append(kv_, k, v, seq, slot, T, stream=stream)
        ctx.paged_prefill(kv_, q, out, start, T, window=50, n_sink=2, stream=stream)
        ctx.paged_evict(kv_, dst, w, w2, budget, n_sink=2, n_recent=9, kept=kept, new_len=new_len, stream=stream)

    def results():
        ctx.check_device()
        r = [t.clone() for t in (out, kept, new_len, *to, w2)]
        for t in (out, kept, new_len, *to, w2):
            t.zero_()
        return r

    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    for counts, lens in (([20, 30, 10], [200, 90, 130]), ([0, 59, 1], [1, 77, 129]), ([60, 0, 0], [60, 0, 41])):
        seq.copy_(torch.repeat_interleave(torch.arange(3), torch.tensor(counts)))
        slot.copy_(torch.cat([torch.arange(n - m, n) for n, m in zip(lens, counts)]))
        start.copy_(torch.tensor(np.concatenate([[0], np.cumsum(counts)])))
        c.len.copy_(torch.tensor(lens))
        step()
        want = results()
        if lens[0] == 200:
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=side):
                step(side)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(want, results()))
    ctx.close()
