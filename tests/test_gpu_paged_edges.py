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
