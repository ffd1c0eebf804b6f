"""The attention block over a paged cache (obs_paged_attn_forward) against the dense
one on the same weights, and the example's serving loop: prompts in chunks, decode
steps with weights, eviction in place."""
import os
import sys

import numpy as np
import pytest

import obsmoe
import oracle as O
from parity_util import REL, dev, host, rel_err

pytestmark = pytest.mark.gpu

H, NQ, NKV, HD, THETA, PAGE = 2048, 32, 4, 128, 1e7, 16
MAX_SEQ, N_SEQS = 256, 3


@pytest.fixture(scope="module")
def pair(cuda):
    """One context with a dense cache per sequence and a paged cache beside it."""
    torch = cuda
    ctx = obsmoe.MoeContext(obsmoe.MoeShape(H, 256, 16, 4, n_layers=1, max_tokens=64), 0)
    ctx.attn_init(NQ, NKV, HD, MAX_SEQ, N_SEQS, THETA)
    ctx.load_attn(0, O.synth_attn(seed=9, layer=0, H=H, nq=NQ, nkv=NKV, hd=HD))
    ctx.paged_init(NQ, NKV, HD, PAGE, max_seqs=N_SEQS, max_kv_len=MAX_SEQ, weights=True)
    per = MAX_SEQ // PAGE
    k, v = (torch.full((N_SEQS * per, PAGE, NKV, HD), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in "kv")
    table = torch.randperm(N_SEQS * per).to(torch.int32).reshape(N_SEQS, per).cuda()
    length = torch.zeros(N_SEQS, dtype=torch.int32, device="cuda")
    yield torch, ctx, obsmoe.PagedKV(k, v, table, length)
    ctx.close()


def test_paged_block_equals_the_dense_block(pair):
    torch, ctx, kv = pair
    k, v, table, length = kv.tensors
    lens = [0] * N_SEQS
    # a prefill of two sequences at once, a chunk of one, decode steps of all three
    steps = [([40, 24, 0], True), ([0, 9, 55], True)] + [([1, 1, 1], False)] * 4
    for i, (counts, prefill) in enumerate(steps):
        T = sum(counts)
        seq = dev(torch, np.repeat(np.arange(N_SEQS), counts).astype(np.int32))
        pos = dev(torch, np.concatenate([np.arange(a, a + c) for a, c in zip(lens, counts)]).astype(np.int32))
        lens = [a + c for a, c in zip(lens, counts)]
        length.copy_(torch.tensor(lens, dtype=torch.int32))
        xh = O.synth_x(300 + i, 0, T, H)
        x = dev(torch, xh)
        dense, paged = (torch.empty((T, H), dtype=torch.int16, device="cuda") for _ in range(2))
        ctx.attn_forward(0, x, dense, T, seq, pos)
        start = dev(torch, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)) if prefill else None
        ctx.paged_attn_forward(0, kv, x, paged, T, seq, pos, pos, start)
        ctx.check_device()
        a, b, xf = host(dense, np.uint16), host(paged, np.uint16), O.bf16_to_f32(xh)
        # both round the o projection and then x + o to bf16: where fp32 sums in another order cross a
        # rounding boundary, each rounding moves by one unit in the last place, 2^-7 of its value at most;
        # the sums themselves (attention rows that differ by such a unit here and there) by far less
        ya, yb = O.bf16_to_f32(a), O.bf16_to_f32(b)
        o = np.abs(ya - xf)
        assert np.all(np.abs(ya - yb) <= 2.0 ** -7 * (np.abs(ya) + o) + 1e-3 * o.max()), i
    # the same rows in both caches, bit for bit
    for s, n in enumerate(lens):
        kc, vc = (torch.empty((NKV, n, HD), dtype=torch.int16, device="cuda") for _ in "kv")
        ctx.kv_read(0, s, 0, n, kc, vc)
        j = torch.arange(n, device="cuda")
        for pool, c in ((k, kc), (v, vc)):
            rows = pool[table[s].long()[j // PAGE], j % PAGE].transpose(0, 1).contiguous()
            assert torch.equal(rows.view(torch.int16), c)


def test_paged_block_refusals(pair):
    torch, ctx, kv = pair
    x, y = (torch.zeros((65, H), dtype=torch.int16, device="cuda") for _ in "xy")
    i = torch.zeros(65, dtype=torch.int32, device="cuda")
    for call, msg in ((lambda: ctx.paged_attn_forward(0, kv, x, y, 65, i, i, i, i), "T out of range"),
                      (lambda: ctx.paged_attn_forward(0, kv, x, x, 3, i, i, i), "alias"),
                      (lambda: ctx.paged_attn_forward(1, kv, x, y, 3, i, i, i), "layer out of range"),
                      (lambda: ctx.paged_attn_forward(0, kv, x, y, 2, i, i, i), "one token per sequence"),
                      (lambda: ctx.paged_attn_forward(0, kv, x, y, 3, i, i, None), "null"),
                      (lambda: ctx.paged_attn_forward(0, kv, x, y, 3, i, i, i, i, weights=torch.zeros((3, NKV, 256), device="cuda")),
                       "decode steps only")):
        with pytest.raises(obsmoe.ObsError, match=msg):
            call()
    other = obsmoe.MoeContext(obsmoe.MoeShape(H, 256, 16, 4, n_layers=1, max_tokens=4), 0)
    with pytest.raises(obsmoe.ObsError, match="attention not initialised"):
        other.paged_attn_forward(0, kv, x, y, 3, i, i, i)
    other.attn_init(NQ, NKV, HD, 32, 1, THETA)
    other.load_attn(0, O.synth_attn(seed=9, layer=0, H=H, nq=NQ, nkv=NKV, hd=HD))
    with pytest.raises(obsmoe.ObsError, match="paged cache not initialised"):
        other.paged_attn_forward(0, kv, x, y, 3, i, i, i)
    other.paged_init(NQ, NKV, HD, PAGE, dtype="f16")
    with pytest.raises((obsmoe.ObsError, ValueError)):
        other.paged_attn_forward(0, kv, x, y, 3, i, i, i)
    other.close()


@pytest.mark.parametrize("kw,msg", [(dict(window=-1), "negative"), (dict(n_sink=-1), "negative"),
                                    (dict(weights=True), "without room for weights")])
def test_a_refused_step_appends_nothing(cuda, kw, msg):
    torch = cuda
    ctx = obsmoe.MoeContext(obsmoe.MoeShape(H, 256, 16, 4, n_layers=1, max_tokens=4), 0)
    ctx.attn_init(NQ, NKV, HD, 32, 1, THETA)
    ctx.load_attn(0, O.synth_attn(seed=9, layer=0, H=H, nq=NQ, nkv=NKV, hd=HD))
    ctx.paged_init(NQ, NKV, HD, PAGE, max_seqs=1, max_kv_len=32)
    k, v = (torch.zeros((2, PAGE, NKV, HD), dtype=torch.bfloat16, device="cuda") for _ in "kv")
    zero, one = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    kv = obsmoe.PagedKV(k, v, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), one)
    x = dev(torch, O.synth_x(5, 0, 1, H))
    y = torch.empty_like(x)
    if "weights" in kw:
        kw = dict(weights=torch.zeros((1, NKV, 32), device="cuda"))
    with pytest.raises(obsmoe.ObsError, match=msg):
        ctx.paged_attn_forward(0, kv, x, y, 1, zero, zero, zero, **kw)
    torch.cuda.synchronize()
    assert not k.any() and not v.any()
    ctx.paged_attn_forward(0, kv, x, y, 1, zero, zero, zero)
    ctx.check_device()
    assert k[0, 0].any() and v[0, 0].any()
    ctx.close()


@pytest.fixture(scope="module")
def example(cuda):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import paged_session

    return paged_session


def test_example_chunked_prefill_equals_one_prefill(cuda, example):
    """The residual stream of the prompts' last tokens does not depend on how the prompts were cut into chunks
    (beyond the order of fp32 sums in the attention, rounded to bf16 in each layer)."""
    torch = cuda
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, example.VOCAB, n).tolist() for n in (45, 7, 12)]
    out = []
    for chunk in (64, 19):
        ctx = example.make_model(2, 64, 64, 3, seed=3)
        s = example.Session(torch, ctx, 2, 3, 64)
        got = []
        s.next_tokens = lambda x: got.append(x.clone())
        s.prefill(prompts, chunk)
        ctx.check_device()
        out.append(host(got[0].view(torch.int16), np.uint16))
        ctx.close()
    assert rel_err(out[1], out[0]) <= REL


def test_example_session_with_eviction(cuda, example):
    """The whole loop: every sequence gets its tokens, the caches stay within their budget, and a budget that
    nothing exceeds changes nothing."""
    lines = []
    out, held = example.run(steps=20, budget=64, lens=(100, 20, 70), log=lines.append)
    assert len({t for o in out for t in o}) > 10  # not one token over and over
    assert [len(o) for o in out] == [20, 20, 20] and all(0 <= t < example.VOCAB for o in out for t in o)
    assert any("evicted" in line for line in lines)
    assert max(held) <= 64 + 8
    whole, held = example.run(steps=20, budget=0, lens=(100, 20, 70), log=lines.append)
    roomy, held2 = example.run(steps=20, budget=120, lens=(100, 20, 70), log=lines.append)
    assert whole == roomy and held == held2 == [119, 39, 89]
    # the short sequence fits the small budget: the others' evictions do not touch it
    assert out[1] == whole[1]
