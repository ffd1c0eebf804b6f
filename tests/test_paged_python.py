"""What the Python calls of the paged cache refuse before they take an address, on the CPU: the
context and the cache are stand-ins, the library is never reached."""
from types import SimpleNamespace

import pytest

import obsmoe

torch = pytest.importorskip("torch")


class OnGpu:
    """A CPU tensor that says it lies on the GPU."""

    def __init__(self, t):
        self.t = t

    is_cuda = True

    def __getattr__(self, name):
        return getattr(self.t, name)

    def __getitem__(self, i):
        return self.t[i]


@pytest.fixture()
def parts(monkeypatch):
    ctx = object.__new__(obsmoe.MoeContext)
    ctx._h, ctx.shape, calls = None, obsmoe.MoeShape(hidden=64), []
    library = SimpleNamespace(**{n: (lambda *a, n=n: calls.append(n) or 0) for n in obsmoe.EXPORTS})
    monkeypatch.setattr(obsmoe, "lib", lambda: library)
    monkeypatch.setattr(obsmoe, "_LIB", None)
    ctx.paged_init(4, 2, 8, 4)
    calls.clear()
    k, v = (OnGpu(torch.zeros((6, 4, 2, 8), dtype=torch.bfloat16)) for _ in "kv")
    kv = obsmoe.PagedKV(k, v, OnGpu(torch.zeros((3, 2), dtype=torch.int32)), OnGpu(torch.zeros(3, dtype=torch.int32)))
    return ctx, kv, calls


def i32(n):
    return OnGpu(torch.zeros(n, dtype=torch.int32))


def bf16(*shape):
    return OnGpu(torch.zeros(shape, dtype=torch.bfloat16))


WRONG = [OnGpu(torch.zeros(64, dtype=torch.int64)), OnGpu(torch.zeros(64)), OnGpu(torch.zeros(2, dtype=torch.int32)),
         OnGpu(torch.zeros(64, dtype=torch.int32)[::2]), torch.zeros(64, dtype=torch.int32)]


@pytest.mark.parametrize("wrong", WRONG, ids=["int64", "float", "short", "strided", "host"])
def test_index_tensors(parts, wrong):
    """int64 would be read as pairs of int32, a short tensor past its end."""
    ctx, kv, calls = parts
    rows, q, x = bf16(3, 2, 8), bf16(3, 4, 8), bf16(3, 64)
    w, kept = OnGpu(torch.zeros((3, 2, 8))), i32(3 * 2 * 4)
    good = {
        "paged_append": lambda **a: ctx.paged_append(kv, rows, rows, **{**dict(seq=i32(3), slot=i32(3)), **a}, T=3),
        "paged_prefill": lambda **a: ctx.paged_prefill(kv, q, q, **{**dict(q_start=i32(4)), **a}, T=3),
        "paged_evict": lambda **a: ctx.paged_evict(kv, kv, w, None, 4, **{**dict(kept=kept, new_len=i32(3)), **a}),
        "paged_attn_forward": lambda **a: ctx.paged_attn_forward(
            0, kv, x, x, 3, **{**dict(seq=i32(3), pos=i32(3), slot=i32(3), q_start=i32(4)), **a}),
    }
    for name, args in (("paged_append", ("seq", "slot")), ("paged_prefill", ("q_start",)), ("paged_evict", ("kept", "new_len")),
                       ("paged_attn_forward", ("seq", "pos", "slot", "q_start"))):
        calls.clear()
        good[name]()
        assert calls == ["obs_" + name]
        for arg in args:
            with pytest.raises(ValueError, match=f"{arg}: .* consecutive int32 on the GPU"):
                good[name](**{arg: wrong})
        assert len(calls) == 1


def test_rows(parts):
    ctx, kv, calls = parts
    rows, q, x = bf16(3, 2, 8), bf16(3, 4, 8), bf16(3, 64)
    host, wide = torch.zeros((3, 2, 8), dtype=torch.bfloat16), OnGpu(torch.zeros((2, 40), dtype=torch.bfloat16)[:, :32])
    for bad in (host, bf16(2, 2, 8), wide, OnGpu(torch.zeros((3, 2, 8), dtype=torch.float16))):
        for a in ((bad, rows), (rows, bad)):
            with pytest.raises(ValueError):
                ctx.paged_append(kv, *a, i32(4), i32(4), 3)
    for bad in (torch.zeros((3, 4, 8), dtype=torch.bfloat16), bf16(2, 4, 8), bf16(4, 4, 8),
                OnGpu(torch.zeros((6, 24), dtype=torch.bfloat16)[:, :16])):
        with pytest.raises(ValueError):
            ctx.paged_decode(kv, bad, q)
    with pytest.raises(ValueError):
        ctx.paged_decode(kv, q, torch.zeros((3, 4, 8), dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        ctx.paged_decode(kv, q, q, weights=torch.zeros((3, 2, 8)))
    for bad in (bf16(2, 64), torch.zeros((3, 64), dtype=torch.bfloat16), OnGpu(torch.zeros((3, 64))),
                OnGpu(torch.zeros((3, 80), dtype=torch.bfloat16)[:, :64])):
        for a in ((bad, x), (x, bad)):
            with pytest.raises(ValueError, match="x and out"):
                ctx.paged_attn_forward(0, kv, *a, 3, i32(3), i32(3), i32(3))
    assert calls == []
    ctx.paged_decode(kv, q, bf16(3, 4, 8))
    ctx.paged_attn_forward(0, kv, x, bf16(3, 64), 3, i32(3), i32(3), i32(3))
    assert calls == ["obs_paged_decode", "obs_paged_attn_forward"]


def test_a_cache_on_the_host_is_refused():
    k = torch.zeros((6, 4, 2, 8), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="on the GPU"):
        obsmoe.PagedKV(k, k, torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
