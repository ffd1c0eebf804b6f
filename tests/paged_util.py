"""The paged cache's operators in 64 bits, one sequence and KV head at a time, and
the bounds the kernels' outputs are held to.

Bound of an attention output o = sum_j p_j v_j against the exact value, element by
element, with u half the unit roundoff of the 16-bit type (u = 2^-9 bf16, 2^-12 f16)
and A = sum_j p_j |v_j| >= |o|:
    u |o| + u A    the one rounding of the output takes 2 u |o| at most; what is left,
                   u (A - |o|), is for p where it is rounded to the type for the product
                   with v, which is therefore allowed only where many p average out (the
                   decode carries p in two pieces, the prefill does for rows that see few
                   positions)
  + 1e-4 A         fp32 scores and exponentials: a score is a sum of head_dim <= 128
                   products, off by at most 128 * 2^-24 * sum |q k| * scale; for rows of
                   unit normal entries sum |q k| scale <= 128 / sqrt(128) = 11.3 on average,
                   so 8.6e-5, and an exponential, the sums and the division add a few 2^-22
  + 2^-24 sum |v_j| / l   (f16 only, over the visible j, l = sum_j e^(x_j - max)): p_j below
                   the smallest normal f16 are rounded to a multiple of 2^-24
The added weights (fp32): 1e-4 of the probabilities' sum by the same count, and two
roundings of the total, 2^-23 each."""
import math

import torch

U = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


class Cache:
    """A paged cache of given lengths on the GPU: every place that holds no position is NaN."""

    def __init__(self, lens, kv, hd, page, dtype, seed=0, order="slots", pages_extra=2, table_extra=0, amp=1.0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.kv, self.hd, self.page, self.dtype = list(lens), kv, hd, page, TYPES[dtype]
        held = [-(-n // page) for n in lens]
        n_pages = sum(held) + pages_extra
        shape = {"slots": (n_pages, page, kv, hd), "heads": (n_pages, kv, page, hd)}[order]

        def pool():
            p = torch.full(shape, float("nan"), dtype=self.dtype, device="cuda")
            return p if order == "slots" else p.transpose(1, 2)

        self.k, self.v = pool(), pool()
        perm = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
        width = max(held + [1]) + table_extra
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
        at = 0
        for s, h in enumerate(held):
            self.table[s, :h] = perm[at:at + h]
            at += h
        self.len = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.kd, self.vd = [], []
        for s, n in enumerate(lens):
            k = (amp * torch.randn((n, kv, hd), generator=gen, device="cuda")).to(self.dtype)
            v = torch.randn((n, kv, hd), generator=gen, device="cuda").to(self.dtype)
            self.put(s, torch.arange(n, device="cuda"), k, v)
            self.kd.append(k)
            self.vd.append(v)

    def places(self, s, j):
        return self.table[s].long()[j // self.page], j % self.page

    def put(self, s, j, k, v):
        if len(j):
            p, o = self.places(s, j)
            self.k[p, o], self.v[p, o] = k, v

    def rows(self, s, n):
        j = torch.arange(n, device="cuda")
        if not n:
            return self.k[0:0, 0], self.v[0:0, 0]
        p, o = self.places(s, j)
        return self.k[p, o], self.v[p, o]


def visible(pos, n, window, sinks):
    """[rows, n]: what the queries at positions pos see of n cached positions."""
    j = torch.arange(n, device="cuda")[None]
    ok = j <= pos[:, None]
    if window:
        ok &= (pos[:, None] - j < window) | (j < sinks)
    return ok


def attend(q, k, v, ok, scale):
    """q [rows, group, hd], k, v [n, hd], ok [rows, n] -> o, A, s [rows, group, hd] and p [rows, group, n] in
    64 bits; s = sum over the visible j of |v_j| / l.  Invisible keys and values are not looked at."""
    k = torch.where(ok.any(0)[:, None], k.double(), 0.0)
    v = torch.where(ok.any(0)[:, None], v.double(), 0.0)
    x = torch.einsum("rgd,nd->rgn", q.double(), k) * scale
    x = x.masked_fill(~ok[:, None], -math.inf)
    some = ok.any(1)[:, None, None]
    top = torch.where(some, x.amax(-1, keepdim=True) if x.shape[-1] else torch.zeros_like(some, dtype=x.dtype), 0.0)
    e = torch.where(ok[:, None], torch.exp(x - top), 0.0)
    l = e.sum(-1, keepdim=True)
    p = torch.where(some, e / torch.where(some, l, 1.0), 0.0)
    absv = v.abs()
    s = torch.where(some, torch.einsum("rn,nd->rd", ok.double(), absv)[:, None] / torch.where(some, l, 1.0), 0.0)
    return torch.einsum("rgn,nd->rgd", p, v), torch.einsum("rgn,nd->rgd", p, absv), s, p


def check_out(got, o, a, s, dtype):
    """got within the bound above of o; raises with the worst ratio."""
    u = U[dtype]
    bound = u * o.abs() + (u + 1e-4) * a + (2.0 ** -24 * s if dtype == torch.float16 else 0.0) + 1e-30
    d = (got.double() - o).abs()
    assert not torch.isnan(got.double()).any(), "NaN in the output"
    worst = float((d / bound).max()) if d.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3f} times the bound"


def evict_ref(w, n, budget, sinks, recent):
    """The kept positions of one (sequence, head): w fp32 [n]."""
    if n <= budget:
        return list(range(n))
    w = w.tolist()
    rest = [j for j in range(sinks, n - recent)]
    key = lambda j: (-math.inf if w[j] != w[j] else w[j])  # noqa: E731
    # NaN after everything else, -inf among it; equal weights by position
    rest.sort(key=lambda j: (w[j] != w[j], -key(j), j))
    return sorted(list(range(sinks)) + rest[: budget - sinks - recent] + list(range(n - recent, n)))
