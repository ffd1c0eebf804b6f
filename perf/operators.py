"""The paged key/value cache's operators, as a serving program meets them: what
is measured, in plain torch and through the library's entry points.

Four operators over one cache of pages ([n_pages, page, n_kv, head_dim], a table
of page ids per sequence):

append   new keys and values into their sequences' pages
decode   attention of one new token per sequence over its pages; a window and a
         few first positions that stay visible (sinks) may limit what it sees;
         optionally the attention weights are added up per cached position
prefill  attention of the new tokens of several prompts (or chunks of them) over
         their pages, causal, with the same window and sinks
evict    the positions with the least accumulated weight leave the cache; the
         kept ones move, in order, to the front of other pages

`own` chooses the side: False computes in plain torch (32 bits, one rounding at
the end), True calls project-obsidian_b200's library.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
SPARE = 3  # pages of the pool that no sequence holds


# ------------------------------------------------------------------- the cases
def listed():
    model = {"heads": 32, "kv_heads": 4, "head_dim": 128, "page": 64, "type": "bf16"}  # Qwen3-30B-A3B's attention
    return [
        # one decode step of 16 sequences: a row each
        {"name": "append 16 rows", "op": "append", "n": 16, "len_lo": 1000, "len_hi": 2049, "q_lo": 1, "q_hi": 1, **model},
        # a whole prompt of the prefill workload
        {"name": "append 4096 rows", "op": "append", "n": 1, "len_lo": 4096, "len_hi": 4096, "q_lo": 4096, "q_hi": 4096, **model},
        # batch 1 after a 2048-token prompt: the latency of a single step
        {"name": "decode 1 x 2049", "op": "decode", "n": 1, "len_lo": 2049, "len_hi": 2049, "window": 0, "sinks": 0, "weights": False, **model},
        # a serving batch of mixed lengths up to the long end, f16, small pages
        {"name": "decode 32 x 61..32768 f16", "op": "decode", "n": 32, "len_lo": 61, "len_hi": 32768, "window": 0, "sinks": 0,
         "weights": False, **model, "page": 16, "type": "f16"},
        # a wide batch that sees a window and four sinks
        {"name": "decode 128 x 8192 window", "op": "decode", "n": 128, "len_lo": 700, "len_hi": 8192, "window": 1024, "sinks": 4,
         "weights": False, **model},
        # the step whose weights a later eviction goes by
        {"name": "decode 16 x 4096 weights", "op": "decode", "n": 16, "len_lo": 1500, "len_hi": 4096, "window": 0, "sinks": 0,
         "weights": True, **model},
        # one prompt of the prefill workload, causal
        {"name": "prefill 4096", "op": "prefill", "n": 1, "len_lo": 4096, "len_hi": 4096, "q_lo": 4096, "q_hi": 4096, "window": 0,
         "sinks": 0, **model},
        # a long prompt with a window and sinks
        {"name": "prefill 8192 window", "op": "prefill", "n": 1, "len_lo": 8192, "len_hi": 8192, "q_lo": 8192, "q_hi": 8192,
         "window": 1024, "sinks": 4, **model},
        # a short follow-up question after a long conversation: few rows, long axis
        {"name": "prefill 48 after 16384", "op": "prefill", "n": 1, "len_lo": 16432, "len_hi": 16432, "q_lo": 48, "q_hi": 48,
         "window": 0, "sinks": 0, **model},
        # a batch of short odd prompts, as many key heads as query heads, head size 64
        {"name": "prefill 9 x 1..700 hd64 f16", "op": "prefill", "n": 9, "len_lo": 1, "len_hi": 700, "q_lo": 1, "q_hi": 700,
         "window": 0, "sinks": 0, "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 16, "type": "f16"},
        # one conversation cut to a quarter
        {"name": "evict 1 x 4096 to 1024", "op": "evict", "n": 1, "len_lo": 4096, "len_hi": 4096, "budget": 1024, "sinks": 4,
         "recent": 256, **model},
        # a batch cut at once; the shorter ones fit already
        {"name": "evict 16 x 8192 to 2048", "op": "evict", "n": 16, "len_lo": 900, "len_hi": 8192, "budget": 2048, "sinks": 4,
         "recent": 512, **model},
    ]


def draw(rng):
    def spread(lo, hi):  # over the logarithm
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["append", "decode", "decode", "prefill", "prefill", "evict"])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 3, 4, 5, 8, 8])
    case = {"op": op, "heads": kv * group, "kv_heads": kv, "head_dim": rng.choice([64, 128, 128, 128, 80]),
            "page": rng.choice([16, 32, 64, 128]), "type": rng.choice(["bf16", "bf16", "f16"])}
    if op == "append":
        q = spread(1, 2048)
        case.update(n=rng.choice([1, 2, 5, 16]), len_lo=q, len_hi=q + spread(1, 4000), q_lo=max(1, q // 3), q_hi=q)
        if case["n"] * q > 4096:
            case["n"] = 1
    elif op == "decode":
        hi = spread(40, 32768)
        n = max(1, min(spread(1, 128), 260000 // hi))
        case.update(n=n, len_lo=max(1, hi // rng.choice([1, 3, 50])), len_hi=hi, window=0, sinks=0, weights=rng.random() < 0.3)
        if rng.random() < 0.4:
            case.update(window=spread(16, 2048), sinks=rng.choice([0, 1, 4, 13]))
    elif op == "prefill":
        q = spread(2, 3000)
        ctx = spread(1, 6000) if rng.random() < 0.5 else 0
        n = max(1, min(spread(1, 12), 3500 // (q + ctx)))
        case.update(n=n, len_lo=max(1, q // 4) + ctx, len_hi=q + ctx, q_lo=max(1, q // 4), q_hi=q, window=0, sinks=0)
        if rng.random() < 0.4:
            case.update(window=spread(16, 2048), sinks=rng.choice([0, 1, 4, 13]))
        if case["heads"] > 32:
            case.update(heads=32, kv_heads=4)
    else:
        hi = spread(200, 12000)
        budget = max(40, hi // rng.choice([2, 3, 5, 9]))
        n = max(1, min(spread(1, 16), 60000 // hi))
        sinks = rng.choice([0, 1, 4, 13])
        case.update(n=n, len_lo=max(1, hi // 4), len_hi=hi, budget=budget, sinks=sinks, recent=min(budget - sinks, spread(1, budget)))
    return case


def _between(lo, hi, n):
    """n whole numbers in [lo, hi], the largest first, then spread by the golden ratio: a ragged batch that the case alone fixes."""
    return [hi if i == 0 else lo + int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _lens(case):
    return _between(case["len_lo"], case["len_hi"], case["n"])


def _qlens(case):
    return [min(a, b) for a, b in zip(_between(case["q_lo"], case["q_hi"], case["n"]), _lens(case))]


def _seen(pos, window, sinks):
    """How many positions the query at `pos` sees."""
    if not window:
        return pos + 1
    first = max(0, pos + 1 - window)
    return pos + 1 - first + min(sinks, first)


def work(case):
    lens, rows = _lens(case), case["kv_heads"] * case["head_dim"]
    size = 2
    if case["op"] == "append":
        t = sum(_qlens(case))
        return {"bytes": 4 * t * rows * size + 8 * t, "flops": 0}
    if case["op"] == "decode":
        seen = sum(_seen(n - 1, case["window"], case["sinks"]) for n in lens)
        io = 2 * case["n"] * case["heads"] * case["head_dim"] * size
        added = 8 * seen * case["kv_heads"] if case["weights"] else 0
        return {"bytes": 2 * seen * rows * size + io + added, "flops": 4 * seen * case["heads"] * case["head_dim"]}
    if case["op"] == "prefill":
        pairs = keys = 0
        for n, q in zip(lens, _qlens(case)):
            pairs += sum(_seen(p, case["window"], case["sinks"]) for p in range(n - q, n))
            first = max(0, n - q + 1 - case["window"]) if case["window"] else 0
            keys += n - first + min(case["sinks"], first)
        io = 2 * sum(_qlens(case)) * case["heads"] * case["head_dim"] * size
        return {"bytes": 2 * keys * rows * size + io, "flops": 4 * pairs * case["heads"] * case["head_dim"]}
    kept = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": 4 * kept * rows * size + 4 * case["kv_heads"] * (sum(lens) + 2 * case["n"] * case["budget"]), "flops": 0}


# ------------------------------------------------------------------ the inputs
class State:
    pass


def _normal(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    s = State()
    s.case, dtype = case, DTYPES[case["type"]]
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    n, page, kv, hd, heads = case["n"], case["page"], case["kv_heads"], case["head_dim"], case["heads"]
    lens = _lens(case)
    s.max_len = max(lens)
    per = -(-s.max_len // page)
    held = [-(-x // page) for x in lens]
    # every sequence's pages, anywhere in the pool; unused places of the table hold page 0
    n_pages = sum(held) + SPARE
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    s.table = torch.zeros((n, per), dtype=torch.int32, device="cuda")
    at = 0
    for i, h in enumerate(held):
        s.table[i, :h] = order[at:at + h]
        at += h
    s.len = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s.k = _normal((n_pages, page, kv, hd), gen, dtype)
    s.v = _normal((n_pages, page, kv, hd), gen, dtype)
    s.scale = hd ** -0.5
    op = case["op"]
    if op in ("append", "prefill"):
        q = _qlens(case)
        s.q_max, s.rows = max(q), sum(q)
        s.q_len = torch.tensor(q, dtype=torch.int32, device="cuda")
        s.q_start = torch.tensor([sum(q[:i]) for i in range(n + 1)], dtype=torch.int32, device="cuda")
    if op == "append":
        s.new_k, s.new_v = _normal((s.rows, kv, hd), gen, dtype), _normal((s.rows, kv, hd), gen, dtype)
        s.seq = torch.repeat_interleave(torch.arange(n, device="cuda"), s.q_len).to(torch.int32)
        s.slot = (torch.arange(s.rows, device="cuda") - s.q_start[s.seq.long()] + (s.len - s.q_len)[s.seq.long()]).to(torch.int32)
    elif op == "decode":
        s.q, s.out = _normal((n, heads, hd), gen, dtype), torch.empty((n, heads, hd), dtype=dtype, device="cuda")
        s.w = torch.rand((n, kv, s.max_len), generator=gen, device="cuda") if case["weights"] else None
    elif op == "prefill":
        s.q, s.out = _normal((s.rows, heads, hd), gen, dtype), torch.empty((s.rows, heads, hd), dtype=dtype, device="cuda")
    else:
        # accumulated weights: a few positions carry most of it
        s.w = torch.exp(2 * torch.randn((n, kv, s.max_len), generator=gen, device="cuda"))
        budget = case["budget"]
        to = -(-budget // page)
        s.to_table = torch.randperm(n * to, generator=gen, device="cuda").to(torch.int32).reshape(n, to)
        s.to_k, s.to_v = (torch.zeros((n * to, page, kv, hd), dtype=dtype, device="cuda") for _ in range(2))
        s.to_w = torch.zeros((n, kv, s.max_len), device="cuda")
        s.kept = torch.empty((n, kv, budget), dtype=torch.int32, device="cuda")
        s.to_len = torch.empty((n,), dtype=torch.int32, device="cuda")
    if own:
        _prepare_own(s)
    return s


def _library():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "project-obsidian_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import obsmoe

    return obsmoe


_contexts = {}  # one for each shape of cache, as a program keeps one for its model


def _prepare_own(s):
    """The context with its workspace, and the caches' descriptors: what a program makes once."""
    lib, c = _library(), s.case
    plan = dict(n_heads=c["heads"], n_kv_heads=c["kv_heads"], head_dim=c["head_dim"], page_size=c["page"], max_seqs=c["n"],
                max_kv_len=s.max_len, dtype=c["type"], weights=c["op"] == "decode" and c["weights"])
    key = tuple(plan.values())
    if key not in _contexts:
        ctx = lib.MoeContext(lib.MoeShape(hidden=2048, inter=256, n_experts=16, top_k=4, n_layers=1, max_tokens=1))
        ctx.paged_init(**plan)
        _contexts[key] = ctx
    s.ctx = _contexts[key]
    s.kv = lib.PagedKV(s.k, s.v, s.table, s.len)
    if c["op"] == "evict":
        s.to_kv = lib.PagedKV(s.to_k, s.to_v, s.to_table, s.to_len)


# -------------------------------------------------------------------- one pass
def run(s):
    return {"append": _append, "decode": _decode, "prefill": _prefill, "evict": _evict}[s.case["op"]](s)


def _rows(pool, table, most):
    """Each sequence's rows in 32 bits: [n, most, n_kv, head_dim]."""
    r = pool[table.long()].flatten(1, 2)[:, :most]
    return r.to(torch.float32)


def _softmax(x):
    """Over the last axis; a row with nothing visible gives zeros."""
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _append(s):
    if own:
        s.ctx.paged_append(s.kv, s.new_k, s.new_v, s.seq, s.slot, s.rows)
        return s.k, s.v
    page = s.case["page"]
    slot = s.slot.long()
    at, off = s.table.long()[s.seq.long(), slot // page], slot % page
    s.k[at, off] = s.new_k
    s.v[at, off] = s.new_v
    return s.k, s.v


def _decode(s):
    c = s.case
    if own:
        s.ctx.paged_decode(s.kv, s.q, s.out, window=c["window"], n_sink=c["sinks"], scale=s.scale, weights=s.w)
        return s.out if s.w is None else (s.out, s.w)
    n, kv, hd = c["n"], c["kv_heads"], c["head_dim"]
    k, v = _rows(s.k, s.table, s.max_len), _rows(s.v, s.table, s.max_len)
    q = s.q.to(torch.float32).reshape(n, kv, -1, hd)
    x = torch.einsum("ngrd,nlgd->ngrl", q, k) * s.scale
    j, last = torch.arange(s.max_len, device="cuda")[None], s.len[:, None]
    seen = j < last
    if c["window"]:
        seen = seen & ((j >= last - c["window"]) | (j < c["sinks"]))
    p = _softmax(x.masked_fill(~seen[:, None, None], float("-inf")))
    out = torch.einsum("ngrl,nlgd->ngrd", p, v).reshape(n, -1, hd).to(s.q.dtype)
    if s.w is None:
        return out
    s.w += p.sum(2)
    return out, s.w


def _prefill(s):
    c = s.case
    if own:
        s.ctx.paged_prefill(s.kv, s.q, s.out, s.q_start, s.rows, window=c["window"], n_sink=c["sinks"], scale=s.scale)
        return s.out
    n, kv, hd = c["n"], c["kv_heads"], c["head_dim"]
    k, v = _rows(s.k, s.table, s.max_len), _rows(s.v, s.table, s.max_len)
    i = torch.arange(s.q_max, device="cuda")[None]
    start, many = s.q_start[:-1, None], s.q_len[:, None]
    q = s.q[(start + torch.minimum(i, many - 1)).long()].to(torch.float32).reshape(n, s.q_max, kv, -1, hd)
    x = torch.einsum("nqgrd,nlgd->ngrql", q, k) * s.scale
    pos = (s.len[:, None] - many + i)[:, :, None]
    j = torch.arange(s.max_len, device="cuda")[None, None]
    seen = j <= pos
    if c["window"]:
        seen = seen & ((pos - j < c["window"]) | (j < c["sinks"]))
    p = _softmax(x.masked_fill_(~seen[:, None, None], float("-inf")))
    out = torch.einsum("ngrql,nlgd->nqgrd", p, v).reshape(n, s.q_max, -1, hd)
    t = torch.arange(s.rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s.q_start[1:], t, right=True)
    return out[seq, (t - s.q_start[seq]).long()].to(s.q.dtype)


def _evict(s):
    c = s.case
    budget, sinks, recent, page = c["budget"], c["sinks"], c["recent"], c["page"]
    if own:
        s.ctx.paged_evict(s.kv, s.to_kv, s.w, s.to_w, budget, n_sink=sinks, n_recent=recent, kept=s.kept, new_len=s.to_len)
        return s.kept, s.to_len, s.to_k, s.to_v, s.to_w
    n, kv = c["n"], c["kv_heads"]
    j, last = torch.arange(s.max_len, device="cuda")[None, None], s.len[:, None, None]
    inf = float("inf")
    w = s.w.masked_fill((j < sinks) | (j >= last - recent), inf).masked_fill(j >= last, -inf)
    few = min(budget, s.max_len)
    first = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :few]
    s.to_len.copy_(torch.clamp(s.len, max=budget))
    i = torch.arange(budget, device="cuda")[None, None]
    first = torch.nn.functional.pad(first, (0, budget - few), value=s.max_len)
    kept = torch.sort(torch.where(i < s.to_len[:, None, None], first, s.max_len), dim=-1).values
    held = kept < s.max_len
    s.kept.copy_(torch.where(held, kept, -1))
    # rows that are not held write their own value again
    seq, head = torch.arange(n, device="cuda")[:, None, None], torch.arange(kv, device="cuda")[None, :, None]
    frm = torch.where(held, kept, 0)
    a, b, off = s.table.long()[seq, frm // page], s.to_table.long()[seq, i // page], i % page
    for_row = held[..., None]
    s.to_k[b, off, head] = torch.where(for_row, s.k[a, frm % page, head], s.to_k[b, off, head])
    s.to_v[b, off, head] = torch.where(for_row, s.v[a, frm % page, head], s.to_v[b, off, head])
    s.to_w.zero_()
    s.to_w[:, :, :few] = torch.where(held, s.w.gather(2, frm), 0.0)[..., :few]
    return s.kept, s.to_len, s.to_k, s.to_v, s.to_w


# ------------------------------------------------------------- in 64 bits, apart
def exact(case, seed):
    """One sequence and one key head at a time, in 64 bits."""
    global own
    mine, own = own, False
    s = prepare(case, seed)
    own = mine
    c, lens = case, _lens(case)
    page, group = c["page"], c["heads"] // c["kv_heads"]
    if c["op"] in ("append", "evict"):  # rows are moved as they are: nothing is computed
        return None

    def cached(pool, i, h, n):
        pages = s.table[i, : -(-n // page)].tolist()
        return torch.cat([pool[p, :, h] for p in pages])[:n].double()

    def visible(pos, n):
        j = torch.arange(n, device="cuda")
        ok = j[None] <= pos[:, None]
        if c["window"]:
            ok &= (j[None] > pos[:, None] - c["window"]) | (j[None] < c["sinks"])
        return ok

    def attend(q, k, v, ok):
        x = (q.double() @ k.T) / math.sqrt(c["head_dim"])
        x[~ok] = -math.inf
        p = torch.softmax(x, -1)
        return p @ v, p

    out = torch.zeros(s.out.shape, dtype=torch.float64, device="cuda")
    added = None if c["op"] != "decode" or s.w is None else s.w.double()
    starts, counts = (s.q_start.tolist(), _qlens(c)) if c["op"] == "prefill" else (list(range(c["n"])), [1] * c["n"])
    for i, n in enumerate(lens):
        pos = torch.arange(n - counts[i], n, device="cuda")
        ok = visible(pos, n)
        rows = slice(starts[i], starts[i] + counts[i])
        for h in range(c["kv_heads"]):
            k, v = cached(s.k, i, h, n), cached(s.v, i, h, n)
            for g in range(h * group, (h + 1) * group):
                o, p = attend(s.q[rows, g], k, v, ok)
                out[rows, g] = o
                if added is not None:
                    added[i, h, :n] += p[0]
    return out if added is None else (out, added)
