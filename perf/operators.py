"""The paged KV cache's operators as measurable cases: writing chunks into pages, copying pages,
attention over pages, and attention for a batch that shares a long prefix.

A pool of pages is ``[2, P, rows, H, D]`` (plane 0 K, plane 1 V). Row ``r`` of a sequence lies in
page ``table[r // rows]`` at row ``r % rows``. Shapes are those of the Wan-5B path (24 heads x 128,
30 layers, 83-token chunks), the Wan-14B path (40 heads x 128), GR00T's grouped-query backbone (16
query heads over 8, token by token) and the other head dims and types that the operators take.

Kinds:

* ``append``  ``kv_page_append``: a chunk per sequence into its pages;
* ``copy``    ``kv_page_copy``: pages to other pages, in every layer's pool at once;
* ``paged``   ``paged_attention``: cached rows by page table, then the chunk's own keys;
* ``shared``  ``shared_prefix_attention``: one prefix for the whole batch, then each sequence's
              own cached rows and its chunk's own keys.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_OPS = None


def _ops():
    global _OPS
    if _OPS is None:
        pkg = str(Path(__file__).resolve().parents[1] / "dexter-labs_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from dexter_amd import ops
        _OPS = ops
    return _OPS


def _append(name, batch, n, heads, dim, page, lo, hi, dtype="bf16"):
    """Sequences start at rows spread over lo..hi."""
    case = {"kind": "append", "batch": batch, "n": n, "kv_heads": heads, "dim": dim,
            "page": page, "lo": lo, "hi": hi, "dtype": dtype}
    return {"name": name, **case} if name else case


def _copy(name, layers, pages, pool, heads, dim, page, dtype="bf16"):
    case = {"kind": "copy", "layers": layers, "pages": pages, "pool": pool, "kv_heads": heads,
            "dim": dim, "page": page, "dtype": dtype}
    return {"name": name, **case} if name else case


def _attn(name, batch, lq, heads, kv_heads, dim, page, lo, hi, *, prefix=0, block=0, causal=False,
          dtype="bf16"):
    """Cached rows per sequence spread over lo..hi; block 0: no block boundaries."""
    case = {"kind": "shared" if prefix else "paged", "batch": batch, "lq": lq, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "lo": lo, "hi": hi, "prefix": prefix,
            "block": block, "causal": causal, "dtype": dtype}
    return {"name": name, **case} if name else case


def listed():
    return [
        # One decoded token of each of 64 sequences of the grouped-query backbone: latency.
        _append("append_tokens", 64, 1, 8, 128, 16, 100, 1500),
        # Eight rollouts write their 83-token chunks, each at its own row.
        _append("append_chunks", 8, 83, 24, 128, 64, 332, 3237),
        # Priming four episodes of the 14B model, 1,826 rows each (two 913-token chunks).
        _append("append_prime", 4, 1826, 40, 128, 128, 0, 0, dtype="f16"),
        # A rollout forks: its last, partly filled page is copied in the backbone's 16 layers.
        _copy("fork_tail", 16, 1, 12, 8, 128, 16),
        # Compaction of the 5B model's pool: 16 pages move down, all 30 layers.
        _copy("compact_5b", 30, 16, 40, 24, 128, 32),
        # Token-by-token decoding of 32 prompts of different lengths, grouped-query.
        _attn("decode_tokens", 32, 1, 16, 8, 128, 16, 300, 3000),
        # Four rollouts at different points of their episodes, frame block + action block, in fp32
        # (the type that results are checked in).
        _attn("chunks_fp32", 4, 99, 24, 24, 128, 32, 0, 1245, block=83, dtype="f32"),
        # A chunk late in a long episode: the cache read is the whole cost.
        _attn("chunk_long", 1, 83, 24, 24, 128, 128, 32768, 32768),
        # Prompts continued over cached turns, token-causal, grouped-query.
        _attn("prompts_causal", 2, 1500, 16, 8, 128, 64, 400, 1000, causal=True),
        # Candidate futures: 16 rollouts' chunks over one episode's history and their own rows.
        _attn("rollouts_5b", 16, 83, 24, 24, 128, 64, 0, 332, prefix=8217),
        # 64 continuations of one prompt, token by token, grouped-query.
        _attn("tokens_shared", 64, 1, 16, 8, 128, 16, 1, 500, prefix=4001),
        # Narrow heads in f16, every rollout still at the fork: no cached rows of its own.
        _attn("rollouts_narrow", 8, 50, 12, 12, 64, 48, 0, 0, prefix=2000, dtype="f16"),
    ]


# ---------------------------------------------------------------------------
# Drawn cases: the same kinds, sizes log-uniform over the range in use.
# ---------------------------------------------------------------------------
def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    rate = 1 / 12 if case["dtype"] == "f32" else 1.0  # fp32 products
    return w["bytes"] / 4e12 + w["flops"] / rate / 1e15


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        case = rng.choice([_draw_append, _draw_copy, _draw_paged, _draw_paged, _draw_shared,
                           _draw_shared])(rng)
        if _cost(case) <= limit:
            return case


def _draw_pool(rng):
    heads, kv = rng.choice([(24, 24), (24, 24), (40, 40), (16, 8), (16, 4), (12, 12), (28, 4)])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([128, 128, 64]) if dtype == "f32" else rng.choice([128, 128, 128, 64, 256])
    return heads, kv, dim, rng.choice([16, 32, 48, 64, 128, 256]), dtype


def _draw_append(rng):
    _, kv, dim, page, dtype = _draw_pool(rng)
    lo = rng.choice([0, _log(rng, 1, 4000)])
    return _append("", _log(rng, 1, 64), _log(rng, 1, 2000), kv, dim, page, lo,
                   lo + rng.choice([0, _log(rng, 1, 4000)]), dtype)


def _draw_copy(rng):
    _, kv, dim, page, dtype = _draw_pool(rng)
    pages = _log(rng, 1, 100)
    return _copy("", _log(rng, 1, 40), pages, 2 * pages + rng.randint(0, 8), kv, dim, page, dtype)


def _draw_attn(rng, prefix):
    heads, kv, dim, page, dtype = _draw_pool(rng)
    lq = rng.choice([1, 1, _log(rng, 2, 128), _log(rng, 2, 128), _log(rng, 100, 1500)])
    top = 4000 if prefix else 32768
    lo = rng.choice([0, _log(rng, 1, top)])
    hi = max(lo, rng.choice([lo, _log(rng, 1, top)]))
    mask = rng.choice(["none", "none", "causal", "block"])
    return _attn("", _log(rng, 2 if prefix else 1, 64), lq, heads, kv, dim, page, lo, hi,
                 prefix=prefix, causal=mask == "causal",
                 block=_log(rng, 1, lq) if mask == "block" else 0, dtype=dtype)


def _draw_paged(rng):
    return _draw_attn(rng, 0)


def _draw_shared(rng):
    return _draw_attn(rng, _log(rng, 100, 32768))


# ---------------------------------------------------------------------------
# Inputs, made on the GPU from the seed alone.
# ---------------------------------------------------------------------------
def _lens(case):
    """Cached rows (or start rows) per sequence, spread over lo..hi."""
    span = case["hi"] - case["lo"]
    return [case["lo"] + round(span * ((0.618034 * i) % 1.0)) for i in range(case["batch"])]


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE).to(dt)

    if case["kind"] == "copy":
        pools = [rand(2, case["pool"], page, kv, dim) for _ in range(case["layers"])]
        order = torch.randperm(case["pool"], generator=g, device=DEVICE).tolist()
        n = case["pages"]
        return {"case": case, "pools": pools, "src": order[:n], "dst": order[n:2 * n]}
    batch, lens = case["batch"], _lens(case)
    new = case["n"] if case["kind"] == "append" else 0
    width = max(1, -(-(max(lens) + new) // page))
    prefix = case.get("prefix", 0)
    prefix_pages = -(-prefix // page)
    held = [-(-(n + new) // page) for n in lens]
    # Pages lie anywhere in the pool, a few of which are free; rows past a sequence's end and
    # free pages hold what earlier sequences left there.
    total = sum(held) + prefix_pages + 3
    order = torch.randperm(total, generator=g, device=DEVICE).tolist()
    table = [[order.pop() if j < n else -1 for j in range(width)] for n in held]
    s = {"case": case, "pages": rand(2, total, page, kv, dim), "table": _i32(table),
         "lens": _i32(lens), "host_lens": lens, "host_table": table}
    if case["kind"] == "append":
        s["k"], s["v"] = rand(batch, new, kv, dim), rand(batch, new, kv, dim)
        return s
    lq = case["lq"]
    s["q"] = rand(batch, lq, case["heads"], dim)
    s["k"], s["v"] = rand(batch, lq, kv, dim), rand(batch, lq, kv, dim)
    s["starts"] = _i32(list(range(0, lq, case["block"]))) if case["block"] else None
    if prefix:
        s["host_prefix"] = [order.pop() for _ in range(prefix_pages)]
        s["prefix_table"], s["prefix_len"] = _i32(s["host_prefix"]), _i32([prefix])
    return s


# ---------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return (_run_own if own else _run_plain)(case["kind"], case, state)


def _run_own(kind, case, s):
    ops = _ops()
    if kind == "append":
        ops.kv_page_append(s["pages"], s["k"], s["v"], s["table"], s["lens"])
        return s["pages"]
    if kind == "copy":
        ops.kv_page_copy(s["pools"], s["src"], s["dst"])
        return s["pools"]
    if kind == "paged":
        return ops.paged_attention(
            s["q"], s["k"], s["v"], pages=s["pages"], block_table=s["table"],
            cache_lens=s["lens"], block_boundaries=s["starts"], causal=case["causal"])
    return ops.shared_prefix_attention(
        s["q"], s["k"], s["v"], pages=s["pages"], prefix_table=s["prefix_table"],
        prefix_len=s["prefix_len"], block_table=s["table"], cache_lens=s["lens"],
        block_boundaries=s["starts"], causal=case["causal"])


def _run_plain(kind, case, s):
    if kind == "copy":
        for pool in s["pools"]:
            pool[:, s["dst"]] = pool[:, s["src"]]
        return s["pools"]
    pages, page = s["pages"], case["page"]
    if kind == "append":
        n = case["n"]
        row = s["lens"].long()[:, None] + torch.arange(n, device=DEVICE)
        at = torch.gather(s["table"].long(), 1, row // page)
        pages[0, at, row % page] = s["k"]
        pages[1, at, row % page] = s["v"]
        return pages
    lq, heads, kv, dim = case["lq"], case["heads"], case["kv_heads"], case["dim"]
    group = heads // kv
    # Visible end of each query among the chunk's own keys.
    i = torch.arange(lq, device=DEVICE)
    if case["causal"]:
        end = i + 1
    elif case["block"]:
        end = torch.clamp((i // case["block"] + 1) * case["block"], max=lq)
    else:
        end = torch.full((lq,), lq, device=DEVICE)
    hidden = (i[None, :] >= end[:, None]).repeat(group, 1)
    lead = []
    if case["prefix"]:
        rows = pages[:, s["prefix_table"].long()].flatten(1, 2)[:, :case["prefix"]]
        lead.append(rows.float().permute(0, 2, 1, 3))
    out = torch.empty_like(s["q"])
    for b, n in enumerate(s["host_lens"]):
        parts = list(lead)
        if n:
            rows = pages[:, s["table"][b, :-(-n // page)].long()].flatten(1, 2)[:, :n]
            parts.append(rows.float().permute(0, 2, 1, 3))
        parts.append(torch.stack((s["k"][b], s["v"][b])).float().permute(0, 2, 1, 3))
        keys = torch.cat([p[0] for p in parts], 1)
        values = torch.cat([p[1] for p in parts], 1)
        # [kv, group * lq, dim]: a K/V head's query heads one after the other.
        q = s["q"][b].float().permute(1, 0, 2).reshape(kv, group * lq, dim)
        x = torch.bmm(q, keys.transpose(1, 2).contiguous()) / math.sqrt(dim)
        x[:, :, -lq:].masked_fill_(hidden, -math.inf)
        p = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.bmm(p, values) / p.sum(-1, keepdim=True)
        out[b] = o.view(heads, lq, dim).permute(1, 0, 2).to(out.dtype)
    return out


# ---------------------------------------------------------------------------
# What one pass cannot do without.
# ---------------------------------------------------------------------------
def _pairs(lq, cached, block, causal):
    if causal:
        return lq * cached + lq * (lq + 1) // 2
    if block:
        return sum((min(lo + block, lq) - lo) * (cached + min(lo + block, lq))
                   for lo in range(0, lq, block))
    return lq * (cached + lq)


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    row = 2 * case["kv_heads"] * case["dim"] * es  # a key and a value of every head
    if case["kind"] == "copy":
        return {"bytes": 2 * case["layers"] * case["pages"] * case["page"] * row, "flops": 0}
    lens, page = _lens(case), case["page"]
    if case["kind"] == "append":
        n = case["n"]
        entries = sum(-(-(c + n) // page) - c // page for c in lens)
        return {"bytes": 2 * len(lens) * n * row + 4 * (entries + len(lens)), "flops": 0}
    lq, prefix = case["lq"], case["prefix"]
    q_out = 2 * len(lens) * lq * case["heads"] * case["dim"] * es
    entries = sum(-(-c // page) for c in lens) + -(-prefix // page)
    pairs = sum(_pairs(lq, prefix + c, case["block"], case["causal"]) for c in lens)
    return {"bytes": q_out + row * (prefix + sum(c + lq for c in lens)) + 4 * (entries + len(lens)),
            "flops": 4 * case["dim"] * case["heads"] * pairs}


# ---------------------------------------------------------------------------
# The definition in 64 bits: one (sequence, head, query) row of keys at a time, found row by row.
# ---------------------------------------------------------------------------
def _slots(table, count, page):
    """Row index in the pool's flattened (page, row) axis of rows 0..count-1 of a sequence."""
    return torch.tensor([table[r // page] * page + r % page for r in range(count)],
                        dtype=torch.long, device=DEVICE)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    page = case["page"]
    if case["kind"] == "copy":
        before = s["pools"]
        after = [p.clone() for p in before]
        for a, b in zip(after, before):
            for i, j in zip(s["src"], s["dst"]):
                a[0, j], a[1, j] = b[0, i], b[1, i]
        return after
    if case["kind"] == "append":
        flat = s["pages"].flatten(1, 2)
        for b, start in enumerate(s["host_lens"]):
            at = _slots(s["host_table"][b], start + case["n"], page)[start:]
            flat[0].index_copy_(0, at, s["k"][b])
            flat[1].index_copy_(0, at, s["v"][b])
        return s["pages"]
    flat = s["pages"].flatten(1, 2)
    lq, group = case["lq"], case["heads"] // case["kv_heads"]
    shared = _slots(s["host_prefix"], case["prefix"], page) if case["prefix"] else None
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(s["host_lens"]):
        slots = _slots(s["host_table"][b], n, page)
        if shared is not None:
            slots = torch.cat((shared, slots))
        first = slots.numel()  # key index of the chunk's first key
        last = [first + lq - 1] * lq  # last visible key of each query
        if case["causal"]:
            last = [first + t for t in range(lq)]
        elif case["block"]:
            last = [first + min(t - t % case["block"] + case["block"], lq) - 1 for t in range(lq)]
        seen = torch.tensor(last, device=DEVICE)[:, None] >= torch.arange(first + lq, device=DEVICE)
        for h in range(case["kv_heads"]):
            kh = torch.cat((flat[0, slots, h], s["k"][b, :, h])).double()
            vh = torch.cat((flat[1, slots, h], s["v"][b, :, h])).double()
            kt = kh.t().contiguous()
            for e in range(h * group, (h + 1) * group):
                x = torch.where(seen, s["q"][b, :, e].double() @ kt * case["dim"] ** -0.5,
                                torch.tensor(-math.inf, dtype=torch.float64, device=DEVICE))
                out[b, :, e] = torch.softmax(x, 1) @ vh
    return out
