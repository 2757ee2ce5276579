"""Operators of a KV cache that is held in 4 bits, and of one that forgets, as measurable cases.

A 4-bit pool of pages is uint8 ``[2, P, H, R * (D / 2 + D / 32)]`` (plane 0 K, plane 1 V): of each
page and head first R rows of D / 2 code bytes (element 2 i in the low half of byte i), then R rows
of D / 32 scale bytes. A code is an E2M1 number (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), and the 32
elements of a block share a scale 2^(byte - 127), 2^e for the least e with every magnitude at most
7 * 2^e (e at least -127 and at most 125 for bf16, -23 and 13 for f16; 255: the block holds what is no number). A 16-bit
pool is ``[2, P, R, H, D]``. Row ``r`` of a sequence lies in page ``table[r // R]`` at row ``r % R``.

Shapes are those of the Wan-5B path (24 heads x 128, 83-token chunks), the Wan-14B path (40 heads
x 128), GR00T's grouped-query backbone (16 query heads over 8, token by token), and the other head
dims and types that the operators take.

Kinds:

* ``write``    ``kv_page_append_fp4``, then ``kv_page_read_fp4`` of the rows written;
* ``attend``   ``paged_attention_fp4``, or ``shared_prefix_attention_fp4`` with a prefix, and each
               query's log-sum-exp;
* ``weights``  ``paged_key_weights``: the softmax weight that each cached row received;
* ``keep``     ``kv_keep_rows``: which rows to keep, by weight, the last ones always;
* ``gather``   ``kv_page_gather``: the kept rows move to the front, in place or into new pages.
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


def _case(name, case):
    return {"name": name, **case} if name else case


def _write(name, batch, n, heads, dim, page, lo, hi, dtype="bf16"):
    """Sequences start at rows spread over lo..hi."""
    return _case(name, {"kind": "write", "batch": batch, "n": n, "kv_heads": heads, "dim": dim,
                        "page": page, "lo": lo, "hi": hi, "dtype": dtype})


def _attend(name, batch, lq, heads, kv_heads, dim, page, lo, hi, *, prefix=0, block=0,
            causal=False, dtype="bf16"):
    """Cached rows per sequence spread over lo..hi; block 0: no block boundaries."""
    return _case(name, {"kind": "attend", "batch": batch, "lq": lq, "heads": heads,
                        "kv_heads": kv_heads, "dim": dim, "page": page, "lo": lo, "hi": hi,
                        "prefix": prefix, "block": block, "causal": causal, "dtype": dtype})


def _weights(name, batch, lq, heads, kv_heads, dim, page, lo, hi, *, fp4, dtype="bf16"):
    return _case(name, {"kind": "weights", "batch": batch, "lq": lq, "heads": heads,
                        "kv_heads": kv_heads, "dim": dim, "page": page, "lo": lo, "hi": hi,
                        "fp4": fp4, "dtype": dtype})


def _keep(name, batch, kv_heads, lo, hi, keep, recent):
    return _case(name, {"kind": "keep", "batch": batch, "kv_heads": kv_heads, "lo": lo, "hi": hi,
                        "keep": keep, "recent": recent})


def _gather(name, batch, kv_heads, dim, page, lo, hi, keep, *, fp4, new_pages, dtype="bf16"):
    return _case(name, {"kind": "gather", "batch": batch, "kv_heads": kv_heads, "dim": dim,
                        "page": page, "lo": lo, "hi": hi, "keep": keep, "fp4": fp4,
                        "new_pages": new_pages, "dtype": dtype})


def listed():
    return [
        # One decoded token of each of 64 sequences of the grouped-query backbone: latency.
        _write("write_tokens", 64, 1, 8, 128, 16, 100, 1500),
        # Priming four episodes of the 14B model, 1,826 rows each (two 913-token chunks).
        _write("write_prime", 4, 1826, 40, 128, 128, 0, 0, dtype="f16"),
        # Token-by-token decoding of 32 prompts of different lengths, grouped-query.
        _attend("tokens_fp4", 32, 1, 16, 8, 128, 16, 300, 3000),
        # A chunk late in a long episode: the cache read is the whole cost.
        _attend("chunk_long_fp4", 1, 83, 24, 24, 128, 128, 32768, 32768),
        # Prompts continued over cached turns, token-causal, grouped-query.
        _attend("prompts_fp4", 2, 1500, 16, 8, 128, 64, 400, 1000, causal=True, dtype="f16"),
        # Candidate futures: 16 rollouts' chunks over one episode's history and their own rows.
        _attend("rollouts_fp4", 16, 83, 24, 24, 128, 64, 0, 332, prefix=8217),
        # What each row of a long episode (a 16-bit cache) gave the newest chunk.
        _weights("weights_chunk", 1, 83, 24, 24, 128, 128, 32768, 32768, fp4=False),
        # The same of 32 decoded tokens over a 4-bit cache: latency.
        _weights("weights_tokens", 32, 1, 16, 8, 128, 16, 300, 3000, fp4=True),
        # Which 1,024 rows each of 32 prompts keeps, the last 64 among them.
        _keep("keep_tokens", 32, 8, 300, 3000, 1024, 64),
        # Four long episodes down to a quarter of their rows.
        _keep("keep_long", 4, 24, 32768, 32768, 8192, 512),
        # A long episode's rows move to the front of its own pages.
        _gather("gather_long", 1, 24, 128, 128, 32768, 32768, 8192, fp4=False, new_pages=False),
        # Forked prompts leave the pages that they share: the kept rows go to new ones.
        _gather("gather_tokens", 32, 8, 128, 16, 300, 3000, 1024, fp4=True, new_pages=True),
    ]


# ---------------------------------------------------------------------------
# Drawn cases: the same kinds, sizes log-uniform over the range in use.
# ---------------------------------------------------------------------------
def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    rate = 1 / 12 if case.get("dtype") == "f32" else 1.0  # fp32 products
    return w["bytes"] / 4e12 + w["flops"] / rate / 1e15


def draw(rng):
    limit = max(_cost(c) for c in listed())
    kinds = [_draw_write, _draw_attend, _draw_attend, _draw_shared, _draw_weights, _draw_keep,
             _draw_gather]
    while True:
        case = rng.choice(kinds)(rng)
        # (The plain form lays every sequence out at the longest one's length.)
        if _cost(case) <= limit and _padded(case) <= 1 << 31:
            return case


def _padded(case):
    """Elements of the longest sequence's keys and scores, times the batch."""
    rows = case["batch"] * (case["hi"] + case.get("prefix", 0) + case.get("lq", 0))
    return rows * max(case["kv_heads"] * case.get("dim", 1), case.get("heads", 0) * case.get("lq", 0))


def _draw_pool(rng, f32=False):
    heads, kv = rng.choice([(24, 24), (24, 24), (40, 40), (16, 8), (16, 4), (12, 12), (28, 4)])
    dtype = rng.choice(["bf16", "bf16", "f16"] + (["f32"] if f32 else []))
    dim = rng.choice([128, 128, 64]) if dtype == "f32" else rng.choice([128, 128, 128, 64, 256])
    return heads, kv, dim, rng.choice([16, 32, 48, 64, 128, 256]), dtype


def _draw_rows(rng, top):
    lo = rng.choice([0, _log(rng, 1, top), _log(rng, 1, top)])
    return lo, max(lo, rng.choice([lo, _log(rng, 1, top)]))


def _draw_write(rng):
    _, kv, dim, page, dtype = _draw_pool(rng)
    lo, hi = _draw_rows(rng, 4000)
    return _write("", _log(rng, 1, 64), _log(rng, 1, 2000), kv, dim, page, lo, hi, dtype)


def _draw_attend(rng, prefix=0):
    heads, kv, dim, page, dtype = _draw_pool(rng)
    lq = rng.choice([1, 1, _log(rng, 2, 128), _log(rng, 2, 128), _log(rng, 100, 1500)])
    lo, hi = _draw_rows(rng, 4000 if prefix else 32768)
    mask = rng.choice(["none", "none", "causal", "block"])
    return _attend("", _log(rng, 2 if prefix else 1, 64), lq, heads, kv, dim, page, lo, hi,
                   prefix=prefix, causal=mask == "causal",
                   block=_log(rng, 1, lq) if mask == "block" else 0, dtype=dtype)


def _draw_shared(rng):
    return _draw_attend(rng, _log(rng, 100, 32768))


def _draw_weights(rng):
    fp4 = rng.random() < 0.5
    heads, kv, dim, page, dtype = _draw_pool(rng, f32=not fp4)
    lq = rng.choice([1, 1, _log(rng, 2, 128), _log(rng, 2, 128), _log(rng, 100, 1500)])
    lo, hi = _draw_rows(rng, 32768)
    return _weights("", _log(rng, 1, 64), lq, heads, kv, dim, page, lo, max(hi, 1), fp4=fp4,
                    dtype=dtype)


def _draw_keep(rng):
    lo, hi = _draw_rows(rng, 40000)
    keep = _log(rng, 1, max(hi, 1))
    return _keep("", _log(rng, 1, 64), rng.choice([24, 40, 8, 4, 12]), lo, max(hi, 1), keep,
                 rng.choice([0, _log(rng, 1, keep), keep]))


def _draw_gather(rng):
    fp4 = rng.random() < 0.5
    _, kv, dim, page, dtype = _draw_pool(rng, f32=not fp4)
    lo, hi = _draw_rows(rng, 16384)
    hi = max(hi, 1)
    return _gather("", _log(rng, 1, 32), kv, dim, page, lo, hi, _log(rng, 1, hi), fp4=fp4,
                   new_pages=rng.random() < 0.5, dtype=dtype)


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
    batch, lens, kv = case["batch"], _lens(case), case["kv_heads"]
    if case["kind"] == "keep":
        # Weights summed over some chunks: a few rows hold most of them.
        w = torch.randn(batch, kv, max(lens), generator=g, device=DEVICE).mul_(2).exp_()
        return {"case": case, "weights": w, "lens": _i32(lens)}
    dt, dim, page = DTYPES[case["dtype"]], case["dim"], case["page"]
    fp4 = case.get("fp4", True)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE).to(dt)

    new = case["n"] if case["kind"] == "write" else 0
    width = max(1, -(-(max(lens) + new) // page))
    prefix = case.get("prefix", 0)
    prefix_pages = -(-prefix // page)
    held = [-(-(n + new) // page) for n in lens]
    kept = -(-case["keep"] // page) if case.get("new_pages") else 0
    # Pages lie anywhere in the pool, a few of which are free; rows past a sequence's end and
    # free pages hold what earlier sequences left there.
    total = sum(held) + prefix_pages + batch * kept + 3
    order = torch.randperm(total, generator=g, device=DEVICE).tolist()
    table = [[order.pop() if j < n else -1 for j in range(width)] for n in held]
    if fp4:
        pool = torch.empty(2, total, kv, page * (dim // 2 + dim // 32), dtype=torch.uint8,
                           device=DEVICE)
        codes, scales = _parts(pool, page, dim)
        for p in range(2):
            c, s = _quantise(rand(total, kv, page, dim), dt)
            codes[p].copy_(c)
            scales[p].copy_(s)
    else:
        pool = rand(2, total, page, kv, dim)
    s = {"case": case, "pages": pool, "table": _i32(table), "lens": _i32(lens), "host_lens": lens,
         "host_table": table}
    if case["kind"] == "write":
        s["k"], s["v"] = rand(batch, new, kv, dim), rand(batch, new, kv, dim)
    elif case["kind"] == "gather":
        # Rows kept: those of the largest of random weights, in order.
        keep = case["keep"]
        score = torch.rand(batch, kv, max(lens), generator=g, device=DEVICE)
        n = s["lens"].long()[:, None, None]
        score.masked_fill_(torch.arange(max(lens), device=DEVICE) >= n, -1.0)
        top, at = score.topk(min(keep, max(lens)), -1)
        at = torch.where(top < 0, max(lens), at).sort(-1).values
        at = torch.where(at >= max(lens), -1, at)
        s["rows"] = torch.full((batch, kv, keep), -1, dtype=torch.int32, device=DEVICE)
        s["rows"][..., :at.shape[-1]] = at
        s["weights"] = torch.rand(batch, kv, width * page, generator=g, device=DEVICE)
        s["host_to"] = [[order.pop() for _ in range(kept)] for _ in range(batch)] if kept else table
        s["to"] = _i32(s["host_to"]) if kept else None
    else:
        lq, heads = case["lq"], case["heads"]
        s["q"] = rand(batch, lq, heads, dim)
        if case["kind"] == "weights":
            # What attention over the cached rows and a few new keys returned.
            x, _ = _scores(case, s)
            lse = torch.logsumexp(x, -1).clamp_(min=-10.0)
            lse = lse + 0.1 * torch.rand(lse.shape, generator=g, device=DEVICE)
            s["lse"] = lse.view(batch, heads, lq).transpose(1, 2).contiguous()
            return s
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
    if kind == "write":
        ops.kv_page_append_fp4(s["pages"], s["k"], s["v"], s["table"], s["lens"])
        return ops.kv_page_read_fp4(s["pages"], s["table"], s["lens"], case["n"], case["dim"],
                                    DTYPES[case["dtype"]])
    if kind == "attend":
        kw = dict(pages=s["pages"], block_table=s["table"], cache_lens=s["lens"],
                  block_boundaries=s["starts"], causal=case["causal"], return_lse=True)
        if not case["prefix"]:
            return ops.paged_attention_fp4(s["q"], s["k"], s["v"], **kw)
        return ops.shared_prefix_attention_fp4(s["q"], s["k"], s["v"], prefix_table=s["prefix_table"],
                                               prefix_len=s["prefix_len"], **kw)
    if kind == "weights":
        return ops.paged_key_weights(s["q"], s["lse"], pages=s["pages"], block_table=s["table"],
                                     cache_lens=s["lens"])
    if kind == "keep":
        return ops.kv_keep_rows(s["weights"], s["lens"], case["keep"], case["recent"])
    ops.kv_page_gather(s["pages"], s["table"], s["rows"], s["to"], s["weights"],
                       head_dim=case["dim"] if case["fp4"] else None)
    return _pool_values(case, s), s["weights"]


def _pool_values(case, s):
    """A pool as it is; of a 4-bit one codes and scale bytes apart, which say what it stands for."""
    return list(_parts(s["pages"], case["page"], case["dim"])) if case["fp4"] else s["pages"]


def _parts(pool, page, dim):
    """Views of a 4-bit pool: codes [2, P, H, R, D / 2], scale bytes [2, P, H, R, D / 32]."""
    at = page * dim // 2
    return (pool[..., :at].unflatten(-1, (page, dim // 2)),
            pool[..., at:].unflatten(-1, (page, dim // 32)))


def _quantise(x, dt):
    """Codes and scale bytes of x [..., D]."""
    lo, hi = (-23, 13) if dt == torch.float16 else (-127, 125)
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    m, e = torch.frexp(top / 7)  # top / 7 in [2^(e - 1), 2^e): rounded, so looked at again
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(top.double() > 7 * torch.exp2(e.double()), e + 1, e)
    e = torch.where(top.double() <= 7 * torch.exp2(e.double() - 1), e - 1, e)
    e = torch.where(top == 0, lo, e).clamp(lo, hi)
    y = b.double().abs() / torch.exp2(e.double())[..., None]
    # Nearest of the eight magnitudes, ties to the even code.
    c = (y > 0.25).to(torch.uint8)
    for i, mid in enumerate((0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        c += (y >= mid) if i % 2 == 0 else (y > mid)
    c += torch.signbit(b).to(torch.uint8) * 8
    c = c.flatten(-2)
    bad = ~torch.isfinite(top)
    return c[..., 0::2] | c[..., 1::2] << 4, torch.where(bad, 255, e + 127).to(torch.uint8)


def _decode(codes, scales):
    """fp32 values [..., D]."""
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device=DEVICE)
    lut = torch.cat((lut, -lut))
    x = lut[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()]
    scale = torch.where(scales == 255, math.nan, torch.exp2(scales.double() - 127)).float()
    return (x.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _cached(case, pool, pages, plane):
    """fp32 rows [B, Hkv, W * R, D] of the pages [B, W]."""
    at = pages.long().clamp(min=0)
    if case.get("fp4", True):
        codes, scales = _parts(pool, case["page"], case["dim"])
        x = _decode(codes[plane][at], scales[plane][at])  # [B, W, H, R, D]
        return x.transpose(1, 2).flatten(2, 3)
    return pool[plane][at].flatten(1, 2).transpose(1, 2).float()


def _queries(case, s):
    """fp32 queries [B, Hkv, group * lq, D]: a K/V head's query heads one after the other."""
    b, lq, heads, dim = s["q"].shape
    return s["q"].float().transpose(1, 2).reshape(b, case["kv_heads"], -1, dim)


def _scores(case, s):
    """Scores of the cached rows [B, Hkv, group * lq, W * R] (-inf past the length), and which exist."""
    q = _queries(case, s)
    keys = _cached(case, s["pages"], s["table"], 0)
    x = torch.bmm(q.flatten(0, 1), keys.flatten(0, 1).transpose(1, 2).contiguous())
    x = x.unflatten(0, q.shape[:2]) / math.sqrt(case["dim"])
    there = torch.arange(keys.shape[2], device=DEVICE) < s["lens"][:, None]
    return x.masked_fill_(~there[:, None, None], -math.inf), there


def _run_plain(kind, case, s):
    if kind == "write":
        return _plain_write(case, s)
    if kind == "attend":
        return _plain_attend(case, s)
    if kind == "weights":
        x, _ = _scores(case, s)
        lse = s["lse"].transpose(1, 2).reshape(*x.shape[:3], 1)
        return torch.exp(x - lse).sum(2)
    if kind == "keep":
        return _plain_keep(case, s)
    return _plain_gather(case, s)


def _plain_write(case, s):
    page, n, dt = case["page"], case["n"], DTYPES[case["dtype"]]
    row = s["lens"].long()[:, None] + torch.arange(n, device=DEVICE)
    at, r = torch.gather(s["table"].long(), 1, row // page), row % page
    codes, scales = _parts(s["pages"], page, case["dim"])
    c, e = _quantise(torch.stack((s["k"], s["v"])), dt)
    codes[:, at, :, r] = c.permute(1, 2, 0, 3, 4)
    scales[:, at, :, r] = e.permute(1, 2, 0, 3, 4)
    x = _decode(codes[:, at, :, r], scales[:, at, :, r]).to(dt)  # [B, n, 2, H, D]
    return x[:, :, 0].contiguous(), x[:, :, 1].contiguous()


def _plain_attend(case, s):
    lq, kv, dim, dt = case["lq"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    batch, group = case["batch"], case["heads"] // case["kv_heads"]
    i = torch.arange(lq, device=DEVICE)
    if case["causal"]:
        end = i + 1
    elif case["block"]:
        end = torch.clamp((i // case["block"] + 1) * case["block"], max=lq)
    else:
        end = torch.full((lq,), lq, device=DEVICE)
    q = _queries(case, s)
    k, v = (s[n].float().transpose(1, 2).flatten(0, 1) for n in "kv")
    x = torch.bmm(q.flatten(0, 1), k.transpose(1, 2).contiguous()).view(batch, kv, group * lq, lq)
    x = x.div_(math.sqrt(dim)).masked_fill_((i[None, :] >= end[:, None]).repeat(group, 1), -math.inf)
    parts = [(x, v)]
    if case["hi"]:
        parts.append((_scores(case, s)[0], _cached(case, s["pages"], s["table"], 1).flatten(0, 1)))
    if case["prefix"]:
        pk, pv = (_cached(case, s["pages"], s["prefix_table"][None], p)[0, :, :case["prefix"]]
                  for p in range(2))
        qs = q.transpose(0, 1).flatten(1, 2)  # [Hkv, B * group * lq, D]
        x = torch.bmm(qs, pk.transpose(1, 2).contiguous()).view(kv, batch, group * lq, -1)
        parts.append((x.div_(math.sqrt(dim)).transpose(0, 1), pv.contiguous()))
    top = torch.stack([x.amax(-1) for x, _ in parts]).amax(0)[..., None]
    total, acc = 0.0, 0.0
    for x, values in parts:
        p = torch.exp(x - top)
        total = total + p.sum(-1, keepdim=True)
        if values.shape[0] == kv and case["prefix"] and values is parts[-1][1]:
            o = torch.bmm(p.transpose(0, 1).flatten(1, 2), values).view(kv, batch, group * lq, dim)
            acc = acc + o.transpose(0, 1)
        else:
            acc = acc + torch.bmm(p.flatten(0, 1), values).view(batch, kv, group * lq, dim)
    out = (acc / total).view(batch, kv * group, lq, dim).transpose(1, 2).contiguous().to(dt)
    lse = (top + torch.log(total)).view(batch, kv * group, lq).transpose(1, 2).contiguous()
    return out, lse


def _plain_keep(case, s):
    keep, recent = case["keep"], min(case["recent"], case["keep"])
    n = s["lens"].long()[:, None, None]
    width = s["weights"].shape[-1]
    row = torch.arange(width, device=DEVICE)
    w = torch.where(row >= n - recent, math.inf, s["weights"])  # (all are finite)
    w = torch.where(row >= n, -math.inf, w)
    at = w.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    at = torch.where(at < n, at, width).sort(-1).values
    rows = torch.full((*at.shape[:2], keep), -1, dtype=torch.int32, device=DEVICE)
    rows[..., :at.shape[-1]] = torch.where(at < width, at, -1)
    return rows


def _plain_gather(case, s):
    page, rows = case["page"], s["rows"].long()
    b, h, i = (rows >= 0).nonzero(as_tuple=True)
    r = rows[b, h, i]
    to = s["table"] if s["to"] is None else s["to"]
    src, dst = s["table"].long()[b, r // page], to.long()[b, i // page]
    if case["fp4"]:
        for part in _parts(s["pages"], page, case["dim"]):
            part[:, dst, h, i % page] = part[:, src, h, r % page]
    else:
        s["pages"][:, dst, i % page, h] = s["pages"][:, src, r % page, h]
    w = s["weights"][b, h, r]
    s["weights"].zero_()
    s["weights"][b, h, i] = w
    return _pool_values(case, s), s["weights"]


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
    lens, kv = _lens(case), case["kv_heads"]
    kept = [min(n, case.get("keep", 0)) for n in lens]
    if case["kind"] == "keep":
        # The kept rows' weights and numbers.
        return {"bytes": 4 * kv * (sum(lens) + len(lens) * case["keep"]) + 4 * len(lens), "flops": 0}
    page, dim = case["page"], case["dim"]
    es = 4 if case["dtype"] == "f32" else 2
    row = kv * dim * es  # a key (or a value) of every head
    held = kv * (dim // 2 + dim // 32) if case.get("fp4", True) else row  # as the cache holds it
    if case["kind"] == "write":
        n = case["n"]
        entries = sum(-(-(c + n) // page) - c // page for c in lens)
        return {"bytes": 2 * len(lens) * n * (2 * row + 2 * held) + 8 * (entries + len(lens)),
                "flops": 0}
    if case["kind"] == "gather":
        return {"bytes": sum(kept) * (4 * held + 12 * kv), "flops": 0}
    lq, prefix = case["lq"], case.get("prefix", 0)
    entries = sum(-(-c // page) for c in lens) + -(-prefix // page)
    queries = len(lens) * lq * case["heads"]
    if case["kind"] == "weights":
        return {"bytes": queries * (dim * es + 4) + sum(lens) * (held + 4 * kv) + 4 * entries,
                "flops": 2 * dim * case["heads"] * lq * sum(lens)}
    pairs = sum(_pairs(lq, prefix + c, case["block"], case["causal"]) for c in lens)
    return {"bytes": queries * (2 * dim * es + 4) + 2 * len(lens) * lq * row +
            2 * held * (prefix + sum(lens)) + 4 * (entries + len(lens)),
            "flops": 4 * dim * case["heads"] * pairs}


# ---------------------------------------------------------------------------
# The definition in 64 bits: one (sequence, head) at a time, rows found row by row.
# ---------------------------------------------------------------------------
def _slots(table, count, page):
    """Row index in the pool's (page, row) axis of rows 0..count-1 of a sequence."""
    return torch.tensor([table[r // page] * page + r % page for r in range(count)],
                        dtype=torch.long, device=DEVICE)


def _stored(case, pool, plane, head, slots):
    """fp64 rows [n, D] of a head, a 4-bit one's from the bits of its codes."""
    page, dim = case["page"], case["dim"]
    if not case.get("fp4", True):
        return pool[plane, :, :, head].flatten(0, 1)[slots].double()
    block = pool[plane, :, head]
    page_of, row_of = slots // page, slots % page
    at = row_of[:, None] * (dim // 2) + torch.arange(dim // 2, device=DEVICE)
    byte = block[page_of[:, None], at].long()
    nibble = torch.stack((byte % 16, byte // 16), 2).reshape(len(slots), dim)
    sign, power, half = nibble // 8, nibble // 2 % 4, nibble % 2
    size = torch.where(power == 0, 0.5 * half, (1 + 0.5 * half) * 2.0 ** (power - 1).double())
    at = page * dim // 2 + row_of[:, None] * (dim // 32) + torch.arange(dim // 32, device=DEVICE)
    scale = block[page_of[:, None], at].double()
    scale = torch.where(scale == 255, math.nan, 2.0 ** (scale - 127)).repeat_interleave(32, 1)
    return (1 - 2 * sign) * size * scale


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "keep":
        return _exact_keep(case, s)
    if case["kind"] == "gather":
        return _exact_gather(case, s)
    if case["kind"] == "write":
        return tuple(_exact_stored(case, s[n]) for n in "kv")
    page, group = case["page"], case["heads"] // case["kv_heads"]
    lq, scale = case["lq"], case["dim"] ** -0.5
    if case["kind"] == "weights":
        got = torch.zeros(case["batch"], case["kv_heads"], len(s["host_table"][0]) * page,
                          dtype=torch.float64, device=DEVICE)
        for b, n in enumerate(s["host_lens"]):
            slots = _slots(s["host_table"][b], n, page)
            for h in range(case["kv_heads"]):
                kt = _stored(case, s["pages"], 0, h, slots).t().contiguous()
                for e in range(h * group, (h + 1) * group):
                    x = s["q"][b, :, e].double() @ kt * scale - s["lse"][b, :, e, None].double()
                    got[b, h, :n] += x.exp().sum(0)
        return got
    shared = _slots(s["host_prefix"], case["prefix"], page) if case["prefix"] else None
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    lse = torch.empty(s["q"].shape[:3], dtype=torch.float64, device=DEVICE)
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
            kh, vh = (torch.cat((_stored(case, s["pages"], p, h, slots), s["kv"[p]][b, :, h].double()))
                      for p in range(2))
            kt = kh.t().contiguous()
            for e in range(h * group, (h + 1) * group):
                x = torch.where(seen, s["q"][b, :, e].double() @ kt * scale,
                                torch.tensor(-math.inf, dtype=torch.float64, device=DEVICE))
                out[b, :, e] = torch.softmax(x, 1) @ vh
                lse[b, :, e] = torch.logsumexp(x, 1)
    return out, lse


def _exact_stored(case, x):
    """What a row reads as once written: the nearest of all values that its block can hold."""
    lo, hi = (-23, 13) if case["dtype"] == "f16" else (-127, 125)
    sizes = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEVICE)
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    power = torch.full_like(top, float(lo))
    for e in range(lo, hi):  # while even 7 of this power are too few, the next one
        power = torch.where(top > 7 * 2.0 ** e, float(e + 1), power)
    y = b.abs() / 2.0 ** power
    best, off = torch.zeros_like(y), y.clone()
    for i in range(1, 8):
        d = (y - sizes[i]).abs()
        better = (d < off) | ((d == off) if i % 2 == 0 else torch.zeros_like(y, dtype=torch.bool))
        best, off = torch.where(better, sizes[i], best), torch.where(better, d, off)
    return (best * 2.0 ** power * torch.where(b < 0, -1.0, 1.0)).flatten(-2)


def _exact_keep(case, s):
    keep = case["keep"]
    rows = torch.full((case["batch"], case["kv_heads"], keep), -1, dtype=torch.int32)
    weights = s["weights"].cpu()
    for b, n in enumerate(_lens(case)):
        count = min(n, keep)
        last = min(case["recent"], count)
        for h in range(case["kv_heads"]):
            w = weights[b, h, :n - last].tolist()
            best = sorted(range(n - last), key=lambda r: (-w[r], r))[:count - last]
            rows[b, h, :count] = torch.tensor(sorted(best) + list(range(n - last, n)),
                                              dtype=torch.int32)
    return rows.to(DEVICE)


def _exact_gather(case, s):
    page, h = case["page"], torch.arange(case["kv_heads"], device=DEVICE)
    before, after = s["pages"].clone(), s["pages"]
    old, weights = s["weights"].clone(), torch.zeros_like(s["weights"])
    rows = s["rows"].long()
    per, tail = case["dim"] // 2, case["dim"] // 32

    def columns(r):  # byte columns of row r of a head's block, [H, D / 2 + D / 32]
        return torch.cat((r[:, None] * per + torch.arange(per, device=DEVICE),
                          page * per + r[:, None] * tail + torch.arange(tail, device=DEVICE)), 1)

    for b, to in enumerate(s["host_to"]):
        table = torch.tensor(s["host_table"][b], device=DEVICE)
        for i in range(min(case["keep"], s["host_lens"][b])):
            r = rows[b, :, i]
            weights[b, h, i] = old[b, h, r]
            p = table[r // page]
            if case["fp4"]:
                x = before[:, p[:, None], h[:, None], columns(r % page)]
                after[:, to[i // page], h[:, None], columns(torch.full_like(r, i % page))] = x
            else:
                after[:, to[i // page], i % page] = before[:, p, r % page, h]
    return _pool_values(case, s), weights
