"""Dense operators over the paged cache: the work that a serving loop has them do.

``extend``   new tokens of a ragged batch go into the cache's pages, keys and queries rotated to
             their positions on the way, the pages' key bounds and the counts kept
             (``paged.extend``)
``attend``   attention of each request's newest tokens over its whole cache: decode, chunks of a
             prompt, whole prompts; scores capped or biased by distance; window, prefix and
             document masks (``paged.attention``)
``shared``   one decode token per request, where groups of requests share their leading blocks
             (``paged.shared_attention``)

A case is a dict of plain values.  With ``own`` false the operators run in their plain form:
elementary torch operations in 32 bits, rounded once.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "strict-topk-overlap_amd"))

own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"


# ----------------------------------------------------------------- cases

def _case(op, hq, hkv, d, b, requests, new, low, high, **more):
    """``requests`` requests of ``low`` to ``high`` tokens (their new ones counted), ``new``
    new tokens in all (or one each)."""
    c = dict(op=op, hq=hq, hkv=hkv, d=d, b=b, requests=requests, new=new, low=low, high=high,
             dtype="bf16")
    if op == "extend":
        c.update(rot=d, interleaved=False)
    else:
        c.update(softcap=0.0, alibi=False, window=0)
    if op == "attend":
        c.update(prefix=0, document=0)
    if op == "shared":
        c.update(groups=1, prefix_blocks=0)
    c.update(more)
    return c


def listed():
    cs = {
        # a small model's decode step, two requests: all launch and host latency
        "extend_decode_small": _case("extend", 16, 8, 128, 32, 2, 2, 500, 1000),
        # a serving batch's decode step
        "extend_decode_batch": _case("extend", 32, 8, 128, 32, 128, 128, 700, 20000),
        # a batch of prompts and chunks of prompts, half-rotated heads with paired elements
        "extend_prefill": _case("extend", 32, 8, 128, 32, 5, 8191, 900, 9000, dtype="fp16",
                                rot=64, interleaved=True),
        # one request decodes at 16K context
        "attend_decode_one": _case("attend", 16, 8, 128, 32, 1, 1, 16000, 16000),
        # the ragged decode batch: 8K to 128K tokens per request
        "attend_decode_ragged": _case("attend", 32, 8, 128, 32, 16, 16, 8192, 131000),
        # a short prompt of a small model
        "attend_prompt_short": _case("attend", 4, 4, 64, 32, 1, 301, 301, 301, dtype="fp16"),
        # a whole prompt, causal
        "attend_prompt": _case("attend", 32, 8, 128, 32, 1, 8192, 8192, 8192),
        # chunks of three prompts, capped scores and a window over large heads
        "attend_chunk_capped": _case("attend", 16, 8, 256, 32, 3, 2900, 2000, 12000,
                                     softcap=50.0, window=4096),
        # packed documents with a distance bias, odd lengths
        "attend_documents": _case("attend", 24, 4, 128, 16, 4, 5001, 1500, 6001, alibi=True,
                                  document=1024),
        # a few requests over one system prompt
        "shared_small": _case("shared", 16, 8, 128, 32, 6, 6, 20, 300, prefix_blocks=64),
        # a large batch over one long prefix
        "shared_large": _case("shared", 32, 8, 128, 32, 96, 96, 1, 2000, prefix_blocks=1024),
        # several prefixes, scores capped, small heads
        "shared_groups": _case("shared", 64, 8, 64, 64, 40, 40, 30, 900, groups=3,
                               prefix_blocks=130, softcap=30.0, dtype="fp16"),
    }
    return [dict(c, name=name) for name, c in cs.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges, at most as much work as the largest of its
    operator."""
    c = _draw(rng)
    most = {"extend": 0.0, "attend": 0.0, "shared": 0.0}
    for x in listed():
        most[x["op"]] = max(most[x["op"]], _cost(x))
    while _cost(c) > most[c["op"]]:
        size = rng.choice(["new", "high", "requests"])
        if size == "requests" and c["requests"] > 1:
            c["requests"] -= -(-c["requests"] // 8)
        elif size == "new" and c["new"] > c["requests"]:
            c["new"] -= -(-(c["new"] - c["requests"]) // 4)
        elif size == "high":
            c["high"] -= c["high"] // 8
            c["low"] = min(c["low"], c["high"])
        if c["op"] == "shared":
            c["prefix_blocks"] -= c["prefix_blocks"] // 8
            c["groups"] = min(c["groups"], c["requests"])
            c["new"] = c["requests"]
        c["new"] = max(c["new"], c["requests"]) if c["op"] != "shared" else c["requests"]
    return c


def _cost(c):
    w = work(c)
    return w["bytes"] / 5e12 + w["flops"] / 8e14


def _draw(rng):
    op = rng.choice(["extend", "attend", "attend", "shared"])
    d = rng.choice([64, 128, 128, 128, 256])
    hq, hkv = rng.choice([(4, 4), (8, 8), (16, 8), (32, 8), (40, 8), (64, 8), (16, 2), (24, 4),
                          (48, 4)])
    b = rng.choice([16, 32, 32, 64])
    kw = dict(dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op == "extend":
        r = _log(rng, 1, 128)
        new = r if rng.random() < 0.5 else r + _log(rng, 10, 8191)
        low = _log(rng, 100, 4000)
        return _case(op, hq, hkv, d, b, r, new, low, low + _log(rng, 100, 16000),
                     rot=rng.choice([d, d, d // 2]), interleaved=rng.random() < 0.3, **kw)
    if rng.random() < 0.3:
        kw["softcap"] = rng.choice([15.0, 30.0, 50.0])
    elif rng.random() < 0.3:
        kw["alibi"] = True
    if op == "shared":
        r = _log(rng, 2, 128)
        if rng.random() < 0.2:
            kw["window"] = _log(rng, 500, 20000)
        return _case(op, hq, hkv, d, b, r, r, rng.randint(1, 200), _log(rng, 200, 2000),
                     groups=min(r, rng.choice([1, 1, 2, 3, 5])),
                     prefix_blocks=_log(rng, 1000, 32768) // b, **kw)
    mask = rng.choice(["none", "none", "window", "prefix", "document"])
    if mask == "window":
        kw["window"] = _log(rng, 200, 8000)
    if rng.random() < 0.5:                       # single tokens
        r = _log(rng, 1, 64)
        low = _log(rng, 200, 16000)
        return _case(op, hq, hkv, d, b, r, r, low, low + _log(rng, 500, 115000), **kw)
    r = _log(rng, 1, 6)
    high = _log(rng, 100, 12000)
    new = r + rng.randint(high // 4, high)
    if mask == "prefix":
        kw["prefix"] = _log(rng, 50, 2000)
    if mask == "document":
        kw["document"] = _log(rng, 60, 2000)
    return _case(op, hq, hkv, d, b, r, new, max(50, high // 3), max(50, high), **kw)


def _lengths(c):
    """Tokens (their new ones counted) and new tokens of each request.  Lengths run over
    [low, high] in a scattered order, both ends taken; with ``shared`` they count the tokens
    behind the shared blocks."""
    r = c["requests"]
    at = [(i * 0.6180339887) % 1.0 for i in range(r)]
    if r > 1:
        at[at.index(min(at))], at[at.index(max(at))] = 0.0, 1.0
    else:
        at = [1.0]
    ns = [round(c["low"] * (c["high"] / c["low"]) ** x) for x in at]
    left, news = c["new"], []
    for i in range(r):                       # uneven shares, at least one token each
        share = left - (r - 1 - i) if i == r - 1 else \
            min(left - (r - 1 - i), max(1, round(left / (r - i) * (0.6 + 0.8 * at[i]))))
        news.append(share)
        left -= share
    ns = [max(n, m) for n, m in zip(ns, news)]
    if c["op"] == "shared":
        pre = c["prefix_blocks"] * c["b"]
        ns = [n + pre for n in ns]
    return ns, news


def _group_starts(c):
    g, r = c["groups"], c["requests"]
    return [i * r // g for i in range(g + 1)]


def _ranges(c):
    """Per request the visible keys [lo, hi) of each new token."""
    out = []
    for n, m in zip(*_lengths(c)):
        p = np.arange(n - m, n, dtype=np.int64)
        lo, hi = np.zeros_like(p), p + 1
        if c["window"]:
            lo = np.maximum(lo, p - c["window"] + 1)
        if c.get("document"):
            lo = np.maximum(lo, p // c["document"] * c["document"])
        if c.get("prefix"):
            hi = np.maximum(hi, min(c["prefix"], n))
        out.append((lo, hi))
    return out


def work(c):
    e = 2
    ns, news = _lengths(c)
    t = sum(news)
    if c["op"] == "extend":
        pages = sum((n - 1) // c["b"] - (n - m) // c["b"] + 1 for n, m in zip(ns, news)) * c["hkv"]
        heads = c["hq"] + 2 * c["hkv"]
        return {"bytes": t * (2 * heads * c["d"] * e + c["rot"] * 4) +
                pages * (2 * c["d"] * e + 4),
                "flops": 3 * t * (c["hq"] + c["hkv"]) * c["rot"]}
    pairs, keys = 0, 0
    spans = _ranges(c)
    for lo, hi in spans:
        pairs += int((hi - lo).sum())
        keys += int(hi.max() - lo.min())
    if c["op"] == "shared":                  # shared blocks are read once per group
        pre, gs = c["prefix_blocks"] * c["b"], _group_starts(c)
        for g in range(c["groups"]):
            seen = [max(0, pre - int(lo[0])) for lo, _ in spans[gs[g]:gs[g + 1]]]
            keys -= sum(seen) - max(seen)
    return {"bytes": keys * c["hkv"] * c["d"] * 2 * e + 2 * t * c["hq"] * c["d"] * e,
            "flops": 4 * c["d"] * c["hq"] * pairs}


# ---------------------------------------------------------------- inputs

class _State:
    """What the program holds: plain attributes."""


def _slopes(hq):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)], device=DEV)


def _pool(c, gen, blocks, s):
    """A page pool with ``blocks[r]`` blocks per request in scattered order; with ``shared`` the
    leading blocks of a group stand once in the pool."""
    hkv, b, d, dt = c["hkv"], c["b"], c["d"], DTYPES[c["dtype"]]
    r, pre = len(blocks), c.get("prefix_blocks", 0)
    gs = _group_starts(c) if c["op"] == "shared" else list(range(r + 1))
    total = sum(n - pre for n in blocks) * hkv + (len(gs) - 1) * pre * hkv
    perm = torch.randperm(total, generator=gen, device=DEV).to(torch.int32).cpu()
    table = torch.full((r, hkv, max(blocks)), -1, dtype=torch.int32)
    at = 0
    for g in range(len(gs) - 1):
        table[gs[g]:gs[g + 1], :, :pre] = perm[at:at + hkv * pre].view(hkv, pre)
        at += hkv * pre
        for i in range(gs[g], gs[g + 1]):
            n = blocks[i] - pre
            table[i, :, pre:blocks[i]] = perm[at:at + hkv * n].view(hkv, n)
            at += hkv * n
    s.k_pages = torch.empty((total, b, d), dtype=dt, device=DEV)
    s.v_pages = torch.empty_like(s.k_pages)
    for x in (s.k_pages, s.v_pages):
        x.view(-1).normal_(generator=gen)
    s.lo = torch.empty((total, d), dtype=dt, device=DEV).normal_(generator=gen).abs_().neg_()
    s.hi = torch.empty_like(s.lo).normal_(generator=gen).abs_()
    s.table = table.to(DEV)


def prepare(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    s = _State()
    s.case, dt = c, DTYPES[c["dtype"]]
    hq, hkv, d, b = c["hq"], c["hkv"], c["d"], c["b"]
    ns, news = _lengths(c)
    s.ns, s.news, t = ns, news, sum(news)
    blocks = [-(-n // b) for n in ns]
    _pool(c, gen, blocks, s)
    starts = np.concatenate(([0], np.cumsum(news)))
    s.host_starts = [int(x) for x in starts]
    s.starts = torch.tensor(s.host_starts, dtype=torch.int32, device=DEV)
    if c["op"] == "extend":
        old = [n - m for n, m in zip(ns, news)]
        s.nblocks = torch.tensor([-(-n // b) for n in old], dtype=torch.int32, device=DEV)
        s.ntokens = torch.tensor(old, dtype=torch.int32, device=DEV)
        s.positions = s.ntokens.clone()
        # one fused projection's output: queries, keys and values of a token side by side
        qkv = torch.empty((t, (hq + 2 * hkv) * d), device=DEV, dtype=dt).normal_(generator=gen)
        s.q = qkv[:, :hq * d].view(t, hq, d)
        s.k = qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
        s.v = qkv[:, (hq + hkv) * d:].view(t, hkv, d)
        half = c["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
        ang = torch.arange(max(blocks) * b, dtype=torch.float64, device=DEV)[:, None] * freq
        s.cos, s.sin = ang.cos().float(), ang.sin().float()
    else:
        s.nblocks = torch.tensor(blocks, dtype=torch.int32, device=DEV)
        s.ntokens = torch.tensor(ns, dtype=torch.int32, device=DEV)
        s.q = torch.empty((t, hq, d), device=DEV, dtype=dt).normal_(generator=gen)
        s.slopes = _slopes(hq) if c["alibi"] else None
        s.prefix = s.first = None
        if c.get("prefix"):
            s.prefix = torch.tensor([min(c["prefix"], n) for n in ns], dtype=torch.int32,
                                    device=DEV)
        if c.get("document"):
            p = np.concatenate([np.arange(n - m, n) for n, m in zip(ns, news)])
            s.first = torch.tensor(p // c["document"] * c["document"], dtype=torch.int32,
                                   device=DEV)
        if c["op"] == "shared":
            s.groups = torch.tensor(_group_starts(c), dtype=torch.int32, device=DEV)
            s.shared = torch.full((c["groups"],), c["prefix_blocks"], dtype=torch.int32,
                                  device=DEV)
    if own:
        from strict_topk import paged
        s.kv = paged.PagedKV(s.k_pages, s.v_pages, s.lo, s.hi, s.table, s.nblocks, s.ntokens)
    return s


# ------------------------------------------------------------ one pass

def run(s):
    c = s.case
    if not own:
        return _plain_extend(s) if c["op"] == "extend" else _plain_attention(s)
    from strict_topk import paged
    if c["op"] == "extend":
        q = paged.extend(s.kv, s.k, s.v, s.starts, s.positions, s.cos, s.sin, q=s.q,
                         interleaved=c["interleaved"])
        return (q, s.k_pages, s.v_pages, s.lo, s.hi, s.nblocks, s.ntokens)
    if c["op"] == "shared":
        return paged.shared_attention(s.q, s.kv, s.groups, s.shared, softcap=c["softcap"],
                                      slopes=s.slopes, window=c["window"])
    return paged.attention(s.q, s.kv, None if c["new"] == c["requests"] else s.starts,
                           softcap=c["softcap"], slopes=s.slopes, window=c["window"],
                           prefix=s.prefix, first=s.first)


def _rotate(x, cos, sin, rot, interleaved):
    """x[T, H, D] in 32 bits rotated by cos, sin[T, rot / 2]."""
    cos, sin = cos[:, None], sin[:, None]
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2] = a * cos - b * sin
        out[..., 1:rot:2] = b * cos + a * sin
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out[..., :rot // 2] = a * cos - b * sin
        out[..., rot // 2:rot] = b * cos + a * sin
    return out


def _plain_extend(s):
    c, dt = s.case, s.q.dtype
    b = c["b"]
    t = s.q.shape[0]
    row = torch.arange(t, device=DEV)
    req = torch.searchsorted(s.starts[1:].contiguous(), row.to(torch.int32), right=True)
    pos = (s.positions[req] + row - s.starts[req]).long()
    cos, sin = s.cos[pos], s.sin[pos]
    q = _rotate(s.q.float(), cos, sin, c["rot"], c["interleaved"]).to(dt)
    k = _rotate(s.k.float(), cos, sin, c["rot"], c["interleaved"]).to(dt)
    blk, off = pos // b, pos % b
    pages = s.table[req, :, blk].long()                   # [T, Hkv]
    s.k_pages[pages, off[:, None]] = k
    s.v_pages[pages, off[:, None]] = s.v
    # bounds: a block that starts with a new token starts over, the others widen
    fresh = pages[off == 0].reshape(-1)
    s.lo[fresh] = math.inf
    s.hi[fresh] = -math.inf
    idx = pages.reshape(-1, 1).expand(-1, c["d"])
    flat = k.reshape(-1, c["d"])
    s.lo.scatter_reduce_(0, idx, flat, "amin")
    s.hi.scatter_reduce_(0, idx, flat, "amax")
    s.ntokens.copy_(s.positions + s.starts[1:] - s.starts[:-1])
    s.nblocks.copy_((s.ntokens + b - 1) // b)
    return (q, s.k_pages, s.v_pages, s.lo, s.hi, s.nblocks, s.ntokens)


def _gather(s, pages, table, r, n):
    """Keys or values [Hkv, n, D] of request r in 32 bits."""
    c = s.case
    nb = -(-n // c["b"])
    x = pages[table[r, :, :nb].long()]
    return x.reshape(c["hkv"], nb * c["b"], c["d"])[:, :n].float()


def _plain_attention(s):
    c = s.case
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    g, scale = hq // hkv, 1.0 / math.sqrt(d)
    out = torch.empty_like(s.q)
    for r, (n, m) in enumerate(zip(s.ns, s.news)):
        a = s.host_starts[r]
        k = _gather(s, s.k_pages, s.table, r, n)
        v = _gather(s, s.v_pages, s.table, r, n)
        q = s.q[a:a + m].float().view(m, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * m, d)
        x = (q @ k.transpose(1, 2)).view(hkv, g, m, n) * scale
        if c["softcap"]:
            x = torch.tanh(x / c["softcap"]) * c["softcap"]
        p = torch.arange(n - m, n, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)[None]
        if s.slopes is not None:
            x -= s.slopes.view(hkv, g, 1, 1) * (p - j).abs()
        top = p + 1
        if s.prefix is not None:
            top = torch.maximum(top, s.prefix[r])
        seen = j < top
        if c["window"]:
            seen &= j > p - c["window"]
        if s.first is not None:
            seen &= j >= s.first[a:a + m, None]
        x = torch.where(seen, x, -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True))
        x /= x.sum(-1, keepdim=True)
        o = (x.view(hkv, g * m, n) @ v).view(hkv, g, m, d)
        out[a:a + m] = o.permute(2, 0, 1, 3).reshape(m, hq, d).to(out.dtype)
    return out


# -------------------------------------------- the definitions in 64 bits

def exact(c, seed):
    s = prepare(c, seed)
    return _exact_extend(s) if c["op"] == "extend" else _exact_attention(s)


def _exact_extend(s):
    c, b, half = s.case, s.case["b"], s.case["rot"] // 2
    q, kp, vp = s.q.double(), s.k_pages.double(), s.v_pages.double()
    lo, hi = s.lo.double(), s.hi.double()
    i = torch.arange(half, device=DEV)
    even, odd = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    for r, (n, m) in enumerate(zip(s.ns, s.news)):
        at, p0 = s.host_starts[r], n - m
        ang_c, ang_s = s.cos[p0:n].double()[:, None], s.sin[p0:n].double()[:, None]
        k = s.k[at:at + m].double()
        for x in (q[at:at + m], k):
            z = torch.complex(x[..., even], x[..., odd]) * torch.complex(ang_c, ang_s)
            x[..., even], x[..., odd] = z.real, z.imag
        v = s.v[at:at + m].double()
        for j in range(p0 // b, (n - 1) // b + 1):
            t0, t1 = max(p0, j * b), min(n, j * b + b)
            pages = s.table[r, :, j].long()
            part = k[t0 - p0:t1 - p0].transpose(0, 1)
            kp[pages, t0 - j * b:t1 - j * b] = part
            vp[pages, t0 - j * b:t1 - j * b] = v[t0 - p0:t1 - p0].transpose(0, 1)
            low, high = part.min(1).values, part.max(1).values
            lo[pages] = low if t0 == j * b else torch.minimum(lo[pages], low)
            hi[pages] = high if t0 == j * b else torch.maximum(hi[pages], high)
    return (q, kp, vp, lo, hi,
            torch.tensor([-(-n // b) for n in s.ns], dtype=torch.int32, device=DEV),
            torch.tensor(s.ns, dtype=torch.int32, device=DEV))


def _exact_attention(s):
    """Head by head; the log of the sum of exponentials first, then the weighted values."""
    c, b = s.case, s.case["b"]
    hq, d = c["hq"], c["d"]
    g = hq // c["hkv"]
    out = torch.empty(s.q.shape, dtype=torch.float64, device=DEV)
    spans = _ranges(c)
    for r, (n, m) in enumerate(zip(s.ns, s.news)):
        at, nb = s.host_starts[r], -(-n // b)
        low, high = (torch.from_numpy(x).to(DEV)[:, None] for x in spans[r])
        j = torch.arange(n, device=DEV)
        hidden = (j < low) | (j >= high)
        dist = (torch.arange(n - m, n, device=DEV)[:, None] - j).abs().double()
        for h in range(c["hkv"]):
            pages = s.table[r, h, :nb].long()
            k = s.k_pages[pages].reshape(-1, d)[:n].double()
            v = s.v_pages[pages].reshape(-1, d)[:n].double()
            for i in range(h * g, h * g + g):
                x = (s.q[at:at + m, i].double() @ k.T) / d ** 0.5
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                if s.slopes is not None:
                    x = x - float(s.slopes[i]) * dist
                x = x.masked_fill(hidden, -math.inf)
                x = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
                out[at:at + m, i] = x @ v
    return out
