"""Plain 64-bit forms of the dense operators over the paged cache, and builders
of their inputs (used by test_gpu_dense.py and test_gpu_extend.py).

Tolerances.  Outputs are rounded once to 16 bits: half a step, eps / 2 of the
value.  The weights are rounded to 16 bits before they multiply the values:
each moves the output by at most eps / 2 of its share, eps / 2 * A in all, with A
= sum p |v| / sum p.  A score is a sum of D products in FP32, at most (D + 8)
2^-24 sum |q k| scale off, and its exponent's argument and the hardware
exponential add a few steps of the score's size; a score off by s moves the
output by at most 2 s A.  Sums of n weights in FP32 are at most n 2^-24 off,
relative to themselves, in numerator and denominator.
"""
import torch

from strict_topk import paged


class Cache:
    """A pool and its logical contents: k, v [R][Hkv, blocks, B, D] in 64 bits on the CPU."""


def make(hkv, d, b, lens, dtype, seed=1, width=None, bounds=None, spare=3, device="cuda"):
    gen = torch.Generator().manual_seed(seed)
    blocks = [-(-n // b) for n in lens]
    width = max(1, max(blocks)) if width is None else width
    total = hkv * sum(blocks)
    order = torch.randperm(total + spare, generator=gen)[:total]
    k = torch.randn((total + spare, b, d), generator=gen).to(dtype)
    v = torch.randn((total + spare, b, d), generator=gen).to(dtype)
    table = torch.full((len(lens), hkv, width), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(blocks):
        table[r, :, :n] = order[at:at + hkv * n].view(hkv, n).to(torch.int32)
        at += hkv * n
    bounds = dtype if bounds is None else bounds
    lo, hi = k.amin(1).to(bounds), k.amax(1).to(bounds)
    dev = torch.device(device)
    return paged.PagedKV(k.to(dev), v.to(dev), lo.to(dev), hi.to(dev), table.to(dev),
                         torch.tensor(blocks, dtype=torch.int32, device=dev),
                         torch.tensor(lens, dtype=torch.int32, device=dev))


def gather(kv, r, h, n):
    """Keys, values [n, D] of request r's KV head h in 64 bits, and which keys have a page."""
    b, table = kv.block, kv.block_table[r, h].cpu()
    nb = -(-n // b)
    page = table[:nb].long()
    ok = (page >= 0) & (page < kv.pages)
    idx = torch.where(ok, page, 0).to(kv.k_pages.device)
    k = kv.k_pages[idx].double().cpu().reshape(-1, kv.dim)[:n]
    v = kv.v_pages[idx].double().cpu().reshape(-1, kv.dim)[:n]
    return k, v, ok.repeat_interleave(b)[:n]


def attention(q, kv, news, scale=None, softcap=0.0, slopes=None, window=0, prefix=None,
              first=None):
    """Output and tolerance [T, Hq, D] in 64 bits."""
    hq, d = q.shape[1:]
    g, scale = hq // kv.hkv, d ** -0.5 if scale is None else scale
    eps = torch.finfo(q.dtype).eps
    q64 = q.double().cpu()
    out = torch.zeros(q64.shape, dtype=torch.float64)
    tol = torch.zeros_like(out)
    full = [min(max(x, 0), kv.width) * kv.block for x in kv.nblocks.tolist()]
    ns = full if kv.ntokens is None else [min(max(x, 0), f)
                                          for x, f in zip(kv.ntokens.tolist(), full)]
    at = 0
    for r, m in enumerate(news):
        n = ns[r]
        for h in range(kv.hkv):
            k, v, ok = gather(kv, r, h, n)
            k = torch.where(ok[:, None], k, 0.)
            for t in range(m):
                p = n - m + t
                lo = max(0, p - window + 1) if window else 0
                if first is not None:
                    lo = max(lo, int(first[at + t]))
                hi = min(p + 1, n)
                if prefix is not None:
                    hi = max(hi, min(int(prefix[r]), n))
                if hi <= lo or not bool(ok[lo:hi].any()):
                    continue
                sel = torch.arange(lo, hi)[ok[lo:hi]]
                kk, vv = k[sel], v[sel]
                qq = q64[at + t, h * g:h * g + g]
                s = (qq @ kk.T) * scale
                off = (d + 8) * 2.0 ** -24 * scale * (qq.abs() @ kk.abs().T)
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                    off = off + softcap * 2.0 ** -21
                if slopes is not None:
                    s = s - slopes.double().cpu()[h * g:h * g + g, None] * (p - sel).abs()
                off = off + (s.abs() + s.abs().amax(-1, keepdim=True) + 16) * 2.0 ** -21
                w = torch.softmax(s, -1)
                o = w @ vv
                a = w @ vv.abs()
                ds = off.amax(-1, keepdim=True)
                out[at + t, h * g:h * g + g] = o
                tol[at + t, h * g:h * g + g] = eps / 2 * o.abs() + \
                    a * (eps / 2 + 2 * ds + 2 * len(sel) * 2.0 ** -24) * 1.01 + \
                    torch.finfo(q.dtype).smallest_normal * eps
        at += m
    return out, tol


def check(got, ref, tol):
    err = (got.double().cpu() - ref).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(err.nan_to_num(1e30).max()),
                                 float(tol.max()), bad.nonzero()[:4].tolist())


def starts_of(news, device="cuda"):
    s = [0]
    for m in news:
        s.append(s[-1] + m)
    return torch.tensor(s, dtype=torch.int32, device=device)


def queries(t, hq, d, dtype, seed=7, device="cuda"):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn((t, hq, d), generator=gen).to(dtype).to(device)


def slopes_of(hq, device="cuda"):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)], device=device)


def tables(rows, rot, device="cuda"):
    half = rot // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    return ang.cos().float().to(device), ang.sin().float().to(device)


def rotate(x, pos, cos, sin, interleaved):
    """x[T, H, D] in 64 bits rotated to pos [T], and the size of the terms."""
    rot = 2 * cos.shape[1]
    c, s = cos.double().cpu()[pos][:, None], sin.double().cpu()[pos][:, None]
    y, size = x.clone(), x.abs()
    i = torch.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, size


