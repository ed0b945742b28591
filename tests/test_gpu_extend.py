"""New tokens into the paged cache (paged.extend) against a plain 64-bit form,
and a run of the dense operators together with the sparse steps, as a serving
loop has them."""
import pytest
import torch

from strict_topk import paged
from tests import dense_ref as R

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _tokens(t, hq, hkv, d, dtype, seed=3):
    fused = R.queries(t, hq + 2 * hkv, d, dtype, seed=seed)
    return fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:]


def _close(got, ref, size, dtype):
    """One rounding to 16 bits of two products and a sum in FP32."""
    eps = torch.finfo(dtype).eps
    err = (got.double().cpu() - ref).abs()
    tol = eps / 2 * ref.abs() * (1 + 2.0 ** -10) + 2.0 ** -22 * size + \
        torch.finfo(dtype).smallest_normal * eps
    assert bool((err <= tol).all()), float((err - tol).max())


def _check(kv, old, q, k, v, news, positions, cos, sin, inter, qout):
    """Every page, bound and count against the plain form; ``old`` the state before."""
    b, dtype = kv.block, kv.k_pages.dtype
    kp, vp = old.k_pages.double().cpu(), old.v_pages.double().cpu()
    size = torch.zeros_like(kp)
    lo, hi = old.lo_pages.double().cpu(), old.hi_pages.double().cpu()
    bsize = torch.zeros_like(lo)
    nb, nt = old.nblocks.tolist(), old.ntokens.tolist()
    table = kv.block_table.cpu()
    at, room = 0, kv.width * b
    for r, m in enumerate(news):
        pos = torch.arange(positions[r], positions[r] + m)
        ok = (pos >= 0) & (pos < room)
        rows = torch.arange(at, at + m)[ok]
        p = pos[ok]
        k64, v64, q64 = (x.double().cpu()[rows] for x in (k, v, q))
        if cos is not None:
            k64, ks = R.rotate(k64, p, cos, sin, inter)
            q64, qs = R.rotate(q64, p, cos, sin, inter)
            if qout is not None:
                _close(qout[rows.to(qout.device)], q64, qs, dtype)
                assert not bool(qout[torch.arange(at, at + m)[~ok].to(qout.device)].any())
        else:
            ks = k64.abs()
        good = bool(ok.all()) and m > 0
        for h in range(kv.hkv):
            for j in sorted(set((p // b).tolist())):
                page = int(table[r, h, j])
                if not 0 <= page < kv.pages:
                    good = False
                    continue
                here = p // b == j
                off = p[here] % b
                kp[page, off], vp[page, off] = k64[here, h], v64[here, h]
                size[page, off] = ks[here, h]
                a, z = k64[here, h].amin(0), k64[here, h].amax(0)
                fresh = int(off[0]) == 0
                lo[page] = a if fresh else torch.minimum(lo[page], a)
                hi[page] = z if fresh else torch.maximum(hi[page], z)
                bsize[page] = ks[here, h].amax(0)
        if good:
            nt[r] = positions[r] + m
            nb[r] = -(-nt[r] // b)
        at += m
    assert torch.equal(kv.v_pages.double().cpu(), vp)
    _close(kv.k_pages, kp, size, dtype)
    _close(kv.lo_pages, lo, bsize, dtype)
    _close(kv.hi_pages, hi, bsize, dtype)
    assert kv.nblocks.tolist() == nb and kv.ntokens.tolist() == nt


def _copy(kv):
    return paged.PagedKV(*(x.clone() for x in (kv.k_pages, kv.v_pages, kv.lo_pages, kv.hi_pages,
                                               kv.block_table, kv.nblocks, kv.ntokens)))


@pytest.mark.parametrize("dtype,hq,hkv,d,b,rot,inter,bounds", [
    (BF, 8, 2, 128, 32, 128, False, None), (FP, 4, 4, 64, 16, 64, True, torch.float32),
    (BF, 3, 1, 256, 24, 48, False, None), (FP, 12, 2, 128, 64, 32, True, None),
    (BF, 5, 5, 64, 7, 16, False, torch.float32), (BF, 8, 2, 256, 32, 256, True, None),
    (FP, 8, 4, 128, 1, 0, False, None)])
def test_ragged_tokens(dtype, hq, hkv, d, b, rot, inter, bounds):
    """Blocks begun and continued, whole blocks, none, one token, rewritten ones."""
    olds, news = [0, 5, 2 * b, 40, 17, 3], [1, 70, 0, 2 * b, 100, 1]
    ends = [o + m for o, m in zip(olds, news)]
    kv = R.make(hkv, d, b, ends, dtype, bounds=bounds)
    kv.ntokens.copy_(torch.tensor(olds, dtype=torch.int32))
    kv.nblocks.copy_(torch.tensor([-(-o // b) for o in olds], dtype=torch.int32))
    old = _copy(kv)
    q, k, v = _tokens(sum(news), hq, hkv, d, dtype)
    cos, sin = R.tables(kv.width * b + 5, rot) if rot else (None, None)
    pos = torch.tensor(olds, dtype=torch.int32, device="cuda")
    qout = paged.extend(kv, k, v, R.starts_of(news), pos, cos, sin, q=q if rot else None,
                        interleaved=inter)
    assert (qout is None) == (rot == 0)
    _check(kv, old, q, k, v, news, olds, cos, sin, inter, qout)
    again = _copy(kv)                              # the same tokens once more change nothing
    paged.extend(kv, k, v, R.starts_of(news), pos, cos, sin, interleaved=inter)
    for x in ("k_pages", "v_pages", "lo_pages", "hi_pages", "nblocks", "ntokens"):
        assert torch.equal(getattr(kv, x), getattr(again, x)), x


def test_positions_outside_and_invalid_pages():
    """Tokens past the table, before it, and on bad pages are not written; their requests keep
    their counts, the others are served."""
    b, news = 16, [40, 10, 30, 5, 20]
    kv = R.make(2, 64, b, [64, 64, 64, 64, 64], BF)
    positions = [40, -4, 10, 2 ** 31 - 2, 44]
    kv.block_table[2, 1, 1] = -1
    kv.block_table[2, 0, 2] = kv.pages + 7
    old = _copy(kv)
    q, k, v = _tokens(sum(news), 4, 2, 64, BF)
    cos, sin = R.tables(64, 64)
    pos = torch.tensor(positions, dtype=torch.int32, device="cuda")
    qout = paged.extend(kv, k, v, R.starts_of(news), pos, cos, sin, q=q)
    _check(kv, old, q, k, v, news, positions, cos, sin, False, qout)
    assert kv.ntokens.tolist() == [64] * 5 and kv.nblocks.tolist() == [4] * 5


def test_padding_and_many_requests():
    """Rows of no request, and more requests than one pass of the prefix sums takes."""
    r, b = 600, 16
    news = [(i * 7) % 4 for i in range(r)]
    olds = [(i * 5) % 40 for i in range(r)]
    kv = R.make(1, 64, b, [o + m for o, m in zip(olds, news)], FP)
    kv.ntokens.copy_(torch.tensor(olds, dtype=torch.int32))
    kv.nblocks.copy_(torch.tensor([-(-o // b) for o in olds], dtype=torch.int32))
    old = _copy(kv)
    t = sum(news)
    q, k, v = _tokens(t + 50, 2, 1, 64, FP)
    cos, sin = R.tables(kv.width * b, 64)
    pos = torch.tensor(olds, dtype=torch.int32, device="cuda")
    qout = paged.extend(kv, k, v, R.starts_of(news), pos, cos, sin, q=q)
    assert not bool(qout[t:].any())
    _check(kv, old, q[:t], k[:t], v[:t], news, olds, cos, sin, False, qout[:t])


@pytest.mark.parametrize("r,hkv,d,b,most", [(300, 3, 64, 16, 3), (270, 12, 256, 4, 2),
                                            (300, 2, 128, 64, 12), (5, 20, 128, 8, 2)])
def test_many_requests_and_heads(r, hkv, d, b, most):
    """Few tokens of many requests, whose KV heads share workgroups, and more of them."""
    news = [(i * 7) % (most + 1) for i in range(r)]
    olds = [(i * 5) % (3 * b) for i in range(r)]
    kv = R.make(hkv, d, b, [o + m for o, m in zip(olds, news)], BF)
    kv.ntokens.copy_(torch.tensor(olds, dtype=torch.int32))
    kv.nblocks.copy_(torch.tensor([-(-o // b) for o in olds], dtype=torch.int32))
    kv.block_table[r // 2, hkv - 1] = -1
    old = _copy(kv)
    t = sum(news)
    q, k, v = _tokens(t, 2 * hkv, hkv, d, BF)
    cos, sin = R.tables(kv.width * b, 32)
    pos = torch.tensor(olds, dtype=torch.int32, device="cuda")
    qout = paged.extend(kv, k, v, R.starts_of(news), pos, cos, sin, q=q)
    _check(kv, old, q, k, v, news, olds, cos, sin, False, qout)


def test_values_that_are_no_numbers():
    """NaN keys give NaN bounds, as the block bounds do; values pass as bits."""
    kv = R.make(1, 64, 16, [20], BF)
    k, v = R.queries(20, 1, 64, BF), R.queries(20, 1, 64, BF, seed=8)
    k[3, 0, 5], v[4, 0, 6], v[5, 0, 7] = float("nan"), float("nan"), float("inf")
    ints = dict(dtype=torch.int32, device="cuda")
    paged.extend(kv, k, v, torch.tensor([0, 20], **ints), torch.tensor([0], **ints))
    page = kv.block_table[0, 0, 0].long()
    assert bool(kv.lo_pages[page, 5].isnan()) and bool(kv.hi_pages[page, 5].isnan())
    assert int(kv.lo_pages[page].isnan().sum()) == 1
    got = kv.v_pages[kv.block_table[0, 0, :2].long()].reshape(-1, 64)[:20]
    assert torch.equal(got.view(torch.int16), v[:, 0].contiguous().view(torch.int16))


def test_one_token_equals_append():
    """Without rotation, one token per request is what paged.append writes, bit for bit."""
    lens = [1, 16, 17, 40]
    a = R.make(2, 128, 16, lens, BF, bounds=torch.float32)
    b = _copy(a)
    _, k, v = _tokens(4, 1, 2, 128, BF)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device="cuda")
    paged.append(a, k.contiguous(), v.contiguous(), pos)
    paged.extend(b, k, v, R.starts_of([1] * 4), pos)
    for x in ("k_pages", "v_pages", "lo_pages", "hi_pages", "nblocks", "ntokens"):
        assert torch.equal(getattr(a, x), getattr(b, x)), x


def test_captured_graph_advances():
    """A decode loop in one captured graph: positions advance on the device."""
    b, steps, lens = 16, 20, [30, 5]
    kv = R.make(2, 64, b, [n + steps + 2 for n in lens], BF)
    kv.ntokens.copy_(torch.tensor(lens, dtype=torch.int32))
    kv.nblocks.copy_(torch.tensor([-(-n // b) for n in lens], dtype=torch.int32))
    eager = _copy(kv)
    q, k, v = _tokens(2, 8, 2, 64, BF)
    cos, sin = R.tables(kv.width * b, 64)
    starts = R.starts_of([1, 1])
    pos = torch.tensor(lens, dtype=torch.int32, device="cuda")
    warm = _copy(kv)
    paged.attention(paged.extend(warm, k, v, starts, pos, cos, sin, q=q), warm)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        qr = paged.extend(kv, k, v, starts, pos, cos, sin, q=q)
        out = paged.attention(qr, kv)
        pos.add_(1)
    for i in range(steps):
        x, y, z = _tokens(2, 8, 2, 64, BF, seed=50 + i)
        q.copy_(x), k.copy_(y), v.copy_(z)
        p = torch.tensor([n + i for n in lens], dtype=torch.int32, device="cuda")
        g.replay()
        want = paged.attention(paged.extend(eager, k, v, starts, p, cos, sin, q=q), eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(kv.k_pages, eager.k_pages) and torch.equal(kv.lo_pages, eager.lo_pages)
        assert kv.ntokens.tolist() == [n + i + 1 for n in lens]


def test_serving_run():
    """A shared prompt prefilled in chunks, then decode steps: extend, dense, shared and sparse
    attention over one cache agree with the plain form."""
    b, hq, hkv, d, dtype = 16, 8, 2, 64, BF
    pre, tails, steps = 64, [9, 30, 1], 3
    kv = R.make(hkv, d, b, [pre + t + steps for t in tails], dtype)
    kv.block_table[:, :, :pre // b] = kv.block_table[:1, :, :pre // b].clone()
    kv.nblocks.zero_()
    kv.ntokens.zero_()
    cos, sin = R.tables(kv.width * b, d)
    ints = dict(dtype=torch.int32, device="cuda")
    # the prompt into request 0, in two chunks; the others take its blocks over
    at = 0
    for m in (40, 24):
        q, k, v = _tokens(m, hq, hkv, d, dtype, seed=at + 1)
        qr = paged.extend(kv, k, v, torch.tensor([0, m, m, m], **ints),
                          torch.tensor([at, 0, 0], **ints), cos, sin, q=q)
        at += m
        out = paged.attention(qr, kv, torch.tensor([0, m, m, m], **ints))
        R.check(out, *R.attention(qr, kv, [m, 0, 0]))
    kv.nblocks.fill_(pre // b)
    kv.ntokens.fill_(pre)
    # each request's own prompt, in one ragged call
    q, k, v = _tokens(sum(tails), hq, hkv, d, dtype, seed=70)
    starts = R.starts_of(tails)
    qr = paged.extend(kv, k, v, starts, torch.full((3,), pre, **ints), cos, sin, q=q)
    R.check(paged.attention(qr, kv, starts), *R.attention(qr, kv, tails))
    gs, sh = torch.tensor([0, 3], **ints), torch.tensor([pre // b], **ints)
    for i in range(steps):
        q, k, v = _tokens(3, hq, hkv, d, dtype, seed=80 + i)
        qr = paged.extend(kv, k, v, R.starts_of([1] * 3), kv.ntokens.clone(), cos, sin, q=q)
        ref = R.attention(qr, kv, [1] * 3)
        R.check(paged.attention(qr, kv), *ref)
        R.check(paged.shared_attention(qr, kv, gs, sh), *ref)
        # the sparse step over all blocks is the same attention (its output is FP32)
        ids, sparse = paged.exact(qr, kv, kv.width)
        assert torch.equal((ids >= 0).sum(-1), kv.nblocks[:, None].expand(-1, hq))
        R.check(sparse, *ref)
    assert kv.ntokens.tolist() == [pre + t + steps for t in tails]


def test_refusals():
    kv = R.make(2, 64, 16, [40, 20], BF)
    q, k, v = _tokens(3, 4, 2, 64, BF)
    ints = dict(dtype=torch.int32, device="cuda")
    starts, pos = torch.tensor([0, 2, 3], **ints), torch.tensor([1, 2], **ints)
    cos, sin = R.tables(kv.width * 16, 64)
    base = dict(kv=kv, k_new=k, v_new=v, starts=starts, positions=pos, cos=cos, sin=sin, q=q)
    before = _copy(kv)
    for kw in (dict(k_new=k[:2]), dict(k_new=k[:, :1]), dict(v_new=v.half()),
               dict(k_new=k.float()), dict(q=q[:2]), dict(q=q[:, :0]), dict(q=q.cpu()),
               dict(k_new=k[:, :, ::2]), dict(starts=starts[:2]), dict(starts=starts.long()),
               dict(positions=pos[:1]), dict(positions=kv.ntokens), dict(positions=kv.nblocks),
               dict(cos=None), dict(cos=None, sin=None), dict(cos=cos[:40], sin=sin[:40]),
               dict(cos=cos[:, :30], sin=sin[:, :30]), dict(cos=cos.double(), sin=sin.double()),
               dict(cos=cos[:, :4].contiguous(), sin=sin[:, :4].contiguous()),
               dict(cos=cos.cpu(), sin=sin.cpu())):
        with pytest.raises(ValueError):
            paged.extend(**dict(base, **kw))
    with pytest.raises(TypeError):
        paged.extend(None, k, v, starts, pos)
    single = R.make(2, 64, 16, [40, 20], BF)
    single.k_pages, single.v_pages = single.k_pages.float(), single.v_pages.float()
    with pytest.raises(ValueError):
        paged.extend(single, k.float(), v.float(), starts, pos)
    for x in ("k_pages", "lo_pages", "nblocks", "ntokens"):
        assert torch.equal(getattr(kv, x), getattr(before, x))
