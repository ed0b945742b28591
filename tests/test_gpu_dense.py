"""Dense attention over the paged cache (paged.attention, paged.shared_attention)
against a plain 64-bit form (dense_ref.py), where it can go wrong: lengths around
the kernels' tiles, every head layout, masks that leave rows empty, values that are
not numbers in hidden places, bad pages, strides, padding, captured graphs."""
import pytest
import torch

from strict_topk import paged
from tests import dense_ref as R

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
MODES = {"plain": {}, "cap": dict(softcap=8.0), "bias": dict(slopes=True),
         "both": dict(softcap=20.0, slopes=True)}


def _kw(hq, mode, **more):
    kw = dict(MODES[mode], **more)
    if kw.get("slopes"):
        kw["slopes"] = R.slopes_of(hq)
    return kw


def _run(q, kv, news, **kw):
    ref = {x: kw[x] for x in kw if x != "out"}
    for x in ("prefix", "first"):
        if ref.get(x) is not None:
            ref[x] = ref[x].tolist()
    starts = None if all(m == 1 for m in news) and not kw.pop("ragged", False) \
        else R.starts_of(news)
    ref.pop("ragged", None)
    got = paged.attention(q, kv, starts, **kw)
    R.check(got, *R.attention(q, kv, news, **ref))
    return got


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype,hq,hkv,d,b", [
    (BF, 8, 2, 128, 32), (FP, 4, 4, 64, 16), (BF, 12, 1, 64, 48), (FP, 16, 2, 256, 64),
    (BF, 40, 1, 128, 16), (FP, 5, 5, 256, 32)])
def test_decode_lengths(dtype, hq, hkv, d, b, mode):
    lens = [1, 0, 15, 16, 17, 31, 33, 127, 128, 129, 300, 700]
    kv = R.make(hkv, d, b, lens, dtype)
    q = R.queries(len(lens), hq, d, dtype)
    out = _run(q, kv, [1] * len(lens), **_kw(hq, mode))
    assert not bool(out[1].any())


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype,hq,hkv,d,b", [
    (BF, 8, 2, 128, 32), (FP, 4, 4, 64, 16), (BF, 12, 1, 64, 48), (FP, 6, 2, 256, 64),
    (FP, 20, 1, 128, 16), (BF, 5, 5, 256, 32)])
def test_ragged_chunks(dtype, hq, hkv, d, b, mode):
    lens = [1, 40, 70, 0, 200, 65, 333]
    news = [1, 40, 1, 0, 131, 17, 5]
    kv = R.make(hkv, d, b, lens, dtype)
    q = R.queries(sum(news), hq, d, dtype)
    _run(q, kv, news, **_kw(hq, mode))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("mask", ["window1", "window40", "prefix", "first", "all"])
def test_masks(d, mask):
    lens, news = [300, 90, 150], [170, 90, 1]
    kv = R.make(2, d, 32, lens, BF)
    q = R.queries(sum(news), 6, d, BF)
    pos = [n - m + t for n, m in zip(lens, news) for t in range(m)]
    kw = {}
    if mask in ("window1", "window40", "all"):
        kw["window"] = 1 if mask == "window1" else 40
    if mask in ("prefix", "all"):
        kw["prefix"] = torch.tensor([200, 1000, -5], dtype=torch.int32, device="cuda")
    if mask in ("first", "all"):
        # documents of 37 tokens, a negative start, and starts past the token: no key
        first = [p // 37 * 37 for p in pos]
        first[3], first[5], first[100], first[171] = -7, pos[5] + 1, 2 ** 31 - 1, 500
        kw["first"] = torch.tensor(first, dtype=torch.int32, device="cuda")
    out = _run(q, kv, news, **kw)
    if mask == "first":
        assert not bool(out[[5, 100, 171]].any())


@pytest.mark.parametrize("window,first", [(1, None), (50, None), (0, [0, 5, 199, 200, 64]),
                                          (33, [300, 0, 180, 7, -1])])
def test_decode_masks(window, first):
    lens = [200, 6, 200, 200, 65]
    kv = R.make(2, 128, 16, lens, FP)
    q = R.queries(5, 8, 128, FP)
    if first is not None:
        first = torch.tensor(first, dtype=torch.int32, device="cuda")
    out = _run(q, kv, [1] * 5, window=window, first=first)
    if window == 0:
        assert not bool(out[3].any())


def test_more_queries_than_tokens():
    """Rows before the request's first token see nothing (or the prefix)."""
    kv = R.make(2, 64, 16, [20, 33], BF)
    q = R.queries(90, 4, 64, BF)
    out = _run(q, kv, [50, 40])
    assert not bool(out[:30].any()) and bool(out[30].any())
    _run(q, kv, [50, 40], prefix=torch.tensor([7, 0], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_hidden_places_do_not_matter(dtype, d, bad):
    """Unused rows of the pages, and tokens after a query's own, hold no numbers: only the
    queries that see them change."""
    lens, news = [140, 77], [100, 1]
    kv = R.make(2, d, 16, lens, dtype)
    q = R.queries(sum(news), 4, d, dtype)
    starts = R.starts_of(news)
    clean = paged.attention(q, kv, starts)
    for r, n in enumerate(lens):                  # behind the last token, and spare pages
        page = kv.block_table[r, :, (n - 1) // 16].long()
        kv.k_pages[page, n % 16:] = bad
        kv.v_pages[page, n % 16:] = bad
    free = torch.ones(kv.pages, dtype=torch.bool, device="cuda")
    free[kv.block_table[kv.block_table >= 0].long()] = False
    kv.k_pages[free] = bad
    kv.v_pages[free] = bad
    assert torch.equal(paged.attention(q, kv, starts), clean)
    # position 90 is seen by the rows from 90 on (row t stands at 40 + t)
    ref, tol = R.attention(q, kv, news)
    page = int(kv.block_table[0, 1, 90 // 16])
    kv.v_pages[page, 90 % 16, 3] = bad
    got = paged.attention(q, kv, starts)
    keep = [i for i in range(d) if i != 3]
    for rows, heads, dims in ((slice(0, 50), slice(0, 4), range(d)), (slice(100, 101), slice(0, 4),
                                                                      range(d)),
                              (slice(50, 100), slice(0, 2), range(d)),
                              (slice(50, 100), slice(2, 4), keep)):
        R.check(got[rows, heads][..., list(dims)], ref[rows, heads][..., list(dims)],
                tol[rows, heads][..., list(dims)])
    hit = got[50:100, 2:, 3].float()
    assert bool((hit.isnan() | hit.isinf()).all())
    kv.k_pages[page, 90 % 16] = bad
    got = paged.attention(q, kv, starts)
    R.check(got[:50], ref[:50], tol[:50])
    # the single token's window hides a bad value inside its first tile
    one = paged.attention(q[100:], _only(kv, 1), window=20)
    page = int(kv.block_table[1, 0, 50 // 16])
    kv.k_pages[page, 50 % 16] = bad
    kv.v_pages[page, 50 % 16] = bad
    assert torch.equal(paged.attention(q[100:], _only(kv, 1), window=20), one)


def _only(kv, r):
    return paged.PagedKV(kv.k_pages, kv.v_pages, kv.lo_pages, kv.hi_pages,
                         kv.block_table[r:r + 1].contiguous(), kv.nblocks[r:r + 1].contiguous(),
                         kv.ntokens[r:r + 1].contiguous())


@pytest.mark.parametrize("news", [[1, 1, 1], [60, 1, 45]])
def test_invalid_pages_are_not_read(news):
    """Entries outside the pool hide their keys; a request with no valid page gets zeros."""
    kv = R.make(2, 128, 16, [200, 50, 45], BF)
    q = R.queries(sum(news), 8, 128, BF)
    kv.block_table[0, 0, 2] = -1
    kv.block_table[0, 1, 5] = kv.pages
    kv.block_table[0, 0, 12] = 2 ** 31 - 1
    kv.block_table[1] = -(2 ** 31)
    out = _run(q, kv, news)
    assert not bool(out[news[0]:news[0] + news[1]].any())


def test_counts_outside_the_table_are_clamped():
    kv = R.make(2, 64, 32, [100, 64, 90], BF)
    q = R.queries(3, 4, 64, BF)
    kv.ntokens[0], kv.nblocks[1], kv.ntokens[2] = 10 ** 9, 10 ** 9, -3
    out = _run(q, kv, [1, 1, 1])
    assert not bool(out[2].any())
    kv.ntokens = None
    kv.nblocks[2] = -1
    out = _run(q, kv, [1, 1, 1])
    assert not bool(out[2].any())


def test_strided_queries_and_padding():
    lens, news = [100, 30], [50, 7]
    kv = R.make(2, 64, 16, lens, BF)
    fused = R.queries(70, 4 + 3, 64, BF)
    q = fused[:, :4]
    starts = R.starts_of(news)
    ref, tol = R.attention(q[:57], kv, news)
    got = paged.attention(q, kv, starts)
    R.check(got[:57], ref, tol)
    assert not bool(got[57:].any())
    out = torch.full((70, 4, 64), 5.0, dtype=BF, device="cuda")
    assert paged.attention(q, kv, starts, out=out) is out
    assert torch.equal(out[:57], got[:57]) and bool((out[57:] == 5).all())
    shifted = starts + 3                           # rows before the first request, too
    got = paged.attention(q, kv, shifted)
    ref, tol = R.attention(q[3:60], kv, news)
    R.check(got[3:60], ref, tol)
    assert not bool(got[:3].any()) and not bool(got[60:].any())


def test_many_requests():
    """More requests than one pass of the kernels' prefix sums takes."""
    lens = [(i * 37) % 90 for i in range(700)]
    kv = R.make(1, 64, 16, lens, BF)
    q = R.queries(700, 2, 64, BF)
    one = _run(q, kv, [1] * 700)
    got = paged.attention(q, kv, R.starts_of([1] * 700))
    assert torch.allclose(one.float(), got.float(), atol=0.02)
    gs = torch.arange(0, 701, 100, dtype=torch.int32, device="cuda")
    none = torch.zeros(7, dtype=torch.int32, device="cuda")
    got = paged.shared_attention(q, kv, gs, none)
    R.check(got, *R.attention(q, kv, [1] * 700))


@pytest.mark.parametrize("requests,groups", [(1500, 1200), (700, 300), (300, 9)])
def test_many_groups(requests, groups):
    """Groups of none, one and several requests, more than one pass of the prefix sums takes;
    requests behind the last group share nothing."""
    lens = [32 + (i * 7) % 20 for i in range(requests)]
    kv = R.make(1, 64, 16, lens, BF)
    at = [(i * (requests - 5) // groups) // 2 * 2 for i in range(groups + 1)]
    shared = [i % 3 for i in range(groups)]
    for g, n in enumerate(shared):
        kv.block_table[at[g]:at[g + 1], :, :n] = kv.block_table[at[g], :, :n]
    q = R.queries(requests, 2, 64, BF)
    ints = dict(dtype=torch.int32, device="cuda")
    got = paged.shared_attention(q, kv, torch.tensor(at, **ints), torch.tensor(shared, **ints))
    R.check(got, *R.attention(q, kv, [1] * requests))


def test_more_requests_than_a_pass():
    lens = [(i * 37) % 40 for i in range(1300)]
    kv = R.make(1, 64, 16, lens, FP)
    _run(R.queries(1300, 2, 64, FP), kv, [1] * 1300)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype,hq,hkv,d,b", [(BF, 16, 8, 64, 32), (FP, 10, 5, 128, 16),
                                              (BF, 40, 2, 256, 16)])
def test_many_short_requests(dtype, hq, hkv, d, b, mode):
    """Short items, several of which lie in one workgroup, of keys all their own and behind
    shared blocks; what the cache holds behind them is NaN."""
    lens = [(i * 37) % 300 for i in range(320)]
    kv = R.make(hkv, d, b, lens, dtype)
    kw = _kw(hq, mode)
    q = R.queries(320, hq, d, dtype)
    ref = R.attention(q, kv, [1] * 320, **kw)
    table = kv.block_table.tolist()
    for r, n in enumerate(lens):
        if n % b:
            for h in range(hkv):
                page = table[r][h][n // b]
                kv.k_pages[page, n % b:] = float("nan")
                kv.v_pages[page, n % b:] = float("inf")
    R.check(paged.attention(q, kv, **kw), *ref)
    ints = dict(dtype=torch.int32, device="cuda")
    at, shared = list(range(0, 321, 2)), [i % 4 for i in range(160)]
    for g, n in enumerate(shared):
        shared[g] = n = min(n, min(lens[2 * g:2 * g + 2]) // b)
        kv.block_table[2 * g + 1, :, :n] = kv.block_table[2 * g, :, :n]
    ref = R.attention(q, kv, [1] * 320, **kw)
    got = paged.shared_attention(q, kv, torch.tensor(at, **ints), torch.tensor(shared, **ints),
                                 **kw)
    R.check(got, *ref)


def test_many_rows_without_splitting():
    """Enough row tiles that none is split."""
    kv = R.make(8, 64, 32, [2100] * 2, FP)
    q = R.queries(4200, 64, 64, FP)
    got = paged.attention(q, kv, R.starts_of([2100, 2100]))
    for t in (0, 1, 77, 2099, 2100, 4199):         # single rows of the reference
        r, n = t // 2100, t % 2100 + 1
        short = paged.PagedKV(kv.k_pages, kv.v_pages, kv.lo_pages, kv.hi_pages,
                              kv.block_table[r:r + 1].contiguous(), kv.nblocks[r:r + 1],
                              torch.tensor([n], dtype=torch.int32, device="cuda"))
        R.check(got[t:t + 1], *R.attention(q[t:t + 1], short, [1]))


def test_large_scores_and_scale():
    lens, news = [150, 70], [80, 1]
    kv = R.make(2, 128, 16, lens, BF)
    q = R.queries(81, 4, 128, BF) * 30
    _run(q, kv, news)
    _run(q, kv, news, scale=0.003)
    _run(q, kv, news, scale=2.0, softcap=60.0)


def test_equal_results_whatever_the_batch():
    """A request's decode result does not depend on chance: the same call gives the same bits."""
    kv = R.make(4, 128, 32, [5000, 33, 1200], BF)
    q = R.queries(3, 16, 128, BF)
    a = paged.attention(q, kv)
    for _ in range(3):
        assert torch.equal(paged.attention(q, kv), a)


def test_pool_past_32_bits():
    """Rows whose element offsets pass 2^31 (and byte offsets 2^32)."""
    pages, b, d = 140000, 64, 256
    k = torch.empty((pages, b, d), dtype=BF, device="cuda")
    v = torch.empty_like(k)
    small = R.make(1, d, b, [500], BF)
    n = small.pages
    k[-n:], v[-n:] = small.k_pages, small.v_pages
    kv = paged.PagedKV(k, v, small.lo_pages, small.hi_pages,
                       torch.where(small.block_table >= 0, small.block_table + (pages - n), -1)
                       .int(), small.nblocks, small.ntokens)
    q = R.queries(9, 4, d, BF)
    starts = R.starts_of([9])
    assert torch.equal(paged.attention(q, kv, starts), paged.attention(q, small, starts))
    assert torch.equal(paged.attention(q[:1], kv), paged.attention(q[:1], small))


def test_captured_graph_follows_lengths():
    lens = [100, 300]
    kv = R.make(2, 128, 16, lens, BF, width=40)
    q = R.queries(2, 8, 128, BF)
    qr = R.queries(60, 8, 128, BF, seed=9)
    starts = R.starts_of([40, 20])
    paged.attention(q, kv), paged.attention(qr, kv, starts)      # warm
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        one = paged.attention(q, kv)
        many = paged.attention(qr, kv, starts)
    for n0, n1, s1 in ((100, 300, 40), (7, 299, 10), (64, 130, 60), (100, 300, 40)):
        kv.ntokens.copy_(torch.tensor([n0, n1], dtype=torch.int32))
        starts.copy_(torch.tensor([0, s1, 60], dtype=torch.int32))
        q.copy_(R.queries(2, 8, 128, BF, seed=n0))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(one, paged.attention(q, kv))
        assert torch.equal(many, paged.attention(qr, kv, starts))
        R.check(one, *R.attention(q, kv, [1, 1]))
        R.check(many, *R.attention(qr, kv, [s1, 60 - s1]))


def test_captured_graph_of_listed_tiles():
    """Tiles that the device lists, cut and leaves whole from one replay to the next."""
    kv = R.make(2, 128, 16, [3000, 600], BF, width=200)
    q = R.queries(600, 8, 128, BF)
    starts = R.starts_of([40, 560])
    paged.attention(q, kv, starts)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = paged.attention(q, kv, starts)
    for n0, n1, s1 in ((3000, 600, 40), (300, 300, 300), (3000, 40, 590), (2, 580, 20), (0, 0, 0)):
        kv.ntokens.copy_(torch.tensor([n0, n1], dtype=torch.int32))
        starts.copy_(torch.tensor([0, s1, 600], dtype=torch.int32))
        q.copy_(R.queries(600, 8, 128, BF, seed=n0 + 1))
        g.replay()
        torch.cuda.synchronize()
        R.check(got, *R.attention(q, kv, [s1, 600 - s1]))
        R.check(paged.attention(q, kv, starts), *R.attention(q, kv, [s1, 600 - s1]))


def test_concurrent_streams():
    kv = R.make(2, 64, 16, [500, 41], FP)
    q = R.queries(2, 4, 64, FP)
    want = paged.attention(q, kv)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([paged.attention(q, kv) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for os in outs for o in os)


# ------------------------------------------------------------ shared blocks

def _share(kv, groups, shared):
    for a, b, n in zip(groups[:-1], groups[1:], shared):
        if b > a:
            kv.block_table[a:b, :, :n] = kv.block_table[a:a + 1, :, :n].clone()
    ints = dict(dtype=torch.int32, device="cuda")
    return torch.tensor(groups, **ints), torch.tensor(shared, **ints)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype,hq,hkv,d,b", [
    (BF, 8, 2, 128, 32), (FP, 4, 4, 64, 16), (BF, 24, 1, 64, 48), (FP, 6, 2, 256, 64)])
def test_shared_lengths(dtype, hq, hkv, d, b, mode):
    pre = 5 * b
    lens = [pre + x for x in (1, 16, 40, 100, 0, 33, 7)]
    kv = R.make(hkv, d, b, lens, dtype)
    groups, shared = _share(kv, [0, 7], [5])
    q = R.queries(7, hq, d, dtype)
    kw = _kw(hq, mode)
    ref = R.attention(q, kv, [1] * 7, **kw)
    R.check(paged.shared_attention(q, kv, groups, shared, **kw), *ref)


@pytest.mark.parametrize("groups,shared", [
    ([0, 3, 3, 9], [4, 2, 6]), ([1, 5, 8], [3, 0]), ([0, 9], [0]), ([2, 3, 4], [6, 5]),
    ([4, 4], [3])])
@pytest.mark.parametrize("kw", [{}, dict(window=30), dict(window=150)])
def test_shared_groups(groups, shared, kw):
    """Groups of one or no request, nothing shared, requests outside every group, windows that
    end in the shared blocks or behind them."""
    lens = [6 * 16 + x for x in (5, 16, 1, 30, 100, 17, 2, 64, 33)]
    kv = R.make(2, 128, 16, lens, BF)
    gs, sh = _share(kv, groups, shared)
    q = R.queries(9, 40, 128, BF)
    R.check(paged.shared_attention(q, kv, gs, sh, **kw), *R.attention(q, kv, [1] * 9, **kw))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [60, 333, 1000, 1300, 2 ** 31 - 1])
def test_shared_windows(d, window):
    """Windows that hide most of the shared blocks, in groups of many and of few shared keys, one
    with requests that hold fewer tokens than are shared."""
    lens = [1280 + x for x in (0, 1, 40, 300, 1290, 77)] + [1000, 500, 0, 1290, 33, 90]
    kv = R.make(2, d, 16, lens, BF)
    gs, sh = _share(kv, [0, 6, 10, 12], [80, 70, 2])
    q = R.queries(12, 40, d, BF)
    R.check(paged.shared_attention(q, kv, gs, sh, window=window),
            *R.attention(q, kv, [1] * 12, window=window))


def test_shared_long_prefix_many_rows():
    """More query rows than one tile and keys enough to be split."""
    lens = [2048 + 1 + 3 * i for i in range(45)]
    kv = R.make(1, 64, 32, lens, BF)
    gs, sh = _share(kv, [0, 45], [64])
    q = R.queries(45, 8, 64, BF)
    first = torch.tensor([40 * i for i in range(45)], dtype=torch.int32, device="cuda")
    ref, tol = R.attention(q, kv, [1] * 45, first=first.tolist())
    R.check(paged.shared_attention(q, kv, gs, sh, first=first), ref, tol)
    out = torch.empty_like(q)
    assert paged.shared_attention(q, kv, gs, sh, first=first, out=out) is out
    R.check(out, ref, tol)


def test_shared_hidden_places():
    """A value that only some requests' windows reach is not a number."""
    lens = [96 + 20, 96 + 50, 96 + 3]
    kv = R.make(2, 128, 16, lens, BF)
    gs, sh = _share(kv, [0, 3], [6])
    q = R.queries(3, 8, 128, BF)
    clean = paged.shared_attention(q, kv, gs, sh, window=25)
    page = int(kv.block_table[0, 0, 70 // 16])
    kv.v_pages[page, 70 % 16] = float("nan")       # windows of 60 begin at 56, 86 and 39
    got = paged.shared_attention(q, kv, gs, sh, window=60)
    want = paged.attention(q, kv, window=60)
    assert torch.equal(got.isnan(), want.isnan())
    assert bool(got[0, 0].isnan().all()) and not bool(got[1].isnan().any())
    got = paged.shared_attention(q, kv, gs, sh, window=25)
    assert torch.equal(got, clean)


def test_shared_captured_graph():
    kv = R.make(2, 64, 16, [100, 130, 90], FP)
    gs, sh = _share(kv, [0, 3], [4])
    q = R.queries(3, 8, 64, FP)
    paged.shared_attention(q, kv, gs, sh)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = paged.shared_attention(q, kv, gs, sh)
    for n, s, last in ((70, 4, 3), (100, 2, 2), (64, 0, 3), (100, 4, 3)):
        kv.ntokens[0] = n
        sh.fill_(s)
        gs[1] = last
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged.shared_attention(q, kv, gs, sh))
        R.check(out, *R.attention(q, kv, [1] * 3))


def test_refusals():
    kv = R.make(2, 64, 16, [40, 20], BF)
    q = R.queries(2, 4, 64, BF)
    ints = dict(dtype=torch.int32, device="cuda")
    bad = [
        dict(q=q[:, :3]), dict(q=q[:, :, :32]), dict(q=q.half()), dict(q=q.float()),
        dict(q=q.cpu()), dict(q=q[:1]), dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)),
        dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(softcap=-1.0),
        dict(softcap=float("inf")), dict(window=-1), dict(window=2 ** 31),
        dict(slopes=R.slopes_of(3)), dict(slopes=R.slopes_of(4).double()),
        dict(prefix=torch.zeros(3, **ints)), dict(prefix=torch.zeros(2, device="cuda")),
        dict(first=torch.zeros(3, **ints)), dict(starts=torch.zeros(2, **ints)),
        dict(starts=torch.zeros(3, dtype=torch.int64, device="cuda")),
        dict(out=torch.empty_like(q).half()), dict(out=torch.empty((2, 8, 64), dtype=BF,
                                                                   device="cuda")[:, ::2])]
    for kw in bad:
        kw = dict(dict(q=q, kv=kv), **kw)
        with pytest.raises(ValueError):
            paged.attention(**kw)
    with pytest.raises(TypeError):
        paged.attention(q, None)
    for gs, sh in ((torch.zeros(1, **ints), torch.zeros(0, **ints)),
                   (torch.zeros(4, **ints), torch.zeros(3, **ints)),
                   (torch.zeros(3, **ints), torch.zeros(1, **ints)),
                   (torch.zeros((2, 1), **ints), torch.zeros(1, **ints)),
                   (torch.zeros(2, device="cuda"), torch.zeros(1, **ints))):
        with pytest.raises(ValueError):
            paged.shared_attention(q, kv, gs, sh)
    for d, b in ((96, 16), (64, 24)):
        with pytest.raises(ValueError):
            paged.attention(R.queries(2, 4, d, BF), R.make(2, d, b, [40, 20], BF))
    odd = torch.zeros(2 * 4 * 64 + 8, dtype=BF, device="cuda")[1:513].view(2, 4, 64)
    with pytest.raises(ValueError):
        paged.attention(odd, kv)
    assert paged.attention(q[:0], kv, torch.zeros(3, **ints)).shape == (0, 4, 64)


# ------------------------------------------- tiles that are listed, and cut

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("mask", ["none", "window", "prefix", "first", "all"])
def test_listed_tiles(d, mask):
    """Short requests in a wide table: the tiles are listed on the device and taken whole."""
    lens, news = [300, 0, 90, 150, 33, 600], [170, 0, 90, 1, 33, 64]
    kv = R.make(2, d, 32, lens, BF, width=400)
    q = R.queries(sum(news), 10, d, BF)
    pos = [n - m + t for n, m in zip(lens, news) for t in range(m)]
    ints = dict(dtype=torch.int32, device="cuda")
    kw = {}
    if mask in ("window", "all"):
        kw["window"] = 70
    if mask in ("prefix", "all"):
        kw["prefix"] = torch.tensor([200, 5, 1000, -5, 33, 580], **ints)
    if mask in ("first", "all"):
        first = [p // 37 * 37 for p in pos]
        first[3], first[5], first[100], first[171] = -7, pos[5] + 1, 2 ** 31 - 1, 500
        kw["first"] = torch.tensor(first, **ints)
    _run(q, kv, news, **kw)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype,hq,hkv,d,b", [(BF, 8, 2, 128, 32), (FP, 3, 1, 64, 16),
                                              (BF, 6, 1, 256, 64)])
def test_cut_tiles(dtype, hq, hkv, d, b, mode):
    """Few long tiles: their keys are cut over many workgroups and the parts joined."""
    lens, news = [2600, 700, 1500, 31], [20, 3, 61, 1]
    kv = R.make(hkv, d, b, lens, dtype, width=200)
    q = R.queries(sum(news), hq, d, dtype)
    _run(q, kv, news, **_kw(hq, mode))


@pytest.mark.parametrize("long", [0, 5000])
def test_many_short_tiles(long):
    """More tiles than workgroups fill the device, of requests with one tile each, listed
    whole and, beside one long request, cut."""
    lens, news = [40 + 3 * (i % 50) for i in range(140)], [1 + i % 4 for i in range(140)]
    lens[70] += long
    kv = R.make(8, 64, 32, lens, BF, width=170)
    _run(R.queries(sum(news), 16, 64, BF), kv, news)


@pytest.mark.parametrize("requests", [1016, 1017])
def test_most_listed_requests(requests):
    """The most tiles that are listed, and more."""
    lens, news = [1 + i % 90 for i in range(requests)], [1] * requests
    kv = R.make(1, 64, 32, lens, FP, width=80)
    _run(R.queries(requests, 1, 64, FP), kv, news, ragged=True)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype,hq,hkv,d,b", [(BF, 8, 2, 128, 32), (FP, 3, 1, 64, 16),
                                              (BF, 6, 1, 256, 64), (FP, 20, 2, 256, 16)])
def test_few_rows(dtype, hq, hkv, d, b, mode):
    """A few tokens of each request, in 16 rows; rows of no request around them."""
    lens, news = [2600, 700, 0, 1500, 31, 2], [4, 1, 0, 7, 2, 3]
    kv = R.make(hkv, d, b, lens, dtype, width=200)
    t = sum(news)
    q = R.queries(t + 5, hq, d, dtype)
    kw = _kw(hq, mode)
    got = paged.attention(q, kv, R.starts_of(news) + 2, **kw)
    R.check(got[2:t + 2], *R.attention(q[2:t + 2], kv, news, **kw))
    assert not bool(got[:2].any()) and not bool(got[t + 2:].any())
    out = torch.full_like(q, 7.0).contiguous()
    paged.attention(q, kv, R.starts_of(news) + 2, out=out, **kw)
    assert torch.equal(out[2:t + 2], got[2:t + 2])
    assert bool((out[:2] == 7).all()) and bool((out[t + 2:] == 7).all())


@pytest.mark.parametrize("mask", ["window", "prefix", "first", "pages", "all"])
def test_few_rows_masks(mask):
    lens, news = [2600, 900, 40], [6, 9, 3]
    kv = R.make(2, 128, 16, lens, FP, width=300)
    q = R.queries(sum(news), 6, 128, FP)
    ints = dict(dtype=torch.int32, device="cuda")
    kw = {}
    if mask in ("window", "all"):
        kw["window"] = 700
    if mask in ("prefix", "all"):
        kw["prefix"] = torch.tensor([2598, 5000, -3], **ints)
    if mask in ("first", "all"):
        first = [p // 37 * 37 for p in range(2594, 2600)] + [890 + i % 3 for i in range(9)] + \
            [39, 2 ** 31 - 1, -7]
        kw["first"] = torch.tensor(first, **ints)
    if mask in ("pages", "all"):
        kv.block_table[0, 0, 20:130:7] = -1
        kv.block_table[1, 1, ::2] = kv.pages
    _run(q, kv, news, **kw)


@pytest.mark.parametrize("dtype,d", [(BF, 64), (FP, 128), (BF, 256)])
def test_few_rows_hidden_places(dtype, d):
    """The last token of a request holds no numbers: the ones before it do not see it."""
    lens, news = [2600, 700, 40], [4, 3, 7]
    kv = R.make(2, d, 16, lens, dtype, width=200)
    q = R.queries(sum(news), 6, d, dtype)
    ref, tol = R.attention(q, kv, news)
    for r, n in enumerate(lens):
        for page in kv.block_table[r, :, (n - 1) // 16].tolist():
            kv.k_pages[page, n % 16:] = float("nan")
            kv.v_pages[page, n % 16:] = float("nan")
            kv.v_pages[page, (n - 1) % 16, 5] = float("inf")
    got = paged.attention(q, kv, R.starts_of(news))
    last = [3, 6, 13]
    rest = [i for i in range(14) if i not in last]
    R.check(got[rest], ref[rest], tol[rest])
    dims = [i for i in range(d) if i != 5]
    R.check(got[last][..., dims], ref[last][..., dims], tol[last][..., dims])
    assert bool(got[last][..., 5].isinf().all())


@pytest.mark.parametrize("mode", MODES)
def test_few_rows_of_many_documents(mode):
    """More tokens of a request than its documents are looked at, and fewer."""
    lens, news = [900, 650], [90, 30]
    kv = R.make(1, 64, 16, lens, BF, width=60)
    q = R.queries(sum(news), 2, 64, BF)
    pos = [n - m + t for n, m in zip(lens, news) for t in range(m)]
    first = torch.tensor([p // 23 * 23 for p in pos], dtype=torch.int32, device="cuda")
    _run(q, kv, news, first=first, **_kw(2, mode))


def test_few_rows_of_many_requests():
    lens, news = [(i * 41) % 500 for i in range(130)], [i % 3 for i in range(130)]
    kv = R.make(1, 64, 16, lens, BF, width=60)
    _run(R.queries(sum(news), 2, 64, BF), kv, news)


@pytest.mark.parametrize("hq,hkv,d,b", [(136, 1, 64, 1024), (258, 2, 128, 16)])
def test_more_heads_than_a_tile_has_rows(hq, hkv, d, b):
    lens = [1500, 3, 0]
    kv = R.make(hkv, d, b, lens, BF)
    _run(R.queries(6, hq, d, BF), kv, [3, 3, 0])
    q = R.queries(3, hq, d, BF)
    _run(q, kv, [1] * 3)
    kv.block_table[1, :, :1] = kv.block_table[0, :, :1]
    ints = dict(dtype=torch.int32, device="cuda")
    kv.ntokens[1] = b
    kv.nblocks[1] = 1
    got = paged.shared_attention(q, kv, torch.tensor([0, 2], **ints), torch.tensor([1], **ints))
    R.check(got, *R.attention(q, kv, [1] * 3))


@pytest.mark.parametrize("mask", ["window", "prefix", "first", "pages"])
def test_cut_tiles_masks(mask):
    lens, news = [2600, 1500], [30, 61]
    kv = R.make(1, 128, 16, lens, FP, width=300)
    q = R.queries(sum(news), 5, 128, FP)
    ints = dict(dtype=torch.int32, device="cuda")
    kw = {}
    if mask == "window":
        kw["window"] = 1333
    if mask == "prefix":
        kw["prefix"] = torch.tensor([2590, 1470], **ints)
    if mask == "first":
        kw["first"] = torch.tensor([(37 * i) % 2700 for i in range(sum(news))], **ints)
    if mask == "pages":
        kv.block_table[0, 0, 20:130:7] = -1
        kv.block_table[1, 0, ::2] = kv.pages
    _run(q, kv, news, **kw)


def test_cut_tiles_hidden_places():
    """A value that is no number, seen by some rows of a cut tile, reaches those rows alone."""
    lens, news = [2600], [100]
    kv = R.make(1, 64, 16, lens, BF, width=300)
    q = R.queries(100, 2, 64, BF)
    starts = R.starts_of(news)
    ref, tol = R.attention(q, kv, news)
    page = int(kv.block_table[0, 0, 2560 // 16])
    kv.v_pages[page, 2560 % 16, 9] = float("nan")      # row t stands at 2500 + t
    got = paged.attention(q, kv, starts)
    R.check(got[:60], ref[:60], tol[:60])
    keep = [i for i in range(64) if i != 9]
    R.check(got[60:][..., keep], ref[60:][..., keep], tol[60:][..., keep])
    assert bool(got[60:, :, 9].isnan().all())


def test_output_over_the_queries():
    """out may be q itself."""
    lens, news = [2600, 90], [20, 90]
    kv = R.make(2, 128, 16, lens, BF, width=200)
    q = R.queries(110, 8, 128, BF)
    starts = R.starts_of(news)
    want = paged.attention(q, kv, starts)
    assert torch.equal(paged.attention(q, kv, starts, out=q), want)
    one = R.queries(2, 8, 128, BF)
    want = paged.attention(one, kv)
    assert torch.equal(paged.attention(one, kv, out=one), want)


def test_malformed_starts_and_groups_stay_in_bounds():
    """starts and groups that decrease or leave the rows give some result, and an intact cache."""
    kv = R.make(2, 64, 16, [700, 90, 40], BF, width=60)
    q = R.queries(40, 4, 64, BF)
    keep = [x.clone() for x in (kv.k_pages, kv.v_pages, kv.block_table)]
    ints = dict(dtype=torch.int32, device="cuda")
    for s in ([0, 30, 10, 40], [5, 1000, -7, 40], [40, 40, 40, 40], [-5, -5, 50, 60],
              [0, 40, 0, 40]):
        paged.attention(q, kv, torch.tensor(s, **ints))
        paged.extend(_scratch(kv), q[:, :2], q[:, 2:], torch.tensor(s, **ints),
                     torch.tensor([3, 4, 5], **ints))
    for g, n in (([0, 3, 1], [2, 2]), ([2, -4, 9], [1000, 3]), ([0, 3, 0, 3], [5, -1, 40])):
        paged.shared_attention(q[:3], kv, torch.tensor(g, **ints), torch.tensor(n, **ints))
    torch.cuda.synchronize()
    for x, y in zip(keep, (kv.k_pages, kv.v_pages, kv.block_table)):
        assert torch.equal(x, y)
    R.check(paged.attention(q[:3], kv), *R.attention(q[:3], kv, [1] * 3))


def _scratch(kv):
    return paged.PagedKV(*(x.clone() for x in (kv.k_pages, kv.v_pages, kv.lo_pages, kv.hi_pages,
                                               kv.block_table, kv.nblocks, kv.ntokens)))
