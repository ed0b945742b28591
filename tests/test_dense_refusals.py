"""Argument errors of the dense operators' C entry points: reported before any device is
touched (no GPU needed)."""
import pytest

X = 4096                                            # any address: nothing is read


@pytest.fixture(scope="module")
def lib():
    from strict_topk import _lib
    if not _lib._PATH.exists():
        import build_lib
        build_lib.build()
    return _lib.lib()


EXTEND = dict(k=X, ks=512, v=X, vs=512, q=X, qs=512, qo=X, dtype=2, tokens=10, requests=2, hq=8,
              hkv=2, nb=4, b=32, d=64, pages=9, starts=X, positions=X, cos=X, sin=X, rows=128,
              rot=64, inter=0, kp=X, vp=X, lo=X, hi=X, bounds=2, table=X, nblocks=X, ntokens=X * 2,
              stream=None)
ATTEND = dict(q=X, qs=512, dtype=2, tokens=10, requests=2, hq=8, hkv=2, nb=4, b=32, d=64, pages=9,
              kp=X, vp=X, table=X, nblocks=X, ntokens=X, starts=X, scale=0.1, softcap=0.0,
              slopes=None, window=0, prefix=None, first=None, out=X, fill=1, ws=X, bytes=1 << 40,
              stream=None)
SHARED = dict(q=X, qs=512, dtype=2, requests=3, hq=8, hkv=2, nb=4, b=32, d=64, pages=9, kp=X,
              vp=X, table=X, nblocks=X, ntokens=X, groups=X, shared=X, ngroups=1, scale=0.1,
              softcap=0.0, slopes=None, window=0, first=None, out=X, ws=X, bytes=1 << 40,
              stream=None)


@pytest.mark.parametrize("kw,why", [
    (dict(dtype=0), "FP16 or BF16"), (dict(d=96), "64, 128 or 256"), (dict(k=None), "null"),
    (dict(kp=None), "null"), (dict(starts=None), "null"), (dict(q=X, qo=None), "q_out"),
    (dict(cos=None, sin=None), "tables"), (dict(cos=None, q=None), "go together"),
    (dict(rot=72), "multiple of 16"), (dict(rot=128), "multiple of 16"),
    (dict(rows=127), "every position"), (dict(bounds=1), "lo and hi"), (dict(k=X + 2), "aligned"),
    (dict(ks=510), "aligned"), (dict(ks=-8), "negative"), (dict(ntokens=X), "ntokens"),
    (dict(requests=0), "bad shape"), (dict(nb=1 << 20, b=1 << 12), "too large"),
    (dict(tokens=-1), "bad shape"), (dict(hq=0), "head")])
def test_extend(lib, kw, why):
    assert lib.stk_paged_extend(*dict(EXTEND, **kw).values()) == -1
    assert why in lib.stk_last_error().decode()


COMMON = [(dict(dtype=0), "FP16 or BF16"), (dict(d=96), "64, 128 or 256"),
          (dict(b=24), "multiple of 16"), (dict(hq=7), "divisible"), (dict(hq=0), "nonempty"),
          (dict(q=None), "null"), (dict(kp=None), "null"), (dict(nblocks=None), "null"),
          (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
          (dict(scale=float("inf")), "scale"), (dict(softcap=-1.0), "softcap"),
          (dict(softcap=float("nan")), "softcap"), (dict(softcap=4097.0), "softcap"),
          (dict(softcap=1e-35), "softcap"), (dict(scale=2e30), "scale"), (dict(window=-1), "window"),
          (dict(q=X + 2), "aligned"), (dict(qs=511), "aligned"), (dict(ws=None), "workspace"),
          (dict(bytes=16), "workspace"), (dict(pages=1 << 30), "too large"),
          (dict(nb=1 << 26), "too large"), (dict(pages=0), "bad shape")]


@pytest.mark.parametrize("kw,why", COMMON + [(dict(starts=None), "one query token"),
                                             (dict(tokens=-1), "bad shape")])
def test_attention(lib, kw, why):
    assert lib.stk_paged_attention(*dict(ATTEND, **kw).values()) == -1
    assert why in lib.stk_last_error().decode()


@pytest.mark.parametrize("kw,why", COMMON + [(dict(groups=None), "null"), (dict(ngroups=0), "groups"),
                                             (dict(ngroups=4), "groups")])
def test_shared(lib, kw, why):
    assert lib.stk_paged_shared_attention(*dict(SHARED, **kw).values()) == -1
    assert why in lib.stk_last_error().decode()


def test_nothing_to_do(lib):
    """No token: no launch, whatever the pointers."""
    assert lib.stk_paged_extend(*dict(EXTEND, tokens=0).values()) == 0
    assert lib.stk_paged_attention(*dict(ATTEND, tokens=0).values()) == 0


def test_workspace_queries(lib):
    size = lib.stk_paged_attention_workspace_bytes
    assert size(0, 2, 8, 2, 4, 32, 64, 1) == 0 and size(4, 2, 8, 3, 4, 32, 64, 1) == 0
    assert 0 < size(2, 2, 8, 2, 4, 32, 64, 0) < size(2, 2, 8, 2, 400, 32, 64, 0)
    shared = lib.stk_paged_shared_workspace_bytes
    assert shared(4, 0, 8, 2, 4, 32, 64) == 0
    assert shared(4, 1, 8, 2, 4, 32, 64) > size(4, 4, 8, 2, 4, 32, 64, 0)
