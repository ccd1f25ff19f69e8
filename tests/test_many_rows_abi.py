"""Refusals of the 8-bit products, the beam selection and the page entry points, before a
device is touched (CPU only)."""
import ctypes

import pytest

FAKE = 0x10000  # never dereferenced


@pytest.fixture(scope="module")
def L(pkg):
    return pkg.gpu_lib()


def test_quantize_rows(pkg, L):
    def call(x=FAKE, t=pkg.F32, xs=0, q=FAKE, qs=0, s=FAKE, n=4, k=64):
        return L.swamp_quantize_rows(x, t, xs, q, qs, s, n, k, None)

    assert call(t=pkg.Q8_0) == pkg.EDTYPE
    assert call(n=-1) == pkg.EINVAL and call(k=-1) == pkg.EINVAL
    assert call(xs=-64) == pkg.EINVAL and call(qs=1 << 41) == pkg.EINVAL
    assert call(xs=63) == pkg.ESHAPE and call(qs=1) == pkg.ESHAPE
    assert call(x=None) == pkg.EINVAL and call(q=None) == pkg.EINVAL and call(s=None) == pkg.EINVAL
    assert call(x=FAKE + 2) == pkg.EINVAL and call(x=FAKE + 1, t=pkg.BF16) == pkg.EINVAL
    assert call(s=FAKE + 2) == pkg.EINVAL
    assert call(n=0, x=None, q=None, s=None) == pkg.OK


def test_gemm_rows_i8(pkg, L):
    def call(x=FAKE, xs=0, sx=FAKE, w=FAKE, ws=0, sw=FAKE, y=FAKE, t=pkg.F32, ys=0, m=4, n=8, k=64):
        return L.swamp_gemm_rows_i8(x, xs, sx, w, ws, sw, y, t, ys, m, n, k, 0, None)

    assert call(t=pkg.Q8_0) == pkg.EDTYPE
    for bad in ({"m": -1}, {"n": -1}, {"k": -1}, {"xs": -16}, {"ws": -16}, {"ys": -8}, {"sx": None},
                {"sw": None}, {"y": None}, {"x": None}, {"w": None}, {"x": FAKE + 8}, {"w": FAKE + 4},
                {"sx": FAKE + 2}, {"sw": FAKE + 1}, {"y": FAKE + 2}, {"y": FAKE + 1, "t": pkg.F16}):
        assert call(**bad) == pkg.EINVAL, bad
    # sums past int32; rows that do not begin at multiples of 16; strides of 8 MB; rows that overlap
    for bad in ({"k": 131072, "xs": 131072, "ws": 131072}, {"k": 60}, {"k": 60, "xs": 64},
                {"xs": 72}, {"ws": 72}, {"xs": 1 << 23}, {"ws": 1 << 23}, {"xs": 48}, {"ys": 7},
                {"m": 1 << 20, "n": 1 << 18}, {"m": (1 << 30) + 1, "n": 1},
                {"m": 1, "n": (1 << 30) + 1}, {"m": 1, "n": (1 << 31) - 1, "k": 1, "xs": 16, "ws": 16}):
        assert call(**bad) == pkg.ESHAPE, bad
    assert call(m=0, x=None, y=None) == pkg.OK and call(n=0, w=None, y=None) == pkg.OK
    for none in ((0, 8, 64), (8, -1, 64), (8, 8, 0), (8, 8, 131072), (1 << 20, 1 << 18, 64),
                 (1, (1 << 30) + 1, 16), ((1 << 30) + 1, 1, 16)):
        assert L.swamp_gemm_rows_i8_workspace(*none) == 0


def test_beam_select(pkg, L):
    def call(n=2, b=4, v=100, k=8, eos=3, t=pkg.F32, st=0, logits=FAKE, score=FAKE, done=FAKE,
             parent=FAKE, token=FAKE, out=FAKE, out_done=FAKE, spec=True):
        return L.swamp_beam_select(pkg.BeamSpec(n, b, v, k, eos) if spec else None, logits, t, st,
                                   score, done, parent, token, out, out_done, None)

    assert call(t=pkg.Q4_0) == pkg.EDTYPE
    for bad in ({"spec": False}, {"n": -1}, {"eos": -2}, {"eos": -1}, {"st": -100}, {"logits": None},
                {"score": None}, {"parent": None}, {"token": None}, {"out": None},
                {"logits": FAKE + 2}, {"logits": FAKE + 1, "t": pkg.F16}, {"done": FAKE + 2},
                {"out_done": FAKE + 1}, {"score": FAKE + 2}, {"parent": FAKE + 2},
                {"token": FAKE + 2}, {"out": FAKE + 2}):
        assert call(**bad) == pkg.EINVAL, bad
    for bad in ({"b": 0}, {"b": 65}, {"k": 0}, {"k": 65}, {"v": 0}, {"v": (1 << 20) + 1},
                {"eos": 100}, {"n": 65536}, {"st": 99}, {"n": 1024, "b": 64, "v": 1 << 20},
                {"n": 65535, "b": 64, "v": 4096 * 4 + 1}):
        assert call(**bad) == pkg.ESHAPE, bad
    assert call(n=0, logits=None, score=None) == pkg.OK
    assert L.swamp_beam_select_workspace(pkg.BeamSpec(0, 4, 100, 8)) == 0
    assert L.swamp_beam_select_workspace(pkg.BeamSpec(2, 65, 100, 8)) == 0
    assert L.swamp_beam_select_workspace(None) == 0


def pool(pkg, n=8, page=16, refs=FAKE, used=FAKE):
    return pkg.PagePool(n, page, refs, used)


def tables(pkg, n=4, lens=FAKE, pages=FAKE, stride=10, bad=0):
    return pkg.PageTables(n, lens, pages, stride, bad)


def moves(pkg, cap=8, src=FAKE, dst=FAKE, count=FAKE):
    return pkg.PageMoves(cap, src, dst, count)


def test_pools_and_tables(pkg, L):
    calls = {
        "fork": lambda p, t, m: L.swamp_pages_fork(p, t, FAKE, None),
        "extend": lambda p, t, m: L.swamp_pages_extend(p, t, FAKE, m, None),
        "trim": lambda p, t, m: L.swamp_pages_trim(p, t, FAKE, None),
        "compact": lambda p, t, m: L.swamp_pages_compact(p, t, m, None),
    }
    for name, call in calls.items():
        good = (pool(pkg), tables(pkg), moves(pkg))
        for bad in (None, pool(pkg, n=-1), pool(pkg, refs=0), pool(pkg, used=0),
                    pool(pkg, refs=FAKE + 2), pool(pkg, used=FAKE + 1)):
            assert call(bad, *good[1:]) == pkg.EINVAL, name
        for page in (0, -16, 24, 131072):
            assert call(pool(pkg, page=page), *good[1:]) == pkg.ESHAPE, name
        for bad in (None, tables(pkg, n=-1), tables(pkg, lens=0), tables(pkg, pages=0),
                    tables(pkg, stride=-1), tables(pkg, stride=1 << 41), tables(pkg, lens=FAKE + 2),
                    tables(pkg, pages=FAKE + 1), tables(pkg, bad=FAKE + 2)):
            assert call(good[0], bad, good[2]) == pkg.EINVAL, name
        assert call(good[0], tables(pkg, n=2049), moves(pkg, cap=4096)) == pkg.ESHAPE, name
        if name in ("extend", "compact"):
            for bad in (None, moves(pkg, cap=-1), moves(pkg, src=0), moves(pkg, dst=0),
                        moves(pkg, count=0), moves(pkg, src=FAKE + 2), moves(pkg, dst=FAKE + 2),
                        moves(pkg, count=FAKE + 1)):
                assert call(*good[:2], bad) == pkg.EINVAL, name
    assert calls["extend"](pool(pkg), tables(pkg), moves(pkg, cap=3)) == pkg.ESHAPE
    assert L.swamp_pages_fork(pool(pkg), tables(pkg), None, None) == pkg.EINVAL
    assert L.swamp_pages_fork(pool(pkg), tables(pkg), FAKE + 2, None) == pkg.EINVAL
    assert L.swamp_pages_extend(pool(pkg), tables(pkg), FAKE + 2, moves(pkg), None) == pkg.EINVAL
    assert L.swamp_pages_trim(pool(pkg), tables(pkg), FAKE + 2, None) == pkg.EINVAL
    assert L.swamp_pages_fork(pool(pkg), tables(pkg, n=0), None, None) == pkg.OK
    assert L.swamp_pages_trim(pool(pkg), tables(pkg, n=0), None, None) == pkg.OK


def test_kv_copy(pkg, L):
    def cache(k=FAKE, v=FAKE, t=pkg.BF16, n=8, page=16, heads=2, dim=64, strides=(0, 0, 0)):
        return pkg.KvPages(k, v, t, n, page, heads, dim, *strides)

    def call(caches, m=True):
        return L.swamp_kv_copy(pkg.kv_caches(caches), len(caches), moves(pkg) if m else None, None)

    assert call([cache()], m=False) == pkg.EINVAL
    assert L.swamp_kv_copy(None, 1, moves(pkg), None) == pkg.EINVAL
    assert L.swamp_kv_copy(pkg.kv_caches([cache()]), -1, moves(pkg), None) == pkg.EINVAL
    assert call([cache(), cache(k=0)]) == pkg.EINVAL and call([cache(v=FAKE + 8)]) == pkg.EINVAL
    assert call([cache(t=pkg.F32)]) == pkg.EDTYPE
    for other in (cache(t=pkg.F16), cache(n=9), cache(page=32), cache(heads=4), cache(dim=128),
                  cache(strides=(4096, 0, 0)), cache(strides=(0, 2048, 0)), cache(strides=(0, 0, 128))):
        assert call([cache(), other]) == pkg.ESHAPE
    # a page of 2^33 elements
    assert call([cache(n=1, page=65536, heads=1024, dim=128)]) == pkg.ESHAPE
    assert call([]) == pkg.OK
    assert L.swamp_kv_copy(pkg.kv_caches([cache()]), 1, moves(pkg, cap=0), None) == pkg.OK
    assert call([cache(k=0, v=0, n=0)]) == pkg.OK


def test_structures_match_the_header(pkg):
    """Sizes that the C structures have (the fields' order is the header's)."""
    sizes = {pkg.BeamSpec: 20, pkg.PagePool: 24, pkg.PageTables: 40, pkg.PageMoves: 32}
    for s, n in sizes.items():
        assert ctypes.sizeof(s) == n
