"""How far the buffers of the paged entry points may reach: sums of strides that
would leave 64 bits are refused, without a GPU."""
import pytest

from test_paging import FAKE, _batch, _cache

BIG = 2 ** 31 - 1


def _attn(pkg, cache=None, batch=None, **more):
    a = dict(qs=0, os_=0, heads=4)
    a.update(more)
    return pkg.gpu_lib().swamp_attn_paged(
        _cache(pkg, **(cache or {})), _batch(pkg, **(batch or {})), FAKE, a["qs"], a["heads"], 0.125,
        0, FAKE, pkg.F32, a["os_"], None)


def _append(pkg, cache=None, batch=None, qs=0, ks=0, vs=0, os_=0):
    return pkg.gpu_lib().swamp_kv_append(
        _cache(pkg, **(cache or {})), _batch(pkg, **(batch or {})), None, FAKE, FAKE, FAKE, pkg.F32,
        qs, ks, vs, FAKE, os_, 4, None)


@pytest.mark.parametrize("n_pages", [2 ** 31 - 1, 2 ** 24, 2 ** 21])
def test_pages_past_64_bits_are_refused(pkg, n_pages):
    """A page id below n_pages is a bound only if the pages' offsets do not wrap:
    2^40 elements apart, these reach 2^71, 2^64 and 2^61 of them."""
    far = dict(n_pages=n_pages, page_stride=2 ** 40)
    assert _attn(pkg, cache=far) == pkg.EINVAL
    assert _append(pkg, cache=far) == pkg.EINVAL
    assert pkg.gpu_lib().swamp_attn_paged_workspace(_cache(pkg, **far), _batch(pkg), 4, 0) == 0


def test_rows_past_64_bits_are_refused(pkg):
    far = 2 ** 40
    tok = dict(n_tok=BIG)
    for more in (dict(qs=far), dict(os_=far)):
        assert _attn(pkg, batch=tok, **more) == pkg.EINVAL
        assert _append(pkg, batch=tok, **more) == pkg.EINVAL
    for more in (dict(ks=far), dict(vs=far)):
        assert _append(pkg, batch=tok, **more) == pkg.EINVAL
    L, r = pkg.gpu_lib(), pkg.Rope(FAKE, 64, 0)
    for xs, os_ in ((far, 0), (0, far)):
        assert L.swamp_rope(r, FAKE, FAKE, pkg.F32, xs, FAKE + 4096, pkg.F32, os_, BIG, 2, 64,
                            None) == pkg.EINVAL


def test_page_tables_past_64_bits_are_refused(pkg):
    for n, stride in ((65535, 2 ** 48), (3, 2 ** 62), (2, 2 ** 63 - 1)):
        assert _attn(pkg, batch=dict(n_seq=n, pages_stride=stride)) == pkg.EINVAL
        assert _append(pkg, batch=dict(n_seq=n, pages_stride=stride)) == pkg.EINVAL
