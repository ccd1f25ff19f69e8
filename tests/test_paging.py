"""Rotary positions, the paged cache's append and attention over it, without a
GPU: the index arithmetic of csrc/paging.hpp (the kernels' own source, built
for the host), what the entry points refuse, and the frequencies."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 0x10000  # never dereferenced: every call below is refused or has no work

SHIM = """
#include "paging.hpp"
extern "C" {
void seq_of(int first, int next, int len, int n_tok, int *o) {
  const swamp::Seq s = swamp::seq_of(first, next, len, n_tok);
  o[0] = s.t0; o[1] = s.n; o[2] = s.len;
}
void seen_by(int pos, int window, int *o) {
  const swamp::Span k = swamp::seen_by(pos, window);
  o[0] = k.lo; o[1] = k.hi;
}
long slot(int id, int pos, int head, int shift, long ps, long hs, long ss, long stride, int n) {
  const int64_t col = swamp::page_col(pos, shift);
  if (!swamp::page_col_ok(pos, col, stride) || !swamp::page_ok(id, n)) return -1;
  return swamp::slot_offset(id, pos, head, shift, ps, hs, ss);
}
}
"""


@pytest.fixture(scope="module")
def paging(tmp_path_factory):
    d = tmp_path_factory.mktemp("paging")
    src, lib = str(d / "paging.cpp"), str(d / "paging.so")
    with open(src, "w") as f:
        f.write(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC",
                    "-I" + os.path.join(REPO, "include"),
                    "-I" + os.path.join(REPO, "llamanyon.rs_amd", "csrc"), src, "-o", lib],
                   check=True)
    so = ctypes.CDLL(lib)
    so.slot.restype = ctypes.c_long
    so.slot.argtypes = [ctypes.c_int] * 4 + [ctypes.c_long] * 4 + [ctypes.c_int]
    return so


def _ints(fn, n, *a):
    o = (ctypes.c_int * n)()
    fn(*a, o)
    return tuple(o)


def test_rows_stay_in_the_batch(paging):
    """Whatever the device arrays hold, a sequence's rows lie in 0 .. n_tok - 1."""
    assert _ints(paging.seq_of, 3, 3, 8, 20, 100) == (3, 5, 20)
    assert _ints(paging.seq_of, 3, 8, 8, 0, 100) == (8, 0, 0)
    big = 2 ** 31 - 1
    for first in (-big - 1, -1, 0, 7, 100, 101, big):
        for nxt in (-big - 1, -1, 0, 6, 7, 100, 101, big):
            for length in (-big - 1, -1, 0, 5, big):
                t0, n, ln = _ints(paging.seq_of, 3, first, nxt, length, 100)
                assert 0 <= t0 <= 100 and 0 <= n and t0 + n <= 100 and ln == max(0, length)


def test_keys_a_row_sees(paging):
    for pos in (-3, -1, 0, 1, 5, 31, 32, 2 ** 31 - 2):
        for window in (0, 1, 2, 32, 1 << 29):
            lo, hi = _ints(paging.seen_by, 2, pos, window)
            want_hi = max(0, pos + 1)
            assert hi == want_hi
            assert lo == (max(0, want_hi - window) if window else 0)
            assert hi == 0 or lo < hi  # a row at a position sees itself


def test_slots_stay_in_the_pages(paging):
    """Page ids outside the cache and positions outside the table have no slot;
    the others' offsets pass 32 bits without wrapping."""
    ps, hs, ss, n = 4 * 16 * 64, 16 * 64, 64, 10
    for id_ in (-2 ** 31, -7, -1, 10, 11, 2 ** 31 - 1):
        assert paging.slot(id_, 5, 1, 4, ps, hs, ss, 8, n) == -1
    for pos in (-2 ** 31, -1, 8 * 16, 8 * 16 + 5, 2 ** 31 - 1):
        assert paging.slot(3, pos, 1, 4, ps, hs, ss, 8, n) == -1
    seen = set()
    for id_ in range(n):
        for pos in range(8 * 16):
            for head in range(4):
                at = paging.slot(id_, pos, head, 4, ps, hs, ss, 8, n)
                assert 0 <= at <= n * ps - 64
                seen.add(at)
    assert len(seen) == n * 4 * 16
    assert paging.slot(9, 127, 3, 4, 2 ** 33, hs, ss, 8, n) == 9 * 2 ** 33 + 3 * hs + 15 * ss


# ------------------------------------------------------------------- refusals

def _cache(pkg, **more):
    a = dict(d_k=FAKE, d_v=FAKE, dtype=pkg.F16, n_pages=8, page_size=16, n_kv_heads=2, head_dim=64)
    a.update(more)
    return pkg.KvPages(**a)


def _batch(pkg, **more):
    a = dict(n_seq=2, n_tok=4, max_new=2, max_len=20, d_first=FAKE, d_len=FAKE, d_pages=FAKE,
             pages_stride=4)
    a.update(more)
    return pkg.SeqBatch(**a)


def test_rope_refusals(pkg):
    L = pkg.gpu_lib()

    def call(rot=64, layout=0, freqs=FAKE, pos=FAKE, x=FAKE, xt=pkg.F32, xs=0, out=FAKE + 4096,
             ot=pkg.F32, os_=0, n=4, heads=2, dim=64, spec=True):
        r = pkg.Rope(freqs, rot, layout) if spec else None
        return L.swamp_rope(r, pos, x, xt, xs, out, ot, os_, n, heads, dim, None)

    assert call(spec=False) == pkg.EINVAL and call(freqs=None) == pkg.EINVAL
    assert call(freqs=FAKE + 4) == pkg.EINVAL and call(layout=2) == pkg.EINVAL
    assert call(rot=0) == pkg.ESHAPE and call(rot=63) == pkg.ESHAPE and call(rot=66) == pkg.ESHAPE
    assert call(dim=65) == pkg.ESHAPE and call(dim=514) == pkg.ESHAPE and call(dim=0) == pkg.EINVAL
    assert call(xt=pkg.Q8_0) == pkg.EDTYPE and call(ot=pkg.Q4_0) == pkg.EDTYPE
    assert call(xs=127) == pkg.ESHAPE and call(os_=127) == pkg.ESHAPE
    assert call(xs=-128) == pkg.EINVAL and call(n=-1) == pkg.EINVAL and call(heads=-1) == pkg.EINVAL
    assert call(pos=None) == pkg.EINVAL and call(x=None) == pkg.EINVAL
    assert call(out=None) == pkg.EINVAL and call(x=FAKE + 2) == pkg.EINVAL
    assert call(xt=pkg.F16, x=FAKE + 1) == pkg.EINVAL and call(out=FAKE + 1) == pkg.EINVAL
    # in place with another type or stride
    assert call(out=FAKE, ot=pkg.F16) == pkg.EINVAL and call(out=FAKE, os_=256) == pkg.EINVAL
    assert call(n=0) == pkg.OK and call(heads=0) == pkg.OK


def test_kv_append_refusals(pkg):
    L = pkg.gpu_lib()

    def call(cache=None, batch=None, rot=64, q=FAKE, k=FAKE, v=FAKE, xt=pkg.F32, qs=0, ks=0, vs=0,
             out=FAKE, os_=0, heads=4):
        return L.swamp_kv_append(_cache(pkg, **(cache or {})), _batch(pkg, **(batch or {})),
                                 pkg.Rope(FAKE, rot, 0) if rot else None, q, k, v, xt, qs, ks, vs,
                                 out, os_, heads, None)

    assert L.swamp_kv_append(None, _batch(pkg), None, FAKE, FAKE, FAKE, 0, 0, 0, 0, FAKE, 0, 4,
                             None) == pkg.EINVAL
    assert L.swamp_kv_append(_cache(pkg), None, None, FAKE, FAKE, FAKE, 0, 0, 0, 0, FAKE, 0, 4,
                             None) == pkg.EINVAL
    for bad, code in ((dict(dtype=pkg.F32), pkg.EDTYPE), (dict(dtype=pkg.Q8_0), pkg.EDTYPE),
                      (dict(page_size=24), pkg.ESHAPE), (dict(page_size=0), pkg.ESHAPE),
                      (dict(page_size=1 << 17), pkg.ESHAPE), (dict(head_dim=60), pkg.ESHAPE),
                      (dict(head_dim=264), pkg.ESHAPE), (dict(head_dim=0), pkg.ESHAPE),
                      (dict(n_kv_heads=0), pkg.EINVAL), (dict(n_pages=-1), pkg.EINVAL),
                      (dict(page_stride=-8), pkg.EINVAL), (dict(slot_stride=56), pkg.ESHAPE),
                      (dict(head_stride=1020), pkg.ESHAPE), (dict(d_k=0), pkg.EINVAL),
                      (dict(d_v=FAKE + 8), pkg.EINVAL)):
        assert call(cache=bad) == code, bad
    for bad in (dict(n_seq=-1), dict(n_tok=-1), dict(max_new=-1), dict(max_len=-1),
                dict(pages_stride=-1), dict(d_first=0), dict(d_len=FAKE + 2), dict(d_pages=0),
                dict(d_bad=FAKE + 1), dict(n_seq=70000)):
        assert call(batch=bad) == pkg.EINVAL, bad
    assert call(rot=66) == pkg.ESHAPE and call(xt=pkg.Q8_0) == pkg.EDTYPE
    assert call(q=None) == pkg.EINVAL and call(out=None) == pkg.EINVAL
    assert call(k=None) == pkg.EINVAL and call(v=FAKE + 2) == pkg.EINVAL
    assert call(qs=255) == pkg.ESHAPE and call(ks=127) == pkg.ESHAPE and call(vs=64) == pkg.ESHAPE
    assert call(os_=64) == pkg.ESHAPE and call(heads=-1) == pkg.EINVAL
    assert call(batch=dict(n_tok=0)) == pkg.OK and call(batch=dict(n_seq=0), k=None) == pkg.OK


def test_attn_paged_refusals(pkg):
    L = pkg.gpu_lib()

    def call(cache=None, batch=None, q=FAKE, qs=0, heads=4, scale=0.125, window=0, out=FAKE,
             ot=pkg.F32, os_=0):
        return L.swamp_attn_paged(_cache(pkg, **(cache or {})), _batch(pkg, **(batch or {})), q, qs,
                                  heads, scale, window, out, ot, os_, None)

    assert L.swamp_attn_paged(None, _batch(pkg), FAKE, 0, 4, 1.0, 0, FAKE, 0, 0, None) == pkg.EINVAL
    assert call(cache=dict(dtype=pkg.F32)) == pkg.EDTYPE and call(ot=pkg.Q8_0) == pkg.EDTYPE
    assert call(heads=3) == pkg.ESHAPE and call(heads=0) == pkg.EINVAL
    assert call(window=-1) == pkg.EINVAL and call(scale=math.inf) == pkg.EINVAL
    assert call(scale=math.nan) == pkg.EINVAL
    assert call(qs=260) == pkg.ESHAPE and call(qs=128) == pkg.ESHAPE and call(os_=258) == pkg.ESHAPE
    assert call(q=None) == pkg.EINVAL and call(q=FAKE + 8) == pkg.EINVAL
    assert call(out=None) == pkg.EINVAL and call(out=FAKE + 8) == pkg.EINVAL
    assert call(cache=dict(d_k=0)) == pkg.EINVAL and call(batch=dict(d_len=0)) == pkg.EINVAL
    assert call(cache=dict(page_size=48)) == pkg.ESHAPE
    for none in (dict(n_seq=0), dict(n_tok=0), dict(max_new=0)):
        assert call(batch=none, q=None) == pkg.OK, none
    with pytest.raises(pkg.GpuError):
        pkg.attn_paged(_cache(pkg), _batch(pkg), FAKE, 3, 1.0, FAKE, pkg.F32)


# ---------------------------------------------------------------- frequencies

def test_rope_freqs_plain_and_linear(pkg):
    i = np.arange(64)
    np.testing.assert_allclose(pkg.rope_freqs(128, 500000.0), 500000.0 ** (-i / 64), rtol=1e-14)
    np.testing.assert_allclose(pkg.rope_freqs(128, factor=4.0), 10000.0 ** (-i / 64) / 4,
                               rtol=1e-14)
    div = np.linspace(1, 8, 64).astype(np.float32)
    np.testing.assert_allclose(pkg.rope_freqs(128, divisors=div), 10000.0 ** (-i / 64) / div,
                               rtol=1e-14)


def test_rope_freqs_ramp(pkg):
    """Pairs that turn more than 32 times in the trained context keep their
    frequency, those that turn less than once are divided, between them a
    straight line."""
    n, base, factor, ctx = 128, 10000.0, 8.0, 4096
    f = pkg.rope_freqs(n, base, factor, ctx)
    plain = base ** (-np.arange(n // 2) / (n // 2))
    turns = plain * ctx / (2 * math.pi)
    share = (plain / f - 1) * f / plain / (1 - 1 / factor)  # 0: kept, 1: divided
    assert np.all(share[turns > 32 * 1.2] < 1e-12) and np.all(share[turns < 1 / 1.2] > 1 - 1e-12)
    assert np.all(np.diff(share) > -1e-12) and np.any((share > 0.1) & (share < 0.9))
    inner = share[(share > 1e-9) & (share < 1 - 1e-9)]
    np.testing.assert_allclose(np.diff(inner), np.diff(inner).mean(), rtol=1e-9)


def test_rope_freqs_refusals(pkg):
    for a in (dict(n_rot=0), dict(n_rot=7)):
        with pytest.raises(pkg.GpuError) as e:
            pkg.rope_freqs(**a)
        assert e.value.code == pkg.ESHAPE
    for a in (dict(base=1.0), dict(base=math.nan), dict(factor=0.0), dict(factor=math.inf),
              dict(orig_ctx=-1), dict(factor=2.0, orig_ctx=100, beta_slow=0.0),
              dict(factor=2.0, orig_ctx=100, beta_fast=1.0), dict(divisors=[1.0, 0.0, 1.0, 1.0])):
        with pytest.raises(pkg.GpuError) as e:
            pkg.rope_freqs(**dict(dict(n_rot=8), **a))
        assert e.value.code == pkg.EINVAL, a
    with pytest.raises(ValueError):
        pkg.rope_freqs(8, divisors=[1.0])
