"""How swamp_attn_paged cuts a call (csrc/attn_plan.hpp, built for the host): block
and piece counts over the whole range of its arguments, without a GPU."""
import ctypes
import os
import random
import subprocess

import pytest

from test_paging import FAKE, _batch, _cache

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256  # MI355X
MOST = 2 ** 32 // 256 - 1  # workgroups of 256 threads that one launch can have

SHIM = """
#include "attn_plan.hpp"
extern "C" void plan(const long *a, int cus, long *o) {
  swamp::AttnCall c = {};
  c.batch.n_seq = int(a[0]); c.batch.n_tok = int(a[1]);
  c.max_new = int(a[2]); c.max_len = int(a[3]);
  c.n_heads = int(a[4]); c.cache.n_kv = int(a[5]); c.cache.dim = int(a[6]);
  c.window = int(a[7]); c.cache.page_shift = int(a[8]); c.batch.pages_stride = a[9];
  const swamp::AttnPlan p = swamp::plan_attn(c, cus);
  o[0] = p.blocks; o[1] = p.few; o[2] = p.splits; o[3] = p.chunk;
  o[4] = long(swamp::attn_part_bytes(c, p.splits) + swamp::attn_stat_bytes(c, p.splits));
}
"""


class Plan:
    def __init__(self, lib, **a):
        a = dict(dict(window=0, shift=5, table=1 << 40), **a)
        keys = ("seqs", "tok", "new", "len", "heads", "kv", "dim", "window", "shift", "table")
        args, out = (ctypes.c_long * 10)(*[a[k] for k in keys]), (ctypes.c_long * 5)()
        lib.plan(args, CUS, out)
        self.blocks, self.few, self.splits, self.chunk, self.bytes = out
        self.groups = self.blocks * a["kv"] * self.splits


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    src, so = str(d / "plan.cpp"), str(d / "plan.so")
    with open(src, "w") as f:
        f.write(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC",
                    "-I" + os.path.join(REPO, "include"),
                    "-I" + os.path.join(REPO, "llamanyon.rs_amd", "csrc"), src, "-o", so],
                   check=True)
    return ctypes.CDLL(so)


def _sound(p, a):
    """Pieces of whole tiles, not more than the keys fill, and one launch holds them."""
    step = 128 if p.few else 64
    assert p.chunk >= step and p.chunk % step == 0 and p.chunk < 2 ** 31, a
    assert p.splits >= 1 and p.blocks >= 1, a
    keys = min(a["len"], 2 ** 31 - 512)
    assert p.splits == 1 or (p.splits - 1) * p.chunk < keys, a
    assert p.groups <= MOST, a


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 64, 2 ** 31 - 65,
                                    2 ** 31 - 512, 2 ** 31 - 513, 2 ** 30])
def test_longest_hints(lib, length):
    """max_len is any int from 0 on; one near the largest is an ordinary hint."""
    for seqs, new, heads, kv, dim in ((64, 512, 64, 8, 128), (64, 4, 64, 8, 128), (1, 1, 8, 1, 8),
                                      (300, 1, 8, 8, 64), (16, 200, 4, 4, 256), (1, 1, 1, 1, 8)):
        for window in (0, 2 ** 30, 2 ** 31 - 1):
            a = dict(seqs=seqs, tok=seqs * new, new=new, len=length, heads=heads, kv=kv, dim=dim,
                     window=window)
            _sound(Plan(lib, **a), a)


def test_pieces_past_the_page_table_are_not_made(lib):
    """Positions that no column of the page table holds are never walked, whatever
    the hint says."""
    for new in (1, 100):
        a = dict(seqs=4, tok=4 * new, new=new, heads=8, kv=2, dim=128, shift=4, table=20)
        p, q = Plan(lib, len=2 ** 31 - 1, **a), Plan(lib, len=16 * 20, **a)
        assert (p.splits, p.chunk) == (q.splits, q.chunk)


def test_plans_over_the_whole_range(lib):
    rng = random.Random(5)

    def span(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    for _ in range(20000):
        kv, group, seqs = span(1, 64), span(1, 64), span(1, 65535)
        new = span(1, 5000)
        a = dict(seqs=seqs, tok=min(seqs * new, 2 ** 22), new=new, len=span(1, 2 ** 31 - 1),
                 heads=kv * group, kv=kv, dim=8 * span(1, 32),
                 window=rng.choice([0, 0, span(1, 2 ** 31 - 1)]))
        p = Plan(lib, **a)
        if p.blocks * kv <= MOST:  # (else the call is refused)
            _sound(p, a)


def test_calls_past_one_launch_are_refused(pkg):
    """More blocks of rows than a launch can have."""
    def call(cache, batch, heads):
        return pkg.gpu_lib().swamp_attn_paged(_cache(pkg, **cache), _batch(pkg, **batch), FAKE, 0,
                                              heads, 0.125, 0, FAKE, pkg.F32, 0, None)
    many = dict(n_seq=65535, n_tok=65535, max_new=1)
    assert call(dict(n_kv_heads=4096, n_pages=1), many, 4096) == pkg.ESHAPE
    assert call(dict(n_kv_heads=257), many, 257) == pkg.ESHAPE
    tokens = dict(n_seq=1, n_tok=2 ** 31 - 1, max_new=2 ** 31 - 1)
    assert call(dict(n_kv_heads=2), tokens, 4) == pkg.ESHAPE


@pytest.mark.parametrize("length", [2 ** 17, 2 ** 20, 2 ** 24, 2 ** 31 - 1])
def test_pieces_and_their_sums_stay_bounded(lib, length):
    """A captured step's max_len is its context's limit, whatever the lengths are: at
    most 16 pieces where the rows alone fill the card, and 256 MB of partial sums."""
    for seqs in (11, 16, 64, 300, 5000):
        for new in (1, 4, 32, 200):
            a = dict(seqs=seqs, tok=seqs * new, new=new, len=length, heads=64, kv=8, dim=128)
            p = Plan(lib, **a)
            assert p.splits == 1 or p.bytes <= 2 ** 28, a
            assert p.splits <= 16, a


def test_piece_counts_of_ordinary_lengths(lib):
    """Where neither bound is met the count is what the measured rules say."""
    def pieces(**a):
        return Plan(lib, **a).splits
    one = dict(seqs=1, tok=1, new=1, heads=32, kv=8, dim=128)
    assert pieces(len=131072, **one) == 32 and pieces(len=512, **one) == 1
    assert pieces(seqs=64, tok=63, new=1, len=8192, heads=64, kv=8, dim=128) == 4
    assert pieces(seqs=8, tok=40, new=5, len=4001, heads=32, kv=8, dim=128) == 4
    assert pieces(seqs=1, tok=512, new=512, len=16384, heads=32, kv=8, dim=128) == 4
    assert pieces(seqs=1, tok=4096, new=4096, len=4096, heads=64, kv=8, dim=128) == 1
