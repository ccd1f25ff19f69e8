"""swamp_pages_fork, _extend, _trim, _compact and swamp_kv_copy on the GPU against one
sequence and one page after the other on the host (tests/pages_reference.py)."""
import random

import pytest
import torch

from pages_reference import OnGpu, Pool, random_pool

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()
    pkg.init()
    return torch.device("cuda")


def say(*a):
    print("[gpu case]", *a, flush=True)


def stream():
    return torch.cuda.current_stream().cuda_stream


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


SIZES = [  # pages, page size, sequences, width of the tables
    (1, 1, 1, 1), (7, 1, 3, 4), (64, 16, 4, 9), (300, 8, 33, 17), (4099, 4, 257, 40),
    (33, 65536, 2, 16), (1000, 32, 64, 1), (140000, 1, 5, 300), (5000, 2, 2048, 3),
]


@pytest.mark.parametrize("size", SIZES)
def test_fork(pkg, dev, size):
    say("fork", size)
    rng = random.Random(str(size))
    p = random_pool(rng, *size)
    n = p.n
    for kind in ("same", "beams", "any", "ends"):
        g = OnGpu(pkg, p)
        if kind == "same":
            parent = list(range(n))
        elif kind == "beams":  # groups of 4 continue one of their own
            parent = [min(s - s % 4 + rng.randrange(4), n - 1) for s in range(n)]
        elif kind == "any":
            parent = [rng.randrange(n) for _ in range(n)]
        else:
            parent = [rng.choice([-1, s, n, -(1 << 31), (1 << 31) - 1]) for s in range(n)]
        d = i32(parent)
        pkg.pages_fork(g.pool, g.tables, d.data_ptr(), stream=stream())
        p.fork(parent)
        g.same(moves=False)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("after", ["fork", "alone"])
def test_extend(pkg, dev, size, after):
    say("extend", size, after)
    rng = random.Random(str(size))
    p = random_pool(rng, *size)
    if after == "fork":
        p.fork([rng.randrange(p.n) for _ in range(p.n)])
    for news in ("one", "some"):
        g = OnGpu(pkg, p)
        if news == "one":
            new, d = [1] * p.n, None
        else:
            new = [rng.choice([0, 1, 2, p.page, 3 * p.page + 1, -5]) for _ in range(p.n)]
            d = i32(new)
        g.bad.fill_(p.bad)
        pkg.pages_extend(g.pool, g.tables, d.data_ptr() if d is not None else 0, g.moves,
                         stream=stream())
        p.extend(new)
        g.same()


def test_extend_runs_out(pkg, dev):
    """Pages run out within a sequence, before a copy, and behind the table's end."""
    say("extend runs out")
    p = Pool(6, 4, 4, 3)
    p.table[0][:2], p.len[0] = [5, 2], 7
    p.table[1][:2], p.len[1] = [5, 2], 7
    p.table[2][:2], p.len[2] = [5, 2], 6
    p.refs[5] = p.refs[2] = 3
    g = OnGpu(pkg, p)
    d = i32([2, 9, 1, 1])
    pkg.pages_extend(g.pool, g.tables, d.data_ptr(), g.moves, stream=stream())
    p.extend([2, 9, 1, 1])
    assert p.bad == 1 and len(p.moves) == 2
    g.same()
    # nothing is free: a copy that finds no page leaves its sequence without one
    p = Pool(1, 4, 2, 1)
    p.table[0][0] = p.table[1][0] = 0
    p.len, p.refs = [3, 2], [2]
    g = OnGpu(pkg, p)
    pkg.pages_extend(g.pool, g.tables, 0, g.moves, stream=stream())
    p.extend([1, 1])
    assert p.table[0][0] == -1 and p.table[1][0] == 0 and p.bad == 1 and not p.moves
    g.same()


def test_free_pages_far_up(pkg, dev):
    """Pages held outside the tables fill the first rounds of the search; the free ones
    lie in a word's middle, at words' ends and past 131072."""
    say("far free pages")
    n_pages = 270000
    p = Pool(n_pages, 1, 3, 9)
    p.refs = [1] * n_pages
    for e in (31, 32, 131071, 131072, 131103, 200000, 262143, 262144, 269999):
        p.refs[e] = 0
    g = OnGpu(pkg, p)
    d = i32([2, 0, 5])
    pkg.pages_extend(g.pool, g.tables, d.data_ptr(), g.moves, stream=stream())
    p.extend([2, 0, 5])
    g.same(whole=False)
    assert p.table[0][:2] == [31, 32] and p.table[2][:2] == [131071, 131072]
    d.fill_(1)
    pkg.pages_extend(g.pool, g.tables, d.data_ptr(), g.moves, stream=stream())
    p.extend([1, 1, 1])
    g.same(whole=False)
    assert p.bad == 1 and p.table[2][5] == -1


def test_extend_to_the_last_position(pkg, dev):
    """Lengths up to 2^31 - 1, on pages of 65536."""
    say("extend last position")
    p = Pool(5, 65536, 2, 32768)
    p.len = [2 ** 31 - 1 - 65536, 0]
    for s in range(2):
        p.table[s] = [-1] * p.width
    g = OnGpu(pkg, p)
    d = i32([65535, 2 ** 31 - 1])
    pkg.pages_extend(g.pool, g.tables, d.data_ptr(), g.moves, stream=stream())
    torch.cuda.synchronize()
    # the first: the room left in its last page is no page's (-1), then one page; the second
    # takes the four others and finds none for the rest
    assert g.len.tolist() == [2 ** 31 - 2, 2 ** 31 - 1] and int(g.bad) == 1
    assert g.table[0, 32767].item() == 0 and g.table[0, :32767].eq(-1).all()
    assert g.table[1, :4].tolist() == [1, 2, 3, 4] and g.table[1, 4:].eq(-1).all()
    # more tokens than there are positions
    d.fill_(5)
    pkg.pages_extend(g.pool, g.tables, d.data_ptr(), g.moves, stream=stream())
    torch.cuda.synchronize()
    assert g.len.tolist() == [2 ** 31 - 1, 2 ** 31 - 1]


@pytest.mark.parametrize("size", SIZES)
def test_trim(pkg, dev, size):
    say("trim", size)
    rng = random.Random(str(size))
    p = random_pool(rng, *size)
    for kind in ("some", "all"):
        g = OnGpu(pkg, p)
        if kind == "all":
            keep, d = [0] * p.n, None
        else:
            keep = [rng.choice([0, n, n // 2, n + 5, -1, 2 ** 31 - 1]) for n in p.len]
            d = i32(keep)
        pkg.pages_trim(g.pool, g.tables, d.data_ptr() if d is not None else 0, stream=stream())
        p.trim(keep)
        g.same(moves=False)
    assert not any(p.refs) and not any(p.words())


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("cap", ["all", 3, 0])
def test_compact(pkg, dev, size, cap):
    say("compact", size, cap)
    rng = random.Random(str(size))
    p = random_pool(rng, *size)
    p.trim([rng.choice([0, n, n // 3]) for n in p.len])
    g = OnGpu(pkg, p, cap=p.n_pages if cap == "all" else cap)
    pkg.pages_compact(g.pool, g.tables, g.moves, stream=stream())
    p.compact(p.n_pages if cap == "all" else cap)
    g.same()
    if cap == "all":
        u = sum(r > 0 for r in p.refs)
        assert all(p.refs[:u]) and not any(p.refs[u:])


def test_empty_calls(pkg, dev):
    """No pages, no sequences, no table: nothing is named, nothing happens."""
    say("empty calls")
    d = i32([0])
    none = pkg.PagePool(0, 16, 0, 0)
    empty = pkg.PageTables(0, 0, 0, 0)
    moves = pkg.PageMoves(1, d.data_ptr(), d.data_ptr(), d.data_ptr())
    length, bad, count, src, dst = i32([5, 0]), i32([0]), i32([9]), i32([1, 1]), i32([1, 1])
    wide = pkg.PageTables(2, length.data_ptr(), 0, 0, bad.data_ptr())
    list2 = pkg.PageMoves(2, src.data_ptr(), dst.data_ptr(), count.data_ptr())
    s = stream()
    for tables in (empty, wide):
        pkg.pages_fork(none, tables, d.data_ptr(), stream=s) if tables is empty else None
        pkg.pages_extend(none, tables, 0, list2, stream=s)
        torch.cuda.synchronize()
        assert int(count) == 0
        count.fill_(9)
        pkg.pages_compact(none, tables, list2, stream=s)
        torch.cuda.synchronize()
        assert int(count) == 0
        pkg.pages_trim(none, tables, stream=s)
    torch.cuda.synchronize()
    assert int(bad) == 1 and length.tolist() == [0, 0]
    pkg.kv_copy(pkg.kv_caches([]), moves, stream=s)


ORDERS = ["head", "slot", "gaps"]


@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("kv,page,dim,n_pages,caches", [
    (8, 16, 128, 40, 3), (1, 1, 8, 70, 1), (3, 2, 24, 33, 65), (2, 64, 80, 9, 2), (1, 4, 256, 500, 2),
])
def test_copy(pkg, dev, order, kv, page, dim, n_pages, caches):
    say("copy", order, kv, page, dim, n_pages, caches)
    g = torch.Generator().manual_seed(dim + page)
    gap = 8 if order == "gaps" else 0
    # in memory: [page][head][slot][dim + gap] or [page][slot][head][dim]
    shape = (n_pages, page, kv, dim) if order == "slot" else (n_pages, kv, page, dim + gap)
    k = torch.randint(-9999, 9999, (caches,) + shape, generator=g, dtype=torch.int16)
    v = torch.randint(-9999, 9999, (caches,) + shape, generator=g, dtype=torch.int16)
    strides = {"head": (0, 0, 0), "slot": (kv * page * dim, dim, kv * dim),
               "gaps": (kv * page * (dim + gap), page * (dim + gap), dim + gap)}[order]
    ids = torch.randperm(n_pages, generator=g).tolist()
    n = n_pages // 3
    src, dst = ids[:n], ids[n:2 * n]
    if n > 2:
        src[1] = src[0]  # one page to two places
        dst[2] = -1      # and a pair that is none
    dk, dv = k.cuda(), v.cuda()
    arrays = pkg.kv_caches([pkg.KvPages(dk[i].data_ptr(), dv[i].data_ptr(), pkg.F16, n_pages, page,
                                        kv, dim, *strides) for i in range(caches)])
    dsrc, ddst, count = i32(src + [0] * 5), i32(dst + [0] * 5), i32([n])
    moves = pkg.PageMoves(n + 5, dsrc.data_ptr(), ddst.data_ptr(), count.data_ptr())
    pkg.kv_copy(arrays, moves, stream=stream())
    torch.cuda.synchronize()
    for t in (k, v):
        was = t.clone()
        for a, b in zip(src, dst):
            if b >= 0:
                t[:, b, ..., :dim] = was[:, a, ..., :dim]
    assert torch.equal(dk.cpu(), k) and torch.equal(dv.cpu(), v)


def test_copy_stays_within_the_list(pkg, dev):
    """A count above the list's room, or below 0, copies what the list holds, or nothing."""
    say("copy counts")
    k = torch.arange(6, dtype=torch.int16).repeat_interleave(8).view(6, 1, 1, 8).cuda()
    v = k.clone()
    src, dst, count = i32([0, 1, 2, 3]), i32([4, 5, 4, 5]), i32([1000])
    caches = pkg.kv_caches([pkg.KvPages(k.data_ptr(), v.data_ptr(), pkg.BF16, 6, 1, 1, 8)])
    moves = pkg.PageMoves(2, src.data_ptr(), dst.data_ptr(), count.data_ptr())
    pkg.kv_copy(caches, moves, stream=stream())
    torch.cuda.synchronize()
    assert k[:, 0, 0, 0].tolist() == [0, 1, 2, 3, 0, 1] == v[:, 0, 0, 7].tolist()
    k[4] = 9
    count.fill_(-4)
    pkg.kv_copy(caches, moves, stream=stream())
    torch.cuda.synchronize()
    assert k[:, 0, 0, 0].tolist() == [0, 1, 2, 3, 9, 1]


@pytest.mark.parametrize("seed", range(3))
def test_a_long_run(pkg, dev, seed):
    """Forks, growth, cuts and compactions in turn, on a stream of their own."""
    say("long run", seed)
    rng = random.Random(seed)
    p = random_pool(rng, 400, rng.choice([1, 4, 16]), 24, 20)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        g = OnGpu(pkg, p)
        for _ in range(40):
            what = rng.choice(["fork", "extend", "extend", "trim", "compact"])
            if what == "fork":
                x = [s - s % 6 + rng.randrange(6) for s in range(24)]
                d = i32(x)
                pkg.pages_fork(g.pool, g.tables, d.data_ptr(), stream=side.cuda_stream)
                p.fork(x)
            elif what == "extend":
                x = [rng.choice([0, 1, 1, 7]) for _ in range(24)]
                d = i32(x)
                pkg.pages_extend(g.pool, g.tables, d.data_ptr(), g.moves, stream=side.cuda_stream)
                p.extend(x)
            elif what == "trim":
                x = [rng.choice([0, n, n, n, n * 2 // 3]) for n in p.len]
                d = i32(x)
                pkg.pages_trim(g.pool, g.tables, d.data_ptr(), stream=side.cuda_stream)
                p.trim(x)
            else:
                pkg.pages_compact(g.pool, g.tables, g.moves, stream=side.cuda_stream)
                p.compact(g.moves.cap)
            g.same(moves=what in ("extend", "compact"))
