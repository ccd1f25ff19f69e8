"""swamp_pages_compact with lists of thousands of moves and tables of more than 1000 columns,
against one page after the other on the host."""
import random

import pytest
import torch

from pages_reference import OnGpu, Pool
from test_gpu_pages import say, stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()
    pkg.init()
    return torch.device("cuda")


def long_pool(n_pages, n, width, short, seed):
    """Pages in any order; every third sequence shares its neighbour's first half."""
    rng = random.Random(seed)
    p = Pool(n_pages, 1, n, width)
    ids = list(range(n_pages))
    rng.shuffle(ids)
    for s in range(n):
        p.len[s] = rng.randint(short, width)
        shared = p.len[s - 1] // 2 if s % 3 == 2 else 0
        shared = min(shared, p.len[s])
        p.table[s][:shared] = p.table[s - 1][:shared]
        for c in range(shared, p.len[s]):
            p.table[s][c] = ids.pop()
        for e in p.held(s):
            p.refs[e] += 1
    return p


def copy_of(p):
    q = Pool(p.n_pages, p.page, p.n, p.width)
    q.refs, q.len, q.table = list(p.refs), list(p.len), [list(t) for t in p.table]
    return q


# pages, sequences, columns, shortest sequence: lists of about 2050, 5300, 15000 and 40000
@pytest.mark.parametrize("size", [(8600, 4, 1500, 900), (22000, 12, 1300, 1000),
                                  (60000, 70, 700, 257), (165000, 90, 1217, 1100)])
def test_long_lists(pkg, dev, size):
    full = long_pool(*size, seed=size[0])
    u = sum(r > 0 for r in full.refs)
    most = sum(r > 0 for r in full.refs[u:])
    assert most > 2000
    # all moves; a list that ends within a step of the probes, with one, at the first long one
    for cap in (full.n_pages, most - 1, most // 2 * 2 - 7, 4096, 2049, 2048):
        p = copy_of(full)
        say("long lists", size, most, cap)
        g = OnGpu(pkg, p, cap=cap)
        pkg.pages_compact(g.pool, g.tables, g.moves, stream=stream())
        p.compact(cap)
        assert len(p.moves) == min(cap, most)
        g.same()


def test_long_run_of_compactions(pkg, dev):
    """What one compaction leaves is the next one's start: cut, compacted 3000 at a time."""
    p = long_pool(40000, 30, 1100, 1000, 5)
    rng = random.Random(1)
    g = OnGpu(pkg, p, cap=3000)
    for turn in range(6):
        say("compactions in turn", turn)
        keep = [rng.choice([n, n, n - 3, n * 3 // 4]) for n in p.len]
        d = torch.tensor(keep, dtype=torch.int32, device=dev)
        pkg.pages_trim(g.pool, g.tables, d.data_ptr(), stream=stream())
        p.trim(keep)
        pkg.pages_compact(g.pool, g.tables, g.moves, stream=stream())
        p.compact(3000)
        g.same()
