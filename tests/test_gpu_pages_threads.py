"""Forks from two host threads at once, of so many sequences that each launch asks for more
LDS than a kernel has without being allowed it, and of different numbers."""
import random
import threading

import pytest
import torch

from pages_reference import OnGpu, random_pool
from test_gpu_pages import i32, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()
    pkg.init()
    return torch.device("cuda")


def test_forks_of_two_threads(pkg, dev):
    say("forks of two threads")
    work, errors = [], []
    for n, seed in ((2048, 1), (900, 2)):
        rng = random.Random(seed)
        p = random_pool(rng, 6000, 2, n, 3)
        parents = [[rng.randrange(n) for _ in range(n)] for _ in range(40)]
        work.append((p, OnGpu(pkg, p), parents, [i32(x) for x in parents], torch.cuda.Stream()))
    torch.cuda.synchronize()
    start = threading.Barrier(2)

    def run(g, lists, stream):
        try:
            start.wait(30)
            for d in lists:
                pkg.pages_fork(g.pool, g.tables, d.data_ptr(), stream=stream.cuda_stream)
        except Exception as e:  # noqa: BLE001 (told by the main thread)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(g, lists, s)) for _, g, _, lists, s in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    assert not errors and not any(t.is_alive() for t in threads)
    for p, g, parents, _, _ in work:
        for x in parents:
            p.fork(x)
        g.same(moves=False)
