"""Pools of pages and their page tables, one sequence and one page after the other on
the host: what swamp_pages_* and swamp_kv_copy are compared with."""
import torch


class Pool:
    """A cache's pages (k, v: one fp32 tag a page, so that copies show), their counts, and
    the tables of n sequences of up to `width` pages."""

    def __init__(self, n_pages, page, n, width):
        self.page, self.n, self.width, self.n_pages = page, n, width, n_pages
        self.refs = [0] * n_pages
        self.table = [[-7] * width for _ in range(n)]
        self.len = [0] * n
        self.moves = []
        self.bad = 0

    def cols(self, tokens):
        return min(-(-max(tokens, 0) // self.page), self.width)

    def held(self, s):
        return self.table[s][:self.cols(self.len[s])]

    def ok(self, e):
        return 0 <= e < self.n_pages

    def lowest(self):
        for e in range(self.n_pages):
            if self.refs[e] == 0:
                self.refs[e] = 1
                return e
        self.bad = 1
        return -1

    def fork(self, parent):
        rows = [self.held(p) if 0 <= p < self.n else [] for p in parent]
        lens = [self.len[p] if 0 <= p < self.n else 0 for p in parent]
        for s in range(self.n):
            for e in self.held(s):
                if self.ok(e):
                    self.refs[e] -= 1
        for s in range(self.n):
            self.table[s][:len(rows[s])] = rows[s]
            for e in rows[s]:
                if self.ok(e):
                    self.refs[e] += 1
        self.len = lens

    def extend(self, new):
        """All pages to copy are taken before any page is handed out."""
        self.moves = []
        parted = [False] * self.n
        left = list(self.refs)
        for s in range(self.n):
            at = self.len[s] // self.page
            if new[s] > 0 and self.len[s] % self.page and at < self.width:
                e = self.table[s][at]
                if not self.ok(e):
                    self.bad = 1
                elif left[e] > 1:
                    left[e] -= 1
                    parted[s] = True
        for s in range(self.n):
            if parted[s]:
                self.refs[self.table[s][self.len[s] // self.page]] -= 1
        for s in range(self.n):
            k = max(new[s], 0)
            at = self.len[s] // self.page
            if parted[s]:
                e = self.lowest()
                if e >= 0:
                    self.moves.append((self.table[s][at], e))
                self.table[s][at] = e
            last = -(-(self.len[s] + k) // self.page)
            if k and last > self.width:
                self.bad = 1
            for c in range(self.cols(self.len[s]), min(last, self.width)):
                self.table[s][c] = self.lowest()
            self.len[s] += k

    def trim(self, keep):
        for s in range(self.n):
            k = min(max(keep[s], 0), self.len[s])
            for e in self.held(s)[self.cols(k):]:
                if self.ok(e):
                    self.refs[e] -= 1
            self.len[s] = k

    def compact(self, cap):
        used = [e for e in range(self.n_pages) if self.refs[e] > 0]
        u = len(used)
        pairs = list(zip([e for e in used if e >= u], [e for e in range(u) if self.refs[e] == 0]))
        self.moves = pairs[:cap]
        to = dict(self.moves)
        for a, b in self.moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        for s in range(self.n):
            k = self.cols(self.len[s])
            self.table[s][:k] = [to.get(e, e) for e in self.table[s][:k]]

    def words(self):
        out = [0] * (-(-self.n_pages // 32))
        for e, r in enumerate(self.refs):
            out[e // 32] |= (r > 0) << (e % 32)
        return [w - (w >> 31 << 32) for w in out]

    def check(self):
        """Counts are the tables' (what every call leaves)."""
        seen = [0] * self.n_pages
        for s in range(self.n):
            for e in self.held(s):
                if self.ok(e):
                    seen[e] += 1
        assert seen == self.refs


class OnGpu:
    """A Pool's state on the device, and the structures of the package."""

    def __init__(self, pkg, pool, cap=None):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        self.pkg, self.ref = pkg, pool
        self.refs, self.used, self.len = i32(pool.refs), i32(pool.words()), i32(pool.len)
        self.table = i32(pool.table).view(pool.n, pool.width)
        cap = max(pool.n_pages, pool.n) if cap is None else cap
        self.src, self.dst = i32([-3] * max(cap, 1)), i32([-3] * max(cap, 1))
        self.count, self.bad = i32([-3]), i32([0])
        self.pool = pkg.PagePool(pool.n_pages, pool.page, self.refs.data_ptr(), self.used.data_ptr())
        self.tables = pkg.PageTables(pool.n, self.len.data_ptr(), self.table.data_ptr(), pool.width,
                                     self.bad.data_ptr())
        self.moves = pkg.PageMoves(cap, self.src.data_ptr(), self.dst.data_ptr(),
                                   self.count.data_ptr())

    def same(self, moves=True, whole=True):
        torch.cuda.synchronize()
        p = self.ref
        assert self.len.tolist() == p.len
        assert self.table.tolist() == p.table
        assert self.refs.tolist() == p.refs
        assert self.used.tolist() == p.words()
        assert int(self.bad) == p.bad
        if moves:
            n = len(p.moves)
            assert int(self.count) == n
            assert list(zip(self.src[:n].tolist(), self.dst[:n].tolist())) == p.moves
        if whole:
            p.check()


def random_pool(rng, n_pages, page, n, width, share=0.5):
    """Sequences with pages of their own and shared prefixes, ids in any order."""
    p = Pool(n_pages, page, n, width)
    ids = list(range(n_pages))
    rng.shuffle(ids)
    for s in range(n):
        if s and rng.random() < share:
            o = rng.randrange(s)
            p.len[s] = rng.choice([p.len[o], rng.randint(0, p.len[o])])
            p.table[s][:p.cols(p.len[s])] = p.table[o][:p.cols(p.len[s])]
        else:
            p.len[s] = rng.randint(0, width * page)
            p.len[s] = min(p.len[s], len(ids) * page)
            for c in range(p.cols(p.len[s])):
                p.table[s][c] = ids.pop()
        for e in p.held(s):
            p.refs[e] += 1
    return p
