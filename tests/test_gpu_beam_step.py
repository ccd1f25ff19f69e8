"""A beam search's decoding steps as an engine runs them: logits from an 8-bit product,
selection, pages that follow the parents, append, attention over the pages, in one
captured graph that is replayed, against histories kept on the host.

The search: row r's hidden state is the last attention's output; its logits are the 8-bit
product of the quantized state with fixed weights.  Tokens' keys, values and queries are
rows of tables.  What attention gives is checked against 64 bits over the row's own history
within the sum of what its roundings add (paged attention, bf16 cache, fp32 output: weights
to 22 bits or more, scores and sums in fp32: 2^-15 of the largest value is far above them);
what follows takes the device's own output, so that nothing adds up."""
import math

import pytest
import torch

from test_gpu_beam import check, reference
from test_gpu_rows_i8 import codes_of, product

pytestmark = pytest.mark.gpu
F32, BF16 = 0, 30


@pytest.fixture(scope="module")
def dev(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()
    pkg.init()
    return torch.device("cuda")


class Search:
    def __init__(self, pkg, n, b, page, layers, vocab, steps, prompt, seed):
        g = torch.Generator().manual_seed(seed)
        self.pkg, self.n, self.b, self.rows, self.page, self.vocab = pkg, n, b, n * b, page, vocab
        self.heads, self.kv, self.dim, self.layers, self.prompt = 4, 2, 64, layers, prompt
        self.width, self.eos = self.heads * self.dim, 7
        table = lambda *s: torch.randn(s, generator=g)
        self.tk, self.tv = table(layers, vocab, self.kv, self.dim), table(layers, vocab, self.kv, self.dim)
        self.tq = table(layers, vocab, self.heads, self.dim)
        self.tk, self.tv, self.tq = (x.bfloat16().cuda() for x in (self.tk, self.tv, self.tq))
        w = table(vocab, self.width) * 0.7
        self.cw, self.sw = (x.cuda() for x in codes_of(w))
        cols = -(-(prompt + steps) // page)
        self.n_pages = n * cols + self.rows * (cols + 2)
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
        self.refs, self.used = i32(self.n_pages), i32(-(-self.n_pages // 32))
        self.lens, self.table, self.bad = i32(self.rows), i32(self.rows, cols), i32(1)
        self.src, self.dst, self.count = i32(self.rows), i32(self.rows), i32(1)
        self.parent, self.token, self.done = i32(self.rows), i32(self.rows), i32(self.rows)
        self.score = torch.full((self.rows,), -math.inf, device="cuda")
        self.score[::b] = 0.0  # one beam of each prompt at first
        shape = (layers, self.n_pages, self.kv, page, self.dim)
        self.k, self.v = (torch.zeros(shape, dtype=torch.bfloat16, device="cuda") for _ in "kv")
        self.pool = pkg.PagePool(self.n_pages, page, self.refs.data_ptr(), self.used.data_ptr())
        self.tables = pkg.PageTables(self.rows, self.lens.data_ptr(), self.table.data_ptr(), cols,
                                     self.bad.data_ptr())
        self.moves = pkg.PageMoves(self.rows, self.src.data_ptr(), self.dst.data_ptr(),
                                   self.count.data_ptr())
        self.caches = [pkg.KvPages(self.k[i].data_ptr(), self.v[i].data_ptr(), pkg.BF16, self.n_pages,
                                   page, self.kv, self.dim) for i in range(layers)]
        self.all = pkg.kv_caches(self.caches)
        self.first = torch.arange(self.rows + 1, dtype=torch.int32, device="cuda")
        self.hidden = torch.randn((self.rows, self.width), generator=g).cuda()
        self.hidden.copy_(self.hidden[::b].repeat_interleave(b, dim=0))
        self.codes = torch.zeros((self.rows, self.width), dtype=torch.int8, device="cuda")
        self.scale = torch.zeros(self.rows, device="cuda")
        self.logits = torch.zeros((self.rows, vocab), device="cuda")
        self.o = torch.zeros((layers, self.rows, self.width), device="cuda")
        self.q = torch.zeros((self.rows, self.width), dtype=torch.bfloat16, device="cuda")
        self.spec = pkg.BeamSpec(n, b, vocab, b, self.eos)
        self.batch = pkg.SeqBatch(self.rows, self.rows, 1, prompt + steps, self.first.data_ptr(),
                                  self.lens.data_ptr(), self.table.data_ptr(), cols,
                                  self.bad.data_ptr())
        self.history = [[] for _ in range(self.rows)]
        # the prompt: one sequence of each group holds it, the beams are forks
        tokens = torch.randint(0, vocab, (n, prompt), generator=g)
        s = torch.cuda.current_stream().cuda_stream
        new = torch.zeros(self.rows, dtype=torch.int32, device="cuda")
        new[::b] = prompt
        pkg.pages_extend(self.pool, self.tables, new.data_ptr(), self.moves, stream=s)
        first = torch.cumsum(torch.cat((torch.zeros(1, dtype=torch.int32), new.cpu())), 0).int().cuda()
        batch = pkg.SeqBatch(self.rows, n * prompt, prompt, prompt, first.data_ptr(),
                             self.lens.data_ptr(), self.table.data_ptr(), cols, self.bad.data_ptr())
        flat = tokens.flatten().cuda()
        for i in range(layers):
            k, v = self.tk[i][flat].contiguous(), self.tv[i][flat].contiguous()
            pkg.kv_append(self.caches[i], batch, None, 0, k.data_ptr(), v.data_ptr(), BF16, 0, 0,
                          stream=s)
        group = (torch.arange(self.rows, dtype=torch.int32) // b * b).cuda()
        pkg.pages_fork(self.pool, self.tables, group.data_ptr(), stream=s)
        torch.cuda.synchronize()
        self.history = [tokens[r // b].tolist() for r in range(self.rows)]

    def need(self):
        L = self.pkg.gpu_lib()
        return max(L.swamp_beam_select_workspace(self.spec),
                   L.swamp_gemm_rows_i8_workspace(self.rows, self.vocab, self.width),
                   L.swamp_attn_paged_workspace(self.caches[0], self.batch, self.heads, 0))

    def step(self, s):
        pkg = self.pkg
        pkg.quantize_rows(self.hidden.data_ptr(), F32, self.codes.data_ptr(), self.scale.data_ptr(),
                          self.rows, self.width, stream=s)
        pkg.gemm_rows_i8(self.codes.data_ptr(), self.scale.data_ptr(), self.cw.data_ptr(),
                         self.sw.data_ptr(), self.logits.data_ptr(), F32, self.rows, self.vocab,
                         self.width, stream=s)
        pkg.beam_select(self.spec, self.logits.data_ptr(), F32, self.score.data_ptr(),
                        self.parent.data_ptr(), self.token.data_ptr(), self.score.data_ptr(),
                        d_done=self.done.data_ptr(), d_out_done=self.done.data_ptr(), stream=s)
        pkg.pages_fork(self.pool, self.tables, self.parent.data_ptr(), stream=s)
        pkg.pages_extend(self.pool, self.tables, 0, self.moves, stream=s)
        pkg.kv_copy(self.all, self.moves, stream=s)
        at = self.token.clamp_min(0).long()
        for i in range(self.layers):
            k, v, q = self.tk[i][at].contiguous(), self.tv[i][at].contiguous(), self.tq[i][at]
            self.q.copy_(q.reshape(self.rows, self.width))
            pkg.kv_append(self.caches[i], self.batch, None, 0, k.data_ptr(), v.data_ptr(), BF16, 0, 0,
                          stream=s)
            pkg.attn_paged(self.caches[i], self.batch, self.q.data_ptr(), self.heads,
                           1 / math.sqrt(self.dim), self.o[i].data_ptr(), F32, stream=s)
        self.hidden.copy_(self.o.sum(dim=0) * 4.0)

    def verify(self, before):
        """before: hidden, score, done as they were."""
        hidden, score, done = before
        codes, scale = codes_of(hidden)
        assert torch.equal(self.codes.cpu(), codes) and torch.equal(self.scale.cpu(), scale)
        logits = product(codes, self.cw.cpu(), scale, self.sw.cpu(), F32)
        assert torch.equal(self.logits.cpu(), logits)
        want = reference(logits, score, done, self.n, self.b, self.b, self.eos)
        check((self.parent.tolist(), self.token.tolist(), self.score.tolist(), self.done.tolist()),
              want)
        self.history = [self.history[w[0]] + [w[1]] for w in want]
        # every page's count is the tables', and the free ones' is 0
        lens, table = self.lens.tolist(), self.table.cpu()
        assert lens == [len(h) for h in self.history] and int(self.bad) == 0
        held = torch.cat([table[r, :-(-lens[r] // self.page)] for r in range(self.rows)])
        assert torch.equal(torch.bincount(held, minlength=self.n_pages).int(), self.refs.cpu())
        # what no two rows write alike: a last page that is not full has one holder
        for r in range(self.rows):
            if lens[r] % self.page:
                assert int(self.refs[table[r, lens[r] // self.page]]) == 1
        g = self.heads // self.kv
        for i in range(self.layers):
            tk, tv, tq = (t[i].cpu().double() for t in (self.tk, self.tv, self.tq))
            for r in range(self.rows):
                h = torch.tensor(self.history[r])
                q = tq[h[-1]]
                k, v = tk[h].repeat_interleave(g, 1), tv[h].repeat_interleave(g, 1)
                p = torch.softmax(torch.einsum("hd,thd->ht", q, k) / math.sqrt(self.dim), dim=1)
                o = torch.einsum("ht,thd->hd", p, v).flatten()
                err = (self.o[i, r].cpu().double() - o).abs().max()
                assert err <= 2.0 ** -15 * v.abs().max()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("n,b,page,prompt", [(3, 4, 8, 21), (1, 1, 4, 1), (2, 6, 16, 32)])
def test_search(pkg, dev, n, b, page, prompt, captured):
    print("[gpu case] search", n, b, page, prompt, captured, flush=True)
    steps = 14
    x = Search(pkg, n, b, page, 2, 300, steps + 1, prompt, seed=n * 10 + b)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    pkg.workspace_reserve(side.cuda_stream, x.need())
    if captured:
        with torch.cuda.graph(graph, stream=side):
            x.step(side.cuda_stream)
    for _ in range(steps):
        before = (x.hidden.cpu(), x.score.cpu(), x.done.cpu())
        if captured:
            graph.replay()
        else:
            with torch.cuda.stream(side):
                x.step(side.cuda_stream)
        torch.cuda.synchronize()
        x.verify(before)


def test_search_then_compact(pkg, dev):
    """Half the prompts end, the others' pages move down, and the search goes on."""
    print("[gpu case] search, compact", flush=True)
    x = Search(pkg, 4, 3, 8, 2, 200, 20, 19, seed=5)
    s = torch.cuda.current_stream().cuda_stream
    for _ in range(5):
        before = (x.hidden.cpu(), x.score.cpu(), x.done.cpu())
        x.step(s)
        torch.cuda.synchronize()
        x.verify(before)
    cap = torch.zeros((3, x.n_pages), dtype=torch.int32, device="cuda")
    moves = pkg.PageMoves(x.n_pages, cap[0].data_ptr(), cap[1].data_ptr(), cap[2].data_ptr())
    keep = torch.full((x.rows,), 1 << 30, dtype=torch.int32, device="cuda")
    keep[:6] = 0
    x.score[:6] = -math.inf
    pkg.pages_trim(x.pool, x.tables, keep.data_ptr(), stream=s)
    pkg.pages_compact(x.pool, x.tables, moves, stream=s)
    pkg.kv_copy(x.all, moves, stream=s)
    torch.cuda.synchronize()
    u = int((x.refs > 0).sum())
    assert int(cap[2, 0]) > 0 and bool((x.refs[:u] > 0).all())
    for r in range(6):
        x.history[r] = []
    for _ in range(4):
        score, done, hidden = x.score.cpu(), x.done.cpu(), x.hidden.cpu()
        x.step(s)
        torch.cuda.synchronize()
        # the ended prompts' rows have no continuation, their tables are empty but for the
        # token that every step appends
        assert x.parent[:6].eq(-1).all() and x.token[:6].eq(-1).all()
        assert x.lens[:6].eq(1).all()
        codes, scale = codes_of(hidden)
        logits = product(codes, x.cw.cpu(), scale, x.sw.cpu(), F32)
        want = reference(logits, score, done, x.n, x.b, x.b, x.eos)
        check((x.parent.tolist(), x.token.tolist(), x.score.tolist(), x.done.tolist()), want)
        x.history = [x.history[w[0]] + [w[1]] if w[0] >= 0 else [0] for w in want]
        assert x.lens.tolist() == [len(h) for h in x.history]
        for r in range(6, x.rows):
            h = torch.tensor(x.history[r])
            tk, tv, tq = (t[1].cpu().double() for t in (x.tk, x.tv, x.tq))
            p = torch.softmax(torch.einsum("hd,thd->ht", tq[h[-1]], tk[h].repeat_interleave(2, 1))
                              / 8.0, dim=1)
            o = torch.einsum("ht,thd->hd", p, tv[h].repeat_interleave(2, 1)).flatten()
            assert (x.o[1, r].cpu().double() - o).abs().max() <= 2.0 ** -15 * tv[h].abs().max()
