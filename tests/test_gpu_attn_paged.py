"""swamp_attn_paged on the GPU against 64 bits on the CPU (tests/
paged_reference.py has the bound and what it counts).  Slots that hold no key
of a sequence are NaN in every cache here."""
import math

import pytest
import torch

from paged_reference import BF16, F16, F32, NAME, TORCH, Paged, attention

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


def queries(c, heads, sigma=1.5):
    return (torch.randn((c.n_tok, heads, c.dim), generator=c.g) * sigma).to(TORCH[c.code])


def run(pkg, c, q, scale, out_code, window=0, cache_batch=None, **more):
    cache, batch = cache_batch or c.on_gpu(pkg, **more)
    dq = q.cuda()
    out = torch.full(q.shape, 77.0, dtype=TORCH[out_code], device="cuda")
    pkg.attn_paged(cache, batch, dq.data_ptr(), q.shape[1], scale, out.data_ptr(), out_code,
                   window=window, stream=stream())
    torch.cuda.synchronize()
    return out.cpu()


def check(pkg, c, heads, out_code, window=0, sigma=1.5, **more):
    q = queries(c, heads, sigma)
    scale = 1 / math.sqrt(c.dim)
    got = run(pkg, c, q, scale, out_code, window, **more)
    want, bound = attention(c, q, scale, window, out_code == F32, out_code)
    err = (got.double() - want).abs()
    worst = (err / bound).max().item() if err.numel() else 0.0
    print(f"[parity] attn: worst error {worst:.3f} of its bound", flush=True)
    assert torch.all(err <= bound), worst
    assert int(c.dev["bad"]) == 0
    return got


# one token each: the form for decoding
@pytest.mark.parametrize("code,out_code", [(BF16, F32), (F16, F32), (F16, F16), (BF16, BF16),
                                           (F16, BF16), (BF16, F16)])
@pytest.mark.parametrize("lens,heads,kv,dim,page", [
    ([1], 1, 1, 8, 1), ([2, 1, 3], 4, 4, 64, 16), ([700], 32, 8, 128, 32),
    ([33, 31, 32, 1, 64], 8, 1, 128, 8), ([513, 100], 14, 2, 80, 64), ([257, 7], 6, 3, 256, 2),
    ([40, 1025], 64, 2, 96, 256)])
def test_decode(pkg, dev, lens, heads, kv, dim, page, code, out_code):
    say("decode", lens, heads, kv, dim, page, NAME[code], NAME[out_code])
    check(pkg, Paged([1] * len(lens), lens, kv, dim, page, code), heads, out_code)


@pytest.mark.parametrize("code,out_code", [(BF16, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("order", ["head", "slot"])
@pytest.mark.parametrize("news,lens,heads,kv,dim,page,window", [
    ([5, 5], [300, 44], 8, 2, 128, 32, 0),
    ([2, 0, 7, 1], [2, 50, 600, 40], 5, 5, 64, 16, 0),
    ([16], [16], 16, 4, 128, 8, 0),
    ([70, 1, 33], [70, 500, 97], 8, 2, 64, 16, 0),
    ([130], [1000], 7, 1, 128, 64, 0),
    ([257], [257], 4, 2, 80, 32, 0),
    ([100, 1], [400, 333], 8, 2, 128, 16, 64),
    ([40], [200], 6, 2, 256, 4, 17),
    ([129, 3], [300, 3], 4, 4, 96, 128, 1),
])
def test_chunks(pkg, dev, news, lens, heads, kv, dim, page, window, order, code, out_code):
    say("chunk", news, lens, heads, kv, dim, page, window, order, NAME[code], NAME[out_code])
    check(pkg, Paged(news, lens, kv, dim, page, code, order=order), heads, out_code, window)


@pytest.mark.parametrize("code", [BF16, F16])
@pytest.mark.parametrize("news,lens,heads,kv", [([1], [20000], 8, 2), ([1, 1], [9001, 5], 4, 1),
                                                ([3], [6000], 8, 1), ([90], [5000], 4, 2)])
def test_long(pkg, dev, news, lens, heads, kv, code):
    """Caches long enough to be split over workgroups; max_len is only a hint."""
    say("long", news, lens, heads, kv, NAME[code])
    c = Paged(news, lens, kv, 64, 64, code)
    a = check(pkg, c, heads, F32)
    c.g.manual_seed(5)
    q = queries(c, heads)
    whole = run(pkg, c, q, 0.125, F32)
    assert torch.equal(whole, run(pkg, c, q, 0.125, F32))  # the same bits again
    for hint in (0, 1, 100000):
        got = run(pkg, c, q, 0.125, F32, max_len=hint)
        want, bound = attention(c, q, 0.125)
        assert torch.all((got.double() - want).abs() <= bound), hint
    assert a.isfinite().all()


@pytest.mark.parametrize("new", [1, 40])
def test_many_sequences(pkg, dev, new):
    say("many sequences", new)
    lens = [new - 1 + 1 + (i * 37) % 211 for i in range(90)]
    news = [0 if i % 11 == 3 else new if i % 5 else 1 for i in range(90)]
    check(pkg, Paged(news, lens, 2, 64, 16, F16), 8, F16)


def test_peaked_and_large_scores(pkg, dev):
    """Scores in the hundreds: the weights of all but a few keys underflow."""
    say("peaked")
    for news, lens in (([1], [900]), ([64], [200])):
        check(pkg, Paged(news, lens, 2, 128, 16, BF16, sigma=8.0), 8, F32, sigma=8.0)


@pytest.mark.parametrize("news,lens,window", [([4], [2], 0), ([40, 3], [7, 0], 0), ([1, 1], [0, 5], 0),
                                              ([200], [150], 9), ([33, 1], [1, -4], 0)])
def test_rows_without_keys(pkg, dev, news, lens, window):
    """More new tokens than the cache holds: rows before position 0 are 0."""
    say("empty rows", news, lens)
    c = Paged(news, lens, 2, 64, 8, F16)
    got = check(pkg, c, 4, F32, window)
    at = 0
    for m, n in zip(news, lens):
        empty = min(m, m - max(n, 0))
        assert torch.all(got[at:at + max(empty, 0)] == 0)
        at += m


def test_padding_rows_and_stale_lengths(pkg, dev):
    """Rows of no sequence keep what they hold; sequence arrays that run out of
    the batch are cut to it."""
    say("padding rows")
    c = Paged([3, 2], [10, 6], 1, 64, 8, F16)
    cache, batch = c.on_gpu(pkg, n_tok=8)
    q = torch.randn((8, 2, 64), generator=c.g).half()
    got = run(pkg, c, q, 0.125, F32, cache_batch=(cache, batch))
    want, bound = attention(c, q[:5], 0.125)
    assert torch.all((got[:5].double() - want).abs() <= bound) and torch.all(got[5:] == 77.0)


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("news,lens,window", [([6], [20], 0), ([70], [100], 0), ([150], [150], 0),
                                              ([6], [100], 10), ([90], [300], 40)])
def test_what_a_row_does_not_see_does_not_reach_it(pkg, dev, news, lens, window, poison):
    """A later token of the same chunk, and one before the window, with NaN or
    infinity in k and v: rows that do not see it are as without it."""
    say("masked poison", news, lens, window, poison)
    c = Paged(news, lens, 2, 64, 16, BF16)
    n, m = lens[0], news[0]
    at = n - m // 3  # a new token's position
    spots = [at] + ([n - m - window - 1, n - m - window + 2] if window else [])
    clean_q = queries(c, 4)
    want, bound = attention(c, clean_q, 0.125, window)
    sees = torch.zeros(m, dtype=torch.bool)
    for spot in spots:
        bad = torch.full((2, 64), poison)
        bad[:, 1::2] = 1.0
        c.put(0, spot, k=bad.bfloat16() if spot == at else None, v=bad.bfloat16())
        pos = torch.arange(n - m, n)
        sees |= (pos >= spot) & ((pos - spot < window) if window else (pos >= 0))
    got = run(pkg, c, clean_q, 0.125, F32, window)
    assert 0 < int(sees.sum()) < m
    assert torch.all((got[~sees].double() - want[~sees]).abs() <= bound[~sees])
    assert not got[sees].isfinite().all(-1).any()  # those that see it, show it


def test_infinite_value_reaches_the_rows_that_see_it(pkg, dev):
    """v = +inf in one dim gives +inf there and leaves the other dims alone."""
    say("visible infinity")
    for m, n in ((1, 40), (30, 70)):
        c = Paged([m], [n], 1, 64, 16, F16)
        spot = n - m // 2 - 1
        k, v = c.keys(0)
        v = v[spot].clone()
        v[:, 5] = math.inf
        q = queries(c, 2)
        want, bound = attention(c, q, 0.125)
        c.put(0, spot, v=v)
        got = run(pkg, c, q, 0.125, F32)
        sees = torch.arange(n - m, n) >= spot
        assert torch.all(got[sees][..., 5] == math.inf)
        got[..., 5], want[..., 5] = 0, 0
        assert torch.all((got.double() - want).abs() <= bound)


@pytest.mark.parametrize("news,lens", [([1, 1, 1], [100, 90, 80]), ([60, 2, 9], [100, 90, 80])])
def test_positions_without_a_page(pkg, dev, news, lens):
    """A page id outside the cache, or a length past the table, gives NaN in its
    sequence's rows that have to read it and sets the flag; the others are right."""
    say("bad pages", news, lens)
    for what in ("id", "negative", "table"):
        c = Paged(news, lens, 2, 64, 16, F16)
        q = queries(c, 4)
        want, bound = attention(c, q, 0.125)
        if what == "table":
            c.len[0] = 16 * c.table.shape[1] + 1 + news[0]
        else:
            c.table[0, 0] = c.n_pages if what == "id" else -3
        got = run(pkg, c, q, 0.125, F32)
        m = news[0]
        assert int(c.dev["bad"]) == 1 and torch.all(got[:m].isnan()), what
        assert torch.all((got[m:].double() - want[m:]).abs() <= bound[m:]), what
        # without a flag to set
        c.on_gpu(pkg, bad=False)
        cache, batch = c.on_gpu(pkg, bad=False)
        assert torch.all(run(pkg, c, q, 0.125, F32, cache_batch=(cache, batch))[:m].isnan())


def test_pages_outside_the_window_are_not_read(pkg, dev):
    """A sliding window's user gives old pages back: their entries may name
    nothing."""
    say("freed pages")
    for m in (1, 4, 200):
        c = Paged([m], [900], 2, 64, 16, BF16)
        q = queries(c, 8)
        want, bound = attention(c, q, 0.125, 100)
        c.table[0, :(900 - m - 100 + 1) // 16] = -1
        got = run(pkg, c, q, 0.125, F32, 100)
        assert torch.all((got.double() - want).abs() <= bound) and int(c.dev["bad"]) == 0


def test_strided_rows(pkg, dev):
    """q and out as parts of wider rows."""
    say("strided rows")
    for m, n in ((1, 50), (40, 90)):
        c = Paged([m], [n], 2, 64, 16, BF16)
        q = queries(c, 4)
        cache, batch = c.on_gpu(pkg)
        wide_q = torch.full((m, 4 * 64 + 24), 9.0, dtype=torch.bfloat16)
        wide_q[:, 8:8 + 256] = q.reshape(m, -1)
        dq = wide_q.cuda()
        out = torch.full((m, 4 * 64 + 40), 9.0, device="cuda")
        pkg.attn_paged(cache, batch, dq.data_ptr() + 16, 4, 0.125, out.data_ptr() + 64, F32,
                       q_stride=280, out_stride=296, stream=stream())
        torch.cuda.synchronize()
        want, bound = attention(c, q, 0.125)
        got = out.cpu()
        assert torch.all((got[:, 16:272].reshape(m, 4, 64).double() - want).abs() <= bound)
        assert torch.all(got[:, :16] == 9.0) and torch.all(got[:, 272:] == 9.0)


def test_offsets_past_32_bits(pkg, dev):
    """Pages 2^31 elements apart."""
    say("far pages")
    page, kv, dim, far = 16, 2, 64, 2 ** 31
    c = Paged([3], [3 * page], kv, dim, page, F16, extra_pages=0)
    q = queries(c, 4)
    want, bound = attention(c, q, 0.125)
    block = kv * page * dim
    buf = torch.empty(2 * far + 2 * block, dtype=torch.float16, device="cuda")
    for i in range(3):
        buf[i * far:i * far + block] = c.k[i].reshape(-1).cuda()
        buf[i * far + block:i * far + 2 * block] = c.v[i].reshape(-1).cuda()
    cache, batch = c.on_gpu(pkg)
    cache = pkg.KvPages(buf.data_ptr(), buf.data_ptr() + 2 * block, F16, 3, page, kv, dim, far,
                        page * dim, dim)
    got = run(pkg, c, q, 0.125, F32, cache_batch=(cache, batch))
    assert torch.all((got.double() - want).abs() <= bound)
    # and written: the newest token's slot
    x = torch.randn((3, kv, dim), generator=c.g).cuda()
    pkg.kv_append(cache, batch, None, 0, x.data_ptr(), x.data_ptr(), F32, 0, 0, stream=stream())
    torch.cuda.synchronize()
    at = int(c.table[0, 2]) * far
    k = buf[at:at + block].view(kv, page, dim)
    assert torch.equal(k[:, page - 3:], x.half().transpose(0, 1))


def test_other_stream(pkg, dev):
    """Work on a stream of its own, behind a producer there."""
    say("other stream")
    c = Paged([1, 9], [3000, 50], 2, 64, 16, BF16)
    q = queries(c, 8)
    cache, batch = c.on_gpu(pkg)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        dq = q.pin_memory().cuda(non_blocking=True)
        out = torch.empty(q.shape, device="cuda")
        pkg.attn_paged(cache, batch, dq.data_ptr(), 8, 0.125, out.data_ptr(), F32,
                       stream=st.cuda_stream)
        got = out.cpu()
    want, bound = attention(c, q, 0.125)
    assert torch.all((got.double() - want).abs() <= bound)


@pytest.mark.parametrize("reserve", [True, False])
def test_graph_replays_with_other_lengths(pkg, dev, reserve):
    """append and attention captured once, replayed as the sequences grow, with
    eager work between; with scratch reserved and without any."""
    say("graph", "reserved" if reserve else "no scratch")
    heads, kv, dim, page, n = 8, 2, 64, 16, 3
    lens = [2000, 31, 700]
    c = Paged([1] * n, [x + 8 for x in lens], kv, dim, page, F16)
    c.len = torch.tensor(lens, dtype=torch.int32)
    cache, batch = c.on_gpu(pkg, max_len=2100)
    freqs = torch.from_numpy(pkg.rope_freqs(dim)).cuda()
    rope = pkg.Rope(freqs.data_ptr(), dim, pkg.ROPE_HALVES)
    x = torch.zeros((n, heads + 2 * kv, dim), device="cuda")
    q = torch.empty((n, heads, dim), dtype=torch.float16, device="cuda")
    out = torch.empty((n, heads, dim), device="cuda")

    def step(s, to_q, to_out):
        w = (heads + 2 * kv) * dim
        pkg.kv_append(cache, batch, rope, x.data_ptr(), x.data_ptr() + 4 * heads * dim,
                      x.data_ptr() + 4 * (heads + kv) * dim, F32, to_q.data_ptr(), heads, q_stride=w,
                      k_stride=w, v_stride=w, stream=s)
        pkg.attn_paged(cache, batch, to_q.data_ptr(), heads, 0.125, to_out.data_ptr(), F32, stream=s)

    st = torch.cuda.Stream()
    if reserve:
        need = pkg.gpu_lib().swamp_attn_paged_workspace(cache, batch, heads, 0)
        pkg.workspace_reserve(st.cuda_stream, max(need, 256))
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step(torch.cuda.current_stream().cuda_stream, q, out)
    q2, out2 = torch.empty_like(q), torch.empty_like(out)
    g = torch.Generator(device="cuda").manual_seed(4)
    for i in range(6):
        x.normal_(generator=g)
        c.dev["len"] += 1
        graph.replay()
        torch.cuda.synchronize()
        step(stream(), q2, out2)
        torch.cuda.synchronize()
        assert torch.equal(q, q2)
        assert torch.all((out - out2).abs() <= 1e-5 * (1 + out2.abs())), i
        assert out.isfinite().all()
    assert int(c.dev["bad"]) == 0
