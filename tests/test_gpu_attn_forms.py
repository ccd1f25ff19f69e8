"""swamp_attn_paged on the GPU where its forms meet: head sizes without a kernel
of their own, pages below a group of 16 keys, strides that need 64 bits, pieces
of a cache and their join, maxima that grow all the way, values that are not
finite in one piece of several.  Oracle and bound: tests/paged_reference.py."""
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


def check(pkg, c, heads, out_code, window=0, scale=None, q=None, **more):
    q = queries(c, heads) if q is None else q
    scale = 1 / math.sqrt(c.dim) if scale is None else scale
    got = run(pkg, c, q, scale, out_code, window, **more)
    want, bound = attention(c, q, scale, window, out_code == F32, out_code)
    err = (got.double() - want).abs()
    worst = (err / bound).max().item()
    print(f"[parity] attn: worst error {worst:.3f} of its bound", flush=True)
    assert torch.all(err <= bound), worst
    assert int(c.dev["bad"]) == 0
    return got


# ------------------------------------------------------- head sizes and pages

@pytest.mark.parametrize("dim", [8, 16, 24, 40, 48, 72, 88, 104, 112, 120, 136, 144, 160, 192, 200,
                                 248])
@pytest.mark.parametrize("code,out_code,page", [(BF16, BF16, 16), (F16, F32, 8), (BF16, F32, 64)])
def test_other_head_sizes(pkg, dev, dim, code, out_code, page):
    say("head size", dim, NAME[code], NAME[out_code], page)
    check(pkg, Paged([1, 3], [150, 37], 2, dim, page, code), 6, out_code)
    check(pkg, Paged([70, 2], [190, 33], 2, dim, page, code), 6, out_code)


@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 512])
@pytest.mark.parametrize("dim", [64, 80, 96, 128, 256])
@pytest.mark.parametrize("order", ["head", "slot"])
def test_pages(pkg, dev, dim, page, order):
    """Pages that end inside a group, a tile, a piece; a window that starts in one."""
    say("pages of", page, dim, order)
    for news, lens, window in (([1, 2], [300, 21], 0), ([100, 1], [300, 21], 0),
                               ([3], [290], 77), ([90], [290], 77)):
        check(pkg, Paged(news, lens, 2, dim, page, BF16, order=order), 4, BF16, window)


@pytest.mark.parametrize("page,dim", [(4, 64), (16, 128), (32, 96)])
def test_strides_past_32_bits(pkg, dev, page, dim):
    """Pages 2^31 elements apart, where no 32-bit way from page to page will do."""
    say("far pages", page, dim)
    far, kv, n = 2 ** 31, 2, 3
    for m in (2, 40):
        c = Paged([min(m, n * page)], [n * page], kv, dim, page, F16, extra_pages=0)
        q = queries(c, 4)
        want, bound = attention(c, q, 0.1)
        block = kv * page * dim
        buf = torch.empty((c.n_pages - 1) * far + 2 * block, dtype=torch.float16, device="cuda")
        for i in range(c.n_pages):
            buf[i * far:i * far + block] = c.k[i].reshape(-1).cuda()
            buf[i * far + block:i * far + 2 * block] = c.v[i].reshape(-1).cuda()
        _, batch = c.on_gpu(pkg)
        cache = pkg.KvPages(buf.data_ptr(), buf.data_ptr() + 2 * block, F16, c.n_pages, page, kv,
                            dim, far, page * dim, dim)
        got = run(pkg, c, q, 0.1, F32, cache_batch=(cache, batch))
        assert torch.all((got.double() - want).abs() <= bound)
        del buf


def test_padded_slots_and_heads(pkg, dev):
    """Rows of a page further apart than a head, K and V in one tensor's halves."""
    say("padded strides")
    for dim, page in ((64, 32), (80, 16), (128, 4)):
        for m in (1, 50):
            c = Paged([m], [110], 2, dim, page, BF16)
            q = queries(c, 4)
            want, bound = attention(c, q, 0.125)
            n, kv = c.n_pages, 2
            both = torch.full((n, page, kv, 2, dim + 8), float("nan"), dtype=torch.bfloat16)
            both[:, :, :, 0, :dim] = c.k.transpose(1, 2)
            both[:, :, :, 1, :dim] = c.v.transpose(1, 2)
            d = both.cuda()
            _, batch = c.on_gpu(pkg)
            row = 2 * (dim + 8)
            cache = pkg.KvPages(d.data_ptr(), d.data_ptr() + 2 * (dim + 8), BF16, n, page, kv, dim,
                                page * kv * row, row, kv * row)
            got = run(pkg, c, q, 0.125, F32, cache_batch=(cache, batch))
            assert torch.all((got.double() - want).abs() <= bound), (dim, page, m)


# ------------------------------------------------------------ pieces and joins

@pytest.mark.parametrize("out_code", [F32, BF16])
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 1), (80, 2, 2), (128, 8, 1), (256, 2, 1)])
def test_pieces_of_every_number(pkg, dev, dim, heads, kv, out_code):
    """Lengths around the borders of pieces, tiles and batches of the join."""
    say("pieces", dim, heads, kv, NAME[out_code])
    for length in (127, 128, 129, 255, 257, 513, 640, 1025, 2049, 4100):
        check(pkg, Paged([1], [length], kv, dim, 32, BF16), heads, out_code)


@pytest.mark.parametrize("new", [1, 60])
def test_pieces_of_unequal_sequences(pkg, dev, new):
    """Pieces that begin past a short sequence's end, rows without keys, slots
    without tokens; the hint far from the lengths."""
    say("unequal", new)
    news, lens = [new, 1, 0, new, 5], [3000, 9, 800, new // 2, 700]
    c = Paged(news, lens, 1, 64, 16, F16)
    q = queries(c, 4)
    for hint in (None, 1, 700, 50000):
        check(pkg, c, 4, F32, q=q, **({} if hint is None else {"max_len": hint}))
        check(pkg, c, 4, F32, 100, q=q, **({} if hint is None else {"max_len": hint}))


def test_padding_rows_of_a_joined_call(pkg, dev):
    """Rows of no sequence keep what they hold where pieces are joined, too."""
    say("padding, joined")
    for m in (2, 40):
        c = Paged([m], [5000], 1, 64, 16, F16)
        q = queries(c, 4)
        want, bound = attention(c, q, 0.125)
        cache, batch = c.on_gpu(pkg, n_tok=m + 7)
        wide = torch.cat((q, torch.full((7, 4, 64), math.nan).half()))
        got = run(pkg, c, wide, 0.125, F32, cache_batch=(cache, batch))
        assert torch.all((got[:m].double() - want).abs() <= bound) and torch.all(got[m:] == 77.0)


@pytest.mark.parametrize("news,lens", [([1], [3000]), ([40], [3000])])
def test_no_page_in_one_piece(pkg, dev, news, lens):
    say("bad page in a piece", news)
    for at in (0, 90, 187):
        c = Paged(news + news, lens + lens, 1, 64, 16, F16)
        q = queries(c, 2)
        want, bound = attention(c, q, 0.125)
        c.table[0, at] = c.n_pages + 5
        got = run(pkg, c, q, 0.125, F32)
        m = news[0]
        # rows that do not see the page may be spared, but not the others
        sees = torch.arange(lens[0] - m, lens[0]) >= 16 * at
        assert int(c.dev["bad"]) == 1 and torch.all(got[:m][sees].isnan())
        assert torch.all((got[m:].double() - want[m:]).abs() <= bound[m:])


def test_cache_without_pages(pkg, dev):
    """n_pages 0: every position is without a page, nothing of k and v is read."""
    say("no pages")
    for page in (4, 16):
        for m in (1, 50):
            c = Paged([m], [60], 1, 64, page, F16)
            q = queries(c, 2)
            cache, batch = c.on_gpu(pkg)
            cache.n_pages = 0
            got = run(pkg, c, q, 0.125, F32, cache_batch=(cache, batch))
            assert torch.all(got.isnan()) and int(c.dev["bad"]) == 1


# -------------------------------------------------------------------- numbers

@pytest.mark.parametrize("code,out_code", [(BF16, F32), (F16, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("falling", [False, True])
def test_maximum_that_grows_all_the_way(pkg, dev, code, out_code, falling):
    """Scores that rise (or fall) from key to key, by 60 in all, so that the
    running maximum moves in every tile."""
    say("growing maximum", NAME[code], NAME[out_code], falling)
    for m, n, dim in ((1, 900, 64), (90, 700, 128), (70, 500, 256)):
        c = Paged([m], [n], 1, dim, 16, code)
        q = queries(c, 2)
        k, _ = c.keys(0)
        ramp = torch.linspace(60.0, 0.0, n) if falling else torch.linspace(0.0, 60.0, n)
        q = (q.float() * 0.1 + 1.0).to(TORCH[code])
        for p in range(n):
            c.put(0, p, k=(k[p].float() * 0.1 + ramp[p] / math.sqrt(dim)).to(TORCH[code]))
        check(pkg, c, 2, out_code, q=q, scale=1.0 / math.sqrt(dim))


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 3.0])
def test_scales(pkg, dev, scale):
    say("scale", scale)
    for m, n in ((2, 300), (80, 200)):
        check(pkg, Paged([m], [n], 2, 64, 16, F16), 4, F32, scale=scale)
        check(pkg, Paged([m], [n], 2, 128, 16, BF16), 4, BF16, 50, scale=scale)


def test_large_values(pkg, dev):
    """Values near the type's largest: sums of weights above 1 do not overflow."""
    say("large values")
    for m, n in ((1, 600), (70, 300)):
        c = Paged([m], [n], 1, 64, 16, F16)
        k, v = c.keys(0)
        for p in range(n):
            c.put(0, p, v=(v[p].float().sign() * 6e4).half())
        check(pkg, c, 2, F32)


def test_keys_of_infinite_score(pkg, dev):
    """A key with score -infinity weighs nothing; a row that sees only such keys
    has no result."""
    say("score -inf")
    for m, n in ((1, 200), (60, 200)):
        c = Paged([m], [n], 1, 64, 16, BF16)
        q = queries(c, 2).abs() + 0.1
        spot = n - m - 5 if m > 1 else 77
        c.put(0, spot, k=torch.full((1, 64), -math.inf).bfloat16())
        k, v = c.keys(0)
        keep = [p for p in range(n) if p != spot]
        got = run(pkg, c, q, 0.125, F32)
        for i in range(m):
            pos = n - m + i
            use = [p for p in keep if p <= pos]
            s = (k[use, 0].double() @ q[i].double().T) * 0.125
            want = torch.softmax(s, 0).T @ v[use, 0].double()
            assert torch.allclose(got[i].double(), want, rtol=1e-4, atol=1e-5)
        one = Paged([1], [1], 1, 64, 16, BF16)
        one.put(0, 0, k=torch.full((1, 64), -math.inf).bfloat16())
        assert torch.all(run(pkg, one, q[:1], 0.125, F32).isnan())


@pytest.mark.parametrize("m,n,window", [(1, 3000, 0), (3, 3000, 0), (60, 3000, 0), (300, 600, 0),
                                        (300, 600, 200)])
@pytest.mark.parametrize("dim", [64, 80, 256])
def test_infinities_in_places(pkg, dev, m, n, window, dim):
    """+infinity and NaN values at single places: they reach the rows and dims that
    see them and no others, in whole caches and in pieces."""
    say("odd values", m, n, window, dim)
    c = Paged([m], [n], 1, dim, 16, BF16)
    q = queries(c, 2)
    scale = 1 / math.sqrt(dim)
    want, bound = attention(c, q, scale, window)
    places = [(0, 3, math.inf), (n - m, dim - 1, math.nan), (n - 1, 0, -math.inf),
              (n // 2, 7, math.inf), (n // 2 + 1, 7, math.inf)]
    for p, d, x in places:
        v = c.keys(0)[1][p].clone()
        v[:, d] = x
        c.put(0, p, v=v)
    got = run(pkg, c, q, scale, F32, window)
    pos = torch.arange(n - m, n)
    expect = want.clone()
    for p, d, x in places:
        sees = (pos >= p) & ((pos - p < window) if window else (pos >= 0))
        expect[sees, :, d] = x
    finite = expect.isfinite()
    assert torch.equal(got.isfinite(), finite)
    assert torch.equal(got.isnan(), expect.isnan())
    assert torch.all((got.double() == expect)[~finite & ~expect.isnan()])
    assert torch.all((got.double() - expect).abs()[finite] <= bound[finite])


@pytest.mark.parametrize("heads,kv", [(1, 1), (7, 1), (33, 1), (64, 1), (5, 5), (40, 5), (12, 3),
                                      (140, 1)])
def test_head_layouts(pkg, dev, heads, kv):
    """Groups that fill less than a wave's rows, more than one, none evenly."""
    say("heads", heads, kv)
    for m, n in ((1, 200), (2, 130), (9, 200), (33, 90)):
        check(pkg, Paged([m, 1], [n, 17], kv, 64, 16, BF16), heads, BF16)
