"""swamp_rope and swamp_kv_append on the GPU against 64 bits on the CPU
(tests/paged_reference.py has the bounds and what they count)."""
import math

import pytest
import torch

from paged_reference import BF16, F16, F32, NAME, TORCH, Paged, half_step, turn, turn_bound

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


def spec(pkg, freqs, n_rot, halves, mscale=1.0):
    return pkg.Rope(freqs.data_ptr(), n_rot, pkg.ROPE_HALVES if halves else pkg.ROPE_PAIRS, mscale)


@pytest.mark.parametrize("xt,ot", [(F32, F32), (F32, BF16), (F16, F16), (BF16, F32), (F32, F16),
                                   (BF16, BF16), (F16, BF16)])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("n,heads,dim,rot", [(1, 32, 128, 128), (5, 3, 80, 32), (7, 1, 64, 2),
                                             (3, 5, 2, 2), (2, 40, 256, 254), (65, 7, 96, 24)])
def test_rope(pkg, dev, n, heads, dim, rot, halves, xt, ot):
    say("rope", n, heads, dim, rot, "halves" if halves else "pairs", NAME[xt], NAME[ot])
    g = torch.Generator().manual_seed(n * 1000 + dim)
    x = torch.randn((n, heads, dim), generator=g).to(TORCH[xt])
    pos = torch.randint(0, 131072, (n,), generator=g, dtype=torch.int32)
    freqs = torch.from_numpy(pkg.rope_freqs(rot, 500000.0))
    dx, dp, df = x.cuda(), pos.cuda(), freqs.cuda()
    out = torch.full((n, heads, dim), 77.0, dtype=TORCH[ot], device=dev)
    pkg.rope(spec(pkg, df, rot, halves, 1.25), dp.data_ptr(), dx.data_ptr(), xt, out.data_ptr(), ot,
             n, heads, dim, stream=stream())
    torch.cuda.synchronize()
    want = turn(x, pos, freqs, rot, halves, 1.25)
    bound = turn_bound(x, rot, halves, 1.25, ot)
    assert torch.all((out.cpu().double() - want).abs() <= bound)
    # what does not turn is the input, rounded
    assert torch.equal(out.cpu()[..., rot:], x[..., rot:].float().to(TORCH[ot]))


@pytest.mark.parametrize("start", [0, 2 ** 20 + 3, 2 ** 31 - 9, -5])
def test_rope_far_positions(pkg, dev, start):
    """The angle's fraction survives positions of any size, and negative ones."""
    say("rope far", start)
    n, dim = 8, 128
    x = torch.randn((n, 2, dim), generator=torch.Generator().manual_seed(3))
    pos = (torch.arange(n) + start).to(torch.int32)
    freqs = torch.from_numpy(pkg.rope_freqs(dim, 10000.0, 8.0, 4096))
    dx, dp, df = x.cuda(), pos.cuda(), freqs.cuda()
    out = torch.empty_like(dx)
    pkg.rope(spec(pkg, df, dim, True), dp.data_ptr(), dx.data_ptr(), F32, out.data_ptr(), F32, n, 2,
             dim, stream=stream())
    torch.cuda.synchronize()
    # the angle's own rounding: two of 2^-53 of up to 2^31 radians, in both
    slack = x.double().abs().amax() * 2 * 4 * 2.0 ** (31 - 53)
    err = (out.cpu().double() - turn(x, pos, freqs, dim, True)).abs()
    assert torch.all(err <= turn_bound(x, dim, True, 1.0, F32) + slack)


@pytest.mark.parametrize("shift", [0, 1])
def test_rope_strided_in_place(pkg, dev, shift):
    """The q part of fused rows turned in place; its neighbours stay; a start
    that is not 16-byte aligned takes single elements."""
    say("rope strided in place", shift)
    n, heads, dim, width = 33, 6, 64, 6 * 64 + 2 * 130 + 1
    buf = torch.randn((n, width), generator=torch.Generator().manual_seed(9))
    pos = torch.arange(n, dtype=torch.int32)
    freqs = torch.from_numpy(pkg.rope_freqs(dim))
    d, dp, df = buf.cuda(), pos.cuda(), freqs.cuda()
    at = d.data_ptr() + 4 * shift
    pkg.rope(spec(pkg, df, dim, False), dp.data_ptr(), at, F32, at, F32, n, heads, dim,
             x_stride=width, out_stride=width, stream=stream())
    torch.cuda.synchronize()
    x = buf[:, shift:shift + heads * dim].reshape(n, heads, dim)
    got = d.cpu()
    turned = got[:, shift:shift + heads * dim].reshape(n, heads, dim).double()
    assert torch.all((turned - turn(x, pos, freqs, dim, False)).abs()
                     <= turn_bound(x, dim, False, 1.0, F32))
    assert torch.equal(got[:, :shift], buf[:, :shift])
    assert torch.equal(got[:, shift + heads * dim:], buf[:, shift + heads * dim:])


@pytest.mark.parametrize("xt,code", [(F32, F16), (F32, BF16), (BF16, BF16), (F16, F16), (BF16, F16)])
@pytest.mark.parametrize("order", ["head", "slot"])
@pytest.mark.parametrize("news,lens,heads,kv,dim,page,rot", [
    ([1], [1], 4, 4, 64, 16, 64),
    ([1, 1, 1], [33, 1, 17], 8, 2, 128, 16, 64),
    ([5, 0, 40, 1], [5, 9, 77, 300], 6, 3, 80, 8, 32),
    ([70] * 3, [70, 100, 4096], 2, 1, 256, 1, 256),
])
def test_append(pkg, dev, news, lens, heads, kv, dim, page, rot, order, xt, code):
    say("append", news, lens, heads, kv, dim, page, order, NAME[xt], NAME[code])
    c = Paged(news, lens, kv, dim, page, code, order=order)
    width = (heads + 2 * kv) * dim + 8
    x = torch.randn((c.n_tok, width), generator=c.g).to(TORCH[xt])
    freqs = torch.from_numpy(pkg.rope_freqs(rot))
    cache, batch = c.on_gpu(pkg)
    dx, df = x.cuda(), freqs.cuda()
    q_out = torch.empty((c.n_tok, heads, dim), dtype=TORCH[code], device=dev)
    size = dx.element_size()
    pkg.kv_append(cache, batch, spec(pkg, df, rot, True), dx.data_ptr(),
                  dx.data_ptr() + heads * dim * size, dx.data_ptr() + (heads + kv) * dim * size, xt,
                  q_out.data_ptr(), heads, q_stride=width, k_stride=width, v_stride=width,
                  stream=stream())
    torch.cuda.synchronize()
    pos = torch.cat([torch.arange(n - m, n) for m, n in zip(news, lens)])
    parts = x[:, :(heads + 2 * kv) * dim].reshape(c.n_tok, -1, dim)
    q, k, v = parts[:, :heads], parts[:, heads:heads + kv], parts[:, heads + kv:]
    assert torch.all((q_out.cpu().double() - turn(q, pos, freqs, rot, True)).abs()
                     <= turn_bound(q, rot, True, 1.0, code))
    # the new tokens' slots hold them, every other one what it held
    want_k, got = turn(k, pos, freqs, rot, True), c.cache_back()
    tol = turn_bound(k, rot, True, 1.0, code)
    k0, v0 = c.k.clone(), c.v.clone()
    t = 0
    for s, m in enumerate(news):
        for i in range(m):
            p = lens[s] - m + i
            page_id, slot = int(c.table[s, p // page]), p % page
            assert torch.all((got[0][page_id, :, slot].double() - want_k[t]).abs() <= tol[t])
            assert torch.equal(got[1][page_id, :, slot], v[t].float().to(TORCH[code]))
            k0[page_id, :, slot], v0[page_id, :, slot] = got[0][page_id, :, slot], got[1][page_id, :, slot]
            t += 1
    as_bits = lambda z: z.contiguous().view(torch.int16)  # noqa: E731
    assert torch.equal(as_bits(got[0]), as_bits(k0)) and torch.equal(as_bits(got[1]), as_bits(v0))
    assert int(c.dev["bad"]) == 0


def test_append_many_sequences_without_rotation(pkg, dev):
    """More sequences than a wave's lanes, empty ones among them; k and v only."""
    say("append 150 sequences")
    news = [(i * 7) % 3 for i in range(150)]
    lens = [n + (i * 5) % 23 for i, n in enumerate(news)]
    c = Paged(news, lens, 2, 64, 4, F16)
    cache, batch = c.on_gpu(pkg)
    k, v = (torch.randn((c.n_tok, 2, 64), generator=c.g) for _ in range(2))
    dk, dv = k.cuda(), v.cuda()
    pkg.kv_append(cache, batch, None, 0, dk.data_ptr(), dv.data_ptr(), F32, 0, 0, stream=stream())
    torch.cuda.synchronize()
    got, t = c.cache_back(), 0
    for s, m in enumerate(news):
        for i in range(m):
            p = lens[s] - m + i
            page_id = int(c.table[s, p // 4])
            assert torch.equal(got[0][page_id, :, p % 4], k[t].half())
            assert torch.equal(got[1][page_id, :, p % 4], v[t].half())
            t += 1
    assert t == c.n_tok and int(c.dev["bad"]) == 0


def test_append_positions_without_a_page(pkg, dev):
    """A token whose page id is outside the cache, whose position is past the
    table or before 0 is left out and flagged; padding rows are not touched."""
    say("append bad pages")
    for what in ("id", "table", "before"):
        c = Paged([3, 2], [20, 9], 1, 64, 8, BF16)
        if what == "id":
            c.table[0, 2] = c.n_pages  # positions 16 ..
        elif what == "table":
            c.len[0] = 8 * c.table.shape[1] + 2  # its last two positions have no column
        else:
            c.len[0] = 2  # its first new token is at position -1
        cache, batch = c.on_gpu(pkg, n_tok=7)
        x = torch.randn((7, 1, 64), generator=c.g).cuda()
        q_out = torch.full((7, 1, 64), 5.0, dtype=torch.bfloat16, device=dev)
        pkg.kv_append(cache, batch, None, x.data_ptr(), x.data_ptr(), x.data_ptr(), F32,
                      q_out.data_ptr(), 1, stream=stream())
        torch.cuda.synchronize()
        assert int(c.dev["bad"]) == 1, what
        assert torch.equal(q_out[:5], x[:5].bfloat16()) and torch.all(q_out[5:] == 5.0)
        got = c.cache_back()[0]
        changed = (got.view(torch.int16) != c.k.view(torch.int16)).any(-1).sum()
        assert int(changed) == {"id": 2, "table": 3, "before": 4}[what], what


def test_append_rounds_to_nearest(pkg, dev):
    """fp32 to 16 bits: ties to even, overflow to infinity, NaN stays NaN."""
    say("append rounding")
    special = torch.tensor([1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 65519.0, 65520.0, -1e30, math.inf,
                            math.nan, 2.0 ** -25, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 3.4e38, -0.0])
    for code in (F16, BF16):
        c = Paged([1], [1], 1, 64, 1, code)
        cache, batch = c.on_gpu(pkg)
        x = torch.zeros((1, 1, 64))
        x[0, 0, :12] = special
        d = x.cuda()
        pkg.kv_append(cache, batch, None, 0, d.data_ptr(), d.data_ptr(), F32, 0, 0, stream=stream())
        torch.cuda.synchronize()
        got = c.cache_back()[1][int(c.table[0, 0]), 0, 0]
        want = x[0, 0].to(TORCH[code])
        assert torch.equal(got.isnan(), want.isnan())
        keep = ~want.isnan()
        assert torch.equal(got[keep].view(torch.int16), want[keep].view(torch.int16))
