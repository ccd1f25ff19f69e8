"""8-bit products, beam selection and pages where offsets pass 32 bits, and products on two
streams at once.  Buffers of many GB of which a few rows are used; values are bit-exact as in
the other tests of these calls."""
import pytest
import torch

pytestmark = pytest.mark.gpu
GB = 1 << 30


@pytest.fixture(scope="module")
def dev(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()
    pkg.init()
    if torch.cuda.mem_get_info()[0] < 60 * GB:
        pytest.skip("less than 60 GB free")
    yield torch.device("cuda")
    torch.cuda.empty_cache()


def say(*a):
    print("[gpu case]", *a, flush=True)


def stream():
    return torch.cuda.current_stream().cuda_stream


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def spread(dev, rows, stride, dtype):
    """[n][width] rows `stride` apart in a buffer that ends with the last one."""
    n, width = rows.shape
    flat = torch.empty((n - 1) * stride + width, dtype=dtype, device=dev)
    out = flat.as_strided((n, width), (stride, 1))
    out.copy_(rows)
    return flat, out


def test_quantize(pkg, dev):
    say("quantize far")
    x = torch.randn((4, 1000), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    xs, qs = (1 << 31) + 8, (1 << 31) + 3
    flat, _ = spread(dev, x, xs, torch.bfloat16)
    q, rows = spread(dev, torch.zeros((4, 1000), dtype=torch.int8), qs, torch.int8)
    scale = torch.empty(4, device=dev)
    pkg.quantize_rows(flat.data_ptr(), pkg.BF16, q.data_ptr(), scale.data_ptr(), 4, 1000,
                      x_stride=xs, q_stride=qs, stream=stream())
    torch.cuda.synchronize()
    want = x.float().abs().amax(dim=1) / 127
    assert torch.equal(scale.cpu(), want)
    assert torch.equal(rows.cpu(), torch.round(x.float() / want[:, None]).to(torch.int8))


@pytest.mark.parametrize("m", [5, 40, 300, 700])
def test_products(pkg, dev, m):
    """Code rows nearly 8 MB apart, rows of y 64 MB."""
    say("products far", m)
    n, k, stride, ys = 600, 100, (1 << 23) - 16, (1 << 24) + 5
    g = torch.Generator().manual_seed(m)
    x = torch.randint(-128, 128, (m, 112), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, 112), generator=g, dtype=torch.int8)
    sx, sw = torch.rand(m, generator=g), torch.rand(n, generator=g)
    dx, _ = spread(dev, x, stride, torch.int8)
    dw, _ = spread(dev, w, stride, torch.int8)
    y, rows = spread(dev, torch.full((m, n), 55.0), ys, torch.float32)
    dsx, dsw = sx.cuda(), sw.cuda()
    pkg.gemm_rows_i8(dx.data_ptr(), dsx.data_ptr(), dw.data_ptr(), dsw.data_ptr(), y.data_ptr(),
                     pkg.F32, m, n, k, x_stride=stride, w_stride=stride, y_stride=ys,
                     stream=stream())
    torch.cuda.synchronize()
    total = torch.matmul(x[:, :k].double(), w[:, :k].double().t())
    assert torch.equal(rows.cpu(), (sx.double()[:, None] * sw.double() * total).float())


def test_products_on_two_streams(pkg, dev):
    """Sums in pieces, each in its stream's scratch, and few rows beside them."""
    say("products on two streams")
    work = []
    for i, (m, n, k) in enumerate(((200, 640, 8192), (200, 640, 8192), (7, 4096, 4096))):
        g = torch.Generator().manual_seed(i)
        x = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
        w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
        sx, sw = torch.rand(m, generator=g), torch.rand(n, generator=g)
        want = (sx.double()[:, None] * sw.double() * torch.matmul(x.double(), w.double().t())).float()
        dx, dw, dsx, dsw = x.cuda(), w.cuda(), sx.cuda(), sw.cuda()
        work.append((torch.cuda.Stream(), dx, dsx, dw, dsw, torch.zeros((m, n), device=dev), want))
    assert pkg.gpu_lib().swamp_gemm_rows_i8_workspace(200, 640, 8192) > 0
    torch.cuda.synchronize()
    for _ in range(10):
        for s, dx, dsx, dw, dsw, y, _ in work:
            pkg.gemm_rows_i8(dx.data_ptr(), dsx.data_ptr(), dw.data_ptr(), dsw.data_ptr(),
                             y.data_ptr(), pkg.F32, dx.shape[0], dw.shape[0], dx.shape[1],
                             stream=s.cuda_stream)
    torch.cuda.synchronize()
    for *_, y, want in work:
        assert torch.equal(y.cpu(), want)


def test_select(pkg, dev):
    say("select far")
    v, stride = 9000, (1 << 31) + 2
    logits = torch.randn((4, v), generator=torch.Generator().manual_seed(8)) * 3
    score = torch.tensor([-1.0, -2.0, -0.5, -3.0])
    flat, _ = spread(dev, logits.half(), stride, torch.float16)
    near = logits.half().cuda()
    ds = score.cuda()
    got = []
    for at, st in ((flat, stride), (near, 0)):
        parent, token, out = i32([7] * 12), i32([7] * 12), torch.full((12,), 7.0, device=dev)
        pkg.beam_select(pkg.BeamSpec(2, 2, v, 6, -1), at.data_ptr(), pkg.F16, ds.data_ptr(),
                        parent.data_ptr(), token.data_ptr(), out.data_ptr(), logits_stride=st,
                        stream=stream())
        torch.cuda.synchronize()
        got.append((parent.tolist(), token.tolist(), out.tolist()))
    assert got[0] == got[1]
    total = (score.double()[:, None] + torch.log_softmax(logits.half().double(), dim=1)).view(2, 2 * v)
    for s in range(2):
        best = torch.sort(total[s], descending=True, stable=True).indices[:6]
        assert got[0][0][6 * s:6 * s + 6] == (2 * s + best // v).tolist()
        assert got[0][1][6 * s:6 * s + 6] == (best % v).tolist()


def test_pages(pkg, dev):
    """Tables 2^30 entries apart, of which each holds a few; the last one ends with its
    entries."""
    say("tables far")
    stride, page, n_pages = 1 << 30, 4, 40
    rows = torch.full((5, 8), -7, dtype=torch.int32)
    rows[:, :3] = torch.tensor([[30, 31, 32], [30, 31, 33], [30, 31, 34], [35, 36, 37], [38, 39, 21]])
    flat, table = spread(dev, rows, stride, torch.int32)
    length = i32([10, 11, 9, 12, 10])
    refs, used = torch.zeros(n_pages, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    for e in rows[:, :3].flatten().tolist():
        refs[e] += 1
        used[e // 32] |= 1 << e % 32
    dr = refs.cuda()
    du = torch.where(used >= 1 << 31, used - (1 << 32), used).to(torch.int32).cuda()
    src, dst, count, bad = i32([0] * 40), i32([0] * 40), i32([0]), i32([0])
    pool = pkg.PagePool(n_pages, page, dr.data_ptr(), du.data_ptr())
    tables = pkg.PageTables(5, length.data_ptr(), flat.data_ptr(), stride, bad.data_ptr())
    moves = pkg.PageMoves(40, src.data_ptr(), dst.data_ptr(), count.data_ptr())
    parent = i32([1, 1, 2, 3, 3])
    pkg.pages_fork(pool, tables, parent.data_ptr(), stream=stream())
    new = i32([1, 1, 3, 1, 4])
    pkg.pages_extend(pool, tables, new.data_ptr(), moves, stream=stream())
    torch.cuda.synchronize()
    # sequence 0 parts from page 33; 2 fills page 34 and none more; 3 and 4 take new ones
    assert length.tolist() == [12, 12, 12, 13, 16] and int(bad) == 0
    assert [src[0].item(), dst[0].item(), count.item()] == [33, 0, 1]
    assert table[:, :4].tolist() == [[30, 31, 0, -7], [30, 31, 33, -7], [30, 31, 34, -7],
                                     [35, 36, 37, 1], [35, 36, 37, 2]]
    keep = i32([12, 12, 0, 13, 9])
    pkg.pages_trim(pool, tables, keep.data_ptr(), stream=stream())
    pkg.pages_compact(pool, tables, moves, stream=stream())
    torch.cuda.synchronize()
    # in use: 0, 1, 30, 31, 33, 35, 36, 37; 2, 3, ... 7 are free below 8
    assert count.item() == 6
    assert src[:6].tolist() == [30, 31, 33, 35, 36, 37] and dst[:6].tolist() == [2, 3, 4, 5, 6, 7]
    assert [table[i, :c].tolist() for i, c in ((0, 3), (1, 3), (3, 4), (4, 3))] == [
        [2, 3, 0], [2, 3, 4], [5, 6, 7, 1], [5, 6, 7]]
    assert dr.tolist() == [1, 1, 2, 2, 1, 2, 2, 2] + [0] * 32
    assert du.tolist() == [255, 0]


def test_copy(pkg, dev):
    say("copy far")
    n_pages, kv, page, dim = 70000, 8, 64, 128  # 2^16 elements a page
    k = torch.empty((n_pages, kv * page * dim), dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    g = torch.Generator().manual_seed(2)
    for t in (k, v):
        for p in (0, 69999, 1, 65537):
            t[p] = torch.randn(kv * page * dim, generator=g).to(torch.bfloat16).cuda()
    src, dst, count = i32([69999, 0]), i32([1, 65537]), i32([2])
    caches = pkg.kv_caches([pkg.KvPages(k.data_ptr(), v.data_ptr(), pkg.BF16, n_pages, page, kv, dim)])
    pkg.kv_copy(caches, pkg.PageMoves(2, src.data_ptr(), dst.data_ptr(), count.data_ptr()),
                stream=stream())
    torch.cuda.synchronize()
    for t in (k, v):
        assert torch.equal(t[1], t[69999]) and torch.equal(t[65537], t[0])
        assert not torch.equal(t[0], t[1])
