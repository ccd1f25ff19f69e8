"""swamp_quantize_rows and swamp_gemm_rows_i8 on the GPU, bit for bit.

Codes: the scale is amax / 127 and a code x / scale, both one fp32 division, so the CPU's
are the same.  Products: a sum of at most 131071 terms of 2^14 is a whole number below
2^31, exact in int32 and in 64 bits; the scales' product (48 bits) is exact in 64, its
product with the sum rounds once there, then to fp32, then to y's type: the same three
roundings here, so the bits are the same.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = 0, 1, 30
TORCH = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}


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


def codes_of(x):
    """(codes, scales) of fp32 rows, on the CPU."""
    top = torch.where(x.isfinite(), x.abs(), math.inf).amax(dim=1) if x.shape[1] else torch.zeros(x.shape[0])
    scale = top / torch.full_like(top, 127.0)
    scale = torch.where(scale < 2.0 ** -126, 0.0, scale)
    fine = torch.isfinite(top) & (scale > 0)
    q = torch.where(fine[:, None], torch.round(x / torch.where(fine, scale, 1.0)[:, None]), 0.0)
    return q.to(torch.int8), torch.where(torch.isfinite(top), scale, math.nan)


@pytest.mark.parametrize("xt", [F32, F16, BF16])
@pytest.mark.parametrize("n,k", [(1, 4096), (3, 1), (5, 7), (257, 64), (2, 5000), (33, 1023),
                                 (4, 28672), (1, 40001), (70, 16)])
def test_quantize(pkg, dev, xt, n, k):
    say("quantize", xt, n, k)
    g = torch.Generator().manual_seed(n * 7 + k)
    x = (torch.randn((n, k), generator=g) * torch.exp(torch.randn((n, 1), generator=g))).to(TORCH[xt])
    if n > 2:
        x[1] = 0
        # codes that lie half way between two
        x[2, ::2] = 0.5
        x[2, 0] = 127.0
    dx = x.cuda()
    q = torch.full((n, k), 77, dtype=torch.int8, device=dev)
    scale = torch.full((n,), 77.0, device=dev)
    pkg.quantize_rows(dx.data_ptr(), xt, q.data_ptr(), scale.data_ptr(), n, k, stream=stream())
    torch.cuda.synchronize()
    want, s = codes_of(x.float())
    assert torch.equal(scale.cpu(), s)
    assert torch.equal(q.cpu(), want)


@pytest.mark.parametrize("xt", [F32, F16, BF16])
@pytest.mark.parametrize("k,x_gap,q_gap,shift", [(64, 0, 0, 1), (100, 3, 12, 0), (4097, 7, 15, 3),
                                                 (256, 4, 16, 0), (8192, 8, 5, 0)])
def test_quantize_strided(pkg, dev, xt, k, x_gap, q_gap, shift):
    """Rows with gaps, starts that no vector load is aligned for; the gaps stay."""
    say("quantize strided", xt, k, x_gap, q_gap, shift)
    n = 9
    x = torch.randn((n, k + x_gap), generator=torch.Generator().manual_seed(k)).to(TORCH[xt])
    flat = torch.zeros(n * (k + x_gap) + 8, dtype=TORCH[xt])
    flat[shift:shift + x.numel()] = x.flatten()
    dx = flat.cuda()
    q = torch.full((n * (k + q_gap) + 8,), 77, dtype=torch.int8, device=dev)
    scale = torch.empty(n, device=dev)
    pkg.quantize_rows(dx.data_ptr() + shift * dx.element_size(), xt, q.data_ptr() + shift,
                      scale.data_ptr(), n, k, x_stride=k + x_gap, q_stride=k + q_gap, stream=stream())
    torch.cuda.synchronize()
    want, s = codes_of(x[:, :k].float())
    got = q.cpu()
    assert torch.equal(scale.cpu(), s)
    rows = got[shift:shift + n * (k + q_gap)].view(n, k + q_gap)
    assert torch.equal(rows[:, :k], want)
    rows[:, :k] = 77
    if q_gap:
        assert torch.all(got == 77)


@pytest.mark.parametrize("xt", [F32, F16, BF16])
def test_quantize_lengths(pkg, dev, xt):
    """Rows about every length where a thread takes more elements."""
    for k in (511, 512, 513, 8192, 8193, 16389, 32768, 32769, 65536, 65537, 131071, 140003):
        say("quantize length", xt, k)
        x = torch.randn((3, k), generator=torch.Generator().manual_seed(k)).to(TORCH[xt])
        x[1, -1] = 9.0
        x[2, 0] = -11.0
        dx = x.cuda()
        q = torch.full((3, k), 77, dtype=torch.int8, device=dev)
        scale = torch.empty(3, device=dev)
        pkg.quantize_rows(dx.data_ptr(), xt, q.data_ptr(), scale.data_ptr(), 3, k, stream=stream())
        torch.cuda.synchronize()
        want, s = codes_of(x.float())
        assert torch.equal(scale.cpu(), s)
        assert torch.equal(q.cpu(), want)


def test_quantize_half_way(pkg, dev):
    """Quotients at half way between two codes and up to 4 steps of fp32 beside it, for
    scales of any mantissa and size."""
    say("quantize half way")
    g = torch.Generator().manual_seed(5)
    n, k = 400, 2048
    s = torch.exp2(torch.rand(n, generator=g) * 200 - 100)
    top = s * 127
    scale = top / 127
    x = (torch.randint(-127, 127, (n, k), generator=g) + 0.5) * scale[:, None]
    bits = x.view(torch.int32) + torch.randint(-4, 5, (n, k), generator=g, dtype=torch.int32)
    x = bits.view(torch.float32)
    x[:, 0] = top
    dx = x.cuda()
    q = torch.full((n, k), 77, dtype=torch.int8, device=dev)
    got = torch.empty(n, device=dev)
    pkg.quantize_rows(dx.data_ptr(), F32, q.data_ptr(), got.data_ptr(), n, k, stream=stream())
    torch.cuda.synchronize()
    want, s = codes_of(x)
    assert torch.equal(got.cpu(), s)
    assert torch.equal(q.cpu(), want)


def test_quantize_limits(pkg, dev):
    """Infinities and NaN take their row, tiny rows are zeros, the largest keep theirs."""
    say("quantize limits")
    x = torch.ones((8, 300))
    x[0, 299] = math.inf
    x[1, 0] = math.nan
    x[2, 5] = -math.inf
    x[3] = 1e-38          # a scale below 2^-126
    x[4] = 2.0 ** -119 * 1.1
    x[5] = 3.4028234e38
    x[6] = -0.0
    x[7, 7] = -3.0
    dx = x.cuda()
    q = torch.full((8, 300), 77, dtype=torch.int8, device=dev)
    scale = torch.empty(8, device=dev)
    pkg.quantize_rows(dx.data_ptr(), F32, q.data_ptr(), scale.data_ptr(), 8, 300, stream=stream())
    torch.cuda.synchronize()
    want, s = codes_of(x)
    assert torch.equal(q.cpu(), want)
    assert torch.equal(scale.isnan().cpu(), s.isnan()) and scale.isnan().sum() == 3
    assert torch.equal(scale.cpu()[3:], s[3:])
    assert scale[3] == 0 and not q[3].any() and (q[5] == 127).all() and not q[:3].any()
    pkg.quantize_rows(0, F32, 0, scale.data_ptr(), 8, 0, stream=stream())
    torch.cuda.synchronize()
    assert not scale.any()


def product(x, w, sx, sw, yt, y=None):
    total = torch.matmul(x.double(), w.double().t())  # whole numbers below 2^53
    v = (sx.double()[:, None] * sw.double()[None, :] * total).float()
    return (v if y is None else y.float() + v).to(TORCH[yt])


def operands(m, n, k, gap=0, seed=0, most=128):
    g = torch.Generator().manual_seed(m * 31 + n * 7 + k + seed)
    stride = -(-k // 16) * 16 + gap
    x = torch.randint(-most, most, (m, stride), generator=g, dtype=torch.int8)
    w = torch.randint(-most, most, (n, stride), generator=g, dtype=torch.int8)
    sx = torch.exp(torch.randn(m, generator=g)) * 1e-2
    sw = torch.exp(torch.randn(n, generator=g)) * 1e-3
    return x, w, sx, sw, stride


def run(pkg, ops, m, n, k, yt, y=None, y_stride=0, accumulate=False):
    x, w, sx, sw, stride = ops
    dx, dw, dsx, dsw = x.cuda(), w.cuda(), sx.cuda(), sw.cuda()
    if y is None:
        y = torch.full((m, y_stride or n), 55.0, dtype=TORCH[yt], device="cuda")
    pkg.gemm_rows_i8(dx.data_ptr(), dsx.data_ptr(), dw.data_ptr(), dsw.data_ptr(), y.data_ptr(), yt,
                     m, n, k, x_stride=stride, w_stride=stride, y_stride=y_stride,
                     accumulate=accumulate, stream=stream())
    torch.cuda.synchronize()
    return y


SHAPES = [  # rows of x, rows of w, columns
    (1, 1, 1), (1, 64, 64), (1, 4096, 4096), (2, 100, 333), (3, 5, 17), (4, 1000, 2048),
    (7, 130, 96), (8, 6144, 4096), (13, 257, 1000), (16, 4096, 512), (17, 33, 129), (31, 700, 4097),
    (32, 512, 8192), (33, 64, 65), (64, 2048, 1111), (65, 300, 640), (100, 129, 15), (128, 128, 128),
    (129, 1000, 777), (200, 5003, 300), (256, 256, 64), (257, 513, 4099), (333, 1031, 2111),
    (512, 4096, 1024), (1000, 70, 130), (1030, 1290, 200), (2048, 2304, 96), (5, 3, 28672),
]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("yt", [F32, F16, BF16])
def test_product(pkg, dev, m, n, k, yt):
    say("product", m, n, k, yt)
    ops = operands(m, n, k)
    y = run(pkg, ops, m, n, k, yt)
    x, w, sx, sw, _ = ops
    assert torch.equal(y.cpu(), product(x[:, :k], w[:, :k], sx, sw, yt))


@pytest.mark.parametrize("m", [1, 2, 5, 16, 40, 90, 300])
def test_every_column_count(pkg, dev, m):
    """Sums that end anywhere in a step; what lies behind a row's end counts for nothing."""
    n = 70
    for k in list(range(1, 70)) + [127, 128, 129, 191, 200, 255, 257, 511, 513, 1023, 1025]:
        say("columns", m, k)
        ops = operands(m, n, k, gap=16 * (k % 3))
        y = run(pkg, ops, m, n, k, F32)
        x, w, sx, sw, _ = ops
        assert torch.equal(y.cpu(), product(x[:, :k], w[:, :k], sx, sw, F32))


@pytest.mark.parametrize("n", [4090, 4100, 8200, 16400])
@pytest.mark.parametrize("m", [1, 16, 30, 33, 61])
def test_few_rows(pkg, dev, m, n):
    """Every way to share out the rows of w among workgroups, columns that end anywhere."""
    for k in (1, 63, 64, 100, 257, 450, 1000, 4100):
        say("few rows", m, n, k)
        ops = operands(m, n, k, gap=16 * (k % 3))
        y = run(pkg, ops, m, n, k, F32)
        x, w, sx, sw, _ = ops
        assert torch.equal(y.cpu(), product(x[:, :k], w[:, :k], sx, sw, F32))


@pytest.mark.parametrize("m", [1, 20, 130])
def test_largest_sum(pkg, dev, m):
    """131071 columns of -128: 2^31 - 2^14, the int32 that is left."""
    say("largest sum", m)
    k, n = 131071, 40
    x = torch.full((m, k + 1), -128, dtype=torch.int8)
    w = torch.full((n, k + 1), -128, dtype=torch.int8)
    w[1::2] = 127
    one = (torch.ones(m), torch.ones(n))
    y = run(pkg, (x, w) + one + (k + 1,), m, n, k, F32).cpu()
    assert torch.all(y[:, ::2] == float(131071 * 16384)) and torch.all(y[:, 1::2] == -float(131071 * 16256))


@pytest.mark.parametrize("yt", [F32, F16, BF16])
@pytest.mark.parametrize("m,n,k", [(1, 700, 512), (9, 65, 100), (70, 300, 1000), (300, 260, 64)])
def test_accumulate_into_wide_rows(pkg, dev, m, n, k, yt):
    say("accumulate", m, n, k, yt)
    ops = operands(m, n, k, gap=32)
    y0 = (torch.randn((m, n + 9), generator=torch.Generator().manual_seed(m)) * 3).to(TORCH[yt])
    y = run(pkg, ops, m, n, k, yt, y=y0.cuda(), y_stride=n + 9, accumulate=True).cpu()
    x, w, sx, sw, _ = ops
    assert torch.equal(y[:, :n], product(x[:, :k], w[:, :k], sx, sw, yt, y0[:, :n]))
    assert torch.equal(y[:, n:], y0[:, n:])


@pytest.mark.parametrize("m", [1, 6, 40, 200])
def test_scales_at_the_ends(pkg, dev, m):
    """NaN scales spoil their row or column alone; tiny and huge ones meet in 64 bits."""
    say("scales", m)
    n, k = 50, 400
    x, w, sx, sw, stride = operands(m, n, k)
    sx[0], sw[3] = 1e-30, 1e38
    sw[7] = math.nan
    sw[9] = 0.0
    if m > 2:
        sx[1], sx[2] = math.nan, 1e30
    y = run(pkg, (x, w, sx, sw, stride), m, n, k, F32).cpu()
    want = product(x[:, :k], w[:, :k], sx, sw, F32)
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


def test_no_columns(pkg, dev):
    say("no columns")
    sx, sw = torch.ones(3, device=dev), torch.ones(5, device=dev)
    y = torch.full((3, 5), 4.0, device=dev)
    pkg.gemm_rows_i8(0, sx.data_ptr(), 0, sw.data_ptr(), y.data_ptr(), F32, 3, 5, 0,
                     accumulate=True, stream=stream())
    torch.cuda.synchronize()
    assert (y == 4).all()
    pkg.gemm_rows_i8(0, sx.data_ptr(), 0, sw.data_ptr(), y.data_ptr(), F32, 3, 5, 0, stream=stream())
    torch.cuda.synchronize()
    assert (y == 0).all()


@pytest.mark.parametrize("m,n,k", [(1, 512, 8192), (20, 256, 4096), (300, 500, 2000)])
def test_with_and_without_scratch(pkg, dev, m, n, k):
    """In a captured graph with nothing reserved the sum is not split: the same bits, on
    every replay, with other inputs."""
    say("scratch", m, n, k)
    ops = operands(m, n, k)
    x, w, sx, sw, stride = ops
    eager = run(pkg, ops, m, n, k, F32).cpu()
    dx, dw, dsx, dsw = x.cuda(), w.cuda(), sx.cuda(), sw.cuda()
    y = torch.zeros((m, n), device=dev)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        pkg.gemm_rows_i8(dx.data_ptr(), dsx.data_ptr(), dw.data_ptr(), dsw.data_ptr(), y.data_ptr(),
                         F32, m, n, k, x_stride=stride, w_stride=stride, stream=side.cuda_stream)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), eager)
    dx.copy_(torch.flip(x, dims=(0,)).contiguous())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y.cpu(), product(x.flip(0)[:, :k], w[:, :k], sx, sw, F32))


@pytest.mark.parametrize("m", [1, 12, 100, 400])
def test_quantized_layer(pkg, dev, m):
    """Activations and weights quantized on the device and multiplied: the sum of products
    of what the codes stand for, and near the product of the originals: each factor is off
    by half a step of its row's scale at most."""
    say("layer", m)
    n, k = 300, 1000
    g = torch.Generator().manual_seed(m)
    x, w = torch.randn((m, k), generator=g), torch.randn((n, k), generator=g) / math.sqrt(k)
    stride = 1008
    dx, dw = x.cuda(), w.cuda()
    qx = torch.zeros((m, stride), dtype=torch.int8, device=dev)
    qw = torch.zeros((n, stride), dtype=torch.int8, device=dev)
    sx, sw = torch.empty(m, device=dev), torch.empty(n, device=dev)
    y = torch.empty((m, n), device=dev)
    pkg.quantize_rows(dx.data_ptr(), F32, qx.data_ptr(), sx.data_ptr(), m, k, q_stride=stride,
                      stream=stream())
    pkg.quantize_rows(dw.data_ptr(), F32, qw.data_ptr(), sw.data_ptr(), n, k, q_stride=stride,
                      stream=stream())
    pkg.gemm_rows_i8(qx.data_ptr(), sx.data_ptr(), qw.data_ptr(), sw.data_ptr(), y.data_ptr(), F32,
                     m, n, k, x_stride=stride, w_stride=stride, stream=stream())
    torch.cuda.synchronize()
    cx, tx = codes_of(x)
    cw, tw = codes_of(w)
    assert torch.equal(y.cpu(), product(cx, cw, tx, tw, F32))
    step = 0.5 * (1 + 2.0 ** -20)  # of a scale
    bound = step * (tx[:, None].double() * w.double().abs().sum(1)[None]
                    + tw[None].double() * x.double().abs().sum(1)[:, None]
                    + step * k * tx[:, None].double() * tw[None].double())
    err = (y.cpu().double() - x.double() @ w.double().t()).abs()
    assert torch.all(err <= bound + 2.0 ** -24 * y.cpu().double().abs())
