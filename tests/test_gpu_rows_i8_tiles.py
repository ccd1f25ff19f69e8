"""swamp_gemm_rows_i8 in each of its tiles, bit for bit: sizes for which the plan takes the
tile (rows_plan_sizes.py), the three output types, results added to what is there, rows of y
with gaps that no 16-byte store is aligned for.

The reference's sums are whole numbers below 2^53 in float64, exact in any order, so the
device's own product gives them; then the same three roundings as in test_gpu_rows_i8.py."""
import pytest
import torch

from rows_plan_sizes import ONE, PIECES
from test_gpu_rows_i8 import BF16, F16, F32, TORCH, say, stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()
    pkg.init()
    yield torch.device("cuda")
    torch.cuda.empty_cache()


@pytest.mark.parametrize("m,n,k", [size for sizes in (ONE, PIECES) for each in sizes.values()
                                   for size in each])
def test_tile(pkg, dev, m, n, k):
    g = torch.Generator(device=dev).manual_seed(m + 3 * n + 7 * k)
    stride = -(-k // 16) * 16 + 16 * (n % 2)
    x, w = (torch.randint(-128, 128, (rows, stride), generator=g, dtype=torch.int8, device=dev)
            for rows in (m, n))
    sx = torch.exp(torch.randn(m, generator=g, device=dev)) * 1e-2
    sw = torch.exp(torch.randn(n, generator=g, device=dev)) * 1e-3
    value = torch.matmul(x[:, :k].double(), w[:, :k].double().t())
    value.mul_(sx.double()[:, None] * sw.double()[None, :])
    value = value.float()
    for t, add, gap in ((F32, 0, 0), (F16, 0, 0), (BF16, 0, 0), (F32, 0, 3), (BF16, 0, 1), (F32, 1, 0),
                        (F16, 1, 5), (BF16, 1, 0)):
        say("tile", m, n, k, t, add, gap)
        y = torch.full((m, n + gap), 55.0, dtype=TORCH[t], device=dev)
        if add:
            y[:, :n] = torch.randn((m, n), generator=g, device=dev)
        want = (y[:, :n].float() + value if add else value).to(TORCH[t])
        pkg.gemm_rows_i8(x.data_ptr(), sx.data_ptr(), w.data_ptr(), sw.data_ptr(), y.data_ptr(), t,
                         m, n, k, x_stride=stride, w_stride=stride, y_stride=n + gap,
                         accumulate=bool(add), stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(y[:, :n], want)
        assert torch.all(y[:, n:] == 55)
