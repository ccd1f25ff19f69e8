"""A sliding window of 2^30 keys and more, over a cache whose pages are one page
many times over."""
import pytest
import torch

from paged_reference import F16, F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 32])
def test_window_of_a_billion_keys(pkg, new):
    """Positions reach 2^31: a window of 2^30 keys still ends.  Keys before it score
    40 above all others and have another value; keys within it all score 0 and hold
    1, so that a row that sees none of the former is 1."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    pkg.init()
    print("[gpu case] window of 2^30", new, flush=True)
    page, dim, window = 65536, 8, 2 ** 30
    last = window + 100  # the last row's position
    cols = last // page + 1
    k = torch.zeros((2, 1, page, dim), dtype=torch.float16)
    v = torch.ones_like(k)
    hidden = last - new + 1 - window + 1  # positions that no row sees
    k[0, 0, :hidden], v[0, 0, :hidden] = 5.0, -3.0
    table = torch.ones((1, cols), dtype=torch.int32)
    table[0, 0] = 0
    dk, dv, dt = k.cuda(), v.cuda(), table.cuda()
    first = torch.tensor([0, new], dtype=torch.int32).cuda()
    length = torch.tensor([last + 1], dtype=torch.int32).cuda()
    q = torch.ones((new, 1, dim), dtype=torch.float16).cuda()
    out = torch.zeros((new, 1, dim), device="cuda")
    cache = pkg.KvPages(dk.data_ptr(), dv.data_ptr(), F16, 2, page, 1, dim)
    batch = pkg.SeqBatch(1, new, new, last + 1, first.data_ptr(), length.data_ptr(), dt.data_ptr(),
                         cols)
    pkg.attn_paged(cache, batch, q.data_ptr(), 1, 1.0, out.data_ptr(), F32, window=window,
                   stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    # sums of ones are exact up to 2^24; what a wave sums (2^30 keys over 256 pieces of
    # four waves) is below, and the join's 260 additions round by 2^-24 each, above and
    # below the line: 2 * 260 * 2^-25 < 2^-15 at worst, but for equal numbers alike
    assert torch.all((out - 1).abs() <= 2.0 ** -15), out
