"""The forms of swamp_kv_append on the GPU: both layouts of the rotation, rows that
take four elements at a time and rows that take single ones, a magnitude, and q
written into wider rows.  Oracle and bounds: tests/paged_reference.py."""
import pytest
import torch

from paged_reference import BF16, F16, F32, NAME, TORCH, Paged, turn, turn_bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("xt,code", [(F32, F16), (F32, BF16), (BF16, BF16), (F16, F16), (F16, BF16)])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("rot,shift,gap", [
    (64, 0, 0),    # four at a time
    (64, 0, 24),   # and into wider rows of q
    (20, 0, 0),    # pairs that are not whole units of four: single elements
    (36, 0, 8),
    (64, 1, 0),    # rows that do not begin on 16 (8) bytes: single elements
    (2, 1, 3),     # and an odd stride of q's rows
])
@pytest.mark.parametrize("news,lens,heads,kv,dim,page", [([1, 3], [40, 3], 6, 2, 64, 16),
                                                         ([9, 0, 1], [70, 5, 1], 4, 4, 80, 8)])
def test_append_forms(pkg, news, lens, heads, kv, dim, page, rot, shift, gap, halves, xt, code):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    pkg.init()
    print("[gpu case] append form", lens, dim, rot, shift, gap, halves, NAME[xt], NAME[code],
          flush=True)
    mscale = 1.25
    c = Paged(news, lens, kv, dim, page, code)
    used = (heads + 2 * kv) * dim
    x = torch.randn((c.n_tok, used + 16), generator=c.g).to(TORCH[xt])
    freqs = torch.from_numpy(pkg.rope_freqs(rot))
    cache, batch = c.on_gpu(pkg)
    dx, df = x.cuda(), freqs.cuda()
    wide = torch.full((c.n_tok, heads * dim + gap), 5.0, dtype=TORCH[code], device="cuda")
    size = dx.element_size()
    at = dx.data_ptr() + shift * size
    spec = pkg.Rope(df.data_ptr(), rot, pkg.ROPE_HALVES if halves else pkg.ROPE_PAIRS, mscale)
    pkg.kv_append(cache, batch, spec, at, at + heads * dim * size, at + (heads + kv) * dim * size, xt,
                  wide.data_ptr(), heads, q_stride=used + 16, k_stride=used + 16,
                  v_stride=used + 16, q_out_stride=heads * dim + gap,
                  stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    pos = torch.cat([torch.arange(n - m, n) for m, n in zip(news, lens)])
    parts = x[:, shift:shift + used].reshape(c.n_tok, -1, dim)
    q, k, v = parts[:, :heads], parts[:, heads:heads + kv], parts[:, heads + kv:]
    got_q = wide.cpu()
    assert torch.all(got_q[:, heads * dim:] == 5.0)  # what lies between the rows
    got_q = got_q[:, :heads * dim].reshape(c.n_tok, heads, dim)
    assert torch.all((got_q.double() - turn(q, pos, freqs, rot, halves, mscale)).abs()
                     <= turn_bound(q, rot, halves, mscale, code))
    want_k, tol = turn(k, pos, freqs, rot, halves, mscale), turn_bound(k, rot, halves, mscale, code)
    got, k0, v0 = c.cache_back(), c.k.clone(), c.v.clone()
    t = 0
    for s, m in enumerate(news):
        for i in range(m):
            p = lens[s] - m + i
            page_id, slot = int(c.table[s, p // page]), p % page
            assert torch.all((got[0][page_id, :, slot].double() - want_k[t]).abs() <= tol[t])
            assert torch.equal(got[0][page_id, :, slot, rot:], k[t, :, rot:].float().to(TORCH[code]))
            assert torch.equal(got[1][page_id, :, slot], v[t].float().to(TORCH[code]))
            k0[page_id, :, slot], v0[page_id, :, slot] = got[0][page_id, :, slot], got[1][page_id, :, slot]
            t += 1
    assert torch.equal(got[0].view(torch.int16), k0.view(torch.int16))
    assert torch.equal(got[1].view(torch.int16), v0.view(torch.int16))
    assert int(c.dev["bad"]) == 0
