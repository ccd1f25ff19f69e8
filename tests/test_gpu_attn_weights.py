"""The softmax weights of swamp_attn_paged on the GPU, against 64 bits on the CPU,
where the keys that make a row's result weigh far less than its largest one: a
first key that takes nearly all of the weight and whose own value is 0."""
import copy
import math

import pytest
import torch

from paged_reference import BF16, F16, F32, NAME, TORCH, Paged, attention, half_step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()
    pkg.init()
    return torch.device("cuda")


def _run(pkg, c, q, scale, out_code, **more):
    cache, batch = c.on_gpu(pkg, **more)
    dq, out = q.cuda(), torch.full(q.shape, 77.0, dtype=TORCH[out_code], device="cuda")
    pkg.attn_paged(cache, batch, dq.data_ptr(), q.shape[1], scale, out.data_ptr(), out_code,
                   stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert int(c.dev["bad"]) == 0
    return out.cpu()


def _sink(new, n, dim, code, below, spread):
    """A cache whose key 0 scores `below` nats above all others, which score within
    `spread` of one another, and whose value there is 0.  The others' values are
    large, so that the result is one of the type's ordinary numbers.  q is 1 in dim 0
    and 0 in dim 1 and after, so that scores are the keys' dim 0, exactly."""
    c = Paged([new], [n], 1, dim, 16, code)
    k, v = (x.clone() for x in c.keys(0))
    s = (torch.rand(n, generator=c.g) * spread - 0.3).to(TORCH[code])
    s[0] = below - 0.3
    k[:, 0, 0] = s
    v[0] = 0
    # (positive, between half and all of the size: a sum that no chance takes to 0)
    v[1:] = ((v[1:].float().abs().clamp(max=4) / 8 + 0.5) * (30000 if code == F16 else 1)).to(v.dtype)
    for p in range(n):
        c.put(0, p, k=k[p], v=v[p])
    q = torch.zeros((new, 2, dim), dtype=TORCH[code])
    q[:, :, 0] = 1
    return c, q


def _bound(c, q, out_code, weight):
    """As paged_reference.attention's, with the scores exact and each weight off by
    `weight` of itself at most, for values that are all positive: 2^-24 (1 + 1 + 1 + 1)
    for the product with log2 e, the distance to the maximum, the exponential and the
    sum's share of each, of the largest score (20), and 8 sqrt(n) 2^-24 for n
    additions."""
    want, _ = attention(c, q, 1.0)
    n = c.lens[0]
    rel = weight + 2.0 ** -24 * (4 * 24 + 4 + 2 * 8 * math.sqrt(n))
    return want, want.abs() * (rel + half_step(out_code)) + (2.0 ** -25 if out_code == F16 else 0)


@pytest.mark.parametrize("whole", [False, True])  # (a max_len of 0: in one piece)
@pytest.mark.parametrize("out_code", [F16, BF16, F32])
@pytest.mark.parametrize("below,spread", [(14.0, 1.0), (16.0, 0.0), (18.0, 1.0), (20.0, 0.0)])
@pytest.mark.parametrize("new,n,dim", [(1, 5000, 64), (1, 4000, 128), (90, 3000, 64), (70, 2500, 128),
                                       (40, 2000, 256), (1, 2000, 256)])
def test_small_weights_of_an_fp16_cache(pkg, dev, new, n, dim, below, spread, out_code, whole):
    """Weights are rounded to fp16's 11 bits, by 2^-11 of each (with fp32 output by
    2^-22 of each), also those of keys that the largest outweighs by e^20.  Only keys
    that share a tile of 64 with the sink meet the end of fp16's range: half of its
    smallest step, 2^-25, where the sink's own weight is held as 2^7 (fp32: 2^14)."""
    print("[gpu case] small weights", new, n, dim, below, spread, NAME[out_code], whole, flush=True)
    c, q = _sink(new, n, dim, F16, below, spread)
    near, far = (2.0 ** -22, 2.0 ** -39) if out_code == F32 else (2.0 ** -11, 2.0 ** -32)
    beside = 63 / (n - new) * far * math.exp(below)
    want, bound = _bound(c, q, out_code, near + 2 * beside)
    got = _run(pkg, c, q, 1.0, out_code, **({"max_len": 0} if whole else {}))
    err = (got.double() - want).abs()
    print(f"[parity] attn: worst error {(err / bound).max().item():.3f} of its bound", flush=True)
    assert torch.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("new,n,dim", [(1, 700, 128), (1, 3000, 64), (60, 400, 128), (50, 300, 96),
                                       (40, 300, 256)])
def test_fp16_output_of_a_bf16_cache(pkg, dev, new, n, dim):
    """An output of 11 bits: the weights carry at least as many, and not bf16's 8.
    Two keys whose values differ by their sign: what a weight's rounding moves is not
    averaged away."""
    print("[gpu case] fp16 of bf16", new, n, dim, flush=True)
    c = Paged([new], [n], 1, dim, 16, BF16)
    k, v = (x.clone() for x in c.keys(0))
    k[:, 0, 0] = -60.0
    k[0, 0, 0], k[1, 0, 0] = 0.0, -0.4921875  # its weight lies between two bf16 numbers
    v[0], v[1] = 1.0, -1.0
    for p in range(n):
        c.put(0, p, k=k[p], v=v[p])
    q = torch.zeros((new, 2, dim), dtype=torch.bfloat16)
    q[:, :, 0] = 1
    want, _ = attention(c, q, 1.0)
    # sum p |v| / sum p is 1: half an fp16 step of each weight, and of the output; the
    # exponential's and the sums' 8 roundings of 2^-24
    bound = 2.0 ** -11 + want.abs() * 2.0 ** -11 + 8 * 2.0 ** -24
    err = (_run(pkg, c, q, 1.0, F16).double() - want).abs()
    assert torch.all(err <= bound), (err / bound).max()
    c2 = Paged([new], [n], 2, dim, 16, BF16)
    q2 = (torch.randn((new, 4, dim), generator=c2.g) * 1.5).bfloat16()
    want, bound = attention(c2, q2, 1 / math.sqrt(dim), 0, True, F16)
    err = (_run(pkg, c2, q2, 1 / math.sqrt(dim), F16).double() - want).abs()
    assert torch.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("code,out_code", [(F16, F16), (F16, F32), (BF16, BF16)])
@pytest.mark.parametrize("new,n,dim", [(1, 1500, 64), (80, 900, 128), (40, 600, 256)])
def test_maximum_that_falls_and_rises(pkg, dev, code, out_code, new, n, dim):
    """Tiles whose largest scores go down by up to 70 nats and up again, several
    times: what the sums are scaled by follows both ways, and no weight leaves the
    type's range."""
    print("[gpu case] falling and rising", new, n, dim, NAME[code], NAME[out_code], flush=True)
    c = Paged([new], [n], 1, dim, 16, code)
    k, _ = c.keys(0)
    pos = torch.arange(n)
    level = 35.0 * torch.cos(pos / 110.0) + torch.randn(n, generator=c.g)
    for p in range(n):
        row = k[p].float() * 0.05
        row[:, 0] = level[p]
        c.put(0, p, k=row.to(TORCH[code]))
    q = torch.zeros((new, 2, dim))
    q[:, :, 0] = 1
    q = q.to(TORCH[code])
    want, bound = attention(c, q, 1.0, 0, out_code == F32, out_code)
    err = (_run(pkg, c, q, 1.0, out_code).double() - want).abs()
    assert torch.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("out_code", [F16, F32])
@pytest.mark.parametrize("new,n,dim", [(1, 300, 64), (60, 300, 64), (50, 200, 128), (40, 200, 256)])
def test_fp16_scores_far_from_0(pkg, dev, new, n, dim, out_code):
    """Scores of 2^25, whose own step is 4, and a maximum that grows by one such step
    where it may or may not be followed: the weights' ratios are what the scores'
    differences say, and none leaves fp16's range."""
    print("[gpu case] scores of 2^25", new, n, dim, NAME[out_code], flush=True)
    c = Paged([new], [n], 1, dim, 16, F16)
    k, v = (x.clone() for x in c.keys(0))
    k[:, 0, 0], k[:, 0, 1] = 16384.0, 0.0
    k[n // 2:, 0, 1] = 4.0
    for p in range(n):
        c.put(0, p, k=k[p])
    q = torch.zeros((new, 2, dim), dtype=torch.float16)
    q[:, :, 0], q[:, :, 1] = 2048.0, 1.0
    for scale in (0.55, 0.9, 1.0, 1.3, 1.4, 1.44, 1.47, 1.5, 1.56, 1.6, 1.8, -1.0):
        want, _ = attention(c, q, scale)
        mean, _ = attention(_with_values(c, v.abs()), q, scale)
        # scores are exact, and what their products with c are off by is common to all
        # keys but for 2^-24 of their difference, 4; weights as stated, in numerator only
        # (the sum has them whole), and 8 sqrt(n) 2^-24 for the additions of either
        rel = (2.0 ** -22 if out_code == F32 else 2.0 ** -11) + 2.0 ** -24 * (40 + 16 * math.sqrt(n))
        bound = mean * rel + want.abs() * half_step(out_code) + 2.0 ** -25
        got = _run(pkg, c, q, scale, out_code)
        assert got.isfinite().all(), scale
        err = (got.double() - want).abs()
        assert torch.all(err <= bound), (scale, (err / bound).max())


def _with_values(c, v):
    """The cache with other values, for the oracle."""
    other = copy.copy(c)
    other.v = c.v.clone()
    for p in range(c.lens[0]):
        other.put(0, p, v=v[p])
    return other
