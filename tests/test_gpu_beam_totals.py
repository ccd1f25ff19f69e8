"""swamp_beam_select's totals where 64 bits are few: totals that agree in all of them (by
beam, then the larger logit, then the lower token, whatever the number of best, of chunks and
of tokens that reach the bound), and rows whose largest logit is far from 0.

Parents and tokens have to be equal: the rows are made so that totals are far apart or the
same by the formula, not by the last bit of a sum.  Scores: one rounding to fp32, 2^-24 of the
score, and 1e-13 for the 64-bit sums (score, x - top and the log of the sum, each of them in
64 bits and small where the total is).
"""
import math

import pytest
import torch

from test_gpu_beam import BF16, F16, F32, TORCH, check, select

pytestmark = pytest.mark.gpu
INF = math.inf


@pytest.fixture(scope="module")
def dev(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()
    pkg.init()
    return torch.device("cuda")


def say(*a):
    print("[gpu case]", *a, flush=True)


def plain(logits, score, n, b, k, eos=-1, done=None):
    """(parent, token, 64-bit score, done) of each sequence's k best."""
    out = []
    for s in range(n):
        found = []
        for r in range(s * b, (s + 1) * b):
            x = logits[r].double()
            top = x.max()
            if not math.isfinite(score[r]):
                continue
            if done is not None and done[r]:
                found.append((-score[r].double().item(), r - s * b, 0.0, eos))
                continue
            if not math.isfinite(top):
                continue
            total = score[r].double() + ((x - top) - torch.exp(x - top).sum().log())
            token = torch.nonzero(x > -INF)[:, 0]
            token = token[torch.sort(x[token], descending=True, stable=True).indices[:k]]
            found += [(-t, r - s * b, -l, v) for t, l, v in
                      zip(total[token].tolist(), x[token].tolist(), token.tolist())]
        found.sort()
        rows = [(s * b + beam, v, -t, int(v == eos or (done is not None and bool(done[s * b + beam]))))
                for t, beam, _, v in found[:k]]
        out += rows + [(-1, -1, -INF, 0)] * (k - len(rows))
    return out


@pytest.mark.parametrize("v,far", [(100, 9), (4096, 4000), (9000, 5000), (70000, 69999)])
def test_logits_below_the_last_bit(pkg, dev, v, far):
    """Two logits that no total of 64 bits tells apart, in one chunk and in two: the larger
    one first, alone as well as before the other."""
    say("below the last bit", v, far)
    logits = torch.full((1, v), -5.0)
    logits[0, 5], logits[0, far] = 0.0, 1e-20
    score = torch.tensor([-1.0])
    for k, first in ((1, [far]), (2, [far, 5]), (3, [far, 5, 0]), (64, [far, 5] + list(range(5)))):
        got = select(pkg, logits, F32, score, None, 1, 1, k, -1)
        want = plain(logits, score, 1, 1, k)
        assert [w[1] for w in want[:len(first)]] == first
        check(got, want)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n,b,v", [(1, 1, 60), (2, 3, 4097), (1, 4, 20000), (1, 64, 300), (1, 20, 9000)])
def test_one_logit_forced(pkg, dev, t, n, b, v):
    """A logit of 1e18 leaves every other of its row at one total: they follow by logit."""
    say("one logit forced", t, n, b, v)
    g = torch.Generator().manual_seed(v + b)
    logits = torch.randn((n * b, v), generator=g) * 3
    logits[torch.arange(n * b), torch.randint(0, v, (n * b,), generator=g)] = 1e18
    logits = logits.to(TORCH[t])
    score = -torch.rand(n * b, generator=g)
    last = None
    for k in (64, 33, 3, 2, 1):
        want = plain(logits, score, n, b, k)
        got = select(pkg, logits, t, score, None, n, b, k, -1)
        check(got, want)
        tokens = torch.tensor(got[1]).view(n, k)
        assert last is None or torch.equal(tokens, last[:, :k])
        last = tokens


@pytest.mark.parametrize("b,v", [(64, 300), (40, 9000), (3, 90000)])
def test_more_equal_totals_than_are_listed(pkg, dev, b, v):
    """All totals of all beams equal, 64 tokens a list: more than a workgroup ranks at once
    (64 x 64, 40 x 3 x 64) and less.  Logits that differ below the last bit keep their order
    within a beam, and beams theirs."""
    say("more than are listed", b, v)
    logits = torch.zeros((b, v))
    g = torch.Generator().manual_seed(b)
    for r in range(b):
        logits[r, torch.randperm(v, generator=g)[:5]] = torch.arange(1, 6) * 1e-20
    score = torch.zeros(b)
    for k in (1, 4, 64):
        check(select(pkg, logits, F32, score, None, 1, b, k, -1), plain(logits, score, 1, b, k))
    # a beam of three tokens comes first; the others' scores agree to 32 bits, not to 64
    logits[1] = -INF
    logits[1, 7:10] = torch.tensor([0.0, 2e-20, 1e-20])
    score = torch.randperm(b, generator=g) * 1e-9
    score[1] = 5.0
    want = plain(logits, score, 1, b, 64)
    assert [w[:2] for w in want[:3]] == [(1, 8), (1, 9), (1, 7)]
    check(select(pkg, logits, F32, score, None, 1, b, 64, -1), want)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("v", [1, 60, 6000, 50257])
def test_row_far_from_zero(pkg, dev, t, v):
    """Rows at the type's lowest value, at -1e15 and at 1e15 throughout (60000 in fp16): every
    token scores its beam's score less log(vocabulary), which 64 bits would lose beside the
    row's largest logit, and stands behind those of a beam of the same score that has a choice."""
    say("far from zero", t, v)
    kind = TORCH[t]
    for value in (torch.finfo(kind).min, -1e15, 1e15):
        value = max(min(value, 60000.0), torch.finfo(kind).min) if t == F16 else value
        logits = torch.full((4, v), value, dtype=kind)
        logits[1] = 0.0
        logits[1, v // 2] = 20.0
        score = torch.tensor([-1.0, -1.0, -2.0, -1.5])
        for k in (1, 5, 64):
            want = plain(logits, score, 2, 2, k)
            if v > 1:
                assert want[0][:2] == (1, v // 2) and abs(want[k][2] + 1.5 + math.log(v)) < 1e-9
            check(select(pkg, logits, t, score, None, 2, 2, k, -1), want)


@pytest.mark.parametrize("v", [300, 9000])
def test_row_far_from_zero_with_others(pkg, dev, v):
    """Differences of a few units at 1e7 and at -3e9 (one step of fp32: 1 and 256)."""
    say("far from zero, with others", v)
    g = torch.Generator().manual_seed(v)
    logits = torch.randint(0, 12, (4, v), generator=g).float() + 1e7
    logits[2:] = torch.randint(0, 2, (2, v), generator=g) * 256.0 - 3e9
    score = -torch.rand(4, generator=g)
    for k in (3, 64):
        check(select(pkg, logits, F32, score, None, 1, 4, k, -1), plain(logits, score, 1, 4, k))


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("v,every", [(60, 2), (64, 63), (9000, 2), (9000, 3), (9000, 1000), (50257, 7)])
def test_lowest_beside_masked(pkg, dev, t, v, every):
    """A row of the type's lowest value and -infinity: the masked tokens count for nothing in
    its sum, in their wave, their chunk and the row."""
    say("lowest beside masked", t, v, every)
    low = torch.finfo(TORCH[t]).min
    logits = torch.full((4, v), -INF, dtype=TORCH[t])
    logits[0, ::every] = low
    logits[1, every - 1::every] = low
    logits[2, v - 1] = low
    logits[3, : v // 2] = low
    score = torch.tensor([-1.0, -2.0, -9.0, -3.0])
    for k in (1, 8, 64):
        want = plain(logits, score, 1, 4, k)
        left = (logits[0] == low).sum().item()
        assert abs(want[0][2] + 1.0 + math.log(left)) < 1e-9 or left > 600
        check(select(pkg, logits, t, score, None, 1, 4, k, -1), want)


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_masks_limits_and_ended_beams(pkg, dev, t):
    """Masked tokens, rows of the lowest value beside a row of one token, infinities, NaN, beams
    that are dead or have ended."""
    say("masks, limits, ended", t)
    n, b, v, k = 7, 4, 6000, 12
    g = torch.Generator().manual_seed(t)
    logits = (torch.randn((n * b, v), generator=g) * 3).to(TORCH[t])
    score = -5 * torch.rand(n * b, generator=g)
    low = torch.finfo(TORCH[t]).min
    logits[0:4, 5:] = -INF               # 5 tokens a beam
    logits[4:9] = -INF                   # none
    logits[8, 4500] = 1.0                # one
    logits[9] = low                      # all at the lowest value
    logits[10, 100] = INF                # the row is spoilt
    logits[11, 5999] = math.nan
    logits[12:16, ::2] = low
    score[8], score[9] = -3.0, -3.0
    score[16:19] = torch.tensor([-INF, math.nan, INF])
    done = torch.zeros(n * b, dtype=torch.int32)
    done[20:24] = torch.tensor([1, 5, -1, 0], dtype=torch.int32)
    logits[20] = math.nan                # not read
    score[24:28] = -INF                  # nobody
    for d, eos in ((None, 3), (done, 4500)):
        want = plain(logits, score, n, b, k, eos, d)
        assert want[2 * k][:2] == (8, 4500) and want[2 * k + 1][:2] == (9, 0)
        assert abs(want[2 * k + 1][2] + 3.0 + math.log(v)) < 1e-9
        check(select(pkg, logits, t, score, d, n, b, k, eos), want)
