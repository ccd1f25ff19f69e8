"""swamp_beam_select on the GPU against a sequence after the other in 64 bits.

Tokens and parents have to be equal: totals are 64-bit on both sides and differ by about
1e-15 of themselves, random ones by far more, and equal logits of one beam by nothing.
Scores: one rounding to fp32, 2^-24 of the score, and 1e-13 for the 64-bit sums."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = 0, 1, 30
TORCH = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
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


def stream():
    return torch.cuda.current_stream().cuda_stream


def reference(logits, score, done, n, b, k, eos):
    """Parents, tokens, 64-bit scores, done of each sequence's k best."""
    v = logits.shape[1]
    out = []
    for s in range(n):
        found = []
        for r in range(s * b, (s + 1) * b):
            sc = score[r].double().item()
            if not math.isfinite(sc):
                continue
            if done is not None and done[r]:
                found.append((torch.tensor([sc], dtype=torch.float64), torch.tensor([eos]), r))
                continue
            x = logits[r].double()
            lse = torch.logsumexp(x, 0)
            if not math.isfinite(lse.item()):
                continue
            t = torch.nonzero(x > -INF)[:, 0]
            best = torch.sort(x[t], descending=True, stable=True)
            t = t[best.indices[:k]]
            found.append((sc + (x[t] - lse), t, r))
        rows = []
        if found:
            total = torch.cat([f[0] for f in found])
            token = torch.cat([f[1] for f in found])
            row = torch.cat([torch.full((f[0].numel(),), f[2]) for f in found])
            order = torch.sort(total, descending=True, stable=True).indices[:k]
            for i in order.tolist():
                ended = int(token[i]) == eos or (done is not None and bool(done[row[i]]))
                rows.append((int(row[i]), int(token[i]), float(total[i]), int(ended)))
        out += rows + [(-1, -1, -INF, 0)] * (k - len(rows))
    return out


def select(pkg, logits, t, score, done, n, b, k, eos, stride=0, want_done=True):
    v = stride or logits.shape[1]
    dl, ds = logits.cuda(), score.cuda()
    dd = done.cuda() if done is not None else None
    parent = torch.full((n * k,), 77, dtype=torch.int32, device="cuda")
    token, out_done = parent.clone(), parent.clone()
    out = torch.full((n * k,), 77.0, device="cuda")
    pkg.beam_select(pkg.BeamSpec(n, b, v, k, eos), dl.data_ptr(), t, ds.data_ptr(),
                    parent.data_ptr(), token.data_ptr(), out.data_ptr(),
                    d_done=dd.data_ptr() if dd is not None else 0,
                    d_out_done=out_done.data_ptr() if want_done else 0,
                    logits_stride=logits.shape[1] if stride else 0, stream=stream())
    torch.cuda.synchronize()
    return parent.tolist(), token.tolist(), out.tolist(), out_done.tolist()


def check(got, want):
    parent, token, score, done = got
    assert parent == [w[0] for w in want]
    assert token == [w[1] for w in want]
    assert done == [w[3] for w in want]
    for g, w in zip(score, want):
        assert g == w[2] or abs(g - w[2]) <= 2.0 ** -24 * abs(w[2]) * (1 + 1e-6) + 1e-13


def inputs(n, b, v, t, seed=0):
    g = torch.Generator().manual_seed(n * 1000 + b * 100 + v + seed)
    logits = (torch.randn((n * b, v), generator=g) * 3).to(TORCH[t])
    score = -5 * torch.rand(n * b, generator=g)
    return logits, score, g


SHAPES = [  # sequences, beams, vocabulary, best
    (1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 2, 4), (3, 4, 100, 4), (1, 2, 4096, 64), (2, 5, 4097, 10),
    (5, 1, 32000, 1), (1, 4, 50257, 8), (3, 8, 8191, 16), (1, 64, 300, 64), (2, 64, 9000, 64),
    (17, 2, 1000, 3), (1, 2, 262145, 33), (70, 4, 640, 4), (1, 1, 1 << 20, 64), (1, 3, 12288, 63),
]


@pytest.mark.parametrize("n,b,v,k", SHAPES)
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_select(pkg, dev, n, b, v, k, t):
    say("select", n, b, v, k, t)
    logits, score, g = inputs(n, b, v, t)
    done = (torch.rand(n * b, generator=g) < 0.3).to(torch.int32)
    for d, eos in ((None, -1), (None, v - 1), (done, 0)):
        check(select(pkg, logits, t, score, d, n, b, k, eos),
              reference(logits, score, d, n, b, k, eos))


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("v,gap", [(1001, 3), (4100, 1), (9001, 8)])
def test_rows_with_gaps(pkg, dev, t, v, gap):
    """Rows that begin at any element; what lies between them is not read as a token."""
    say("gaps", t, v, gap)
    logits, score, _ = inputs(2, 3, v + gap, t)
    logits[:, v:] = 1000.0
    got = select(pkg, logits, t, score, None, 2, 3, 6, 7, stride=v)
    check(got, reference(logits[:, :v], score, None, 2, 3, 6, 7))


@pytest.mark.parametrize("n,b,v,k", [(2, 4, 5000, 8), (1, 3, 9000, 64), (1, 64, 4100, 64),
                                     (1, 1, 20000, 33)])
def test_equal_logits(pkg, dev, n, b, v, k):
    """All logits equal: the first tokens of the first beam of the largest score; equal
    scores too: by beam, then token.  -0 equals 0."""
    say("equal", n, b, v, k)
    logits = torch.zeros((n * b, v))
    logits[:, 1::2] = -0.0
    score = torch.zeros(n * b)
    check(select(pkg, logits, F32, score, None, n, b, k, -1),
          [(s * b, i, -math.log(v), 0) for s in range(n) for i in range(k)])
    score = -torch.arange(n * b).float() % b
    check(select(pkg, logits, F32, score, None, n, b, k, -1),
          reference(logits, score, None, n, b, k, -1))


@pytest.mark.parametrize("k", [1, 5, 64])
def test_few_values(pkg, dev, k):
    """Logits of a handful of values, sorted rows, and all large ones in one place."""
    say("few values", k)
    g = torch.Generator().manual_seed(k)
    for make in (lambda: torch.randint(0, 3, (4, 10000), generator=g).float(),
                 lambda: torch.linspace(5, -5, 10000).repeat(4, 1),
                 lambda: torch.linspace(-5, 5, 10000).repeat(4, 1),
                 lambda: torch.where((torch.arange(10000) // 16) % 256 == 3, 4.0,
                                     torch.randn((4, 10000), generator=g)),
                 lambda: torch.where(torch.arange(10000) % 16 == 3, 4.0,
                                     torch.rand((4, 10000), generator=g))):
        logits = make()
        score = -torch.rand(4, generator=g)
        check(select(pkg, logits, F32, score, None, 2, 2, k, 3),
              reference(logits, score, None, 2, 2, k, 3))


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_masks_and_limits(pkg, dev, t):
    """Masked tokens, the type's lowest value, rows of nothing, infinities, NaN, beams
    that are dead or have ended."""
    say("masks", t)
    n, b, v, k = 7, 4, 6000, 12
    logits, score, g = inputs(n, b, v, t)
    low = torch.finfo(TORCH[t]).min
    logits[0:4, 5:] = -INF               # 5 tokens a beam
    logits[4:8] = -INF                   # none
    logits[8, :] = -INF
    logits[8, 4500] = 1.0                # one
    logits[9, :] = low                   # all at the lowest value
    logits[10, 100] = INF                # the row is spoilt
    logits[11, 5999] = math.nan
    logits[12:16, ::2] = low
    score[16] = -INF
    score[17] = math.nan
    score[18] = INF
    done = torch.zeros(n * b, dtype=torch.int32)
    done[20:24] = torch.tensor([1, 5, -1, 0], dtype=torch.int32)
    logits[20] = math.nan                # not read
    score[24:28] = -INF                  # nobody
    for d, eos in ((None, 3), (done, 4500)):
        check(select(pkg, logits, t, score, d, n, b, k, eos),
              reference(logits, score, d, n, b, k, eos))


def test_far_apart(pkg, dev):
    """Logits up to fp32's end, and scores that agree to 32 bits."""
    say("far apart")
    logits = torch.zeros((4, 9000))
    logits[0, 17] = 3e38
    logits[0, 8000] = -3e38
    logits[1] = -3e38
    logits[1, 5000] = -2.9e38
    logits[2:] = torch.randn((1, 9000), generator=torch.Generator().manual_seed(1))
    logits[3, 77] += 1e-6                # its lse a little larger
    score = torch.tensor([-1.0, -1.0, -2.0, -2.0])
    check(select(pkg, logits, F32, score, None, 1, 4, 20, -1),
          reference(logits, score, None, 1, 4, 20, -1))


def test_in_place_and_replayed(pkg, dev):
    """Scores and ended beams updated in place by a captured call, step after step; without
    scratch reserved the capture is refused."""
    say("in place, replayed")
    n, b, v, eos = 3, 4, 5000, 9
    logits, score, g = inputs(n, b, v, F32)
    dl, ds = logits.cuda(), score.cuda()
    done = torch.zeros(n * b, dtype=torch.int32, device=dev)
    parent, token = torch.zeros_like(done), torch.zeros_like(done)
    spec = pkg.BeamSpec(n, b, v, b, eos)

    def call(s):
        pkg.beam_select(spec, dl.data_ptr(), F32, ds.data_ptr(), parent.data_ptr(),
                        token.data_ptr(), ds.data_ptr(), d_done=done.data_ptr(),
                        d_out_done=done.data_ptr(), stream=s)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with pytest.raises(pkg.GpuError) as e:
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            dl.add_(0.0)
            call(side.cuda_stream)
    assert e.value.code == pkg.EWORKSPACE
    torch.cuda.synchronize()
    pkg.workspace_reserve(side.cuda_stream, pkg.gpu_lib().swamp_beam_select_workspace(spec))
    with torch.cuda.graph(graph, stream=side):
        call(side.cuda_stream)
    ref_score, ref_done = score.clone(), torch.zeros(n * b, dtype=torch.int32)
    for step in range(5):
        x = torch.randn((n * b, v), generator=g) * 3
        x[step % (n * b), eos] = 30.0
        dl.copy_(x.cuda())
        graph.replay()
        torch.cuda.synchronize()
        want = reference(x, ref_score, ref_done, n, b, b, eos)
        check((parent.tolist(), token.tolist(), ds.tolist(), done.tolist()), want)
        ref_score, ref_done = ds.cpu(), done.cpu()
    assert ref_done.any()


def test_two_streams(pkg, dev):
    """Two selections at once, each with its stream's scratch."""
    say("two streams")
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    work = []
    for i, side in enumerate(sides):
        logits, score, _ = inputs(4, 4, 30000, F32, seed=i)
        dl, ds = logits.cuda(), score.cuda()
        out = [torch.zeros(32, dtype=torch.int32, device=dev) for _ in range(3)]
        val = torch.zeros(32, device=dev)
        work.append((logits, score, dl, ds, out, val))
    torch.cuda.synchronize()
    spec = pkg.BeamSpec(4, 4, 30000, 8, 2)
    for _ in range(5):
        for side, (_, _, dl, ds, out, val) in zip(sides, work):
            pkg.beam_select(spec, dl.data_ptr(), F32, ds.data_ptr(), out[0].data_ptr(),
                            out[1].data_ptr(), val.data_ptr(), d_out_done=out[2].data_ptr(),
                            stream=side.cuda_stream)
    torch.cuda.synchronize()
    for logits, score, _, _, out, val in work:
        check((out[0].tolist(), out[1].tolist(), val.tolist(), out[2].tolist()),
              reference(logits, score, None, 4, 4, 8, 2))
