"""examples/attention_layer.py on the GPU: a layer's prompt, its chunks and its
decoded tokens against the layer in 64 bits on the CPU."""
import importlib.util
import math
import os

import pytest
import torch

from paged_reference import turn

pytestmark = pytest.mark.gpu
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

HEADS, KV, DIM, WIDTH, PAGE = 8, 2, 64, 512, 16

# Relative error of the layer's output, in the 2-norm: at most five values on the
# way to it are rounded to bf16 (the normalized row, k, v, the weights, the
# attention's output), each by at most half a step of 2^-8 relative; q's rounding
# and k's move scores, whose own size is about 1, by as much.
TOLERANCE = 6 * 2.0 ** -8


@pytest.fixture(scope="module")
def example(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    spec = importlib.util.spec_from_file_location(
        "attention_layer", os.path.join(REPO, "examples", "attention_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _weights(pkg, raw, rows, cols):
    out = torch.empty(rows * cols, device="cuda")
    pkg.qdequant(pkg.Q4_0, raw.data_ptr(), raw.numel(), out.data_ptr(), rows * cols)
    torch.cuda.synchronize()
    return out.cpu().double().view(rows, cols)


def _layer(layer, pkg, hidden):
    """The layer over one whole sequence, in 64 bits."""
    w = _weights(pkg, layer.w_qkv, layer.qkv_rows, WIDTH)
    wo = _weights(pkg, layer.w_o, WIDTH, HEADS * DIM)
    x = hidden.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)
    y = (x @ w.T).view(-1, HEADS + 2 * KV, DIM)
    pos = torch.arange(y.shape[0])
    qk = turn(y[:, :HEADS + KV], pos, layer.freqs.cpu(), DIM, True)
    q, k, v = qk[:, :HEADS], qk[:, HEADS:], y[:, HEADS + KV:]
    k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, v))
    s = (q.transpose(0, 1) @ k.permute(1, 2, 0)) / math.sqrt(DIM)
    s = s.masked_fill(pos[None, :, None] < pos[None, None, :], -math.inf)
    o = (torch.softmax(s, -1) @ v.transpose(0, 1)).transpose(0, 1).reshape(-1, HEADS * DIM)
    return o @ wo.T


def _error(got, hidden, want):
    return ((got.double() - hidden.double() - want).norm(dim=-1) / want.norm(dim=-1)).max().item()


@pytest.mark.parametrize("prompt", [1, 37, 200])
def test_prompt_and_decoding(example, pkg, prompt):
    """Two sequences: their prompts in one call, then ten tokens each in steps of
    both together; every row against the whole layer."""
    print("[gpu case] layer, prompt of", prompt, flush=True)
    n, more = 2, 10
    total = prompt + more
    layer = example.AttentionLayer(HEADS, KV, DIM, WIDTH, n_pages=64, page=PAGE)
    g = torch.Generator().manual_seed(3)
    hidden = torch.randn((n, total, WIDTH), generator=g)
    want = torch.stack([_layer(layer, pkg, h) for h in hidden])
    table = example.page_tables(n, total, PAGE)
    lens = torch.full((n,), prompt, dtype=torch.int32, device="cuda")
    first = torch.arange(0, n * prompt + 1, prompt, dtype=torch.int32).cuda()
    rows = hidden[:, :prompt].reshape(-1, WIDTH).contiguous()
    batch = layer.batch(first, lens, table, prompt, prompt)
    got = layer(rows.cuda(), batch, layer.buffers(n * prompt, True)).cpu()
    assert _error(got, rows, want[:, :prompt].reshape(-1, WIDTH)) <= TOLERANCE
    first1 = torch.arange(n + 1, dtype=torch.int32).cuda()
    batch1, buf = layer.batch(first1, lens, table, 1, total), layer.buffers(n, False)
    for i in range(prompt, total):
        lens += 1
        token = hidden[:, i].contiguous()
        got = layer(token.cuda(), batch1, buf).cpu()
        assert _error(got, token, want[:, i]) <= TOLERANCE, i


def test_chunks_beside_decoding(example, pkg):
    """A prompt in three ragged chunks, beside a sequence that decodes."""
    print("[gpu case] layer, chunks", flush=True)
    layer = example.AttentionLayer(HEADS, KV, DIM, WIDTH, n_pages=64, page=PAGE)
    g = torch.Generator().manual_seed(4)
    a, b = torch.randn((150, WIDTH), generator=g), torch.randn((3, WIDTH), generator=g)
    want_a, want_b = _layer(layer, pkg, a), _layer(layer, pkg, b)
    table = example.page_tables(2, 150, PAGE)
    at = 0
    for i, size in enumerate((71, 1, 78)):
        lens = torch.tensor([at + size, i + 1], dtype=torch.int32).cuda()
        first = torch.tensor([0, size, size + 1], dtype=torch.int32).cuda()
        rows = torch.cat((a[at:at + size], b[i:i + 1]))
        batch = layer.batch(first, lens, table, size, 150)
        got = layer(rows.cuda(), batch, layer.buffers(size + 1, True)).cpu()
        want = torch.cat((want_a[at:at + size], want_b[i:i + 1]))
        assert _error(got, rows, want) <= TOLERANCE
        at += size
