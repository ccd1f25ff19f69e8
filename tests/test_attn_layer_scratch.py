"""examples/attention_layer.py: what a captured step reserves is the most that one of
its calls takes."""
import importlib.util
import os
from types import SimpleNamespace

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location(
        "attention_layer", os.path.join(REPO, "examples", "attention_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _layer(lib):
    pkg = SimpleNamespace(gpu_lib=lambda: lib, BF16=30)
    return SimpleNamespace(pkg=pkg, qkv_rows=6144, width=4096, n_heads=32, dim=128, dtype=2,
                           cache="cache")


@pytest.mark.parametrize("most", ["attention", "qkv", "o"])
@pytest.mark.parametrize("prompt", [False, True])
def test_a_step_reserves_its_largest_need(most, prompt):
    batch = SimpleNamespace(n_tok=24)
    need = {"attention": 1000, "qkv": 2000, "o": 3000}
    need[most] = 1 << 30

    def gemm(dtype, x_type, n, rows, cols):
        assert prompt and (dtype, x_type, n) == (2, 30, 24)
        return need[{(6144, 4096): "qkv", (4096, 4096): "o"}[rows, cols]]

    def batched(dtype, n, rows, cols, accumulate):
        assert not prompt and (dtype, n) == (2, 24)
        return need[{(6144, 4096, 0): "qkv", (4096, 4096, 1): "o"}[rows, cols, accumulate]]

    def attn(cache, b, heads, window):
        assert (cache, b, heads, window) == ("cache", batch, 32, 0)
        return need["attention"]

    lib = SimpleNamespace(swamp_attn_paged_workspace=attn, swamp_qgemm_workspace=gemm,
                          swamp_qgemv_batched_workspace=batched)
    assert _example().AttentionLayer.scratch(_layer(lib), batch, prompt) == 1 << 30


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [1, 24, 64])
def test_captured_step_has_the_bits_of_an_eager_one(seqs):
    """With its scratch reserved, a captured step takes the paths of an eager one."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    print("[gpu case] captured step of", seqs, flush=True)
    ex = _example()
    length, page = 700, 32
    table = ex.page_tables(seqs, length, page)
    layer = ex.AttentionLayer(8, 2, 64, 1024, n_pages=int(table.numel()), page=page)
    layer.k.normal_()
    layer.v.normal_()
    first = torch.arange(seqs + 1, dtype=torch.int32).cuda()
    lens = torch.full((seqs,), length, dtype=torch.int32, device="cuda")
    batch, buf = layer.batch(first, lens, table, 1, length), layer.buffers(seqs, False)
    token = torch.randn((seqs, layer.width), device="cuda")
    eager = layer(token.clone(), batch, buf)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    need = layer.scratch(batch, prompt=False)
    if need:
        layer.pkg.workspace_reserve(side.cuda_stream, need)
    hidden = token.clone()
    with torch.cuda.graph(graph, stream=side):
        layer(hidden, batch, buf)
    for _ in range(3):
        hidden.copy_(token)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(hidden, eager)
        assert torch.equal(layer(token.clone(), batch, buf), eager)
