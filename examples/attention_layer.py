"""An attention layer on quantized weights, prompt and decoding, as an engine
runs it: RMSNorm, the fused QKV product, rotation and append to a paged cache,
attention over the cache, the O product and the residual.

    python examples/attention_layer.py [--tokens 2048] [--decode 64] [--seqs 4]

runs the prompts of a few sequences (4096 wide, 32 query and 8 cache heads of
128 dims, Q4_0 weights made at random), decodes further tokens of all of them
together from one captured graph, and prints the time of each part.
"""
import argparse
import importlib.util
import math
import os
import sys

import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def package():
    if "llamanyon_rs_amd" not in sys.modules:
        spec = importlib.util.spec_from_file_location(
            "llamanyon_rs_amd", os.path.join(REPO, "llamanyon.rs_amd", "__init__.py"))
        sys.modules["llamanyon_rs_amd"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["llamanyon_rs_amd"])
    return sys.modules["llamanyon_rs_amd"]


class AttentionLayer:
    """Weights, rotation and paged cache of one layer.  The caller's sequences own
    pages of the cache by their page tables."""

    def __init__(self, n_heads=32, n_kv=8, head_dim=128, width=4096, n_pages=1024, page=32, seed=1):
        self.pkg = pkg = package()
        pkg.init()
        self.n_heads, self.n_kv, self.dim, self.width, self.page = n_heads, n_kv, head_dim, width, page
        self.qkv_rows = (n_heads + 2 * n_kv) * head_dim
        self.dtype, sigma = pkg.Q4_0, 1.0 / math.sqrt(width)
        self.w_qkv = self._upload(pkg.synth_quantized(pkg.Q4_0, seed, sigma, self.qkv_rows, width))
        self.w_o = self._upload(pkg.synth_quantized(pkg.Q4_0, seed + 1, sigma, width,
                                                    n_heads * head_dim))
        self.norm = torch.ones(width, device="cuda")
        self.freqs = torch.from_numpy(pkg.rope_freqs(head_dim, 500000.0)).cuda()
        self.rope = pkg.Rope(self.freqs.data_ptr(), head_dim, pkg.ROPE_HALVES)
        shape = (n_pages, n_kv, page, head_dim)
        self.k = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        self.v = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        self.cache = pkg.KvPages(self.k.data_ptr(), self.v.data_ptr(), pkg.BF16, n_pages, page, n_kv,
                                 head_dim)

    @staticmethod
    def _upload(blocks):
        return torch.from_numpy(blocks).cuda()

    def batch(self, first, lens, table, max_new, max_len):
        """first, lens, table: int32 tensors on the device, kept by the caller."""
        return self.pkg.SeqBatch(lens.numel(), self._rows(first), max_new, max_len, first.data_ptr(),
                                 lens.data_ptr(), table.data_ptr(), table.shape[1])

    @staticmethod
    def _rows(first):
        return int(first[-1])

    def buffers(self, n_tok, prompt):
        """What a step of n_tok tokens writes on its way; kept from call to call."""
        act = torch.bfloat16 if prompt else torch.float32
        return {
            "prompt": prompt,
            "x": torch.empty((n_tok, self.width), dtype=act, device="cuda"),
            "qkv": torch.empty((n_tok, self.qkv_rows), device="cuda"),
            "q": torch.empty((n_tok, self.n_heads * self.dim), dtype=torch.bfloat16, device="cuda"),
            "o": torch.empty((n_tok, self.n_heads * self.dim), dtype=act, device="cuda"),
            "y": torch.empty((n_tok, self.width), device="cuda"),
        }

    def scratch(self, batch, prompt):
        """Bytes that the calls of a step take from the stream's scratch: what to reserve
        before a capture.  They run one after the other and share it, so the most of them."""
        lib, n = self.pkg.gpu_lib(), batch.n_tok
        shapes = ((self.qkv_rows, self.width, 0), (self.width, self.n_heads * self.dim, 1))
        needs = [lib.swamp_attn_paged_workspace(self.cache, batch, self.n_heads, 0)]
        for rows, cols, accumulate in shapes:
            needs.append(lib.swamp_qgemm_workspace(self.dtype, self.pkg.BF16, n, rows, cols) if prompt
                         else lib.swamp_qgemv_batched_workspace(self.dtype, n, rows, cols,
                                                                accumulate))
        return max(needs)

    def __call__(self, hidden, batch, buf):
        """hidden [tokens][width] fp32 += the layer's attention, on the current stream:
        the new tokens of `batch`, all of them (buffers(..., prompt=True)) or one a
        sequence."""
        pkg, s = self.pkg, torch.cuda.current_stream().cuda_stream
        n, h, kv, d = hidden.shape[0], self.n_heads, self.n_kv, self.dim
        act = pkg.BF16 if buf["prompt"] else pkg.F32
        pkg.rmsnorm_rows(hidden.data_ptr(), self.norm.data_ptr(), 1e-5, buf["x"].data_ptr(), act, n,
                         self.width, stream=s)
        qkv = buf["qkv"].data_ptr()
        if buf["prompt"]:
            pkg.qgemm(self.dtype, self.w_qkv.data_ptr(), self.w_qkv.numel(), buf["x"].data_ptr(),
                      act, qkv, n, self.qkv_rows, self.width, stream=s)
        else:
            pkg.qgemv_batched(self.dtype, self.w_qkv.data_ptr(), self.w_qkv.numel(),
                              buf["x"].data_ptr(), qkv, n, self.qkv_rows, self.width, stream=s)
        # q, k and v of a token lie side by side in its row of the product
        pkg.kv_append(self.cache, batch, self.rope, qkv, qkv + 4 * h * d, qkv + 4 * (h + kv) * d,
                      pkg.F32, buf["q"].data_ptr(), h, q_stride=self.qkv_rows,
                      k_stride=self.qkv_rows, v_stride=self.qkv_rows, stream=s)
        pkg.attn_paged(self.cache, batch, buf["q"].data_ptr(), h, 1 / math.sqrt(d),
                       buf["o"].data_ptr(), act, stream=s)
        if buf["prompt"]:
            pkg.qgemm(self.dtype, self.w_o.data_ptr(), self.w_o.numel(), buf["o"].data_ptr(), act,
                      buf["y"].data_ptr(), n, self.width, h * d, stream=s)
            hidden += buf["y"]
        else:
            pkg.qgemv_batched(self.dtype, self.w_o.data_ptr(), self.w_o.numel(), buf["o"].data_ptr(),
                              hidden.data_ptr(), n, self.width, h * d, accumulate=True, stream=s)
        return hidden


def page_tables(n_seq, length, page):
    """Pages for sequences of up to `length` tokens, dealt out in turn."""
    need = -(-length // page)
    return (torch.arange(need, dtype=torch.int32)[None, :] * n_seq
            + torch.arange(n_seq, dtype=torch.int32)[:, None]).cuda()


def timed(f, n=10):
    f()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    for _ in range(n):
        f()
    b.record()
    b.synchronize()
    return a.elapsed_time(b) / n * 1e3


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=2048, help="prompt of each sequence")
    ap.add_argument("--decode", type=int, default=64, help="tokens decoded after it")
    ap.add_argument("--seqs", type=int, default=4)
    a = ap.parse_args()
    n, t = a.seqs, a.tokens
    table = page_tables(n, t + a.decode, 32)
    layer = AttentionLayer(n_pages=int(table.numel()))

    # the prompts, together
    first = torch.arange(0, n * t + 1, t, dtype=torch.int32).cuda()
    lens = torch.full((n,), t, dtype=torch.int32, device="cuda")
    batch, buf = layer.batch(first, lens, table, t, t), layer.buffers(n * t, True)
    hidden = torch.randn((n * t, layer.width), device="cuda")
    us = timed(lambda: layer(hidden.clone(), batch, buf))
    print(f"prompt   {n} x {t} tokens: {us:9.1f} us, {n * t / us * 1e6:.3g} tokens/s a layer")

    # one token of each sequence a step, captured once: the lengths grow on the device
    first1 = torch.arange(n + 1, dtype=torch.int32).cuda()
    batch1, buf1 = layer.batch(first1, lens, table, 1, t + a.decode), layer.buffers(n, False)
    token = torch.randn((n, layer.width), device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    layer.pkg.workspace_reserve(side.cuda_stream, layer.scratch(batch1, prompt=False))
    with torch.cuda.graph(graph, stream=side):
        lens += 1
        layer(token, batch1, buf1)
    lens.fill_(t)
    torch.cuda.synchronize()
    us = timed(graph.replay, max(1, a.decode - 1))
    print(f"decode   {n} x 1 token after {t}: {us:9.1f} us a step")


if __name__ == "__main__":
    main()
