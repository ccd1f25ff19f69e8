"""Attention between the QKV and the O product, as timed cases: the rotation of
positions, the paged cache's append and the attention that reads the cache.

A case is one pass through one public entry point.  Its ops:

  rope    rows of heads turned by their positions: swamp_rope
  append  the projections' q, k, v of new tokens: q turned, k turned and v
          written to the cache's pages: swamp_kv_append
  attn    the new tokens' attention over the paged cache: swamp_attn_paged

Lengths: `seqs` sequences; the first has `len` tokens in the cache, the others
(where `ragged`) from a tenth of it up.  `new` of them are new, all sequences
alike ("new"), or of the first only while the others decode one token
("mixed").  An `idle` batch has one slot without new tokens.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _package():
    if "llamanyon_rs_amd" not in sys.modules:
        path = os.path.join(ROOT, "llamanyon.rs_amd", "__init__.py")
        spec = importlib.util.spec_from_file_location("llamanyon_rs_amd", path)
        mod = importlib.util.module_from_spec(spec)
        sys.modules["llamanyon_rs_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["llamanyon_rs_amd"]


# ------------------------------------------------------------------ the cases

def _attn(name, seqs, new, length, heads, kv, dim, page, dtype, out, **more):
    case = {"op": "attn", "seqs": seqs, "new": new, "len": length, "heads": heads, "kv": kv,
            "dim": dim, "page": page, "dtype": dtype, "out": out, "ragged": False, "mixed": False,
            "idle": False, "window": 0}
    case.update(more)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # The smallest call: one token's query heads of an 8B model.
        {"name": "rope_decode", "op": "rope", "tokens": 1, "heads": 32, "dim": 128, "rot": 128,
         "layout": "pairs", "scaling": "none", "start": 1000, "x": "f32", "out": "f32"},
        # A chunk of a prompt far into a context that was extended eightfold.
        {"name": "rope_prompt_far", "op": "rope", "tokens": 4096, "heads": 32, "dim": 128,
         "rot": 128, "layout": "halves", "scaling": "yarn", "start": 100000, "x": "bf16",
         "out": "bf16"},
        # A model that turns part of each head, a ragged number of tokens.
        {"name": "rope_partial", "op": "rope", "tokens": 777, "heads": 20, "dim": 80, "rot": 32,
         "layout": "halves", "scaling": "linear", "start": 0, "x": "f32", "out": "f16"},
        # Continuous batching: 16 sequences decode together.
        {"name": "append_decode16", "op": "append", "seqs": 16, "new": 1, "len": 2000,
         "heads": 32, "kv": 8, "dim": 128, "rot": 128, "layout": "pairs", "page": 32,
         "x": "f32", "dtype": "f16", "ragged": True, "mixed": False, "idle": False},
        # Four ragged prompts of an 8B model handed over together.
        {"name": "append_prompts", "op": "append", "seqs": 4, "new": 1999, "len": 1999,
         "heads": 32, "kv": 8, "dim": 128, "rot": 128, "layout": "halves", "page": 16,
         "x": "f32", "dtype": "bf16", "ragged": True, "mixed": False, "idle": False},
        # One chat decodes: a short context, latency counts.
        _attn("attn_decode_short", 1, 1, 700, 32, 8, 128, 32, "bf16", "f32"),
        # One long document: 131072 tokens of cache for one token.
        _attn("attn_decode_long", 1, 1, 131072, 32, 8, 128, 64, "bf16", "f32"),
        # A full serving batch, ragged, an idle slot, 70B heads.
        _attn("attn_decode_batch", 64, 1, 8192, 64, 8, 128, 16, "f16", "bf16", ragged=True,
              idle=True),
        # Speculative verify: five tokens of each of eight sequences.
        _attn("attn_verify", 8, 5, 4001, 32, 8, 128, 32, "bf16", "f32", ragged=True),
        # Chunked prefill: 512 tokens on top of a long context.
        _attn("attn_chunk", 1, 512, 16384, 32, 8, 128, 64, "bf16", "bf16"),
        # One chunk beside 15 decoding sequences, small heads, a sliding window.
        _attn("attn_mixed_window", 16, 509, 5000, 32, 4, 64, 16, "f16", "f16", ragged=True,
              mixed=True, window=2048),
        # A prompt of 4096 tokens through a 70B layer.
        _attn("attn_prompt", 1, 4096, 4096, 64, 8, 128, 64, "bf16", "bf16"),
    ]


def _span(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["rope", "append", "attn", "attn", "attn", "attn"])
    dim = rng.choice([64, 128, 128, 80, 96, 256])
    kv = rng.choice([1, 2, 4, 5, 8])
    heads = kv * rng.choice([1, 2, 4, 7, 8])
    layout = rng.choice(["pairs", "halves"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "rope":
        return {"op": op, "tokens": _span(rng, 1, 4096), "heads": heads, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2, dim // 4]), "layout": layout,
                "scaling": rng.choice(["none", "linear", "yarn", "divisors"]),
                "start": _span(rng, 1, 1000000), "x": rng.choice(["f32", "f16", "bf16"]),
                "out": rng.choice(["f32", "f16", "bf16"])}
    seqs = _span(rng, 1, 64)
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "append":
        length = _span(rng, 1, 8000 // max(1, seqs // 2))
        new = 1 if rng.random() < 0.5 else _span(rng, 1, length)
        return {"op": op, "seqs": seqs, "new": new, "len": length, "heads": heads, "kv": kv,
                "dim": dim, "rot": rng.choice([dim, dim, dim // 2]), "layout": layout,
                "page": page, "x": rng.choice(["f32", "f32", "bf16"]), "dtype": dtype,
                "ragged": True, "mixed": rng.random() < 0.2, "idle": rng.random() < 0.2}
    kind = rng.choice(["decode", "few", "chunk", "prompt"])
    if kind in ("decode", "few"):
        new = 1 if kind == "decode" else _span(rng, 2, 16)
        length = max(new, _span(rng, 1, min(60000, 400000 // seqs)))
    else:
        seqs = min(seqs, 8)
        length = _span(rng, 64, 16384 // seqs if kind == "chunk" else 4096 // seqs)
        new = length if kind == "prompt" else _span(rng, 17, min(length, 1024))
    case = _attn(None, seqs, new, length, heads, kv, dim, page, dtype,
                 rng.choice(["f32", dtype, "bf16"]), ragged=seqs > 1,
                 mixed=kind == "chunk" and rng.random() < 0.5, idle=rng.random() < 0.2,
                 window=rng.choice([0, 0, 0, _span(rng, 16, 4096)]))
    while work(case)["flops"] > 2.5e11 or work(case)["bytes"] > 1e9:
        case["len"] = case["len"] * 3 // 4
        case["new"] = min(case["new"], case["len"])
    return case


def _lengths(case):
    """(new tokens, cached tokens) of each sequence."""
    n = case["seqs"]
    lens, news = [], []
    for i in range(n):
        part = 1.0 - 0.9 * ((i * 0.6180339887498949) % 1.0) if case["ragged"] else 1.0
        length = max(1, int(case["len"] * part))
        new = case["new"] if not case["mixed"] or i == 0 else 1
        if case["idle"] and n > 1 and i == n - 1:
            new = 0
        lens.append(length)
        news.append(min(new, length))
    return news, lens


# ----------------------------------------------------------------- the inputs

def _freqs(n_rot, scaling, base=500000.0):
    """Radians per position of each pair, in 64 bits, and the magnitude."""
    i = torch.arange(n_rot // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / n_rot)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "divisors":  # a table of a file: low frequencies slowed down
        return f / torch.clamp(i - n_rot / 8, 1.0, 8.0), 1.0
    if scaling == "yarn":
        factor, ctx, fast, slow = 8.0, 8192, 32.0, 1.0
        at = [n_rot * math.log(ctx / (b * 2 * math.pi)) / (2 * math.log(base))
              for b in (fast, slow)]
        lo, hi = max(0, math.floor(at[0])), min(n_rot - 1, math.ceil(at[1]))
        ramp = torch.clamp((i - lo) / max(0.001, hi - lo), 0.0, 1.0)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _randn(g, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * sigma).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    st = {"case": case}
    if case["op"] == "rope":
        n, h, d = case["tokens"], case["heads"], case["dim"]
        st["x"] = _randn(g, (n, h, d), TYPES[case["x"]])
        st["pos"] = torch.arange(case["start"], case["start"] + n, dtype=torch.int32,
                                 device=DEVICE)
        f, st["mscale"] = _freqs(case["rot"], case["scaling"])
        st["freqs"] = f.to(DEVICE)
        st["out"] = torch.empty((n, h, d), dtype=TYPES[case["out"]], device=DEVICE)
        if own:
            pkg = _package()
            st["rope"] = pkg.Rope(st["freqs"].data_ptr(), case["rot"], _layout(pkg, case),
                                  st["mscale"])
        return st
    news, lens = _lengths(case)
    h, kv, d, page = case["heads"], case["kv"], case["dim"], case["page"]
    dtype, n_tok = TYPES[case["dtype"]], sum(news)
    need = [-(-x // page) for x in lens]
    n_pages = sum(need) + max(4, sum(need) // 4)
    perm = torch.randperm(n_pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.zeros((case["seqs"], max(need)), dtype=torch.int32)
    perm_host, at = perm.cpu(), 0
    for s, k in enumerate(need):
        table[s, :k] = perm_host[at:at + k]
        at += k
    st["table"] = table.to(DEVICE)
    st["first"] = torch.tensor([sum(news[:s]) for s in range(case["seqs"] + 1)],
                               dtype=torch.int32, device=DEVICE)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    st["max_new"], st["max_len"] = max(news), max(lens)
    # which sequence and position each new token has
    st["seq"] = torch.cat([torch.full((k,), s, dtype=torch.int64)
                           for s, k in enumerate(news)]).to(DEVICE)
    st["pos"] = torch.cat([torch.arange(m - k, m, dtype=torch.int64)
                           for k, m in zip(news, lens)]).to(DEVICE)
    st["k_cache"] = _randn(g, (n_pages, kv, page, d), dtype)
    st["v_cache"] = _randn(g, (n_pages, kv, page, d), dtype)
    if case["op"] == "append":
        # the fused QKV product's rows: q, k and v of a token side by side
        st["qkv"] = _randn(g, (n_tok, (h + 2 * kv) * d), TYPES[case["x"]])
        f, st["mscale"] = _freqs(case["rot"], "none")
        st["freqs"] = f.to(DEVICE)
        st["out"] = torch.empty((n_tok, h, d), dtype=dtype, device=DEVICE)
    else:
        st["q"] = _randn(g, (n_tok, h, d), dtype, 1.5)
        st["out"] = torch.empty((n_tok, h, d), dtype=TYPES[case["out"]], device=DEVICE)
    if own:
        pkg = _package()
        st["cache"] = pkg.KvPages(st["k_cache"].data_ptr(), st["v_cache"].data_ptr(),
                                  _code(pkg, case["dtype"]), n_pages, page, kv, d)
        st["batch"] = pkg.SeqBatch(case["seqs"], n_tok, st["max_new"], st["max_len"],
                                   st["first"].data_ptr(), st["lens"].data_ptr(),
                                   st["table"].data_ptr(), st["table"].shape[1])
        if case["op"] == "append":
            st["rope"] = pkg.Rope(st["freqs"].data_ptr(), case["rot"], _layout(pkg, case),
                                  st["mscale"])
    return st


def _code(pkg, name):
    return {"f32": pkg.F32, "f16": pkg.F16, "bf16": pkg.BF16}[name]


def _layout(pkg, case):
    return pkg.ROPE_PAIRS if case["layout"] == "pairs" else pkg.ROPE_HALVES


# ------------------------------------------------------------- the plain forms

def _turn(x, pos, freqs, layout, mscale):
    """x [tokens][heads][dim] in 32 bits, the first 2 len(freqs) dims turned;
    the angles of far positions in 64 bits."""
    angle = pos.double()[:, None] * freqs[None, :]
    c = (torch.cos(angle) * mscale).float()[:, None, :]
    s = (torch.sin(angle) * mscale).float()[:, None, :]
    rot = 2 * freqs.numel()
    head, tail = x[..., :rot], x[..., rot:]
    if layout == "pairs":
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat((a * c - b * s, a * s + b * c), dim=-1)
    return torch.cat((head, tail), dim=-1)


def _plain_append(st):
    case = st["case"]
    h, kv, d = case["heads"], case["kv"], case["dim"]
    dtype = TYPES[case["dtype"]]
    x = st["qkv"].float().view(-1, h + 2 * kv, d)
    qk = _turn(x[:, :h + kv], st["pos"], st["freqs"], case["layout"], st["mscale"])
    page = st["table"][st["seq"], st["pos"] // case["page"]].long()
    slot = st["pos"] % case["page"]
    st["k_cache"][page, :, slot] = qk[:, h:].to(dtype)
    st["v_cache"][page, :, slot] = x[:, h + kv:].to(dtype)
    return {"q": qk[:, :h].to(dtype), "k": st["k_cache"], "v": st["v_cache"]}


def _plain_attn(st):
    """Every sequence padded to the longest, one product for all scores."""
    case = st["case"]
    n, h, kv, d = case["seqs"], case["heads"], case["kv"], case["dim"]
    group, new = h // kv, st["max_new"]
    start = st["lens"].long() - (st["first"][1:] - st["first"][:-1]).long()  # first new position
    row = st["pos"] - start[st["seq"]]
    q = torch.zeros((n, new, h, d), device=DEVICE)
    q[st["seq"], row] = st["q"].float()
    q = q.view(n, new, kv, group, d).permute(0, 2, 3, 1, 4).reshape(n, kv, group * new, d)
    pages = st["table"].long()
    k = st["k_cache"][pages].float().permute(0, 2, 1, 3, 4).reshape(n, kv, -1, d)
    v = st["v_cache"][pages].float().permute(0, 2, 1, 3, 4).reshape(n, kv, -1, d)
    score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    at = (start[:, None] + torch.arange(new, device=DEVICE))[:, :, None]
    key = torch.arange(k.shape[2], device=DEVICE)[None, None, :]
    seen = key <= at
    if case["window"]:
        seen &= key > at - case["window"]
    seen = seen[:, None, None].expand(n, kv, group, new, -1).reshape(score.shape)
    score = score.masked_fill_(~seen, -math.inf)
    p = torch.exp(score - score.max(dim=-1, keepdim=True).values)
    o = torch.matmul(p, v) / p.sum(dim=-1, keepdim=True)
    o = o.view(n, kv, group, new, d).permute(0, 3, 1, 2, 4).reshape(n, new, h, d)
    return o[st["seq"], row].to(TYPES[case["out"]])


def run(st):
    case = st["case"]
    if not own:
        if case["op"] == "rope":
            return _turn(st["x"].float(), st["pos"], st["freqs"], case["layout"],
                         st["mscale"]).to(TYPES[case["out"]])
        return _plain_append(st) if case["op"] == "append" else _plain_attn(st)
    pkg, s = _package(), torch.cuda.current_stream().cuda_stream
    if case["op"] == "rope":
        pkg.rope(st["rope"], st["pos"].data_ptr(), st["x"].data_ptr(), _code(pkg, case["x"]),
                 st["out"].data_ptr(), _code(pkg, case["out"]), case["tokens"], case["heads"],
                 case["dim"], stream=s)
        return st["out"]
    if case["op"] == "append":
        x, width = st["qkv"], st["qkv"].shape[1]
        k_at = case["heads"] * case["dim"] * x.element_size()
        v_at = k_at + case["kv"] * case["dim"] * x.element_size()
        pkg.kv_append(st["cache"], st["batch"], st["rope"], x.data_ptr(), x.data_ptr() + k_at,
                      x.data_ptr() + v_at, _code(pkg, case["x"]), st["out"].data_ptr(),
                      case["heads"], q_stride=width, k_stride=width, v_stride=width, stream=s)
        return {"q": st["out"], "k": st["k_cache"], "v": st["v_cache"]}
    pkg.attn_paged(st["cache"], st["batch"], st["q"].data_ptr(), case["heads"],
                   1.0 / math.sqrt(case["dim"]), st["out"].data_ptr(), _code(pkg, case["out"]),
                   window=case["window"], stream=s)
    return st["out"]


# -------------------------------------------------------- the work, the values

def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        turned = case["tokens"] * case["heads"] * case["rot"]
        return {"bytes": n * (_size(case["x"]) + _size(case["out"])) + 4 * case["tokens"]
                + 4 * case["rot"], "flops": 3 * turned}
    news, lens = _lengths(case)
    h, kv, d = case["heads"], case["kv"], case["dim"]
    tokens = sum(news)
    if case["op"] == "append":
        n = tokens * (h + 2 * kv) * d
        return {"bytes": n * (_size(case["x"]) + 2), "flops": 3 * tokens * (h + kv) * case["rot"]}
    seen = pairs = 0
    for new, length in zip(news, lens):
        w = case["window"] or length
        if new:
            seen += length - max(0, length - new - w + 1)
            whole = min(new, max(0, length - w))  # tokens whose window is full
            first = length - new
            pairs += whole * w + sum(p + 1 for p in range(first, length - whole))
    return {"bytes": 2 * seen * kv * d * 2 + tokens * h * d * (2 + _size(case["out"])),
            "flops": 4 * pairs * h * d}


def _exact_turn(x, pos, freqs, layout, mscale):
    """The pairs as complex numbers times mscale e^(i p f), in 64 bits."""
    half = freqs.numel()
    turn = torch.polar(torch.full((1, 1), float(mscale), dtype=torch.float64, device=DEVICE),
                       torch.outer(pos.double(), freqs))[:, None, :]
    y = x.double().clone()
    if layout == "pairs":
        z = torch.view_as_complex(y[..., :2 * half].reshape(*y.shape[:-1], half, 2).contiguous())
        y[..., :2 * half] = torch.view_as_real(z * turn).reshape(*y.shape[:-1], 2 * half)
    else:
        z = torch.complex(y[..., :half].clone(), y[..., half:2 * half].clone()) * turn
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_turn(st["x"], st["pos"], st["freqs"], case["layout"], st["mscale"])
    h, kv, d, page = case["heads"], case["kv"], case["dim"], case["page"]
    news, lens = _lengths(case)
    if case["op"] == "append":
        x = st["qkv"].double().view(-1, h + 2 * kv, d)
        k_all, v_all = st["k_cache"].double(), st["v_cache"].double()
        q, at = torch.empty((x.shape[0], h, d), dtype=torch.float64, device=DEVICE), 0
        for s, (new, length) in enumerate(zip(news, lens)):
            pos = torch.arange(length - new, length, device=DEVICE)
            part = x[at:at + new]
            q[at:at + new] = _exact_turn(part[:, :h], pos, st["freqs"], case["layout"],
                                         st["mscale"])
            k = _exact_turn(part[:, h:h + kv], pos, st["freqs"], case["layout"], st["mscale"])
            flat = st["table"][s].long()[torch.div(pos, page, rounding_mode="floor")]
            for j in range(kv):
                k_all[flat, j, pos % page] = k[:, j]
                v_all[flat, j, pos % page] = part[:, h + kv + j]
            at += new
        return {"q": q, "k": k_all, "v": v_all}
    out = torch.zeros((sum(news), h, d), dtype=torch.float64, device=DEVICE)
    at = 0
    for s, (new, length) in enumerate(zip(news, lens)):
        used = st["table"][s, :-(-length // page)].long()
        for j in range(kv):
            k = st["k_cache"][used, j].reshape(-1, d)[:length].double()
            v = st["v_cache"][used, j].reshape(-1, d)[:length].double()
            heads = slice(j * (h // kv), (j + 1) * (h // kv))
            q = st["q"][at:at + new, heads].double()
            logit = torch.einsum("thd,kd->thk", q, k) / math.sqrt(d)
            gap = (torch.arange(length - new, length, device=DEVICE)[:, None]
                   - torch.arange(length, device=DEVICE)[None, :])
            hidden = (gap < 0) | (gap >= (case["window"] or length + 1))
            logit = logit.masked_fill(hidden[:, None, :], -math.inf)
            out[at:at + new, heads] = torch.softmax(logit, dim=-1) @ v
        at += new
    return out
