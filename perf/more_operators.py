"""A decoding step of many sequences that share prompts (beam search, parallel
samples), as timed cases: the 8-bit products of its rows, the selection among
its logits, and the pages of the cache that follow the selection.

A case is one pass as a program makes it.  Its ops:

  linear   rows of activations to 8-bit codes with a scale each, times 8-bit
           weights with a scale for each output row: swamp_quantize_rows,
           swamp_gemm_rows_i8
  beam     the best continuations of every sequence over its beams and the
           vocabulary: swamp_beam_select
  step     the beams' page tables follow their parents, every sequence gets
           pages for its new tokens, and pages that several would write are
           copied in every layer: swamp_pages_fork, swamp_pages_extend,
           swamp_kv_copy
  compact  finished and cut sequences give their pages back, and the pages in
           use move to the lowest places: swamp_pages_trim,
           swamp_pages_compact, swamp_kv_copy

`step` and `compact` change the tables and counts that they are given; a pass
begins with the same ones put back, so that every pass does the same work.
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

def listed():
    return [
        # One sequence decodes: the fused QKV product of an 8B layer, one row.
        {"name": "linear_one", "op": "linear", "m": 1, "rows": 6144, "cols": 4096, "x": "f32",
         "y": "f32"},
        # 16 prompts of 4 beams: gate and up of an 8B layer.
        {"name": "linear_beams", "op": "linear", "m": 64, "rows": 28672, "cols": 4096, "x": "f32",
         "y": "f32"},
        # Odd sizes on every side, a batch between the two regimes.
        {"name": "linear_odd", "op": "linear", "m": 333, "rows": 5003, "cols": 2111, "x": "f16",
         "y": "f16"},
        # A prompt of 4096 tokens through gate and up of an 8B layer.
        {"name": "linear_prompt", "op": "linear", "m": 4096, "rows": 28672, "cols": 4096,
         "x": "bf16", "y": "bf16"},
        # One prompt, four beams, twice as many candidates: latency counts.
        {"name": "beam_one", "op": "beam", "seqs": 1, "beams": 4, "vocab": 128256, "out": 8,
         "x": "f32", "done": False, "allowed": 1.0},
        # A serving batch: 16 prompts of 4 beams.
        {"name": "beam_batch", "op": "beam", "seqs": 16, "beams": 4, "vocab": 128256, "out": 4,
         "x": "f32", "done": True, "allowed": 1.0},
        # A wide search over a small vocabulary, logits in 16 bits (many are equal).
        {"name": "beam_wide", "op": "beam", "seqs": 4, "beams": 32, "vocab": 32000, "out": 64,
         "x": "bf16", "done": False, "allowed": 1.0},
        # A grammar leaves a few tokens of an odd vocabulary in hundreds of rows.
        {"name": "beam_grammar", "op": "beam", "seqs": 50, "beams": 5, "vocab": 50257, "out": 10,
         "x": "f16", "done": True, "allowed": 0.003},
        # One prompt, four beams, short: latency counts.
        {"name": "step_one", "op": "step", "seqs": 1, "beams": 4, "len": 100, "new": 1, "page": 16,
         "kv": 8, "dim": 128, "layers": 2, "dtype": "bf16"},
        # 16 prompts of 4 beams, pages of 32 tokens, four layers of an 8B model.
        {"name": "step_batch", "op": "step", "seqs": 16, "beams": 4, "len": 1001, "new": 1,
         "page": 32, "kv": 8, "dim": 128, "layers": 4, "dtype": "bf16"},
        # Eight documents of 8 beams each: long page tables, little to copy.
        {"name": "step_long", "op": "step", "seqs": 8, "beams": 8, "len": 32768, "new": 5,
         "page": 16, "kv": 2, "dim": 64, "layers": 2, "dtype": "f16"},
        # 128 sequences, a third ended and a third cut back: a cache full of holes.
        {"name": "compact_batch", "op": "compact", "seqs": 128, "len": 1500, "page": 32, "kv": 4,
         "dim": 128, "layers": 2, "dtype": "bf16"},
    ]


def _span(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["linear", "linear", "beam", "beam", "step", "compact"])
    if op == "linear":
        case = {"op": op, "m": _span(rng, 1, 4096), "rows": _span(rng, 64, 32768),
                "cols": _span(rng, 32, 16384), "x": rng.choice(["f32", "f16", "bf16"]),
                "y": rng.choice(["f32", "f32", "f16", "bf16"])}
        while work(case)["flops"] > 9e11:
            case["m"] = case["m"] * 3 // 4
        return case
    if op == "beam":
        beams = _span(rng, 1, 64)
        case = {"op": op, "seqs": _span(rng, 1, 64), "beams": beams,
                "vocab": _span(rng, 100, 160000), "out": min(64, beams * rng.choice([1, 1, 2, 3])),
                "x": rng.choice(["f32", "f32", "f16", "bf16"]), "done": rng.random() < 0.5,
                "allowed": rng.choice([1.0, 1.0, 1.0, 0.5, 0.01])}
        while case["seqs"] * beams * case["vocab"] > 1.2e7:
            case["seqs"], case["vocab"] = max(1, case["seqs"] // 2), max(100, case["vocab"] * 3 // 4)
        return case
    case = {"op": op, "seqs": _span(rng, 1, 64), "len": _span(rng, 1, 20000),
            "page": rng.choice([1, 8, 16, 16, 32, 64, 128]), "kv": rng.choice([1, 2, 4, 5, 8]),
            "dim": rng.choice([64, 80, 128, 256]), "layers": rng.choice([1, 2, 3, 4]),
            "dtype": rng.choice(["f16", "bf16"])}
    if op == "step":
        case.update(beams=rng.choice([1, 2, 4, 5, 8]), new=rng.choice([1, 1, 1, 4, 17]))
    else:
        case["seqs"] *= rng.choice([1, 2, 4])
    while _n_pages(case) * _page_bytes(case) * 2 * case["layers"] > 5e8 or _n_pages(case) > 60000:
        case["len"], case["layers"] = max(1, case["len"] * 3 // 4), 1 + case["layers"] // 2
        case["seqs"] = max(1, case["seqs"] * 7 // 8)
    return case


def _length(case, g):
    """Tokens of prompt (or sequence) g: from the longest down to a quarter of it."""
    return max(1, int(case["len"] * (1.0 - 0.75 * ((g * 0.6180339887498949) % 1.0))))


def _page_bytes(case):
    return case["page"] * case["kv"] * case["dim"] * 2


def _shared(case, g):
    """Pages that the beams of prompt g share: all but those of its last 48 tokens."""
    return max(0, _length(case, g) - 48) // case["page"]


def _parent(case, g, j):
    """Whom beam j of prompt g continues: the first beams more often."""
    return int(case["beams"] * ((((g + 1) * 0.7548776662 + j * 0.5698402910) % 1.0) ** 2))


def _used_pages(case):
    if case["op"] == "compact":
        return sum(-(-_length(case, g) // case["page"]) for g in range(case["seqs"]))
    return sum(_shared(case, g)
               + case["beams"] * (-(-_length(case, g) // case["page"]) - _shared(case, g))
               for g in range(case["seqs"]))


def _n_pages(case):
    used = _used_pages(case)
    if case["op"] == "compact":
        return used + used // 4 + 2
    return used + case["seqs"] * case["beams"] * (2 + case["new"] // case["page"]) + used // 8


def _kept(case, g):
    """Tokens that sequence g keeps: a third none, a third a part, a third all."""
    n = _length(case, g)
    return (0, n * 3 // 5, n)[g % 3]


# ----------------------------------------------------------------- the inputs

def _randn(g, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * sigma).to(dtype)


def _prepare_linear(case, g, st):
    m, n, k = case["m"], case["rows"], case["cols"]
    # activations: a few columns far above the others
    col = torch.exp(0.8 * torch.randn(k, generator=g, device=DEVICE))
    st["x"] = (torch.randn((m, k), generator=g, device=DEVICE) * col).to(TYPES[case["x"]])
    # the codes' rows begin at multiples of 16 bytes
    st["stride"] = stride = -(-k // 16) * 16
    st["w"] = torch.zeros((n, stride), dtype=torch.int8, device=DEVICE)
    w = torch.randn((n, k), generator=g, device=DEVICE)
    st["w_scale"] = w.abs().amax(dim=1) * (1.0 / 127.0) / math.sqrt(k)
    st["w"][:, :k] = torch.round(w * (127.0 / w.abs().amax(dim=1, keepdim=True))).to(torch.int8)
    st["y"] = torch.empty((m, n), dtype=TYPES[case["y"]], device=DEVICE)
    st["q"] = torch.zeros((m, stride), dtype=torch.int8, device=DEVICE)
    st["x_scale"] = torch.empty(m, device=DEVICE)


def _prepare_beam(case, g, st):
    n, b, v, k = case["seqs"], case["beams"], case["vocab"], case["out"]
    logits = torch.randn((n * b, v), generator=g, device=DEVICE) * 2.5
    # (a few tokens stand out, as they do in text)
    hot = torch.randint(0, v, (n * b, min(v, 32)), generator=g, device=DEVICE)
    logits.scatter_add_(1, hot, 6.0 * torch.rand(hot.shape, generator=g, device=DEVICE))
    if case["allowed"] < 1.0:
        keep = torch.rand((n * b, v), generator=g, device=DEVICE) < case["allowed"]
        logits.masked_fill_(~keep, -math.inf)
    st["logits"] = logits.to(TYPES[case["x"]])
    st["score"] = -8.0 * torch.rand(n * b, generator=g, device=DEVICE) - 4.0
    st["eos"] = 2
    st["done"] = None
    if case["done"]:
        st["done"] = (torch.rand(n * b, generator=g, device=DEVICE) < 0.2).to(torch.int32)
    st["parent"] = torch.empty(n * k, dtype=torch.int32, device=DEVICE)
    st["token"] = torch.empty(n * k, dtype=torch.int32, device=DEVICE)
    st["out_score"] = torch.empty(n * k, device=DEVICE)
    st["out_done"] = torch.empty(n * k, dtype=torch.int32, device=DEVICE)
    if own:
        pkg = _package()
        st["spec"] = pkg.BeamSpec(n, b, v, k, st["eos"])


def _prepare_pages(case, g, st):
    step, page = case["op"] == "step", case["page"]
    beams = case["beams"] if step else 1
    n, n_pages = case["seqs"] * beams, _n_pages(case)
    lens = [_length(case, i // beams) for i in range(n)]
    width = -(-(max(lens) + (case["new"] if step else 0)) // page)
    words = -(-n_pages // 32)
    # every count and table in one buffer, a view for each (rows of 16 bytes)
    sizes = {"table": n * width, "len": n, "refs": n_pages, "used": words, "src": n_pages,
             "dst": n_pages, "count": 1}
    at, total = {}, 0
    for name, size in sizes.items():
        at[name] = total
        total += -(-size // 4) * 4
    flat = torch.zeros(total, dtype=torch.int32)
    part = {name: flat[at[name]:at[name] + size] for name, size in sizes.items()}
    order = torch.randperm(n_pages, generator=g, device=DEVICE).to(torch.int32).cpu()
    table, taken = part["table"].view(n, width), 0
    for s in range(n):
        i, j = divmod(s, beams)
        need, shared = -(-lens[s] // page), _shared(case, i) if step else 0
        if j == 0:
            table[s, :shared] = order[taken:taken + shared]
            taken += shared
        else:
            table[s, :shared] = table[s - j, :shared]
        table[s, shared:need] = order[taken:taken + need - shared]
        taken += need - shared
        part["refs"].index_add_(0, table[s, :need].long(), torch.ones(need, dtype=torch.int32))
    part["len"].copy_(torch.tensor(lens, dtype=torch.int32))
    bits = torch.zeros(words * 32, dtype=torch.int64)
    bits[:n_pages] = (part["refs"] > 0).long()
    part["used"].copy_((bits.view(-1, 32) << torch.arange(32)).sum(dim=1).to(torch.int32))
    st["start"] = flat.to(DEVICE)
    st["now"] = st["start"].clone()
    for name, size in sizes.items():
        st[name] = st["now"][at[name]:at[name] + size]
    st["table"] = st["table"].view(n, width)
    st["n_pages"] = n_pages
    shape = (case["layers"], n_pages, case["kv"], page, case["dim"])
    st["k_cache"] = _randn(g, shape, TYPES[case["dtype"]])
    st["v_cache"] = _randn(g, shape, TYPES[case["dtype"]])
    if step:
        st["parent"] = torch.tensor([s - s % beams + _parent(case, s // beams, s % beams)
                                     for s in range(n)], dtype=torch.int32, device=DEVICE)
        st["new"] = torch.full((n,), case["new"], dtype=torch.int32, device=DEVICE)
    else:
        st["keep"] = torch.tensor([_kept(case, s) for s in range(n)], dtype=torch.int32,
                                  device=DEVICE)
    if own:
        pkg = _package()
        code = {"f16": pkg.F16, "bf16": pkg.BF16}[case["dtype"]]
        st["pool"] = pkg.PagePool(n_pages, page, st["refs"].data_ptr(), st["used"].data_ptr())
        st["tables"] = pkg.PageTables(n, st["len"].data_ptr(), st["table"].data_ptr(), width)
        st["moves"] = pkg.PageMoves(n_pages, st["src"].data_ptr(), st["dst"].data_ptr(),
                                    st["count"].data_ptr())
        st["caches"] = pkg.kv_caches([
            pkg.KvPages(st["k_cache"][i].data_ptr(), st["v_cache"][i].data_ptr(), code, n_pages,
                        page, case["kv"], case["dim"]) for i in range(case["layers"])])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    st = {"case": case}
    if case["op"] == "linear":
        _prepare_linear(case, g, st)
    elif case["op"] == "beam":
        _prepare_beam(case, g, st)
    else:
        _prepare_pages(case, g, st)
    return st


# ------------------------------------------------------------- the plain forms

def _plain_linear(st):
    k = st["case"]["cols"]
    x = st["x"].float()
    scale = x.abs().amax(dim=1, keepdim=True)
    scale = scale / torch.full_like(scale, 127.0)
    q = torch.round(x / scale.clamp_min(1e-37))
    y = torch.matmul(q, st["w"][:, :k].float().t()) * scale * st["w_scale"]
    return y.to(st["y"].dtype)


def _plain_beam(st):
    """Scores in 64 bits, so that near ones keep their order; a stable sort keeps
    the lowest index first among equal ones."""
    case = st["case"]
    n, b, v, k = case["seqs"], case["beams"], case["vocab"], case["out"]
    x = st["logits"].double()
    top = x.max(dim=1, keepdim=True).values
    lse = torch.log(torch.exp(x - top).sum(dim=1, keepdim=True)) + top
    total = st["score"].double()[:, None] + (x - lse)
    total = torch.where(torch.isnan(total), -math.inf, total)  # rows without a token
    if st["done"] is not None:  # an ended beam has one continuation: itself
        token = torch.arange(v, device=DEVICE)
        same = torch.where(token == st["eos"], st["score"].double()[:, None], -math.inf)
        total = torch.where(st["done"][:, None] != 0, same, total)
    value, at = torch.sort(total.view(n, b * v), dim=1, descending=True, stable=True)
    value, at = value[:, :k], at[:, :k]
    if b * v < k:
        value = torch.nn.functional.pad(value, (0, k - b * v), value=-math.inf)
        at = torch.nn.functional.pad(at, (0, k - b * v))
    none = value == -math.inf
    beam = at // v
    parent = beam + b * torch.arange(n, device=DEVICE)[:, None]
    token = at - beam * v
    done = token == st["eos"]
    if st["done"] is not None:
        done = done | (st["done"][parent] != 0)
    return {"parent": torch.where(none, -1, parent).int().flatten(),
            "token": torch.where(none, -1, token).int().flatten(),
            "score": value.float().flatten(), "done": (done & ~none).int().flatten()}


def _plain_used(st):
    bits = torch.zeros(st["used"].numel() * 32, dtype=torch.int64, device=DEVICE)
    bits[:st["n_pages"]] = (st["refs"] > 0).long()
    words = (bits.view(-1, 32) << torch.arange(32, device=DEVICE)).sum(dim=1)
    st["used"].copy_(words.to(torch.int32))


def _count(st, ids, mask, by):
    """refs += by for every id of the mask."""
    st["refs"].index_add_(0, ids.flatten().long(), (mask.int() * by).flatten())


def _columns(st, lens):
    """Which entries of the tables hold a sequence's pages."""
    col = torch.arange(st["table"].shape[1], device=DEVICE)
    return col[None, :] < -(-lens // st["case"]["page"])[:, None]


def _plain_fork(st):
    parent = st["parent"].long()
    lens = st["len"].long()
    _count(st, st["table"], _columns(st, lens), -1)
    lens = lens[parent]
    mine = _columns(st, lens)
    st["table"].copy_(torch.where(mine, st["table"][parent], st["table"]))
    st["len"].copy_(lens)
    _count(st, st["table"], mine, 1)
    _plain_used(st)


def _plain_extend(st):
    page, table = st["case"]["page"], st["table"]
    n, width = table.shape
    lens = st["len"].long()
    last = torch.div(lens, page, rounding_mode="floor")
    tail = table.gather(1, last.clamp_max(width - 1)[:, None])[:, 0].long()
    held = (lens % page != 0) & (st["new"] > 0)
    refs = st["refs"][torch.where(held, tail, 0)].long()
    # how many sequences before this one would write the same page
    seq = torch.arange(n, device=DEVICE)
    before = (tail[:, None] == tail[None, :]) & held[None, :] & (seq[None, :] < seq[:, None])
    copies = held & (before.sum(dim=1) < refs - 1)
    first = -(-lens // page)
    fresh = -(-(lens + st["new"]) // page) - first
    need = copies.long() + fresh
    offset = torch.cumsum(need, 0) - need
    free = torch.argsort((st["refs"] > 0).int(), stable=True)  # the lowest free pages first
    free = torch.nn.functional.pad(free, (0, int(n * (width + 1))), value=-1)
    room = st["n_pages"] - (st["refs"] > 0).sum()
    # the pages that are copied, and their places in the list
    place = torch.where(copies, torch.cumsum(copies.long(), 0) - 1, st["src"].numel())
    to = free[offset]
    src = torch.nn.functional.pad(st["src"], (0, 1)).scatter(0, place, tail.int())
    dst = torch.nn.functional.pad(st["dst"], (0, 1)).scatter(0, place, to.int())
    st["src"].copy_(src[:-1])
    st["dst"].copy_(dst[:-1])
    st["count"].copy_(copies.sum().int()[None])
    _count(st, tail, copies, -1)
    col = torch.arange(width, device=DEVICE)[None, :]
    new = (col >= first[:, None]) & (col < (first + fresh)[:, None])
    which = (offset + copies.long())[:, None] + col - first[:, None]
    new_ids = torch.where(new, which, 0)
    ids = torch.where(new_ids < room, free[new_ids], -1)
    ids = torch.where(copies[:, None] & (col == last[:, None]), to[:, None], ids).int()
    new = new | (copies[:, None] & (col == last[:, None]))
    table.copy_(torch.where(new, ids, table))
    _count(st, torch.where(new, ids, 0), new, 1)
    st["len"].add_(st["new"])
    _plain_used(st)


def _plain_trim(st):
    keep = torch.minimum(st["len"], st["keep"])
    gone = _columns(st, st["len"].long()) & ~_columns(st, keep.long())
    _count(st, torch.where(gone, st["table"], 0), gone, -1)
    st["len"].copy_(keep)
    _plain_used(st)


def _plain_compact(st):
    used = st["refs"] > 0
    page = torch.arange(st["n_pages"], device=DEVICE)
    n = used.sum()
    src, dst = page[used & (page >= n)], page[~used & (page < n)]
    st["src"][:src.numel()] = src.int()
    st["dst"][:dst.numel()] = dst.int()
    st["count"].fill_(src.numel())
    to = page.clone()
    to[src] = dst
    st["refs"][dst] = st["refs"][src]
    st["refs"][src] = 0
    mine = _columns(st, st["len"].long())
    moved = to[torch.where(mine, st["table"], 0).long()].int()
    st["table"].copy_(torch.where(mine, moved, st["table"]))
    _plain_used(st)


def _plain_copy(st):
    n = int(st["count"])
    src, dst = st["src"][:n].long(), st["dst"][:n].long()
    st["k_cache"][:, dst] = st["k_cache"][:, src]
    st["v_cache"][:, dst] = st["v_cache"][:, src]


def _pages_out(st):
    return {name: st[name] for name in ("table", "len", "refs", "used", "src", "dst", "count",
                                        "k_cache", "v_cache")}


def run(st):
    case = st["case"]
    if not own:
        if case["op"] == "linear":
            return _plain_linear(st)
        if case["op"] == "beam":
            return _plain_beam(st)
        st["now"].copy_(st["start"])
        if case["op"] == "step":
            _plain_fork(st)
            _plain_extend(st)
        else:
            _plain_trim(st)
            _plain_compact(st)
        _plain_copy(st)
        return _pages_out(st)
    pkg, s = _package(), torch.cuda.current_stream().cuda_stream
    code = {"f32": pkg.F32, "f16": pkg.F16, "bf16": pkg.BF16}
    if case["op"] == "linear":
        m, n, k, stride = case["m"], case["rows"], case["cols"], st["stride"]
        pkg.quantize_rows(st["x"].data_ptr(), code[case["x"]], st["q"].data_ptr(),
                          st["x_scale"].data_ptr(), m, k, q_stride=stride, stream=s)
        pkg.gemm_rows_i8(st["q"].data_ptr(), st["x_scale"].data_ptr(), st["w"].data_ptr(),
                         st["w_scale"].data_ptr(), st["y"].data_ptr(), code[case["y"]], m, n, k,
                         x_stride=stride, w_stride=stride, stream=s)
        return st["y"]
    if case["op"] == "beam":
        pkg.beam_select(st["spec"], st["logits"].data_ptr(), code[case["x"]],
                        st["score"].data_ptr(), st["parent"].data_ptr(), st["token"].data_ptr(),
                        st["out_score"].data_ptr(),
                        d_done=0 if st["done"] is None else st["done"].data_ptr(),
                        d_out_done=st["out_done"].data_ptr(), stream=s)
        return {"parent": st["parent"], "token": st["token"], "score": st["out_score"],
                "done": st["out_done"]}
    st["now"].copy_(st["start"])
    if case["op"] == "step":
        pkg.pages_fork(st["pool"], st["tables"], st["parent"].data_ptr(), stream=s)
        pkg.pages_extend(st["pool"], st["tables"], st["new"].data_ptr(), st["moves"], stream=s)
    else:
        pkg.pages_trim(st["pool"], st["tables"], st["keep"].data_ptr(), stream=s)
        pkg.pages_compact(st["pool"], st["tables"], st["moves"], stream=s)
    pkg.kv_copy(st["caches"], st["moves"], stream=s)
    return _pages_out(st)


# -------------------------------------------------------- the work, the values

def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["rows"], case["cols"]
        return {"bytes": m * k * _size(case["x"]) + n * k + 4 * n + m * n * _size(case["y"]),
                "flops": 2 * m * n * k}
    if case["op"] == "beam":
        rows = case["seqs"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * _size(case["x"]) + 8)
                + 16 * case["seqs"] * case["out"],
                "flops": 4 * rows * case["vocab"]}
    page = case["page"]
    if case["op"] == "step":
        b = case["beams"]
        entries = copies = fresh = 0
        for g in range(case["seqs"]):
            n = _length(case, g)
            parents = [_parent(case, g, j) for j in range(b)]
            cols = -(-n // page)
            entries += cols * (len(set(parents)) + sum(p != j for j, p in enumerate(parents)))
            fresh += b * (-(-(n + case["new"]) // page) - cols)
            if n % page:
                copies += b - len(set(parents))
        n_seq = case["seqs"] * b
    else:
        kept = sum(-(-_kept(case, g) // page) for g in range(case["seqs"]))
        entries = _used_pages(case) - kept + 2 * kept  # those given back, those kept: read, moved
        copies = int(kept * (1 - kept / _n_pages(case)))  # what lies above the pages in use
        fresh, n_seq = 0, case["seqs"]
    return {"bytes": 4 * (entries + 2 * fresh + 4 * copies + 3 * n_seq)
            + 4 * copies * case["layers"] * _page_bytes(case), "flops": 0}


def _exact_pages(case, st):
    """One sequence after the other, one page after the other, on the host."""
    page, step = case["page"], case["op"] == "step"
    lens, table = st["len"].tolist(), st["table"].tolist()
    refs = st["refs"].tolist()
    src, dst = st["src"].tolist(), st["dst"].tolist()
    n = len(lens)
    if step:
        parent, new = st["parent"].tolist(), st["new"].tolist()
        rows = [table[p][:-(-lens[p] // page)] for p in parent]
        for s in range(n):
            for e in table[s][:-(-lens[s] // page)]:
                refs[e] -= 1
        for s in range(n):
            table[s][:len(rows[s])] = rows[s]
            for e in rows[s]:
                refs[e] += 1
        lens = [lens[p] for p in parent]
        free = iter([e for e in range(len(refs)) if refs[e] == 0])
        moves = []
        for s in range(n):
            at = lens[s] // page
            if new[s] and lens[s] % page and refs[table[s][at]] > 1:
                e = next(free)
                moves.append((table[s][at], e))
                refs[table[s][at]] -= 1
                refs[e] = 1
                table[s][at] = e
            for col in range(-(-lens[s] // page), -(-(lens[s] + new[s]) // page)):
                table[s][col] = next(free)
                refs[table[s][col]] = 1
            lens[s] += new[s]
    else:
        for s, keep in enumerate(st["keep"].tolist()):
            for e in table[s][-(-min(keep, lens[s]) // page):-(-lens[s] // page)]:
                refs[e] -= 1
            lens[s] = min(keep, lens[s])
        used = [e for e in range(len(refs)) if refs[e] > 0]
        high = [e for e in used if e >= len(used)]
        moves = list(zip(high, [e for e in range(len(used)) if refs[e] == 0]))
        to = dict(moves)
        for a, b in moves:
            refs[a], refs[b] = 0, refs[a]
        for s in range(n):
            k = -(-lens[s] // page)
            table[s][:k] = [to.get(e, e) for e in table[s][:k]]
    for i, (a, b) in enumerate(moves):
        src[i], dst[i] = a, b
    words = [0] * st["used"].numel()
    for e, r in enumerate(refs):
        words[e // 32] |= (r > 0) << (e % 32)
    found = {"table": table, "len": lens, "refs": refs, "src": src, "dst": dst,
             "used": [w - (w >> 31 << 32) for w in words], "count": [len(moves)]}
    found = {name: torch.tensor(x, dtype=torch.int32, device=DEVICE) for name, x in found.items()}
    for name in ("k_cache", "v_cache"):
        found[name] = st[name].double()
        if moves:
            a, b = (torch.tensor(x, device=DEVICE) for x in zip(*moves))
            found[name][:, b] = st[name][:, a].double()
    return found


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("step", "compact"):
        return _exact_pages(case, st)
    if case["op"] == "linear":
        x, w = st["x"].double(), st["w"][:, :case["cols"]].double()
        # the scale is a number of 32 bits, and so is the quotient that is rounded
        scale = (x.abs().max(dim=1).values / torch.tensor(127.0, dtype=torch.float64,
                                                          device=DEVICE)).float().double()
        codes = (x / scale[:, None]).float().double().round()
        return torch.einsum("mk,nk->mn", codes, w) * torch.outer(scale, st["w_scale"].double())
    n, b, v, k = case["seqs"], case["beams"], case["vocab"], case["out"]
    found = {"parent": [], "token": [], "score": [], "done": []}
    for s in range(n):
        value, at = [], []
        for j in range(s * b, (s + 1) * b):
            row = st["logits"][j].double()
            if st["done"] is not None and int(st["done"][j]):
                value.append(st["score"][j:j + 1].double())
                at.append(torch.tensor([st["eos"]], device=DEVICE) + j * v)
            elif bool((row > -math.inf).any()):
                logp = torch.log_softmax(row, dim=0) + st["score"][j].double()
                live = torch.nonzero(row > -math.inf)[:, 0]
                value.append(logp[live])
                at.append(live + j * v)
        value = torch.cat(value + [torch.empty(0, dtype=torch.float64, device=DEVICE)])
        at = torch.cat(at + [torch.empty(0, dtype=torch.int64, device=DEVICE)])
        best = torch.sort(value, descending=True, stable=True)
        m = min(k, value.numel())
        at = at[best.indices[:m]]
        pad = (0, k - m)
        ended = at % v == st["eos"]
        if st["done"] is not None:
            ended |= st["done"][at // v] != 0
        found["parent"].append(torch.nn.functional.pad(at // v, pad, value=-1))
        found["token"].append(torch.nn.functional.pad(at % v, pad, value=-1))
        found["score"].append(torch.nn.functional.pad(best.values[:m], pad, value=-math.inf))
        found["done"].append(torch.nn.functional.pad(ended.long(), pad))
    return {name: torch.cat(parts) for name, parts in found.items()}
