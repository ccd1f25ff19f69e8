"""Batches over a paged cache for the tests of swamp_rope, swamp_kv_append and
swamp_attn_paged, and their plain implementations in 64 bits on the CPU."""
import math

import torch

F32, F16, BF16 = 0, 1, 30
TORCH = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
NAME = {F32: "f32", F16: "f16", BF16: "bf16"}


def half_step(code):
    """Largest relative rounding of a value to the type."""
    return torch.finfo(TORCH[code]).eps / 2


def turn(x, pos, freqs, n_rot, halves, mscale=1.0):
    """x [tokens][heads][dim], in 64 bits."""
    x = x.double().clone()
    ang = pos.double()[:, None, None] * freqs.double()[None, None, :]
    c, s = torch.cos(ang) * mscale, torch.sin(ang) * mscale
    if halves:
        a, b = x[..., :n_rot // 2].clone(), x[..., n_rot // 2:n_rot].clone()
        x[..., :n_rot // 2], x[..., n_rot // 2:n_rot] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., 0:n_rot:2].clone(), x[..., 1:n_rot:2].clone()
        x[..., 0:n_rot:2], x[..., 1:n_rot:2] = a * c - b * s, a * s + b * c
    return x


def turn_bound(x, n_rot, halves, mscale, out_code):
    """|error| allowed: sine and cosine within 3 steps of 2^-24 (two roundings
    of the reduced angle, the polynomial's last), two products, a sum and the
    magnitude's product one each: 8 steps of 2^-24 of |a| + |b|, and the
    output's rounding (fp16: at least half its smallest subnormal)."""
    mag = x.double().abs().clone()
    if halves:
        t = mag[..., :n_rot // 2] + mag[..., n_rot // 2:n_rot]
        mag[..., :n_rot // 2], mag[..., n_rot // 2:n_rot] = t, t
    else:
        t = mag[..., 0:n_rot:2] + mag[..., 1:n_rot:2]
        mag[..., 0:n_rot:2], mag[..., 1:n_rot:2] = t, t
    return mag * mscale * (8 * 2.0 ** -24 + half_step(out_code)) + 2.0 ** -25


class Paged:
    """Sequences with `news` new tokens of `lens` cached ones on shuffled pages.
    Slots that hold no key of a sequence are filled with `stale`."""

    def __init__(self, news, lens, n_kv, dim, page, code, seed=1, order="head", stale=math.nan,
                 sigma=1.0, extra_pages=3):
        g = torch.Generator().manual_seed(seed)
        self.news, self.lens, self.n_kv, self.dim, self.page = list(news), list(lens), n_kv, dim, page
        self.code, self.order, self.g = code, order, g
        need = [-(-max(n, 0) // page) for n in lens]
        self.n_pages = sum(need) + extra_pages
        perm = torch.randperm(self.n_pages, generator=g)
        self.table = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = perm[at:at + n].int()
            at += n
        self.first = torch.tensor([sum(self.news[:s]) for s in range(len(news) + 1)],
                                  dtype=torch.int32)
        self.len = torch.tensor(lens, dtype=torch.int32)
        self.n_tok = sum(self.news)
        # logical [page][head][slot][dim]
        shape = (self.n_pages, n_kv, page, dim)
        self.k = torch.full(shape, stale, dtype=TORCH[code])
        self.v = torch.full(shape, stale, dtype=TORCH[code])
        for s, n in enumerate(lens):
            for p0 in range(0, max(n, 0), page):
                m, i = min(page, n - p0), int(self.table[s, p0 // page])
                self.k[i, :, :m] = (torch.randn((n_kv, m, dim), generator=g) * sigma).to(TORCH[code])
                self.v[i, :, :m] = torch.randn((n_kv, m, dim), generator=g).to(TORCH[code])

    def keys(self, s, n=None):
        """(k, v) of the sequence's first n positions, [n][head][dim] views' copies."""
        n = self.lens[s] if n is None else n
        pos = torch.arange(max(n, 0))
        ids = self.table[s].long()[pos // self.page]
        return self.k[ids, :, pos % self.page], self.v[ids, :, pos % self.page]

    def put(self, s, pos, k=None, v=None):
        i = int(self.table[s, pos // self.page])
        if k is not None:
            self.k[i, :, pos % self.page] = k
        if v is not None:
            self.v[i, :, pos % self.page] = v

    def on_gpu(self, pkg, max_new=None, max_len=None, n_tok=None, bad=True):
        """(cache, batch) over device copies, kept in self.dev."""
        def lay(x):  # the memory order of the cache
            return x.cuda() if self.order == "head" else x.transpose(1, 2).contiguous().cuda()
        d = {"k": lay(self.k), "v": lay(self.v), "first": self.first.cuda(),
             "len": self.len.cuda(), "table": self.table.cuda(),
             "bad": torch.zeros(1, dtype=torch.int32, device="cuda")}
        self.dev = d
        strides = () if self.order == "head" else (self.page * self.n_kv * self.dim, self.dim,
                                                   self.n_kv * self.dim)
        cache = pkg.KvPages(d["k"].data_ptr(), d["v"].data_ptr(), self.code, self.n_pages,
                            self.page, self.n_kv, self.dim, *strides)
        batch = pkg.SeqBatch(len(self.lens), self.n_tok if n_tok is None else n_tok,
                             max(self.news + [0]) if max_new is None else max_new,
                             max(self.lens + [0]) if max_len is None else max_len,
                             d["first"].data_ptr(), d["len"].data_ptr(), d["table"].data_ptr(),
                             self.table.shape[1], d["bad"].data_ptr() if bad else 0)
        return cache, batch

    def cache_back(self):
        """The device's (k, v) in logical order."""
        def lay(x):
            return x.cpu() if self.order == "head" else x.cpu().transpose(1, 2)
        return lay(self.dev["k"]), lay(self.dev["v"])


def attention(paged, q, scale, window=0, precise=True, out_code=F32):
    """(out, bound) in 64 bits.  Keys that a row does not see are left out of
    its sums, whatever they hold.  The bound, per element, from the roundings
    on the way (2^-24 each where not said; sums of n roundings as 8 sqrt(n)):
      score: dim roundings of at most |q||k|; the product with the scale and
        the distance to the maximum: 4 of |score|; exp2: 4;
      weights: to the cache's type where the output has 16 bits, else 2^-22;
      sums over n keys, numerator and denominator; the output's rounding."""
    h, dim = q.shape[1], q.shape[2]
    group = h // paged.n_kv
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    u = 2.0 ** -24
    weight = 2.0 ** -22 if precise else half_step(paged.code)
    at = 0
    for s, (new, n) in enumerate(zip(paged.news, paged.lens)):
        if n > 0:
            k, v = (x.double() for x in paged.keys(s))
        for i in range(new):
            pos = n - new + i
            if pos >= 0:
                lo = max(0, pos + 1 - window) if window else 0
                kk = k[lo:pos + 1].repeat_interleave(group, 1)
                vv = v[lo:pos + 1].repeat_interleave(group, 1)
                x = q[at + i].double()
                sc = (kk * x[None]).sum(-1) * scale
                p = torch.exp(sc - sc.max(0).values[None])
                l = p.sum(0)
                out[at + i] = (p[..., None] * vv).sum(0) / l[:, None]
                size = (x.norm(dim=-1)[None] * kk.norm(dim=-1)) * abs(scale)
                e = u * (8 * math.sqrt(dim) * size + 4 * sc.abs() + 4 * sc.abs().max(0).values + 4)
                n_seen = pos + 1 - lo
                each = e + weight + u * 8 * math.sqrt(n_seen)
                mean = (p[..., None] * vv.abs()).sum(0) / l[:, None]
                bound[at + i] = ((p * each)[..., None] * vv.abs()).sum(0) / l[:, None] \
                    + mean * ((p * each).sum(0) / l)[:, None] + mean * 4 * u
        at += new
    bound += out.abs() * half_step(out_code) + (2.0 ** -25 if out_code == F16 else 1e-37)
    return out, bound
