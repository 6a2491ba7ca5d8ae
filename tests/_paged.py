"""Plain 64-bit implementations and batch builders for the tests of the paged K/V cache (host tensors)."""
import math

import torch

D = 128
BF16_HALF = torch.finfo(torch.bfloat16).eps / 2  # 2^-8: the most a rounding to bf16 is off, relative to the value


def rotate64(x, cos, sin, pairing):
    """x [.., 128] f64, cos / sin [128] rows broadcast against it."""
    y = torch.empty_like(x)
    lo, hi = (slice(0, D, 2), slice(1, D, 2)) if pairing == "interleaved" else (slice(0, 64), slice(64, D))
    y[..., lo] = x[..., lo] * cos[..., lo] - x[..., hi] * sin[..., lo]
    y[..., hi] = x[..., lo] * sin[..., lo] + x[..., hi] * cos[..., lo]
    return y


def rotate32(x, cos, sin, pairing):
    """The kernel's own arithmetic: f32, products and sums rounded separately (bit for bit)."""
    x, cos, sin = x.float(), cos.float(), sin.float()
    y = torch.empty_like(x)
    lo, hi = (slice(0, D, 2), slice(1, D, 2)) if pairing == "interleaved" else (slice(0, 64), slice(64, D))
    y[..., lo] = x[..., lo] * cos[..., lo] - x[..., hi] * sin[..., lo]
    y[..., hi] = x[..., lo] * sin[..., lo] + x[..., hi] * cos[..., lo]
    return y


def quantize(x):
    """(codes 0..15 uint8, (step, zero) bf16) of f32 rows, as the format defines them."""
    lo, hi = x.amin(-1), x.amax(-1)
    step = ((hi - lo) / torch.full_like(hi, 15.0)).to(torch.bfloat16).float()
    zero = (lo + 8.0 * step).to(torch.bfloat16).float()
    c = torch.round((x - zero[..., None]) / step[..., None]).clamp(-8, 7)
    c = torch.where(step[..., None] > 0, c, torch.zeros_like(c))
    return (c + 8).to(torch.uint8), torch.stack([step, zero], -1).to(torch.bfloat16)


def pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def stands_for(packed, scale):
    """f64 values of 4-bit rows."""
    s = scale.double()
    return s[..., 1:] + s[..., :1] * (unpack(packed).double() - 8.0)


def allows(p, j, block, window, sink):
    tq, tk = p // block, j // block
    return tk <= tq and (window == 0 or tq - tk < window or tk < sink)


def seen_matrix(nq, n, mask):
    """[nq, n] truth values: which of n keys the last nq positions see; mask (block, window, sink) or None."""
    p = torch.arange(n - nq, n)[:, None]
    j = torch.arange(n)[None]
    if mask is None:
        return torch.ones(nq, n, dtype=torch.bool)
    block, window, sink = mask
    tq, tk = torch.div(p, block, rounding_mode="floor"), j // block
    seen = (tk <= tq) & (p >= 0)
    if window:
        seen &= (tq - tk < window) | (tk < sink)
    return seen


def attend64(q, k, v, mask, scale=None):
    """q [nq, heads, 128], k / v [n, kv_heads, 128] f64 -> (out, sum of w |v|) [nq, heads, 128] f64; rows without keys 0."""
    nq, heads, _ = q.shape
    n, hk, _ = k.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, mag = torch.zeros(nq, heads, D, dtype=torch.float64), torch.zeros(nq, heads, D, dtype=torch.float64)
    if n == 0 or nq == 0:
        return out, mag
    seen = seen_matrix(nq, n, mask)
    for h in range(heads):
        kk, vv = k[:, h * hk // heads], v[:, h * hk // heads]
        s = (q[:, h] @ kk.T * scale).masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(top > -math.inf, top, torch.zeros_like(top)))
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        # (a key that a row does not see has weight 0 whatever its value is)
        some = seen.any(0)
        vv = torch.where(some[:, None], vv, torch.zeros_like(vv))
        out[:, h], mag[:, h] = w @ vv, w @ vv.abs()
    return out, mag


class Case:
    """A ragged batch over a shuffled pool, on the host; `device()` puts it on the GPU."""

    def __init__(self, fmt, kv_len, nq, heads, kv_heads, page_rows, seed=0, spare=3, pad=0, drop=None, poison=False, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.fmt, self.kv_len, self.nq, self.heads, self.kv_heads, self.page_rows = fmt, list(kv_len), list(nq), heads, kv_heads, page_rows
        self.tokens = sum(nq) + pad
        self.max_q, self.max_kv = max(max(nq, default=0), 1), max(max(kv_len, default=0), 1)
        self.width = (self.max_kv + page_rows - 1) // page_rows
        counts = [(n + page_rows - 1) // page_rows for n in kv_len]
        self.pages = sum(counts) + spare
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((len(kv_len), self.width), -1, dtype=torch.int32)
        at = 0
        for s, c in enumerate(counts):
            self.table[s, :c] = order[at:at + c]
            at += c
        self.cu = torch.zeros(len(nq) + 1, dtype=torch.int32)
        self.cu[1:] = torch.tensor(nq, dtype=torch.int32).cumsum(0) if nq else 0
        bf = lambda *sh: torch.randn(*sh, generator=g).to(torch.bfloat16)
        self.q = bf(self.tokens, heads, D) * scale
        self.rows = {}
        shape = (self.pages, kv_heads, page_rows)
        self.pool, self.scales = {}, {}
        for name in ("k", "v"):
            if fmt == "bf16":
                self.pool[name] = torch.full((*shape, D), math.nan).to(torch.bfloat16) if poison else bf(*shape, D)
                vals = [bf(n, kv_heads, D) for n in kv_len]
                put = [(x,) for x in vals]
                self.rows[name] = [x.double() for x in vals]
            else:
                self.pool[name] = torch.randint(0, 256, (*shape, 64), generator=g, dtype=torch.uint8)
                self.scales[name] = torch.full((*shape, 2), math.nan).to(torch.bfloat16) if poison else bf(*shape, 2)
                put, self.rows[name] = [], []
                for n in kv_len:
                    codes, sc = quantize(torch.randn(n, kv_heads, D, generator=g)) if n else (
                        torch.zeros(0, kv_heads, D, dtype=torch.uint8), torch.zeros(0, kv_heads, 2, dtype=torch.bfloat16))
                    put.append((pack(codes), sc))
                    self.rows[name].append(stands_for(pack(codes), sc))
            for s, n in enumerate(kv_len):
                j = torch.arange(n)
                page, row = self.table[s].long()[j // page_rows], j % page_rows
                self.pool[name][page, :, row] = put[s][0]
                if fmt != "bf16":
                    self.scales[name][page, :, row] = put[s][1]
        if drop is not None:  # (block, window, sink): pages of which no row of the call sees a key are given back
            for s, (n, m) in enumerate(zip(kv_len, nq)):
                some = seen_matrix(m, n, drop).any(0)
                for i in range(counts[s]):
                    if not some[i * page_rows:(i + 1) * page_rows].any():
                        self.table[s, i] = -1

    def device(self):
        from fastvideo_rs_b200 import paged
        self.dev = {n: t.cuda() for n, t in self.pool.items()}
        sc = {n: t.cuda() for n, t in self.scales.items()}
        kv = paged.PagedKv(self.dev["k"], self.dev["v"], sc.get("k"), sc.get("v"))
        batch = paged.PagedBatch(self.table.cuda(), torch.tensor(self.kv_len, dtype=torch.int32).cuda(), self.cu.cuda(),
                                 max_q=self.max_q, max_kv=self.max_kv)
        return kv, batch, self.q.cuda()

    def expect(self, mask, scale=None):
        """(out, bound) [tokens, heads, 128] f64 of the rows that belong to a sequence.

        The bound: the output's own rounding 2^-8 |o|; P (4 bits: P times the step) rounded to bf16, 2^-8 of each term, so
        2^-8 sum w |v| (4 bits: |step code| <= |v| + |zero|); scores and sums in f32, whose errors (128 products of size
        |q k| at 2^-24 and, in 4 bits, up to 143 |q| step against an offset) stay below 2^-10 of the terms."""
        outs, bounds = [], []
        for s, (n, m) in enumerate(zip(self.kv_len, self.nq)):
            q = self.q[self.cu[s]:self.cu[s + 1]].double()
            o, mag = attend64(q, self.rows["k"][s], self.rows["v"][s], mask, scale)
            if self.fmt == "q4" and n:
                mag = mag + self._zero(s)
            outs.append(o)
            bounds.append(BF16_HALF * o.abs() + (BF16_HALF + 2.0 ** -10) * mag + 1e-30)
        return torch.cat(outs), torch.cat(bounds)

    def _zero(self, s):
        n, r = self.kv_len[s], self.page_rows
        j = torch.arange(n)
        page = self.table[s].long()[j // r]
        live = page >= 0
        return self.scales["v"][page[live], :, (j % r)[live]][..., 1].double().abs().amax()
