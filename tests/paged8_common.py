"""Ragged batches over a paged cache of 8-bit codes for the tests, and the operators' definitions in float64 on the CPU."""
import math

import numpy as np
import torch

from tests.paged_common import F32, Batch, half_step

I8, E4M3 = torch.int8, torch.float8_e4m3fn
BLOCK = 16
TOP = {I8: 127.0, E4M3: 448.0}
OVER = {I8: 127.5, E4M3: 464.0}


def values(codes, kind):
    """float64 values of codes given as uint8 bytes; the two e4m3 codes of no number are 480 and -480."""
    if kind == I8:
        return codes.view(torch.int8).double()
    v = codes.view(E4M3).float().double()
    no = (codes & 0x7F) == 0x7F
    return torch.where(no, torch.where(codes >= 0x80, -480.0, 480.0).double(), v)


def encode(y, kind):
    """Codes (uint8 bytes) of float64 values in units of their scale: to nearest, ties to even."""
    if kind == I8:
        return y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    exponent = torch.frexp(y)[1].clamp(min=-5)  # 2^(exponent - 1) at most |y|; 2^-9 is the smallest step
    step = torch.ldexp(torch.ones_like(y), exponent - 4)
    return ((y / step).round() * step).clamp(-448, 448).float().to(E4M3).view(torch.uint8)


class Batch8(Batch):
    """As Batch, of 8-bit codes: blocks that hold tokens have random scales (log2 uniform in `spread`) and random codes
    where tokens are, every other byte is arbitrary and every other scale `fill`. k, v: float64 values."""

    def __init__(self, seqs, kv_heads, hd, page, kind, order="head", seed=0, spare_rows=0, fill=float("nan"),
                 spread=(-7, -4), tokens=True):
        super().__init__(seqs, kv_heads, hd, page, F32, order, seed, spare_rows, tokens=False, fill=0.0)
        self.kind, self.order = kind, order
        self.pool = None
        shape = (self.pages, page, kv_heads, hd)
        self.codes = [torch.randint(0, 256, shape, generator=self.g).to(torch.uint8) for _ in (0, 1)]
        self.scales = [torch.full((self.pages, kv_heads, page // BLOCK), fill) for _ in (0, 1)]
        for s, t in enumerate(self.lens if tokens else []):
            for b in range(-(-max(t, 0) // BLOCK)):
                at, lo = int(self.table[s, b * BLOCK // page]), b * BLOCK % page
                n = min(BLOCK, t - b * BLOCK)
                for i in (0, 1):
                    c = torch.randint(0, 255, (n, kv_heads, hd), generator=self.g)
                    if kind == I8:
                        c = (c - 127).to(torch.int8).view(torch.uint8)
                    else:
                        c = (c + (c >= 127).long()).clamp(max=254).to(torch.uint8)  # (127 and 255 are no numbers)
                    self.codes[i][at, lo:lo + n] = c
                    e = spread[0] + (spread[1] - spread[0]) * torch.rand(kv_heads, generator=self.g)
                    top = 1.0 if kind == I8 else 127 / 448 * 4
                    self.scales[i][at, :, lo // BLOCK] = 2.0 ** e * top
        self.refresh()

    def refresh(self):
        """k and v anew from codes and scales."""
        self.k, self.v = [values(c, self.kind) * s.double().transpose(1, 2).repeat_interleave(BLOCK, 1)[..., None]
                          for c, s in zip(self.codes, self.scales)]

    def device(self, gphq, max_rows=None, max_len=None):
        """(PagedKv8, PagedBatch) on the GPU; the pool's memory in its order."""
        def up(c):
            c = c if self.order == "token" else c.transpose(1, 2)
            c = c.contiguous().cuda().view(self.kind)
            return c if self.order == "token" else c.transpose(1, 2)

        kv = gphq.PagedKv8(*[up(c) for c in self.codes], *[s.cuda() for s in self.scales])
        ints = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()
        b = gphq.PagedBatch(ints(self.starts), ints(self.lens), ints(self.table), self.rows,
                            max(self.new + [0]) if max_rows is None else max_rows,
                            max(self.lens + [0]) if max_len is None else max_len)
        return kv, b

    def block_tops(self, s, n, i):
        """[n][KV heads]: 127 (480) times the scale of each of sequence s's first n tokens: above all its block's values."""
        at = [self.token(s, p) for p in range(n)]
        pg, sl = torch.tensor([a for a, _ in at], dtype=torch.long), torch.tensor([b for _, b in at], dtype=torch.long)
        return (127.0 if self.kind == I8 else 480.0) * self.scales[i][pg, :, sl // BLOCK].double()


def attention64_8(b, q, heads, scale, window=0, floor=2.0 ** -25):
    """The definition in float64, and a bound of what the arithmetic may lose on every output.

    With u = 2^-24. A score: fp32 rows are taken to 2^-23 of the row's largest value (bfloat16 ones of less than 2^-39
    of it, FP16 ones exactly), which costs 2^-22 max |q| sum |k| at most; sums of hd products lose (hd + 4) u of
    the sum of their magnitudes (each term may be cut 2^-25 below the largest), scales and factors 4 u more. An error e
    of the scores changes the quotient by at most (exp(2 e) - 1) sum p |v|. Sums over m keys, exponentials, rescales:
    (2 m + 64) u sum p |v|. A probability times its block's scale is cut off 2^-25 under units in which the largest
    probability is 2^7 or more and the largest block scale 1/2 or more: m 2^-31 of the largest |code| times scale. Of
    16-bit rows in sequences of more than 64 columns it is rounded to FP16: 2^-11 sum p |v|. The result's own rounding:
    half a step of itself, and `floor`, its half step below the type's normal numbers or more."""
    rows, width = q.shape
    hd, group = b.hd, heads // b.kv_heads
    out, tol = (torch.zeros(rows, heads, hd, dtype=torch.float64) for _ in range(2))
    u, half = 2.0 ** -24, half_step(q.dtype)
    q = q.reshape(rows, heads, hd).double()
    for s, (n, t) in enumerate(zip(b.new, b.lens)):
        if n == 0 or t <= 0:
            continue
        k, v = b.keys(s, t)
        tops = b.block_tops(s, t, 1)
        pos = torch.arange(t - n, t)[:, None]
        key = torch.arange(t)
        sees = (key <= pos) & (key > pos - window) if window else key <= pos
        m = sees.sum(1, keepdim=True).double()
        for h in range(heads):
            g, x = h // group, q[b.starts[s]:b.starts[s] + n, h]
            kh, vh = k[:, g], v[:, g]
            w = (x @ kh.T * scale).masked_fill(~sees, -math.inf)
            w = torch.softmax(w, 1).nan_to_num(0.0)
            o, a = w @ vh, w @ vh.abs()
            mag = (x.abs() @ kh.abs().T).masked_fill(~sees, 0).amax(1, keepdim=True)
            span = kh.abs().sum(1).expand(n, -1).masked_fill(~sees, 0).amax(1, keepdim=True)
            e = abs(scale) * ((hd + 8) * u * mag + 2.0 ** -22 * x.abs().amax(1, keepdim=True) * span)
            top = tops[:, g].expand(n, -1).masked_fill(~sees, 0).amax(1, keepdim=True)
            d = (torch.expm1(2 * e) + (2 * m + 64) * u) * a + m * 2.0 ** -31 * top
            if half > u and n * group > 64:
                d = d + 2.0 ** -11 * a
            r = slice(b.starts[s], b.starts[s] + n)
            out[r, h], tol[r, h] = o, d + half * o.abs() * (1 + 2.0 ** -9) + floor
    return out.reshape(rows, width), tol.reshape(rows, width)


def rotated64(x, w, eps, cos, sin, pos):
    """Head RMSNorm (w given) and rotation (cos given) of float64 rows [rows][heads][hd] at their positions."""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if cos is not None:
        c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
        lo, hi = x.chunk(2, -1)
        x = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
    return x


def append64(b, qkv, heads, kn, eps, cos, sin, limit=None):
    """Writes the new tokens' codes and scales into b (block by block, by the definition); tokens at positions past
    `limit` and before 0 are left out, bad pages skipped."""
    G, D, kind = b.kv_heads, b.hd, b.kind
    for s, (n, t) in enumerate(zip(b.new, b.lens)):
        first, end = max(0, t - n), t if limit is None else min(t, limit)
        if end <= first:
            continue
        rows = qkv[b.starts[s] + first - (t - n):b.starts[s] + end - (t - n)].double().view(-1, heads + 2 * G, D)
        pos = torch.arange(first, end)
        both = (rotated64(rows[:, heads:heads + G], kn, eps, cos, sin, pos), rows[:, heads + G:])
        for i, y in enumerate(both):
            y = torch.where(y.abs() <= torch.finfo(F32).max, y, 0.0)
            p = first
            while p < end:
                lo = p // BLOCK * BLOCK
                stop = min(end, lo + BLOCK)
                at, slot = int(b.table[s, p // b.page]), lo % b.page
                if 0 <= at < b.pages:
                    for g in range(G):
                        mine = y[p - first:stop - first, g]
                        most = float(mine.abs().max())
                        scale = float(np.float32(most / TOP[kind]))
                        if most > 0:
                            scale = max(scale, 2.0 ** -126)
                        old = float(b.scales[i][at, g, slot // BLOCK])
                        if p > lo and 0 < old < math.inf:
                            grown, k = old, 0
                            while most > OVER[kind] * grown:
                                grown, k = 2 * grown, k + 1
                            if k:
                                c = b.codes[i][at, slot:slot + p - lo, g]
                                b.codes[i][at, slot:slot + p - lo, g] = encode(values(c, kind) * 2.0 ** -k, kind)
                            scale = grown
                        b.scales[i][at, g, slot // BLOCK] = scale
                        b.codes[i][at, slot + p - lo:slot + stop - lo, g] = encode(mine / scale if scale else mine, kind)
                p = stop
    b.refresh()
