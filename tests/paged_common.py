"""Ragged batches over a paged cache for the tests, and the operators' definitions in float64 on the CPU."""
import math

import numpy as np
import torch

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAN = float("nan")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Batch:
    """`seqs`: (new tokens, tokens in all) of every sequence. Pages are handed out in a shuffled order; every slot
    that holds no token, in its own pages or others, holds `fill`; unused table entries are -1."""

    def __init__(self, seqs, kv_heads, hd, page, dtype, order="head", seed=0, spare_rows=0, fill=NAN, tokens=True):
        self.g = torch.Generator().manual_seed(seed)
        self.new, self.lens = [n for n, _ in seqs], [t for _, t in seqs]
        self.starts = [0]
        for n in self.new:
            self.starts.append(self.starts[-1] + n)
        self.rows = self.starts[-1] + spare_rows
        self.kv_heads, self.hd, self.page, self.dtype = kv_heads, hd, page, dtype
        need = [-(-max(t, 0) // page) for t in self.lens]
        self.pages = sum(need) + 2
        perm = torch.randperm(self.pages, generator=self.g).tolist()
        self.entries = max(need + [1]) + 1
        self.table = np.full((len(seqs), self.entries), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = perm[at:at + n]
            at += n
        shape = (self.pages, page, kv_heads, hd) if order == "token" else (self.pages, kv_heads, page, hd)
        self.pool = [torch.full(shape, fill, dtype=dtype) for _ in range(2)]
        self.k, self.v = [p if order == "token" else p.transpose(1, 2) for p in self.pool]
        if tokens:
            for s, t in enumerate(self.lens):
                for p in range(t):
                    at = (self.table[s, p // page], p % page)
                    self.k[at] = torch.randn(kv_heads, hd, generator=self.g).to(dtype)
                    self.v[at] = (torch.randn(kv_heads, hd, generator=self.g) + 0.25).to(dtype)

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.g)

    def token(self, s, p):
        """The (page, slot) of token p of sequence s."""
        return int(self.table[s, p // self.page]), p % self.page

    def keys(self, s, n):
        """float64 keys and values [n][KV heads][hd] of sequence s's first n tokens."""
        at = [self.token(s, p) for p in range(n)]
        pg, sl = torch.tensor([a for a, _ in at], dtype=torch.long), torch.tensor([b for _, b in at], dtype=torch.long)
        return self.k[pg, sl].double(), self.v[pg, sl].double()

    def device(self, gphq, max_rows=None, max_len=None):
        """(PagedKv, PagedBatch) on the GPU; the pool keeps its order."""
        k, v = [t.clone().cuda() if t.is_contiguous() else t.transpose(1, 2).contiguous().cuda().transpose(1, 2)
                for t in (self.k, self.v)]
        ints = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()
        kv = gphq.PagedKv(k, v)
        b = gphq.PagedBatch(ints(self.starts), ints(self.lens), ints(self.table), self.rows,
                            max(self.new + [0]) if max_rows is None else max_rows,
                            max(self.lens + [0]) if max_len is None else max_len)
        return kv, b


def attention64(b, q, heads, scale, window=0):
    """The definition in float64, and a bound of what fp32 arithmetic may lose on every output.

    With u = 2^-24, a score is a sum of hd products taken in some order, scaled: off by at most (hd + 4) u times the
    sum of its products' magnitudes; a 22-bit split of a row's values adds 2^-22 of the row's largest value times
    the sum of |k|. An error e of the scores changes every probability by a factor within exp(+-e) and so the
    quotient by at most (exp(2 e) - 1) of sum p |v|. The sums over n keys, the exponentials (2 units), the running
    rescales (at most one per 32 keys) and the joins lose at most (2 n + 64) u of sum p |v|; probabilities that
    FP16 pieces cut off at 2^-32 of the largest lose n 2^-32 max |v|. With 16-bit rows each probability is rounded
    to their type once: half a step of sum p |v|. The result's own rounding: half a step of itself."""
    rows, width = q.shape
    hd, group = b.hd, heads // b.kv_heads
    out, tol, mean = (torch.zeros(rows, heads, hd, dtype=torch.float64) for _ in range(3))
    u, half = 2.0 ** -24, half_step(q.dtype)
    q = q.reshape(rows, heads, hd).double()
    for s, (n, t) in enumerate(zip(b.new, b.lens)):
        k, v = b.keys(s, t)
        for i in range(n):
            p = t - n + i
            if p < 0:
                continue
            r, lo = b.starts[s] + i, max(0, p - window + 1) if window else 0
            m = p + 1 - lo
            for h in range(heads):
                kh, vh, x = k[lo:p + 1, h // group], v[lo:p + 1, h // group], q[r, h]
                w = torch.softmax(kh @ x * scale, 0)
                out[r, h] = w @ vh
                a = w @ vh.abs()
                e = abs(scale) * ((hd + 4) * u * float((kh.abs() @ x.abs()).max())
                                  + 2.0 ** -22 * float(x.abs().max() * kh.abs().sum(1).max()))
                tol[r, h] = (math.expm1(2 * e) + (2 * m + 64) * u) * a + m * 2.0 ** -32 * vh.abs().max()
                if half > u:
                    tol[r, h] += half * a
                tol[r, h] += half * out[r, h].abs() + 2.0 ** -25
    return out.reshape(rows, width), tol.reshape(rows, width)
