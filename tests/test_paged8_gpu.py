"""The paged cache in 8 bits on the GPU: append and attention against their definitions in float64, over ragged batches
whose unused bytes are arbitrary and whose unused scales are NaN."""
import functools
import math

import numpy as np
import pytest
import torch

from gophonic_amd import gphq
from tests.paged8_common import BLOCK, E4M3, I8, Batch8, append64, attention64_8, encode, rotated64, values
from tests.paged_common import BF16, F16, F32, NAN, half_step

pytestmark = pytest.mark.gpu

KINDS, KIND_IDS = [I8, E4M3], ["i8", "e4m3"]
ROWS, ROW_IDS = [F32, F16, BF16], ["f32", "f16", "bf16"]


def rope(positions, hd, theta=1e4):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * theta ** (-torch.arange(hd // 2, dtype=torch.float64) * 2 / hd)
    return a.cos().float(), a.sin().float()


def up(t):
    return None if t is None else t.cuda()


def bytes_of(kv):
    return [t.contiguous().view(torch.uint8).cpu() for t in (kv.k, kv.v)]


def same_pool(kv, b):
    """The device's codes and scales are b's, bit for bit."""
    for got, want in zip(bytes_of(kv), b.codes):
        assert torch.equal(got, want), int((got != want).sum())
    for got, want in zip((kv.k_scales, kv.v_scales), b.scales):
        assert torch.equal(got.cpu().view(torch.int32), want.view(torch.int32))


@functools.lru_cache(None)
def two_streams():
    """The file's streams. A process has more streams than hardware queues: each one more that a test takes changes which
    of the streams of later tests share a queue, and wait for each other."""
    return [torch.cuda.Stream() for _ in (0, 1)]


# ---- append ---------------------------------------------------------------------

APPEND = [
    # (new, in all) of the sequences, heads, KV heads, head dim, page, order
    ([(1, 1)], 1, 1, 128, 16, "head"),
    ([(1, 17)], 16, 8, 128, 16, "head"),
    ([(3, 3), (0, 5), (1, 40), (7, 33)], 8, 2, 128, 16, "token"),
    ([(5, 70), (64, 64), (1, 128)], 5, 5, 64, 64, "head"),
    ([(1, n) for n in range(1, 71)], 4, 1, 64, 32, "token"),
    ([(130, 150), (1, 1), (33, 34)], 10, 2, 128, 128, "head"),
    ([(17, 17), (16, 32), (15, 31), (2, 17)], 2, 2, 64, 16, "head"),
    ([(n % 8, n % 8 + n) for n in range(150)], 2, 1, 64, 32, "head"),
]


@pytest.mark.parametrize("form", ["norm+rope", "rope", "norm", "plain"])
@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("rt", ROWS, ids=ROW_IDS)
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(case, rt, kind, form):
    """Codes and scales bit for bit (64-bit arithmetic on both sides; a code would have to lie within 2^-40 of a border
    to differ), queries within fp32's rounding: the norm's sum, root and quotient (hd / 2 + 4) u of a value, the
    rotation 3 u of both magnitudes, the last product u."""
    seqs, heads, G, D, page, order = APPEND[case]
    b = Batch8(seqs, G, D, page, kind, order, seed=case, spare_rows=2)
    width = (heads + 2 * G) * D
    qkv = (b.randn(b.rows, width) * 3).to(rt)
    qn, kn = (1 + 0.2 * b.randn(D), 1 + 0.2 * b.randn(D)) if "norm" in form else (None, None)
    cos, sin = rope(160, D) if "rope" in form else (None, None)
    kv, dev = b.device(gphq)
    wide = torch.full((b.rows, width + 16), NAN, dtype=rt, device="cuda")  # rows in wider buffers
    wide[:, :width] = qkv.cuda()
    q = torch.full((b.rows, heads * D + 8), 7.0, dtype=rt, device="cuda")
    gphq.paged8_append(kv, dev, wide[:, :width], q[:, :heads * D], heads, up(qn), up(kn), 1e-5, up(cos), up(sin), 0.25)
    dev.check()
    append64(b, qkv, heads, kn, 1e-5, cos, sin)
    same_pool(kv, b)
    rows = b.starts[-1]
    pos = torch.tensor([b.lens[s] - b.new[s] + i for s, n in enumerate(b.new) for i in range(n)], dtype=torch.long)
    x = qkv[:rows].double().view(rows, heads + 2 * G, D)[:, :heads]
    want = rotated64(x, qn, 1e-5, cos, sin, pos) * 0.25
    big = rotated64(x, qn, 1e-5, None, None, pos).abs() * 0.25
    big = torch.cat([big[..., :D // 2] + big[..., D // 2:]] * 2, -1) if cos is not None else big
    err = (q[:rows, :heads * D].cpu().double().view(rows, heads, D) - want).abs()
    assert (err <= big * (D / 2 + 8) * 2.0 ** -24 + half_step(rt) * want.abs() * (1 + 2.0 ** -9) + 2.0 ** -25).all()
    assert (q[rows:] == 7).all() and (q[:, heads * D:] == 7).all()


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("hd", [64, 128])
def test_tokens_one_by_one(kind, hd):
    """40 steps of one token, growing and shrinking: scales double when they have to, earlier codes with them; an int8
    value ends within one step of what was stored, an e4m3 value within half a step of its own or of the smallest."""
    G, page = 2, 32
    b = Batch8([(0, 0)], G, hd, page, kind, seed=1, tokens=False)
    b.pages, b.entries = 3, 2
    b.table = np.array([[2, 0]], np.int32)
    b.codes = [torch.randint(0, 256, (3, page, G, hd), generator=b.g).to(torch.uint8) for _ in (0, 1)]
    b.scales = [torch.full((3, G, 2), NAN) for _ in (0, 1)]
    kv, _ = b.device(gphq)
    rows = b.randn(40, 3 * G * hd) * 2.0 ** torch.randint(-3, 4, (40, 1), generator=b.g).float()
    rows[5] *= 1e6
    rows[20:30] *= 1e-8
    rows[30] = 0
    q = torch.empty(1, G * hd, device="cuda")
    for t in range(40):
        b.new, b.lens, b.starts, b.rows = [1], [t + 1], [0, 1], 1
        dev = gphq.PagedBatch(*[torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 1], [t + 1])],
                              torch.from_numpy(b.table).cuda(), 1, 1, 40)
        gphq.paged8_append(kv, dev, rows[t:t + 1].cuda(), q, G)
        dev.check()
        append64(b, rows[t:t + 1], G, None, 0.0, None, None)
    same_pool(kv, b)
    x = rows.double().view(40, 3 * G, hd)
    for i, y in enumerate((b.k, b.v)):
        got = torch.stack([y[b.token(0, p)] for p in range(40)])
        at = [b.token(0, p) for p in range(40)]
        step = torch.stack([b.scales[i][pg, :, sl // BLOCK] for pg, sl in at]).double()[..., None]
        err = (got - x[:, (1 + i) * G:(2 + i) * G]).abs()
        if kind == I8:
            assert (err <= step * (1 + 1e-6)).all()
        else:  # (a first rounding at half a step, and one more where the scale grew below the normal range)
            assert (err <= 2.0 ** -4 * (1 + 1e-6) * x[:, (1 + i) * G:(2 + i) * G].abs() + 2.0 ** -9 * step).all()


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("split", [[40], [1, 39], [15, 1, 24], [16, 16, 8], [7, 9, 16, 8]])
def test_chunks_of_a_prompt(kind, split):
    """A prompt in one call or several: whole blocks come out the same however it is cut."""
    b = Batch8([(40, 40)], 2, 128, 16, kind, seed=2)
    rows = b.randn(40, 6 * 128)
    kv, _ = b.device(gphq)
    q = torch.empty(40, 2 * 128, device="cuda")
    at = 0
    for n in split:
        b.new, b.lens, b.starts, b.rows = [n], [at + n], [0, n], n
        dev = gphq.PagedBatch(*[torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, n], [at + n])],
                              torch.from_numpy(b.table).cuda(), n, n, 40)
        gphq.paged8_append(kv, dev, rows[at:at + n].cuda(), q, 2)
        append64(b, rows[at:at + n], 2, None, 0.0, None, None)
        at += n
    same_pool(kv, b)


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("scale", [0.0, -1.0, math.inf, -math.inf, NAN])
def test_a_block_without_a_scale_gets_one(kind, scale):
    """A block with earlier tokens whose scale is no positive finite number counts as empty."""
    b = Batch8([(2, 20)], 1, 64, 16, kind, seed=3)
    at = int(b.table[0, 1])
    for s in b.scales:
        s[at, 0, 0] = scale
    rows = b.randn(2, 3 * 64)
    kv, dev = b.device(gphq)
    gphq.paged8_append(kv, dev, rows.cuda(), torch.empty(2, 64, device="cuda"), 1)
    append64(b, rows, 1, None, 0.0, None, None)
    same_pool(kv, b)


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("mag", [1e-45, 1e-38, 1e-30, 1.0, 1e30, 3.4e38, 0.0])
def test_magnitudes(kind, mag):
    """From the smallest fp32 number to the largest, and zero; then a token of ordinary size behind them."""
    b = Batch8([(3, 3), (4, 20)], 1, 64, 16, kind, seed=4, spread=(-140, -130))
    rows = (torch.rand(7, 3 * 64, generator=b.g) * 2 - 1).double().mul(mag).float()
    rows[0, 64:] = mag
    rows[3, 64:] = -mag
    kv, dev = b.device(gphq)
    gphq.paged8_append(kv, dev, rows.cuda(), torch.empty(7, 64, device="cuda"), 1)
    dev.check()
    append64(b, rows, 1, None, 0.0, None, None)
    same_pool(kv, b)


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, NAN])
def test_values_that_are_not_finite(kind, bad):
    """Code 0, reported; the block's other values as without them. A normalized key row of one is not finite whole."""
    b = Batch8([(3, 19), (2, 2)], 2, 64, 16, kind, seed=5)
    rows = b.randn(5, 6 * 64)
    rows[1, 2 * 64 + 3] = bad   # a key
    rows[4, 5 * 64 + 60] = bad  # a value
    for kn in (None, torch.ones(64)):
        kv, dev = b.device(gphq)
        gphq.paged8_append(kv, dev, rows.cuda(), torch.empty(5, 128, device="cuda"), 2, None, up(kn))
        with pytest.raises(gphq.GphqError) as e:
            dev.check()
        assert e.value.status == gphq.ERR_NON_FINITE
        dev.check()
        mine = Batch8([(3, 19), (2, 2)], 2, 64, 16, kind, seed=5)
        append64(mine, rows, 2, kn, 1e-6, None, None)
        same_pool(kv, mine)


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
def test_keys_turned_past_fp32_s_range(kind):
    """Finite keys whose rotation is above the largest fp32 number: code 0, reported, in a new block and in one with a
    scale, which stays finite."""
    rows = torch.zeros(3, 3 * 64)
    rows[0, 64], rows[0, 64 + 32] = 3e38, -3e38  # a pair that a turn by 45 degrees makes (4.2e38, 0)
    rows[1] = rows[0]
    rows[1, 65] = 1e38
    rows[2, 64:] = torch.linspace(-1, 1, 128)
    half = torch.full((32, 32), 0.5 ** 0.5)
    b = Batch8([(1, 20), (2, 2)], 1, 64, 16, kind, seed=6)
    kv, dev = b.device(gphq)
    gphq.paged8_append(kv, dev, rows.cuda(), torch.empty(3, 64, device="cuda"), 1, None, None, 0.0, half.cuda(), half.cuda())
    with pytest.raises(gphq.GphqError) as e:
        dev.check()
    assert e.value.status == gphq.ERR_NON_FINITE
    append64(b, rows, 1, None, 0.0, half, half)
    same_pool(kv, b)
    assert kv.k_scales[int(b.table[0, 1]), 0, 0].isfinite()


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("scale", [49.0, 41.0, 2.0 ** 23 + 1])
def test_values_between_two_codes(kind, scale):
    """Quotients that lie between two codes, or so near to there that fp32 has no number between: 49 * (1 / 49) is not
    1 in 64 bits, and (19 * 2^19 + 1) / (2^23 + 1) is 2^-26 of itself below 19 / 16."""
    b = Batch8([(3, 20)], 1, 64, 16, kind, seed=7)
    at = int(b.table[0, 1])
    for s in b.scales:
        s[at] = scale
    if kind == I8:
        ties = torch.arange(-62, 66).double() + 0.5
    else:
        codes = torch.arange(1, 127, dtype=torch.uint8).view(E4M3).double()
        ties = torch.cat([(codes[1:] + codes[:-1]) / 2, torch.tensor([1.1875] * 3).double()])
    y = ties * scale
    below = (y - y.abs() * 2.0 ** -25).float()  # the fp32 number at most y, mostly
    rows = torch.zeros(3, 3 * 64)
    rows[0, 64:], rows[1, 64:], rows[2, 64:] = y.float(), -y.float(), below
    kv, dev = b.device(gphq)
    gphq.paged8_append(kv, dev, rows.cuda(), torch.empty(3, 64, device="cuda"), 1)
    dev.check()
    append64(b, rows, 1, None, 0.0, None, None)
    same_pool(kv, b)
    if kind == E4M3:  # to nearest, said another way: no other code is nearer, of two as near the even one
        all_codes = torch.arange(0, 127, dtype=torch.uint8).view(E4M3).double()
        for r in range(3):
            x = (rows[r, 64:].double() / scale)[:, None]
            d = (x.abs() - all_codes).abs()
            near = d.min(1).values
            even = (d == near[:, None]).long() * (2 - torch.arange(127) % 2)
            want = even.argmax(1) + 128 * (x[:, 0] < 0)
            got = torch.cat([b.codes[i][at, 1 + r, 0].long() for i in (0, 1)])
            assert torch.equal(got, want)


def test_append_in_place_of_the_queries():
    b = Batch8([(5, 9), (1, 20)], 2, 128, 16, I8, seed=3)
    heads, D = 8, 128
    qkv = b.randn(b.rows, (heads + 4) * D).cuda()
    cos, sin = (t.cuda() for t in rope(64, D))
    qn, kn = (1 + 0.1 * b.randn(D)).cuda(), (1 + 0.1 * b.randn(D)).cuda()
    kv, dev = b.device(gphq)
    q = torch.empty(b.rows, heads * D, device="cuda")
    gphq.paged8_append(kv, dev, qkv, q, heads, qn, kn, 1e-6, cos, sin, 0.5)
    kv2, dev2 = b.device(gphq)
    both = qkv.clone()
    gphq.paged8_append(kv2, dev2, both, both, heads, qn, kn, 1e-6, cos, sin, 0.5)
    assert torch.equal(both[:, :heads * D], q) and torch.equal(both[:, heads * D:], qkv[:, heads * D:])
    assert all(torch.equal(x, y) for x, y in zip(bytes_of(kv), bytes_of(kv2)))


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
def test_append_reports_what_it_cannot_place(kind):
    """A bad page stores nothing of its tokens, a bad sequence is skipped whole, a position past the table or before 0
    is skipped; the other rows are as without them."""
    heads, D, page = 2, 64, 16
    b = Batch8([(2, 20), (3, 40), (2, 5), (3, 52), (2, 1), (2, 18)], 1, D, page, kind, seed=4)
    b.table[1, 2] = b.pages  # the page of tokens 37, 38 and 39, all that sequence 1 brings: one past the pool
    b.table[5, 1] = -7       # tokens 16, 17 of the last sequence
    qkv = b.randn(b.rows, (heads + 2) * D)
    cos, sin = rope(50, D)   # positions 50 and 51 are past it, 49 is not
    kv, dev = b.device(gphq)
    q = torch.full((b.rows, heads * D), 7.0, device="cuda")
    gphq.paged8_append(kv, dev, qkv.cuda(), q, heads, None, None, 0.0, cos.cuda(), sin.cuda())
    with pytest.raises(gphq.GphqError) as e:
        dev.check()
    assert e.value.status == gphq.ERR_PAGED_BATCH
    dev.check()  # cleared
    assert (q[[8, 9, 10]] == 7).all()  # positions 50, 51, and token -1 of sequence 4, whose length is below its rows
    assert (q[[0, 1, 2, 3, 4, 5, 6, 7, 11, 12, 13]] != 7).all()
    append64(b, qkv, heads, None, 0.0, cos, sin, limit=50)
    same_pool(kv, b)


@pytest.mark.parametrize("starts,good", [([0, 4, 2, 6], []), ([0, 2, 4, 9], [0, 1, 2, 3]), ([-1, 2, 4, 6], [2, 3, 4, 5]),
                                         ([0, 5, 5, 6], [5]), ([2 ** 31 - 1, -2 ** 31, 4, 6], [4, 5])])
def test_bad_sequences_are_left_alone(starts, good):
    """Starts that descend, leave the rows or give a sequence more than max_rows rows: flagged, its rows untouched."""
    b = Batch8([(2, 20)] * 3, 1, 64, 16, I8, seed=6)
    kv, _ = b.device(gphq)
    dev = gphq.PagedBatch(*[torch.tensor(v, dtype=torch.int32, device="cuda") for v in (starts, b.lens)],
                          torch.from_numpy(b.table).cuda(), 6, 2, 20)
    q, out = (torch.full((6, 64), 7.0, device="cuda") for _ in (0, 1))
    other = [r for r in range(6) if r not in good]
    rows = b.randn(6, 3 * 64)
    gphq.paged8_append(kv, dev, rows.cuda(), q, 1)
    with pytest.raises(gphq.GphqError) as e:
        dev.check()
    assert e.value.status == gphq.ERR_PAGED_BATCH
    gphq.paged8_attention(kv, dev, rows[:, :64].contiguous().cuda(), out, 1, 1.0)
    with pytest.raises(gphq.GphqError) as e:
        dev.check()
    assert e.value.status == gphq.ERR_PAGED_BATCH
    for t in (q, out):
        assert (t[other] == 7).all() and (t[good] != 7).all()
    live = [s for s in range(3) if starts[s] in good]
    b.starts = [starts[s] if s in live else 0 for s in range(3)] + [6]
    b.new = [starts[s + 1] - starts[s] if s in live else 0 for s in range(3)]
    append64(b, rows, 1, None, 0.0, None, None)
    same_pool(kv, b)


@pytest.mark.parametrize("starts,good", [([0, 20, 40, 90], range(40)), ([0, 50, 50, 60], range(50, 60)),
                                         ([-10, 20, 40, 60], range(20, 60)), ([0, 40, 20, 60], []),
                                         ([2 ** 31 - 1, -2 ** 31, 40, 60], range(40, 60))])
def test_bad_sequences_of_many_rows_are_left_alone(starts, good):
    """The same where a sequence has more than a few rows."""
    b = Batch8([(20, 50)] * 3, 2, 64, 16, I8, seed=6)
    kv, _ = b.device(gphq)
    dev = gphq.PagedBatch(*[torch.tensor(v, dtype=torch.int32, device="cuda") for v in (starts, b.lens)],
                          torch.from_numpy(b.table).cuda(), 60, 20, 50)
    q, good = torch.full((60, 128), 7.0, device="cuda"), list(good)
    other = [r for r in range(60) if r not in good]
    rows = b.randn(60, 6 * 64)
    gphq.paged8_append(kv, dev, rows.cuda(), q, 2)
    with pytest.raises(gphq.GphqError) as e:
        dev.check()
    assert e.value.status == gphq.ERR_PAGED_BATCH
    assert (q[other] == 7).all() and (q[good] != 7).all()
    live = [s for s in range(3) if starts[s] in good]
    b.starts = [starts[s] if s in live else 0 for s in range(3)] + [60]
    b.new = [starts[s + 1] - starts[s] if s in live else 0 for s in range(3)]
    append64(b, rows, 2, None, 0.0, None, None)
    same_pool(kv, b)


def test_append_in_a_batch_of_many_idle_sequences():
    """More sequences than the first search takes at once, most without rows; single tokens beside short prompts."""
    seqs = [((0, 5), (1, 1 + n % 40), (0, 1), (n % 30, n % 30 + 7))[n % 4] if n % 11 == 0 else (0, 3) for n in range(5000)]
    b = Batch8(seqs, 1, 64, 16, I8, seed=8)
    rows = b.randn(b.rows, 3 * 64)
    for few in (False, True):  # (fewer sequences than rows: blocks by their numbers; else by rows)
        if few:
            b = Batch8([s for s in seqs if s[0]], 1, 64, 16, I8, seed=8)
        kv, dev = b.device(gphq)
        gphq.paged8_append(kv, dev, rows.cuda(), torch.empty(b.rows, 64, device="cuda"), 1)
        dev.check()
        append64(b, rows, 1, None, 0.0, None, None)
        same_pool(kv, b)


# ---- attention ------------------------------------------------------------------

ATTEND = [
    ([(1, 1)], 1, 1, 128, 16, "head"),
    ([(1, 17)], 16, 8, 128, 16, "head"),
    ([(1, 1500)], 8, 2, 64, 16, "token"),
    ([(3, 3), (0, 5), (1, 40), (7, 33)], 8, 2, 128, 16, "token"),
    ([(5, 70), (64, 64), (1, 128)], 5, 5, 64, 64, "head"),
    ([(1, n) for n in range(1, 71)], 4, 1, 64, 32, "token"),
    ([(130, 150), (1, 1), (33, 34)], 10, 2, 128, 128, "head"),
    ([(70, 600)], 8, 1, 128, 32, "head"),
    ([(300, 300), (1, 299), (2, 700)], 4, 2, 128, 32, "token"),
    ([(200, 900)], 2, 1, 64, 256, "token"),
]


def attend(b, q, heads, scale, window=0, **over):
    kv, dev = b.device(gphq, **over)
    out = torch.full((b.rows, heads * b.hd), 7.0, dtype=q.dtype, device="cuda")
    gphq.paged8_attention(kv, dev, q.cuda(), out, heads, scale, window)
    dev.check()
    return out.cpu()


def close(b, q, heads, scale, window, got):
    want, tol = attention64_8(b, q, heads, scale, window)
    rows = b.starts[-1]
    err = (got[:rows].double() - want[:rows]).abs()
    assert (err <= tol[:rows]).all(), (float((err / tol[:rows]).max()), float(err.max()))
    assert (got[rows:] == 7).all()


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("rt", ROWS, ids=ROW_IDS)
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention(case, rt, kind):
    seqs, heads, G, D, page, order = ATTEND[case]
    b = Batch8(seqs, G, D, page, kind, order, seed=case, spare_rows=2)
    q = (b.randn(b.rows, heads * D)).to(rt)
    close(b, q, heads, D ** -0.5, 0, attend(b, q, heads, D ** -0.5))


@pytest.mark.parametrize("window", [1, 15, 100])
@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("rt", ROWS, ids=ROW_IDS)
def test_attention_window(rt, kind, window):
    b = Batch8([(1, 5), (3, 300), (90, 400), (1, 1000), (17, 17)], 2, 128, 16, kind, seed=20)
    q = b.randn(b.rows, 8 * 128).to(rt)
    close(b, q, 8, 0.1, window, attend(b, q, 8, 0.1, window))


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-30, 30.0])
@pytest.mark.parametrize("rt", ROWS, ids=ROW_IDS)
def test_scales_of_every_kind(rt, scale):
    b = Batch8([(1, 100), (40, 90)], 1, 64, 16, I8, seed=21)
    q = (b.randn(b.rows, 4 * 64) * 0.1).to(rt)
    close(b, q, 4, scale, 0, attend(b, q, 4, scale))


@pytest.mark.parametrize("spread", [(-100, -100), (90, 100), (-40, 0), (-118, -117)])
@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("rt", [F32, BF16], ids=["f32", "bf16"])
def test_block_scales_of_every_size(rt, kind, spread):
    """Values far from 1, and blocks whose scales lie 2^40 apart."""
    b = Batch8([(1, 200), (40, 100), (3, 33)], 1, 64, 16, kind, seed=22, spread=spread)
    for s in b.scales[:1]:  # keys of ordinary size
        s.copy_(torch.where(s.isnan(), s, 2.0 ** -6))
    b.refresh()
    q = b.randn(b.rows, 2 * 64).to(rt)
    got = attend(b, q, 2, 0.125).double()
    # fp32 and bfloat16 results below 2^-126 have steps of 2^-149 and 2^-133. (A floor of 2^-25, added to bounds of
    # 1e-33 and taken off again, would leave 0 of them: float64 has 53 bits.)
    want, tol = attention64_8(b, q, 2, 0.125, floor=2.0 ** -133)
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("rt", ROWS, ids=ROW_IDS)
def test_what_a_row_does_not_see_does_not_reach_it(rt, kind):
    """Later blocks of the sequence with scales of any kind, seen by some rows of a tile and not by others: those that
    do not see them are as without them, bit for bit; those that do are not finite where the scale is not."""
    for seqs, first in (([(20, 40)], 32), ([(100, 120)], 96), ([(3, 34)], 32)):
        b = Batch8(seqs, 1, 128, 16, kind, seed=23)
        n, t = seqs[0]
        q = b.randn(b.rows, 2 * 128).to(rt)
        plain = attend(b, q, 2, 0.1)
        early = max(0, first - (t - n))
        for scale in (NAN, math.inf, 1e30, 0.0):
            for which in (0, 1):
                c = Batch8(seqs, 1, 128, 16, kind, seed=23)
                for p in range(first, t, BLOCK):
                    pg, sl = c.token(0, p)
                    c.scales[which][pg, 0, sl // BLOCK] = scale
                assert torch.equal(attend(c, q, 2, 0.1)[:early], plain[:early])
        # (every row behind `first` sees a block whose scale of V is NaN: none of its values is a number)
        c = Batch8(seqs, 1, 128, 16, kind, seed=23)
        pg, sl = c.token(0, first)
        c.scales[1][pg, 0, sl // BLOCK] = NAN
        assert attend(c, q, 2, 0.1)[early:].isnan().all()


def test_codes_of_no_number_read_as_480():
    b = Batch8([(1, 30), (70, 90)], 1, 64, 16, E4M3, seed=24)
    for c in b.codes:
        c[:, 3] = 0x7F
        c[:, 9, :, ::2] = 0xFF
    b.refresh()
    q = (b.randn(b.rows, 2 * 64) * 0.1).half()
    close(b, q, 2, 0.1, 0, attend(b, q, 2, 0.1))


@pytest.mark.parametrize("seqs", [[(1, 100)], [(80, 100)]])
@pytest.mark.parametrize("rt", ROWS, ids=ROW_IDS)
def test_bad_pages_read_as_masked_keys(seqs, rt):
    """A page number outside the pool: its keys are not seen, reported; a row of bad pages alone is 0."""
    for bad in (-1, None, 2 ** 31 - 1):
        b = Batch8(seqs, 1, 64, 16, I8, seed=25)
        q = b.randn(b.rows, 64).to(rt)
        n, t = seqs[0]
        b.table[0, 2] = b.pages if bad is None else bad
        kv, dev = b.device(gphq)
        out = torch.full((b.rows, 64), 7.0, dtype=rt, device="cuda")
        gphq.paged8_attention(kv, dev, q.cuda(), out, 1, 0.2)
        with pytest.raises(gphq.GphqError) as e:
            dev.check()
        assert e.value.status == gphq.ERR_PAGED_BATCH
        k, v = [torch.cat([x[int(p)] if 0 <= p < b.pages else torch.full_like(x[0], NAN) for p in b.table[0, :7]])[:t, 0]
                for x in (b.k, b.v)]
        good = ~k[:, 0].isnan()
        for i in range(n):
            sees = good & (torch.arange(t) <= t - n + i)
            w = torch.softmax(k[sees] @ q[i].double() * 0.2, 0)
            want = w @ v[sees]
            assert (out[i].cpu().double() - want).abs().max() <= 2.0 ** -7 * (w @ v[sees].abs()).max()
        b.table[0, :-1] = -1
        kv, dev = b.device(gphq)
        gphq.paged8_attention(kv, dev, q.cuda(), out, 1, 0.2)
        assert (out == 0).all()


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("rt", ROWS, ids=ROW_IDS)
def test_few_rows_in_a_batch_of_many_sequences(rt, kind):
    """A batch made for many sequences, of which three bring rows: the row kernel's grid is by row."""
    seqs = [(0, 30 if i % 7 == 0 else 0) for i in range(300)]
    for i, v in ((3, (1, 200)), (150, (2, 70)), (299, (1, 1))):
        seqs[i] = v
    b = Batch8(seqs, 2, 128, 16, kind, seed=26)
    q = b.randn(b.rows, 6 * 128).to(rt)
    close(b, q, 6, 0.1, 0, attend(b, q, 6, 0.1))


@pytest.mark.parametrize("rt", ROWS, ids=ROW_IDS)
@pytest.mark.parametrize("hd", [64, 128])
def test_long_splits(hd, rt):
    """Caches long enough that a split is many steps, and the table of one passes 64 entries."""
    b = Batch8([(1, 9000), (2, 3000), (1, 1025)], 1, hd, 16, I8, seed=27)
    q = b.randn(b.rows, 4 * hd).to(rt)
    close(b, q, 4, hd ** -0.5, 0, attend(b, q, 4, hd ** -0.5))
    b = Batch8([(40, 5000)], 1, hd, 16, E4M3, seed=28)
    q = b.randn(b.rows, 4 * hd).to(rt)
    close(b, q, 4, hd ** -0.5, 0, attend(b, q, 4, hd ** -0.5))


@pytest.mark.parametrize("rt,mag", [(F32, 1e-38), (F32, 1e30), (F16, 6e4), (BF16, 1e30), (BF16, 1e-30)])
def test_rows_out_of_fp16_s_range(rt, mag):
    b = Batch8([(1, 50), (70, 80)], 1, 128, 16, I8, seed=29)
    q = (b.randn(b.rows, 2 * 128).clamp(-1, 1).double() * mag).to(rt)
    scale = 0.3 / mag
    if scale > 1e29:
        scale = 1e29
    close(b, q, 2, scale, 0, attend(b, q, 2, scale))


@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("hd,page,order", [(128, 16, "head"), (64, 64, "token")])
@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("rt", ROWS, ids=ROW_IDS)
def test_long_prompts(rt, kind, hd, page, order, window):
    """Sequences of a thousand columns and more, whose tiles are the widest, split and whole."""
    b = Batch8([(260, 700)], 1, hd, page, kind, order, seed=33)
    q = b.randn(b.rows, 8 * hd).to(rt)
    close(b, q, 8, hd ** -0.5, window, attend(b, q, 8, hd ** -0.5, window))
    b = Batch8([(200, 200), (257, 300), (300, 301)], 2, hd, page, kind, order, seed=34)
    q = b.randn(b.rows, 10 * hd).to(rt)
    close(b, q, 10, hd ** -0.5, window, attend(b, q, 10, hd ** -0.5, window))


@pytest.mark.parametrize("heads,kv_heads", [(32, 1), (64, 2), (17, 1), (33, 1), (64, 1), (65, 1), (128, 1)])
@pytest.mark.parametrize("rt", ROWS, ids=ROW_IDS)
def test_groups_of_every_size_among_idle_sequences(rt, heads, kv_heads):
    """Single rows of more than one set of columns, in batches of few and of many sequences."""
    for idle in (0, 150):
        seqs = [(1, 300), (1, 33)] + [(0, 20)] * idle + [(1, 100)]
        b = Batch8(seqs, kv_heads, 64, 16, I8, seed=35)
        q = b.randn(b.rows, heads * 64).to(rt)
        close(b, q, heads, 0.125, 0, attend(b, q, heads, 0.125))


@pytest.mark.parametrize("heads,kv_heads,rows", [(4, 1, 4), (4, 1, 5), (4, 1, 8), (4, 1, 9), (4, 1, 16), (4, 1, 17), (8, 8, 64),
                                                 (8, 8, 65), (5, 1, 6), (5, 1, 13)])
@pytest.mark.parametrize("rt", ROWS, ids=ROW_IDS)
def test_columns_on_both_sides_of_the_kernels(rt, heads, kv_heads, rows):
    b = Batch8([(rows, 700), (1, 40)], kv_heads, 64, 16, E4M3, seed=36)
    q = b.randn(b.rows, heads * 64).to(rt)
    close(b, q, heads, 0.125, 0, attend(b, q, heads, 0.125))
    b = Batch8([(rows, 700)], kv_heads, 64, 16, I8, seed=37)
    q = b.randn(b.rows, heads * 64).to(rt)
    close(b, q, heads, 0.125, 0, attend(b, q, heads, 0.125))


def test_pages_of_4096_tokens_and_pools_of_one():
    """The largest page, one page, one head: strides that are never taken."""
    b = Batch8([(3, 700), (70, 4100)], 1, 64, 4096, I8, seed=38)
    q = b.randn(b.rows, 2 * 64)
    close(b, q, 2, 0.125, 0, attend(b, q, 2, 0.125))
    qkv = b.randn(b.rows, 4 * 64)
    kv, dev = b.device(gphq)
    gphq.paged8_append(kv, dev, qkv.cuda(), torch.empty(b.rows, 128, device="cuda"), 2)
    dev.check()
    append64(b, qkv, 2, None, 0.0, None, None)
    same_pool(kv, b)
    k = torch.zeros(1, 16, 1, 64, dtype=torch.int8, device="cuda")
    s = torch.zeros(1, 1, 1, device="cuda")
    kv = gphq.PagedKv8(k, k.clone(), s, s.clone())
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    dev = gphq.PagedBatch(ints([0, 16]), ints([16]), ints([[0]]), 16, 16, 16)
    qkv, q, out = torch.randn(16, 192, device="cuda"), torch.empty(16, 64, device="cuda"), torch.empty(16, 64, device="cuda")
    gphq.paged8_append(kv, dev, qkv, q, 1)
    gphq.paged8_attention(kv, dev, q, out, 1, 0.125)
    dev.check()
    x = values(kv.v.view(torch.uint8).cpu(), I8)[0, :, 0] * float(kv.v_scales)
    assert (out[0].cpu().double() - x[0]).abs().max() <= 2.0 ** -20 * x[0].abs().max()


def test_two_calls_at_once():
    """Two streams over one pool, each with a workspace of its own."""
    b = Batch8([(1, 3000), (1, 2500)], 2, 128, 16, I8, seed=39)
    q = b.randn(b.rows, 8 * 128)
    want = attend(b, q, 8, 0.1)
    kv, dev = b.device(gphq)
    qd = q.cuda()
    streams, outs = two_streams(), [torch.zeros(2, 1024, device="cuda") for _ in (0, 1)]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, out in zip(streams, outs):
            gphq.paged8_attention(kv, dev, qd, out, 8, 0.1, stream=st)
    torch.cuda.synchronize()
    assert all(torch.equal(out.cpu(), want) for out in outs)


def test_views_strides_another_stream_and_repeats():
    """Pages and scales that are views of larger pools, rows of wider buffers, a side stream; the same bits each time."""
    b = Batch8([(1, 700), (66, 90), (3, 40)], 2, 128, 32, I8, seed=30)
    q = b.randn(b.rows, 4 * 128)
    plain = attend(b, q, 4, 0.1)
    kv, dev = b.device(gphq)
    big = [torch.zeros(b.pages, 3, 2, 32, 128 + 16, dtype=torch.int8, device="cuda") for _ in (0, 1)]
    bs = [torch.full((b.pages, 5, 2, 2), NAN, device="cuda") for _ in (0, 1)]
    views = []
    for i, (t, s) in enumerate(((kv.k, kv.k_scales), (kv.v, kv.v_scales))):
        big[i][:, 1, :, :, :128] = t.transpose(1, 2)
        bs[i][:, 3] = s
        views.append((big[i][:, 1, :, :, :128].transpose(1, 2), bs[i][:, 3]))
    kv2 = gphq.PagedKv8(views[0][0], views[1][0], views[0][1], views[1][1])
    wide = torch.zeros(b.rows, 4 * 128 + 32, device="cuda")
    wide[:, 16:16 + 512] = q.cuda()
    out = torch.zeros(b.rows, 512 + 64, device="cuda")
    side = two_streams()[0]
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            gphq.paged8_attention(kv2, dev, wide[:, 16:528], out[:, :512], 4, 0.1)
        gphq.paged8_attention(kv2, dev, wide[:, 16:528], out[:, :512], 4, 0.1, stream=side)
        side.synchronize()
        assert torch.equal(out[:, :512].cpu(), plain) and (out[:, 512:] == 0).all()


def test_offsets_past_32_bits():
    """Pages far into a pool of more than 4 GiB."""
    pages, G, T, D = 40000, 8, 128, 128
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GiB of device memory")
    k = torch.zeros(pages, G, T, D, dtype=torch.int8, device="cuda").transpose(1, 2)
    v = torch.zeros(pages, G, T, D, dtype=torch.int8, device="cuda").transpose(1, 2)
    assert k.numel() > 1 << 32
    ks, vs = (torch.full((pages, G, T // 16), NAN, device="cuda") for _ in (0, 1))
    kv = gphq.PagedKv8(k, v, ks, vs)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(200, 3 * G * D, generator=g)
    far = gphq.PagedBatch(ints([0, 200]), ints([200]), ints([[pages - 1, pages - 2]]), 200, 200, 200)
    near = gphq.PagedBatch(ints([0, 200]), ints([200]), ints([[0, 1]]), 200, 200, 200)
    outs = []
    for batch in (far, near):
        q, out = torch.empty(200, G * D, device="cuda"), torch.empty(200, G * D, device="cuda")
        gphq.paged8_append(kv, batch, qkv.cuda(), q, G)
        gphq.paged8_attention(kv, batch, q, out, G, 0.1)
        batch.check()
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and outs[0].isfinite().all()
    for t in (k, v):
        assert torch.equal(t[pages - 1], t[0]) and t[0].count_nonzero() > 0 and t[pages // 2].count_nonzero() == 0


def test_captured_steps_follow_the_lengths():
    """One captured append and attention of three requests, replayed as they grow; each replay against an eager call."""
    heads, G, D, page = 4, 2, 128, 16
    b = Batch8([(1, 20), (1, 33), (1, 47)], G, D, page, I8, seed=31)
    kv, _ = b.device(gphq)
    kv2, _ = b.device(gphq)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    starts, lens = ints([0, 1, 2, 3]), ints([20, 33, 47])
    table = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    table[:, :b.entries] = torch.from_numpy(b.table).cuda()
    spare = [p for p in range(b.pages) if p not in set(b.table.flatten().tolist())]
    table[2, 3] = spare[0]
    dev = gphq.PagedBatch(starts, lens, table, 3, 1, 60)
    qkv, q, out = (torch.randn(3, n * D, device="cuda") for n in (heads + 2 * G, heads, heads))
    work = torch.empty(max(16, gphq.paged8_attention_workspace_bytes(kv, dev, F32, heads)), dtype=torch.uint8, device="cuda")

    def step(kv, q, out):
        gphq.paged8_append(kv, dev, qkv, q, heads)
        gphq.paged8_attention(kv, dev, q, out, heads, 0.1, work=work)

    side = two_streams()[0]
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step(kv, q, out)
    torch.cuda.synchronize()
    q2, out2 = torch.empty_like(q), torch.empty_like(out)
    for _ in range(5):
        qkv.normal_()
        graph.replay()
        torch.cuda.synchronize()
        step(kv2, q2, out2)
        assert torch.equal(q, q2) and torch.equal(out, out2)
        assert all(torch.equal(x, y) for x, y in zip(bytes_of(kv), bytes_of(kv2)))
        lens += 1
    dev.check()


def test_loose_bounds_and_no_rows():
    """Bounds wider than the batch, rows before the first sequence: the same rows; a batch of none leaves all alone."""
    b = Batch8([(1, 300), (5, 40)], 1, 64, 16, E4M3, seed=32)
    q = b.randn(b.rows, 4 * 64)
    tight = attend(b, q, 4, 0.1)
    entries = -(-1000 // 16)
    b.table = np.concatenate([b.table, np.full((2, entries - b.entries), -1, np.int32)], 1)
    loose = attend(b, q, 4, 0.1, max_rows=6, max_len=1000)
    close(b, q, 4, 0.1, 0, tight)
    close(b, q, 4, 0.1, 0, loose)
    kv, _ = b.device(gphq)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    dev = gphq.PagedBatch(ints([2, 2, 2]), ints(b.lens), torch.from_numpy(b.table).cuda(), 6, 6, 1000)
    out = torch.full((6, 256), 7.0, device="cuda")
    before = bytes_of(kv)
    gphq.paged8_attention(kv, dev, q.cuda(), out, 4, 0.1)
    gphq.paged8_append(kv, dev, torch.randn(6, 6 * 64, device="cuda"), out, 4)
    dev.check()
    assert (out == 7).all() and all(torch.equal(x, y) for x, y in zip(before, bytes_of(kv)))


def test_wrong_tensors_are_refused():
    k = torch.zeros(2, 16, 1, 64, dtype=torch.int8, device="cuda")
    s = torch.ones(2, 1, 1, device="cuda")
    kv = gphq.PagedKv8(k, k.clone(), s, s.clone())
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    dev = gphq.PagedBatch(ints([0, 1]), ints([3]), ints([[0]]), 1, 1, 3)
    q = torch.zeros(1, 64, device="cuda")
    for f in (lambda: gphq.paged8_attention(kv, dev, q, q.half(), 1, 1.0),
              lambda: gphq.paged8_attention(kv, dev, q, q.cpu(), 1, 1.0),
              lambda: gphq.paged8_attention(kv, dev, q, q[:, :32], 1, 1.0),
              lambda: gphq.paged8_attention(kv, dev, q, q, 1, 1.0),
              lambda: gphq.paged8_append(kv, dev, q, q.clone(), 1),
              lambda: gphq.paged8_append(kv, dev, torch.zeros(1, 192, device="cuda"), q, 1, q_norm=q[0, :32]),
              lambda: gphq.paged_attention(kv, dev, q, q.clone(), 1, 1.0)):
        with pytest.raises((gphq.GphqError, AttributeError)):
            f()


# ---- the batched pass over a pool of codes ----------------------------------------

GEOM = dict(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=128, intermediate=1024, vocab=300, max_positions=640,
            eps=1e-6, rope_theta=1e6)


@pytest.fixture(scope="module")
def lm():
    return gphq.lm_random(GEOM, gphq.FMT_Q8B, 5)[0]


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
def test_paged_pass_stores_the_rounded_rows_of_an_fp32_pool(lm, kind):
    """Layer 0 sees the same inputs in both: its values are off by half a code at most (int8: half a scale; e4m3: 2^-4
    of the value, or half of 2^-9 of the scale), where a block is whole; and the passes' states stay near: an int8
    value of the two layers is off by less than 1/254 of its block's largest, an e4m3 one by 1/16 of itself."""
    rng = np.random.default_rng(2)
    ids = rng.integers(0, GEOM["vocab"], 77).astype(np.int32)
    table = rng.permutation(9)[None, :5].astype(np.int32)
    pf, states, pools = gphq.Prefill(lm, 512), [], []
    for dtype in (F32, kind):
        pool = gphq.PagedPool(lm, 9, 16, dtype)
        h = torch.empty(1, GEOM["hidden"], device="cuda")
        pf.paged(pool, [ids], [0], table, h)
        pf.check()
        states.append(h.double().flatten())
        pools.append(pool)
    wide, mine = pools[0].layer(0), pools[1].layer(0)
    for x, c, s in ((wide.k, mine.k, mine.k_scales), (wide.v, mine.v, mine.v_scales)):
        for p in range(77):
            pg, sl = int(table[0, p // 16]), p % 16
            scale = s[pg, :, 0].double()[:, None]
            got = values(c[pg, sl].view(torch.uint8).cpu(), kind).cuda() * scale
            want = x[pg, sl].double()
            room = 0.5 * scale if kind == I8 else torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * scale)
            assert ((got - want).abs() <= room * (1 + 1e-4) + 1e-6 * want.abs().max()).all()
    a, b = states
    assert float(a @ b / (a.norm() * b.norm())) >= (0.999 if kind == I8 else 0.98)


def test_paged_pass_in_pieces(lm):
    """Prompts whole and in chunks of one block, two requests, then single tokens over the same int8 pages."""
    rng = np.random.default_rng(3)
    ids = [rng.integers(0, GEOM["vocab"], n).astype(np.int32) for n in (64, 48)]
    table = np.array([[3, 1, 4, 9], [2, 6, 5, -1]], np.int32)
    pools = [gphq.PagedPool(lm, 12, 16, I8) for _ in (0, 1)]
    pf = gphq.Prefill(lm, 128)
    h = torch.empty(2, GEOM["hidden"], device="cuda")
    pf.paged(pools[0], ids, [0, 0], table, h)
    h2 = torch.empty(2, GEOM["hidden"], device="cuda")
    for lo in (0, 16, 32):
        pf.paged(pools[1], [x[lo:lo + 16] for x in ids], [lo, lo], table, h2)
    one = torch.empty(1, GEOM["hidden"], device="cuda")
    pf.paged(pools[1], [ids[0][48:]], [48], table[:1], one)
    pf.check()
    # The same tokens, whole blocks each time: rows' projections may differ in their last bits between passes of other
    # sizes, so a code may be the next one.
    for layer in range(GEOM["layers"]):
        a, b = pools[0].layer(layer), pools[1].layer(layer)
        for p in (3, 1, 4, 9, 2, 6, 5):
            assert (a.k[p].int() - b.k[p].int()).abs().max() <= 2 and (a.v[p].int() - b.v[p].int()).abs().max() <= 2
    x, y = h[0].double(), one[0].double()
    assert float(x @ y / (x.norm() * y.norm())) >= 0.999
    pf.paged(pools[1], [[7], [8]], [64, 48], np.array([[3, 1, 4, 9, 0], [2, 6, 5, 7, -1]], np.int32), h2)
    pf.check()
    assert h2.isfinite().all()


def test_pool_of_codes(lm):
    pool = gphq.PagedPool(lm, 5, 32, E4M3)
    kv = pool.layer(1)
    assert kv.k.shape == (5, 32, 2, 128) and kv.k.dtype == E4M3 and kv.k_scales.shape == (5, 2, 2)
    other = gphq.PagedPool(lm, 5, 32, F16)
    import ctypes

    d = gphq.PagedKv8Desc()
    assert gphq.load().gphq_paged_pool_layer8(other.h, 0, ctypes.byref(d)) == gphq.ERR_UNSUPPORTED
    assert gphq.load().gphq_paged_pool_layer8(pool.h, 2, ctypes.byref(d)) == gphq.ERR_PAGED_SHAPE
    with pytest.raises(gphq.GphqError):
        gphq.PagedPool(lm, 5, 32, torch.uint8)
