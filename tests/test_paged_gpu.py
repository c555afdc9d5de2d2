"""The paged cache on the GPU: append and attention against their definitions in float64, over ragged batches whose
unused slots hold NaN."""
import math

import numpy as np
import pytest
import torch

from gophonic_amd import gphq
from tests.paged_common import BF16, F16, F32, NAN, Batch, attention64, half_step

pytestmark = pytest.mark.gpu

TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]
TYPE_IDS = ["f32-f32", "f32-f16", "f32-bf16", "f16-f16", "bf16-bf16"]


def rope(positions, hd, theta=1e4):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * theta ** (-torch.arange(hd // 2, dtype=torch.float64) * 2 / hd)
    return a.cos().float(), a.sin().float()


# ---- append ---------------------------------------------------------------------


def append64(b, qkv, heads, qn, kn, eps, cos, sin, q_scale):
    """float64 queries, and the pools with the new tokens; bounds of what fp32 arithmetic may lose of each: the norm's
    sum of hd squares, root and quotient are off by at most (hd / 2 + 4) u of a value, the rotation's two products and
    their sum by 3 u of both magnitudes, the last product by u."""
    G, D, u = b.kv_heads, b.hd, 2.0 ** -24
    x = qkv.double().view(b.rows, heads + 2 * G, D)
    seq = [s for s, n in enumerate(b.new) for _ in range(n)]
    pos = torch.tensor([b.lens[s] - b.starts[s + 1] + r for r, s in enumerate(seq)], dtype=torch.long)
    rows = len(seq)

    def head(h, w):
        if w is not None:
            h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double()
        big = h.abs()
        if cos is not None:
            c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
            lo, hi = h[..., :D // 2], h[..., D // 2:]
            h = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
            big = torch.cat([big[..., :D // 2] + big[..., D // 2:]] * 2, -1)
        return h, big * (D / 2 + 8) * u

    x = x[:rows]
    q, qt = head(x[:, :heads], qn)
    k, kt = head(x[:, heads:heads + G], kn)
    return (q * q_scale, qt * abs(q_scale)), (k, kt), x[:, heads + G:], [b.token(s, int(p)) for s, p in zip(seq, pos)]


APPEND = [
    # (new, in all) of the sequences, heads, KV heads, head dim, page, order
    ([(1, 1)], 1, 1, 128, 16, "head"),
    ([(1, 17)], 16, 8, 128, 16, "head"),
    ([(3, 3), (0, 5), (1, 40), (7, 33)], 8, 2, 128, 16, "token"),
    ([(5, 70), (64, 64), (1, 128)], 5, 5, 64, 64, "head"),
    ([(1, n) for n in range(1, 71)], 4, 1, 64, 32, "token"),
    ([(130, 150), (1, 1), (33, 34)], 10, 2, 128, 128, "head"),
]


@pytest.mark.parametrize("form", ["norm+rope", "rope", "norm", "plain"])
@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(case, rt, ct, form):
    seqs, heads, G, D, page, order = APPEND[case]
    b = Batch(seqs, G, D, page, ct, order, seed=case, spare_rows=2, tokens=False)
    width = (heads + 2 * G) * D
    qkv = (b.randn(b.rows, width) * 3).to(rt)
    qn, kn = (1 + 0.2 * b.randn(D), 1 + 0.2 * b.randn(D)) if "norm" in form else (None, None)
    cos, sin = rope(160, D) if "rope" in form else (None, None)
    kv, dev = b.device(gphq)
    # Row strides of their own: the rows sit in wider buffers.
    wide = torch.full((b.rows, width + 16), NAN, dtype=rt, device="cuda")
    wide[:, :width] = qkv.cuda()
    q = torch.full((b.rows, heads * D + 8), 7.0, dtype=rt, device="cuda")
    up = lambda t: None if t is None else t.cuda()
    gphq.paged_append(kv, dev, wide[:, :width], q[:, :heads * D], heads, up(qn), up(kn), 1e-5, up(cos), up(sin), 0.25)
    dev.check()
    (q64, qt), (k64, kt), v64, places = append64(b, qkv, heads, qn, kn, 1e-5, cos, sin, 0.25)
    rows = len(places)
    got = q[:rows, :heads * D].cpu().double().view(rows, heads, D)
    err = (got - q64).abs()
    assert (err <= qt + half_step(rt) * q64.abs() * (1 + 2.0 ** -10) + 2.0 ** -25).all(), float((err - qt).max())
    assert (q[rows:] == 7).all() and (q[:, heads * D:] == 7).all()
    k, v = kv.k.cpu(), kv.v.cpu()
    for r, at in enumerate(places):
        e = (k[at].double() - k64[r]).abs()
        assert (e <= kt[r] + half_step(ct) * k64[r].abs() * (1 + 2.0 ** -10) + 2.0 ** -25).all()
        assert torch.equal(v[at], v64[r].to(rt).float().to(ct))
        k[at], v[at] = NAN, NAN
    assert k.isnan().all() and v.isnan().all()  # every other slot as it was


def test_append_in_place_of_the_queries():
    b = Batch([(5, 9), (1, 20)], 2, 128, 16, F16, seed=3, tokens=False)
    heads, D = 8, 128
    qkv = b.randn(b.rows, (heads + 4) * D).cuda()
    cos, sin = (t.cuda() for t in rope(64, D))
    qn, kn = (1 + 0.1 * b.randn(D)).cuda(), (1 + 0.1 * b.randn(D)).cuda()
    kv, dev = b.device(gphq)
    q = torch.empty(b.rows, heads * D, device="cuda")
    gphq.paged_append(kv, dev, qkv, q, heads, qn, kn, 1e-6, cos, sin, 0.5)
    kv2, dev2 = b.device(gphq)
    both = qkv.clone()
    gphq.paged_append(kv2, dev2, both, both, heads, qn, kn, 1e-6, cos, sin, 0.5)
    assert torch.equal(both[:, :heads * D], q) and torch.equal(both[:, heads * D:], qkv[:, heads * D:])
    assert torch.equal(kv.k.nan_to_num(9), kv2.k.nan_to_num(9)) and torch.equal(kv.v.nan_to_num(9), kv2.v.nan_to_num(9))


def test_append_reports_what_it_cannot_place():
    """A bad page stores nothing of its token, a bad sequence is skipped whole, a position past the table is skipped;
    the other rows are as without them."""
    heads, D, page = 2, 64, 16
    b = Batch([(2, 20), (3, 40), (2, 5), (1, 63), (2, 1), (2, 18)], 1, D, page, F32, seed=4, tokens=False)
    b.table[1, 2] = b.pages  # the page of tokens 37, 38 and 39, all that sequence 1 brings: one past the pool
    b.table[5, 1] = -7       # tokens 16, 17 of the last sequence
    qkv = b.randn(b.rows, (heads + 2) * D)
    cos, sin = rope(50, D)   # position 62 is past it
    kv, dev = b.device(gphq)
    q = torch.full((b.rows, heads * D), 7.0, device="cuda")
    gphq.paged_append(kv, dev, qkv.cuda(), q, heads, None, None, 0.0, cos.cuda(), sin.cuda())
    with pytest.raises(gphq.GphqError) as e:
        dev.check()
    assert e.value.status == gphq.ERR_PAGED_BATCH
    dev.check()  # cleared
    assert (q[[7, 8]] == 7).all()  # position 62, and token -1 of sequence 4, whose length is below its rows
    assert (q[[0, 1, 2, 3, 4, 5, 6, 9, 10, 11]] != 7).all()
    stored = {b.token(0, 18), b.token(0, 19), b.token(2, 3), b.token(2, 4), b.token(4, 0)}
    k = kv.k.cpu()
    have = {(p, s) for p in range(b.pages) for s in range(page) if not k[p, s].isnan().any()}
    assert have == stored


@pytest.mark.parametrize("starts,good", [([0, 4, 2, 6], []), ([0, 2, 4, 9], [0, 1, 2, 3]), ([-1, 2, 4, 6], [2, 3, 4, 5]),
                                         ([0, 5, 5, 6], [5]), ([2 ** 31 - 1, -2 ** 31, 4, 6], [4, 5])])
def test_bad_sequences_are_left_alone(starts, good):
    """Starts that descend, leave the rows or give a sequence more than max_rows rows: flagged, its rows untouched."""
    heads, D = 2, 64
    b = Batch([(2, 20), (2, 30), (2, 40)], 1, D, 16, F32, seed=5)
    kv, dev = b.device(gphq)
    dev.starts.copy_(torch.tensor(starts, dtype=torch.int32))
    rest = [r for r in range(b.rows) if r not in good]
    for call in (lambda o: gphq.paged_attention(kv, dev, b.randn(b.rows, heads * D).cuda(), o, heads, 0.1),
                 lambda o: gphq.paged_append(kv, dev, b.randn(b.rows, (heads + 2) * D).cuda(), o, heads)):
        out = torch.full((b.rows, heads * D), 7.0, device="cuda")
        call(out)
        with pytest.raises(gphq.GphqError):
            dev.check()
        assert (out[rest] == 7).all() and (out[good] != 7).all() and out.isfinite().all()


def test_bad_lengths_are_left_alone():
    b = Batch([(1, 20), (1, 30), (1, 40)], 1, 64, 16, F32, seed=6)
    for lens in ([20, -1, 40], [20, 41, 40], [20, 2 ** 31 - 1, 40]):
        kv, dev = b.device(gphq)
        dev.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        out = torch.full((3, 128), 7.0, device="cuda")
        gphq.paged_attention(kv, dev, b.randn(3, 128).cuda(), out, 2, 0.1)
        with pytest.raises(gphq.GphqError):
            dev.check()
        assert (out[1] == 7).all() and (out[[0, 2]] != 7).all()


# ---- attention ------------------------------------------------------------------


def attend(b, q, heads, scale, window=0, **over):
    kv, dev = b.device(gphq, **over)
    out = torch.full((b.rows, heads * b.hd), 7.0, dtype=q.dtype, device="cuda")
    gphq.paged_attention(kv, dev, q.cuda(), out, heads, scale, window)
    dev.check()
    return out


def check_attention(b, heads, rt, window=0, scale=None, **over):
    scale = b.hd ** -0.5 if scale is None else scale
    q = (b.randn(b.rows, heads * b.hd) * 1.5).to(rt)
    out = attend(b, q, heads, scale, window, **over)
    want, tol = attention64(b, q, heads, scale, window)
    n = b.starts[-1]
    err = (out[:n].cpu().double() - want[:n]).abs()
    worst = float((err / tol[:n].clamp(min=1e-30)).max()) if n else 0.0
    assert (err <= tol[:n]).all(), f"worst {worst} of the bound"
    assert (out[n:] == 7).all()  # rows behind the last sequence


SINGLE = [1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 300, 1000]
ATTEND = [
    # sequences, heads, KV heads, head dim, page, order
    ([(1, n) for n in SINGLE], 4, 1, 128, 16, "head"),
    ([(1, n) for n in SINGLE], 16, 8, 64, 64, "token"),
    ([(1, 200), (0, 30), (1, 0), (2, 1), (3, 3), (0, 0)], 6, 2, 128, 32, "head"),       # empty, and rows that see nothing
    ([(5, 40), (4, 4), (6, 70), (1, 9)], 8, 2, 128, 16, "token"),                        # a few rows each
    ([(1, 77), (1, 600)], 40, 1, 64, 16, "head"),                                        # 40 heads on one KV head
    ([(40, 40)], 4, 2, 128, 16, "head"),
    ([(33, 50), (130, 300), (1, 500), (65, 64), (7, 260)], 8, 2, 128, 32, "token"),      # mixed
    ([(129, 129), (31, 1000)], 5, 1, 64, 128, "head"),
    ([(257, 300)], 3, 3, 128, 16, "head"),                                               # every head its own KV head
    ([(17, 2100)], 8, 1, 128, 64, "head"),                                               # few rows, long: split
]


@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention(case, rt, ct):
    seqs, heads, G, D, page, order = ATTEND[case]
    check_attention(Batch(seqs, G, D, page, ct, order, seed=case, spare_rows=3), heads, rt)


@pytest.mark.parametrize("window", [1, 2, 16, 33, 100, 5000])
@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
def test_attention_window(rt, ct, window):
    b = Batch([(1, 700), (1, 20), (5, 90), (70, 400), (40, 40)], 2, 128, 16, ct, seed=window)
    # Pages wholly behind every row's window may have been given back.
    for s, (n, t) in enumerate(zip(b.new, b.lens)):
        gone = max(0, t - n - window + 1) // 16
        b.table[s, :gone] = -1
    q = (b.randn(b.rows, 8 * 128) * 1.5).to(rt)
    out = attend(b, q, 8, 0.1, window)
    full = Batch([(1, 700), (1, 20), (5, 90), (70, 400), (40, 40)], 2, 128, 16, ct, seed=window)
    want, tol = attention64(full, q, 8, 0.1, window)
    assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf, "lowest"])
@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("seqs", [[(8, 40)], [(70, 150)]], ids=["rows", "chunk"])
def test_what_a_row_does_not_see_does_not_reach_it(seqs, rt, ct, bad):
    """Keys and values of later tokens of the same call, and of tokens that only the first rows' windows reach, hold
    NaN, infinities or the type's lowest value: rows that do not see them keep to the definition."""
    heads, D, (n, t) = 8, 128, seqs[0]
    b = Batch(seqs, 2, D, 16, ct, seed=7)
    q = (b.randn(b.rows, heads * D) * 1.5).to(rt)
    window = t - n - n // 4 + 1
    want, tol = attention64(b, q, heads, 0.1, window)
    late, early = t - n // 2, n // 4 + 2  # tokens from `late` on, and before `early`; the first row sees from n / 4
    value = torch.finfo(ct).min if bad == "lowest" else bad
    for p in list(range(late, t)) + list(range(early)):
        b.k[b.token(0, p)] = value
        b.v[b.token(0, p)] = value
    got = attend(b, q, heads, 0.1, window).cpu().double()
    free = [i for i in range(n) if early <= t - n + i - window + 1 and t - n + i < late]
    assert len(free) >= 2
    assert ((got[free] - want[free]).abs() <= tol[free]).all()
    if bad != "lowest":  # and rows that see them are not finite
        assert not got[[i for i in range(n) if i not in free]].isfinite().all(-1).any()


@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
def test_extreme_scores(rt, ct):
    """Scores that grow along the keys by far more than the rescale's lag, and rows of zeros."""
    b = Batch([(1, 300), (70, 200)], 2, 64, 16, ct, seed=9)
    for s, t in enumerate(b.lens):
        for p in range(t):
            b.k[b.token(s, p)] = (b.k[b.token(s, p)].double() * (0.05 + 3.0 * p / t)).to(ct)
    check_attention(b, 4, rt, scale=1.0)
    q = torch.zeros(b.rows, 4 * 64, dtype=rt)
    out = attend(b, q, 4, 1.0)
    want, tol = attention64(b, q, 4, 1.0)
    assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("mag", [2.0 ** -60, 2.0 ** 40])
@pytest.mark.parametrize("ct", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
def test_fp32_rows_out_of_a_16_bit_type_s_range(ct, mag):
    b = Batch([(1, 100), (40, 90)], 1, 128, 16, ct, seed=11)
    q = b.randn(b.rows, 2 * 128) * mag
    scale = 0.1 / mag
    out = attend(b, q, 2, scale)
    want, tol = attention64(b, q, 2, scale)
    assert ((out.cpu().double() - want).abs() <= tol).all()


def test_bad_pages_read_as_masked_keys():
    b = Batch([(1, 100), (50, 100)], 2, 64, 16, F16, seed=12)
    q = b.randn(b.rows, 4 * 64)
    for s in range(2):
        b.table[s, 2] = b.pages + 5
    kv, dev = b.device(gphq)
    out = torch.empty(b.rows, 4 * 64, device="cuda")
    gphq.paged_attention(kv, dev, q.cuda(), out, 4, 0.1)
    with pytest.raises(gphq.GphqError):
        dev.check()
    # The definition without tokens 32 .. 47.
    rows = q.double().view(b.rows, 4, 64)
    for s in range(2):
        for i in range(b.new[s]):
            p, r = b.lens[s] - b.new[s] + i, b.starts[s] + i
            keep = [j for j in range(p + 1) if not 32 <= j < 48]
            at = [b.token(s, j) for j in keep]
            for h in range(4):
                k = torch.stack([b.k[a][h // 2] for a in at]).double()
                v = torch.stack([b.v[a][h // 2] for a in at]).double()
                want = torch.softmax(k @ rows[r, h] * 0.1, 0) @ v
                # fp32 throughout: far inside 2^-14 for 100 keys of unit size.
                assert torch.allclose(out[r].view(4, 64)[h].cpu().double(), want, rtol=2.0 ** -14, atol=2.0 ** -14)


def test_a_call_of_loose_bounds_gives_the_same_rows():
    """max_rows, max_len and the row buffers may be larger than what the sequences bring."""
    b = Batch([(1, 300), (40, 200), (3, 3)], 2, 128, 16, BF16, seed=13, spare_rows=20)
    q = b.randn(b.rows, 8 * 128)
    want, tol = attention64(b, q, 8, 0.09)
    n = b.starts[-1]
    for max_rows, max_len in ((40, 300), (64, 320), (10 ** 6, 320)):
        out = attend(b, q, 8, 0.09, max_rows=max_rows, max_len=max_len)
        assert ((out[:n].cpu().double() - want[:n]).abs() <= tol[:n]).all()
        assert (out[n:] == 7).all()


@pytest.mark.parametrize("new", [1, 3, 9, 60])
def test_one_sequence_of_fewer_rows_than_its_bound(new):
    b = Batch([(new, 333)], 2, 128, 16, F16, seed=20, spare_rows=4)
    q = b.randn(b.rows, 8 * 128)
    out = attend(b, q, 8, 0.1, max_rows=64, max_len=16 * b.entries)
    want, tol = attention64(b, q, 8, 0.1)
    assert ((out[:new].cpu().double() - want[:new]).abs() <= tol[:new]).all()
    assert (out[new:] == 7).all()


@pytest.mark.parametrize("scale", [-0.15, 0.0, 1e-32, -1e-32])
@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
def test_scales_of_every_kind(rt, ct, scale):
    check_attention(Batch([(1, 200), (40, 70), (1, 0)], 2, 64, 16, ct, seed=21), 4, rt, scale=scale)


@pytest.mark.parametrize("heads,kv_heads,rows", [(2, 2, (63, 64, 65)), (8, 2, (15, 16, 17)), (14, 2, (9, 10, 1)),
                                                 (64, 1, (1, 2, 1)), (65, 1, (1, 1, 2))])
@pytest.mark.parametrize("rt,ct", [(F32, F32), (F32, F16), (torch.bfloat16, torch.bfloat16)])
def test_columns_on_both_sides_of_the_two_kernels(heads, kv_heads, rows, rt, ct):
    """Rows times group about 64: each sequence in one kernel or the other, alone and with the rest."""
    shape = [(n, n + 150 + 700 * i) for i, n in enumerate(rows)]
    check_attention(Batch(shape, kv_heads, 64, 16, ct, seed=25), heads, rt)
    for one in shape:
        check_attention(Batch([one], kv_heads, 64, 16, ct, seed=26), heads, rt)


def test_a_slice_of_a_batch():
    """Sequences 1 and 2 of three, by views of the tables: rows of the others stay as they are, and none is bad."""
    b = Batch([(3, 40), (1, 700), (50, 90), (2, 30)], 2, 64, 16, F16, seed=24)
    q = b.randn(b.rows, 4 * 64)
    kv, dev = b.device(gphq)
    part = gphq.PagedBatch(dev.starts[1:4], dev.lens[1:3], dev.table[1:3], b.rows, 50, 700)
    out = torch.full((b.rows, 4 * 64), 7.0, device="cuda")
    gphq.paged_attention(kv, part, q.cuda(), out, 4, 0.1)
    part.check()
    want, tol = attention64(b, q, 4, 0.1)
    assert ((out[3:54].cpu().double() - want[3:54]).abs() <= tol[3:54]).all()
    assert (out[:3] == 7).all() and (out[54:] == 7).all()
    out.fill_(7.0)
    gphq.paged_append(kv, part, b.randn(b.rows, 8 * 64).cuda(), out, 4)
    part.check()
    assert (out[:3] == 7).all() and (out[54:] == 7).all() and (out[3:54] != 7).all()


def test_without_a_word_for_bad_values():
    b = Batch([(1, 40), (2, 50)], 1, 64, 16, F32, seed=22)
    kv, dev = b.device(gphq)
    dev.desc.bad_dev = None
    dev.lens.copy_(torch.tensor([40, 51], dtype=torch.int32))
    out = torch.full((3, 128), 7.0, device="cuda")
    q = b.randn(3, 128)
    gphq.paged_attention(kv, dev, q.cuda(), out, 2, 0.1)
    torch.cuda.synchronize()
    want, tol = attention64(b, q, 2, 0.1)
    assert ((out[0].cpu().double() - want[0]).abs() <= tol[0]).all() and (out[1:] == 7).all()


def test_scratch_of_a_call_on_another_stream():
    """Calls without a workspace on a side stream, with work on the current stream taking and giving back memory."""
    b = Batch([(1, 3000), (1, 2500)], 1, 128, 16, BF16, seed=23)
    q = b.randn(2, 4 * 128)
    kv, dev = b.device(gphq)
    dq, side = q.cuda(), torch.cuda.Stream()
    want, tol = attention64(b, q, 4, 0.1)
    torch.cuda.synchronize()
    outs = [torch.empty(2, 512, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    for o in outs:
        gphq.paged_attention(kv, dev, dq, o, 4, 0.1, stream=side)
        torch.full((1 << 16,), float("nan"), device="cuda")
    torch.cuda.synchronize()
    for o in outs:
        assert ((o.cpu().double() - want).abs() <= tol).all()


def test_strided_rows_another_stream_and_repeats():
    b = Batch([(1, 900), (1, 40), (20, 500)], 2, 128, 32, F16, seed=14)
    heads, D = 8, 128
    q = b.randn(b.rows, heads * D + 32)
    kv, dev = b.device(gphq)
    wide = q.cuda()
    outs = [torch.full((b.rows, heads * D + 4), 7.0, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    work = torch.empty(gphq.paged_attention_workspace_bytes(kv, dev, F32, heads), dtype=torch.uint8, device="cuda")
    for o in outs:
        gphq.paged_attention(kv, dev, wide[:, 16:16 + heads * D], o[:, :heads * D], heads, 0.1, work=work, stream=side)
    side.synchronize()
    want, tol = attention64(b, q[:, 16:16 + heads * D].contiguous(), heads, 0.1)
    assert ((outs[0][:, :heads * D].cpu().double() - want).abs() <= tol).all()
    assert (outs[0][:, heads * D:] == 7).all()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])  # the same bits every time


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements whose tokens lie in its last pages."""
    page, G, D = 4096, 8, 128
    pages = 2 ** 32 // (page * G * D) + 3
    pool = [torch.empty(pages, page, G, D, dtype=BF16, device="cuda") for _ in range(2)]
    b = Batch([(1, 50), (40, 60)], G, D, page, BF16, "token", seed=15)
    kv = gphq.PagedKv(*pool)
    last = {int(b.table[s, 0]): pages - 1 - s for s in range(2)}
    for mine, theirs in zip((b.k, b.v), pool):
        for a, z in last.items():
            theirs[z] = mine[a].cuda()
    _, dev = b.device(gphq)
    dev.table.copy_(torch.tensor([[last.get(int(x), -1) for x in row] for row in b.table], dtype=torch.int32))
    q = b.randn(b.rows, 16 * D)
    out = torch.empty(b.rows, 16 * D, device="cuda")
    gphq.paged_attention(kv, dev, q.cuda(), out, 16, 0.1)
    dev.check()
    want, tol = attention64(b, q, 16, 0.1)
    assert ((out.cpu().double() - want).abs() <= tol).all()
    qkv = b.randn(b.rows, 18 * D + 14 * D).to(BF16)
    gphq.paged_append(kv, dev, qkv.cuda(), torch.empty(b.rows, 16 * D, dtype=BF16, device="cuda"), 16)
    dev.check()
    assert torch.equal(pool[1][pages - 1, 49].cpu(), qkv[0, 24 * D:].view(G, D))
    assert torch.equal(pool[0][pages - 2, 20].cpu(), qkv[1, 16 * D:24 * D].view(G, D))


def test_captured_steps_follow_the_lengths():
    """Append and attention captured once, replayed as the sequences grow, with eager work between the replays."""
    heads, G, D, page, steps = 8, 2, 128, 16, 5
    b = Batch([(1, 30 + steps), (1, 14 + steps), (1, 200 + steps)], G, D, page, F16, seed=16)
    grow = [t - steps + 1 for t in b.lens]
    qkvs = [b.randn(3, (heads + 2 * G) * D).cuda() for _ in range(steps)]
    cos, sin = (t.cuda() for t in rope(256, D))
    kv, dev = b.device(gphq)
    kv2, dev2 = b.device(gphq)
    qkv, q, out = qkvs[0].clone(), torch.empty(3, heads * D, device="cuda"), torch.empty(3, heads * D, device="cuda")
    q2, out2 = torch.empty_like(q), torch.empty_like(out)
    work = torch.empty(gphq.paged_attention_workspace_bytes(kv, dev, F32, heads), dtype=torch.uint8, device="cuda")

    def step(kv, dev, rows, q, out):
        gphq.paged_append(kv, dev, rows, q, heads, None, None, 0.0, cos, sin, D ** -0.5)
        gphq.paged_attention(kv, dev, q, out, heads, 1.0, work=work)

    dev.lens.copy_(torch.tensor(grow, dtype=torch.int32))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(kv, dev, qkv, q, out)
    for i in range(steps):
        now = torch.tensor([t + i for t in grow], dtype=torch.int32)
        dev.lens.copy_(now)
        dev2.lens.copy_(now)
        qkv.copy_(qkvs[i])
        graph.replay()
        torch.cuda.synchronize()
        step(kv2, dev2, qkvs[i], q2, out2)
        torch.cuda.synchronize()
        assert torch.equal(q, q2) and torch.equal(out, out2)
    dev.check()
    assert torch.equal(kv.k.nan_to_num(9), kv2.k.nan_to_num(9)) and torch.equal(kv.v.nan_to_num(9), kv2.v.nan_to_num(9))


def test_shared_pages():
    """Two sequences over the same prompt pages see the same keys."""
    b = Batch([(1, 70), (1, 70)], 2, 64, 16, F32, seed=17)
    b.table[1, :4] = b.table[0, :4]
    check_attention(b, 4, F32)


def test_wrong_tensors_are_refused():
    b = Batch([(1, 20)], 2, 64, 16, F32, seed=18)
    kv, dev = b.device(gphq)
    q, out = torch.zeros(1, 256, device="cuda"), torch.zeros(1, 256, device="cuda")
    for call in (
        lambda: gphq.paged_attention(kv, dev, q.cpu(), out, 4, 1.0),
        lambda: gphq.paged_attention(kv, dev, q[:, :200], out, 4, 1.0),
        lambda: gphq.paged_attention(kv, dev, q, out.half(), 4, 1.0),
        lambda: gphq.paged_attention(kv, dev, q.t(), out, 4, 1.0),
        lambda: gphq.paged_append(kv, dev, q, out, 4),
        lambda: gphq.PagedKv(kv.k, kv.v.half()),
        lambda: gphq.PagedKv(kv.k, kv.v[:, :, :1]),
        lambda: gphq.PagedBatch(dev.starts.long(), dev.lens, dev.table, 1, 1, 20),
        lambda: gphq.PagedBatch(dev.starts[:1], dev.lens, dev.table, 1, 1, 20),
        lambda: gphq.PagedBatch(dev.starts, dev.lens, dev.table[0], 1, 1, 20),
    ):
        with pytest.raises(gphq.GphqError):
            call()
    assert np.isfinite(out.cpu().numpy()).all()
