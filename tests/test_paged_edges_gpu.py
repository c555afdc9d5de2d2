"""Paged attention where a batch is unusual: rows whose pages are bad, values at the ends of a type's range, batches of
mostly idle sequences, walks over many pages. Against the definition in float64, on sampled rows."""
import math

import pytest
import torch

from gophonic_amd import gphq
from tests.paged_common import BF16, F16, F32, NAN, Batch, half_step

pytestmark = pytest.mark.gpu

TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]
TYPE_IDS = ["f32-f32", "f32-f16", "f32-bf16", "f16-f16", "bf16-bf16"]


def run(b, q, heads, scale, window=0, bad=False, **over):
    kv, dev = b.device(gphq, **over)
    out = torch.full((b.rows, heads * b.hd), 7.0, dtype=q.dtype, device="cuda")
    gphq.paged_attention(kv, dev, q.cuda(), out, heads, scale, window)
    if bad:
        with pytest.raises(gphq.GphqError) as e:
            dev.check()
        assert e.value.status == gphq.ERR_PAGED_BATCH
    dev.check()
    return out.cpu()


def row64(b, q, heads, scale, r, window=0, pieces=1):
    """The definition of one row in float64 and a bound of fp32 arithmetic's error, as paged_common.attention64 derives
    it, over the keys that lie in pages of the pool. Probabilities of 16-bit rows in `pieces` pieces of the type, each
    off by at most half a step of what is left of them."""
    s = max(i for i in range(len(b.new)) if b.starts[i] <= r)
    p = b.lens[s] - b.new[s] + r - b.starts[s]
    keys = torch.arange(max(0, p - window + 1) if window else 0, p + 1)
    page = torch.from_numpy(b.table[s]).long()[keys // b.page]
    good = (page >= 0) & (page < b.pages)
    keys, page = keys[good], page[good]
    m, group, u, half = len(keys), heads // b.kv_heads, 2.0 ** -24, half_step(q.dtype)
    if m == 0:
        zero = torch.zeros(heads * b.hd, dtype=torch.float64)
        return zero, zero
    k = b.k[page, keys % b.page].double().transpose(0, 1)  # [KV heads][keys][hd]
    v = b.v[page, keys % b.page].double().transpose(0, 1)
    x = q[r].double().view(b.kv_heads, group, b.hd)
    w = torch.softmax(x @ k.transpose(1, 2) * scale, -1)
    out, a = w @ v, w @ v.abs()
    e = abs(scale) * ((b.hd + 4) * u * (x.abs() @ k.abs().transpose(1, 2)).amax(-1)
                      + 2.0 ** -22 * x.abs().amax(-1) * k.abs().sum(-1).amax(-1)[:, None])
    tol = (torch.expm1(2 * e)[..., None] + (2 * m + 64) * u) * a + m * 2.0 ** -32 * v.abs().amax((1, 2))[:, None, None]
    if half > u:
        tol = tol + half ** pieces * a
    return out.reshape(-1), (tol + half * out.abs() + 2.0 ** -25).reshape(-1)


def check_rows(b, q, heads, scale, got, rows, window=0, pieces=1):
    for r in rows:
        want, tol = row64(b, q, heads, scale, r, window, pieces)
        err = (got[r].double() - want).abs()
        assert (err <= tol).all(), f"row {r}: {float((err / tol.clamp(min=1e-30)).max())} of the bound"


# ---- rows that see no key because their pages are bad ------------------------------


@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("seqs,bad,window", [
    ([(1, 9)], [(0, 0)], 0),                                    # the only page
    ([(1, 9), (1, 2000)], [(0, 0)], 0),                         # beside one that is split
    ([(1, 2000)], [(0, e) for e in range(125)], 0),             # every split's pages
    ([(1, 2000), (3, 700)], [(0, 124), (1, 43), (1, 42)], 16),  # a window inside bad pages, or partly
    ([(70, 70)], [(0, 0)], 0),                                  # a chunk whose first rows have no other page
    ([(70, 70), (80, 3000)], [(0, 0), (0, 1)], 0),              # the same, beside one that is split
    ([(90, 600)], [(0, e) for e in range(32, 38)], 20),         # a chunk's windows
    ([(80, 3000)], [(0, e) for e in range(188)], 0),            # a split chunk without a page
], ids=range(8))
def test_rows_without_a_good_page_are_zero(seqs, bad, window, rt, ct):
    heads = 4
    b = Batch(seqs, 2, 64, 16, ct, seed=40)
    for i, (s, e) in enumerate(bad):
        b.table[s, e] = (b.pages, -1, 2 ** 31 - 1)[i % 3]
    q = b.randn(b.rows, heads * 64).to(rt)
    got = run(b, q, heads, 0.1, window, bad=True)
    check_rows(b, q, heads, 0.1, got, range(b.rows), window)
    empty = [r for r in range(b.rows) if not row64(b, q, heads, 0.1, r, window)[0].any()]
    assert empty and (got[empty] == 0).all()


@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("seqs", [[(1, 9)], [(1, 2000)], [(70, 70)], [(80, 3000)]], ids=str)
def test_rows_whose_scores_are_all_minus_infinity_are_not_finite(seqs, rt, ct):
    """They do see keys, so they are not the rows above: the quotient is 0 / 0."""
    b = Batch(seqs, 2, 64, 16, ct, seed=41)
    b.k.fill_(-math.inf)
    q = (b.randn(b.rows, 4 * 64).abs() + 0.1).to(rt)
    got = run(b, q, 4, 0.1)
    assert not got.isfinite().any()


# ---- batches of mostly idle sequences ----------------------------------------------


def idle(seqs, live):
    """`seqs` sequences of which those in `live`, {number: (new, tokens)}, bring rows; the others hold tokens or none."""
    return [live.get(s, (0, 5 * (s % 3))) for s in range(seqs)]


@pytest.mark.parametrize("rt,ct", [(F32, F32), (F32, F16), (BF16, BF16)], ids=["f32-f32", "f32-f16", "bf16-bf16"])
@pytest.mark.parametrize("seqs,live,spare", [
    (300, {17: (1, 3000)}, 0), (300, {0: (1, 2500), 64: (3, 2900), 299: (2, 700)}, 0),
    (300, {0: (1, 2500), 64: (3, 2900), 299: (2, 700)}, 5), (150, {3: (1, 2600), 70: (40, 2100), 128: (5, 2200)}, 0),
], ids=range(4))
def test_few_rows_in_a_batch_of_many_sequences(seqs, live, spare, rt, ct):
    b = Batch(idle(seqs, live), 2, 64, 16, ct, seed=50, spare_rows=spare)
    q = (b.randn(b.rows, 8 * 64) * 1.5).to(rt)
    got = run(b, q, 8, 0.125)
    check_rows(b, q, 8, 0.125, got, range(b.starts[-1]))
    assert (got[b.starts[-1]:] == 7).all()


@pytest.mark.parametrize("heads,kv_heads", [(40, 1), (16, 1), (17, 1), (2, 2), (64, 1), (65, 1)])
@pytest.mark.parametrize("rt,ct", [(F32, F16), (F32, F32)], ids=["f32-f16", "f32-f32"])
def test_few_rows_of_every_group_size_among_idle_sequences(heads, kv_heads, rt, ct):
    """Rows of one to five tiles each, of sequences of one to three rows."""
    b = filled(idle(400, {3: (3, 700), 200: (1, 90), 399: (2, 1300)}), kv_heads, 64, 16, ct, seed=52)
    q = (b.randn(b.rows, heads * 64) * 1.5).to(rt)
    got = run(b, q, heads, 0.125)
    check_rows(b, q, heads, 0.125, got, range(b.rows))


@pytest.mark.parametrize("what", ["idle length", "live length", "descending starts", "rows past the end"])
def test_bad_sequences_among_idle_ones_are_reported(what):
    """As in a batch without idle sequences: the bad one is skipped and reported, rows of good ones are as they were."""
    b = filled(idle(400, {3: (1, 700), 200: (1, 90), 399: (1, 1300)}), 2, 64, 16, F16, seed=53)
    q = b.randn(b.rows, 8 * 64)
    kv, dev = b.device(gphq)
    if what == "idle length":
        dev.lens[77] = 5000
        good = [0, 1, 2]
    elif what == "live length":
        dev.lens[200] = -1
        good = [0, 2]
    elif what == "descending starts":
        dev.starts[201] = 0  # sequence 200 ends before it starts, sequence 201 has two rows where one may be
        good = [0, 2]
    else:
        dev.starts[400] = 9
        good = [0, 1]
    out = torch.full((b.rows, 8 * 64), 7.0, device="cuda")
    gphq.paged_attention(kv, dev, q.cuda(), out, 8, 0.125)
    with pytest.raises(gphq.GphqError) as e:
        dev.check()
    assert e.value.status == gphq.ERR_PAGED_BATCH
    dev.check()
    out = out.cpu()
    check_rows(b, q, 8, 0.125, out, good)
    assert (out[[r for r in range(3) if r not in good]] == 7).all()


def test_a_batch_of_all_the_sequences_that_fit():
    """65536 sequences over one KV head, three of them with a row: the most that a batch may hold."""
    n, page, heads = 65536, 16, 4
    lens = {5: 40, 40000: 3000, 65535: 700}
    need = 188
    b = Batch([(1, t) for t in lens.values()], 1, 64, page, F16, seed=51)
    starts = torch.zeros(n + 1, dtype=torch.int32)
    for s in lens:
        starts[s + 1:] += 1
    table = torch.full((n, need), -1, dtype=torch.int32)
    length = torch.zeros(n, dtype=torch.int32)
    for i, (s, t) in enumerate(lens.items()):
        length[s] = t
        table[s, :b.entries] = torch.from_numpy(b.table[i])[:need]
    kv, _ = b.device(gphq)
    dev = gphq.PagedBatch(starts.cuda(), length.cuda(), table.cuda(), 3, 1, 3000)
    q = b.randn(3, heads * 64)
    out = torch.full((3, heads * 64), 7.0, device="cuda")
    gphq.paged_attention(kv, dev, q.cuda(), out, heads, 0.125)
    dev.check()
    check_rows(b, q, heads, 0.125, out.cpu(), range(3))


# ---- what a call found out of bounds ------------------------------------------------


def test_check_keeps_to_its_stream():
    """The check reads and clears the batch's word on the stream that it is given: it does not wait for the default
    stream's work, and what the next call on its own stream finds is not lost."""
    b = Batch([(1, 40)], 1, 64, 16, F16, seed=60)
    b.table[0, 1] = -5
    kv, dev = b.device(gphq)
    q, out = b.randn(1, 128).half().cuda(), torch.empty(1, 128, dtype=F16, device="cuda")
    work = torch.empty(16, dtype=torch.uint8, device="cuda")
    x, side, done = torch.randn(8192, 8192, device="cuda"), torch.cuda.Stream(), torch.cuda.Event()
    y = x @ x
    torch.cuda.synchronize()
    for _ in range(60):  # some hundreds of milliseconds
        torch.matmul(x, x, out=y)
    done.record()
    for _ in range(3):
        gphq.paged_attention(kv, dev, q, out, 2, 0.1, work=work, stream=side)
        with pytest.raises(gphq.GphqError):
            dev.check(side)
    dev.check(side)
    assert not done.query()
    torch.cuda.synchronize()


def test_the_current_stream_s_handle():
    side = torch.cuda.Stream()
    for s in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(s):
            assert gphq.stream_handle() == s.cuda_stream == gphq.stream_handle(s)


# ---- values at the end of their type's range -----------------------------------------


@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("ahead", [0.0, 7.5], ids=["level", "ahead"])
@pytest.mark.parametrize("seqs", [[(1, 1)], [(1, 300), (3, 40)], [(1, 3000)], [(70, 200)], [(80, 3000)]], ids=str)
def test_values_at_the_end_of_the_range(seqs, ahead, rt, ct):
    """One finite value of nearly the type's largest magnitude among small ones: a weighted mean of them is finite, also
    where its key's score is `ahead` (in log2) of all before it."""
    b = Batch(seqs, 2, 64, 16, ct, seed=70)
    big = 0.99 * torch.finfo(ct).max
    for s, (n, t) in enumerate(seqs):
        for p in range(t):
            b.k[b.token(s, p)] = 0.0
        at = b.token(s, t - n)  # the first new token, which every row sees
        b.k[at] = ahead * math.log(2) / 64
        b.v[at] = big
        b.v[at][:, ::2] = -big
    q = torch.ones(b.rows, 4 * 64, dtype=rt)
    got = run(b, q, 4, 1.0)
    assert got.isfinite().all()
    check_rows(b, q, 4, 1.0, got, range(b.rows))


# ---- 16-bit rows of single tokens -----------------------------------------------------


@pytest.mark.parametrize("ct", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_single_16_bit_rows_are_rounded_once(ct, hd):
    """Sequences of up to 64 columns: only the result is rounded to 16 bits, not the probabilities."""
    b = Batch([(1, 40), (1, 100), (1, 700), (1, 3000), (5, 300), (16, 90)], 2, hd, 16, ct, seed=80)
    q = (b.randn(b.rows, 8 * hd) * 1.5).to(ct)
    got = run(b, q, 8, hd ** -0.5)
    check_rows(b, q, 8, hd ** -0.5, got, range(b.rows), pieces=2)


# ---- long walks ------------------------------------------------------------------------


def filled(seqs, kv_heads, hd, page, dtype, seed, **over):
    """A Batch whose tokens are drawn all at once, unused slots NaN."""
    b = Batch(seqs, kv_heads, hd, page, dtype, seed=seed, tokens=False, **over)
    used = torch.zeros(b.pages, page, dtype=torch.bool)
    for s, t in enumerate(b.lens):
        p = torch.arange(t)
        used[torch.from_numpy(b.table[s]).long()[p // page], p % page] = True
    n = int(used.sum())
    b.k[used] = b.randn(n, kv_heads, hd).to(dtype)
    b.v[used] = (b.randn(n, kv_heads, hd) + 0.25).to(dtype)
    return b


def splits(b, rt, heads, rows, window=0):
    """How many splits of `rows` rows the call's workspace holds."""
    kv, dev = b.device(gphq)
    n = gphq.paged_attention_workspace_bytes(kv, dev, rt, heads, window)
    assert n % (rows * heads * (b.hd + 2) * 4) == 0
    return n // (rows * heads * (b.hd + 2) * 4)


def spread(rows, count=24):
    return sorted({round(i * (rows - 1) / (count - 1)) for i in range(count)})


def in_blocks(rt, blocks):
    """Rows of group 8 and eight KV heads that make as many blocks of the chunk kernel as `blocks` times what runs at
    once: 128 columns and two blocks a CU, 256 and one for fp32 rows."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    return int(blocks * (2 * cus * 128 if rt != F32 else cus * 256) / 64)


@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 16), (128, 256)])
def test_chunks_that_are_not_split(hd, page, rt, ct):
    """A block walks all of a chunk's keys: some forty steps, more table entries than a wavefront holds at once."""
    rows = in_blocks(rt, 1)
    b = filled([(rows, rows + 1537)], 8, hd, page, ct, seed=90)
    q = b.randn(rows, 64 * hd).to(rt)
    assert splits(b, rt, 64, rows) == 0
    got = run(b, q, 64, 0.1)
    check_rows(b, q, 64, 0.1, got, spread(rows))


@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("hd", [64, 128])
def test_chunks_of_two_long_splits(hd, rt, ct):
    rows = in_blocks(rt, 0.5)
    b = filled([(rows, 6033)], 8, hd, 16, ct, seed=91)
    q = b.randn(rows, 64 * hd).to(rt)
    assert splits(b, rt, 64, rows) == 2
    got = run(b, q, 64, 0.1)
    check_rows(b, q, 64, 0.1, got, spread(rows))


@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("hd", [64, 128])
def test_single_tokens_of_long_splits(hd, rt, ct):
    """Sixteen single tokens over ragged caches of small pages, two splits of some 2000 keys each."""
    b = filled([(1, 4000 - 177 * i) for i in range(16)], 8, hd, 16, ct, seed=92)
    q = (b.randn(16, 32 * hd) * 1.5).to(rt)
    assert splits(b, rt, 32, 16) == 2
    got = run(b, q, 32, hd ** -0.5)
    check_rows(b, q, 32, hd ** -0.5, got, range(16))


@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
def test_many_sequences_of_every_kind(rt, ct):
    """170 sequences, chunks, a few rows, single tokens and none, both kernels split: more than the 64 that a wavefront
    looks at together."""
    kinds = [(0, 0), (1, 1400), (1, 33), (0, 50), (5, 900), (1, 17), (70, 1300), (1, 1), (3, 2), (40, 40)]
    seqs = [(n, t + 3 * i if t > 2 else t) for i in range(17) for n, t in kinds]
    b = filled(seqs, 1, 64, 16, ct, seed=93, spare_rows=3)
    q = (b.randn(b.rows, 4 * 64) * 1.5).to(rt)
    small = 170 * (64 // 4)  # places of the row kernel's split results: up to 16 rows a sequence
    kv, dev = b.device(gphq)
    n = gphq.paged_attention_workspace_bytes(kv, dev, rt, 4)
    places, rest = n // (4 * (64 + 2) * 4), min(small, b.rows)
    assert any((places - i * b.rows) > 0 and (places - i * b.rows) % rest == 0 for i in range(2, 40))
    got = run(b, q, 4, 0.125)
    last = b.starts[-1]
    check_rows(b, q, 4, 0.125, got, sorted(set(spread(last, 150)) | {r for r in b.starts[:-1] if r < last}))
    assert (got[last:] == 7).all()


@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("window", [0, 300])
def test_infinite_values_on_many_steps(window, rt, ct):
    """Infinities in some dims of many values of a chunk, on every step of the tiles' edges, LDS buffers used many times
    over: exactly the rows that see one are not finite in that dim (NaN where a probability has several pieces, of
    which one may be 0 or negative), every other value keeps to the definition."""
    heads, hd = 8, 64  # group 1: a tile is 128 or 256 rows, its edges several steps
    rows = in_blocks(rt, 1) * 8
    b = filled([(rows, rows + 200)], 8, hd, 16, ct, seed=94)
    q = b.randn(rows, heads * hd).to(rt)
    assert splits(b, rt, heads, rows, window) == 0
    # Token p holds an infinity in KV head p % 8, dim p % 64 or the next: three of 64 neighbouring tokens, from half
    # of the rows on (without a window, all rows behind it see the early ones).
    bad = [p for p in range(200 + rows // 2, 200 + rows) if p % 64 in (0, 17, 50)]
    held = torch.zeros(rows + 200, 8, hd, dtype=torch.bool)
    clean = b.v.clone()
    for p in bad:
        at, d = b.token(0, p), (p + p // 64) % hd
        b.v[at][p // 64 % 8, d] = math.inf
        clean[at][p // 64 % 8, d] = 0.0
        held[p, p // 64 % 8, d] = True
    got = run(b, q, heads, 0.1, window)
    b.v = clean
    for r in sorted(set(spread(rows, 16)) | set(range(rows // 2 - 2, rows, rows // 29)) | {rows // 2 + i for i in range(5)}):
        p = 200 + r
        lo = max(0, p - window + 1) if window else 0
        inf = held[lo:p + 1].any(0).reshape(-1)
        assert torch.equal(~got[r].isfinite(), inf), f"row {r}"
        want, tol = row64(b, q, heads, 0.1, r, window)
        # Where a token's own value is infinite the definition is too; the other dims have the values as they are.
        err = (got[r].double() - want).abs()[~inf]
        assert (err <= tol[~inf]).all(), f"row {r}"


@pytest.mark.parametrize("rt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("seqs,split", [([(1, 9000)], True), ([(1, 9000)] * 2 + [(1, 2500)] * 130, False),
                                        ([(80, 9000)], True), ("chunk", False)], ids=["rows", "rows whole", "chunk", "chunk whole"])
def test_long_runs_of_bad_pages(seqs, split, rt, ct):
    """Hundreds of bad table entries before the only good one, whose keys give scores of -inf to some KV heads: those
    are not finite, the others are that page's mean, and without a good entry the row is 0."""
    rows = in_blocks(rt, 1)
    heads, G = (64, 8) if seqs == "chunk" else (8, 2)
    b = filled([(rows, rows + 5000)] if seqs == "chunk" else seqs, G, 64, 16, ct, seed=95)
    q = (b.randn(b.rows, heads * 64).abs() + 0.1).to(rt)
    assert (splits(b, rt, heads, b.rows) == 0) != split
    first = b.lens[0] - b.new[0]  # the first row's position
    for s in range(min(2, len(b.new))):
        b.table[s, :first // 16] = -1
    at, before = int(b.table[0, first // 16]), first % 16
    b.k[at][:before + 1, 0] = -math.inf  # what the first row sees, in the KV head 0
    if len(b.new) > 1:
        b.table[1] = b.pages
    got = run(b, q, heads, 0.1, bad=True)
    group = heads // G * 64
    assert not got[0, :group].isfinite().any()
    want, tol = row64(b, q, heads, 0.1, 0)
    assert ((got[0].double() - want).abs() <= tol)[group:].all()
    if len(b.new) > 1:
        assert (got[1] == 0).all()
        check_rows(b, q, heads, 0.1, got, range(2, b.rows, 9))
