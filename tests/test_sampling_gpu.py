"""gphq_probabilities and gphq_verify_drafts on the GPU against their definitions in float64."""
import math

import numpy as np
import pytest
import torch

from gophonic_amd import gphq

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


# ---- probabilities ----------------------------------------------------------------


def softmax64(x, t):
    """The definition of one row, t > 0, in float64; and a bound of fp32's error relative to each value: the exponent
    (x - max) / t, off by 2^-23 of itself (difference, rate and product, 3 u), the exponentials and the division a few
    units, a sum of n terms in tiles of 16 and trees at most (16 + 24) u and as much as its terms."""
    x = x.double()
    z = (x - x.max()) / t
    p = z.exp() / z.exp().sum()
    w = torch.where(p > 0, z.abs() * p, 0.0).sum()  # of the sum's error
    return p, 2.0 ** -22 * (z.abs() + w) + 64 * 2.0 ** -24


def check_row(got, x, t):
    got = got.double()
    x = x.double()
    if t > 0:
        if x.isnan().any() or (x == INF).any():
            assert got.isnan().all()
        elif (x == -INF).all():
            assert (got == 0).all()
        else:
            p, rel = softmax64(x, max(t, 1.5e-38))
            p, rel = p.nan_to_num(0.0), torch.where(p > 0, rel, 0.0)
            assert ((got - p).abs() <= rel * p * 1.01 + 2.0 ** -126).all(), float(((got - p).abs() / p.clamp(min=1e-30)).max())
    else:
        best = torch.where(x.isnan(), -INF, x)
        want = torch.zeros_like(best)
        if best.max() > -INF:
            want[int((best == best.max()).nonzero()[0])] = 1
        assert torch.equal(got, want)


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 257, 1000, 4095, 4096, 4097, 12345, 151936])
@pytest.mark.parametrize("rows", [1, 2, 7])
def test_rows(rows, vocab):
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=g) * 4
    t = torch.tensor([1.0, 0.0, 0.3, 2.5, 0.0, 1e-3, 50.0])[:rows]
    out = torch.empty(rows, vocab, device="cuda")
    gphq.probabilities(x.cuda(), out, t.cuda())
    for r in range(rows):
        check_row(out[r].cpu(), x[r], float(t[r]))
    gphq.probabilities(x.cuda(), out)
    for r in range(rows):
        check_row(out[r].cpu(), x[r], 1.0)


@pytest.mark.parametrize("rows,vocab", [(300, 5000), (2500, 33), (40, 70001), (9000, 1)])
def test_many_rows(rows, vocab):
    """Parts of several tiles, and more rows than blocks are wanted."""
    x = torch.randn(rows, vocab, device="cuda") * 3
    t = torch.rand(rows, device="cuda").clamp(min=0.2)
    t[::5] = 0
    out = torch.empty_like(x)
    gphq.probabilities(x, out, t)
    z = (x.double() - x.double().amax(1, keepdim=True)) / t.double()[:, None].clamp(min=0.1)
    p = z.exp() / z.exp().sum(1, keepdim=True)
    live = t > 0
    rel = 2.0 ** -22 * (z.abs() + (z.abs() * p).sum(1, keepdim=True)) + 64 * 2.0 ** -24
    assert ((out.double() - p).abs() <= rel * p * 1.01 + 2.0 ** -126)[live].all()
    one = torch.zeros_like(x)
    one[torch.arange(rows, device="cuda"), (x == x.amax(1, keepdim=True)).float().argmax(1)] = 1
    assert torch.equal(out[~live], one[~live])


@pytest.mark.parametrize("pad", [0, 1, 3, 4, 32])
@pytest.mark.parametrize("off", [0, 1, 4])
def test_strides_and_alignment(pad, off):
    """Rows of wider buffers, of any alignment; what lies between them is left alone."""
    V = 5003
    wide = torch.randn(5, V + pad + off, device="cuda")
    dst = torch.full((5, V + 2 * pad + off), 7.0, device="cuda")
    gphq.probabilities(wide[:, off:off + V], dst[:, off:off + V])
    x = wide[:, off:off + V].contiguous()
    out = torch.empty_like(x)
    gphq.probabilities(x, out)
    for r in range(5):
        check_row(dst[r, off:off + V].cpu(), x[r].cpu(), 1.0)
    assert (dst[:, :off] == 7).all() and (dst[:, off + V:] == 7).all()


@pytest.mark.parametrize("vocab", [5, 4096, 9001])
def test_rows_that_are_not_finite(vocab):
    """Masked logits (-inf), the type's lowest value, rows of -inf alone, NaN and +inf, at t = 0 and above."""
    low = float(torch.finfo(torch.float32).min)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(12, vocab, generator=g)
    x[0, : vocab // 2] = -INF
    x[1] = -INF
    x[2, 3] = NAN
    x[3, 2] = INF
    x[4] = low
    x[5, 1:] = low
    x[6] = -INF
    x[6, vocab - 1] = low
    x[7, 4] = INF
    x[7, 1] = INF
    x[8] = NAN
    x[9] = float(torch.finfo(torch.float32).max)
    x[10] = 0.0
    x[11, ::2] = -INF
    for temp in (1.0, 0.0, 0.25, -1.0, NAN):
        out = torch.empty(12, vocab, device="cuda")
        gphq.probabilities(x.cuda(), out, torch.full((12,), temp, device="cuda"))
        for r in range(12):
            check_row(out[r].cpu(), x[r], temp if temp > 0 else 0.0)


@pytest.mark.parametrize("t", [1e-45, 1e-38, 1e-20, 1e20, 3e38, INF])
def test_temperatures_of_every_size(t):
    x = torch.randn(3, 777)
    x[1, 5] = -INF
    out = torch.empty(3, 777, device="cuda")
    gphq.probabilities(x.cuda(), out, torch.full((3,), t, device="cuda"))
    got = out.cpu().double()
    if t < 1:
        for r in range(3):
            assert int(got[r].argmax()) == int(x[r].argmax()) and abs(float(got[r].sum()) - 1) < 1e-6
    else:
        for r in range(3):
            live = x[r] > -INF
            assert ((got[r][live] - 1 / int(live.sum())).abs() < 1e-8).all() and (got[r][~live] == 0).all()


def test_in_place_repeats_and_another_stream():
    x = torch.randn(70, 30011, device="cuda") * 5
    out = torch.empty_like(x)
    gphq.probabilities(x, out)
    both = x.clone()
    gphq.probabilities(both, both)
    assert torch.equal(both, out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        two = torch.empty_like(x)
        side.wait_stream(torch.cuda.current_stream())
        gphq.probabilities(x, two, stream=side)
        side.synchronize()
        assert torch.equal(two, out)


# ---- drafts ---------------------------------------------------------------------


def verified(starts, drafts, p, q, u, v, rows):
    """The definition: tokens (None: left alone), accepted, and the decisions' distance from a border."""
    tokens, accepted = [None] * rows, []
    p = p.astype(np.float64)
    q = None if q is None else q.astype(np.float64)
    V = p.shape[1]
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        b -= 1
        if a < 0 or b < a - 1 or b >= rows or a > rows:
            accepted.append(-1)
            continue
        if b == a - 1:
            accepted.append(0)
            continue
        r = a
        while r < b:
            x = drafts[r]
            if not 0 <= x < V:
                break
            if not float(u[r]) * (1.0 if q is None else q[r, x]) < p[r, x]:
                break
            r += 1
        w = np.where(p[r] > 0, p[r], 0)
        if r < b and 0 <= drafts[r] < V:
            if q is None:
                less = w.copy()
                less[drafts[r]] = 0
            else:
                with np.errstate(invalid="ignore"):
                    less = p[r] - q[r]
                less = np.where(less > 0, less, 0)
            if less.sum() > 0:
                w = less
        cum = np.cumsum(w)
        vs = float(v[s])
        vs = min(max(vs, 0.0), 1 - 2.0 ** -24) if vs == vs else 0.0
        with np.errstate(invalid="ignore"):
            over = np.nonzero((cum > vs * cum[-1]) & (w > 0))[0]
        pos = np.nonzero(w > 0)[0]
        token = int(over[0]) if len(over) else int(pos[-1]) if len(pos) else 0
        tokens[a:b + 1] = [int(x) for x in drafts[a:r]] + [token] + [-1] * (b - r)
        accepted.append(r - a)
    return tokens, accepted


def run(starts, drafts, p, q, u, v, lens=None, in_place=False):
    rows = p.shape[0]
    up = lambda a, t: torch.as_tensor(np.asarray(a), dtype=t).cuda()
    d = up(drafts, torch.int32)
    tokens = d if in_place else torch.full((rows,), 7, dtype=torch.int32, device="cuda")
    accepted = torch.full((len(starts) - 1,), 9, dtype=torch.int32, device="cuda")
    l = None if lens is None else up(lens, torch.int32)
    kept = None if lens is None else l if in_place else torch.empty_like(l)
    gphq.verify_drafts(up(starts, torch.int32), d, up(p, torch.float32), None if q is None else up(q, torch.float32),
                       up(u, torch.float32), up(v, torch.float32), tokens, accepted, l, kept)
    return tokens.tolist(), accepted.tolist(), None if kept is None else kept.tolist()


def rows_of(r, rows, vocab, sharp=3.0):
    x = r.standard_normal((rows, vocab)) * sharp
    e = np.exp(x - x.max(1, keepdims=True))
    return (e / e.sum(1, keepdims=True)).astype(np.float32)


def compare(starts, drafts, p, q, u, v, in_place=False):
    rows = p.shape[0]
    lens = [100 + i for i in range(len(starts) - 1)]
    tokens, accepted, kept = run(starts, drafts, p, q, u, v, lens, in_place)
    want, count = verified(starts, drafts, p, q, u, v, rows)
    assert accepted == count
    for r in range(rows):
        assert tokens[r] == (want[r] if want[r] is not None else drafts[r] if in_place else 7), r
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        assert kept[s] == lens[s] - (max(b - a - 1, 0) - count[s] if count[s] >= 0 and b > a else 0)


@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in place"])
@pytest.mark.parametrize("certain", [False, True], ids=["probabilities", "certain"])
@pytest.mark.parametrize("vocab", [1, 2, 5, 64, 1000, 4096, 4097, 20011])
@pytest.mark.parametrize("lens", [[0], [5], [0, 3, 0, 1, 8, 2], [1] * 70, [64, 65, 130]])
def test_drafts(lens, vocab, certain, in_place):
    r = np.random.default_rng(vocab + len(lens))
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n + 1)
    rows = starts[-1]
    p = rows_of(r, rows, vocab)
    q = rows_of(r, rows, vocab) * 0.3 + p * 0.7
    # Drafts that are likely, so that some sequences get far.
    drafts = [int(x) for x in np.where(r.random(rows) < 0.9, p.argmax(1), r.integers(0, vocab, rows))]
    compare(starts, drafts, p, None if certain else q.astype(np.float32), r.random(rows, np.float32),
            r.random(len(lens), np.float32), in_place)


@pytest.mark.parametrize("certain", [False, True])
def test_random_numbers_at_their_ends(certain):
    """0 accepts whatever the target can give and takes the first token with a weight, 1 - 2^-24 takes the last ones;
    numbers outside 0 .. 1, and NaN, are taken into it."""
    r = np.random.default_rng(3)
    p, q = rows_of(r, 24, 300), rows_of(r, 24, 300)
    p[:, :5] = 0
    p[:, -5:] = 0
    starts = list(range(0, 25, 3))
    drafts = [int(x) for x in q.argmax(1)]
    for u in (0.0, 0.5, 1 - 2.0 ** -24, 1.0):
        for v in (0.0, 2.0 ** -24, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, NAN):
            compare(starts, drafts, p, None if certain else q, np.full(24, u, np.float32), np.full(8, v, np.float32))


def test_drafts_the_target_cannot_give():
    """A draft of probability 0 (u = 0 too), outside the vocabulary, certain of the only token; equal rows, whose rest
    is empty; rows of zeros."""
    p = np.zeros((12, 70), np.float32)
    p[:, 10:20] = 0.1
    q = p.copy()
    drafts = [5, 0, -1, 0, 70, 0, 12, 0, 2 ** 31 - 1, 0, -2 ** 31, 0]
    starts = [0, 2, 4, 6, 8, 10, 12]
    for u in (0.0, 0.99):
        for v in (0.0, 0.3, 0.999):
            compare(starts, drafts, p, q, np.full(12, u, np.float32), np.full(6, v, np.float32))
            compare(starts, drafts, p, None, np.full(12, u, np.float32), np.full(6, v, np.float32))
    zero = np.zeros_like(p)
    compare(starts, drafts, zero, q, np.full(12, 0.5, np.float32), np.full(6, 0.5, np.float32))
    one = np.zeros((4, 70), np.float32)
    one[:, 33] = 1
    compare([0, 2, 4], [33, 0, 32, 0], one, None, np.full(4, 0.999, np.float32), np.full(2, 0.999, np.float32))


@pytest.mark.parametrize("bad", [NAN, INF, -1.0, -INF])
def test_weights_that_are_no_probabilities(bad):
    r = np.random.default_rng(4)
    p, q = rows_of(r, 8, 5000), rows_of(r, 8, 5000)
    p[:, 77] = bad
    q[3, 99] = bad
    drafts = [0] * 8
    compare([0, 2, 4, 6, 8], drafts, p, q, np.full(8, 0.9, np.float32), np.array([0.1, 0.5, 0.7, 0.99], np.float32))


def test_starts_that_are_no_rows():
    """Sequences without rows, descending starts, starts outside the rows; rows of no sequence are left alone."""
    r = np.random.default_rng(5)
    p, q = rows_of(r, 10, 100), rows_of(r, 10, 100)
    u, drafts = r.random(10, np.float32), [int(x) for x in q.argmax(1)]
    for starts in ([2, 4, 4, 7], [0, 3, 2, 5], [-2, 3, 6], [5, 8, 11], [10, 10], [11, 11], [-1, -1], [2 ** 31 - 1, -2 ** 31, 3],
                   [3, 3]):
        v = r.random(len(starts) - 1, np.float32)
        lens = [50] * (len(starts) - 1)
        tokens, accepted, kept = run(starts, drafts, p, q, u, v, lens)
        want, count = verified(starts, drafts, p, q, u, v, 10)
        assert accepted == count, starts
        # (Where starts descend two sequences may have a row each for its own; it holds the token of either.)
        may = [{7} if w is None else set() for w in want]
        for s, (a, b) in enumerate(zip(starts, starts[1:])):
            mine, _ = verified([a, b], drafts, p, q, u, v[s:s + 1], 10)
            for row, t in enumerate(mine):
                may[row] |= set() if t is None else {t}
        assert all(t in m for t, m in zip(tokens, may)), starts
        assert all(k == 50 for k, c in zip(kept, count) if c < 0)


def test_the_whole_vocabulary():
    """151936 tokens, odd strides; sums in the definition's order of blocks against numpy's: a token is the same unless
    a number lies within 2^-45 of a border."""
    r = np.random.default_rng(6)
    V, lens = 151936, [0, 4, 2, 5, 0, 1]
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n + 1)
    rows = starts[-1]
    p = rows_of(r, rows, V, 2.0)
    q = (p * (1 + 0.5 * r.standard_normal(p.shape))).clip(0).astype(np.float32)
    drafts = [int(x) for x in p.argmax(1)]
    compare(starts, drafts, p, q, r.random(rows, np.float32), r.random(6, np.float32))
    wide = torch.zeros(rows, V + 3, device="cuda")
    wide[:, 1:V + 1] = torch.from_numpy(p).cuda()
    u, v = torch.from_numpy(r.random(rows, np.float32)).cuda(), torch.from_numpy(r.random(6, np.float32)).cuda()
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    tokens, accepted = ints([7] * rows), ints([9] * 6)
    gphq.verify_drafts(ints(starts), ints(drafts), wide[:, 1:V + 1], None, u, v, tokens, accepted)
    want, count = verified(starts, drafts, p, None, u.cpu().numpy(), v.cpu().numpy(), rows)
    assert tokens.tolist() == want and accepted.tolist() == count


@pytest.mark.parametrize("certain", [False, True])
def test_tokens_are_distributed_as_the_target_s(certain):
    """One draft of q, 60000 times with random numbers of their own: the first token is p's, the counts within five
    standard deviations; a draft is accepted as often as sum min(p, q)."""
    n, V = 60000, 12
    r = np.random.default_rng(7)
    p, q = rows_of(r, 1, V, 1.0)[0], rows_of(r, 1, V, 1.0)[0]
    drafts = r.choice(V, n, p=q.astype(np.float64) / q.astype(np.float64).sum())
    if certain:
        drafts[:] = 3
    starts = np.arange(0, 2 * n + 1, 2)
    both = np.stack([drafts, np.zeros(n, int)], 1).reshape(-1)
    P, Q = np.tile(p, (2 * n, 1)), np.tile(q, (2 * n, 1))
    tokens, accepted, _ = run(starts, both, P, None if certain else Q, r.random(2 * n, np.float32), r.random(n, np.float32))
    first = np.array(tokens)[::2]
    got = np.bincount(first, minlength=V)
    assert (np.abs(got - n * p) <= 5 * np.sqrt(n * p * (1 - p)) + 1).all()
    rate = float(p[3]) if certain else float(np.minimum(p, q).sum())
    assert abs(sum(accepted) - n * rate) <= 5 * math.sqrt(n * rate * (1 - rate))


def test_captured_and_repeated():
    """One captured chain of probabilities and verification, replayed with other logits; the same as eager calls."""
    V, lens = 9001, [3, 0, 5]
    starts = [0, 4, 5, 11]
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    st, drafts = ints(starts), ints([0] * 11)
    x, q = torch.randn(11, V, device="cuda"), torch.randn(11, V, device="cuda")
    p = torch.empty_like(x)
    t = torch.tensor([1.0, 0.5, 0.0, 1.0] * 2 + [0.7] * 3, device="cuda")
    u, v = torch.rand(11, device="cuda"), torch.rand(3, device="cuda")
    tokens, accepted = ints([0] * 11), ints([0] * 3)
    w1 = torch.empty(gphq.probabilities_workspace_bytes(11, V), dtype=torch.uint8, device="cuda")
    w2 = torch.empty(gphq.verify_drafts_workspace_bytes(3, V), dtype=torch.uint8, device="cuda")

    def step(p, tokens, accepted, w1=None, w2=None):
        gphq.probabilities(x, p, t, w1)
        gphq.verify_drafts(st, drafts, p, q, u, v, tokens, accepted, work=w2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step(p, tokens, accepted, w1, w2)
    torch.cuda.synchronize()
    for i in range(5):
        x.normal_().mul_(4)
        q.copy_(torch.softmax(x + torch.randn_like(x), 1))
        drafts.copy_(q.argmax(1))
        u.uniform_()
        v.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        p2, tokens2, accepted2 = torch.empty_like(p), torch.full_like(tokens, -9), torch.full_like(accepted, -9)
        step(p2, tokens2, accepted2)
        assert torch.equal(p, p2) and torch.equal(tokens, tokens2) and torch.equal(accepted, accepted2)
