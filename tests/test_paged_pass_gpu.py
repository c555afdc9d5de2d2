"""The operators together, as a serving step runs them: the paged pass against passes over private prefixes, and one
layer's steps by hand (projection, adapters, append, attention, projection) against float64."""
import math

import numpy as np
import pytest
import torch

from gophonic_amd import gphq
from tests import lm_common as lc
from tests.paged_common import BF16, F16, F32

pytestmark = pytest.mark.gpu

GEOM = dict(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=128, intermediate=1024, vocab=300, max_positions=640,
            eps=1e-6, rope_theta=1e6)


@pytest.fixture(scope="module")
def lm():
    return gphq.lm_random(GEOM, gphq.FMT_Q8B, 5)[0]


def cos(a, b):
    a, b = a.double().flatten(), b.double().flatten()
    return float(a @ b / (a.norm() * b.norm()))


def private(lm, tokens, split):
    """Last-token states of a private prefix extended by the pieces of `tokens` that end at `split`."""
    pf, kv = gphq.Prefill(lm, 512), gphq.Prefix(lm, GEOM["max_positions"])
    out, at = [], 0
    for end in split:
        h = torch.empty(GEOM["hidden"], device="cuda")
        pf.extend(kv, at, tokens[at:end], h)
        out.append(h)
        at = end
    pf.check()
    return out, kv


# fp32 and FP16 pages hold what the private pass's own arithmetic keeps (it rounds keys and values to FP16): the
# reference's bound of a pass against token-by-token evaluation, cosine 0.99999. bfloat16 pages round keys and values
# at 2^-8 each, 2^-7.5 of a value in all, over two layers: 1 - cosine is about half the square of the relative error.
@pytest.mark.parametrize("dtype,bound", [(F32, 0.99999), (F16, 0.99999), (BF16, 1 - 2 * 2.0 ** -15)],
                         ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [512, 60])
def test_paged_pass_against_private_prefixes(lm, dtype, bound, rows):
    """Three requests of different ages in shared passes: prompts in chunks, then single tokens, then both; passes
    of 60 rows cut the prompts again."""
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, GEOM["vocab"], n).astype(np.int32) for n in (150, 40, 301)]
    steps = [[100, 0, 300], [120, 33, 301], [121, 34, 301], [150, 40, 301]]  # tokens of each after each step
    pool = gphq.PagedPool(lm, 48, 16, dtype)
    pf = gphq.Prefill(lm, rows)
    table = np.full((3, 20), -1, np.int32)
    pages = list(rng.permutation(48))
    for s, p in enumerate(prompts):
        need = -(-len(p) // 16)
        table[s, :need] = pages[:need]
        pages = pages[need:]
    had = [0, 0, 0]
    ends = [sorted({st[s] for st in steps if st[s]}) for s in range(3)]
    want = [private(lm, p, e)[0] for p, e in zip(prompts, ends)]
    for step in steps:
        live = [s for s in range(3) if step[s] > had[s]]
        h = torch.empty(len(live), GEOM["hidden"], device="cuda")
        pf.paged(pool, [prompts[s][had[s]:step[s]] for s in live], [had[s] for s in live], table[live], h)
        pf.check()
        for i, s in enumerate(live):
            assert cos(h[i], want[s][ends[s].index(step[s])]) >= bound
            had[s] = step[s]


def test_first_layer_rows_are_the_private_prefix_s_bits(lm):
    """fp32 pages: layer 0's keys and values of a prompt equal, bit for bit, the rows that a private prefix holds."""
    rng = np.random.default_rng(2)
    ids = rng.integers(0, GEOM["vocab"], 77).astype(np.int32)
    _, kv = private(lm, ids, [77])
    pool, pf = gphq.PagedPool(lm, 9, 16, F32), gphq.Prefill(lm, 512)
    table = rng.permutation(9)[None, :5].astype(np.int32)
    h = torch.empty(1, GEOM["hidden"], device="cuda")
    pf.paged(pool, [ids], [0], table, h)
    layer = pool.layer(0)
    kc, vc, cap = kv.kv()

    class Rows:
        def __init__(self, a):
            self.__cuda_array_interface__ = dict(shape=(cap, 2, 128), typestr="<f4", data=(a, False), version=2)

    for mine, theirs in ((layer.k, kc), (layer.v, vc)):
        rows = torch.as_tensor(Rows(theirs), device="cuda")
        got = torch.stack([mine[int(table[0, p // 16]), p % 16] for p in range(77)])
        assert torch.equal(got, rows[:77])


def test_shared_prompt_pages(lm):
    """Two continuations of one prompt whose whole pages they share, each with pages of its own behind them."""
    rng = np.random.default_rng(3)
    ids = rng.integers(0, GEOM["vocab"], 64).astype(np.int32)
    more = [rng.integers(0, GEOM["vocab"], n).astype(np.int32) for n in (5, 20)]
    pool, pf = gphq.PagedPool(lm, 12, 16, F16), gphq.Prefill(lm, 128)
    first = np.array([[3, 1, 4, 9]], np.int32)
    h = torch.empty(1, GEOM["hidden"], device="cuda")
    pf.paged(pool, [ids], [0], first, h)
    table = np.array([[3, 1, 4, 9, 2, -1], [3, 1, 4, 9, 6, 5]], np.int32)
    h2 = torch.empty(2, GEOM["hidden"], device="cuda")
    pf.paged(pool, more, [64, 64], table, h2)
    pf.check()
    for i, m in enumerate(more):
        want, _ = private(lm, np.concatenate([ids, m]), [64, 64 + len(m)])
        assert cos(h2[i], want[1]) >= 0.99999


def test_int8_route(lm):
    lm8 = gphq.lm_random(GEOM, gphq.FMT_Q8, 6)[0]
    rng = np.random.default_rng(4)
    ids = rng.integers(0, GEOM["vocab"], 90).astype(np.int32)
    pf, kv = gphq.Prefill(lm8, 128), gphq.Prefix(lm8, 128)
    pf.set_arith(gphq.PASS_INT8)
    want = torch.empty(GEOM["hidden"], device="cuda")
    pf.extend(kv, 0, ids, want)
    pool = gphq.PagedPool(lm8, 8, 32, F32)
    h = torch.empty(1, GEOM["hidden"], device="cuda")
    pf.paged(pool, [ids], [0], np.array([[0, 2, 7]], np.int32), h)
    pf.check()
    # The same int8 projections around attention in FP16 tiles there and fp32 here: an activation near a rounding
    # border may take the next code, 2^-7 of its row's largest.
    assert cos(h, want) >= 0.999


@pytest.mark.parametrize("seqs,past,table,status", [
    ([[1, 2]], [0], [[12]], gphq.ERR_PAGED_BATCH), ([[1, 2]], [0], [[-1]], gphq.ERR_PAGED_BATCH),
    ([[1], [2]], [0, 0], [[3], [3]], gphq.ERR_PAGED_BATCH), ([[1] * 20], [0], [[3, 3]], gphq.ERR_PAGED_BATCH),
    ([[1] * 20], [0], [[3]], gphq.ERR_PAGED_SHAPE), ([[1]], [-1], [[3]], gphq.ERR_KEEP_RANGE),
    ([[]], [0], [[3]], gphq.ERR_EMPTY_SEQUENCE), ([[1]], [640], [[3] * 41], gphq.ERR_CONTEXT),
    ([[1]], [2 ** 62], [[3]], gphq.ERR_CONTEXT), ([[300]], [0], [[3]], gphq.ERR_TOKEN_VOCAB),
    ([], [], np.zeros((0, 1)), gphq.ERR_SEQUENCE_COUNT),
], ids=lambda v: None)
def test_paged_pass_refuses(lm, seqs, past, table, status):
    pool, pf = gphq.PagedPool(lm, 12, 16, F16), gphq.Prefill(lm, 128)
    h = torch.full((max(len(seqs), 1), GEOM["hidden"]), 7.0, device="cuda")
    with pytest.raises(gphq.GphqError) as e:
        pf.paged(pool, seqs, past, np.asarray(table), h[:len(seqs)])
    assert e.value.status == status
    assert (h == 7).all()


@pytest.mark.parametrize("seqs,past,table", [
    ([[1]], [16], [[3, 3]]), ([[1], [2]], [16, 0], [[3, 4], [3, 5]]), ([[1], [2]], [5, 40], [[3, 0, 0], [4, 3, 5]]),
])
def test_paged_pass_refuses_to_write_a_page_that_is_read(lm, seqs, past, table):
    """A page of earlier tokens, of the same sequence or another's, that this step would write over."""
    pool, pf = gphq.PagedPool(lm, 12, 16, F16), gphq.Prefill(lm, 128)
    with pytest.raises(gphq.GphqError) as e:
        pf.paged(pool, seqs, past, np.asarray(table), torch.empty(len(seqs), GEOM["hidden"], device="cuda"))
    assert e.value.status == gphq.ERR_PAGED_BATCH


@pytest.mark.parametrize("ids,table,status", [
    ([2 ** 32 + 5], [[3]], gphq.ERR_TOKEN_VOCAB), ([-2 ** 32 + 5], [[3]], gphq.ERR_TOKEN_VOCAB),
    ([5], [[2 ** 32 + 3]], gphq.ERR_PAGED_BATCH), ([5], [[-2 ** 32 + 3]], gphq.ERR_PAGED_BATCH),
])
def test_paged_pass_refuses_numbers_past_32_bits(lm, ids, table, status):
    """They are not taken for their low halves, which name a token and a page."""
    pool, pf = gphq.PagedPool(lm, 12, 16, F16), gphq.Prefill(lm, 128)
    with pytest.raises(gphq.GphqError) as e:
        pf.paged(pool, [np.array(ids)], [0], np.array(table), torch.empty(1, GEOM["hidden"], device="cuda"))
    assert e.value.status == status


@pytest.mark.parametrize("make", [lambda h: h.half(), lambda h: h.cpu(), lambda h: h.t().contiguous().t(),
                                  lambda h: h.repeat(1, 2)[:, :h.shape[1]], lambda h: h[:, :1].expand(*h.shape)],
                         ids=["half", "host", "transposed", "wider", "expanded"])
def test_paged_pass_refuses_a_result_that_is_not_rows_of_float32(lm, make):
    pool, pf = gphq.PagedPool(lm, 12, 16, F16), gphq.Prefill(lm, 128)
    with pytest.raises(gphq.GphqError):
        pf.paged(pool, [[1], [2, 3]], [0, 0], [[3], [4]], make(torch.empty(2, GEOM["hidden"], device="cuda")))


def test_paged_pass_refuses_another_model_s_pool(lm):
    other = gphq.lm_random(dict(GEOM, layers=1), gphq.FMT_Q8B, 7)[0]
    pool, pf = gphq.PagedPool(other, 4, 16, F16), gphq.Prefill(lm, 16)
    with pytest.raises(gphq.GphqError) as e:
        pf.paged(pool, [[1]], [0], [[0]], torch.empty(1, GEOM["hidden"], device="cuda"))
    assert e.value.status == gphq.ERR_FOREIGN_PREFIX
    for args in ((0, 16, F16), (4, 24, F16), (4, 8, F16)):
        with pytest.raises(gphq.GphqError):
            gphq.PagedPool(lm, *args)
    with pytest.raises(gphq.GphqError):
        pool.layer(1)


def test_one_layer_by_hand_with_adapters(lm):
    """QKV projection of a mixed batch, the rows' adapters, append, attention, O projection: the library's calls in a
    row against float64 from the projection's own output on."""
    H, heads, G, D = GEOM["hidden"], GEOM["heads"], GEOM["kv_heads"], 128
    width, rank = (heads + 2 * G) * D, 8
    g = torch.Generator().manual_seed(11)
    new, old = [1, 37, 1, 5], [90, 0, 16, 20]
    rows = sum(new)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    lens = [a + b for a, b in zip(new, old)]
    x = torch.randn(rows, H, generator=g).cuda()
    a, b = torch.randn(2, rank, H, generator=g) * 0.05, torch.randn(2, width, rank, generator=g) * 0.05
    a, b = a.bfloat16().cuda(), b.bfloat16().cuda()
    slot_of = [1, 0, -1, 1]
    slots = torch.tensor([s for n, s in zip(new, slot_of) for _ in range(n)], dtype=torch.int32).cuda()
    pf = gphq.Prefill(lm, 64)
    qkv = torch.empty(rows, width, device="cuda")
    pf.project(0, 0, x, rows, qkv)
    base = qkv.double().cpu()
    gphq.lora_add(a, b, x, qkv, slots)

    pool = gphq.PagedPool(lm, 20, 16, F32)
    kv = pool.layer(1)
    table = np.full((4, 7), -1, np.int32)
    perm = torch.randperm(20, generator=g).tolist()
    for s, n in enumerate(lens):
        for e in range(-(-n // 16)):
            table[s, e] = perm.pop()
    past = [[(torch.randn(G, D, generator=g), torch.randn(G, D, generator=g)) for _ in range(o)] for o in old]
    for s, o in enumerate(old):
        for p in range(o):
            kv.k[int(table[s, p // 16]), p % 16] = past[s][p][0].cuda()
            kv.v[int(table[s, p // 16]), p % 16] = past[s][p][1].cuda()
    batch = gphq.PagedBatch(torch.from_numpy(starts).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                            torch.from_numpy(table).cuda(), rows, max(new), max(lens))
    qn, kn = 1 + 0.1 * torch.randn(D, generator=g), 1 + 0.1 * torch.randn(D, generator=g)
    ang = torch.arange(128, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(64, dtype=torch.float64) / 64)
    c, s_ = ang.cos().float(), ang.sin().float()
    gphq.paged_append(kv, batch, qkv, qkv, heads, qn.cuda(), kn.cuda(), 1e-6, c.cuda(), s_.cuda(), D ** -0.5)
    ctx = torch.empty(rows, heads * D, device="cuda")
    gphq.paged_attention(kv, batch, qkv, ctx, heads, 1.0)
    out = torch.zeros(rows, H, device="cuda")
    pf.project(0, 1, ctx, rows, out)
    batch.check()

    # float64, with the rows the projection gave.
    full = base.clone()
    for r in range(rows):
        s = int(slots[r])
        if s >= 0:
            full[r] += b[s].double().cpu() @ (a[s].double().cpu() @ x[r].double().cpu())
    head = full.view(rows, heads + 2 * G, D)

    def prep(h, w, p):
        h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w.double()
        lo, hi = h[:, :64], h[:, 64:]
        return torch.cat([lo * c[p].double() - hi * s_[p].double(), hi * c[p].double() + lo * s_[p].double()], -1)

    want = torch.zeros(rows, heads, D, dtype=torch.float64)
    for s in range(4):
        k, v = [p[0].double() for p in past[s]], [p[1].double() for p in past[s]]
        for i in range(new[s]):
            r, p = starts[s] + i, old[s] + i
            k.append(prep(head[r, heads:heads + G], kn, p))
            v.append(head[r, heads + G:])
            q = prep(head[r, :heads], qn, p) * D ** -0.5
            K, V = torch.stack(k), torch.stack(v)
            for h in range(heads):
                want[r, h] = torch.softmax(K[:, h // 4] @ q[h], 0) @ V[:, h // 4]
    want = want.view(rows, heads * D)
    # fp32 throughout. Adapters add rank + H products in fp32 (520 u of their magnitudes, here below the row's own
    # size), the norm and rotation 72 u, a score of 128 products and size up to 6: 140 u * 6 twice, the sums over up
    # to 91 keys 250 u: under 3000 u = 2^-12.4 of a value's size.
    err = (ctx.cpu().double() - want).abs()
    assert (err <= 2.0 ** -12.4 * (1 + want.abs().amax(1, keepdim=True))).all(), float(err.max())
    ref = torch.zeros(rows, H, device="cuda")
    pf.project(0, 1, want.float().cuda(), rows, ref)
    # The O projection of both: its activations are rounded to FP16 per row (2^-11 of the row's largest).
    assert cos(out, ref) >= 0.99999
    assert math.isfinite(float(out.sum()))


def test_memory_that_is_not_there_leaves_no_error(lm):
    """A pool too large for the device is refused; neither the next call nor torch's next kernel reports it again."""
    for _ in range(2):
        with pytest.raises(gphq.GphqError):
            gphq.PagedPool(lm, 2 ** 31 - 1, 4096, F32)
        x = torch.zeros(64, device="cuda") + 1
        pool, pf = gphq.PagedPool(lm, 4, 16, F16), gphq.Prefill(lm, 16)
        h = torch.empty(1, GEOM["hidden"], device="cuda")
        with pytest.raises(gphq.GphqError):
            gphq.PagedPool(lm, 2 ** 31 - 1, 4096, F32)
        pf.paged(pool, [[1, 2, 3]], [0], [[2]], h)
        pf.check()
        assert h.isfinite().all() and float(x.sum()) == 64


def test_adapters_beside_a_layer_s_projections(lm):
    """The adapters of QKV on the rows that the projection multiplies (normalized by the caller), those of O on the
    context: what they add is B (A x) of those rows, on top of what the projections give alone."""
    H, heads, G, D, rank, rows = GEOM["hidden"], GEOM["heads"], GEOM["kv_heads"], 128, 16, 45
    g = torch.Generator().manual_seed(21)
    x, ctx = torch.randn(rows, H, generator=g).cuda() * 2, torch.randn(rows, heads * D, generator=g).cuda()
    slots = torch.arange(rows, dtype=torch.int32).cuda() % 4 - 1
    pf = gphq.Prefill(lm, 64)
    xn = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + GEOM["eps"])
    for proj, rows_in, width, y in ((0, xn, (heads + 2 * G) * D, torch.empty(rows, (heads + 2 * G) * D, device="cuda")),
                                    (1, ctx, H, x.clone())):
        a = (torch.randn(3, rank, rows_in.shape[1], generator=g) * 0.05).bfloat16().cuda()
        b = (torch.randn(3, width, rank, generator=g) * 0.05).bfloat16().cuda()
        pf.project(0, proj, x if proj == 0 else ctx, rows, y)
        alone = y.double()
        gphq.lora_add(a, b, rows_in, y, slots)
        A, B, v = a.double()[slots.clamp(min=0).long()], b.double()[slots.clamp(min=0).long()], rows_in.double()
        on = (slots >= 0).double()[:, None]
        low = (A * v[:, None]).sum(-1)
        want = alone + on * (B * low[:, None]).sum(-1)
        # (k + rank + 8) u of the products' magnitudes, and one u of the sum with what was there.
        size = (B.abs() * (A.abs() * v.abs()[:, None]).sum(-1)[:, None]).sum(-1)
        tol = (rows_in.shape[1] + rank + 8) * 2.0 ** -24 * size + 2.0 ** -24 * (alone.abs() + want.abs())
        assert ((y.double() - want).abs() <= tol).all()
        assert torch.equal(y[0].double(), alone[0])  # no adapter
