"""gphq_lora_add against its definition in float64."""
import pytest
import torch

from gophonic_amd import gphq

pytestmark = pytest.mark.gpu
NAN = float("nan")


def make(rows, k, n, slots, max_rank, ranks, dtype, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    a, b = (r(slots, max_rank, k) * 0.1).to(dtype), (r(slots, n, max_rank) * 0.1).to(dtype)
    for s, rank in enumerate(ranks):  # what an adapter does not use may hold anything
        a[s, rank:] = NAN
        b[s, :, rank:] = NAN
    x, y = r(rows, k + pad) * 3, r(rows, n + pad)
    return a, b, x, y, r(slots).abs() + 0.5


def expect(a, b, x, y, row_slots, ranks, scales):
    """float64 y, and what fp32 may lose of it: with u = 2^-24 a sum of k products is off by at most (k + 2) u of their
    magnitudes, whatever its order; the second product carries that on and adds (rank + 2) u, the scale and the last
    sum one u each of what they meet."""
    y = y.double().clone()
    tol = y.abs() * 2.0 ** -24
    for r, s in enumerate(row_slots):
        if 0 <= s < len(ranks):
            rank, sc = ranks[s], float(scales[s])
            A, B, v = a[s, :rank].double(), b[s, :, :rank].double(), x[r].double()
            t, ta = A @ v, A.abs() @ v.abs()
            y[r] += sc * (B @ t)
            tol[r] += (x.shape[1] + rank + 8) * 2.0 ** -24 * sc * (B.abs() @ ta) + y[r].abs() * 2.0 ** -24
    return y, tol


CASES = [
    # rows, k, n, slots, max_rank, ranks, slot of every row
    (1, 32, 1, 1, 8, [8], [0]),
    (1, 256, 70, 3, 16, [16, 1, 5], [2]),
    (5, 64, 33, 2, 8, [3, 8], [0, -1, 1, 2, 0]),
    (16, 128, 257, 16, 16, list(range(1, 17)), list(range(16))),
    (37, 160, 300, 4, 64, [64, 17, 0, 33], [(7 * i) % 6 - 1 for i in range(37)]),
    (64, 1024, 1500, 2, 32, [32, 31], [0] * 30 + [1] * 34),
    (300, 512, 260, 3, 128, [128, 100, 65], [i // 110 for i in range(300)]),
    (513, 96, 64, 5, 24, [24, 24, 9, 24, 16], [(i // 50) % 7 - 1 for i in range(513)]),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_lora(case, dtype):
    rows, k, n, slots, max_rank, ranks, row_slots = CASES[case]
    a, b, x, y, scales = make(rows, k, n, slots, max_rank, ranks, dtype, case)
    want, tol = expect(a, b, x, y, row_slots, ranks, scales)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    d = y.cuda()
    gphq.lora_add(a.cuda(), b.cuda(), x.cuda(), d, i32(row_slots), i32(ranks), scales.cuda())
    err = (d.cpu().double() - want).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-30)).max())
    free = [r for r, s in enumerate(row_slots) if not 0 <= s < slots]
    assert torch.equal(d[free].cpu(), y[free])  # rows without an adapter keep their bits


def test_strides_defaults_stream_and_repeats():
    """Rows in wider buffers at odd strides; no ranks and no scales; another stream; the same bits every time."""
    rows, k, n, slots, R = 50, 128, 131, 2, 16
    a, b, x, y, _ = make(rows, k, n, slots, R, [R, R], torch.bfloat16, 5, pad=4)
    row_slots = [i % 3 for i in range(rows)]
    want, tol = expect(a, b, x[:, :k].contiguous(), y[:, :n].contiguous(), row_slots, [R, R], [1.0, 1.0])
    rs = torch.tensor(row_slots, dtype=torch.int32).cuda()
    xs, da, db = x.cuda(), a.cuda(), b.cuda()
    outs = [y.cuda() for _ in range(3)]
    work = torch.empty(gphq.lora_workspace_bytes(rows, k, R), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for o in outs:
        gphq.lora_add(da, db, xs[:, :k], o[:, :n], rs, work=work, stream=side)
    side.synchronize()
    assert ((outs[0][:, :n].cpu().double() - want).abs() <= tol).all()
    assert torch.equal(outs[0][:, n:].cpu(), y[:, n:])
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("what", ["adapter", "row"])
def test_what_is_not_finite_stays_where_it_is(what):
    """NaN in one adapter reaches its own rows only, NaN in one row's x that row only, in tiles that hold others."""
    rows, k, n, slots, R = 40, 64, 80, 3, 16
    a, b, x, y, scales = make(rows, k, n, slots, R, [R] * 3, torch.float16, 6)
    row_slots = [i % 3 for i in range(rows)]
    if what == "adapter":
        a[1, 3, 5], b[1, 7, 2] = NAN, float("inf")
        mine = [r for r in range(rows) if row_slots[r] == 1]
    else:
        x[17, 9] = NAN
        mine = [17]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    d = y.cuda()
    gphq.lora_add(a.cuda(), b.cuda(), x.cuda(), d, i32(row_slots), None, scales.cuda())
    want, tol = expect(a, b, x, y, row_slots, [R] * 3, scales)
    rest = [r for r in range(rows) if r not in mine]
    assert ((d[rest].cpu().double() - want[rest]).abs() <= tol[rest]).all()
    assert d[mine].isnan().any(1).all()


def test_captured_and_replayed_with_other_adapters():
    rows, k, n, slots, R = 33, 256, 200, 4, 32
    a, b, x, y, scales = make(rows, k, n, slots, R, [R] * 4, torch.bfloat16, 7)
    da, db, dx, sc = a.cuda(), b.cuda(), x.cuda(), scales.cuda()
    rs, d = torch.zeros(rows, dtype=torch.int32, device="cuda"), y.cuda()
    work = torch.empty(gphq.lora_workspace_bytes(rows, k, R), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        gphq.lora_add(da, db, dx, d, rs, None, sc, work=work)
    for i in range(4):
        row_slots = [(r * (i + 1)) % 5 - 1 for r in range(rows)]
        rs.copy_(torch.tensor(row_slots, dtype=torch.int32))
        d.copy_(y.cuda())
        graph.replay()
        torch.cuda.synchronize()
        e = y.cuda()
        gphq.lora_add(da, db, dx, e, rs, None, sc)
        torch.cuda.synchronize()
        assert torch.equal(d, e)
        want, tol = expect(a, b, x, y, row_slots, [R] * 4, scales)
        assert ((d.cpu().double() - want).abs() <= tol).all()


def test_beside_a_projection():
    """gphq_gemv_vec, then the adapters of its lanes: the whole against float64."""
    lanes, k, n, slots, R = 12, 256, 320, 3, 8
    g = torch.Generator().manual_seed(8)
    codes = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    wscale = torch.rand(n, generator=g) * 0.01
    a, b, x, _, scales = make(lanes, k, n, slots, R, [R] * 3, torch.bfloat16, 9)
    row_slots = [(5 * i) % 4 - 1 for i in range(lanes)]
    y = torch.empty(lanes, n, device="cuda")
    work = torch.empty(gphq.gemv_vec_workspace_bytes(lanes, k), dtype=torch.uint8, device="cuda")
    dx = x.cuda()
    gphq.gemv_vec(gphq.FMT_Q8, codes.cuda(), wscale.cuda(), dx, y, lanes, k, n, work)
    gphq.lora_add(a.cuda(), b.cuda(), dx, y, torch.tensor(row_slots, dtype=torch.int32).cuda(), None, scales.cuda())
    base = (x.double() @ codes.double().T) * wscale.double()
    want, tol = expect(a, b, x, base, row_slots, [R] * 3, scales)
    # the projection's own bound: 1e-4 absolute and 1e-5 relative to the serial product
    assert ((y.cpu().double() - want).abs() <= tol + 1e-4 + 1e-5 * base.abs()).all()


def test_wrong_tensors_are_refused():
    a, b, x, y, _ = make(4, 32, 8, 1, 8, [8], torch.float16, 10)
    da, db, dx, dy, rs = a.cuda(), b.cuda(), x.cuda(), y.cuda(), torch.zeros(4, dtype=torch.int32, device="cuda")
    for call in (
        lambda: gphq.lora_add(da, db.float(), dx, dy, rs), lambda: gphq.lora_add(da, db[:, :, :4], dx, dy, rs),
        lambda: gphq.lora_add(da, db, dx.half(), dy, rs), lambda: gphq.lora_add(da, db, dx, dy, rs.long()),
        lambda: gphq.lora_add(da, db, dx, dy, rs[:3]), lambda: gphq.lora_add(da, db, x, dy, rs),
        lambda: gphq.lora_add(da, db, dx, dy[:, :7], rs), lambda: gphq.lora_add(da.double(), db.double(), dx, dy, rs),
    ):
        with pytest.raises(gphq.GphqError):
            call()
