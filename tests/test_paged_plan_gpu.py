"""gphq_paged_plan on the GPU against the definition, one request after another on the host."""
import numpy as np
import pytest
import torch

from gophonic_amd import gphq

pytestmark = pytest.mark.gpu


def planned(held, count, taken, shared, table, free, have, page, rows, max_rows, max_len):
    """The definition. table: lists; free: a list of the list's whole memory, of which `have` are free."""
    table, free, taken = [list(t) for t in table], list(free), list(taken)
    room, bad = len(free), set()
    if have < 0 or have > room:
        bad.add("page")
    have = min(max(have, 0), room)
    ok = [h >= 0 and 0 <= c <= max_rows and 0 <= t <= len(tb) and s >= 0 and h + c <= max_len
          for h, c, t, s, tb in zip(held, count, taken, shared, table)]
    if not all(ok):
        bad.add("seq")
    need = [-(-(h + c) // page) if g else t for h, c, t, g in zip(held, count, taken, ok)]
    for i, t in enumerate(taken):
        keep = max(need[i], min(shared[i], t)) if ok[i] else t
        for e in range(keep, t):
            if have < room:
                free[have] = table[i][e]
                have += 1
            else:
                bad.add("page")
        taken[i] = min(t, keep)
    starts, lens, wanted, asked, used = [0], [], 0, 0, 0
    for i, c in enumerate(count):
        wants = max(0, need[i] - taken[i])
        wanted += wants
        n = c if ok[i] else 0
        if wants and wanted > have:
            bad.add("full")
            n = 0
        else:
            for e in range(wants):
                table[i][taken[i] + e] = free[have - 1 - used]
                used += 1
            taken[i] += wants
        asked += n
        if n and asked > rows:
            bad.add("seq")
            n = 0
        starts.append(starts[-1] + n)
        lens.append(held[i] + n)
    place = [((held[i] + j), i, table[i][(held[i] + j) // page] * page + (held[i] + j) % page)
             for i in range(len(held)) for j in range(starts[i + 1] - starts[i])]
    place += [(-1, -1, -1)] * (rows - len(place))
    return starts, lens, taken, have - used, table, free, place, bad


def ints(a, dtype=torch.int32):
    return torch.tensor(a, dtype=dtype, device="cuda")


def check(held, count, taken, shared, table, free, have, page, rows, max_rows, max_len, alias=False, maps=True):
    seqs = len(held)
    want = planned(held, count, taken, shared or [0] * seqs, table, free, have, page, rows, max_rows, max_len)
    h, t, fc = ints(held), ints(taken), ints([have])
    tab = ints(table).view(seqs, -1)
    more = dict(lens=h, taken_out=t, free_count_out=fc) if alias else {}
    if not maps:
        more.update(positions=False, sequences=False, slots=False)
    p = gphq.PagedPlan(h, ints(count), t, tab, ints(free), fc, page, rows, max_rows, max_len,
                       shared=ints(shared) if shared else None, **more)
    p.run()
    starts, lens, taken_out, left, wtable, wfree, place, bad = want
    assert p.starts.tolist() == starts
    assert p.lens.tolist() == lens
    assert p.taken_out.tolist() == taken_out
    assert p.free_count_out.tolist() == [left]
    assert p.table.tolist() == wtable
    assert p.free.tolist() == wfree
    if maps:
        assert list(zip(p.positions.tolist(), p.sequences.tolist(), p.slots.tolist())) == place
    status = (gphq.ERR_PAGED_BATCH if bad & {"seq", "page"} else gphq.ERR_PREFIX_FULL if bad else gphq.OK)
    if status == gphq.OK:
        p.batch.check()
    else:
        with pytest.raises(gphq.GphqError) as e:
            p.batch.check()
        assert e.value.status == status
        p.batch.check()  # cleared
    return p


def batch(seed, seqs, page, new_hi, old_hi, back=0, spare=9, share=True):
    """A random batch whose pages come from one shuffled list."""
    r = np.random.default_rng(seed)
    count = [int(c) for c in r.integers(0, new_hi + 1, seqs)]
    held = [int(h) for h in r.integers(0, old_hi + 1, seqs)]
    taken = [-(-(h + int(r.integers(0, back + 1))) // page) for h in held]
    for i in np.nonzero(r.random(seqs) < 0.1)[0]:
        held[i] = count[i] = 0
    shared = [int(r.integers(0, 3)) if share and r.random() < 0.3 else 0 for _ in held]
    max_len = max(h + c for h, c in zip(held, count))
    stride = max(max(taken), -(-max_len // page)) + 1
    wants = sum(max(0, -(-(h + c) // page) - t) for h, c, t in zip(held, count, taken))
    pages = sum(taken) + wants + spare
    order = [int(x) for x in r.permutation(pages)]
    table, at = [], 0
    for t in taken:
        table.append(order[at:at + t] + [-1] * (stride - t))
        at += t
    free = order[at:] + [-5] * at
    return dict(held=held, count=count, taken=taken, shared=shared, table=table, free=free, have=pages - at, page=page,
                rows=sum(count) + 3, max_rows=max(count), max_len=max_len)


@pytest.mark.parametrize("alias", [False, True], ids=["apart", "in place"])
@pytest.mark.parametrize("seqs,page,new_hi,old_hi,back", [
    (1, 16, 1, 0, 0), (1, 16, 1, 15, 0), (1, 16, 40, 100, 0), (3, 64, 5, 200, 40), (64, 16, 1, 500, 20),
    (65, 16, 1, 300, 0), (200, 16, 30, 300, 60), (1000, 32, 9, 400, 12), (1024, 16, 1, 100, 0), (1025, 16, 3, 100, 40),
    (3000, 16, 2, 60, 33), (5, 4096, 3, 9000, 0), (70, 16, 0, 100, 50),
])
def test_plans(seqs, page, new_hi, old_hi, back, alias):
    check(**batch(seqs + page, seqs, page, new_hi, old_hi, back), alias=alias)


@pytest.mark.parametrize("have", [0, 1, 2, 3, 4, 5, 6, 7, 40, -1, 41])
def test_a_list_that_runs_short(have):
    """Served in order while the pages last: one that does not fit brings nothing, nor does any that wants pages behind
    it; one that wants none does. What is given back in the same step can be taken."""
    d = dict(held=[16, 0, 5, 31, 16, 0], count=[20, 1, 3, 1, 1, 17], taken=[1, 0, 1, 2, 3, 1], shared=None,
             table=[[i * 6 + e for e in range(6)] for i in range(6)], free=list(range(100, 140)), have=have, page=16,
             rows=60, max_rows=20, max_len=64)
    check(**d)
    check(**{**d, "count": [64 - 16, 1, 3, 1, 1, 17], "max_rows": 64})


def test_rows_and_lists_without_room():
    """A sequence whose rows pass the rows brings none; a page for which the list has no room is dropped."""
    d = batch(5, 40, 16, 10, 100, 40)
    for rows in (0, 1, 7, 20, sum(d["count"]) - 1):
        check(**{**d, "rows": rows})
    free = d["free"][:d["have"] + 3]
    check(**{**d, "free": free})
    check(**{**d, "free": [], "have": 0})


@pytest.mark.parametrize("name,value", [("held", -1), ("held", 2 ** 31 - 1), ("count", -1), ("count", 100), ("taken", -1),
                                        ("taken", 100), ("shared", -1), ("count", 2 ** 31 - 1), ("held", -2 ** 31)])
def test_bad_numbers_are_left_alone(name, value):
    d = batch(6, 20, 16, 10, 100, 20)
    for at in (0, 7, 19):
        v = list(d[name])
        v[at] = value
        check(**{**d, name: v})


def test_without_maps_and_without_requests():
    check(**batch(7, 30, 16, 8, 100), maps=False)
    p = gphq.PagedPlan(ints([]), ints([]), ints([]), ints([]).view(0, 4), ints([1, 2]), ints([2]), 16, 3, 1, 64)
    p.run()
    assert p.starts.tolist() == [0] and p.free_count_out.tolist() == [2]
    assert p.positions.tolist() == [-1] * 3 and p.slots.tolist() == [-1] * 3
    p.batch.check()


def test_slots_past_32_bits():
    n = 2 ** 31 - 2
    check([10], [10], [1], None, [[n, -1]], [n - 1, 7], 1, 4096, 12, 10, 4096 * 2)
    p = check([4090], [10], [1], None, [[n, -1]], [n - 1, 7], 1, 4096, 12, 10, 4096 * 2)
    assert int(p.slots.max()) > 2 ** 42


def test_large_batches():
    """One prompt of many thousand rows between single tokens; as many sequences as a call takes, most of them idle."""
    d = batch(8, 70, 16, 1, 300)
    d["count"][33], d["held"][33] = 30000, 0
    d["max_rows"], d["max_len"] = 30000, 30000
    stride = -(-30000 // 16) + 1
    d["table"] = [t + [-1] * (stride - len(t)) for t in d["table"]]
    d["free"] = d["free"] + list(range(10 ** 6, 10 ** 6 + 2000))
    d["free"] = d["free"][:d["have"]] + list(range(10 ** 6, 10 ** 6 + 3000))
    d["have"] += 2500
    d["rows"] = sum(d["count"]) + 70
    check(**d)
    seqs = 65536
    held, count, taken = [0] * seqs, [0] * seqs, [0] * seqs
    for i, (h, c) in {0: (3, 2), 40000: (15, 3), 65535: (0, 1)}.items():
        held[i], count[i], taken[i] = h, c, -(-h // 16)
    check(held, count, taken, None, [[i, -1] for i in range(seqs)], list(range(10 ** 6, 10 ** 6 + 9)), 9, 16, 8, 4, 32)


def test_captured_plans_follow_the_requests():
    """A captured plan in place, replayed: each step from what the last one left, with requests that come, grow, take
    drafts back and end in between; against the definition step by step."""
    page, seqs, stride, pages, rows = 16, 6, 8, 60, 40
    r = np.random.default_rng(9)
    held, count, taken = (torch.zeros(seqs, dtype=torch.int32, device="cuda") for _ in range(3))
    table = torch.full((seqs, stride), -1, dtype=torch.int32, device="cuda")
    free, have = ints([int(x) for x in r.permutation(pages)]), ints([pages])
    p = gphq.PagedPlan(held, count, taken, table, free, have, page, rows, 20, 120, lens=held, taken_out=taken,
                       free_count_out=have)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            p.run()
    torch.cuda.synchronize()
    for step in range(25):
        h = held.tolist()
        for s in range(seqs):
            h[s] = 0 if h[s] > 90 else max(0, h[s] - int(r.integers(0, 4)))  # drafts taken back, requests that end
        c = [int(x) for x in r.integers(0, 7, seqs)]
        want = planned(h, c, taken.tolist(), [0] * seqs, table.tolist(), free.tolist(), int(have), page, rows, 20, 120)
        held.copy_(ints(h))
        count.copy_(ints(c))
        graph.replay()
        torch.cuda.synchronize()
        assert p.starts.tolist() == want[0] and held.tolist() == want[1] and taken.tolist() == want[2]
        assert int(have) == want[3] and table.tolist() == want[4] and free.tolist() == want[5]
        assert list(zip(p.positions.tolist(), p.sequences.tolist(), p.slots.tolist())) == want[6]
        p.batch.check()
        # No page is lost or held twice.
        mine = [x for t, n in zip(table.tolist(), taken.tolist()) for x in t[:n]] + free.tolist()[:int(have)]
        assert sorted(mine) == list(range(pages))


def test_on_another_stream():
    d = batch(10, 100, 16, 4, 200, 30)
    want = planned(*[d[k] for k in ("held", "count", "taken", "shared", "table", "free", "have", "page", "rows",
                                    "max_rows", "max_len")])
    p = gphq.PagedPlan(ints(d["held"]), ints(d["count"]), ints(d["taken"]), ints(d["table"]), ints(d["free"]),
                       ints([d["have"]]), 16, d["rows"], d["max_rows"], d["max_len"], shared=ints(d["shared"]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    p.run(stream=side)
    side.synchronize()
    assert p.starts.tolist() == want[0] and p.table.tolist() == want[4]
