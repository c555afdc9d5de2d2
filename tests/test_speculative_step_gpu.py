"""The operators of a speculative step together, as a server runs them: requests' pages planned on the device, their
rows appended to and attended over 8-bit pages, logits made probabilities, drafts verified, and the accepted lengths
fed to the next plan; nothing of it is read back between the calls."""
import numpy as np
import pytest
import torch

from gophonic_amd import gphq
from tests.paged8_common import BLOCK, E4M3, I8, values
from tests.paged_common import F32

pytestmark = pytest.mark.gpu

SEQS, DRAFTS, HEADS, G, D, PAGE, VOCAB, STEPS = 5, 3, 4, 2, 64, 16, 97, 12
ROWS, MAX_LEN, PAGES = SEQS * (DRAFTS + 1), 200, 64


class Server:
    """A model of one attention layer: token t at position p has the fused row table[t], its logits are out . head."""

    def __init__(self, kind, seed):
        g = torch.Generator().manual_seed(seed)
        up = lambda *s: torch.randn(*s, generator=g).cuda()
        self.table, self.head = up(VOCAB, (HEADS + 2 * G) * D), up(HEADS * D, VOCAB) * 0.4
        self.noise = up(VOCAB, VOCAB)  # what the proposer gets wrong
        a = torch.arange(MAX_LEN, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(D // 2, dtype=torch.float64) * 2 / D)
        self.cos, self.sin = a.cos().float().cuda(), a.sin().float().cuda()
        self.kn = (1 + 0.1 * torch.randn(D, generator=g)).cuda()
        codes = lambda: torch.zeros(PAGES, G, PAGE, D, dtype=torch.uint8, device="cuda").view(kind).transpose(1, 2)
        scales = lambda: torch.full((PAGES, G, PAGE // BLOCK), float("nan"), device="cuda")
        self.kv, self.kind = gphq.PagedKv8(codes(), codes(), scales(), scales()), kind
        i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
        self.held, self.count, self.taken = i(SEQS), i(SEQS), i(SEQS)
        self.pages = torch.full((SEQS, -(-MAX_LEN // PAGE) + 1), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(PAGES, generator=g).int().cuda()
        self.have = torch.tensor([PAGES], dtype=torch.int32, device="cuda")
        self.plan = gphq.PagedPlan(self.held, self.count, self.taken, self.pages, self.free, self.have, PAGE, ROWS,
                                   DRAFTS + 1, MAX_LEN, taken_out=self.taken, free_count_out=self.have)
        f = lambda *s: torch.zeros(*s, device="cuda")
        self.tokens, self.out_tokens, self.accepted = i(ROWS), i(ROWS), i(SEQS)
        self.q, self.out, self.logits, self.probs, self.draft = f(ROWS, HEADS * D), f(ROWS, HEADS * D), f(ROWS, VOCAB), \
            f(ROWS, VOCAB), f(ROWS, VOCAB)
        self.accept_u, self.sample_u = f(ROWS), f(SEQS)
        self.temperatures = torch.ones(ROWS, device="cuda")
        self.drafts = i(ROWS)
        byte = lambda n: torch.zeros(max(16, n), dtype=torch.uint8, device="cuda")
        self.work = [byte(gphq.paged8_attention_workspace_bytes(self.kv, self.plan.batch, F32, HEADS)),
                     byte(gphq.probabilities_workspace_bytes(ROWS, VOCAB)),
                     byte(gphq.verify_drafts_workspace_bytes(SEQS, VOCAB))]

    def step(self):
        """Row r of sequence s holds its last token or a draft; the drafts that row r's logits answer are the next rows'."""
        self.plan.run()
        qkv = self.table.index_select(0, self.tokens)
        gphq.paged8_append(self.kv, self.plan.batch, qkv, self.q, HEADS, None, self.kn, 1e-6, self.cos, self.sin, D ** -0.5)
        gphq.paged8_attention(self.kv, self.plan.batch, self.q, self.out, HEADS, 1.0, work=self.work[0])
        torch.mm(self.out, self.head, out=self.logits)
        gphq.probabilities(self.logits, self.probs, self.temperatures, work=self.work[1])
        gphq.verify_drafts(self.plan.starts, self.drafts, self.probs, self.draft, self.accept_u, self.sample_u,
                           self.out_tokens, self.accepted, lens=self.plan.lens, kept=self.held, work=self.work[2])


def propose(sv, r, tokens, last):
    """Host side of a proposer: DRAFTS tokens for each request (fewer for some), their probabilities, random numbers."""
    starts = [0]
    rows, drafts, probs = [], [], []
    for s in range(SEQS):
        n = int(r.integers(0, DRAFTS + 1))
        seq = [last[s]]
        for i in range(n):
            p = torch.softmax(sv.noise[seq[-1]].cpu(), 0).numpy().astype(np.float64)
            seq.append(int(r.choice(VOCAB, p=p / p.sum())))
            probs.append(p)
        probs.append(np.zeros(VOCAB))
        rows += seq
        drafts += seq[1:] + [0]
        starts.append(len(rows))
    pad = ROWS - len(rows)
    return starts, rows + [0] * pad, drafts + [0] * pad, np.concatenate([np.stack(probs), np.zeros((pad, VOCAB))])


@pytest.mark.parametrize("kind", [I8, E4M3], ids=["i8", "e4m3"])
def test_steps(kind):
    sv, r = Server(kind, 3), np.random.default_rng(4)
    last = [int(x) for x in r.integers(0, VOCAB, SEQS)]
    text = [[] for _ in range(SEQS)]
    for step in range(STEPS):
        if step == 7:  # a request ends and another takes its place
            sv.held[2] = 0
            text[2] = []
        starts, rows, drafts, draft = propose(sv, r, text, last)
        sv.count.copy_(torch.tensor(np.diff(starts), dtype=torch.int32))
        sv.tokens.copy_(torch.tensor(rows, dtype=torch.int32))
        sv.drafts.copy_(torch.tensor(drafts, dtype=torch.int32))
        sv.draft.copy_(torch.from_numpy(draft))
        sv.accept_u.copy_(torch.from_numpy(r.random(ROWS, np.float32)))
        sv.sample_u.copy_(torch.from_numpy(r.random(SEQS, np.float32)))
        sv.step()
        sv.plan.batch.check()
        assert sv.plan.starts.tolist() == starts
        held, lens, accepted, out = sv.held.tolist(), sv.plan.lens.tolist(), sv.accepted.tolist(), sv.out_tokens.tolist()
        for s in range(SEQS):
            a, n = starts[s], starts[s + 1] - starts[s]
            assert 0 <= accepted[s] < n and lens[s] == len(text[s]) + n and held[s] == len(text[s]) + accepted[s] + 1
            assert out[a:a + accepted[s]] == drafts[a:a + accepted[s]] and 0 <= out[a + accepted[s]] < VOCAB
            assert out[a + accepted[s] + 1:a + n] == [-1] * (n - accepted[s] - 1)
            # Attention of the step's rows over what the pages hold, in float64.
            attend(sv, s, lens[s], a, n)
            text[s] += rows[a:a + accepted[s] + 1]
            last[s] = out[a + accepted[s]]
        # The pages hold the text: every kept token's value is its row's, within its code's rounding.
        for s in range(SEQS):
            stored(sv, s, text[s], kind)
        mine = [x for t, n in zip(sv.pages.tolist(), sv.taken.tolist()) for x in t[:n]]
        mine += sv.free.tolist()[:int(sv.have)]
        assert sorted(mine) == list(range(PAGES))


def places(sv, s, n):
    table = sv.pages[s].tolist()
    return [(table[p // PAGE], p % PAGE) for p in range(n)]


def held(sv, s, n, i):
    """float64 [n][G][D] of the keys (0) or values (1) that the pages hold for a sequence, and the scales of each."""
    c, sc = ((sv.kv.k, sv.kv.k_scales), (sv.kv.v, sv.kv.v_scales))[i]
    at = places(sv, s, n)
    pg, sl = torch.tensor([a for a, _ in at]).cuda(), torch.tensor([b for _, b in at]).cuda()
    scale = sc[pg, :, sl // BLOCK].double()[..., None]
    return values(c.view(torch.uint8)[pg, sl].cpu(), sv.kind).cuda() * scale, scale


def stored(sv, s, text, kind):
    """int8: within one step of the scale, whatever it has grown by; e4m3: half a step of the value or of the smallest."""
    if not text:
        return
    want = sv.table[torch.tensor(text).cuda()].double().view(-1, HEADS + 2 * G, D)[:, HEADS + G:]
    got, scale = held(sv, s, len(text), 1)
    room = scale * (1 + 1e-6) if kind == I8 else 2.0 ** -4 * (1 + 1e-6) * want.abs() + 2.0 ** -9 * scale
    assert ((got - want).abs() <= room).all()


def attend(sv, s, n, row, rows):
    k, _ = held(sv, s, n, 0)
    v, _ = held(sv, s, n, 1)
    for i in range(rows):
        p = n - rows + i
        q = sv.q[row + i].double().view(G, HEADS // G, D)
        w = torch.softmax(torch.einsum("ghd,kgd->ghk", q.cpu(), k[:p + 1].cpu()), 2)
        want = torch.einsum("ghk,kgd->ghd", w, v[:p + 1].cpu())
        mag = torch.einsum("ghk,kgd->ghd", w, v[:p + 1].cpu().abs())
        got = sv.out[row + i].double().view(G, HEADS // G, D).cpu()
        # Scores to (hd + 8) 2^-24 of their terms' magnitudes, which change the quotient by twice that; sums of n.
        e = float((q.cpu().abs()[..., None, :] * k[:p + 1].cpu().abs().permute(1, 0, 2)[:, None]).sum(-1).max())
        assert ((got - want).abs() <= (2.5 * (D + 16) * 2.0 ** -24 * e + (2 * n + 64) * 2.0 ** -24) * mag + 1e-7 * mag.max()).all()


def test_a_captured_step():
    """The same steps from a graph, replayed with the host's inputs copied in between: every replay gives what an eager
    server gives."""
    a, b = Server(I8, 5), Server(I8, 5)
    r = np.random.default_rng(6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        a.step()  # (the library's products make their handles; no request has a row)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            a.step()
    torch.cuda.synchronize()
    b.step()
    last = [int(x) for x in r.integers(0, VOCAB, SEQS)]
    for step in range(8):
        starts, rows, drafts, draft = propose(a, r, None, last)
        u, v = r.random(ROWS, np.float32), r.random(SEQS, np.float32)
        for sv in (a, b):
            sv.count.copy_(torch.tensor(np.diff(starts), dtype=torch.int32))
            sv.tokens.copy_(torch.tensor(rows, dtype=torch.int32))
            sv.drafts.copy_(torch.tensor(drafts, dtype=torch.int32))
            sv.draft.copy_(torch.from_numpy(draft))
            sv.accept_u.copy_(torch.from_numpy(u))
            sv.sample_u.copy_(torch.from_numpy(v))
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        for x, y in ((a.held, b.held), (a.out_tokens, b.out_tokens), (a.accepted, b.accepted), (a.pages, b.pages),
                     (a.taken, b.taken), (a.have, b.have), (a.plan.slots, b.plan.slots)):
            assert torch.equal(x, y)
        n = starts[-1]
        assert torch.equal(a.out[:n], b.out[:n]) and torch.equal(a.probs[:n], b.probs[:n])
        acc, out = a.accepted.tolist(), a.out_tokens.tolist()
        last = [out[starts[s] + acc[s]] for s in range(SEQS)]
