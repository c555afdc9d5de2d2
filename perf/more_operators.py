"""One speculative step of many requests over a paged cache held in 8 bits: its operators, measured.

One case is a dict of plain values; `kind` names the operator:

  plan    pages handed out and given back, page tables, row starts and the slot
          of every new token, from the requests' lengths (gphq.PagedPlan.run)
  append  a batch's fused QKV rows: head RMSNorm and rotary position, queries
          written out, keys and values stored as 8-bit codes with a scale for
          every 16 tokens and KV head (gphq.paged8_append)
  attend  causal attention of the batch's new tokens over such pages
          (gphq.paged8_attention)
  probs   logits to probabilities at a temperature of each row's own
          (gphq.probabilities)
  verify  drafted tokens accepted or replaced by the target's probabilities,
          from given random numbers (gphq.verify_drafts)

A batch is `seqs` sequences; sequence s brings new[s] tokens to old[s] that the
cache holds already. `lay` numbers the draw of those lengths, so a case alone
fixes its work; everything else is made from the seed. With `own` false the
operators run in their plain form: elementary torch operations in float32,
rounded once at the end; in float64 what decides a code or a token.
"""
import math
import random

import torch

own = False

POSITIONS = 40960  # the rotary table's rows: the context of the measured model shapes
VOCAB = 151936  # and their vocabulary
THETA, EPS = 1e6, 1e-6
BLOCK = 16  # tokens that share a scale
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CODES = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"i8": 127.0, "e4m3": 448.0}  # the largest code
OVER = {"i8": 127.5, "e4m3": 464.0}  # what still rounds to it


def listed():
    qwen8 = dict(heads=32, kv_heads=8, hd=128)
    small = dict(heads=16, kv_heads=8, hd=128)
    return [
        # 32 requests' next tokens: one page in two or so is new. All latency.
        dict(name="plan_lanes32", kind="plan", page=16, seqs=32, new=1, new_hi=1, old=100, old_hi=4000, back=0, lay=1),
        # A continuous batch of a thousand requests: prompt chunks, single tokens, drafts taken back, requests that end.
        dict(name="plan_batch1000", kind="plan", page=16, seqs=1000, new=1, new_hi=64, old=0, old_hi=2000, back=12,
             lay=2),
        # 64 requests, one token each, in the middle of their answers.
        dict(name="append8_lanes64", kind="append", **qwen8, rows="f32", codes="i8", page=64, order="head", seqs=64,
             new=1, new_hi=1, old=100, old_hi=4000, lay=3),
        # Prompt chunks of five requests in one pass.
        dict(name="append8_chunks", kind="append", **qwen8, rows="f32", codes="i8", page=64, order="head", seqs=5,
             new=300, new_hi=1300, old=0, old_hi=2000, lay=4),
        # One token of one request over a short cache: latency of the attention step.
        dict(name="attend8_token", kind="attend", **small, rows="f32", codes="i8", page=16, order="head", seqs=1, new=1,
             new_hi=1, old=1023, old_hi=1023, window=0, lay=5),
        # Two long documents being answered, four drafted tokens beside each: the cache's whole length, small pages.
        dict(name="attend8_long", kind="attend", **qwen8, rows="bf16", codes="i8", page=16, order="head", seqs=2, new=5,
             new_hi=5, old=32000, old_hi=40900, window=0, lay=6),
        # A follow-up message of 512 tokens over a long conversation, floating-point codes.
        dict(name="attend8_chunk", kind="attend", **qwen8, rows="f16", codes="e4m3", page=64, order="head", seqs=1,
             new=512, new_hi=512, old=16000, old_hi=16000, window=0, lay=7),
        # A continuous batch: prompt chunks of odd lengths and single tokens side by side, token-major pages.
        dict(name="attend8_mixed", kind="attend", **qwen8, rows="f32", codes="i8", page=32, order="token", seqs=12,
             new=1, new_hi=300, old=0, old_hi=4000, window=0, lay=8),
        # One request's logits: latency.
        dict(name="probs_row", kind="probs", rows=1, vocab=VOCAB, pad=0),
        # 32 requests' logits for the last token and four drafts each.
        dict(name="probs_drafts160", kind="probs", rows=160, vocab=VOCAB, pad=0),
        # One token sampled for one request, nothing drafted: latency.
        dict(name="verify_sample", kind="verify", seqs=1, new=0, new_hi=0, vocab=VOCAB, draft="none", lay=9),
        # 64 requests with one to five drafts of a model whose probabilities are kept.
        dict(name="verify_lanes64", kind="verify", seqs=64, new=1, new_hi=5, vocab=VOCAB, draft="probs", lay=10),
    ]


def draw(rng):
    def log(lo, hi, step=1):
        return max(1, round(lo * (hi / lo) ** rng.random() / step)) * step

    kind = rng.choice(["plan", "append", "attend", "attend", "probs", "verify"])
    lay = rng.randrange(1 << 20)
    if kind == "plan":
        return dict(kind=kind, page=rng.choice([16, 32, 64, 128]), seqs=log(1, 1000), new=rng.choice([0, 1]),
                    new_hi=rng.choice([1, log(2, 64)]), old=0, old_hi=log(16, 2000), back=rng.choice([0, 12]), lay=lay)
    if kind == "probs":
        return dict(kind=kind, rows=log(1, 160), vocab=log(500, VOCAB), pad=rng.choice([0, 0, 1, 7, 64]))
    if kind == "verify":
        return dict(kind=kind, seqs=log(1, 64), new=0, new_hi=rng.randint(0, 5), vocab=log(500, VOCAB),
                    draft=rng.choice(["probs", "probs", "none"]), lay=lay)
    kv_heads = rng.choice([1, 2, 4, 8])
    shape = rng.choice(["tokens", "chunks", "mixed"])
    c = dict(kind=kind, heads=kv_heads * rng.choice([1, 2, 4, 5, 8] if shape == "tokens" else [1, 2, 4, 5]),
             kv_heads=kv_heads, hd=rng.choice([64, 128, 128]), rows=rng.choice(["f32", "f16", "bf16"]),
             codes=rng.choice(["i8", "e4m3"]), page=rng.choice([16, 32, 64, 128]), order=rng.choice(["head", "token"]))
    window = dict(window=rng.choice([0, 0, log(100, 4000)])) if kind == "attend" else {}
    if shape == "tokens":
        seqs = log(1, 32)
        lo = rng.randint(1, 6)  # single tokens, or with a few drafts beside them
        return dict(c, seqs=seqs, new=lo, new_hi=lo, old=0, old_hi=log(16, 32768 // seqs if seqs > 1 else 40000),
                    **window, lay=lay)
    seqs = rng.randint(1, 3) if shape == "chunks" else rng.randint(3, 10)
    lo = log(2, 200) if shape == "chunks" else 1
    return dict(c, seqs=seqs, new=lo, new_hi=max(lo, log(lo + 1, 600 if shape == "chunks" else 200)), old=0,
                old_hi=log(16, 3000), **window, lay=lay)


# ---- lengths and work ---------------------------------------------------------


def _lengths(c):
    """(new tokens, tokens before them) of every sequence; where single tokens are allowed, half bring the fewest."""
    r = random.Random(c["lay"])
    new = [c["new"] if c["new"] <= 1 and r.random() < 0.5 else r.randint(c["new"], c["new_hi"])
           for _ in range(c["seqs"])]
    if c["seqs"] == 1:
        new = [c["new_hi"]]
    return new, [r.randint(c["old"], c["old_hi"]) for _ in new] if "old" in c else None


def _requests(c):
    """(held, new, pages taken, pages shared) of every request of a plan: some take drafts back, some end."""
    r = random.Random(c["lay"] + 1)
    new, old = _lengths(c)
    held, taken, shared = [], [], []
    for i, o in enumerate(old):
        had = o + (r.randint(0, c["back"]) if r.random() < 0.5 else 0)
        taken.append(-(-had // c["page"]))
        shared.append(min(r.randint(0, 3), taken[-1]) if r.random() < 0.25 else 0)
        if c["back"] and r.random() < 0.05:
            o, new[i] = 0, 0
        held.append(o)
    return held, new, taken, shared


def work(case):
    c = case
    if c["kind"] == "plan":
        held, new, taken, _ = _requests(c)
        moved = sum(abs(-(-(h + n) // c["page"]) - t) for h, n, t in zip(held, new, taken))
        return {"bytes": 28 * c["seqs"] + 8 * moved + 16 * sum(new), "flops": 0}
    if c["kind"] == "probs":
        return {"bytes": 8 * c["rows"] * c["vocab"], "flops": 4 * c["rows"] * c["vocab"]}
    if c["kind"] == "verify":
        sides = 2 if c["draft"] == "probs" else 1
        return {"bytes": 4 * sides * c["seqs"] * c["vocab"], "flops": 3 * c["seqs"] * c["vocab"]}
    new, old = _lengths(c)
    rows = sum(new)
    rb, q, kv = SIZE[c["rows"]], c["heads"] * c["hd"], c["kv_heads"] * c["hd"]
    if c["kind"] == "append":
        return {"bytes": rows * ((2 * q + 2 * kv) * rb + 2 * kv + 4 * c["hd"]), "flops": rows * (q + 2 * kv) * 8}
    read = pairs = 0
    for n, o in zip(new, old):
        w = c["window"] or o + n
        read += o + n - max(0, o + 1 - w)
        pairs += sum(min(o + i + 1, w) for i in range(n))
    return {"bytes": 2 * rows * q * rb + 2 * read * (kv + 4 * c["kv_heads"] // BLOCK), "flops": 4 * pairs * q}


# ---- inputs -------------------------------------------------------------------


def _randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _rand(g, *shape):
    return torch.rand(shape, device="cuda", generator=g)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _rope_tables(hd):
    """cos and sin [positions][hd / 2], the angles in float64."""
    inv = THETA ** (-torch.arange(0, hd // 2, dtype=torch.float64, device="cuda") * 2 / hd)
    a = torch.arange(POSITIONS, dtype=torch.float64, device="cuda")[:, None] * inv
    return a.cos().float(), a.sin().float()


def _pool(g, c, pages):
    """Codes of keys and values [2][pages][page tokens][KV heads][head dim], their memory in token or head order, and
    scales [2][pages][KV heads][blocks]: what earlier requests left there, quantized as they were stored."""
    G, D, T = c["kv_heads"], c["hd"], c["page"]
    codes = torch.empty(2, pages, G, T, D, dtype=torch.uint8, device="cuda")
    scales = torch.empty(2, pages, G, T // BLOCK, device="cuda")
    for i in (0, 1):
        for p in range(0, pages, 512):
            x = _randn(g, *codes[i, p:p + 512].shape) * (1.0, 0.7)[i] + (0.0, 0.1)[i]
            x = (x + x[:, :, :1] * 0.5).view(-1, G, T // BLOCK, BLOCK, D)  # keys of a page that are somewhat alike
            scale = x.abs().amax((-1, -2)) / TOP[c["codes"]]
            x = (x / scale[..., None, None]).view(-1, G, T, D)
            x = x.round().to(torch.int8) if c["codes"] == "i8" else x.clamp(-448, 448).to(CODES["e4m3"])
            codes[i, p:p + 512], scales[i, p:p + 512] = x.view(torch.uint8), scale
    if c["order"] == "token":
        codes = codes.transpose(2, 3).contiguous()
    else:
        codes = codes.transpose(2, 3)
    return codes.view(CODES[c["codes"]]), scales


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(1_000_003 * seed + 31)
    if c["kind"] == "plan":
        return _prepare_plan(c, g)
    if c["kind"] == "probs":
        return _prepare_probs(c, g)
    if c["kind"] == "verify":
        return _prepare_verify(c, g)
    new, old = _lengths(c)
    rows, lens = sum(new), [o + n for o, n in zip(old, new)]
    s = dict(case=c, rows=rows, max_rows=max(new), max_len=max(lens))
    need = [-(-n // c["page"]) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((c["seqs"], max(need) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):  # pages as a free list hands them out; the table's rest is unset
        table[i, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s.update(starts=_ints(starts), lens=_ints(lens), table=table)
    s["codes"], s["scales"] = _pool(g, c, pages)
    rdt, H, G, D = TYPES[c["rows"]], c["heads"], c["kv_heads"], c["hd"]
    if c["kind"] == "append":
        s["qkv"] = (_randn(g, rows, (H + 2 * G) * D) * 3).to(rdt)
        s["q"] = torch.empty((rows, H * D), dtype=rdt, device="cuda")
        s["q_norm"], s["k_norm"] = 1 + 0.1 * _randn(g, D), 1 + 0.1 * _randn(g, D)
        s["cos"], s["sin"] = _rope_tables(D)
    else:
        s["q"] = (_randn(g, rows, H * D) * 1.5).to(rdt)
        s["out"] = torch.empty((rows, H * D), dtype=rdt, device="cuda")
    if own:
        from gophonic_amd import gphq

        s["kv"] = gphq.PagedKv8(s["codes"][0], s["codes"][1], s["scales"][0], s["scales"][1])
        s["batch"] = gphq.PagedBatch(s["starts"], s["lens"], s["table"], rows, s["max_rows"], s["max_len"])
        if c["kind"] == "attend":
            s["work"] = torch.empty(gphq.paged8_attention_workspace_bytes(s["kv"], s["batch"], s["q"].dtype, H,
                                                                          c["window"]),
                                    dtype=torch.uint8, device="cuda")
    return s


def _prepare_plan(c, g):
    held, new, taken, shared = _requests(c)
    page = c["page"]
    s = dict(case=c, held=_ints(held), new=_ints(new), taken=_ints(taken), shared=_ints(shared))
    s["rows"], s["max_rows"] = sum(new) + 5, max(new)  # room for a few rows more than the step brings
    s["max_len"] = max(h + n for h, n in zip(held, new))
    stride = max(max(taken), -(-s["max_len"] // page)) + 1
    wants = sum(max(0, -(-(h + n) // page) - t) for h, n, t in zip(held, new, taken))
    pages = sum(taken) + wants + 9
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    s["table"] = torch.full((c["seqs"], stride), -1, dtype=torch.int32, device="cuda")
    live = torch.arange(stride, device="cuda") < s["taken"][:, None]
    s["table"][live] = order[:sum(taken)]
    s["free"] = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    s["free"][:pages - sum(taken)] = order[sum(taken):]
    s["free_count"] = _ints([pages - sum(taken)])
    for name, n in (("starts", c["seqs"] + 1), ("lens", c["seqs"]), ("taken_out", c["seqs"]), ("free_count_out", 1),
                    ("positions", s["rows"]), ("sequences", s["rows"])):
        s[name] = torch.zeros(n, dtype=torch.int32, device="cuda")
    s["slots"] = torch.zeros(s["rows"], dtype=torch.int64, device="cuda")
    if own:
        from gophonic_amd import gphq

        s["plan"] = gphq.PagedPlan(s["held"], s["new"], s["taken"], s["table"], s["free"], s["free_count"], page,
                                   s["rows"], s["max_rows"], s["max_len"], shared=s["shared"], starts=s["starts"],
                                   lens=s["lens"], taken_out=s["taken_out"], free_count_out=s["free_count_out"],
                                   positions=s["positions"], sequences=s["sequences"], slots=s["slots"])
    return s


def _logits(g, rows, vocab):
    """Logits as a head gives them: some tokens are far likelier than the rest."""
    x = _randn(g, rows, vocab) * 2
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 40), device="cuda", generator=g), 6 + 2 * _randn(g, rows, 40))
    return x


def _prepare_probs(c, g):
    R, V = c["rows"], c["vocab"]
    s = dict(case=c, logits=torch.full((R, V + c["pad"]), 100.0, device="cuda"))
    s["logits"][:, :V] = _logits(g, R, V)
    s["temperatures"] = 0.3 + 1.2 * _rand(g, R)
    s["temperatures"][_rand(g, R) < 0.2] = 0.0  # requests that ask for the likeliest token
    s["probs"] = torch.zeros(R, V, device="cuda")
    if own:
        from gophonic_amd import gphq

        s["work"] = torch.empty(gphq.probabilities_workspace_bytes(R, V), dtype=torch.uint8, device="cuda")
    return s


def _prepare_verify(c, g):
    new, _ = _lengths(c)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n + 1)
    R, V = starts[-1], c["vocab"]
    x = _logits(g, R, V)
    s = dict(case=c, rows=R, starts=_ints(starts), target=torch.softmax(x, 1), draft=None)
    if c["draft"] == "probs":  # a smaller model's probabilities, near the target's
        s["draft"] = torch.softmax(x.add_(_randn(g, R, V)), 1)
        del x
    s["drafts"] = torch.multinomial(s["draft"] if s["draft"] is not None else s["target"], 1,
                                    generator=g).flatten().int()
    s["accept_u"], s["sample_u"] = _rand(g, R), _rand(g, c["seqs"])
    s["lens"] = torch.randint(10, 4000, (c["seqs"],), device="cuda", generator=g).int()
    s["tokens"] = torch.zeros(R, dtype=torch.int32, device="cuda")
    s["accepted"], s["kept"] = (torch.zeros(c["seqs"], dtype=torch.int32, device="cuda") for _ in range(2))
    if own:
        from gophonic_amd import gphq

        s["work"] = torch.empty(gphq.verify_drafts_workspace_bytes(c["seqs"], V), dtype=torch.uint8, device="cuda")
    return s


# ---- plain forms --------------------------------------------------------------


def _places(s):
    """Of every row: its sequence, its position, and the (page, slot) its token takes."""
    c = s["case"]
    r = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"], r, right=True) - 1
    pos = (s["lens"][seq] - s["starts"][seq + 1] + r).long()
    return seq, pos, s["table"][seq, pos // c["page"]].long(), pos % c["page"]


def _rotate(x, w, cos, sin):
    """Head RMSNorm with weight w, then the rotation of the pairs (l, l + hd/2); x [rows][heads][hd]."""
    x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _encode(y, kind):
    """Codes of float64 values in units of their scale, as float64."""
    if kind == "i8":
        return y.round().clamp(-127, 127)
    return y.float().clamp(-448, 448).to(CODES["e4m3"]).double()


def _append(s):
    """The new tokens' blocks, 16 slots each: a slot holds an earlier token, a new one, or none of this sequence's."""
    c = s["case"]
    H, G, D, kind = c["heads"], c["kv_heads"], c["hd"], c["codes"]
    seq, pos, page, slot = _places(s)
    x = s["qkv"].view(s["rows"], H + 2 * G, D)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = _rotate(x[:, :H].float(), s["q_norm"], cos, sin) * D ** -0.5
    s["q"].copy_(q.reshape(s["rows"], H * D))
    k = _rotate(x[:, H:H + G].double(), s["k_norm"].double(), cos.double(), sin.double())
    y = torch.stack([k, x[:, H + G:].double()])  # [2][rows][G][D]
    # Every row's block, numbered by the first row that lies in it.
    first = pos - (s["lens"][seq] - (s["starts"][seq + 1] - s["starts"][seq])).long()  # the row's place in its sequence
    lead = torch.arange(s["rows"], device="cuda") - torch.minimum(first, pos % BLOCK)
    most = torch.zeros(2, s["rows"], G, dtype=torch.float64, device="cuda")
    most.scatter_reduce_(1, lead[None, :, None].expand(2, -1, G), y.abs().amax(-1), "amax")
    most = most[:, lead]
    old = s["scales"][:, page, :, slot // BLOCK].movedim(0, 1).double()  # (indexing puts rows first)
    keep = ((pos[lead] % BLOCK) > 0)[None, :, None] & (old > 0)
    fresh = (most / TOP[kind]).float().clamp(min=2.0 ** -126).double()
    fresh = torch.where(most > 0, fresh, 0.0)
    f, e = torch.frexp(most / (OVER[kind] * torch.where(keep, old, 1.0)))
    grow = torch.where(f == 0.5, e - 1, e).clamp(min=0)
    scale = torch.where(keep, torch.ldexp(old, grow), fresh)
    y = _encode(y * torch.where(scale > 0, 1 / scale, 0.0)[..., None], kind)
    # Earlier tokens of a block whose scale grew: written by the block's first row alone.
    earlier = (torch.arange(BLOCK, device="cuda") < (pos % BLOCK)[:, None]) & (lead == torch.arange(
        s["rows"], device="cuda"))[:, None]  # [rows][slots]
    slots = (slot // BLOCK * BLOCK)[:, None] + torch.arange(BLOCK, device="cuda")
    codes = s["codes"].view(torch.uint8)
    was = codes[:, page[:, None], slots].view(CODES[kind]).double()  # [2][rows][slots][G][D]
    less = torch.where(keep, grow, 0)[:, :, None, :, None]
    now = _encode(torch.ldexp(was, -less), kind).to(CODES[kind] if kind == "i8" else torch.float32)
    now = now.to(CODES[kind]).view(torch.uint8)
    # (A slot that is not an earlier token's is written to itself here, and the new tokens over it below.)
    where = torch.where(earlier, slots, slot[:, None])
    now = torch.where(earlier[None, :, :, None, None], now, codes[:, page, slot][:, :, None])
    codes[:, page[:, None], where] = now
    codes[:, page, slot] = (y if kind == "i8" else y.float()).to(CODES[kind]).view(torch.uint8)
    s["scales"][:, page, :, slot // BLOCK] = scale.float().movedim(1, 0)
    return s["q"], _values(s)


def _values(s):
    """The keys and values that the pool stands for."""
    scales = s["scales"].transpose(2, 3)[:, :, :, None, :, None]  # [2][pages][blocks][1][G][1]
    codes = s["codes"] if s["case"]["codes"] == "i8" else s["codes"].float()
    return (codes.unflatten(2, (-1, BLOCK)) * scales).flatten(2, 3)


def _padded(s):
    """Row of (sequence, i), which of them exist, and the mask [seq][i][key] of what each may see."""
    c = s["case"]
    i = torch.arange(s["max_rows"], device="cuda")
    n = (s["starts"][1:] - s["starts"][:-1])[:, None]
    live = i < n
    row = (s["starts"][:-1, None] + i).clamp_(max=s["rows"] - 1).long()
    pos = (s["lens"][:, None] - n + i)[..., None]
    key = torch.arange(-(-s["max_len"] // c["page"]) * c["page"], device="cuda")
    sees = key <= pos
    if c["window"]:
        sees &= key > pos - c["window"]
    return row, live, sees


def _gathered(s, i, table):
    """float32 keys (i = 0) or values (1) [sequence][key][G][D] of the pages of a table."""
    c = s["case"]
    x = s["codes"].view(torch.uint8)[i][table].view(CODES[c["codes"]]).float()  # [S][entries][T][G][D]
    x = x.unflatten(2, (-1, BLOCK)) * s["scales"][i][table].transpose(2, 3)[:, :, :, None, :, None]
    return x.reshape(c["seqs"], -1, c["kv_heads"], c["hd"])


def _attend(s):
    c = s["case"]
    H, G, D = c["heads"], c["kv_heads"], c["hd"]
    S, N = c["seqs"], s["max_rows"]
    row, live, sees = _padded(s)
    table = s["table"][:, :sees.shape[-1] // c["page"]].clamp(min=0).long()
    k = _gathered(s, 0, table).permute(0, 2, 3, 1).contiguous()
    v = _gathered(s, 1, table).permute(0, 2, 1, 3).contiguous()
    q = s["q"].float().view(-1, G, H // G, D)[row].permute(0, 2, 3, 1, 4).reshape(S, G, H // G * N, D)
    p = torch.matmul(q, k).mul_(D ** -0.5).view(S, G, H // G, N, -1)
    p.masked_fill_(~sees[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    den = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, G, H // G * N, -1), v).view(S, G, H // G, N, D) / den
    s["out"][row[live]] = o.permute(0, 3, 1, 2, 4).reshape(S, N, H * D)[live].to(s["out"].dtype)
    return s["out"]


def _plan(s):
    page, rows = s["case"]["page"], s["rows"]
    held, new, taken, shared = (s[n].long() for n in ("held", "new", "taken", "shared"))
    need = (held + new + page - 1) // page
    keep = torch.maximum(need, torch.minimum(shared, taken))
    gives, wants = (taken - keep).clamp(min=0), (need - taken).clamp(min=0)
    give_end, want_end = gives.cumsum(0), wants.cumsum(0)
    count = s["free_count"].long()
    e = torch.arange(s["table"].shape[1], device="cuda")
    given = (e >= keep[:, None]) & (e < taken[:, None])
    at = torch.where(given, count + (give_end - gives - keep)[:, None] + e, s["free"].numel())
    free = torch.cat([s["free"], s["free"][:1]])
    free.scatter_(0, at.flatten(), s["table"].flatten())
    s["free"].copy_(free[:-1])
    total = count + give_end[-1:]
    served = (wants == 0) | (want_end <= total)
    take = served[:, None] & (e >= taken[:, None]) & (e < need[:, None])
    at = (total - 1 - (want_end - wants - taken)[:, None] - e).clamp(0, s["free"].numel() - 1)
    s["table"].copy_(torch.where(take, s["free"][at], s["table"]))
    n = torch.where(served, new, 0)
    n = torch.where(n.cumsum(0) <= rows, n, 0)
    ends = n.cumsum(0)
    s["starts"][1:] = ends
    s["lens"].copy_(held + n)
    s["taken_out"].copy_(torch.where(served, keep, taken))
    s["free_count_out"].copy_(total - torch.where(served, wants, 0).sum())
    r = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(ends, r, right=True).clamp(max=len(new) - 1)
    pos = held[seq] + r - (ends - n)[seq]
    live = r < ends[-1]
    slot = s["table"][seq, (pos // page).clamp(max=s["table"].shape[1] - 1)].long() * page + pos % page
    s["positions"].copy_(torch.where(live, pos, -1))
    s["sequences"].copy_(torch.where(live, seq, -1))
    s["slots"].copy_(torch.where(live, slot, -1))
    return _planned(s)


def _planned(s):
    return [s[n] for n in ("starts", "lens", "taken_out", "free_count_out", "table", "free", "positions", "sequences",
                           "slots")]


def _probs(s):
    x, t = s["logits"][:, :s["case"]["vocab"]], s["temperatures"][:, None]
    most, at = x.max(1, keepdim=True)
    at = torch.where(x == most, torch.arange(x.shape[1], device="cuda"), x.shape[1]).amin(1, keepdim=True)
    p = ((x - most) / torch.where(t > 0, t, 1.0)).exp_()
    p = p / p.sum(1, keepdim=True)
    one = torch.arange(x.shape[1], device="cuda") == at
    s["probs"].copy_(torch.where(t > 0, p, one.float()))
    return s["probs"]


def _verify(s):
    """Sums and the values next to a border in float64: a token is one or another."""
    R, V = s["rows"], s["case"]["vocab"]
    r = torch.arange(R, device="cuda")
    starts = s["starts"].long()
    first, last = starts[:-1], starts[1:] - 1
    seq = torch.searchsorted(starts, r, right=True) - 1
    x = s["drafts"].long()[:, None]
    px = s["target"].gather(1, x).double().flatten()
    qx = s["draft"].gather(1, x).double().flatten() if s["draft"] is not None else torch.ones_like(px)
    fails = ~(s["accept_u"].double() * qx < px) | (r == last[seq])
    at = torch.full_like(first, R).scatter_reduce_(0, seq, torch.where(fails, r, R), "amin")
    p = s["target"][at].double()
    if s["draft"] is not None:
        rest = (p - s["draft"][at].double()).clamp_(min=0)
    else:
        rest = torch.where(torch.arange(V, device="cuda") == x[at], 0.0, p)
    rest = torch.where(((at == last) | (rest.sum(1) == 0))[:, None], p, rest)
    cum = rest.cumsum(1)
    token = torch.searchsorted(cum, s["sample_u"].double()[:, None] * cum[:, -1:], right=True).flatten()
    token = torch.minimum(token, torch.where(rest > 0, torch.arange(V, device="cuda"), 0).amax(1))
    s["accepted"].copy_(at - first)
    s["kept"].copy_(s["lens"] - (last - at))
    s["tokens"].copy_(torch.where(r < at[seq], s["drafts"].long(), torch.where(r == at[seq], token[seq], -1)))
    return s["tokens"], s["accepted"], s["kept"]


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if own:
        from gophonic_amd import gphq

        if kind == "plan":
            s["plan"].run()
            return _planned(s)
        if kind == "append":
            gphq.paged8_append(s["kv"], s["batch"], s["qkv"], s["q"], c["heads"], s["q_norm"], s["k_norm"], EPS,
                               s["cos"], s["sin"], c["hd"] ** -0.5)
            return s["q"], _values(s)
        if kind == "attend":
            gphq.paged8_attention(s["kv"], s["batch"], s["q"], s["out"], c["heads"], c["hd"] ** -0.5, c["window"],
                                  work=s["work"])
            return s["out"]
        if kind == "probs":
            gphq.probabilities(s["logits"][:, :c["vocab"]], s["probs"], s["temperatures"], work=s["work"])
            return s["probs"]
        gphq.verify_drafts(s["starts"], s["drafts"], s["target"], s["draft"], s["accept_u"], s["sample_u"],
                           s["tokens"], s["accepted"], lens=s["lens"], kept=s["kept"], work=s["work"])
        return s["tokens"], s["accepted"], s["kept"]
    return {"plan": _plan, "append": _append, "attend": _attend, "probs": _probs, "verify": _verify}[kind](s)


# ---- 64 bits ------------------------------------------------------------------


def exact(case, seed):
    c, s = case, prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attend": _exact_attend, "probs": _exact_probs,
            "verify": _exact_verify}[c["kind"]](c, s)


def _exact_plan(c, s):
    """One request after another, on the host."""
    held, new, taken, shared, table, free = (s[n].tolist() for n in ("held", "new", "taken", "shared", "table", "free"))
    page, stack = c["page"], free[:int(s["free_count"])]
    need = [-(-(h + n) // page) for h, n in zip(held, new)]
    for i, t in enumerate(taken):
        left = min(t, max(need[i], min(shared[i], t)))
        stack += table[i][left:t]
        taken[i] = left
    free[:len(stack)] = stack
    starts, lens, short, asked = [0], [], False, 0
    for i, n in enumerate(new):
        want = max(0, need[i] - taken[i])
        short |= want > len(stack)
        if want and short:
            n = 0
        else:
            for e in range(want):
                table[i][taken[i] + e] = stack.pop()
            taken[i] += want
        asked += n
        if asked > s["rows"]:
            n = 0
        lens.append(held[i] + n)
        starts.append(starts[-1] + n)
    place = [(h + j, i, table[i][(h + j) // page] * page + (h + j) % page)
             for i, h in enumerate(held) for j in range(starts[i + 1] - starts[i])]
    place += [(-1, -1, -1)] * (s["rows"] - len(place))
    return [_ints(v, torch.int64) for v in (starts, lens, taken, [len(stack)], table, free, *zip(*place))]


def _exact_append(c, s):
    H, G, D, T, kind = c["heads"], c["kv_heads"], c["hd"], c["page"], c["codes"]
    starts, lens, table = s["starts"].tolist(), s["lens"].tolist(), s["table"].tolist()
    x = s["qkv"].double().view(s["rows"], H + 2 * G, D)
    pos = torch.cat([torch.arange(n - (b - a), n) for a, b, n in zip(starts, starts[1:], lens)]).cuda()
    ang = [t[pos].double()[:, None, :] for t in (s["cos"], s["sin"])]

    def head(h, w):
        h = h * torch.rsqrt((h * h).sum(-1, keepdim=True) / D + EPS) * w.double()
        lo, hi = h[..., :D // 2], h[..., D // 2:]
        return torch.cat((lo * ang[0] - hi * ang[1], lo * ang[1] + hi * ang[0]), dim=-1)

    y = torch.stack([head(x[:, H:H + G], s["k_norm"]), x[:, H + G:]])
    codes, scales = s["codes"].view(torch.uint8), s["scales"]
    values = (codes.view(CODES[kind]).double().unflatten(2, (-1, BLOCK))
              * scales.double().transpose(2, 3)[:, :, :, None, :, None]).flatten(2, 3)

    def code(v):
        if kind == "i8":
            return v.round().clamp(-127, 127)
        return v.float().clamp(-448, 448).to(CODES[kind]).double()

    for i, (a, b, n) in enumerate(zip(starts, starts[1:], lens)):
        p = n - (b - a)
        while p < n:  # one block of one sequence after another
            end, at = min(n, (p // BLOCK + 1) * BLOCK), table[i][p // T]
            t0, t1, u0 = p % T // BLOCK * BLOCK, end - 1, p % T
            mine = y[:, b - n + p:b - n + end]  # [2][tokens][G][D]
            most = mine.abs().amax((1, 3))
            scale = (most / TOP[kind]).float().double()
            if u0 > t0:
                was = scales[:, at, :, t0 // BLOCK].double()
                grown = was.clone()
                while bool((most > OVER[kind] * grown).any()):
                    grown = torch.where(most > OVER[kind] * grown, 2 * grown, grown)
                before = codes[:, at, t0:u0].view(CODES[kind]).double()
                values[:, at, t0:u0] = code(before * (was / grown)[:, None, :, None]) * grown[:, None, :, None]
                scale = grown
            values[:, at, u0:t1 % T + 1] = code(mine / scale[:, None, :, None]) * scale[:, None, :, None]
            if u0 > t0 or end % BLOCK:  # slots behind the tokens: codes of earlier requests, by the new scale
                stale = codes[:, at, t1 % T + 1:t0 + BLOCK].view(CODES[kind]).double()
                values[:, at, t1 % T + 1:t0 + BLOCK] = stale * scale.float().double()[:, None, :, None]
            p = end
    return (head(x[:, :H], s["q_norm"]) / math.sqrt(D)).reshape(s["rows"], H * D), values


def _exact_attend(c, s):
    H, G, D, page = c["heads"], c["kv_heads"], c["hd"], c["page"]
    starts, lens, table = s["starts"].tolist(), s["lens"].tolist(), s["table"].tolist()
    out = torch.empty(s["rows"], H, D, dtype=torch.float64, device="cuda")
    for i, (a, b, n) in enumerate(zip(starts, starts[1:], lens)):
        pages = torch.tensor(table[i][:-(-n // page)]).cuda()
        j = torch.arange(n, device="cuda")
        at = torch.arange(n - (b - a), n, device="cuda")[:, None]
        hide = (j > at) | (j <= at - c["window"]) if c["window"] else j > at
        for g in range(G):
            k, v = ((s["codes"].view(torch.uint8)[t][pages, :, g].view(CODES[c["codes"]]).double().reshape(-1, D)
                     * s["scales"][t][pages, g].double().reshape(-1).repeat_interleave(BLOCK)[:, None])[:n]
                    for t in (0, 1))
            for h in range(g * (H // G), (g + 1) * (H // G)):
                w = (s["q"][a:b, h * D:(h + 1) * D].double() @ k.T) / math.sqrt(D)
                out[a:b, h] = torch.softmax(w.masked_fill(hide, -math.inf), -1) @ v
    return out.reshape(s["rows"], H * D)


def _exact_probs(c, s):
    out = torch.zeros(c["rows"], c["vocab"], dtype=torch.float64, device="cuda")
    for r, t in enumerate(s["temperatures"].double().tolist()):
        x = s["logits"][r, :c["vocab"]].double()
        if t > 0:
            out[r] = torch.softmax(x / t, 0)
        else:
            out[r, (x == x.max()).nonzero()[0]] = 1
    return out


def _exact_verify(c, s):
    """One sequence after another."""
    tokens, accepted, kept = [], [], []
    starts, drafts, u, v = (s[n].tolist() for n in ("starts", "drafts", "accept_u", "sample_u"))
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        row = a
        while row < b - 1:
            x = drafts[row]
            q = float(s["draft"][row, x]) if s["draft"] is not None else 1.0
            if not u[row] * q < float(s["target"][row, x]):
                break
            row += 1
        w = s["target"][row].double()
        if row < b - 1:
            less = w.clone()
            if s["draft"] is not None:
                less -= s["draft"][row].double()
                less[less < 0] = 0
            else:
                less[drafts[row]] = 0
            w = less if float(less.sum()) > 0 else w
        cum = torch.cumsum(w, 0)
        over = (cum > v[i] * cum[-1]).nonzero()
        token = int(over[0] if len(over) else w.nonzero()[-1])
        tokens += drafts[a:row] + [token] + [-1] * (b - 1 - row)
        accepted.append(row - a)
        kept.append(int(s["lens"][i]) - (b - 1 - row))
    return _ints(tokens, torch.int64), _ints(accepted, torch.int64), _ints(kept, torch.int64)
