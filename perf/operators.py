"""Serving many requests over one paged K/V cache: the operators of a step, measured.

One case is a dict of plain values; `kind` names the operator:

  append   a batch's fused QKV rows: head RMSNorm and rotary position of every
           query and key head, queries written out, keys and values stored at
           their places in the pages (gphq.paged_append)
  attend   causal attention of the batch's new tokens, one or many per
           sequence, over the pages of their sequences (gphq.paged_attention)
  lora     low-rank adapters of several requests added beside one shared
           projection's output (gphq.lora_add)

A batch is `seqs` sequences; sequence s brings new[s] tokens to old[s] tokens
that the cache already holds. `lay` numbers the draw of those lengths (and of
the adapters' ranks), so a case alone fixes its work; everything else is made
from the seed. With `own` false the operators run in their plain form:
elementary torch operations in float32, rounded once at the end.
"""
import math
import random

import torch

own = False

POSITIONS = 40960  # the rotary table's rows: the context of the measured model shapes
THETA, EPS = 1e6, 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    qwen8 = dict(heads=32, kv_heads=8, hd=128)
    small = dict(heads=16, kv_heads=8, hd=128)
    return [
        # One request's next token: the smallest append, all latency.
        dict(name="append_token", kind="append", **small, rows="f32", cache="f16", page=16, order="head", seqs=1,
             new=1, new_hi=1, old=1024, old_hi=1024, lay=1),
        # 64 requests, one token each, in the middle of their answers.
        dict(name="append_lanes64", kind="append", **qwen8, rows="f32", cache="bf16", page=64, order="head", seqs=64,
             new=1, new_hi=1, old=100, old_hi=4000, lay=2),
        # Prompt chunks of five requests in one pass, token-major fp32 pages (the private prefix's row order).
        dict(name="append_chunks", kind="append", **qwen8, rows="f32", cache="f32", page=64, order="token", seqs=5,
             new=300, new_hi=1300, old=0, old_hi=2000, lay=3),
        # One token of one request over a short cache: latency of the attention step.
        dict(name="attend_token", kind="attend", **small, rows="f32", cache="f16", page=16, order="head", seqs=1,
             new=1, new_hi=1, old=1023, old_hi=1023, window=0, lay=4),
        # 16 requests' next tokens over ragged caches, fp32 pages: what the decode step's private caches hold.
        dict(name="attend_lanes16", kind="attend", **qwen8, rows="f32", cache="f32", page=64, order="head", seqs=16,
             new=1, new_hi=1, old=2000, old_hi=4095, window=0, lay=5),
        # Two long documents being answered: few rows, the cache's whole length, small pages.
        dict(name="attend_long", kind="attend", **qwen8, rows="bf16", cache="bf16", page=16, order="head", seqs=2,
             new=1, new_hi=1, old=32000, old_hi=40900, window=0, lay=6),
        # A follow-up message of 512 tokens over a conversation of several thousand.
        dict(name="attend_chunk", kind="attend", **qwen8, rows="f16", cache="f16", page=64, order="head", seqs=1,
             new=512, new_hi=512, old=7000, old_hi=7000, window=0, lay=7),
        # A whole 4096-token prompt in one pass, fp32 rows as the batched pass has them, FP16 pages.
        dict(name="attend_prompt", kind="attend", **qwen8, rows="f32", cache="f16", page=64, order="head", seqs=1,
             new=4096, new_hi=4096, old=0, old_hi=0, window=0, lay=8),
        # A continuous batch: prompt chunks of odd lengths and single tokens side by side.
        dict(name="attend_mixed", kind="attend", **qwen8, rows="f32", cache="bf16", page=32, order="token", seqs=12,
             new=1, new_hi=300, old=0, old_hi=4000, window=0, lay=9),
        # One token of one request with a rank-16 adapter beside o_proj: latency.
        dict(name="lora_token", kind="lora", weights="bf16", seqs=1, new=1, new_hi=1, slots=4, max_rank=16, k=4096,
             n=4096, lay=10),
        # 32 decode lanes over eight adapters of mixed ranks beside gate/up.
        dict(name="lora_lanes32", kind="lora", weights="f16", seqs=32, new=1, new_hi=1, slots=8, max_rank=64, k=4096,
             n=24576, lay=11),
        # Prompt chunks of six requests beside the QKV projection.
        dict(name="lora_chunks", kind="lora", weights="bf16", seqs=6, new=300, new_hi=1000, slots=4, max_rank=64,
             k=4096, n=6144, lay=12),
    ]


def draw(rng):
    def log(lo, hi, step=1):
        return max(1, round(lo * (hi / lo) ** rng.random() / step)) * step

    kind = rng.choice(["append", "attend", "attend", "lora"])
    lay = rng.randrange(1 << 20)
    if kind == "lora":
        tokens = rng.random() < 0.5
        seqs = log(1, 64) if tokens else rng.randint(1, 8)
        hi = 1 if tokens else log(2, 500)
        return dict(kind=kind, weights=rng.choice(["bf16", "f16", "f32"]), seqs=seqs, new=1, new_hi=hi,
                    slots=rng.randint(1, 8), max_rank=8 * rng.randint(1, 8), k=log(512, 6144, 32), n=log(500, 12000),
                    lay=lay)
    kv_heads = rng.choice([1, 2, 4, 8])
    c = dict(kind=kind, heads=kv_heads * rng.choice([1, 2, 4, 5, 8]), kv_heads=kv_heads, hd=rng.choice([64, 128, 128]))
    c["cache"] = rng.choice(["f32", "f16", "bf16"])
    c["rows"] = rng.choice(["f32", c["cache"]])
    c["page"] = rng.choice([16, 32, 64, 128])
    c["order"] = rng.choice(["head", "token"])
    shape = rng.choice(["tokens", "chunks", "mixed"])
    if shape == "tokens":
        seqs = log(1, 32)
        return dict(c, seqs=seqs, new=1, new_hi=1, old=0, old_hi=log(16, 32768 // seqs if seqs > 1 else 40000),
                    **(dict(window=rng.choice([0, 0, log(100, 4000)])) if kind == "attend" else {}), lay=lay)
    seqs = rng.randint(1, 3) if shape == "chunks" else rng.randint(3, 10)
    lo = log(2, 200) if shape == "chunks" else 1
    return dict(c, seqs=seqs, new=lo, new_hi=max(lo, log(lo + 1, 1000 if shape == "chunks" else 200)), old=0,
                old_hi=log(16, 3000), **(dict(window=rng.choice([0, 0, log(100, 4000)])) if kind == "attend" else {}),
                lay=lay)


# ---- lengths and work ---------------------------------------------------------


def _lengths(c):
    """(new tokens, tokens before them) of every sequence; in a mixed batch half of the sequences bring one token."""
    r = random.Random(c["lay"])
    new = [r.randint(c["new"], c["new_hi"]) if c["new"] > 1 or r.random() < 0.5 else 1 for _ in range(c["seqs"])]
    if c["seqs"] == 1:
        new = [c["new_hi"]]
    return new, [r.randint(c["old"], c["old_hi"]) for _ in new] if "old" in c else None


def _adapters(c):
    """(rank of every slot, slot of every sequence or -1)."""
    r = random.Random(c["lay"] + 1)
    ranks = [c["max_rank"]] + [r.randint(1, c["max_rank"]) for _ in range(c["slots"] - 1)]
    slots = [0] + [r.randint(-1, c["slots"] - 1) for _ in range(c["seqs"] - 1)]
    return ranks, slots


def work(case):
    c = case
    new, old = _lengths(c)
    rows = sum(new)
    if c["kind"] == "lora":
        ranks, slots = _adapters(c)
        live = sum(n for n, s in zip(new, slots) if s >= 0)
        used = sum(ranks[s] for s in set(slots) if s >= 0)
        return {"bytes": live * (4 * c["k"] + 8 * c["n"]) + used * (c["k"] + c["n"]) * SIZE[c["weights"]],
                "flops": 2 * sum(n * ranks[s] for n, s in zip(new, slots) if s >= 0) * (c["k"] + c["n"])}
    rb, cb, q, kv = SIZE[c["rows"]], SIZE[c["cache"]], c["heads"] * c["hd"], c["kv_heads"] * c["hd"]
    if c["kind"] == "append":
        return {"bytes": rows * ((2 * q + 2 * kv) * rb + 2 * kv * cb + 4 * c["hd"]), "flops": rows * (q + kv) * 8}
    read = pairs = 0
    for n, o in zip(new, old):
        w = c["window"] or o + n
        read += o + n - max(0, o + 1 - w)
        pairs += sum(min(o + i + 1, w) for i in range(n))
    return {"bytes": 2 * rows * q * rb + 2 * read * kv * cb, "flops": 4 * pairs * q}


# ---- inputs -------------------------------------------------------------------


def _randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _rope_tables(hd):
    """cos and sin [positions][hd / 2], the angles in float64."""
    inv = THETA ** (-torch.arange(0, hd // 2, dtype=torch.float64, device="cuda") * 2 / hd)
    a = torch.arange(POSITIONS, dtype=torch.float64, device="cuda")[:, None] * inv
    return a.cos().float(), a.sin().float()


def _pool(g, c, pages, dtype, offset):
    """A pool seen as [pages][page tokens][KV heads][head dim]: page memory in token or head order, filled with
    what earlier requests left there."""
    shape = (pages, c["page"], c["kv_heads"]) if c["order"] == "token" else (pages, c["kv_heads"], c["page"])
    t = torch.empty(*shape, c["hd"], dtype=dtype, device="cuda")
    for p in range(0, pages, 512):
        t[p:p + 512] = _randn(g, *t[p:p + 512].shape) + offset
    return t if c["order"] == "token" else t.transpose(1, 2)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(1_000_003 * seed + 29)
    new, old = _lengths(c)
    rows = sum(new)
    s = dict(case=c, rows=rows, max_rows=max(new))

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    if c["kind"] == "lora":
        ranks, slots = _adapters(c)
        dt = TYPES[c["weights"]]
        s["a"] = (_randn(g, c["slots"], c["max_rank"], c["k"]) / c["k"] ** 0.5).to(dt)
        s["b"] = (_randn(g, c["slots"], c["n"], c["max_rank"]) * 0.05).to(dt)
        s["ranks"], s["scales"] = ints(ranks), 2 * torch.rand(c["slots"], device="cuda", generator=g) + 0.5
        s["row_slots"] = ints([a for n, a in zip(new, slots) for _ in range(n)])
        s["x"], s["y"] = _randn(g, rows, c["k"]), _randn(g, rows, c["n"])
        s["x"][:, 5::256] *= 8  # a few large channels, as activations have
        if own:
            from gophonic_amd import gphq

            s["work"] = torch.empty(gphq.lora_workspace_bytes(rows, c["k"], c["max_rank"]), dtype=torch.uint8,
                                    device="cuda")
        return s
    lens = [o + n for o, n in zip(old, new)]
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
    s.update(starts=ints(starts), lens=ints(lens), table=table, max_len=max(lens))
    rdt, cdt = TYPES[c["rows"]], TYPES[c["cache"]]
    s["k"], s["v"] = _pool(g, c, pages, cdt, 0.0), _pool(g, c, pages, cdt, 0.1)
    H, G, D = c["heads"], c["kv_heads"], c["hd"]
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

        s["kv"] = gphq.PagedKv(s["k"], s["v"])
        s["batch"] = gphq.PagedBatch(s["starts"], s["lens"], s["table"], rows, s["max_rows"], s["max_len"])
        if c["kind"] == "attend":
            s["work"] = torch.empty(gphq.paged_attention_workspace_bytes(s["kv"], s["batch"], s["q"].dtype, H,
                                                                         c["window"]),
                                    dtype=torch.uint8, device="cuda")
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


def _append(s):
    c = s["case"]
    H, G, D = c["heads"], c["kv_heads"], c["hd"]
    _, pos, page, slot = _places(s)
    x = s["qkv"].float().view(s["rows"], H + 2 * G, D)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = _rotate(x[:, :H], s["q_norm"], cos, sin) * D ** -0.5
    k = _rotate(x[:, H:H + G], s["k_norm"], cos, sin)
    s["q"].copy_(q.reshape(s["rows"], H * D))
    s["k"][page, slot] = k.to(s["k"].dtype)
    s["v"][page, slot] = x[:, H + G:].to(s["v"].dtype)
    return s["q"], s["k"], s["v"]


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


def _attend(s):
    c = s["case"]
    H, G, D = c["heads"], c["kv_heads"], c["hd"]
    S, N = c["seqs"], s["max_rows"]
    row, live, sees = _padded(s)
    table = s["table"][:, :sees.shape[-1] // c["page"]].clamp(min=0).long()
    k = s["k"][table].float().reshape(S, -1, G, D).permute(0, 2, 3, 1).contiguous()
    v = s["v"][table].float().reshape(S, -1, G, D).permute(0, 2, 1, 3).contiguous()
    q = s["q"].float().view(-1, G, H // G, D)[row].permute(0, 2, 3, 1, 4).reshape(S, G, H // G * N, D)
    p = torch.matmul(q, k).mul_(D ** -0.5).view(S, G, H // G, N, -1)
    p.masked_fill_(~sees[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    den = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, G, H // G * N, -1), v).view(S, G, H // G, N, D) / den
    s["out"][row[live]] = o.permute(0, 3, 1, 2, 4).reshape(S, N, H * D)[live].to(s["out"].dtype)
    return s["out"]


def _lora(s):
    c = s["case"]
    R = c["max_rank"]
    mine = s["row_slots"][:, None] == torch.arange(c["slots"], device="cuda")
    keep = mine[..., None] & (torch.arange(R, device="cuda") < s["ranks"][:, None])
    t = torch.matmul(s["x"], s["a"].float().view(-1, c["k"]).t()).view(-1, c["slots"], R)
    t = torch.where(keep, t * s["scales"][:, None], 0.0).view(-1, c["slots"] * R)
    s["y"] += torch.matmul(t, s["b"].float().permute(0, 2, 1).reshape(-1, c["n"]))
    return s["y"]


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if own:
        from gophonic_amd import gphq

        if kind == "append":
            gphq.paged_append(s["kv"], s["batch"], s["qkv"], s["q"], c["heads"], s["q_norm"], s["k_norm"], EPS,
                              s["cos"], s["sin"], c["hd"] ** -0.5)
            return s["q"], s["k"], s["v"]
        if kind == "attend":
            gphq.paged_attention(s["kv"], s["batch"], s["q"], s["out"], c["heads"], c["hd"] ** -0.5, c["window"],
                                 work=s["work"])
            return s["out"]
        gphq.lora_add(s["a"], s["b"], s["x"], s["y"], s["row_slots"], s["ranks"], s["scales"], work=s["work"])
        return s["y"]
    return {"append": _append, "attend": _attend, "lora": _lora}[kind](s)


# ---- 64 bits ------------------------------------------------------------------


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "lora":
        y = s["y"].double()
        ranks, slots = s["ranks"].tolist(), s["row_slots"]
        for a, rank in enumerate(ranks):
            r = (slots == a).nonzero().flatten()
            if r.numel():
                low = s["x"][r].double() @ s["a"][a, :rank].double().T
                y[r] += float(s["scales"][a]) * (low @ s["b"][a, :, :rank].double().T)
        return y
    H, G, D, page = c["heads"], c["kv_heads"], c["hd"], c["page"]
    starts, lens, table = s["starts"].tolist(), s["lens"].tolist(), s["table"].tolist()
    if c["kind"] == "append":
        x = s["qkv"].double().view(s["rows"], H + 2 * G, D)
        k, v = s["k"].double(), s["v"].double()
        pos = torch.cat([torch.arange(n - (b - a), n) for a, b, n in zip(starts, starts[1:], lens)])
        where = [table[i][p // page] for i, (a, b, n) in enumerate(zip(starts, starts[1:], lens))
                 for p in range(n - (b - a), n)]
        where, pos = torch.tensor(where).cuda(), pos.cuda()
        ang = [t[pos].double()[:, None, :] for t in (s["cos"], s["sin"])]

        def head(h, w):
            h = h * torch.rsqrt((h * h).sum(-1, keepdim=True) / D + EPS) * w.double()
            lo, hi = h[..., :D // 2], h[..., D // 2:]
            return torch.cat((lo * ang[0] - hi * ang[1], lo * ang[1] + hi * ang[0]), dim=-1)

        k[where, pos % page] = head(x[:, H:H + G], s["k_norm"])
        v[where, pos % page] = x[:, H + G:]
        return (head(x[:, :H], s["q_norm"]) / math.sqrt(D)).reshape(s["rows"], H * D), k, v
    out = torch.empty(s["rows"], H, D, dtype=torch.float64, device="cuda")
    for i, (a, b, n) in enumerate(zip(starts, starts[1:], lens)):
        pages = torch.tensor(table[i][:-(-n // page)]).cuda()
        j = torch.arange(n, device="cuda")
        at = torch.arange(n - (b - a), n, device="cuda")[:, None]
        hide = (j > at) | (j <= at - c["window"]) if c["window"] else j > at
        for h in range(H):
            kh = s["k"][pages, :, h // (H // G)].reshape(-1, D)[:n].double()
            vh = s["v"][pages, :, h // (H // G)].reshape(-1, D)[:n].double()
            w = (s["q"][a:b, h * D:(h + 1) * D].double() @ kh.T) / math.sqrt(D)
            out[a:b, h] = torch.softmax(w.masked_fill(hide, -math.inf), -1) @ vh
    return out.reshape(s["rows"], H * D)
