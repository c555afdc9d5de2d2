"""CPU checks of the 8-bit paged cache's, the plan's and the sampling entry points: bad arguments are refused before any
device work."""
import ctypes

import pytest
import torch

from gophonic_amd import gphq
from tests import test_paged as tp
from tests.test_paged import P, batch


def kv8(**over):
    codes = {n: over.pop(n) for n in list(over) if n in dict(gphq.PagedKvDesc._fields_)}
    codes.setdefault("dtype", gphq.DTYPE_I8)
    d = dict(codes=tp.kv(**codes), k_scales_dev=P, v_scales_dev=P, scale_page_stride=1, scale_head_stride=1)
    d.update(over)
    return gphq.PagedKv8Desc(*[d[n] for n, _ in gphq.PagedKv8Desc._fields_])


def append(k=None, b=None, **over):
    d = dict(dtype=gphq.DTYPE_F32, qkv=P, qkv_stride=4 * 128, heads=2, qn=P, kn=P, eps=1e-6, cos=P, sin=P, rope=64,
             scale=1.0, q=P, q_stride=256)
    d.update(over)
    return gphq.load().gphq_paged8_append(ctypes.byref(k or kv8()), ctypes.byref(b or batch()), *d.values(), None)


def attend(k=None, b=None, **over):
    d = dict(dtype=gphq.DTYPE_F32, q=P, q_stride=256, heads=2, scale=1.0, window=0, out=P + (1 << 20), out_stride=256,
             work=P, bytes=1 << 30)
    d.update(over)
    return gphq.load().gphq_paged8_attention(ctypes.byref(k or kv8()), ctypes.byref(b or batch()), *d.values(), None)


BAD_KV = [
    (dict(dtype=gphq.DTYPE_F16), gphq.ERR_UNSUPPORTED), (dict(dtype=0), gphq.ERR_UNSUPPORTED),
    (dict(dtype=6), gphq.ERR_UNSUPPORTED), (dict(head_dim=96), gphq.ERR_UNSUPPORTED),
    (dict(page_tokens=8), gphq.ERR_UNSUPPORTED), (dict(page_tokens=48), gphq.ERR_UNSUPPORTED),
    (dict(pages=0), gphq.ERR_PAGED_SHAPE), (dict(kv_heads=0), gphq.ERR_PAGED_SHAPE),
    (dict(token_stride=64), gphq.ERR_PAGED_SHAPE), (dict(token_stride=136), gphq.ERR_PAGED_SHAPE),
    (dict(head_stride=0), gphq.ERR_PAGED_SHAPE), (dict(page_stride=1 << 62), gphq.ERR_PAGED_SHAPE),
    (dict(k_dev=None), gphq.ERR_PAGED_SHAPE), (dict(v_dev=P + 8), gphq.ERR_PAGED_SHAPE),
    (dict(k_scales_dev=None), gphq.ERR_PAGED_SHAPE), (dict(v_scales_dev=P + 2), gphq.ERR_PAGED_SHAPE),
    (dict(scale_page_stride=0), gphq.ERR_PAGED_SHAPE), (dict(scale_head_stride=0), gphq.ERR_PAGED_SHAPE),
    (dict(page_tokens=64, scale_head_stride=3, scale_page_stride=4), gphq.ERR_PAGED_SHAPE),
    (dict(scale_page_stride=1 << 60), gphq.ERR_PAGED_SHAPE),
]


@pytest.mark.parametrize("over,want", BAD_KV, ids=lambda v: str(v))
def test_bad_pools_are_refused(over, want):
    assert append(kv8(**dict(over))) == want
    assert attend(kv8(**dict(over))) == want


@pytest.mark.parametrize("over,want", tp.BAD_BATCH, ids=lambda v: str(v))
def test_bad_batches_are_refused(over, want):
    assert append(b=batch(**over)) == want
    assert attend(b=batch(**over)) == want


@pytest.mark.parametrize("over,want", [
    (dict(dtype=gphq.DTYPE_I8), gphq.ERR_UNSUPPORTED), (dict(dtype=0), gphq.ERR_UNSUPPORTED),
    (dict(heads=0), gphq.ERR_PAGED_SHAPE), (dict(heads=1025), gphq.ERR_PAGED_SHAPE),
    (dict(qkv_stride=508), gphq.ERR_PAGED_SHAPE), (dict(qkv_stride=514), gphq.ERR_PAGED_SHAPE),
    (dict(q_stride=252), gphq.ERR_PAGED_SHAPE), (dict(cos=None), gphq.ERR_PAGED_SHAPE),
    (dict(sin=None), gphq.ERR_PAGED_SHAPE), (dict(rope=0), gphq.ERR_PAGED_SHAPE), (dict(eps=-1.0), gphq.ERR_PAGED_SHAPE),
    (dict(eps=float("nan")), gphq.ERR_PAGED_SHAPE), (dict(qkv=None), gphq.ERR_PAGED_SHAPE),
    (dict(q=P + 4), gphq.ERR_PAGED_SHAPE), (dict(qn=P + 8), gphq.ERR_PAGED_SHAPE),
    (dict(q=P + 64, q_stride=512), gphq.ERR_OVERLAP), (dict(q=P, q_stride=256), gphq.ERR_OVERLAP),
], ids=lambda v: str(v))
def test_append_refuses(over, want):
    assert append(**over) == want


@pytest.mark.parametrize("over,want", [
    (dict(dtype=gphq.DTYPE_E4M3), gphq.ERR_UNSUPPORTED), (dict(heads=0), gphq.ERR_PAGED_SHAPE),
    (dict(scale=float("nan")), gphq.ERR_PAGED_SHAPE), (dict(scale=float("-inf")), gphq.ERR_PAGED_SHAPE),
    (dict(window=-1), gphq.ERR_PAGED_SHAPE), (dict(q_stride=252), gphq.ERR_PAGED_SHAPE),
    (dict(out_stride=258), gphq.ERR_PAGED_SHAPE), (dict(q=None), gphq.ERR_PAGED_SHAPE),
    (dict(out=P + (1 << 20) + 8), gphq.ERR_PAGED_SHAPE), (dict(out=P), gphq.ERR_OVERLAP),
    (dict(out=P + 1024), gphq.ERR_OVERLAP),
], ids=lambda v: str(v))
def test_attention_refuses(over, want):
    assert attend(**over) == want


def test_attention_refuses_a_short_workspace():
    lib = gphq.load()
    k, b = kv8(pages=1 << 16), batch(max_len=1 << 16, table_stride=1 << 12)
    need = lib.gphq_paged8_attention_workspace_bytes(ctypes.byref(k), ctypes.byref(b), gphq.DTYPE_F32, 2, 0)
    assert need > 0
    assert attend(k, b, bytes=need - 1) == gphq.ERR_PAGED_SHAPE
    assert attend(k, b, work=None) == gphq.ERR_PAGED_SHAPE
    assert attend(k, b, work=P + 8) == gphq.ERR_PAGED_SHAPE
    assert lib.gphq_paged8_attention_workspace_bytes(None, ctypes.byref(b), gphq.DTYPE_F32, 2, 0) < 0
    assert lib.gphq_paged8_attention_workspace_bytes(ctypes.byref(k), None, gphq.DTYPE_F32, 2, 0) < 0


@pytest.mark.parametrize("seqs,rows,max_rows,max_len", [(2, 8192, 8192, 40960), (16, 1 << 20, 1 << 20, 40960),
                                                        (65536, 40, 1, 40960), (300, 4096, 2048, 40960)])
def test_the_workspace_stays_small(seqs, rows, max_rows, max_len):
    k = kv8(kv_heads=8, pages=1 << 20, head_stride=2048, page_stride=16384, scale_page_stride=8)
    b = batch(seqs=seqs, rows=rows, max_rows=max_rows, max_len=max_len, table_stride=max_len // 16)
    for heads in (8, 32, 64):
        n = gphq.load().gphq_paged8_attention_workspace_bytes(ctypes.byref(k), ctypes.byref(b), gphq.DTYPE_F16, heads, 0)
        assert 0 <= n < 256 << 20


@pytest.mark.parametrize("over", [dict(seqs=0), dict(rows=0), dict(max_rows=0)], ids=lambda v: str(v))
def test_an_empty_batch_is_no_work(over):
    b = batch(starts_dev=P, **over)
    assert append(b=b) == gphq.OK
    assert attend(b=b) == gphq.OK


def test_a_pool_of_codes_is_no_pool_of_values():
    """The calls for values refuse codes, and the other way round."""
    k = tp.kv(dtype=gphq.DTYPE_I8)
    assert tp.append(k) == gphq.ERR_UNSUPPORTED and tp.attend(k) == gphq.ERR_UNSUPPORTED
    lib, h = gphq.load(), ctypes.c_void_p(1)
    assert lib.gphq_paged_pool_new(None, 4, 16, gphq.DTYPE_I8, ctypes.byref(h)) == gphq.ERR_WORKSPACE
    assert lib.gphq_paged_pool_layer8(None, 0, ctypes.byref(kv8())) == gphq.ERR_PAGED_SHAPE


@pytest.mark.parametrize("make", [
    lambda c, s: (c, c[:1], s, s), lambda c, s: (c.float(), c.float(), s, s), lambda c, s: (c, c, s.double(), s.double()),
    lambda c, s: (c, c, s[:, :, :1], s[:, :, :1]), lambda c, s: (c, c, s, s.transpose(0, 1).contiguous().transpose(0, 1)),
    lambda c, s: (c, c.view(torch.uint8), s, s), lambda c, s: (c.view(torch.uint8), c.view(torch.uint8), s, s),
    lambda c, s: (c, c, s.repeat(1, 1, 2)[..., ::2], s.repeat(1, 1, 2)[..., ::2]),
    lambda c, s: (c, c, s.to("meta"), s.to("meta")),
], ids=range(9))
def test_descriptions_that_do_not_fit_are_refused(make):
    c, s = torch.zeros(3, 32, 2, 64, dtype=torch.int8), torch.zeros(3, 2, 2)
    gphq.PagedKv8(c, c, s, s)
    with pytest.raises(gphq.GphqError):
        gphq.PagedKv8(*make(c, s))


# ---- the plan -------------------------------------------------------------------


def requests(**over):
    d = dict(held_dev=P, count_dev=P, taken_dev=P, shared_dev=None, table_dev=P, free_dev=P, free_count_dev=P,
             starts_dev=P, lens_dev=P, taken_out_dev=P, free_count_out_dev=P, positions_dev=None, sequences_dev=None,
             slots_dev=None, bad_dev=None, seqs=2, table_stride=4, free_len=8, page_tokens=16, rows=8, max_rows=4,
             max_len=64)
    d.update(over)
    return gphq.PagedRequestsDesc(*[d[n] for n, _ in gphq.PagedRequestsDesc._fields_])


@pytest.mark.parametrize("over,want", [
    (dict(page_tokens=8), gphq.ERR_UNSUPPORTED), (dict(page_tokens=48), gphq.ERR_UNSUPPORTED),
    (dict(page_tokens=8192), gphq.ERR_UNSUPPORTED), (dict(seqs=-1), gphq.ERR_PAGED_SHAPE),
    (dict(seqs=65537), gphq.ERR_PAGED_SHAPE), (dict(rows=-1), gphq.ERR_PAGED_SHAPE),
    (dict(rows=(1 << 20) + 1), gphq.ERR_PAGED_SHAPE), (dict(max_rows=-1), gphq.ERR_PAGED_SHAPE),
    (dict(max_len=-1), gphq.ERR_PAGED_SHAPE), (dict(max_len=65), gphq.ERR_PAGED_SHAPE),
    (dict(free_len=-1), gphq.ERR_PAGED_SHAPE), (dict(free_len=1 << 31), gphq.ERR_PAGED_SHAPE),
    (dict(table_stride=1 << 31), gphq.ERR_PAGED_SHAPE), (dict(held_dev=None), gphq.ERR_PAGED_SHAPE),
    (dict(count_dev=None), gphq.ERR_PAGED_SHAPE), (dict(taken_dev=None), gphq.ERR_PAGED_SHAPE),
    (dict(table_dev=None), gphq.ERR_PAGED_SHAPE), (dict(free_dev=None), gphq.ERR_PAGED_SHAPE),
    (dict(free_count_dev=None), gphq.ERR_PAGED_SHAPE), (dict(starts_dev=None), gphq.ERR_PAGED_SHAPE),
    (dict(lens_dev=None), gphq.ERR_PAGED_SHAPE), (dict(taken_out_dev=None), gphq.ERR_PAGED_SHAPE),
    (dict(free_count_out_dev=None), gphq.ERR_PAGED_SHAPE), (dict(slots_dev=P + 4), gphq.ERR_PAGED_SHAPE),
    (dict(positions_dev=P + 2), gphq.ERR_PAGED_SHAPE), (dict(bad_dev=P + 1), gphq.ERR_PAGED_SHAPE),
], ids=lambda v: str(v))
def test_plan_refuses(over, want):
    assert gphq.load().gphq_paged_plan(ctypes.byref(requests(**over)), None) == want


def test_plan_refuses_no_requests_and_wrong_tensors():
    assert gphq.load().gphq_paged_plan(None, None) == gphq.ERR_PAGED_SHAPE
    i = lambda n: torch.zeros(n, dtype=torch.int32)
    args = lambda **o: {**dict(held=i(2), count=i(2), taken=i(2), table=i((2, 4)), free=i(8), free_count=i(1),
                               page_tokens=16, rows=8, max_rows=4, max_len=64), **o}
    gphq.load()
    gphq.PagedPlan(**args())
    for bad in (dict(held=i(2).long()), dict(count=i(1)), dict(table=i((3, 4))), dict(free_count=i(0)),
                dict(starts=i(2)), dict(slots=i(8)), dict(positions=i(7)), dict(taken=i(4)[::2]),
                dict(shared=i(2).to("meta"))):
        with pytest.raises(gphq.GphqError) as e:
            gphq.PagedPlan(**args(**bad))
        assert e.value.status == gphq.ERR_PAGED_SHAPE


# ---- probabilities and drafts -----------------------------------------------------


def probs(**over):
    d = dict(x=P, x_stride=64, t=None, out=P + (1 << 20), out_stride=64, rows=3, vocab=50, work=P, bytes=1 << 20)
    d.update(over)
    return gphq.load().gphq_probabilities(*d.values(), None)


@pytest.mark.parametrize("over,want", [
    (dict(rows=-1), gphq.ERR_DIMENSIONS), (dict(rows=(1 << 20) + 1), gphq.ERR_DIMENSIONS),
    (dict(vocab=-1), gphq.ERR_DIMENSIONS), (dict(vocab=(1 << 24) + 1, x_stride=1 << 25, out_stride=1 << 25), gphq.ERR_DIMENSIONS),
    (dict(x_stride=49), gphq.ERR_DIMENSIONS), (dict(out_stride=49), gphq.ERR_DIMENSIONS),
    (dict(x_stride=1 << 60), gphq.ERR_DIMENSIONS), (dict(x=None), gphq.ERR_DIMENSIONS),
    (dict(out=None), gphq.ERR_DIMENSIONS), (dict(x=P + 2), gphq.ERR_DIMENSIONS), (dict(t=P + 1), gphq.ERR_DIMENSIONS),
    (dict(work=None), gphq.ERR_DIMENSIONS), (dict(work=P + 8), gphq.ERR_DIMENSIONS), (dict(bytes=16), gphq.ERR_DIMENSIONS),
    (dict(out=P + 64), gphq.ERR_OVERLAP), (dict(out=P, out_stride=65), gphq.ERR_OVERLAP),
], ids=lambda v: str(v))
def test_probabilities_refuses(over, want):
    assert probs(**over) == want


@pytest.mark.parametrize("over", [dict(rows=0), dict(vocab=0)], ids=lambda v: str(v))
def test_probabilities_of_nothing(over):
    assert probs(**over) == gphq.OK


def verify(**over):
    d = dict(starts=P, drafts=P, target=P, target_stride=64, draft=P, draft_stride=64, accept_u=P, sample_u=P, seqs=2,
             rows=5, vocab=50, tokens=P, accepted=P, lens=P, kept=P, work=P, bytes=1 << 20)
    d.update(over)
    return gphq.load().gphq_verify_drafts(*d.values(), None)


@pytest.mark.parametrize("over", [
    dict(seqs=-1), dict(seqs=65537), dict(rows=-1), dict(rows=(1 << 20) + 1), dict(vocab=0), dict(vocab=(1 << 24) + 1),
    dict(seqs=65536, vocab=1 << 24, target_stride=1 << 24, draft_stride=1 << 24), dict(target_stride=49),
    dict(draft_stride=49), dict(target_stride=1 << 60), dict(draft_stride=1 << 60), dict(starts=None), dict(drafts=None),
    dict(target=None), dict(accept_u=None), dict(sample_u=None), dict(tokens=None), dict(accepted=None), dict(lens=None),
    dict(starts=P + 2), dict(kept=P + 2), dict(draft=P + 1), dict(work=None), dict(work=P + 8), dict(bytes=32),
], ids=lambda v: str(v))
def test_verify_refuses(over):
    assert verify(**over) == gphq.ERR_DIMENSIONS


def test_verify_of_no_sequences():
    assert verify(seqs=0, bytes=0) == gphq.OK


@pytest.fixture
def on_the_cpu(monkeypatch):
    """The binding's checks on tensors in host memory; what they let through finds no device here."""
    gphq.load()
    monkeypatch.setattr(gphq, "_here", lambda *tensors: None)
    monkeypatch.setattr(gphq, "stream_handle", lambda stream=None: None)


def test_wrong_tensors_are_refused(on_the_cpu):
    f = lambda *s: torch.zeros(*s)
    i = lambda n: torch.zeros(n, dtype=torch.int32)
    work = torch.zeros(1 << 16, dtype=torch.uint8)
    for x, out, t, w in ((f(3, 50), f(3, 49), None, work), (f(3, 50).double(), f(3, 50).double(), None, work),
                         (f(150), f(150), None, work), (f(3, 100)[:, ::2], f(3, 50), None, work),
                         (f(3, 50), f(3, 50), f(2), work), (f(3, 50), f(3, 50), f(3), work[:16]),
                         (f(3, 50), f(3, 50), f(3), work[::2]), (f(1, 50).expand(3, 50), f(3, 50), None, work)):
        with pytest.raises(gphq.GphqError) as e:
            gphq.probabilities(x, out, t, w)
        assert e.value.status == gphq.ERR_DIMENSIONS
    good = dict(starts=i(3), drafts=i(5), target=f(5, 50), draft=f(5, 50), accept_u=f(5), sample_u=f(2), tokens=i(5),
                accepted=i(2), lens=i(2), kept=i(2), work=work)
    for bad in (dict(starts=i(0)), dict(starts=i(3).long()), dict(drafts=i(4)), dict(target=f(50)), dict(draft=f(4, 50)),
                dict(draft=f(5, 50).half()), dict(accept_u=f(4)), dict(sample_u=f(1)), dict(tokens=i(10)[::2]),
                dict(accepted=i(1)), dict(lens=None), dict(kept=i(1)), dict(work=work[:16]),
                dict(target=f(5, 100)[:, ::2])):
        with pytest.raises(gphq.GphqError) as e:
            gphq.verify_drafts(**{**good, **bad})
        assert e.value.status == gphq.ERR_DIMENSIONS
