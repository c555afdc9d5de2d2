"""CPU checks of the paged cache's and the adapters' entry points: bad arguments are refused before any device work."""
import ctypes

import pytest

from gophonic_amd import gphq

P = 4096  # a non-null, aligned address that is never read


def kv(**over):
    d = dict(k_dev=P, v_dev=P, page_stride=2048, token_stride=128, head_stride=128, pages=4, page_tokens=16, kv_heads=1,
             head_dim=128, dtype=gphq.DTYPE_F16, reserved=0)
    d.update(over)
    return gphq.PagedKvDesc(*[d[n] for n, _ in gphq.PagedKvDesc._fields_])


def batch(**over):
    d = dict(starts_dev=P, lens_dev=P, table_dev=P, table_stride=4, seqs=2, rows=8, max_rows=4, max_len=64, bad_dev=None)
    d.update(over)
    return gphq.PagedBatchDesc(*[d[n] for n, _ in gphq.PagedBatchDesc._fields_])


def append(k=None, b=None, **over):
    d = dict(dtype=gphq.DTYPE_F32, qkv=P, qkv_stride=4 * 128, heads=2, qn=P, kn=P, eps=1e-6, cos=P, sin=P, rope=64,
             scale=1.0, q=P, q_stride=256)
    d.update(over)
    return gphq.load().gphq_paged_append(ctypes.byref(k or kv()), ctypes.byref(b or batch()), *d.values(), None)


def attend(k=None, b=None, **over):
    d = dict(dtype=gphq.DTYPE_F32, q=P, q_stride=256, heads=2, scale=1.0, window=0, out=P + (1 << 20), out_stride=256,
             work=P, bytes=1 << 30)
    d.update(over)
    return gphq.load().gphq_paged_attention(ctypes.byref(k or kv()), ctypes.byref(b or batch()), *d.values(), None)


BAD_KV = [
    (dict(dtype=7), gphq.ERR_UNSUPPORTED), (dict(head_dim=96), gphq.ERR_UNSUPPORTED),
    (dict(page_tokens=8), gphq.ERR_UNSUPPORTED), (dict(page_tokens=48), gphq.ERR_UNSUPPORTED),
    (dict(page_tokens=8192), gphq.ERR_UNSUPPORTED), (dict(pages=0), gphq.ERR_PAGED_SHAPE),
    (dict(pages=1 << 31), gphq.ERR_PAGED_SHAPE), (dict(kv_heads=0), gphq.ERR_PAGED_SHAPE),
    (dict(token_stride=64), gphq.ERR_PAGED_SHAPE), (dict(token_stride=132), gphq.ERR_PAGED_SHAPE),
    (dict(page_stride=-2048), gphq.ERR_PAGED_SHAPE), (dict(head_stride=0), gphq.ERR_PAGED_SHAPE),
    (dict(page_stride=1 << 61), gphq.ERR_PAGED_SHAPE), (dict(k_dev=None), gphq.ERR_PAGED_SHAPE),
    (dict(v_dev=P + 8), gphq.ERR_PAGED_SHAPE),
]
BAD_BATCH = [
    (dict(seqs=-1), gphq.ERR_PAGED_SHAPE), (dict(rows=-1), gphq.ERR_PAGED_SHAPE),
    (dict(rows=(1 << 20) + 1), gphq.ERR_PAGED_SHAPE), (dict(seqs=1 << 20), gphq.ERR_PAGED_SHAPE),
    (dict(max_rows=-1), gphq.ERR_PAGED_SHAPE), (dict(max_len=-1), gphq.ERR_PAGED_SHAPE),
    (dict(max_len=65), gphq.ERR_PAGED_SHAPE), (dict(table_stride=3), gphq.ERR_PAGED_SHAPE),
    (dict(table_stride=1 << 31), gphq.ERR_PAGED_SHAPE), (dict(starts_dev=None), gphq.ERR_PAGED_SHAPE),
    (dict(lens_dev=None), gphq.ERR_PAGED_SHAPE), (dict(table_dev=None), gphq.ERR_PAGED_SHAPE),
    (dict(bad_dev=P + 2), gphq.ERR_PAGED_SHAPE), (dict(table_dev=P + 2), gphq.ERR_PAGED_SHAPE),
]


@pytest.mark.parametrize("over,want", BAD_KV, ids=lambda v: str(v))
def test_bad_pools_are_refused(over, want):
    assert append(kv(**over)) == want
    assert attend(kv(**over)) == want


@pytest.mark.parametrize("over,want", BAD_BATCH, ids=lambda v: str(v))
def test_bad_batches_are_refused(over, want):
    assert append(b=batch(**over)) == want
    assert attend(b=batch(**over)) == want


@pytest.mark.parametrize("over,want", [
    (dict(dtype=gphq.DTYPE_BF16), gphq.ERR_UNSUPPORTED), (dict(dtype=0), gphq.ERR_UNSUPPORTED),
    (dict(heads=0), gphq.ERR_PAGED_SHAPE), (dict(heads=1025), gphq.ERR_PAGED_SHAPE),
    (dict(qkv_stride=508), gphq.ERR_PAGED_SHAPE), (dict(qkv_stride=514), gphq.ERR_PAGED_SHAPE),
    (dict(q_stride=252), gphq.ERR_PAGED_SHAPE), (dict(cos=None), gphq.ERR_PAGED_SHAPE),
    (dict(sin=None), gphq.ERR_PAGED_SHAPE), (dict(rope=0), gphq.ERR_PAGED_SHAPE), (dict(eps=-1.0), gphq.ERR_PAGED_SHAPE),
    (dict(eps=float("nan")), gphq.ERR_PAGED_SHAPE), (dict(qkv=None), gphq.ERR_PAGED_SHAPE),
    (dict(q=P + 4), gphq.ERR_PAGED_SHAPE), (dict(qn=P + 8), gphq.ERR_PAGED_SHAPE),
], ids=lambda v: str(v))
def test_append_refuses(over, want):
    assert append(**over) == want


def test_append_refuses_queries_laid_over_other_rows():
    assert append(q=P + 64, q_stride=512) == gphq.ERR_OVERLAP
    assert append(q=P, q_stride=256) == gphq.ERR_OVERLAP  # the same address with another stride


@pytest.mark.parametrize("over,want", [
    (dict(dtype=gphq.DTYPE_BF16), gphq.ERR_UNSUPPORTED), (dict(heads=0), gphq.ERR_PAGED_SHAPE),
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
    k, b = kv(pages=1 << 16), batch(max_len=1 << 16, table_stride=1 << 12)
    need = lib.gphq_paged_attention_workspace_bytes(ctypes.byref(k), ctypes.byref(b), gphq.DTYPE_F32, 2, 0)
    assert need > 0
    assert attend(k, b, bytes=need - 1) == gphq.ERR_PAGED_SHAPE
    assert attend(k, b, work=None) == gphq.ERR_PAGED_SHAPE
    assert attend(k, b, work=P + 8) == gphq.ERR_PAGED_SHAPE
    for over in (dict(dtype=gphq.DTYPE_BF16), dict(heads=0), dict(window=-1)):
        d = dict(dtype=gphq.DTYPE_F32, heads=2, window=0)
        d.update(over)
        assert lib.gphq_paged_attention_workspace_bytes(ctypes.byref(k), ctypes.byref(b), *d.values()) < 0


@pytest.mark.parametrize("seqs,rows,max_rows,max_len", [(2, 8192, 8192, 40960), (16, 1 << 20, 1 << 20, 40960),
                                                        (1, 2048, 2048, 1 << 20), (300, 4096, 2048, 40960)])
def test_the_workspace_stays_small(seqs, rows, max_rows, max_len):
    """Splits are cut so that the blocks in flight hold them, at most a few rounds of the chip's: under 256 MiB."""
    k = kv(kv_heads=8, pages=1 << 20, head_stride=2048, page_stride=16384)
    b = batch(seqs=seqs, rows=rows, max_rows=max_rows, max_len=max_len, table_stride=max_len // 16)
    for heads in (8, 32, 64):
        n = gphq.load().gphq_paged_attention_workspace_bytes(ctypes.byref(k), ctypes.byref(b), gphq.DTYPE_F32, heads, 0)
        assert 0 <= n < 256 << 20


@pytest.mark.parametrize("seqs,rows", [(2048, 1), (16384, 1), (65536, 1), (65536, 40), (4096, 4096), (65536, 1 << 16)])
@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (8, 1), (64, 64)])
@pytest.mark.parametrize("max_rows", [1, 16])
def test_idle_sequences_cost_no_workspace(seqs, rows, heads, kv_heads, max_rows):
    """A batch made for many sequences of which few bring rows: at most `rows` of them hold split results, and it is
    not refused while its tiles, kv_heads seqs ceil(min(max_rows g, 64) / 16), are under 2^23."""
    k = kv(kv_heads=kv_heads, pages=1 << 20, head_stride=2048, page_stride=2048 * kv_heads)
    b = batch(seqs=seqs, rows=rows, max_rows=max_rows, max_len=40960, table_stride=2560)
    for dtype in (gphq.DTYPE_F16, gphq.DTYPE_F32):
        n = gphq.load().gphq_paged_attention_workspace_bytes(ctypes.byref(k), ctypes.byref(b), dtype, heads, 0)
        assert 0 <= n < 256 << 20


@pytest.mark.parametrize("over,heads,kv_heads,fits", [
    (dict(seqs=65536, rows=65536, max_rows=1), 127, 127, True), (dict(seqs=65536, rows=65536, max_rows=1), 128, 128, False),
    (dict(seqs=65536, rows=1 << 20, max_rows=16), 128, 32, False),
    (dict(seqs=1, rows=1 << 20, max_rows=1 << 20), 512, 8, True), (dict(seqs=1, rows=1 << 20, max_rows=1 << 20), 1024, 8, False),
    (dict(seqs=2, rows=1 << 20, max_rows=1 << 20), 128, 2, False),
])
def test_attention_refuses_more_blocks_than_a_launch_takes(over, heads, kv_heads, fits):
    k = kv(kv_heads=kv_heads, head_stride=2048, page_stride=2048 * kv_heads)
    b = batch(max_len=4096, table_stride=256, **over)
    n = gphq.load().gphq_paged_attention_workspace_bytes(ctypes.byref(k), ctypes.byref(b), gphq.DTYPE_F16, heads, 0)
    assert (n >= 0) == fits and (fits or n == gphq.ERR_PAGED_SHAPE)


def test_null_descriptions_are_refused():
    lib = gphq.load()
    assert lib.gphq_paged_attention_workspace_bytes(None, ctypes.byref(batch()), 3, 2, 0) == gphq.ERR_PAGED_SHAPE
    assert lib.gphq_paged_attention_workspace_bytes(ctypes.byref(kv()), None, 3, 2, 0) == gphq.ERR_PAGED_SHAPE
    assert lib.gphq_paged_check(None, None) == gphq.ERR_PAGED_SHAPE


@pytest.mark.parametrize("over", [dict(seqs=0), dict(rows=0), dict(max_rows=0)], ids=lambda v: str(v))
def test_an_empty_batch_is_no_work(over):
    b = batch(starts_dev=P, **over)
    assert append(b=b) == gphq.OK
    assert attend(b=b) == gphq.OK
    assert gphq.load().gphq_paged_attention_workspace_bytes(ctypes.byref(kv()), ctypes.byref(b), 3, 2, 0) == 0


def lora(**over):
    d = dict(dtype=gphq.DTYPE_BF16, a=P, b=P, ranks=P, scales=P, slots=2, max_rank=16, row_slots=P, x=P, x_stride=64,
             y=P + (1 << 20), y_stride=40, rows=3, k=64, n=40, work=P, bytes=1 << 24)
    d.update(over)
    return gphq.load().gphq_lora_add(*d.values(), None)


@pytest.mark.parametrize("over,want", [
    (dict(dtype=9), gphq.ERR_UNSUPPORTED), (dict(slots=-1), gphq.ERR_DIMENSIONS), (dict(max_rank=12), gphq.ERR_DIMENSIONS),
    (dict(max_rank=136), gphq.ERR_DIMENSIONS), (dict(k=48), gphq.ERR_DIMENSIONS), (dict(k=-32), gphq.ERR_DIMENSIONS),
    (dict(n=-1), gphq.ERR_DIMENSIONS), (dict(rows=-1), gphq.ERR_DIMENSIONS), (dict(x_stride=60), gphq.ERR_DIMENSIONS),
    (dict(x_stride=66), gphq.ERR_DIMENSIONS), (dict(y_stride=39), gphq.ERR_DIMENSIONS), (dict(a=None), gphq.ERR_DIMENSIONS),
    (dict(row_slots=None), gphq.ERR_DIMENSIONS), (dict(x=P + 8), gphq.ERR_DIMENSIONS), (dict(b=P + 8), gphq.ERR_DIMENSIONS),
    (dict(work=None), gphq.ERR_DIMENSIONS), (dict(bytes=191), gphq.ERR_DIMENSIONS), (dict(y=P + 2), gphq.ERR_DIMENSIONS),
    (dict(y=P), gphq.ERR_OVERLAP),
    (dict(k=(1 << 31) - 32, x_stride=1 << 31, y=1 << 60, bytes=1 << 60), gphq.ERR_DIMENSIONS),
    (dict(rows=256, n=1 << 27, y_stride=1 << 27, x=1 << 60, slots=16, bytes=1 << 60), gphq.ERR_DIMENSIONS),
    (dict(rows=1 << 20, n=1 << 30, y_stride=1 << 30, x=1 << 60, bytes=1 << 60), gphq.ERR_DIMENSIONS),
], ids=lambda v: str(v))
def test_lora_refuses(over, want):
    assert lora(**over) == want


@pytest.mark.parametrize("over", [dict(rows=0), dict(n=0), dict(slots=0), dict(max_rank=0), dict(k=0, x_stride=0)],
                         ids=lambda v: str(v))
def test_lora_without_work_is_ok(over):
    assert lora(**over) == gphq.OK


def test_pool_and_paged_pass_refuse_null_handles():
    lib = gphq.load()
    h = ctypes.c_void_p(1)
    assert lib.gphq_paged_pool_new(None, 4, 16, gphq.DTYPE_F32, ctypes.byref(h)) == gphq.ERR_WORKSPACE
    assert not h.value
    assert lib.gphq_paged_pool_new(None, 4, 16, gphq.DTYPE_F32, None) == gphq.ERR_DIMENSIONS
    assert lib.gphq_paged_pool_layer(None, 0, ctypes.byref(kv())) == gphq.ERR_PAGED_SHAPE
    assert lib.gphq_prefill_paged(None, None, None, None, None, 1, None, 1, None, 0, None) == gphq.ERR_WORKSPACE
    lib.gphq_paged_pool_free(None)


def test_descriptions_over_two_devices_are_refused():
    import torch

    def ints(n, device="cpu"):
        return torch.zeros(n, dtype=torch.int32, device=device)

    pages = torch.zeros(2, 16, 1, 64)
    cases = [lambda: gphq.PagedKv(pages, torch.empty_like(pages, device="meta")),
             lambda: gphq.PagedBatch(ints(3, "meta"), ints(2), ints((2, 1)), 2, 1, 16),
             lambda: gphq.PagedBatch(ints(3), ints(2), ints((2, 1), "meta"), 2, 1, 16),
             lambda: gphq.PagedBatch(ints(3, "meta"), ints(2, "meta"), ints((2, 1)), 2, 1, 16)]
    for make in cases:
        with pytest.raises(gphq.GphqError) as e:
            make()
        assert e.value.status == gphq.ERR_PAGED_SHAPE


@pytest.fixture
def on_the_cpu(monkeypatch):
    """The binding's checks on tensors in host memory; what they let through finds no device here."""
    import torch

    gphq.load()
    monkeypatch.setattr(gphq, "_here", lambda *tensors: None)
    monkeypatch.setattr(gphq, "stream_handle", lambda stream=None: None)
    return torch


@pytest.mark.parametrize("view", [lambda w: w[:1].expand(1 << 24), lambda w: w[::2], lambda w: w[:64].view(8, 8).t()],
                         ids=["expanded", "every other", "transposed"])
def test_a_workspace_that_is_not_one_piece_is_refused(on_the_cpu, view):
    """Its numbers of values would pass for more bytes than lie behind its address."""
    torch = on_the_cpu
    work = view(torch.zeros(1 << 20, dtype=torch.uint8))
    ints = lambda *v: torch.tensor(v, dtype=torch.int32)
    pages, row = torch.zeros(2, 16, 1, 64), torch.zeros(1, 64)
    kv, b = gphq.PagedKv(pages, pages.clone()), gphq.PagedBatch(ints(0, 1), ints(5), ints(0).view(1, 1), 1, 1, 5)
    with pytest.raises(gphq.GphqError) as e:
        gphq.paged_attention(kv, b, row, row.clone(), 1, 1.0, work=work)
    assert e.value.status == gphq.ERR_PAGED_SHAPE
    a, x = torch.zeros(1, 8, 32), torch.zeros(1, 32)
    with pytest.raises(gphq.GphqError) as e:
        gphq.lora_add(a, torch.zeros(1, 16, 8), x, torch.zeros(1, 16), ints(0), work=work)
    assert e.value.status == gphq.ERR_DIMENSIONS


def test_a_pool_s_layers_lie_on_its_own_device(monkeypatch):
    """Made while device 1 is current and described while device 0 is: views of device 1's memory, not copies."""
    import torch

    gphq.load()
    asked = []

    class Lib:
        def gphq_paged_pool_new(self, lm, pages, page_tokens, dtype, out):
            out._obj.value = P
            return gphq.OK

        def gphq_paged_pool_layer(self, pool, layer, out):
            for name, value in dict(k_dev=P, v_dev=2 * P, pages=3, page_tokens=16, kv_heads=2, head_dim=64,
                                    dtype=gphq.DTYPE_F32).items():
                setattr(out._obj, name, value)
            return gphq.OK

        def gphq_paged_pool_free(self, pool):
            pass

    def as_tensor(memory, device):
        asked.append((memory.__cuda_array_interface__["data"][0], torch.device(device)))
        return torch.zeros(memory.__cuda_array_interface__["shape"])

    monkeypatch.setattr(gphq, "load", Lib)
    monkeypatch.setattr(torch, "as_tensor", as_tensor)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    pool = gphq.PagedPool(type("Lm", (), dict(h=None)), 3, 16, torch.float32)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    kv = pool.layer(0)
    assert asked == [(P, torch.device("cuda", 1)), (2 * P, torch.device("cuda", 1))]
    assert kv.k.shape == (3, 16, 2, 64)
    pool.close()


def test_the_current_stream_s_handle_without_torch_s_private_call(monkeypatch):
    """A torch that has no such call is asked for the stream in the public way."""
    import torch

    gphq.load()
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    monkeypatch.setattr(gphq, "_raw_stream", None, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: type("Stream", (), dict(cuda_stream=1234)))
    assert gphq.stream_handle() == 1234
