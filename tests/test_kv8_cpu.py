"""What the 8-bit cache's operators and matvec refuse, and how a decode step is cut, without a GPU."""
import pytest
import torch

from sdcguard_b200.ops import attention, kv8, layers
from sdcguard_b200.ops.kv8 import KV8Cache
from sdcguard_b200.ops.quant import QuantWeights


def _cache(blocks=4, nkv=2):
    return KV8Cache.empty(blocks, nkv, device="cpu")


@pytest.mark.parametrize("change", ["dtype", "dims", "page", "scales", "contiguous"])
def test_cache_refuses(change):
    c = _cache()
    codes, scales = c.codes, c.scales
    if change == "dtype":
        codes = codes.view(torch.uint8)
    elif change == "dims":
        codes = codes[0]
    elif change == "page":
        codes = codes.view(torch.uint8).view(4, 2, 2, 32, 64).view(torch.float8_e4m3fn)
    elif change == "scales":
        scales = scales.double()
    else:
        scales = scales.transpose(1, 2)
    with pytest.raises(ValueError):
        KV8Cache(codes, scales)


def test_cache_layers_and_values():
    c = KV8Cache.empty(3, 1, layers=2, device="cpu")
    assert len(c) == 2 and c[1].num_blocks == 3 and c[1].nkv == 1
    with pytest.raises(IndexError):
        c[0][0]
    c.codes.view(torch.uint8)[1, 2, 1, 0, 4, 7] = 0x40        # 2.0
    c.scales[1, 2, 0, 1] = 0.25
    v = c[1].values(torch.tensor([2]))
    assert v[0, 1, 0, 4, 7] == 0.5 and v.abs().sum() == 0.5


def _append_args(t=3, nq=4, nkv=2):
    return dict(qkv=torch.zeros(t, (nq + 2 * nkv) * 128, dtype=torch.bfloat16), nq=nq, nkv=nkv,
                pos=torch.zeros(t, dtype=torch.int32), slots=torch.zeros(t, dtype=torch.int64), q_norm=None, k_norm=None,
                eps=1e-6, cos_sin=torch.zeros(8, 64, 2), q_out=torch.zeros(t, nq, 128, dtype=torch.bfloat16),
                cache=_cache(nkv=nkv))


@pytest.mark.parametrize("name,value", [
    ("qkv", torch.zeros(3, 8 * 128)), ("qkv", torch.zeros(3, 7 * 128, dtype=torch.bfloat16)),
    ("qkv", torch.zeros(8 * 128, 3, dtype=torch.bfloat16).t()),
    ("pos", torch.zeros(3, dtype=torch.int64)), ("slots", torch.zeros(2, dtype=torch.int64)),
    ("q_norm", torch.ones(128)), ("k_norm", torch.ones(64, dtype=torch.bfloat16)),
    ("cos_sin", torch.zeros(8, 65, 2)), ("cos_sin", torch.zeros(8, 6, 2)), ("cos_sin", torch.zeros(8, 128)[:, :64]),
    ("q_out", torch.zeros(3, 4, 64, dtype=torch.bfloat16)), ("cache", KV8Cache.empty(4, 3, device="cpu")),
    ("cache", KV8Cache.empty(4, 2, layers=1, device="cpu")), ("rows", torch.zeros(1, dtype=torch.int32)),
    ("check", torch.zeros(4, dtype=torch.int64)), (None, None)])
def test_append_refuses(name, value):
    """Each wrong argument, and (last) tensors that are not on a GPU."""
    args = _append_args()
    if name:
        args[name] = value
    with pytest.raises((ValueError, IndexError)):
        layers.qk_norm_rope_kv8(**args)


@pytest.mark.parametrize("bad", [dict(nseq=0), dict(nq=17, nkv=1), dict(nq=5, nkv=2), dict(max_ctx=0),
                                 dict(max_ctx=(1 << 24) + 1), dict(nkv=0)])
def test_decode_plan_refuses(bad):
    with pytest.raises(ValueError):
        attention.decode8_plan(**{**dict(nseq=2, nq=8, nkv=2, max_ctx=100, device="cpu"), **bad})


def _decode_args(b=2, nq=4, nkv=2):
    return dict(q=torch.zeros(b, nq, 128, dtype=torch.bfloat16), cache=_cache(nkv=nkv),
                block_table=torch.zeros(b, 3, dtype=torch.int32), seq_req=torch.zeros(b, dtype=torch.int32),
                ctx=torch.ones(b, dtype=torch.int32), plan=attention.decode8_plan(b, nq, nkv, 48, "cpu"))


@pytest.mark.parametrize("name,value", [
    ("q", torch.zeros(2, 4, 128)), ("q", torch.zeros(2, 6, 128, dtype=torch.bfloat16)),
    ("q", torch.zeros(3, 4, 128, dtype=torch.bfloat16)), ("q", torch.zeros(2, 4, 64, dtype=torch.bfloat16)),
    ("block_table", torch.zeros(2, 3, dtype=torch.int64)), ("block_table", torch.zeros(3, 2, dtype=torch.int32).t()),
    ("seq_req", torch.zeros(3, dtype=torch.int32)), ("ctx", torch.ones(2, dtype=torch.int64)),
    ("out", torch.zeros(2, 4, 128)), ("seq_idx", torch.zeros(2, dtype=torch.int64)),
    ("check", torch.zeros(4, dtype=torch.int64)), ("row_sq", torch.zeros(3)),
    ("plan", attention.decode8_plan(2, 8, 2, 48, "cpu")), (None, None)])
def test_decode_refuses(name, value):
    args = _decode_args()
    if name:
        args[name] = value
    with pytest.raises(ValueError):
        attention.decode8(**args)


def test_decode_cut():
    """Every length fits its cut, within what one combine takes; a cut does not depend on anything but the sizes."""
    for nseq in (1, 7, 256):
        for nkv in (1, 8):
            for ctx in (1, 16, 17, 64, 65, 1000, 8192, 40960, 131072, 1 << 24):
                seg, segs = attention.decode8_cut(nseq, nkv, ctx)
                assert seg >= 1 and 1 <= segs <= 256 and (segs - 1) * seg * 16 < ctx <= segs * seg * 16
    assert attention.decode8_cut(256, 8, 1600)[1] == 1         # a full batch: a CTA takes a whole row


@pytest.mark.parametrize("table,lens", [(torch.zeros(2, 3, dtype=torch.int64), [5, 5]),
                                        (torch.zeros(2, 3, dtype=torch.int32), [5]),
                                        (torch.zeros(2, 3, dtype=torch.int32), [5, 49]),
                                        (torch.zeros(2, 3, dtype=torch.int32), [5, 0])])
def test_prefill_plan_refuses(table, lens):
    with pytest.raises(ValueError):
        attention.prefill8_plan(table, lens, 2)


def test_prefill_plan_lists_the_pages():
    bt = torch.tensor([[4, 9, 1], [7, 0, 0], [2, 3, 8]], dtype=torch.int32)
    p = attention.prefill8_plan(bt, [33, 16, 17], 2)
    assert p.pages.tolist() == [4, 9, 1, 7, 2, 3] and p.table.tolist() == [[0, 1, 2], [3, 0, 0], [4, 5, 0]]
    assert p.work.shape == (6, 2, 2, 16, 128)
    with pytest.raises(ValueError):
        attention.prefill8_plan(bt, [33, 16, 17], 2, torch.zeros(100, dtype=torch.bfloat16))


@pytest.mark.parametrize("name,value", [
    ("q", torch.zeros(5, 6, 128, dtype=torch.bfloat16)), ("pos", torch.zeros(5)), ("tiles", torch.zeros(2, 3)),
    ("check", torch.zeros(4, dtype=torch.int64)), (None, None)])
def test_prefill_refuses(name, value):
    bt = torch.tensor([[1, 2]], dtype=torch.int32)
    args = dict(q=torch.zeros(5, 4, 128, dtype=torch.bfloat16), cache=_cache(),
                plan=attention.prefill8_plan(bt, [20], 2), pos=torch.zeros(5, dtype=torch.int32),
                tiles=torch.zeros(2, 4, dtype=torch.int32))
    if name:
        args[name] = value
    with pytest.raises(ValueError):
        attention.prefill8(**args)


def test_matvec_refuses():
    w = torch.randn(8, 64)
    x = torch.zeros(1, 64, dtype=torch.bfloat16)
    for qw in (QuantWeights.quantize(w, bits=8, group=32), QuantWeights.quantize(w, bits=4, group=16),
               QuantWeights.quantize(w, bits=4, group=32)):                         # the last: not on a GPU
        with pytest.raises(ValueError):
            qw.matvec(x)


@pytest.mark.parametrize("check", [torch.zeros(4), torch.zeros(3, dtype=torch.int64), torch.zeros(8, dtype=torch.int64)[::2]])
def test_check_takes_a_state_row(check):
    """Check modes write the whole row: anything else is refused before a launch."""
    idx = torch.zeros(1, dtype=torch.int32)
    d, out = _decode_args(), torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    plan = attention.prefill8_plan(torch.tensor([[1]], dtype=torch.int32), [2], 2)
    qw, x = QuantWeights.quantize(torch.randn(8, 64), bits=4, group=32), torch.zeros(1, 64, dtype=torch.bfloat16)
    y = torch.zeros(1, 8, dtype=torch.bfloat16)
    for call in (lambda c: layers.qk_norm_rope_kv8(**_append_args(), rows=idx, check=c),
                 lambda c: attention.decode8(**d, out=out, seq_idx=idx, check=c),
                 lambda c: attention.prefill8(d["q"], d["cache"], plan, d["ctx"], torch.zeros(1, 4, dtype=torch.int32),
                                              out=out, row_idx=idx, check=c),
                 lambda c: qw.matvec(x, out=y, blocks=idx, check=c)):
        with pytest.raises(ValueError, match="state row"):
            call(check)


def test_check_needs_the_output():
    """A check mode without `out` would compare with memory that nothing wrote."""
    idx, st = torch.zeros(1, dtype=torch.int32), torch.zeros(4, dtype=torch.int64)
    d = _decode_args()
    plan = attention.prefill8_plan(torch.tensor([[1]], dtype=torch.int32), [2], 2)
    qw, x = QuantWeights.quantize(torch.randn(8, 64), bits=4, group=32), torch.zeros(1, 64, dtype=torch.bfloat16)
    for call in (lambda: attention.decode8(**d, seq_idx=idx, check=st),
                 lambda: attention.prefill8(d["q"], d["cache"], plan, d["ctx"], torch.zeros(1, 4, dtype=torch.int32),
                                            row_idx=idx, check=st),
                 lambda: qw.matvec(x, blocks=idx, check=st)):
        with pytest.raises(ValueError, match="out"):
            call()


def test_page_transfer_refuses_the_8_bit_cache():
    """Its scales lie apart from the pages' bytes, so hashing or copying the codes alone would be no transfer."""
    from sdcguard_b200.ops import kv_transfer
    c = KV8Cache.empty(3, 1, layers=2, device="cpu")
    for call in (lambda: kv_transfer.page_checksums(c, torch.zeros(1, dtype=torch.int32)),
                 lambda: kv_transfer.page_bytes(c),
                 lambda: kv_transfer.pull_pages(c, c, *[torch.zeros(1, dtype=torch.int32)] * 2,
                                                torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(ValueError, match="KV8Cache"):
            call()
    assert kv_transfer.page_bytes(torch.zeros(2, 3, 2, 1, 16, 128, dtype=torch.bfloat16)) == 2 * 2 * 16 * 128 * 2


@pytest.mark.parametrize("layers_", [1, 7, 28, 32, 36, 64])
@pytest.mark.parametrize("pages", [1, 5, 64, 1000])
def test_replayed_pages_reach_every_page_of_every_layer(layers_, pages):
    from sdcguard_b200.models.decoder import page_offset
    for layer in (0, layers_ - 1):
        seen = {page_offset(1 + step * layers_ + layer, pages) for step in range(64 * 64)}
        assert seen == set(range(min(64, pages)))


def test_want():
    t = torch.zeros(4, 8)
    cpu = torch.device("cpu")
    assert kv8.want(t, torch.float32, (4, 8), cpu, "t") is t
    for bad in (lambda: kv8.want(t.t(), torch.float32, (8, 4), cpu, "t"),
                lambda: kv8.want(t, torch.float32, (8, 4), cpu, "t"),
                lambda: kv8.want(t.view(-1)[1:], torch.float32, (31,), cpu, "t", align=16)):
        with pytest.raises(ValueError):
            bad()


def test_matvec_refuses_an_output_whose_rows_overlap():
    qw = QuantWeights.quantize(torch.randn(8, 64), bits=4, group=32)
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    buf = torch.zeros(64, dtype=torch.bfloat16)
    for out in (buf[:8].expand(3, 8), buf.as_strided((3, 8), (7, 1))):
        with pytest.raises(ValueError, match="rows"):
            qw.matvec(x, out=out)
    with pytest.raises(ValueError, match="CUDA"):                # every other call of these arguments ends at the device
        qw.matvec(x, out=buf.as_strided((3, 8), (8, 1)))
