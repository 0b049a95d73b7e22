"""Products of a few rows with 4-bit weights, read as codes: against float64 products with the effective weights, and
the exact replay of sampled outputs. Tolerance: one rounding to bf16 (2^-8 of the value) and K fp32 sums, each rounded or
cut (2^-23 of sum |x w| each)."""
import math

import pytest
import torch

from sdcguard_b200.ops import gemm
from sdcguard_b200.ops.quant import CheckedQuantLinear, QuantWeights

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _weights(n, k, group, zeros, mode="subtract", seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV, generator=g)
    scales = (0.01 * torch.exp(torch.randn(n, k // group, device=DEV, generator=g))).bfloat16()
    z = torch.randint(0, 16, (n, k // group), dtype=torch.uint8, device=DEV, generator=g) if zeros else None
    return QuantWeights(codes, scales, z, 4, group, zero_mode=mode)


def _holds(y, x, qw, bias=None):
    w = qw.reference_weight().to(x.device)
    ref = x.double() @ w.t() + (0 if bias is None else bias.double())
    mag = x.double().abs() @ w.abs().t() + (0 if bias is None else bias.double().abs())
    return bool(((y.double() - ref).abs() <= ref.abs() * 2 ** -8 + mag * qw.k * 2.0 ** -23).all())


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 31, 32])
@pytest.mark.parametrize("n,k,group,zeros", [(1, 32, 32, False), (17, 96, 32, True), (1000, 1024, 128, True),
                                             (64, 4128, 96, False), (33, 2112, 64, True), (130, 256, 256, False)])
def test_matvec_matches_64_bits(m, n, k, group, zeros):
    qw = _weights(n, k, group, zeros, seed=m)
    x = torch.randn(m, k, device=DEV).bfloat16()
    y = qw.matvec(x)
    assert _holds(y, x, qw)
    assert torch.equal(qw.matvec(x[:1]), y[:1])         # a row's bits do not depend on the rows beside it


@pytest.mark.parametrize("mode", ["subtract", "fma", "two_roundings"])
def test_matvec_multiplies_by_the_effective_weights_bit_for_bit(mode):
    qw = _weights(70, 128, 64, True, mode)
    eye = torch.eye(128, device=DEV).bfloat16()
    got = torch.cat([qw.matvec(eye[i:i + 32]) for i in range(0, 128, 32)])
    assert torch.equal(got.t().double(), qw.reference_weight().to(DEV))


def test_matvec_strides_bias_empty_and_values_that_are_not_finite():
    qw = _weights(100, 256, 32, True)
    buf = torch.randn(5, 300, device=DEV).bfloat16()
    x = buf[:, 8:264]
    bias = torch.randn(100, device=DEV)
    wide = torch.full((5, 128), 7.0, device=DEV).bfloat16()
    y = qw.matvec(buf.new_zeros(5, 304)[:, :256].copy_(x), bias, out=wide[:, 9:109])
    assert _holds(y, x, qw, bias) and (wide[:, :9] == 7).all() and (wide[:, 109:] == 7).all()
    assert qw.matvec(torch.empty(0, 256, dtype=torch.bfloat16, device=DEV)).shape == (0, 100)
    x = torch.randn(3, 256, device=DEV).bfloat16()
    want = qw.matvec(x)
    x[1, 7] = float("nan")
    y = qw.matvec(x)
    assert y[1].isnan().all() and torch.equal(y[[0, 2]], want[[0, 2]])
    x[1, 7] = float("inf")
    y, w = qw.matvec(x), qw.reference_weight()[:, 7].to(DEV)
    assert torch.equal(y[1].isnan(), w == 0) and (y[1][w > 0] == math.inf).all() and (y[1][w < 0] == -math.inf).all()


def test_matvec_replay_and_stream():
    from sdcguard_b200.numerics import abft
    qw = _weights(200, 512, 128, True)
    for m in (3, 12, 30):
        x = torch.randn(m, 512, device=DEV).bfloat16()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y = qw.matvec(x)
        torch.cuda.current_stream().wait_stream(s)
        st = torch.zeros(2, 4, dtype=torch.int64, device=DEV)
        blocks = torch.tensor([12, 0, 5], dtype=torch.int32, device=DEV)
        qw.matvec(x, out=y, blocks=blocks, check=st[0])
        y.view(torch.int16)[m - 1, 199] ^= 1
        qw.matvec(x, out=y, blocks=blocks, check=st[1])
        a, b = (abft.decode_state_row(r) for r in st.cpu().tolist())
        assert a["z"] == 0 and a["checks"] == 1
        assert b["z"] == math.inf and b["flat"] == (m - 1) * 200 + 199 and b["checks"] == 1


def test_checked_layer_reads_the_codes_in_small_batches():
    qw = _weights(2000, 256, 64, True)
    bias = torch.randn(2000, device=DEV)
    layer = CheckedQuantLinear(qw, bias)
    st = gemm.StateTable(DEV, 2)
    s0, s1 = st.add("quant (ABFT GEMM)", layer.cw.nb), st.add("quant.decode (replay)", 1)
    x = torch.randn(40, 256, device=DEV).bfloat16()
    for _ in range(70):                                   # more turns than there are samples
        y = layer(x[:5], st.state, s0, decode_slot=s1)
    assert _holds(y, x[:5], qw, bias) and torch.equal(y, qw.matvec(x[:5], bias))
    rows = st.read()
    assert rows[0]["checks"] == 0 and rows[1]["checks"] == 70 and rows[1]["z"] == 0
    big = layer(x, st.state, s0, decode_slot=s1)          # more rows than matvec takes: the checked GEMM
    assert st.read()[0]["checks"] > 0 and _holds(big, x, qw, bias)
    with pytest.raises(ValueError):
        layer(x[:5], st.state, s0, decode_slot=s1, inject=(0, 0, 1))


def test_checked_layer_captured_at_its_first_call():
    """A graph holds the layer and its replay check; the recomputed outputs rotate with the graph's replays."""
    qw = _weights(2000, 256, 64, True)
    layer = CheckedQuantLinear(qw)
    st = gemm.StateTable(DEV, 2)
    s0, s1 = st.add("quant (ABFT GEMM)", layer.cw.nb), st.add("quant.decode (replay)", 1)
    x = torch.randn(3, 256, device=DEV).bfloat16()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer(x, st.state, s0, decode_slot=s1)
    seen = set()
    for i in range(64):
        x.copy_(torch.randn(3, 256, device=DEV))
        g.replay()
        assert torch.equal(y, qw.matvec(x))
        seen |= set(layer._sampled.tolist())
    assert seen >= set(range(125))                        # all blocks of 16 outputs
    row = st.read()[1]
    assert row["checks"] == 64 and row["z"] == 0


@pytest.mark.parametrize("m", [1, 8, 13, 16, 27, 32])
@pytest.mark.parametrize("n,k,group,zeros", [(40, 8224, 32, True), (2400, 8192, 128, False), (2049, 8224, 32, True),
                                             (4752, 8192, 64, False)])
def test_matvec_long_products(m, n, k, group, zeros):
    """More warps take the products of a long k: 64 bits, the same bits in every batch and in the replay."""
    qw = _weights(n, k, group, zeros, seed=m)
    x = torch.randn(m, k, device=DEV).bfloat16()
    y = qw.matvec(x)
    assert _holds(y, x, qw)
    assert torch.equal(qw.matvec(x[:1]), y[:1]) and torch.equal(qw.matvec(x[m - 1:]), y[m - 1:])
    st = torch.zeros(4, dtype=torch.int64, device=DEV)
    qw.matvec(x, out=y, blocks=torch.arange(-(-n // 16), dtype=torch.int32, device=DEV), check=st)
    assert st.tolist()[2] == 1 and st.tolist()[0] == 0
