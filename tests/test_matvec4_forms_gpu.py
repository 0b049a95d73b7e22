"""Every form of the 4-bit products: wide and narrow tiles, packed and unpacked x, 8 and 16 warps, all readings of the zero
points; against float64 products with the effective weights, with the same bits in every batch and in the replay.
Tolerance: one rounding to bf16 (2^-8 of the value) and K fp32 sums, each rounded or cut (2^-23 of sum |x w| each)."""
import pytest
import torch

from sdcguard_b200.ops.quant import QuantWeights

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
READINGS = ["eight", "subtract", "fma", "two_roundings"]


def _weights(n, k, group, reading, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV, generator=g)
    scales = (0.01 * torch.exp(torch.randn(n, k // group, device=DEV, generator=g))).bfloat16()
    z = None if reading == "eight" else torch.randint(0, 16, (n, k // group), dtype=torch.uint8, device=DEV, generator=g)
    return QuantWeights(codes, scales, z, 4, group, zero_mode="subtract" if reading == "eight" else reading)


def _effective(qw):
    """W as float64: the reading's roundings, the products before them exact."""
    def spread(t):
        return t.double().repeat_interleave(qw.group, 1)

    q = torch.stack([qw.codes & 15, qw.codes >> 4], -1).flatten(1).double()
    s = spread(qw.scales)
    if qw.zeros is None or qw.zero_mode == "subtract":
        return ((q - (8 if qw.zeros is None else spread(qw.zeros))) * s).bfloat16().double()
    zs = -spread((qw.scales.double() * qw.zeros.double()).bfloat16())
    qs = (q * s).bfloat16().double() if qw.zero_mode == "two_roundings" else q * s
    return (qs + zs).bfloat16().double()


def _holds(y, x, w, k):
    ref, mag = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    return bool(((y.double() - ref).abs() <= ref.abs() * 2 ** -8 + mag * k * 2.0 ** -23).all())


@pytest.mark.parametrize("reading", READINGS)
@pytest.mark.parametrize("n,k,group", [
    (8200, 2080, 32),        # wide, packed (n k above 2^24)
    (8193, 1056, 96),        # wide, x as it is; the last k block is short
    (4800, 4128, 32),        # one group of 16 outputs a warp, packed
    (4740, 8224, 32),        # above the sizes that take 16 warps
    (2401, 8224, 257 * 32),  # 16 warps, one group a row
    (2000, 8448, 96),        # 16 warps, packed
    (300, 8224, 32)])        # 16 warps, x as it is
def test_every_form(n, k, group, reading):
    qw = _weights(n, k, group, reading, seed=n)
    w = _effective(qw)
    x = torch.randn(32, k, device=DEV).bfloat16()
    blocks = torch.arange(-(-n // 16), dtype=torch.int32, device=DEV)
    first = qw.matvec(x[:1])
    for m in (1, 8, 9, 13, 16, 17, 32):
        y = qw.matvec(x[:m])
        assert _holds(y, x[:m], w, k), m
        assert torch.equal(y[:1], first), m
        st = torch.zeros(4, dtype=torch.int64, device=DEV)
        qw.matvec(x[:m], out=y, blocks=blocks, check=st)
        assert st.tolist()[2] == 1 and st.tolist()[0] == 0, m
    assert torch.equal(qw.matvec(x[31:]), y[31:])


@pytest.mark.parametrize("reading", READINGS)
def test_wide_and_packed_products_multiply_by_the_effective_weights_bit_for_bit(reading):
    qw = _weights(8200, 2080, 32, reading)
    w = _effective(qw)
    for lo in (0, 31, 1000, 2048):
        eye = torch.eye(2080, device=DEV).bfloat16()[lo:lo + 32]
        for m in (1, 16, 32):
            assert torch.equal(qw.matvec(eye[:m]).double(), w.t()[lo:lo + m])
