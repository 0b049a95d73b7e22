"""A checked quantized layer with a decode slot, where the products from the codes do not serve the layer or the call: the
GEMM on the effective weights takes it. Tolerance as in the products' own tests (fp32 sums of K products, one rounding)."""
import pytest
import torch

from sdcguard_b200.ops import gemm
from sdcguard_b200.ops.quant import CheckedQuantLinear, QuantWeights

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _layer(bits=4, group=64, n=512, k=256, scale=0.01):
    g = torch.Generator(device=DEV).manual_seed(bits)
    codes = torch.randint(0, 256, (n, k // 2 if bits == 4 else k), dtype=torch.uint8, device=DEV, generator=g)
    scales = (scale * torch.exp(torch.randn(n, k // group, device=DEV, generator=g))).bfloat16()
    layer = CheckedQuantLinear(QuantWeights(codes, scales, None, bits, group))
    st = gemm.StateTable(DEV, 2)
    return layer, st, st.add("quant (ABFT GEMM)", layer.cw.nb), st.add("quant.decode (replay)", 1)


def _holds(y, x, qw):
    w = qw.reference_weight().to(DEV)
    ref, mag = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    return bool(((y.double() - ref).abs() <= ref.abs() * 2 ** -8 + mag * qw.k * 2.0 ** -23).all())


@pytest.mark.parametrize("form", [dict(bits=8), dict(group=16), dict(scale=2.0 ** 34)])
@pytest.mark.parametrize("m", [1, 5, 32, 33])
def test_layers_that_the_codes_path_does_not_serve(form, m):
    """8-bit codes, groups of 16, scales of 2^27 and more."""
    layer, st, s0, s1 = _layer(**form)
    x = torch.randn(m, 256, device=DEV).bfloat16()
    y = layer(x, st.state, s0, decode_slot=s1)
    assert _holds(y, x, layer.qw)
    rows = st.read()
    assert rows[0]["checks"] > 0 and rows[0]["z"] < 6 and rows[1]["checks"] == 0


@pytest.mark.parametrize("m", [5, 33])
def test_arguments_of_the_gemm_are_refused_at_every_size(m):
    layer, st, s0, s1 = _layer()
    x = torch.randn(m, 256, device=DEV).bfloat16()
    for kw in (dict(inject=(0, 0, 1)), dict(z_alarm=6.0)):
        with pytest.raises(ValueError, match="GEMM"):
            layer(x, st.state, s0, decode_slot=s1, **kw)
    layer(x, st.state, s0, z_alarm=6.0)                   # without a decode slot they are the GEMM's
