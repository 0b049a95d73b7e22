"""Decode attention over the bf16 cache: what a page holds behind its sequence's end reaches no row."""
import pytest
import torch

from sdcguard_b200.ops import attention

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("nq,nkv", [(2, 2), (4, 2), (8, 2), (8, 1)])
@pytest.mark.parametrize("batch", [1, 400])                 # a CTA for each segment, or for a whole row
def test_places_behind_a_sequence_may_hold_anything(nq, nkv, batch):
    lens = [1, 15, 16, 17, 50, 64, 65, 300] * (batch // 8) if batch > 1 else [300]
    g = torch.Generator(device=DEV).manual_seed(nq)
    cache = torch.randn(19 * batch + 1, 2, nkv, 16, 128, device=DEV, generator=g).bfloat16()
    bt = (1 + torch.arange(19 * batch, dtype=torch.int32, device=DEV)).view(batch, 19)
    q = torch.randn(batch, nq, 128, device=DEV, generator=g).bfloat16()
    req = torch.arange(batch, dtype=torch.int32, device=DEV)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def run():
        return attention.decode(q, cache, bt, req, ctx, nq, nkv, max_ctx=512)

    want = run()
    assert torch.isfinite(want).all()
    for b, n in enumerate(lens):
        for page in range(n // 16, 19):
            cache[bt[b, page].long(), :, :, n % 16 if page == n // 16 else 0:] = float("nan")
    assert torch.equal(run(), want)


def test_rows_that_do_not_fit_have_a_norm_of_nan():
    """8-bit cache: a row of NaN adds NaN to its sum of squares, whatever made it NaN; a row without keys adds nothing."""
    from sdcguard_b200.ops.kv8 import KV8Cache
    cache = KV8Cache.empty(8, 1, device=DEV)
    q = torch.randn(5, 2, 128, device=DEV).bfloat16()
    q[4, 1, 0] = float("nan")
    bt = torch.tensor([[1, 2], [3, 4], [5, 99], [6, 7], [6, 7]], dtype=torch.int32, device=DEV)
    req = torch.tensor([0, 9, 2, 3, 4], dtype=torch.int32, device=DEV)
    ctx = torch.tensor([0, 20, 20, 33, 20], dtype=torch.int32, device=DEV)
    sq = torch.zeros(5, device=DEV)
    out = attention.decode8(q, cache, bt, req, ctx, attention.decode8_plan(5, 2, 1, 32, DEV), row_sq=sq)
    assert out.isnan().any(-1).any(-1).tolist() == sq.isnan().tolist() == [False, True, True, True, True] and sq[0] == 0
