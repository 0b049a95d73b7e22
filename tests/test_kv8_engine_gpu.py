"""The serving engine over the 8-bit cache, at sizes whose prefill goes through the expanded pages: against the bf16 engine
(what the first layer stores; with the same stored values, the same bits) and against 64 bits (the decode step), and its
replays."""
import math

import pytest
import torch

from sdcguard_b200.ops import attention, layers
from sdcguard_b200.ops.kv8 import KV8Cache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
LENS = [230, 77, 16, 1, 149]            # 473 tokens of two kv heads
BLOCKS = 96


def _engine(kv_cache, **kw):
    from sdcguard_b200.models.decoder import TINY
    from sdcguard_b200.serve.engine import LLMEngine
    kw.setdefault("cuda_graph", False)
    return LLMEngine(TINY, device="cuda:0", num_blocks=BLOCKS, max_prefill_tokens=512, max_num_seqs=8, max_model_len=512,
                     sample_every=4, kv_cache=kv_cache, **kw)


def _prompts():
    return torch.randint(0, 1024, (len(LENS), max(LENS)), generator=torch.Generator().manual_seed(0))


def _logits(eng):
    """The logits that the engine samples from, call by call."""
    seen, real = [], eng.model.sample

    def sample(x):
        seen.append(x.clone())
        return real(x)

    eng.model.sample = sample
    return seen


def _store_8_bits(monkeypatch):
    """The bf16 engine's append stores what the 8-bit cache would hold: its values are exact in bf16."""
    sides = {}

    def append(qkv, nq, nkv, pos, slots, qn, kn, eps, table, q, lc, rows=None, check=None):
        if check is not None:
            return q
        side = sides.setdefault(lc.data_ptr(), KV8Cache.empty(BLOCKS, nkv, device=DEV))
        layers.qk_norm_rope_kv8(qkv, nq, nkv, pos, slots, qn, kn, eps, table, q, side)
        lc.copy_(side.values())
        return q

    monkeypatch.setattr(layers, "qk_norm_rope_kv", append)


def test_large_prefills_are_the_expanded_ones():
    assert sum(LENS) * 2 > attention.FEW_ROWS


@pytest.mark.parametrize("checked", [True, False])
def test_prefill_is_the_bf16_engines_over_the_stored_values(monkeypatch, checked):
    eng = _engine("fp8", checked=checked)
    got = _logits(eng)
    tokens = eng.generate(_prompts(), LENS, 1)
    scores = eng.score([_prompts()[0].tolist()], topk=1024)
    _store_8_bits(monkeypatch)
    ref = _engine("bf16", checked=checked)
    want = _logits(ref)
    assert torch.equal(ref.generate(_prompts(), LENS, 1), tokens)
    assert len(got) == len(want) == 1 and torch.equal(got[0], want[0])
    for a, b in zip(scores[0], ref.score([_prompts()[0].tolist()], topk=1024)[0]):
        assert torch.equal(a, b)


def test_the_first_layer_stores_the_bf16_engines_keys_and_values():
    """Half a step of E4M3 (2^-4 of the value, 2^-10 of the scale below its normal range); the bf16 engine's keys are rounded
    to bf16 (2^-8) behind the norm, behind its weight and behind the rotation, which adds up the first two of both numbers
    of a pair: at most 2 x 2^-8 of the pair's length. The length is taken from the rounded pair (1.02: its own error and
    products of roundings). Values are not computed with."""
    eng, ref = _engine("fp8"), _engine("bf16")
    eng.generate(_prompts(), LENS, 1)
    ref.generate(_prompts(), LENS, 1)
    a, b = eng.cache[0].values().double(), ref.cache[0].double()
    scale = eng.cache[0].scales.double().transpose(1, 2)[..., None, None]
    place = (b != 0).any(-1).any(1).any(1)                   # (pages, places) that hold tokens
    assert place.sum() == sum(LENS)
    used = place[:, None, None, :, None].expand_as(a)
    pair = torch.hypot(b[..., :64], b[..., 64:]).repeat(1, 1, 1, 1, 2)
    bf16 = 1.02 * 2 ** -8 * (b.abs() + 2 * pair)
    bf16[:, 1] = 0
    tol = b.abs() * 2 ** -4 + bf16 * (1 + 2 ** -4) + scale * 2 ** -10
    assert ((a - b).abs() <= tol)[used].all()


def test_decode_steps_attend_to_what_is_stored(monkeypatch):
    """Each decode step's attention against 64 bits over the cache as it stands: output to bf16, weights to f16, sums and
    scores in fp32 (128 products, each rounded or cut)."""
    real, calls = attention.decode8, []

    def decode8(q, cache, bt, req, ctx, plan, out=None, **kw):
        out = real(q, cache, bt, req, ctx, plan, out=out, **kw)
        if kw.get("check") is None:
            calls.append(ctx.tolist())
            G = q.shape[1] // cache.nkv
            for b, n in enumerate(ctx.tolist()):
                x = cache.values(bt[int(req[b]), :-(-n // 16)].long()).double().permute(1, 2, 0, 3, 4)
                k, v = (t[:, :n].repeat_interleave(G, 0) for t in x.flatten(2, 3))
                qd = q[b].double()[:, :, None]
                w = torch.softmax((k @ qd)[..., 0] * 128 ** -0.5, -1)[:, None]
                ref, mag = (w @ v)[:, 0], (w @ v.abs())[:, 0]
                ds = (k.abs() @ qd.abs()).amax((1, 2))[:, None] * 128 ** -0.5 * 128 * 2.0 ** -23
                tol = ref.abs() * 2 ** -8 + mag * (2 ** -11 + 2 ** -18 + 2 * ds) + 1e-30
                assert ((out[b].double() - ref).abs() <= tol).all()
        return out

    eng = _engine("fp8")
    monkeypatch.setattr(attention, "decode8", decode8)
    eng.generate(_prompts(), LENS, 4)
    assert calls == [[n + s for n in LENS] for s in (1, 2, 3) for _ in range(2)]     # three steps of two layers


def test_replays_of_a_large_prefill_are_clean_and_see_a_flipped_page(monkeypatch):
    """The rows' and the expanded pages' replays on the side stream, while the layers share the expanded pages."""
    eng = _engine("fp8", cuda_graph=True)
    for _ in range(3):
        eng.generate(_prompts(), LENS, 3)
    rows = {r["name"]: r for r in eng.model.read_checks()}
    for i in range(2):
        for op in ("rope_kv", "attn"):
            r = rows[f"layers.{i}.{op} (replay)"]
            assert r["checks"] > 0 and r["z"] == 0, r
    assert all(r["z"] < 6 for r in rows.values())
    real, hit = attention.prefill8, []

    def flipped(q, cache, plan, *a, **kw):
        if kw.get("check") is not None:
            hit.append(1)
            if len(hit) == 2:                                # the second layer's pages, behind their expansion
                plan.work.view(torch.int16)[:] ^= 1
        return real(q, cache, plan, *a, **kw)

    monkeypatch.setattr(attention, "prefill8", flipped)
    eng.generate(_prompts(), LENS, 1)
    z = {r["name"]: r["z"] for r in eng.model.read_checks()}
    assert len(hit) == 2 and z["layers.0.attn (replay)"] == 0 and z["layers.1.attn (replay)"] == math.inf


def test_pages_used_before_do_not_change_a_prefill():
    """Pages of a request that stored NaN serve another one: the places behind its end still hold them."""
    eng = _engine("fp8")
    want = eng.score([_prompts()[0, :201].tolist()], topk=5)
    eng.cache.codes.view(torch.uint8).fill_(0x7F)
    got = eng.score([_prompts()[0, :201].tolist()], topk=5)
    assert all(torch.equal(a, b) for a, b in zip(want[0], got[0]))


def test_engine_refuses_an_8_bit_cache_it_was_not_asked_for():
    from sdcguard_b200.models.decoder import TINY
    from sdcguard_b200.serve.engine import LLMEngine
    with pytest.raises(ValueError, match="bf16"):
        LLMEngine(TINY, device="cuda:0", max_num_seqs=8, cache=KV8Cache.empty(8, 2, 2, DEV))
