"""The 8-bit KV cache: append (norm, rotation, page scales), decode and prefill over it, against the formulas in 64
bits, and their exact replays. Tolerances are sums of the roundings that the kernels make (half a step each: bf16 2^-8
of the value, E4M3 2^-4, f16 2^-11, fp32 2^-24)."""
import math

import pytest
import torch

from sdcguard_b200.ops import attention, kv8, layers
from sdcguard_b200.ops.kv8 import KV8Cache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
NAN = float("nan")


def _state(n=1):
    return torch.zeros(n, 4, dtype=torch.int64, device=DEV)


def _flat(row):
    from sdcguard_b200.numerics import abft
    d = abft.decode_state_row(row.cpu().tolist())
    return d["z"], d["flat"], d["checks"]


def _scale64(amax):
    s = torch.exp2(torch.ceil(torch.log2((amax / 448).clamp_min(2.0 ** -70))))
    s = torch.where(s * 448 < amax, s * 2, torch.where(s * 224 >= amax, s / 2, s))
    return s.clamp_min(2.0 ** -60)


def _rand_cache(blocks, nkv, seed=0, spread=3.0):
    """Random values whose size differs from page to page by up to 2^(2 spread)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    v = torch.randn(blocks, 2, nkv, 16, 128, device=DEV, generator=g)
    v *= torch.exp2(spread * (2 * torch.rand(blocks, 2, nkv, 1, 1, device=DEV, generator=g) - 1))
    s = _scale64(v.double().abs().amax((-1, -2)))
    return KV8Cache((v / s[..., None, None].float()).to(torch.float8_e4m3fn), s.float().transpose(1, 2).contiguous())


# ------------------------------------------------------------------------------------------------ append
def _append_ref(qkv, nq, nkv, pos, qn, kn, eps, table, interleaved):
    """(q, kv (T, 2, nkv, 128)) in float64."""
    t = qkv.shape[0]
    x = qkv.double().reshape(t, nq + 2 * nkv, 128).clone()
    for lo, hi, w in ((0, nq, qn), (nq, nq + nkv, kn)):
        if w is not None:
            h = x[:, lo:hi]
            x[:, lo:hi] = h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if table is not None:
        half = table.shape[1]
        c, s = (table.double()[pos.long()][:, None, :, i] for i in (0, 1))
        h = x[:, :nq + nkv]
        a, b = (h[..., 0:2 * half:2], h[..., 1:2 * half:2]) if interleaved else (h[..., :half], h[..., half:2 * half])
        ra, rb = a * c - b * s, b * c + a * s
        if interleaved:
            x[:, :nq + nkv, 0:2 * half:2], x[:, :nq + nkv, 1:2 * half:2] = ra, rb
        else:
            x[:, :nq + nkv, :half], x[:, :nq + nkv, half:2 * half] = ra, rb
    return x[:, :nq], torch.stack([x[:, nq:nq + nkv], x[:, nq + nkv:]], 1)


def _check_append(before, cache, slots, kv):
    """The cache after an append of kv at slots, given what it was before: scales, new codes, kept and other codes."""
    old_v, old_s = before
    page, off = slots // 16, slots % 16
    live = slots >= 0
    want_s = old_s.double().clone()
    untouched = torch.ones(cache.num_blocks, 16, dtype=torch.bool, device=DEV)
    for pg in page[live].unique().tolist():
        sel = (page == pg) & live
        first = int(off[sel].min())
        need = _scale64(kv[sel].abs().amax((0, 3)))                                   # 2, nkv
        had = old_s[pg].double().t() if first else torch.zeros_like(need)
        want_s[pg] = torch.maximum(need, had).t()
        untouched[pg, :first] = False
        untouched[pg, off[sel]] = False
    assert torch.equal(cache.scales.double(), want_s)
    s5 = cache.scales.double().transpose(1, 2)[..., None, None]
    now = cache.codes.double() * s5
    # new tokens: one rounding to E4M3 (half a step: 2^-4 of the value, 2^-10 of the scale below the normal range), and
    # the fp32 arithmetic before it (norm and rotation: under 16 roundings of the row's largest)
    got = now[page[live], :, :, off[live]]
    ref = kv[live]
    s4 = s5[page[live], :, :, 0]
    tol = torch.maximum(ref.abs() * 2 ** -4, s4 * 2 ** -10) + ref.abs().amax(-1, keepdim=True) * 2 ** -19
    assert ((got - ref).abs() <= tol).all()
    # kept tokens: one rounding at the new scale
    for pg in page[live].unique().tolist():
        first = int(off[(page == pg) & live].min())
        if first:
            d = (now[pg, :, :, :first] - old_v[pg, :, :, :first]).abs()
            assert (d <= torch.maximum(old_v[pg, :, :, :first].abs() * 2 ** -4, s5[pg] * 2 ** -10)).all()
            same = (cache.scales[pg] == old_s[pg]).t()[..., None, None]
            assert (torch.where(same, d, 0) == 0).all()
    return untouched


def _run_append(nq, nkv, slots, pos, norm=True, rotary=128, interleaved=False, seed=0, blocks=None, size=1.0, ld=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = len(slots)
    slots = torch.tensor(slots, dtype=torch.int64, device=DEV)
    pos = torch.tensor(pos, dtype=torch.int32, device=DEV)
    blocks = blocks or int(slots.max()) // 16 + 2
    cache = _rand_cache(blocks, nkv, seed + 1)
    width = (nq + 2 * nkv) * 128
    buf = torch.randn(t, ld or width, device=DEV, generator=g).mul_(size).bfloat16()
    qkv = buf[:, (ld or width) - width:]
    qn, kn = ((1 + 0.3 * torch.randn(128, device=DEV, generator=g)).bfloat16() if norm else None for _ in range(2))
    table = layers.rope_table(int(pos.max()) + 1, rotary, 10000.0, device=DEV) if rotary else None
    q = torch.full((t, nq, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    before = (cache.values().double(), cache.scales.clone())
    raw = cache.codes.view(torch.uint8).clone()
    args = (qkv, nq, nkv, pos, slots, qn, kn, 1e-6, table, q, cache)
    layers.qk_norm_rope_kv8(*args, interleaved=interleaved)
    rq, kv = _append_ref(qkv, nq, nkv, pos, qn, kn, 1e-6, table, interleaved)
    assert ((q.double() - rq).abs() <= rq.abs() * 2 ** -8 + rq.abs().amax(-1, keepdim=True) * 2 ** -19).all()
    untouched = _check_append(before, cache, slots, kv)
    m = untouched[:, None, None, :, None].expand_as(raw)
    assert torch.equal(cache.codes.view(torch.uint8)[m], raw[m])
    return args, cache


@pytest.mark.parametrize("nq,nkv,norm,rotary,interleaved", [
    (16, 8, True, 128, False), (4, 1, False, 128, True), (3, 3, True, 64, False), (10, 2, False, 40, True),
    (2, 1, True, 8, False), (32, 8, False, 0, False)])
@pytest.mark.parametrize("tokens,start", [(1, 0), (1, 5), (1, 31), (16, 0), (37, 9), (1030, 3)])
def test_append_one_sequence(nq, nkv, norm, rotary, interleaved, tokens, start):
    perm = torch.randperm(start // 16 + tokens // 16 + 2, generator=torch.Generator().manual_seed(tokens)).tolist()
    pos = list(range(start, start + tokens))
    _run_append(nq, nkv, [perm[p // 16] * 16 + p % 16 for p in pos], pos, norm, rotary, interleaved, seed=tokens)


def test_append_batch_of_sequences_padding_and_strided_rows():
    """Sequences at their own places, rows without a slot between and behind them, a projection inside a wider buffer."""
    lens, starts, pages = [1, 40, 16, 3, 1], [7, 13, 0, 30, 15], [[4], [9, 1, 7, 3], [2], [11, 5], [8]]
    slots, pos = [], []
    for n, s, pg in zip(lens, starts, pages):
        slots += [pg[(s + i) // 16 - s // 16] * 16 + (s + i) % 16 for i in range(n)] + [-1]
        pos += [s + i for i in range(n)] + [0]
    _run_append(6, 2, slots + [-1] * 3, pos + [0] * 3, blocks=13, ld=10 * 128 + 24)
    _run_append(6, 2, slots * 1 + [-1] * 1100, pos + [0] * 1100, blocks=13, ld=10 * 128 + 24)     # long: grouped rows
    _run_append(2, 1, [-1], [3], blocks=2)


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_does_not_depend_on_how_tokens_are_grouped(interleaved):
    """How many tokens a warp looks at follows from the call's length: runs that start at every place of such a group and
    reach over its end, between rows without a slot, give the same bits in calls of 500 to 2100 rows."""
    g = torch.Generator().manual_seed(5)
    slots, pos, page = [], [], 0
    while len(slots) < 450:
        n, start = int(torch.randint(1, 24, (1,), generator=g)), int(torch.randint(0, 16, (1,), generator=g))
        slots += [page * 16 + start + i for i in range(n)] + [-1] * int(torch.randint(0, 3, (1,), generator=g))
        pos += [start + i for i in range(n)] + [0] * (len(slots) - len(pos) - n)
        page += (start + n) // 16 + 1
    used, got = len(slots), []
    for pad in (500, 511, 512, 2047, 2048, 2100):          # against 64 bits
        (qkv, _, _, _, _, qn, kn, eps, table, _, _), _ = _run_append(
            6, 2, slots + [-1] * (pad - used), pos + [0] * (pad - used), interleaved=interleaved, seed=3, blocks=page + 1)
    slots = torch.tensor(slots + [-1] * (2100 - used), dtype=torch.int64, device=DEV)
    pos = torch.tensor(pos + [0] * (2100 - used), dtype=torch.int32, device=DEV)
    for pad in (500, 511, 512, 2047, 2048, 2100):          # the same rows in each call
        cache, q = _rand_cache(page + 1, 2, 4), torch.zeros(pad, 6, 128, dtype=torch.bfloat16, device=DEV)
        layers.qk_norm_rope_kv8(qkv[:pad], 6, 2, pos[:pad], slots[:pad], qn, kn, eps, table, q, cache, interleaved=interleaved)
        got.append((cache.codes.view(torch.uint8), cache.scales, q[:used]))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


@pytest.mark.parametrize("size", [2.0 ** -90, 2.0 ** -20, 300.0, 2.0 ** 60])
def test_append_small_and_large_values(size):
    _run_append(2, 2, [5 + 16 * 3 + i for i in range(9)], list(range(5, 14)), norm=False, size=size)


def test_append_scale_edges_and_values_that_are_not_finite():
    """amax of exactly 448 s keeps s; the next bf16 value doubles it. NaN and infinities are stored as NaN, each in its
    own place, and raise no scale."""
    v = torch.zeros(4, 3, 128, device=DEV)
    v[0, 2, 3] = 448.0
    v[1, 2, 5] = 450.0
    v[2, 2, 0], v[2, 2, 1], v[2, 2, 2], v[2, 2, 127] = 1.0, float("inf"), -float("inf"), NAN
    v[3, 1, 9], v[3, 2, 77] = -56.0, 0.0
    cache = KV8Cache.empty(5, 1, device=DEV)
    q = torch.empty(4, 1, 128, dtype=torch.bfloat16, device=DEV)
    pos = torch.zeros(4, dtype=torch.int32, device=DEV)
    slots = torch.tensor([16, 32, 48, 64], device=DEV)
    layers.qk_norm_rope_kv8(v.bfloat16().view(4, -1), 1, 1, pos, slots, None, None, 1e-6, None, q, cache)
    assert cache.scales[1, 0].tolist() == [2.0 ** -60, 1.0] and cache.scales[2, 0].tolist() == [2.0 ** -60, 2.0]
    assert cache.scales[3, 0, 1] == 2.0 ** -8 and cache.scales[4, 0].tolist() == [0.125, 2.0 ** -60]
    x = cache.values()
    assert x[1, 1, 0, 0, 3] == 448 and x[2, 1, 0, 0, 5] == 448         # 450 / 2 = 225 lies between 224 and 240
    assert x[3, 1, 0, 0].isnan().nonzero().flatten().tolist() == [1, 2, 127] and x[3, 1, 0, 0, 0] == 1
    # a page with a NaN keeps it when its scale grows, and its other tokens stay
    w = torch.full((1, 3, 128), 1000.0, device=DEV)
    layers.qk_norm_rope_kv8(w.bfloat16().view(1, -1), 1, 1, pos[:1], torch.tensor([49], device=DEV), None, None, 1e-6,
                            None, q[:1], cache)
    x = cache.values()
    assert cache.scales[3, 0, 1] == 4.0 and x[3, 1, 0, 0].isnan().nonzero().flatten().tolist() == [1, 2, 127]
    assert x[3, 1, 0, 0, 0] == 1 and (x[3, 1, 0, 1] - 1000).abs().max() <= 1000 * 2 ** -4


def test_append_outside_the_cache_or_the_table():
    """A slot or position outside gives a NaN row of q and stores nothing; the other rows are as ever."""
    cache = _rand_cache(4, 2)
    raw, scales = cache.codes.view(torch.uint8).clone(), cache.scales.clone()
    qkv = torch.randn(5, 6 * 128, device=DEV).bfloat16()
    q = torch.zeros(5, 2, 128, dtype=torch.bfloat16, device=DEV)
    table = layers.rope_table(8, 128, 10000.0, device=DEV)
    pos = torch.tensor([0, 8, -1, 7, 1], dtype=torch.int32, device=DEV)
    slots = torch.tensor([64, 17, 33, 50, 1 << 40], device=DEV)
    layers.qk_norm_rope_kv8(qkv, 2, 2, pos, slots, None, None, 1e-6, table, q, cache)
    assert q.isnan().all(-1).all(-1).tolist() == [True, True, True, False, True] and not q[3].isnan().any()
    assert torch.equal(cache.codes.view(torch.uint8)[:3], raw[:3]) and torch.equal(cache.scales[:3], scales[:3])
    assert not torch.equal(cache.codes.view(torch.uint8)[3], raw[3])


def test_append_one_by_one_and_at_once():
    """A prompt appended token by token ends at the same scales; its codes differ by the rounding of each move only
    where values lie below the normal range of the last scale."""
    g = torch.Generator(device=DEV).manual_seed(5)
    qkv = (torch.randn(50, 4 * 128, device=DEV, generator=g) * torch.logspace(-2, 2, 50, device=DEV)[:, None]).bfloat16()
    pos = torch.arange(50, dtype=torch.int32, device=DEV)
    slots = pos.long() + 16
    table = layers.rope_table(50, 128, 10000.0, device=DEV)
    a, b = KV8Cache.empty(5, 1, device=DEV), KV8Cache.empty(5, 1, device=DEV)
    q = torch.empty(50, 2, 128, dtype=torch.bfloat16, device=DEV)
    layers.qk_norm_rope_kv8(qkv, 2, 1, pos, slots, None, None, 1e-6, table, q, a)
    q1 = torch.empty_like(q)
    for i in range(50):
        layers.qk_norm_rope_kv8(qkv[i:i + 1], 2, 1, pos[i:i + 1], slots[i:i + 1], None, None, 1e-6, table,
                                q1[i:i + 1], b)
    assert torch.equal(q, q1) and torch.equal(a.scales, b.scales)
    x, y = a.values().double(), b.values().double()
    s = a.scales.double().transpose(1, 2)[..., None, None]
    assert torch.equal(x[x.abs() >= 2 ** -5 * s.expand_as(x)], y[x.abs() >= 2 ** -5 * s.expand_as(x)])
    assert ((x - y).abs() <= s * 2 ** -9).all()        # below: a step at most, half a step for each of two roundings


def test_append_check_mode():
    args, cache = _run_append(4, 2, [21 + i for i in range(30)], list(range(5, 35)))
    st = _state(6)
    rows = torch.tensor([0, 11, 29], dtype=torch.int32, device=DEV)
    layers.qk_norm_rope_kv8(*args, rows=rows, check=st[0])
    q, codes = args[9], cache.codes.view(torch.uint8)
    q.view(torch.int16)[11, 3, 100] ^= 1
    layers.qk_norm_rope_kv8(*args, rows=rows, check=st[1])
    q.view(torch.int16)[11, 3, 100] ^= 1
    codes[(21 + 29) // 16, 1, 1, (21 + 29) % 16, 64] ^= 8
    layers.qk_norm_rope_kv8(*args, rows=rows, check=st[2])
    codes[(21 + 29) // 16, 1, 1, (21 + 29) % 16, 64] ^= 8
    cache.scales[(21 + 11) // 16, 0, 0] /= 4
    layers.qk_norm_rope_kv8(*args, rows=rows, check=st[3])
    cache.scales[(21 + 11) // 16, 0, 0] *= 4
    layers.qk_norm_rope_kv8(*args, rows=rows, check=st[4])
    assert _flat(st[0]) [::2] == (0, 1) and _flat(st[4])[::2] == (0, 1)
    assert _flat(st[1]) == (math.inf, (11 * 8 + 3) * 128 + 100, 1)
    assert _flat(st[2]) == (math.inf, (29 * 8 + 7) * 128 + 64, 1)
    z, flat, _ = _flat(st[3])
    assert z == math.inf and flat // 128 == 11 * 8 + 4


# ------------------------------------------------------------------------------------------------ decode
def _attend64(q, k, v, scale=128 ** -0.5):
    """One query row of one head in float64: output and sum of the weighted magnitudes."""
    w = torch.softmax((k @ q) * scale, 0)
    return w @ v, w @ v.abs()


def _decode_case(ctxs, nq, nkv, seed=0, spread=3.0, max_ctx=None, extra_pages=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // 16) for n in ctxs]
    blocks = sum(need) + 2
    cache = _rand_cache(blocks, nkv, seed + 1, spread)
    perm = (torch.randperm(blocks - 1, generator=torch.Generator().manual_seed(seed)) + 1).tolist()
    bt = torch.zeros(len(ctxs), max(max(need), 1) + extra_pages, dtype=torch.int32)
    o = 0
    for r, n in enumerate(need):
        bt[r, :n] = torch.tensor(perm[o:o + n], dtype=torch.int32)
        o += n
    q = torch.randn(len(ctxs), nq, 128, device=DEV, generator=g).bfloat16()
    plan = attention.decode8_plan(len(ctxs), nq, nkv, max_ctx or max(max(ctxs), 1), DEV)
    return (q, cache, bt.to(DEV), torch.arange(len(ctxs), dtype=torch.int32, device=DEV),
            torch.tensor(ctxs, dtype=torch.int32, device=DEV), plan)


def _check_decode(args, out, rows=None):
    """|out - ref| <= bf16 rounding of the output + sum_j p_j |v_j| times (f16 rounding of the weights 2^-11, the ex2 and
    fp32 sums of the weights 2^-18, and the error of the scores: 128 products in fp32, each rounded or cut, so at most
    128 * 2^-23 of sum |q k| scale, in the exponent of weight and of the sum)."""
    q, cache, bt, req, ctx, _ = args
    nkv, G = cache.nkv, q.shape[1] // cache.nkv
    for b in (range(q.shape[0]) if rows is None else rows):
        n = int(ctx[b])
        if n == 0:
            assert (out[b] == 0).all()
            continue
        x = cache.values(bt[int(req[b]), :-(-n // 16)].long()).double().permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n]
        for h in range(q.shape[1]):
            k, v, qd = x[0, h // G], x[1, h // G], q[b, h].double()
            ref, mag = _attend64(qd, k, v)
            ds = float((k.abs() @ qd.abs()).max()) * 128 ** -0.5 * 128 * 2.0 ** -23
            tol = ref.abs() * 2 ** -8 + mag * (2 ** -11 + 2 ** -18 + 2 * ds) + 1e-30
            assert ((out[b, h].double() - ref).abs() <= tol).all(), (b, h, n)


@pytest.mark.parametrize("nq,nkv", [(16, 8), (32, 8), (4, 1), (8, 8), (3, 1), (10, 2), (7, 1), (8, 1), (9, 1), (16, 1),
                                    (28, 2)])
def test_decode_matches_64_bits_and_replays_exactly(nq, nkv):
    args = _decode_case([1, 0, 15, 16, 17, 64, 65, 300, 1029], nq, nkv, seed=nq)
    rs = torch.zeros(9, device=DEV)
    out = attention.decode8(*args, row_sq=rs)
    _check_decode(args, out)
    assert torch.allclose(rs, out.float().square().sum((1, 2)), rtol=2e-5)
    idx = torch.tensor([8, 0, 4], dtype=torch.int32, device=DEV)
    again = torch.full_like(out, 3.0)
    attention.decode8(*args, out=again, seq_idx=idx)
    assert torch.equal(again[idx.long()], out[idx.long()])
    rest = [i for i in range(9) if i not in (8, 0, 4)]
    assert (again[rest] == 3).all()
    st = _state(2)
    attention.decode8(*args, out=out, seq_idx=idx, check=st[0])
    out.view(torch.int16)[8, nq - 1, 77] ^= 1
    attention.decode8(*args, out=out, seq_idx=idx, check=st[1])
    assert _flat(st[0])[::2] == (0, 1) and _flat(st[1]) == (math.inf, (8 * nq + nq - 1) * 128 + 77, 1)


@pytest.mark.parametrize("seqs,ctx,nq,nkv,segs", [(16, 1200, 8, 8, 4), (98, 3200, 8, 4, 2), (40, 1600, 8, 8, 3)])
def test_decode_few_segments_of_many_rows(seqs, ctx, nq, nkv, segs):
    """Rows that end before, in and at the end of a segment (the last one shorter), each as if it were alone."""
    seg = attention.decode8_cut(seqs, nkv, ctx)[0] * 16
    assert attention.decode8_cut(seqs, nkv, ctx)[1] == segs
    ends = [ctx, seg - 1, seg, seg + 1, seg * (segs - 1), seg * (segs - 1) + 1, 0, 1]
    ctxs = (ends + [1 + (i * 7919) % ctx for i in range(seqs)])[:seqs]
    args = _decode_case(ctxs, nq, nkv, seed=ctx)
    out = attention.decode8(*args)
    _check_decode(args, out, rows=range(8))
    pick = torch.tensor([seqs - 1, 5, 3, 0], dtype=torch.int32, device=DEV)
    again = torch.empty_like(out)
    attention.decode8(*args, out=again, seq_idx=pick)
    assert torch.equal(again[pick.long()], out[pick.long()])


@pytest.mark.parametrize("seqs,ctx,nq,nkv", [(1, 4097, 8, 2), (2, 20000, 4, 1), (40, 700, 8, 8), (300, 90, 4, 2)])
def test_decode_cut_of_the_keys(seqs, ctx, nq, nkv):
    """Batches that are cut into one, few and many segments; a row's bits do not depend on the rows around it."""
    ctxs = [ctx] + [1 + (i * 7919) % ctx for i in range(1, seqs)]
    args = _decode_case(ctxs, nq, nkv, seed=ctx)
    out = attention.decode8(*args)
    _check_decode(args, out, rows=range(min(seqs, 6)))
    pick = torch.tensor([seqs - 1, 0], dtype=torch.int32, device=DEV)
    again = torch.empty_like(out)
    attention.decode8(*args, out=again, seq_idx=pick)
    assert torch.equal(again[pick.long()], out[pick.long()])


@pytest.mark.parametrize("spread", [0.0, 20.0, 40.0])
def test_decode_pages_of_very_different_scales(spread):
    args = _decode_case([200, 1029], 4, 2, seed=9, spread=spread)
    if spread:
        # K alike on all pages (or one page takes all the weight), V as it is
        args[1].scales[:, :, 0] = 2.0 ** -8
    _check_decode(args, attention.decode8(*args))


@pytest.mark.parametrize("size", [2.0 ** -120, 1e-6, 8.0, 1e4, 1e30])
def test_decode_small_and_large_queries(size):
    args = _decode_case([100, 333], 8, 2, seed=4, spread=0.0)
    args[0].mul_(size)
    _check_decode(args, attention.decode8(*args))


def test_decode_masked_places_may_hold_anything():
    """NaN codes and scales behind the end of a sequence reach no result; inside it they give NaN where they must."""
    args = _decode_case([21, 40, 64], 4, 2, seed=6)
    q, cache, bt, req, ctx, plan = args
    want = attention.decode8(*args)
    codes = cache.codes.view(torch.uint8)
    codes[bt[0, 1].long(), :, :, 5:] = 0x7F
    codes[bt[1, 2].long(), :, :, 8:] = 0xFF
    cache.scales[0] = NAN
    codes[0] = 0x7F
    assert torch.equal(attention.decode8(*args), want)
    codes[bt[1, 0].long(), 1, 1, 3, 17] = 0x7F                 # one value of V: its dim, the heads of kv head 1
    out = attention.decode8(*args)
    bad = out.isnan().nonzero().tolist()
    assert bad == [[1, 2, 17], [1, 3, 17]]
    codes[bt[2, 3].long(), 0, 0, 15, 0] = 0x7F                 # one value of K: the rows of kv head 0
    out = attention.decode8(*args)
    assert out[2, :2].isnan().all() and not out[2, 2:].isnan().any()


def test_decode_queries_that_are_not_finite_and_pages_never_written():
    args = _decode_case([50, 50], 2, 1, seed=2)
    args[0][0, 0, 5] = NAN
    args[0][0, 1, 5] = float("inf")
    out = attention.decode8(*args)
    assert out[0].isnan().all() and not out[1].isnan().any()
    cache = KV8Cache.empty(8, 1, device=DEV)
    q, _, bt, req, ctx, plan = args
    q = torch.randn_like(q)
    assert (attention.decode8(q, cache, bt.clamp(max=7), req, ctx, plan) == 0).all()
    cache.codes.view(torch.uint8)[3] = 0x38                    # ones, at a scale of 1, next to pages of zeros
    cache.scales[3] = 1.0
    t = torch.tensor([[3, 1, 2, 4], [4, 3, 1, 2]], dtype=torch.int32, device=DEV)
    args = (q, cache, t, req, ctx, plan)
    _check_decode(args, attention.decode8(*args))


def test_decode_rows_that_do_not_fit_give_nan():
    args = _decode_case([30, 40, 50, 60, 33], 4, 2, seed=8, extra_pages=0)
    q, cache, bt, req, ctx, plan = args
    want = attention.decode8(*args)
    bt[1, 1] = cache.num_blocks                 # a page outside
    bt[2, 0] = -1
    req[3] = 5                                  # no such row
    ctx[4] = 65                                 # more than the table row
    out = attention.decode8(q, cache, bt, req, ctx, plan)
    assert torch.equal(out[0], want[0]) and out[1:].isnan().all()
    ctx[4] = -1
    assert attention.decode8(q, cache, bt, req, ctx, plan)[4].isnan().all()
    q, cache, bt, req, ctx, _ = _decode_case([200, 64], 4, 2, seed=8)
    small = attention.decode8_plan(2, 4, 2, 64, DEV)              # shorter than the first sequence
    out = attention.decode8(q, cache, bt, req, ctx, small)
    assert out[0].isnan().all() and not out[1].isnan().any()


def test_decode_table_views_requests_and_scale():
    """A block table that is a slice of a wider one, sequences that share requests, a batch below the plan's, a scale."""
    args = _decode_case([100, 200, 300], 4, 2, seed=3)
    q, cache, bt, req, ctx, plan = args
    wide = torch.full((3, 64), -7, dtype=torch.int32, device=DEV)
    wide[:, 3:3 + bt.shape[1]] = bt
    view = wide[:, 3:3 + bt.shape[1]]
    assert torch.equal(attention.decode8(q, cache, view, req, ctx, plan), attention.decode8(*args))
    r2 = torch.tensor([2, 2], dtype=torch.int32, device=DEV)
    c2 = torch.tensor([300, 17], dtype=torch.int32, device=DEV)
    sub = (q[:2], cache, view, r2, c2, plan)
    _check_decode((q[:2], cache, view, r2, c2, plan), attention.decode8(*sub))
    out = attention.decode8(*sub, scale=0.0)
    x = cache.values(bt[2, :19].long()).double()[:, 1].permute(1, 0, 2, 3).flatten(1, 2)[:, :300].mean(1)
    assert ((out[0].double() - x.repeat_interleave(2, 0)).abs() <= x.repeat_interleave(2, 0).abs() * 2 ** -8 +
            (2 ** -11 + 2 ** -18) * cache.values().abs().max().double()).all()


@pytest.mark.parametrize("nq,nkv", [(4, 4), (16, 2)])
def test_decode_of_several_tokens_of_a_request(nq, nkv):
    """A sequence for each new token, its request's pages and its own length: what a prefill of those tokens gives."""
    lens, prior = [9, 4, 1], [394, 1317, 0]
    ctxs = [a + b for a, b in zip(lens, prior)]
    _, cache, bt, _, _, _ = _decode_case(ctxs, nq, nkv, seed=2)
    q = torch.randn(14, nq, 128, device=DEV).bfloat16()
    pos = torch.cat([torch.arange(p, p + n) for p, n in zip(prior, lens)]).int().to(DEV)
    req = torch.repeat_interleave(torch.arange(3), torch.tensor(lens)).int().to(DEV)
    args = (q, cache, bt, req, pos + 1, attention.decode8_plan(14, nq, nkv, max(ctxs), DEV))
    _check_decode(args, attention.decode8(*args))


def test_decode_offsets_beyond_32_bits():
    """Pages more than 2^31 bytes into the codes, and a long sequence."""
    nkv, blocks = 8, 150000                       # 4.9 GB of codes
    cache = KV8Cache.empty(blocks, nkv, device=DEV)
    small = _rand_cache(600, nkv, 3, 0.0)
    cache.codes[-600:], cache.scales[-600:] = small.codes, small.scales
    n = 9001
    bt = (blocks - 1 - torch.arange(563, device=DEV)).int()[None].contiguous()
    q = torch.randn(1, 16, 128, device=DEV).bfloat16()
    args = (q, cache, bt, torch.zeros(1, dtype=torch.int32, device=DEV),
            torch.tensor([n], dtype=torch.int32, device=DEV), attention.decode8_plan(1, 16, nkv, n, DEV))
    _check_decode(args, attention.decode8(*args))
    qkv = torch.randn(1, 32 * 128, device=DEV).bfloat16()
    layers.qk_norm_rope_kv8(qkv, 16, 8, torch.zeros(1, dtype=torch.int32, device=DEV),
                            torch.tensor([(blocks - 1) * 16], device=DEV), None, None, 1e-6, None, q, cache)
    got = cache.values(torch.tensor([blocks - 1], device=DEV))[0, 1, :, 0].double()
    ref = qkv.double().view(32, 128)[24:]
    assert ((got - ref).abs() <= ref.abs() * 2 ** -4 + ref.abs().max() * 2 ** -15).all()


# ------------------------------------------------------------------------------------------------ prefill
@pytest.mark.parametrize("nq,nkv,lens,prior", [
    (16, 8, [200, 77, 1, 130], [0, 40, 300, 16]), (32, 8, [200, 77, 1, 130], [0, 40, 300, 16]),
    (4, 1, [200, 77, 1, 130], [0, 40, 300, 16]), (2, 2, [200, 77, 1, 130], [0, 40, 300, 16]),
    (2, 1, [1500, 77, 1, 130], [700, 40, 3000, 0])])                 # many key tiles: every barrier turns often
def test_prefill_matches_64_bits_and_replays_exactly(nq, nkv, lens, prior):
    ctxs = [a + b for a, b in zip(lens, prior)]
    _, cache, bt, _, _, _ = _decode_case(ctxs, nq, nkv, seed=nq, spread=1.0)
    T, G = sum(lens), nq // nkv
    q = torch.randn(T, nq, 128, device=DEV).bfloat16()
    starts = [sum(lens[:i]) for i in range(len(lens))]
    pos = torch.cat([torch.arange(p, p + n) for p, n in zip(prior, lens)]).int().to(DEV)
    tiles = attention.prefill_tiles(starts, lens, G).to(DEV)
    plan = attention.prefill8_plan(bt, ctxs, nkv)
    rs = torch.zeros(T, device=DEV)
    out = attention.prefill8(q, cache, plan, pos, tiles, row_sq=rs)
    assert torch.allclose(rs, out.float().square().sum((1, 2)), rtol=2e-5)
    for r, (n, p0) in enumerate(zip(lens, prior)):
        x = cache.values(bt[r, :-(-ctxs[r] // 16)].long()).double().permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :ctxs[r]]
        late = torch.arange(ctxs[r], device=DEV)[None] > torch.arange(p0, p0 + n, device=DEV)[:, None]
        for h in range(nq):
            k, v, qd = x[0, h // G], x[1, h // G], q[starts[r]:starts[r] + n, h].double()
            w = torch.softmax((qd @ k.t() * 128 ** -0.5).masked_fill(late, -math.inf), -1)
            ref, mag = w @ v, w @ v.abs()
            ds = float((qd.abs() @ k.abs().t()).max()) * 128 ** -0.5 * 128 * 2.0 ** -23
            # output to bf16; the weights to bf16, in the sum too; ex2, sums and scores as in decode
            tol = ref.abs() * 2 ** -8 + mag * (2 * 2 ** -8 + 2 ** -17 + 2 * ds)
            assert ((out[starts[r]:starts[r] + n, h].double() - ref).abs() <= tol).all(), (r, h)
    rt, ridx = attention.replay_tiles([[3, 150], [starts[1] + 76], [], [starts[3] + 129]], G)
    rt, ridx = rt.to(DEV), ridx.to(DEV)
    st = _state(4)
    attention.prefill8(q, cache, plan, pos, rt, out=out, row_idx=ridx, check=st[0])
    out.view(torch.int16)[starts[1] + 76, nq - 1, 9] ^= 1
    attention.prefill8(q, cache, plan, pos, rt, out=out, row_idx=ridx, check=st[1])
    out.view(torch.int16)[starts[1] + 76, nq - 1, 9] ^= 1
    last = bt[3, -(-ctxs[3] // 16) - 1].long()                    # a page changes after it was expanded
    cache.codes.view(torch.uint8)[last, 1, 0, 1, 3] ^= 1
    n = plan.pages.shape[0]
    attention.prefill8(q, cache, plan, pos, rt, out=out, row_idx=ridx, check=st[2], pages_from=n - 1, pages_step=64)
    attention.prefill8(q, cache, plan, pos, rt, out=out, row_idx=ridx, check=st[3], pages_from=0, pages_step=n)
    assert _flat(st[0])[0] == 0 and _flat(st[3])[0] == 0
    assert _flat(st[1])[:2] == (math.inf, ((starts[1] + 76) * nq + nq - 1) * 128 + 9)
    assert _flat(st[2])[:2] == (math.inf, (n - 1) * 2 * nkv + nkv)


@pytest.mark.parametrize("nq,nkv,lens,prior", [
    (4, 4, [9, 9, 1], [3945, 0, 700]), (16, 2, [23, 4], [1682, 16]), (8, 8, [1], [0]), (16, 1, [160, 200], [40, 3]),
    (2, 2, [40, 33, 1], [0, 7, 5000])])
def test_prefill_of_few_tokens(nq, nkv, lens, prior):
    """The decode kernel's path: 64 bits, replays, rows that no tile names, positions and pages outside."""
    ctxs = [a + b for a, b in zip(lens, prior)]
    _, cache, bt, _, _, _ = _decode_case(ctxs, nq, nkv, seed=nq, spread=1.0)
    T, G = sum(lens), nq // nkv
    assert (T + 3) * nkv <= attention.FEW_ROWS
    q = torch.randn(T + 3, nq, 128, device=DEV).bfloat16()
    starts = [sum(lens[:i]) for i in range(len(lens))]
    pos = torch.cat([torch.arange(p, p + n) for p, n in zip(prior, lens)] + [torch.zeros(3)]).int().to(DEV)
    tiles = attention.prefill_tiles(starts, lens, G).to(DEV)
    plan = attention.prefill8_plan(bt, ctxs, nkv)
    rs, out = torch.zeros(T + 3, device=DEV), torch.full_like(q, 7.0)
    attention.prefill8(q, cache, plan, pos, tiles, out=out, row_sq=rs)
    assert (out[T:] == 7).all() and (rs[T:] == 0).all()
    assert torch.allclose(rs[:T], out[:T].float().square().sum((1, 2)), rtol=2e-5)
    req = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).int().to(DEV)
    _check_decode((q[:T], cache, bt, req, pos[:T] + 1, None), out[:T])
    small = attention.prefill8_plan(bt, ctxs, nkv)           # where the plan's pages are too small for the partial sums
    small.work = small.work[:0]
    again = torch.full_like(q, 7.0)
    attention.prefill8(q, cache, small, pos, tiles, out=again)
    assert torch.equal(again, out)
    rt, ridx = attention.replay_tiles([[s + n - 1] for s, n in zip(starts, lens)], G)
    rt, ridx = rt.to(DEV), ridx.to(DEV)
    st = _state(2)
    attention.prefill8(q, cache, plan, pos, rt, out=out, row_idx=ridx, check=st[0])
    out.view(torch.int16)[T - 1, nq - 1, 9] ^= 1
    attention.prefill8(q, cache, plan, pos, rt, out=out, row_idx=ridx, check=st[1])
    assert _flat(st[0])[0] == 0 and st[:, 2].tolist() == [1, 1]
    assert _flat(st[1])[:2] == (math.inf, ((T - 1) * nq + nq - 1) * 128 + 9)
    want = attention.prefill8(q, cache, plan, pos, tiles)[:T]
    pos[0] = 1 << 20
    out = attention.prefill8(q, cache, plan, pos, tiles)[:T]
    assert (out[0] == 0).all() and torch.equal(out[1:], want[1:])
    pos[0] = prior[0]
    bt[-1, 0] = 1 << 20
    out = attention.prefill8(q, cache, attention.prefill8_plan(bt, ctxs, nkv), pos, tiles)[:T]
    assert out[starts[-1]:].isnan().all() and torch.equal(out[:starts[-1]], want[:starts[-1]])


def test_prefill_tensors_on_16_byte_boundaries():
    """Views whose rows begin 16 bytes behind a 32-byte boundary, over both caches: the same bits."""
    lens, nq, nkv = [300, 77], 8, 2
    _, cache, bt, _, _, _ = _decode_case(lens, nq, nkv, seed=6, spread=1.0)
    q = torch.randn(377, nq, 128, device=DEV).bfloat16()
    pos = torch.cat([torch.arange(n) for n in lens]).int().to(DEV)
    tiles = attention.prefill_tiles([0, 300], lens, nq // nkv).to(DEV)
    plain = cache.values().bfloat16().contiguous()
    off = [torch.zeros(q.numel() + 16, dtype=torch.bfloat16, device=DEV)[8:8 + q.numel()].view(q.shape) for _ in range(2)]
    off[0].copy_(q)
    assert all(t.data_ptr() % 32 == 16 for t in off)
    plan = attention.prefill8_plan(bt, lens, nkv)
    want = attention.prefill8(q, cache, plan, pos, tiles)
    assert torch.equal(attention.prefill8(off[0], cache, plan, pos, tiles, out=off[1]), want)
    off[1].zero_()
    assert torch.equal(attention.prefill(off[0], plain, bt, pos, tiles, nq, nkv, out=off[1]), want)
    few = torch.zeros_like(want[:40])
    plan = attention.prefill8_plan(bt[:1], [40], nkv)
    tiles = attention.prefill_tiles([0], [40], nq // nkv).to(DEV)
    attention.prefill8(q[:40], cache, plan, pos[:40].contiguous(), tiles, out=few)
    off[1].zero_()
    attention.prefill8(off[0][:40], cache, plan, pos[:40].contiguous(), tiles, out=off[1][:40])
    assert torch.equal(off[1][:40], few) and (off[1][40:] == 0).all()


def test_prefill_pages_and_positions_outside():
    """A page outside the cache gives NaN to its request alone; a position outside the plan's table gives zeros."""
    lens = [40, 33]
    _, cache, bt, _, _, _ = _decode_case(lens, 4, 2, seed=1)
    q = torch.randn(73, 4, 128, device=DEV).bfloat16()
    pos = torch.cat([torch.arange(40), torch.arange(33)]).int().to(DEV)
    tiles = attention.prefill_tiles([0, 40], lens, 2).to(DEV)
    want = attention.prefill8(q, cache, attention.prefill8_plan(bt, lens, 2), pos, tiles)
    bt[1, 0] = 1 << 20
    work = torch.empty(20 * 4096 * 2, dtype=torch.bfloat16, device=DEV)
    plan = attention.prefill8_plan(bt, lens, 2, work)
    pos[7] = 1 << 20
    out = attention.prefill8(q, cache, plan, pos, tiles)
    rows = [i for i in range(40) if i != 7]
    assert torch.equal(out[rows], want[rows]) and (out[7] == 0).all() and out[40:].isnan().all()


# ------------------------------------------------------------------------------------------------ together
def test_graphs_streams_and_a_run_of_the_operators():
    """Prompt append, prefill, then steps of append and decode (eager on a side stream, and captured twice, each graph
    with its own plan): the graphs' replays give the eager bits, and decode agrees with 64 bits over the cache."""
    nq, nkv, lens = 8, 2, [35, 18, 64]
    g = torch.Generator(device=DEV).manual_seed(1)
    table = layers.rope_table(128, 128, 10000.0, device=DEV)
    bt = torch.tensor([[1, 2, 3, 4, 5], [6, 7, 8, 0, 0], [9, 10, 11, 12, 13]], dtype=torch.int32, device=DEV)

    def at(r, p):
        return int(bt[r, p // 16]) * 16 + p % 16

    T = sum(lens)
    qkv = torch.randn(T, 12 * 128, device=DEV, generator=g).bfloat16()
    pos = torch.cat([torch.arange(n) for n in lens]).int().to(DEV)
    slots = torch.tensor([at(r, p) for r, n in enumerate(lens) for p in range(n)], device=DEV)
    w = (torch.ones(128, device=DEV) * 1.1).bfloat16()
    cache = KV8Cache.empty(14, nkv, device=DEV)
    q = torch.empty(T, nq, 128, dtype=torch.bfloat16, device=DEV)
    layers.qk_norm_rope_kv8(qkv, nq, nkv, pos, slots, w, w, 1e-6, table, q, cache)
    starts = [0, 35, 53]
    pre = attention.prefill8(q, cache, attention.prefill8_plan(bt, lens, nkv), pos,
                             attention.prefill_tiles(starts, lens, 4).to(DEV))
    step = torch.randn(3, 12 * 128, device=DEV, generator=g).bfloat16()
    p1 = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s1 = torch.tensor([at(r, n) for r, n in enumerate(lens)], device=DEV)
    req = torch.arange(3, dtype=torch.int32, device=DEV)
    ctx = p1 + 1

    def run(cache, plan, q, out):
        layers.qk_norm_rope_kv8(step, nq, nkv, p1, s1, w, w, 1e-6, table, q, cache)
        return attention.decode8(q, cache, bt, req, ctx, plan, out=out)

    def fresh():
        return (KV8Cache(cache.codes.clone(), cache.scales.clone()), attention.decode8_plan(3, nq, nkv, 4096, DEV),
                torch.empty(3, nq, 128, dtype=torch.bfloat16, device=DEV),
                torch.empty(3, nq, 128, dtype=torch.bfloat16, device=DEV))

    sides = [fresh() for _ in range(3)]
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        eager = run(*sides[0])
    torch.cuda.current_stream().wait_stream(other)
    c, plan, qq, _ = sides[0]
    _check_decode((qq, c, bt, req, ctx, plan), eager)
    # the last prompt token, seen by prefill (weights in bf16) and by decode (in f16), is the same to their roundings
    last = [s + n - 1 for s, n in zip(starts, lens)]
    dec = attention.decode8(q[last], cache, bt, req, p1, plan)
    _check_decode((q[last], cache, bt, req, p1, plan), dec)
    top = cache.values().abs().max()
    assert (dec.float() - pre[last].float()).abs().max() <= top * (2 * 2 ** -8 + 2 * 2 ** -8 + 2 ** -10)
    graphs = []
    for side in sides[1:]:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            run(*side)
        graphs.append(gr)
    for _ in range(2):
        for gr in graphs:
            gr.replay()
    torch.cuda.synchronize()
    for side in sides[1:]:
        assert torch.equal(side[3], eager)
        assert torch.equal(side[0].codes.view(torch.uint8), c.codes.view(torch.uint8))
        assert torch.equal(side[0].scales, c.scales)


def test_layers_of_a_cache():
    cache = KV8Cache.empty(6, 2, layers=3, device=DEV)
    assert len(cache) == 3 and cache[1].codes.shape == (6, 2, 2, 16, 128) and cache[1] is cache[1]
    assert cache[2].codes.data_ptr() == cache.codes[2].data_ptr() and kv8.page_bytes(2) == 2 * 2 * (2048 + 4)


def _engine(**kw):
    from sdcguard_b200.models.decoder import TINY
    from sdcguard_b200.serve.engine import LLMEngine
    return LLMEngine(TINY, device="cuda:0", num_blocks=64, max_prefill_tokens=512, max_num_seqs=8, max_model_len=512,
                     sample_every=4, kv_cache="fp8", **kw)


def test_engine_with_an_8_bit_cache():
    """Serving with kv_cache="fp8": the checks of append and attention run and stay clean, graph and eager steps give
    the same tokens, and pages that were used before give them again."""
    prompts = torch.randint(0, 1024, (5, 70), generator=torch.Generator().manual_seed(0))
    lens = [70, 33, 16, 1, 48]
    eng = _engine(checked=True)
    out = eng.generate(prompts, lens, 20)
    rows = {r["name"]: r for r in eng.model.read_checks()}
    for i in range(2):
        for op in ("rope_kv", "attn"):
            r = rows[f"layers.{i}.{op} (replay)"]
            assert r["checks"] > 0 and r["z"] == 0, r
    assert all(r["z"] < 6 for r in rows.values())
    assert eng.describe()["kv_cache"] == "fp8" and eng.describe()["kv_page_bytes"] == 2 * kv8.page_bytes(2)
    eager = _engine(checked=True, cuda_graph=False)
    assert torch.equal(eager.generate(prompts, lens, 20), out)
    assert torch.equal(eager.generate(prompts, lens, 20), out)          # pages used before
    scores = eng.score([prompts[0, :40].tolist()], topk=3)
    assert scores[0][0].shape == (40, 3) and torch.isfinite(scores[0][0]).all()


def test_engine_attention_replay_sees_a_flipped_page():
    """A code that changes between the attention and its replay is reported in the layer's attention slot."""
    eng = _engine(checked=True, cuda_graph=False)
    real, hit = attention.decode8, []

    def flipped(q, cache, *a, **kw):
        if kw.get("check") is not None and not hit:
            hit.append(1)
            cache.codes.view(torch.uint8)[1:, 0] ^= 0x40
        return real(q, cache, *a, **kw)

    attention.decode8 = flipped
    try:
        eng.generate(torch.randint(0, 1024, (2, 20), generator=torch.Generator().manual_seed(0)), [20, 20], 3)
    finally:
        attention.decode8 = real
    z = {r["name"]: r["z"] for r in eng.model.read_checks()}
    assert hit and z["layers.0.attn (replay)"] == math.inf


def test_engine_refuses():
    from sdcguard_b200.models.decoder import TINY
    from sdcguard_b200.serve.engine import LLMEngine
    with pytest.raises(ValueError):
        LLMEngine(TINY, device="cuda:0", num_blocks=8, kv_cache="int8")
    with pytest.raises(ValueError):
        LLMEngine(TINY, device="cuda:0", max_num_seqs=8, kv_cache="fp8",
                  cache=torch.zeros(2, 8, 2, 2, 16, 128, dtype=torch.bfloat16, device=DEV))
