"""Prefill attention on the tensor cores, over the 8-bit and over the bf16 cache: values that are not finite (in masked
places, behind a sequence's end, in queries and keys), rows without keys, and pages outside the cache. Comparisons are of
bits: what a row must not see does not change it."""
import math
import os
import subprocess
import sys

import pytest
import torch

from sdcguard_b200.ops import attention
from sdcguard_b200.ops.kv8 import KV8Cache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
NAN, INF = float("nan"), float("inf")
OUTSIDE = 1 << 20


def _flat(row):
    from sdcguard_b200.numerics import abft
    d = abft.decode_state_row(row.cpu().tolist())
    return d["z"], d["flat"], d["checks"]


class Case:
    """A prefill batch whose sequences end inside pages; `run` takes it over either cache. `few`: through the decode kernel."""

    def __init__(self, lens, prior, nq, nkv, seed=0, few=False):
        self.lens, self.prior, self.nq, self.nkv = lens, prior, nq, nkv
        self.ctxs = [a + b for a, b in zip(lens, prior)]
        self.T = sum(lens)
        assert (self.T * nkv <= attention.FEW_ROWS) == few
        g = torch.Generator(device=DEV).manual_seed(seed)
        need = [-(-n // 16) for n in self.ctxs]
        blocks = sum(need) + 2
        v = torch.randn(blocks, 2, nkv, 16, 128, device=DEV, generator=g)
        self.cache = KV8Cache((v * 64).to(torch.float8_e4m3fn), torch.full((blocks, nkv, 2), 2.0 ** -6, device=DEV))
        perm = torch.randperm(blocks - 2, generator=torch.Generator().manual_seed(seed)) + 1
        self.bt = torch.zeros(len(lens), max(need) + 1, dtype=torch.int32)
        o = 0
        for r, n in enumerate(need):
            self.bt[r, :n] = perm[o:o + n]
            o += n
        self.bt = self.bt.to(DEV)
        self.starts = [sum(lens[:i]) for i in range(len(lens))]
        self.pos = torch.cat([torch.arange(p, p + n) for p, n in zip(prior, lens)]).int().to(DEV)
        self.tiles = attention.prefill_tiles(self.starts, lens, nq // nkv).to(DEV)
        self.q = torch.randn(self.T, nq, 128, device=DEV, generator=g).bfloat16()

    def codes(self):
        return self.cache.codes.view(torch.uint8)

    def plan(self):
        return attention.prefill8_plan(self.bt, self.ctxs, self.nkv)

    def run(self, kind, **kw):
        out = kw.pop("out", None)
        if out is None:
            out = torch.full_like(self.q, 7.0)
        tiles = kw.pop("tiles", self.tiles)
        if kind == "fp8":
            return attention.prefill8(self.q, self.cache, kw.pop("plan", None) or self.plan(), self.pos, tiles, out=out, **kw)
        kw.pop("plan", None)
        return attention.prefill(self.q, self.cache.values().bfloat16(), self.bt, self.pos, tiles, self.nq, self.nkv,
                                 out=out, **kw)


SHAPES = [(16, 8), (2, 1), (8, 8), (16, 1)]


@pytest.mark.parametrize("kind", ["fp8", "bf16"])
@pytest.mark.parametrize("nq,nkv", SHAPES)
def test_places_behind_a_sequence_may_hold_anything(kind, nq, nkv):
    c = Case([300, 77, 130], [0, 21, 1016], nq, nkv)
    want = c.run(kind)
    assert torch.isfinite(want).all()
    for r, n in enumerate(c.ctxs):
        assert n % 16
        c.codes()[c.bt[r, n // 16].long(), :, :, n % 16:] = (0x7F, 0xFF)[r % 2]
    c.cache.scales[0] = NAN                       # the page that fills up the table's rows
    assert torch.equal(c.run(kind), want)


def test_places_behind_a_sequence_of_few_tokens():
    c = Case([30, 17], [3, 40], 4, 2, few=True)
    want = c.run("fp8")
    for r, n in enumerate(c.ctxs):
        c.codes()[c.bt[r, n // 16].long(), :, :, n % 16:] = 0x7F
    assert torch.equal(c.run("fp8"), want)


@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("kind", ["fp8", "bf16"])
def test_queries_that_are_not_finite(kind, few):
    c = Case([40, 33], [0, 7], 4, 2, few=True) if few else Case([300, 77], [0, 150], 4, 2)
    want = c.run(kind)
    a, b = c.starts[1] - 1, c.starts[1] + 5
    c.q[0] = NAN                                  # a row with one key
    c.q[a, 1] = NAN                               # one head
    c.q[a, 2, 5] = INF
    c.q[b, 3, 100] = NAN
    out = c.run(kind)
    bad = out.isnan().any(-1)
    assert bad.nonzero().tolist() == [[0, 0], [0, 1], [0, 2], [0, 3], [a, 1], [a, 2], [b, 3]]
    assert out[bad].isnan().all() and torch.equal(out[~bad], want[~bad])


@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("kind", ["fp8", "bf16"])
@pytest.mark.parametrize("lo,hi", [(0, 1), (130, 131), (0, 128)])
def test_keys_that_are_not_finite_reach_the_rows_that_see_them(kind, few, lo, hi):
    """K of NaN at the first place (all that the first row sees), in the second key tile, in all of the first tile (rows with
    finite scores behind it)."""
    c = Case([150], [0], 4, 2, few=True) if few else Case([300, 77], [0, 150], 4, 2)
    want = c.run(kind)
    for at in range(lo, hi):
        c.codes()[c.bt[0, at // 16].long(), 0, 1, at % 16, 9] = 0x7F         # of kv head 1: query heads 2 and 3
    out = c.run(kind)
    hit = torch.zeros(c.T, 4, dtype=torch.bool, device=DEV)
    hit[lo:c.lens[0], 2:] = True
    assert out[hit].isnan().all() and torch.equal(out[~hit], want[~hit])


@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("kind", ["fp8", "bf16"])
def test_a_value_that_is_not_finite_reaches_its_dim(kind, few):
    """A V of NaN that every row sees: its dim in the heads of its kv head, and nothing else."""
    c = Case([150], [7], 4, 2, few=True) if few else Case([300, 77], [7, 150], 4, 2)
    want = c.run(kind)
    c.codes()[c.bt[0, 0].long(), 1, 0, 3, 17] = 0x7F
    out = c.run(kind)
    n = c.lens[0]
    assert out[:n, :2, 17].isnan().all()
    out[:n, :2, 17] = want[:n, :2, 17]
    assert torch.equal(out, want)


def test_scores_of_minus_infinity_alone_give_nan():
    """exp(-inf - max) with a maximum of -inf: 0 / 0, as in the formula, on every path."""
    for few in (True, False):
        c = Case([40], [0], 2, 1, few=True) if few else Case([450], [0], 2, 1)
        c.codes()[:, 0] = 0x38                    # keys of ones
        c.q[1, 0] = -INF
        for kind in ("fp8", "bf16"):
            out = c.run(kind)
            assert out[1, 0].isnan().all() and out.isnan().any(-1).sum() == 1
    c = Case([40], [0], 2, 1, few=True)
    c.codes()[:, 0] = 0x38
    c.q[:2, 0] = -INF
    for segs in (1, 2):
        plan = attention.decode8_plan(2, 2, 1, 40, DEV)
        if segs == 2:
            plan = attention.Decode8Plan(2, 2, 1, 40, 2, 2, torch.empty(2 * 2 * 2 * 132, device=DEV))
        out = attention.decode8(c.q[:2], c.cache, c.bt, torch.zeros(2, dtype=torch.int32, device=DEV),
                                torch.tensor([40, 20], dtype=torch.int32, device=DEV), plan)
        assert out[:, 0].isnan().all() and torch.isfinite(out[:, 1]).all()


@pytest.mark.parametrize("nq,nkv", [(16, 8), (4, 1), (8, 8)])
def test_positions_outside_the_table_give_rows_of_zeros(nq, nkv):
    """One row of a live tile, a tile of one token, every row of a request (both tiles of its pairs)."""
    per = 128 // (nq // nkv)                                 # tokens of a tile
    c = Case([2 * per + 1, 300, 5, 40], [0, 9, 30, 0], nq, nkv)
    want = c.run("fp8")
    c.pos[7] = OUTSIDE
    c.pos[2 * per] = OUTSIDE                                 # the remainder tile
    c.pos[c.starts[2]:c.starts[3]] = OUTSIDE
    c.pos[c.starts[3] + 3] = -1
    rows = [7, 2 * per, c.starts[3] + 3] + list(range(c.starts[2], c.starts[3]))
    rest = [i for i in range(c.T) if i not in rows]
    sq = torch.zeros(c.T, device=DEV)
    plan = c.plan()
    out = c.run("fp8", row_sq=sq, plan=plan)
    assert (out[rows] == 0).all() and torch.equal(out[rest], want[rest])
    assert (sq[rows] == 0).all() and torch.allclose(sq, out.float().square().sum((1, 2)), rtol=2e-5)
    # the replay compares such rows too
    tiles, idx = attention.replay_tiles([[2 * per], [], [c.starts[2] + 1], []], nq // nkv)
    tiles, idx = tiles.to(DEV), idx.to(DEV)
    st = torch.zeros(2, 4, dtype=torch.int64, device=DEV)
    c.run("fp8", out=out, row_idx=idx, tiles=tiles, check=st[0], plan=plan)
    out[c.starts[2] + 1, nq - 1, 70] = 1.0
    c.run("fp8", out=out, row_idx=idx, tiles=tiles, check=st[1], plan=plan)
    assert _flat(st[0])[::2] == (0, 1)
    assert _flat(st[1]) == (math.inf, ((c.starts[2] + 1) * nq + nq - 1) * 128 + 70, 1)


def test_pages_outside_the_cache_give_nan_to_their_request():
    c = Case([300, 77], [0, 150], 4, 2)
    want = c.run("fp8")
    c.bt[1, 0] = OUTSIDE
    out = c.run("fp8")
    assert torch.equal(out[:300], want[:300]) and out[300:].isnan().all()
    c.bt[1, 0] = -1
    assert c.run("fp8")[300:].isnan().all()


def test_many_pairs_a_cta():
    """More pairs than SMs: a CTA takes over others, with rows and whole tiles that have no keys among them."""
    lens = [700 + 37 * i for i in range(12)]
    c = Case(lens, [0] * 12, 16, 8)
    assert c.tiles.shape[0] // 2 * 8 > 148 * 2
    want = c.run("fp8")
    keep = torch.ones(c.T, dtype=torch.bool, device=DEV)
    for r in (1, 4, 11):
        keep[c.starts[r]:c.starts[r] + 64 * (r + 3)] = False
    c.pos[~keep] = OUTSIDE
    for r, n in enumerate(c.ctxs):
        if n % 16:
            c.codes()[c.bt[r, n // 16].long(), :, :, n % 16:] = 0x7F
    out = c.run("fp8")
    assert (out[~keep] == 0).all() and torch.equal(out[keep], want[keep])


def test_one_tile_a_cta():
    """The kernel that takes one query tile a CTA (its choice is read once in a process) answers the same calls."""
    if os.environ.get("SDCGUARD_PREFILL_PINGPONG") == "0":
        pytest.skip("this is that process")
    env = dict(os.environ, SDCGUARD_PREFILL_PINGPONG="0")
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-p", "no:cacheprovider",
                        os.path.join(here, "test_prefill_rows_gpu.py"),
                        os.path.join(here, "test_kv8_gpu.py") + "::test_prefill_matches_64_bits_and_replays_exactly"],
                       env=env, capture_output=True, text=True, timeout=600, cwd=os.path.dirname(here))
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-1000:]


@pytest.mark.parametrize("kind", ["fp8", "bf16"])
@pytest.mark.parametrize("nq,nkv", [(32, 1), (128, 1), (128, 4)])
def test_many_heads_of_a_kv_head(kind, nq, nkv):
    """Four tokens a tile and one, in calls of few tokens too: output to bf16 (2^-8), weights to bf16 in the products and the
    sum (2 x 2^-8), ex2 and sums (2^-17), scores of 128 products in fp32, each rounded or cut (in weight and sum)."""
    lens, prior = [37, 1, 20], [100, 0, 333]
    c = Case(lens, prior, nq, nkv, few=True)
    out = c.run(kind)
    for r, (n, p0, s) in enumerate(zip(lens, prior, c.starts)):
        x = c.cache.values(c.bt[r, :-(-c.ctxs[r] // 16)].long()).double().permute(1, 2, 0, 3, 4).flatten(2, 3)
        late = torch.arange(c.ctxs[r], device=DEV)[None] > torch.arange(p0, p0 + n, device=DEV)[:, None]
        for h in range(nq):
            k, v = (t[:c.ctxs[r]] for t in x[:, h // (nq // nkv)])
            qd = c.q[s:s + n, h].double()
            w = torch.softmax((qd @ k.t() * 128 ** -0.5).masked_fill(late, -math.inf), -1)
            ds = float((qd.abs() @ k.abs().t()).max()) * 128 ** -0.5 * 128 * 2.0 ** -23
            tol = (w @ v).abs() * 2 ** -8 + w @ v.abs() * (2 * 2 ** -8 + 2 ** -17 + 2 * ds)
            assert ((out[s:s + n, h].double() - w @ v).abs() <= tol).all(), (r, h)


@pytest.mark.parametrize("kind", ["fp8", "bf16"])
def test_rows_that_no_tile_names_stay(kind):
    c = Case([300, 77], [0, 150], 4, 2)
    want = c.run(kind)
    c.q = torch.cat([c.q, torch.full((3, 4, 128), NAN, device=DEV).bfloat16()])
    c.pos = torch.cat([c.pos, torch.zeros(3, dtype=torch.int32, device=DEV)])
    sq = torch.zeros(c.T + 3, device=DEV)
    out = c.run(kind, row_sq=sq)
    assert torch.equal(out[:c.T], want) and (out[c.T:] == 7).all() and (sq[c.T:] == 0).all()


@pytest.mark.parametrize("few", [False, True])
def test_captured_and_on_two_streams(few):
    """Two graphs with a plan each, replayed on two streams at once over caches that change between the replays, and eager
    calls on a side stream: the eager bits."""
    cases = [Case([40, 33], [0, 7], 4, 2, seed=s, few=True) if few else Case([700, 77], [0, 150], 4, 2, seed=s)
             for s in (0, 1)]
    other = [Case(c.lens, c.prior, 4, 2, seed=5 + i, few=few).cache.codes.view(torch.uint8) for i, c in enumerate(cases)]
    plans, outs = [c.plan() for c in cases], [torch.zeros_like(c.q) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    graphs = []
    for c, plan, out in zip(cases, plans, outs):
        c.run("fp8", plan=plan, out=out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run("fp8", plan=plan, out=out)
        graphs.append(g)
    for turn in range(3):
        want = [c.run("fp8") for c in cases]
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out, w)
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(c.run("fp8", plan=plans[0 if c is cases[0] else 1]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for c, o in zip(cases, other):
            c.codes().copy_(o if turn == 0 else c.codes().flip(0))
        torch.cuda.synchronize()


@pytest.mark.parametrize("few", [False, True])
def test_scale(few):
    """A scale of zero weighs all keys alike: the mean of the values that the row sees."""
    c = Case([40, 33], [0, 7], 4, 2, few=True) if few else Case([300, 77], [0, 150], 4, 2)
    out = c.run("fp8", scale=0.0).double()
    for r, (n, p0, s) in enumerate(zip(c.lens, c.prior, c.starts)):
        v = c.cache.values(c.bt[r, :-(-c.ctxs[r] // 16)].long()).double().permute(1, 2, 0, 3, 4).flatten(2, 3)[1]
        at = torch.arange(p0, p0 + n, device=DEV)
        mean, mag = (t.cumsum(1)[:, at] / (at + 1)[:, None] for t in (v, v.abs()))
        ref = mean.transpose(0, 1).repeat_interleave(2, 1)
        tol = ref.abs() * 2 ** -8 + mag.transpose(0, 1).repeat_interleave(2, 1) * 2 ** -11
        assert ((out[s:s + n] - ref).abs() <= tol).all()
