"""Paged attention entry points (`csrc/attention.cu`): causal prefill over a batch of requests and single-token
decode, both over a paged KV cache with 16-token pages, plus the host-side tiling of prefill work; `decode8` and
`prefill8` do the same over a cache held in 8 bits (`csrc/kv8.cu`, `ops.kv8`).

Rows of both kernels are deterministic (see the kernel file), so `replay_*` recompute a sample of rows on
separate CTAs and `ops.layers.compare_rows` checks them bit for bit. The reference samples (token, head) pairs
and recomputes them in fp32 against an error bound (src/sdcguard/serve_attn.py:5-48, `attn_check_triton`
:574); the replay needs no bound, so every flipped bit in a sampled row is seen.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np
import torch

from .. import _native
from . import kv8
from .kv8 import PAGE, KV8Cache

ROWS = 128


def _s(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _pairs(per_request: list[list[tuple]]) -> list[tuple]:
    """Tiles two by two within each request (the prefill kernel runs the two tiles of a pair in one CTA on shared
    key / value tiles); a request with an odd number of tiles gets an empty partner (0 tokens)."""
    pairs = []
    for tiles in per_request:
        for i in range(0, len(tiles), 2):
            a = tiles[i]
            b = tiles[i + 1] if i + 1 < len(tiles) else (a[0], a[1] + a[2], 0, -1)
            pairs.append((a, b))
    return pairs


def prefill_tiles(q_starts: Sequence[int], q_lens: Sequence[int], group: int) -> torch.Tensor:
    """(2 n, 4) int32 tiles (request, first token, tokens, -1) covering every request's new tokens, as n pairs of
    consecutive tiles of one request (entries 2i and 2i + 1), pairs ordered by the keys they attend to, most first
    (later tiles of a causal prompt attend to more keys), so the longest CTAs start first."""
    tpc = ROWS // group
    per = [[(r, s + off, min(tpc, n - off), -1) for off in range(0, n, tpc)] for r, (s, n) in
           enumerate(zip(q_starts, q_lens))]
    pairs = _pairs(per)
    # keys a pair attends to: its last token's position within its request
    pairs.sort(key=lambda pr: -(pr[0][1] - q_starts[pr[0][0]] + pr[0][2] + pr[1][2]))
    flat = [t for pr in pairs for t in pr]
    return torch.tensor(flat, dtype=torch.int32).view(-1, 4)


def replay_tiles(sampled: Sequence[Sequence[int]], group: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Tiles for a replay of sampled tokens (sampled[r] lists request r's sampled token indices), in pairs of one
    request as `prefill_tiles` makes them; returns (tiles, row_idx)."""
    tpc = ROWS // group
    per, idx = [], []
    for r, toks in enumerate(sampled):
        mine = []
        for off in range(0, len(toks), tpc):
            chunk = list(toks[off:off + tpc])
            mine.append((r, 0, len(chunk), len(idx)))
            idx.extend(chunk)
        per.append(mine)
    flat = [t for pr in _pairs(per) for t in pr]
    t = torch.tensor(flat, dtype=torch.int32).view(-1, 4)
    return t, torch.tensor(idx, dtype=torch.int32)


def prefill(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, pos: torch.Tensor,
            tiles: torch.Tensor, nq: int, nkv: int, out: Optional[torch.Tensor] = None,
            row_idx: Optional[torch.Tensor] = None, row_sq: Optional[torch.Tensor] = None,
            scale: Optional[float] = None, check: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q: (T, nq, 128) bf16; tiles/row_idx/pos/block_table int32 on the device. out: (T, nq, 128) or, for a
    replay, any tensor indexed by the same token ids. What a page holds behind its sequence's end reaches no row. With `check` (a state row; replay tiles and row_idx
    given), the sampled rows are recomputed and compared with `out` instead of written."""
    if out is None:
        out = torch.empty_like(q)
    scale = 1.0 / math.sqrt(128) if scale is None else scale
    _native.check(_native.lib().sdc_attn_prefill(
        q.data_ptr(), out.data_ptr(), cache.data_ptr(), cache.shape[0], block_table.data_ptr(), block_table.shape[1],
        pos.data_ptr(), tiles.data_ptr(), tiles.shape[0], None if row_idx is None else row_idx.data_ptr(), nq, nkv,
        128, float(scale), None if row_sq is None else row_sq.data_ptr(), None if check is None else check.data_ptr(),
        _s(q)), "attention prefill")
    return out


def decode_scratch(nseq_rows: int, nq: int, nkv: int, max_ctx: int, device) -> torch.Tensor:
    """Partial-result scratch for `decode` (one record per sequence, kv head and 256-key segment)."""
    splits = int(_native.lib().sdc_attn_decode_splits(int(max_ctx)))
    return torch.empty(nseq_rows * nkv * splits * (nq // nkv) * 132, dtype=torch.float32, device=device)


def decode(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, seq_req: torch.Tensor,
           ctx: torch.Tensor, nq: int, nkv: int, max_ctx: int, out: Optional[torch.Tensor] = None,
           seq_idx: Optional[torch.Tensor] = None, nseq: Optional[int] = None,
           row_sq: Optional[torch.Tensor] = None, scale: Optional[float] = None,
           scratch: Optional[torch.Tensor] = None, check: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q: (B, nq, 128); split-KV: a CTA per (sequence, kv head) and every z-th 256-key segment (64-key chunks merged
    in order inside the segment), then a fixed-order combine of the segments.
    seq_idx selects sequences to run (replay). scratch: from `decode_scratch` (allocated here if absent).
    With `check` (a state row; seq_idx given), the selected rows are recomputed and compared with `out`."""
    if out is None:
        out = torch.empty_like(q)
    scale = 1.0 / math.sqrt(128) if scale is None else scale
    n = nseq if nseq is not None else (seq_idx.shape[0] if seq_idx is not None else q.shape[0])
    if scratch is None:
        scratch = decode_scratch(q.shape[0], nq, nkv, max_ctx, q.device)
    _native.check(_native.lib().sdc_attn_decode(
        q.data_ptr(), out.data_ptr(), cache.data_ptr(), cache.shape[0], block_table.data_ptr(), block_table.shape[1],
        seq_req.data_ptr(), ctx.data_ptr(), None if seq_idx is None else seq_idx.data_ptr(), n, nq, nkv, 128,
        int(max_ctx), float(scale), scratch.data_ptr(), None if row_sq is None else row_sq.data_ptr(),
        None if check is None else check.data_ptr(), _s(q)), "attention decode")
    return out


# ------------------------------------------------------------------------------------ cache in 8 bits (csrc/kv8.cu)
_SCALE = 1.0 / math.sqrt(128)
DECODE8_CTAS = 148 * 3      # CTAs of one long sequence: three per SM
DECODE8_MAX_SEGS = 256


@dataclass
class Decode8Plan:
    """How `decode8` cuts the keys of up to nseq sequences of up to max_ctx keys, and its scratch. A replay (check mode)
    takes the plan of the call that it repeats: the cut decides the order of the sums. One launch at a time may use a
    plan; two streams, or two graphs that may run at once, take a plan each."""
    nseq: int
    nq: int
    nkv: int
    max_ctx: int
    seg_pages: int
    max_segs: int
    part: Optional[torch.Tensor]


def decode8_cut(nseq: int, nkv: int, max_ctx: int) -> tuple[int, int]:
    """(pages a segment, segments of the longest sequence) of a decode step. Segments of equal size: fewer leave SMs
    idle, more pay the start of a CTA and the merge again. One sequence is cut into as many as run at once (131072 keys,
    8 kv heads: 149 pages a segment 51.6 us, 112 pages 55.8 us, 74 pages 62 us). Several differ in length and
    balance better in twice as many (8 of up to 8000: 39 pages 21.3 us, 64 pages 27.0 us). At least 12 pages (1 x 20000
    keys, one kv head: 12 pages 11.2 us, 8 pages 12.9 us, 24 pages 12.4 us), of several sequences 20 (16 x 1200: 15.2 us, 12
    pages 18.5), at most 256, at most 256 segments (what
    one combine CTA merges), and no cut up to 24 pages, where the merge costs more than it saves (4 x 300 keys: 6.3 us,
    in two 7.7 us).

    Several sequences with 200 rows (a sequence and kv head) or more fill the SMs by themselves, and what a cut saves in
    the longest row's time it pays in starts and merges. Ragged and uniform lengths, uncut against two segments: 320 rows
    of up to 44 pages 12.2 and 16.0 us, 14.1 and 21.5 (of 100 pages, three segments: 24.7 and 28.4, 21.2 and 34.1: cut);
    448 of 177 pages 48.9 and 58.6, 50.4 and 80.6; 640 of 57 pages 22.3 and 39.1, 27.4 and 41.3 (720 of 125 pages 44.8 and
    80.8, 44.9 and 74.6: cut); 880 of 125 pages 53.7 and 84.2, 58.3 and 97.2. Two segments are 3/5 and 2/5 of the longest
    row, which leaves more rows whole than halves do: 488 rows of 257 pages 58.5 and 98.0 us, halves 63.9 and 99.2."""
    pages = -(-max_ctx // PAGE)
    if pages <= 24:
        return pages, 1
    rows = nseq * nkv
    if nseq > 1 and rows >= 200:
        if pages <= (64 if rows < 388 else 192 if rows <= 148 * 4 else 96 if rows < 800 else 256):
            return pages, 1
        if 388 <= rows < 800 and pages * 3 // 5 <= 252:
            return -(-pages * 3 // 20) * 4, 2
    ctas = DECODE8_CTAS if nseq == 1 else 2 * DECODE8_CTAS
    seg = max(12 if nseq == 1 else 20, min(256, -(-nseq * nkv * pages // ctas)), -(-pages // DECODE8_MAX_SEGS))
    segs = -(-pages // seg)
    seg = -(-pages // segs)                       # alike, and a multiple of the four warps where that adds no segment
    seg = min(-(-seg // 4) * 4, pages)
    return seg, -(-pages // seg)


def decode8_plan(nseq: int, nq: int, nkv: int, max_ctx: int, device) -> Decode8Plan:
    """Plan and scratch of `decode8` for up to nseq sequences of up to max_ctx keys."""
    if nseq < 1 or nkv < 1 or nq % nkv or not 1 <= nq // nkv <= 16 or not 1 <= max_ctx <= 1 << 24:
        raise ValueError(f"nseq {nseq}, nq {nq}, nkv {nkv}, max_ctx {max_ctx}: at least one sequence, 1 to 16 query "
                         "heads per kv head, 1 to 2^24 keys")
    seg, segs = decode8_cut(nseq, nkv, max_ctx)
    part = torch.empty(nseq * nq * segs * 132, dtype=torch.float32, device=device) if segs > 1 else None
    return Decode8Plan(nseq, nq, nkv, max_ctx, seg, segs, part)


def _want_q(q: torch.Tensor, cache: KV8Cache, out: Optional[torch.Tensor]) -> tuple:
    """(rows, query heads, out) of queries that fit the cache."""
    shape = q.shape
    if not cache.one_layer or len(shape) != 3 or shape[2] != 128:
        raise ValueError(f"q must be (rows, heads, 128), got {tuple(shape)}, and the cache one layer of a KV8Cache")
    kv8.want(q, torch.bfloat16, shape, cache.device, "q", align=16)
    if out is None:
        out = torch.empty_like(q)
    else:
        kv8.want(out, torch.bfloat16, shape, cache.device, "out", align=16)
    return shape[0], shape[1], out


def _want_extra(row_sq, check, rows: int, dev) -> None:
    if row_sq is not None:
        kv8.want(row_sq, torch.float32, (rows,), dev, "row_sq")
    if check is not None:
        kv8.want_state(check, dev)


def decode8(q: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor, seq_req: torch.Tensor, ctx: torch.Tensor,
            plan: Decode8Plan, out: Optional[torch.Tensor] = None, seq_idx: Optional[torch.Tensor] = None,
            row_sq: Optional[torch.Tensor] = None, scale: Optional[float] = None,
            check: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence over a cache of 8 bits: q (B, nq, 128) bf16, ctx[b] keys (the new token's
    among them) in the pages of row seq_req[b] of block_table (int32). Any number of query heads per kv head up to 16.

    A sequence without keys (ctx 0) gives zeros. One with more keys than its table row or the plan holds, a table row
    that does not exist, or a page outside the cache gives NaN. seq_idx selects sequences, each once; with `check` (a
    state row) they are recomputed and compared with `out`. row_sq: += ||row||^2 of the output (cleared by the caller;
    its sum over kv heads is taken in no fixed order)."""
    given = out
    b, nq, out = _want_q(q, cache, out)
    dev, nkv = cache.device, cache.nkv
    if nq != plan.nq or nkv != plan.nkv or b > plan.nseq:
        raise ValueError(f"q {tuple(q.shape)} and {nkv} kv heads do not fit the plan ({plan.nseq} sequences, {plan.nq} "
                         f"query and {plan.nkv} kv heads)")
    table, stride = block_table.shape, block_table.stride()
    if block_table.dtype is not torch.int32 or block_table.device != dev or len(table) != 2 \
            or (stride[1] != 1 and table[1] > 1):
        raise ValueError("block_table must be int32 (requests, pages) with contiguous rows on the cache's device")
    kv8.want(seq_req, torch.int32, (b,), dev, "seq_req")
    kv8.want(ctx, torch.int32, (b,), dev, "ctx")
    if seq_idx is not None:
        kv8.want(seq_idx, torch.int32, (seq_idx.shape[0],), dev, "seq_idx")
    if check is not None and (seq_idx is None or given is None):
        raise ValueError("check needs seq_idx, and out, which it compares")
    if cache.num_blocks * nkv >= 1 << 26 or (scale is not None and not 0 <= scale < math.inf):
        raise ValueError(f"{cache.num_blocks} pages of {nkv} heads (below 2^26 in all) and scale {scale} (not negative)")
    if plan.part is not None and plan.part.device != dev:
        raise ValueError("the plan must be on the cache's device")
    if row_sq is not None or check is not None:
        _want_extra(row_sq, check, b, dev)
    kv8.launch("sdc_kv8_decode", dev, (
        q.data_ptr(), out.data_ptr(), cache.codes.data_ptr(), cache.scales.data_ptr(), cache.num_blocks,
        block_table.data_ptr(), table[0], table[1], stride[0], seq_req.data_ptr(),
        ctx.data_ptr(), kv8.ptr(seq_idx), b if seq_idx is None else seq_idx.shape[0], b, nq, nkv, plan.seg_pages,
        plan.max_segs, _SCALE if scale is None else scale, kv8.ptr(plan.part), kv8.ptr(row_sq), kv8.ptr(check)))
    return out


def expanded_page(nkv: int) -> int:
    """bf16 elements of one expanded page of a layer."""
    return 2 * nkv * PAGE * 128


@dataclass
class Prefill8Plan:
    """The pages of a prefill batch in one list, and the bf16 pages they are expanded to. The same rules as for
    `Decode8Plan`: one launch at a time, and a replay takes the plan of the call that it repeats."""
    pages: torch.Tensor        # (P,) int32 page ids, request after request
    table: torch.Tensor        # (R, W) int32 places in that list
    work: torch.Tensor         # (P, 2, nkv, 16, 128) bf16
    nkv: int
    block_table: torch.Tensor  # (R, W) int32 page ids (a copy)


def prefill8_plan(block_table: torch.Tensor, ctx_lens: Sequence[int], nkv: int,
                  work: Optional[torch.Tensor] = None) -> Prefill8Plan:
    """Plan of `prefill8` for requests of ctx_lens keys (cached and new ones) in the rows of block_table. `work`: bf16
    memory for the expanded pages (`expanded_page` elements each), kept by the caller across layers and steps."""
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.shape[0] != len(ctx_lens):
        raise ValueError("block_table must be int32 with one row for each of ctx_lens")
    dev, width = block_table.device, block_table.shape[1]
    counts = [-(-int(n) // PAGE) for n in ctx_lens]
    if not counts or min(int(n) for n in ctx_lens) < 1 or max(counts) > width:
        raise ValueError(f"ctx_lens {list(ctx_lens)[:8]}: at least one key each, and no more than {width} pages")
    total, w = sum(counts), max(counts)
    c = np.array(counts)
    place = np.arange(w)
    used = place < c[:, None]
    table = np.where(used, (np.cumsum(c) - c)[:, None] + place, 0)
    both = torch.from_numpy(np.concatenate([np.flatnonzero(used), table.ravel()]).astype(np.int32)).to(dev)   # one copy
    bt = block_table[:, :w].clone(memory_format=torch.contiguous_format)
    pages, table = bt.view(-1).index_select(0, both[:total]), both[total:].view(-1, w)
    need = total * expanded_page(nkv)
    if work is None:
        work = torch.empty(need, dtype=torch.bfloat16, device=dev)
    elif work.dtype != torch.bfloat16 or work.numel() < need or not work.is_contiguous() or work.device != dev \
            or work.data_ptr() % 128:
        raise ValueError(f"work must be contiguous bf16 of at least {need} elements on {dev}")
    return Prefill8Plan(pages, table, work.view(-1)[:need].view(total, 2, nkv, PAGE, 128), nkv, bt)


# A prefill's CTA walks over all keys of its rows, 2 us for 128 of them; the decode kernel cuts the keys but reads them for
# every token. So few rows (tokens x kv heads) go there: 54 tokens x 4 heads behind 3945 keys 36 us against 78, 23 x 2 behind
# 1682 11 against 36, 64 x 8 behind 4000 (above the line) 73 against 84, 128 x 8 behind 8000 252 against 142.
FEW_ROWS = 400


def _prefill8_few(q, cache, plan, pos, tiles, out, row_idx, row_sq, scale, check):
    t, nq, nkv, dev, keys = q.shape[0], q.shape[1], plan.nkv, cache.device, plan.table.shape[1] * PAGE
    if cache.num_blocks * nkv >= 1 << 26:
        raise ValueError(f"{cache.num_blocks} pages of {nkv} heads (below 2^26 in all)")
    rows = 0 if row_idx is None else row_idx.shape[0]
    seg, segs = decode8_cut(t, nkv, keys)
    part = t * nq * segs * 132 if segs > 1 else 0         # floats, then the lists, where the expanded pages would go
    need = part + 3 * t + rows
    work = plan.work if plan.work.numel() >= 2 * need else torch.empty(need, dtype=torch.int32, device=dev)
    part_at, bt = work.data_ptr(), plan.block_table
    req_at = part_at + 4 * part
    ctx_at, idx_at = req_at + 4 * t, req_at + 8 * t
    stream = kv8.stream(dev)                              # (of the first half of the arguments)
    kv8.launch("sdc_kv8_prefill_few", dev, (
        tiles.data_ptr(), tiles.shape[0], ROWS // (nq // nkv), kv8.ptr(row_idx), rows, pos.data_ptr(), keys, t, req_at,
        ctx_at, idx_at, stream,
        q.data_ptr(), out.data_ptr(), cache.codes.data_ptr(), cache.scales.data_ptr(), cache.num_blocks, bt.data_ptr(),
        bt.shape[0], bt.shape[1], bt.shape[1], req_at, ctx_at, idx_at, t + rows, t, nq, nkv, seg, segs,
        _SCALE if scale is None else scale, part_at, kv8.ptr(row_sq), kv8.ptr(check)))
    return out


def prefill8(q: torch.Tensor, cache: KV8Cache, plan: Prefill8Plan, pos: torch.Tensor, tiles: torch.Tensor,
             out: Optional[torch.Tensor] = None, row_idx: Optional[torch.Tensor] = None,
             row_sq: Optional[torch.Tensor] = None, scale: Optional[float] = None,
             check: Optional[torch.Tensor] = None, pages_from: int = 0, pages_step: int = 64) -> torch.Tensor:
    """`prefill` over a cache of 8 bits: the plan's pages are expanded to bf16 (exact for power-of-two scales), then the
    tensor-core prefill reads those; a call of few tokens (T kv heads <= FEW_ROWS) runs through the decode kernel instead, a
    sequence for each token, so a row's last bits depend on which of the two its call takes. q (T, nq, 128), tiles from
    `prefill_tiles`, requests numbered as in the plan, each token's position below its request's ctx_lens. A position outside
    the plan's table gives a row of zeros, a page outside the cache NaN. What a page holds behind its sequence's end reaches
    no row; a query of NaN, or a key that a row sees, makes the row NaN. (A value of NaN inside the sequence gives its dim NaN
    in the rows that see it and, in calls that are not of few tokens, in rows up to 254 places before it.) With `check`: the rows of the replay tiles are compared, and every pages_step-th expanded page
    (where there are such) from pages_from on."""
    given = out
    t, nq, out = _want_q(q, cache, out)
    dev, nkv = cache.device, cache.nkv
    if nkv != plan.nkv or nq % nkv or ROWS % (nq // nkv) or nq == 0:
        raise ValueError(f"{nq} query heads on {nkv} kv heads (plan: {plan.nkv}): a power of two up to 128 per kv head")
    kv8.want(pos, torch.int32, (t,), dev, "pos")
    kv8.want(tiles, torch.int32, (tiles.shape[0], 4), dev, "tiles", align=16)
    if plan.work.device != dev:
        raise ValueError("the plan must be on the cache's device")
    if scale is not None and not 0 <= scale < math.inf:
        raise ValueError(f"scale {scale}: finite and not negative")
    if check is not None and (row_idx is None or given is None or pages_from < 0 or pages_step < 1):
        raise ValueError("check needs replay tiles with row_idx, out, which it compares, pages_from >= 0 and "
                         "pages_step >= 1")
    if row_idx is not None:
        kv8.want(row_idx, torch.int32, (row_idx.shape[0],), dev, "row_idx")
    _want_extra(row_sq, check, t, dev)
    if t == 0 or tiles.shape[0] == 0:
        return out
    if t * nkv <= FEW_ROWS and nq // nkv <= 16 and plan.table.shape[1] <= (1 << 24) // PAGE:
        return _prefill8_few(q, cache, plan, pos, tiles, out, row_idx, row_sq, scale, check)
    kv8.launch("sdc_kv8_expand", dev, (
        cache.codes.data_ptr(), cache.scales.data_ptr(), cache.num_blocks, plan.pages.data_ptr(), plan.pages.shape[0],
        nkv, plan.work.data_ptr(), pages_from, pages_step, kv8.ptr(check)))
    kv8.launch("sdc_attn_prefill_expanded", dev, (
        q.data_ptr(), out.data_ptr(), plan.work.data_ptr(), plan.work.shape[0], plan.table.data_ptr(),
        plan.table.shape[1], pos.data_ptr(), tiles.data_ptr(), tiles.shape[0], kv8.ptr(row_idx), nq, nkv,
        _SCALE if scale is None else scale, kv8.ptr(row_sq), kv8.ptr(check)))
    return out


def reference_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_pos: torch.Tensor) -> torch.Tensor:
    """fp32 reference for one request: q (t, nq, d), k/v (n, nkv, d), causal by absolute positions."""
    nq, nkv = q.shape[1], k.shape[1]
    g = nq // nkv
    kf = k.float().repeat_interleave(g, dim=1)
    vf = v.float().repeat_interleave(g, dim=1)
    s = torch.einsum("thd,nhd->htn", q.float(), kf) / math.sqrt(q.shape[-1])
    keys = torch.arange(k.shape[0], device=q.device)
    mask = keys[None, :] > q_pos[:, None]
    s = s.masked_fill(mask[None], float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.einsum("htn,nhd->thd", p, vf)
