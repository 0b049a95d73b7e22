"""Python entry points of the layer kernels in `csrc/layers.cu` and the exact replay comparison in
`csrc/checks.cu`. All take bf16 CUDA tensors and run on the current stream; optional `rows` index tensors
(int32, on the device) select rows for a replay of sampled rows."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _native
from . import kv8
from .kv8 import KV8Cache


def _s(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def add_rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
                resid_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                row_sq: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None,
                check: Optional[torch.Tensor] = None):
    """y = RMSNorm(x (+ residual)) * weight; h = x + residual written to resid_out (may alias residual);
    ||y_row||^2 to row_sq. Returns (y, row_sq). With `rows`, output row i is computed from input row rows[i].
    With `check` (a state row) and `rows`: replay check, rows rows[i] of `out` (the first run's output) are
    recomputed and compared, nothing is written."""
    m = x.shape[0] if rows is None else rows.shape[0]
    h = x.shape[-1]
    if out is None:
        out = torch.empty(m, h, dtype=torch.bfloat16, device=x.device)
    if row_sq is None and check is None:
        row_sq = torch.empty(m, dtype=torch.float32, device=x.device)
    _native.check(_native.lib().sdc_add_rmsnorm_bf16(
        x.data_ptr(), _p(residual), weight.data_ptr(), float(eps), m, h, out.data_ptr(), _p(resid_out),
        _p(row_sq), _p(rows), _p(check), _s(x)), "add_rmsnorm")
    return out, row_sq


def qk_norm_rope_kv(qkv: torch.Tensor, nq: int, nkv: int, pos: torch.Tensor, slots: torch.Tensor,
                    q_norm: Optional[torch.Tensor], k_norm: Optional[torch.Tensor], eps: float,
                    cos_sin: torch.Tensor, q_out: torch.Tensor, cache: torch.Tensor,
                    rows: Optional[torch.Tensor] = None, check: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Split the fused QKV output, per-head RMSNorm of q and k (when weights are given), RoPE, q -> q_out,
    k/v -> paged cache at `slots` (int64; -1 skips). With `check` (a state row), compare instead of write."""
    t = qkv.shape[0] if rows is None else rows.shape[0]
    _native.check(_native.lib().sdc_qk_norm_rope_kv(
        qkv.data_ptr(), qkv.stride(0), t, nq, nkv, 128, pos.data_ptr(), slots.data_ptr(), _p(q_norm), _p(k_norm),
        float(eps), cos_sin.data_ptr(), q_out.data_ptr(), cache.data_ptr(), _p(rows), _p(check), _s(qkv)),
        "qk_norm_rope_kv")
    return q_out


def qk_norm_rope_kv8(qkv: torch.Tensor, nq: int, nkv: int, pos: torch.Tensor, slots: torch.Tensor,
                     q_norm: Optional[torch.Tensor], k_norm: Optional[torch.Tensor], eps: float,
                     cos_sin: Optional[torch.Tensor], q_out: torch.Tensor, cache: KV8Cache, interleaved: bool = False,
                     rows: Optional[torch.Tensor] = None, check: Optional[torch.Tensor] = None) -> torch.Tensor:
    """qk_norm_rope_kv into a cache of 8 bits (`kv8.KV8Cache`, one layer): split the fused QKV projection (T, (nq +
    2 nkv) * 128), normalise q and k per head (where a weight is given), rotate them, q -> q_out (T, nq, 128), k and v
    -> the cache at `slots` (int64 block * 16 + place; negative: q only). All in fp32, each output rounded once.

    cos_sin: (positions, rotary / 2, 2) fp32 from `rope_table(positions, rotary, ...)`; the first `rotary` dims of a
    head (a multiple of 8) are rotated: dim i with dim i + rotary / 2, or, `interleaved`, dims 2i and 2i + 1. None: no
    rotation.

    The tokens that a call writes to one page are adjacent rows at places that follow one another, as a prompt's or a
    step's are: one warp sets the page's scale (a page in two runs, or a place twice, leaves what it holds undefined).
    What the page held before the first of them is kept, at the page's new scale; what it held behind them is dead.
    A token whose slot lies outside the cache, or whose position lies outside the table, is not stored, and its row of
    q_out is NaN. With `check` (a state row) and `rows`: the sampled tokens are recomputed and compared with q_out and
    the cache instead of written; this holds until a later call raises the scale of their page."""
    shape, stride = qkv.shape, qkv.stride()              # (each read of a tensor's attribute costs a tenth of a microsecond)
    t, heads, dev = shape[0], nq + 2 * nkv, cache.device
    if not cache.one_layer or cache.nkv != nkv:
        raise ValueError(f"cache must be one layer with {nkv} kv heads, got {tuple(cache.codes.shape)}")
    at = qkv.data_ptr()
    if shape != (t, heads * 128) or qkv.dtype is not torch.bfloat16 or qkv.device != dev or at % 8 or stride[1] != 1 \
            or (t > 1 and stride[0] % 4):
        raise ValueError(f"qkv must be bf16 (T, {heads * 128}) on {dev} with contiguous rows on 8-byte boundaries")
    kv8.want(q_out, torch.bfloat16, (t, nq, 128), dev, "q_out", align=8)
    kv8.want(pos, torch.int32, (t,), dev, "pos")
    kv8.want(slots, torch.int64, (t,), dev, "slots")
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None:
            kv8.want(w, torch.bfloat16, (128,), dev, name, align=8)
    table_rows = rotary = 0
    if cos_sin is not None:
        shape = cos_sin.shape
        table_rows, rotary = shape[0], 2 * shape[1]
        kv8.want(cos_sin, torch.float32, (table_rows, rotary // 2, 2), dev, "cos_sin", align=16)
        if rotary % 8 or not 0 < rotary <= 128:
            raise ValueError(f"{rotary} rotated dims: a multiple of 8, at most 128")
    if (rows is None) != (check is None):
        raise ValueError("rows and check go together")
    if rows is not None:
        kv8.want(rows, torch.int32, (rows.shape[0],), dev, "rows")
        kv8.want_state(check, dev)
    kv8.launch("sdc_kv8_append", dev, (
        at, stride[0] if t > 1 else heads * 128, t, nq, nkv, pos.data_ptr(), slots.data_ptr(),
        kv8.ptr(q_norm), kv8.ptr(k_norm), eps, kv8.ptr(cos_sin), table_rows, rotary, interleaved, q_out.data_ptr(),
        cache.codes.data_ptr(), cache.scales.data_ptr(), cache.num_blocks, kv8.ptr(rows),
        0 if rows is None else rows.shape[0], kv8.ptr(check)))
    return q_out


def silu_mul(gu: torch.Tensor, out: Optional[torch.Tensor] = None, row_sq: Optional[torch.Tensor] = None,
             rows: Optional[torch.Tensor] = None, check: Optional[torch.Tensor] = None):
    """out = silu(gate) * up with ||out_row||^2; `rows` / `check` as in add_rmsnorm (replay check in place)."""
    m = gu.shape[0] if rows is None else rows.shape[0]
    i = gu.shape[-1] // 2
    if out is None:
        out = torch.empty(m, i, dtype=torch.bfloat16, device=gu.device)
    if row_sq is None and check is None:
        row_sq = torch.empty(m, dtype=torch.float32, device=gu.device)
    _native.check(_native.lib().sdc_silu_mul_bf16(gu.data_ptr(), m, i, out.data_ptr(), _p(row_sq), _p(rows),
                                                   _p(check), _s(gu)), "silu_mul")
    return out, row_sq


def silu_mul_bands(gu: torch.Tensor, gcount: torch.Tensor, out: Optional[torch.Tensor] = None,
                   row_sq: Optional[torch.Tensor] = None):
    """silu_mul over grouped expert rows: only the first 128 * gcount rows (gcount on the device) are computed."""
    m, i = gu.shape[0], gu.shape[-1] // 2
    if out is None:
        out = torch.empty(m, i, dtype=torch.bfloat16, device=gu.device)
    if row_sq is None:
        row_sq = torch.empty(m, dtype=torch.float32, device=gu.device)
    _native.check(_native.lib().sdc_silu_mul_bf16_bands(gu.data_ptr(), m, i, out.data_ptr(), row_sq.data_ptr(),
                                                        gcount.data_ptr(), _s(gu)), "silu_mul (bands)")
    return out, row_sq


def compare_rows(a: torch.Tensor, idx: Optional[torch.Tensor], b: torch.Tensor, state_row: torch.Tensor) -> None:
    """Exact comparison of replayed rows b[i] with a[idx[i]] (2-D bf16); mismatches go to `state_row`."""
    s = b.shape[0]
    _native.check(_native.lib().sdc_compare_rows_bf16(
        a.data_ptr(), a.stride(0), _p(idx), b.data_ptr(), b.stride(0), a.shape[-1], s, state_row.data_ptr(), _s(a)),
        "compare_rows")


def rope_table(max_pos: int, head_dim: int, theta: float, scaling: Optional[dict] = None,
               device="cuda") -> torch.Tensor:
    """(max_pos, head_dim / 2) float2 table of (cos, sin) for the rotate-half RoPE; `scaling` follows the
    Llama-3 frequency rule (factor, low_freq_factor, high_freq_factor, original_max_position_embeddings)."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim))
    if scaling:
        import math
        factor = scaling["factor"]
        lo, hi = scaling["low_freq_factor"], scaling["high_freq_factor"]
        old = scaling["original_max_position_embeddings"]
        lo_wl, hi_wl = old / lo, old / hi
        wl = 2 * math.pi / inv
        smooth = (old / wl - lo) / (hi - lo)
        scaled = torch.where(wl > lo_wl, inv / factor, inv)
        mid = (wl <= lo_wl) & (wl >= hi_wl)
        inv = torch.where(mid, (1 - smooth) * inv / factor + smooth * inv, scaled)
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv[None, :]
    tab = torch.stack([ang.cos(), ang.sin()], dim=-1).float()
    return tab.contiguous().to(device)
