"""Paged KV cache held in 8 bits (`csrc/kv8.cu`): half the bytes of the bf16 cache in memory and in every decode step.

    cache = KV8Cache.empty(num_blocks, nkv, layers=28, device="cuda")
    layers.qk_norm_rope_kv8(qkv, nq, nkv, pos, slots, q_norm, k_norm, eps, cos_sin, q, cache[i])     # append
    attention.prefill8(q, cache[i], prefill_plan, pos, tiles)
    attention.decode8(q, cache[i], block_table, seq_req, ctx, decode_plan)

Keys and values are E4M3 codes with one float32 scale for each page of 16 tokens, kv head and K / V; a value is code *
scale. Appending makes every scale a power of two, the least that holds the page's largest value: moving a page to a
larger scale then changes no code above E4M3's subnormal range, and a value is exact in bf16. A value that is not
finite is stored as NaN. The layout is the bf16 cache's, [blocks][2 (K, V)][kv heads][16][128], a byte an element.
"""
from __future__ import annotations

import contextlib
from typing import Optional

import torch

from .. import _native

PAGE = 16
HEAD_DIM = 128
E4M3_MAX = 448.0
LEAST_SCALE = 2.0 ** -60


def want(t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: torch.device, name: str,
         align: int = 1) -> torch.Tensor:
    """t, if it is a contiguous `dtype` tensor of `shape` on `device` on an `align`-byte boundary (a kernel takes its
    address); ValueError otherwise."""
    if t.dtype is dtype and t.shape == shape and t.device == device and t.is_contiguous() \
            and (align == 1 or t.data_ptr() % align == 0):
        return t
    raise ValueError(f"{name} must be contiguous {dtype} {tuple(shape)} on {device}, aligned to {align} bytes, got "
                     f"{t.dtype} {tuple(t.shape)} on {t.device}")


def want_state(check: torch.Tensor, device: torch.device) -> None:
    """ValueError unless `check` is a state row (a check mode's kernel writes all of it)."""
    if check.dtype is not torch.int64 or check.numel() != 4 or check.device != device or not check.is_contiguous():
        raise ValueError(f"check must be a state row (4 contiguous int64) on {device}, got {check.dtype} "
                         f"{tuple(check.shape)} on {check.device}")


_here, _stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


_same = contextlib.nullcontext()


def on(device: torch.device):
    """The context in which a launch on `device` belongs: a kernel starts on the current device."""
    if device.index is None:
        raise ValueError(f"the kernels run on a CUDA device, not on {device}")
    return _same if _here() == device.index else torch.cuda.device(device.index)


def stream(device: torch.device) -> int:
    """`device`'s current stream as a bare handle."""
    if device.index is None:
        raise ValueError(f"the kernels run on a CUDA device, not on {device}")
    return _stream(device.index)


def launch(entry: str, device: torch.device, args: tuple) -> None:
    """Calls the library's `entry` with args (addresses as integers, 0 for none) and `device`'s current stream. (These
    operators run for a few microseconds: the arguments cross as one struct, and the stream is taken as the bare
    handle.)"""
    index = device.index
    if index is None or index != _here():
        with on(device):
            return launch(entry, device, args)
    rc = getattr(_native.lib(), entry)(_native.STRUCTS[entry].pack(*args, _stream(index)))
    if rc:
        _native.check(rc, entry)


def ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


class KV8Cache:
    """codes float8_e4m3fn [(layers,) blocks, 2, kv heads, 16, 128], scales float32 [(layers,) blocks, kv heads, 2 (K,
    V)]; `cache[i]` is layer i. A page that was never written has scale 0 and reads as zeros."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != torch.float8_e4m3fn or codes.dim() not in (5, 6) or codes.shape[-2:] != (PAGE, HEAD_DIM) \
                or codes.shape[-4] != 2 or not codes.is_contiguous() or codes.data_ptr() % 16:
            raise ValueError(f"codes must be contiguous float8_e4m3fn [(layers,) blocks, 2, kv heads, {PAGE}, "
                             f"{HEAD_DIM}], got {codes.dtype} {tuple(codes.shape)}")
        shape = tuple(codes.shape[:-4]) + (codes.shape[-3], 2)
        if scales.dtype != torch.float32 or tuple(scales.shape) != shape or not scales.is_contiguous() \
                or scales.device != codes.device or scales.data_ptr() % 8:
            raise ValueError(f"scales must be contiguous float32 {shape} on {codes.device}")
        self.codes, self.scales, self.device = codes, scales, codes.device
        self.one_layer = codes.dim() == 5
        self.num_blocks, self.nkv = codes.shape[-5], codes.shape[-3]
        self._layers = [None] * codes.shape[0] if codes.dim() == 6 else []

    @classmethod
    def empty(cls, num_blocks: int, nkv: int, layers: Optional[int] = None, device="cuda") -> "KV8Cache":
        lead = () if layers is None else (layers,)
        codes = torch.zeros(*lead, num_blocks, 2, nkv, PAGE, HEAD_DIM, dtype=torch.uint8, device=device)
        return cls(codes.view(torch.float8_e4m3fn),
                   torch.zeros(*lead, num_blocks, nkv, 2, dtype=torch.float32, device=device))

    def __len__(self) -> int:
        return len(self._layers)

    def __getitem__(self, i: int) -> "KV8Cache":
        if not self._layers:
            raise IndexError("this is one layer's cache")
        if self._layers[i] is None:
            self._layers[i] = KV8Cache(self.codes[i], self.scales[i])
        return self._layers[i]

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def dtype(self) -> torch.dtype:
        return self.codes.dtype

    def values(self, pages: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The stored values in float32 (of one layer; of the given pages): [pages, 2, kv heads, 16, 128]."""
        codes, scales = (self.codes, self.scales) if pages is None else (self.codes[pages], self.scales[pages])
        return codes.float() * scales.transpose(-1, -2)[..., None, None]


def page_bytes(nkv: int) -> int:
    """Bytes of one page of one layer: codes and scales."""
    return 2 * nkv * (PAGE * HEAD_DIM + 4)
