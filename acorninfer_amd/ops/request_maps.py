"""Block tables and slot maps from the lengths of requests, built on the GPU.

- `block_tables`  a flat list of blocks, ceil(length / P) to a request -> padded tables
- `slot_map`      packed rows -> the request, position, page and slot of each

They give what `ops.paged_attention.build_tables` and `PagedCacheView.reserve` give on
the host, as the attention kernels and the caches' writers read it, from a few bytes per
request. `Qwen3DecodeModel.forward_extend` packs its prompts with them, and
`engine.beam.BeamSearch` runs `slot_map` inside its captured step. Kernels:
csrc/request_maps.hip. Everything launches on the current stream of its tensors' device,
never synchronises, and can be captured in a graph.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from acorninfer_amd._lib import launch, one_device


class SlotMap(NamedTuple):
    """Of every packed row [R]: its request (int32), position (int64), page and slot in the cache
    (int64; page -1: none, which writers skip), and length (int32, position + 1); row0 [N] int32:
    each request's first row."""
    seq: torch.Tensor
    positions: torch.Tensor
    pages: torch.Tensor
    slots: torch.Tensor
    lens: torch.Tensor
    row0: torch.Tensor


_MAP_DTYPES = (torch.int32, torch.int64, torch.int64, torch.int64, torch.int32, torch.int32)


def _page_size(page_size: int) -> int:
    P = int(page_size)
    assert 1 <= P <= 1 << 30 and P & (P - 1) == 0, f"page_size {P} must be a power of two"
    return P


def block_tables(blocks: torch.Tensor, lengths: torch.Tensor, page_size: int, width: int, *,
                 pad: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Tables [N, width] int32: request n holds the next ceil(lengths[n] / page_size) entries of
    `blocks` [T] int32 (a length below 1 none), of which its row gets the first `width`; `pad`
    fills the rest, and what the list has no block for. lengths [N] int32."""
    P, width = _page_size(page_size), int(width)
    assert blocks.dtype is torch.int32 and blocks.dim() == 1 and blocks.is_contiguous(), \
        "blocks are contiguous int32 [T]"
    assert lengths.dtype is torch.int32 and lengths.dim() == 1 and lengths.is_contiguous(), \
        "lengths are contiguous int32 [N]"
    assert width >= 1, "tables hold at least one page per request"
    N = lengths.shape[0]
    if out is None:
        dev = one_device(blocks, lengths)
        out = lengths.new_empty((N, width))
    else:
        assert out.dtype is torch.int32 and out.shape == (N, width) and out.is_contiguous(), \
            f"out is contiguous int32 {[N, width]}"
        dev = one_device(blocks, lengths, out)
    launch("block_tables", dev, blocks.data_ptr(), blocks.shape[0], lengths.data_ptr(),
           out.data_ptr(), N, width, P, int(pad))
    return out


def slot_map(tables: torch.Tensor, starts: torch.Tensor, counts: torch.Tensor, page_size: int,
             rows: int, *, out: SlotMap | None = None) -> SlotMap:
    """The map of `rows` packed rows: request n brings counts[n] of them (below 1: none), its tokens
    starts[n], starts[n] + 1, ... (both [N] int32), which lie in the pages of tables[n] [N, width]
    int32. Rows that no request brings are not written (in a new map: undefined); requests past
    `rows` are cut off."""
    P, R = _page_size(page_size), int(rows)
    assert tables.dtype is torch.int32 and tables.dim() == 2 and tables.is_contiguous(), \
        "tables are contiguous int32 [N, pages]"
    N, W = tables.shape
    for t in (starts, counts):
        assert t.dtype is torch.int32 and t.shape == (N,) and t.is_contiguous(), \
            "starts and counts are contiguous int32, one per request"
    assert R >= 0 and (W >= 1 or N == 0), "tables hold at least one page per request"
    if out is None:
        dev = one_device(tables, starts, counts)
        seq, lens, row0 = tables.new_empty((2 * R + N,)).split((R, R, N))
        out = SlotMap(seq, *tables.new_empty((3, R), dtype=torch.int64).unbind(), lens, row0)
    else:
        for name, t, dtype in zip(SlotMap._fields, out, _MAP_DTYPES):
            n = N if name == "row0" else R
            assert t.dtype is dtype and t.shape == (n,) and t.is_contiguous(), \
                f"out.{name} is contiguous {dtype} [{n}]"
        dev = one_device(tables, starts, counts, *out)
    launch("slot_map", dev, tables.data_ptr(), starts.data_ptr(), counts.data_ptr(),
           *(t.data_ptr() for t in out), N, R, max(1, W), P)
    return out
