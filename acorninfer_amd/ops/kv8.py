"""The 8-bit paged KV cache: its pages, writing and reading them, and attention.

A layer's cache is a `KV8Pages` of three uint8 tensors: K and V tiles of 16
tokens each, e4m3 bytes, and per (token, kv head) a power-of-two scale code for
k and one for v (2 D + 2 bytes, against 4 D in 16 bits). Format and layout are
stated in include/acorn_hip.h; tiles lie in the order the attention kernels
load them, so programs go through the functions here:

- `kv8_scatter`                   rows of k and v into the cache
- `qkv_norm_rope_kv8`             a qkv projection's output into q and the cache
- `kv8_gather`                    tokens of sequences back into 16 or 32 bits
- `paged_decode_attention_kv8`    one new token per sequence
- `paged_prefill_attention_kv8`   packed prompt rows, causal
- `paged_verify_attention_kv8`    a window of drafted tokens per sequence

They stand beside ops/paged_attention.py and ops/paged_verify.py (the 16-bit
cache) with the same block tables, lengths and row metadata. Kernels:
csrc/kv8_cache.hip, csrc/kv8_attention.hip. Shapes: head_dim 64 or 128, pages of
a power-of-two multiple of 16 tokens; attention in bf16 or fp16 with 1, 2, 4 or
8 q heads per kv head. Everything launches on the current stream of its
tensors' device, never synchronises, and can be captured in a graph. Calls that
overlap must not share an `out` or `workspace`.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from acorninfer_amd._lib import check, dtype_code, lib, ptr, require_gpu, stream_ptr

GROUP = 16               # tokens of a tile
MI355X_CUS = 256


class KV8Pages(NamedTuple):
    """One layer's pages: k, v uint8 [num_blocks, KV, P // 16, 16 * D], scales uint8
    [num_blocks, KV, P // 16, 32]. Zeros are an empty cache."""
    k: torch.Tensor
    v: torch.Tensor
    scales: torch.Tensor

    @property
    def num_blocks(self) -> int:
        return self.k.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2] * GROUP

    @property
    def head_dim(self) -> int:
        return self.k.shape[3] // GROUP


def kv8_supported(head_dim: int, page_size: int) -> bool:
    """Shapes the 8-bit cache is built for."""
    return (head_dim in (64, 128) and page_size >= GROUP and page_size <= 65536
            and page_size & (page_size - 1) == 0)


def kv8_attention_supported(dtype: torch.dtype, head_dim: int, page_size: int, num_heads: int,
                            kv_heads: int) -> bool:
    """Shapes the attention over it is built for."""
    return (dtype in (torch.bfloat16, torch.float16) and kv8_supported(head_dim, page_size)
            and num_heads % kv_heads == 0 and num_heads // kv_heads in (1, 2, 4, 8))


def kv8_pages(num_blocks: int, kv_heads: int, head_dim: int, page_size: int, device) -> KV8Pages:
    """Empty pages of one layer."""
    if not kv8_supported(head_dim, page_size):
        raise NotImplementedError(f"8-bit cache: head_dim {head_dim}, page_size {page_size}")
    shape = (num_blocks, kv_heads, page_size // GROUP)
    return KV8Pages(*(torch.zeros(*shape, n, dtype=torch.uint8, device=device)
                      for n in (GROUP * head_dim, GROUP * head_dim, 2 * GROUP)))


def _check_pages(kv: KV8Pages) -> None:
    k, v, s = kv
    assert k.dim() == 4 and k.shape == v.shape and k.shape[3] % GROUP == 0, \
        "tiles are [num_blocks, KV, P // 16, 16 * D]"
    assert s.shape == (*k.shape[:3], 2 * GROUP), "scales are [num_blocks, KV, P // 16, 32]"
    for t in kv:
        assert t.dtype == torch.uint8 and t.is_contiguous(), "pages are contiguous uint8"


def _on(device: torch.device, *tensors) -> None:
    """Kernels launch on one device's stream and reach every tensor by its pointer."""
    require_gpu(*tensors)
    for t in tensors:
        assert t is None or t.device == device, f"tensors on {t.device} and {device}"


def _check_targets(pages: torch.Tensor, slots: torch.Tensor, rows: int) -> None:
    for t in (pages, slots):
        assert t.shape == (rows,) and t.dtype == torch.int64 and t.is_contiguous(), \
            "pages and slots are contiguous int64, one per row"


def _check_tables(kv: KV8Pages, N: int, tables: torch.Tensor, *meta: torch.Tensor) -> int:
    """Block tables and per-sequence metadata; the table's width (1 for an empty batch)."""
    assert tables.dim() == 2 and tables.shape[0] == N
    for t in meta:
        assert t.shape == (N,)
    for t in (tables, *meta):
        assert t.dtype == torch.int32 and t.is_contiguous(), "tables and metadata are int32"
    assert N == 0 or tables.shape[1] >= 1, "tables must hold at least one page per sequence"
    return max(1, tables.shape[1])


def _check_out(out: torch.Tensor, shape: tuple, dtype: torch.dtype, device) -> None:
    assert tuple(out.shape) == tuple(shape), f"out must be {tuple(shape)}, not {tuple(out.shape)}"
    assert out.dtype == dtype, f"out dtype {out.dtype} != {dtype}"
    assert out.device == device and out.is_contiguous(), "out must be contiguous on the inputs' device"


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [R, KV, D] as the kernel reads it: dims side by side, each lane's D / 16 values aligned."""
    size = x.element_size()
    step = min(16, x.shape[2] // 16 * size)
    if x.stride(2) != 1 or x.data_ptr() % step or any(x.stride(i) * size % step for i in (0, 1)):
        x = x.contiguous()
        if x.data_ptr() % step:
            x = x.clone()
    return x


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """x contiguous from a 16-byte boundary (a view into a tensor may start anywhere)."""
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def kv8_scatter(k: torch.Tensor, v: torch.Tensor, kv: KV8Pages, pages: torch.Tensor,
                slots: torch.Tensor) -> None:
    """Quantise rows k, v [R, KV, D] (fp32 / fp16 / bf16, any strides) into the cache at
    (pages[i], slots[i]) (int64). A target outside the pool is skipped, as in
    PagedKVCache.scatter_decode; two rows with one target leave it undefined."""
    _check_pages(kv)
    dev = kv.k.device
    _on(dev, *kv, k, v, pages, slots)
    assert k.dim() == 3 and k.shape == v.shape and k.shape[1:] == (kv.kv_heads, kv.head_dim), \
        f"k is {tuple(k.shape)}, v {tuple(v.shape)}; the pool holds {kv.kv_heads} kv heads of " \
        f"{kv.head_dim}"
    assert k.dtype == v.dtype
    R = k.shape[0]
    _check_targets(pages, slots, R)
    k, v = _rows(k), _rows(v)
    with torch.cuda.device(dev):
        rc = lib().acorn_kv8_scatter(
            ptr(k), ptr(v), *map(ptr, kv), ptr(pages), ptr(slots), R, kv.kv_heads, kv.head_dim,
            kv.page_size, kv.num_blocks, k.stride(0), k.stride(1), v.stride(0), v.stride(1),
            dtype_code(k), stream_ptr(dev))
    check(rc, "kv8_scatter")


def kv8_gather(kv: KV8Pages, tables: torch.Tensor, seq_row0: torch.Tensor, seq_pos0: torch.Tensor,
               seq_nq: torch.Tensor, max_nq: int, rows: int, *,
               dtype: torch.dtype = torch.bfloat16,
               out: tuple[torch.Tensor, torch.Tensor] | None = None
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """The cache read back: k, v [rows, KV, D] of `dtype`, where row seq_row0[n] + j holds token
    seq_pos0[n] + j (j < seq_nq[n] <= max_nq) of the sequence with block table tables[n]. Rows
    that no sequence covers, or past their table row's pages, are not written."""
    _check_pages(kv)
    dev = kv.k.device
    _on(dev, *kv, tables, seq_row0, seq_pos0, seq_nq)
    W = _check_tables(kv, seq_row0.shape[0], tables, seq_row0, seq_pos0, seq_nq)
    shape = (int(rows), kv.kv_heads, kv.head_dim)
    assert int(rows) >= 0 and int(max_nq) >= 0
    if out is None:
        out = (torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev))
    for o in out:
        _check_out(o, shape, dtype, dev)
    with torch.cuda.device(dev):
        rc = lib().acorn_kv8_gather(
            *map(ptr, kv), ptr(tables), ptr(seq_row0), ptr(seq_pos0), ptr(seq_nq), ptr(out[0]),
            ptr(out[1]), seq_row0.shape[0], int(rows), int(max_nq), kv.kv_heads, kv.head_dim,
            kv.page_size, kv.num_blocks, W, dtype_code(out[0]), stream_ptr(dev))
    check(rc, "kv8_gather")
    return out


def qkv_norm_rope_kv8(qkv: torch.Tensor, kv: KV8Pages, pages: torch.Tensor, slots: torch.Tensor,
                      positions: torch.Tensor, inv_freq: torch.Tensor, q_weight: torch.Tensor,
                      k_weight: torch.Tensor, eps: float, q_heads: int, *,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Between the qkv projection and attention: qkv [R, (H + 2 KV) * D] in the activation dtype,
    or fp32 [S, R, (H + 2 KV) * D] (the planes of a split product, added in order). Returns q
    [R, H, D] (per-head RMSNorm with q_weight [D], RoPE at positions [R] int64 with inv_freq
    [D / 2] fp32) in q_weight's dtype; k (the same with k_weight) and v are quantised into the
    cache at (pages[i], slots[i]), straight from their 32-bit values."""
    _check_pages(kv)
    dev = kv.k.device
    _on(dev, *kv, qkv, pages, slots, positions, inv_freq, q_weight, k_weight)
    H, KV, D = int(q_heads), kv.kv_heads, kv.head_dim
    dtype = q_weight.dtype
    assert qkv.dim() in (2, 3) and qkv.shape[-1] == (H + 2 * KV) * D and H >= 1, \
        f"qkv rows hold {(H + 2 * KV) * D} values"
    assert qkv.dtype == (torch.float32 if qkv.dim() == 3 else dtype), \
        "qkv is [S, R, width] fp32 or [R, width] of the weights' dtype"
    planes = qkv.shape[0] if qkv.dim() == 3 else 0
    assert qkv.dim() == 2 or planes >= 1
    R = qkv.shape[-2]
    _check_targets(pages, slots, R)
    assert positions.shape == (R,) and positions.dtype == torch.int64 and positions.is_contiguous()
    assert inv_freq.shape == (D // 2,) and inv_freq.dtype == torch.float32 and inv_freq.is_contiguous()
    assert q_weight.shape == k_weight.shape == (D,) and k_weight.dtype == dtype
    qkv, qw, kw = _aligned(qkv), _aligned(q_weight), _aligned(k_weight)
    if out is None:
        out = torch.empty((R, H, D), dtype=dtype, device=dev)
    _check_out(out, (R, H, D), dtype, dev)
    with torch.cuda.device(dev):
        rc = lib().acorn_qkv_epilogue_kv8(
            ptr(qkv), planes, ptr(out), *map(ptr, kv), ptr(pages), ptr(slots), R, H, KV, D,
            kv.page_size, kv.num_blocks, ptr(qw), ptr(kw), float(eps), ptr(positions),
            ptr(inv_freq), dtype_code(out), stream_ptr(dev))
    check(rc, "qkv_norm_rope_kv8")
    return out


def kv8_splits(batch: int, kv_heads: int, max_pages: int, page_size: int) -> int:
    """Splits of the cache's length for paged_decode_attention_kv8 over block tables max_pages
    wide."""
    groups = max_pages * (page_size // GROUP)
    pairs = max(1, batch * kv_heads)
    if groups <= 64 or pairs >= 4 * MI355X_CUS:
        return 1
    unit = max(1, 16 // (page_size // GROUP))
    return max(1, min(-(-max_pages // unit), 64))


def kv8_workspace(batch: int, num_heads: int, head_dim: int, num_splits: int, device
                  ) -> tuple[torch.Tensor, torch.Tensor] | None:
    """The partials of num_splits splits (None for one)."""
    if num_splits <= 1:
        return None
    n = batch * num_heads * num_splits
    return (torch.empty(n * head_dim, dtype=torch.float32, device=device),
            torch.empty(2 * n, dtype=torch.float32, device=device))


def _check_attention(q: torch.Tensor, kv: KV8Pages) -> None:
    assert q.shape[-1] == kv.head_dim and q.shape[-2] % kv.kv_heads == 0, \
        f"q heads {tuple(q.shape[-2:])} over {kv.kv_heads} kv heads of {kv.head_dim}"
    if not kv8_attention_supported(q.dtype, kv.head_dim, kv.page_size, q.shape[-2], kv.kv_heads):
        raise NotImplementedError(
            f"attention over the 8-bit cache: {q.dtype}, head_dim {kv.head_dim}, page_size "
            f"{kv.page_size}, {q.shape[-2]} / {kv.kv_heads} heads")


def paged_decode_attention_kv8(q: torch.Tensor, kv: KV8Pages, tables: torch.Tensor,
                               seq_lens: torch.Tensor, num_splits: int | None = None, *,
                               out: torch.Tensor | None = None,
                               workspace: tuple[torch.Tensor, torch.Tensor] | None = None
                               ) -> torch.Tensor:
    """paged_decode_attention over the 8-bit cache. q [B, H, D] bf16 / fp16 (normed + roped);
    tables [B, MP] int32; seq_lens [B] int32 (including the current token); returns [B, H, D].
    num_splits page-aligned splits of a sequence (None: kv8_splits). `out` / `workspace`
    (kv8_workspace of the same sizes) let a caller pass address-stable buffers. A length is taken
    as at most the tokens its table row has pages for; a row that sees no token is NaN."""
    _check_pages(kv)
    dev = q.device
    _on(dev, q, *kv, tables, seq_lens)
    assert q.dim() == 3
    B, H, D = q.shape
    _check_attention(q, kv)
    W = _check_tables(kv, B, tables, seq_lens)
    S = kv8_splits(B, kv.kv_heads, W, kv.page_size) if num_splits is None else int(num_splits)
    assert S >= 1
    q2 = _aligned(q)
    if out is None:
        out = torch.empty((B, H, D), dtype=q.dtype, device=dev)
    _check_out(out, (B, H, D), q.dtype, dev)
    if workspace is None:
        workspace = kv8_workspace(B, H, D, S, dev)
    acc, ml = workspace if workspace is not None and S > 1 else (None, None)
    if S > 1:
        for t, n in ((acc, B * H * S * D), (ml, 2 * B * H * S)):
            assert t.dtype == torch.float32 and t.is_contiguous() and t.numel() >= n and \
                t.device == dev, "workspace: kv8_workspace of the same sizes"
    with torch.cuda.device(dev):
        rc = lib().acorn_paged_attention_kv8(
            ptr(q2), *map(ptr, kv), ptr(tables), ptr(seq_lens), ptr(out), ptr(acc), ptr(ml), B, H,
            kv.kv_heads, D, kv.page_size, kv.num_blocks, W, S, float(D ** -0.5), dtype_code(q2),
            stream_ptr(dev))
    check(rc, "paged_decode_attention_kv8")
    return out


@functools.lru_cache(maxsize=1024)
def _prefill_workspace_bytes(*sizes: int) -> int:
    n = ctypes.c_int64(0)
    check(lib().acorn_paged_prefill_workspace_kv8(*sizes, ctypes.byref(n)),
          "paged_prefill_workspace_kv8")
    return n.value


def prefill_workspace_kv8(N: int, R: int, max_nq: int, H: int, KV: int, D: int, P: int,
                          table_width: int, device) -> torch.Tensor | None:
    """The workspace a prefill launch of these sizes splits its keys over, or None."""
    n = _prefill_workspace_bytes(N, R, max_nq, H, KV, D, P, table_width)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _prefill(q2, kv, tables, row0, pos0, nq, out, N, R, max_nq, W) -> None:
    H, D = q2.shape[-2:]
    dev = q2.device
    ws = prefill_workspace_kv8(N, R, max_nq, H, kv.kv_heads, D, kv.page_size, W, dev)
    with torch.cuda.device(dev):
        rc = lib().acorn_paged_prefill_attention_kv8(
            ptr(q2), *map(ptr, kv), ptr(tables), ptr(row0), ptr(pos0), ptr(nq), ptr(out), N, R,
            max_nq, H, kv.kv_heads, D, kv.page_size, kv.num_blocks, W, float(D ** -0.5),
            dtype_code(q2), ptr(ws), 0 if ws is None else ws.numel(), stream_ptr(dev))
    check(rc, "paged_prefill_attention_kv8")


def paged_prefill_attention_kv8(q: torch.Tensor, kv: KV8Pages, tables: torch.Tensor,
                                seq_row0: torch.Tensor, seq_pos0: torch.Tensor,
                                seq_nq: torch.Tensor, max_nq: int, *,
                                out: torch.Tensor | None = None) -> torch.Tensor:
    """paged_prefill_attention over the 8-bit cache. q [R, H, D]: the prompt rows of N sequences,
    packed; row j of sequence n, q[seq_row0[n] + j] (j < seq_nq[n] <= max_nq), sits at position
    seq_pos0[n] + j and attends to the sequence's tokens 0 .. its own position, which are in the
    cache. Rows not covered by a sequence, or past their table row's pages, are left as they were
    in `out`."""
    _check_pages(kv)
    dev = q.device
    _on(dev, q, *kv, tables, seq_row0, seq_pos0, seq_nq)
    assert q.dim() == 3
    R, H, D = q.shape
    _check_attention(q, kv)
    N = seq_row0.shape[0]
    W = _check_tables(kv, N, tables, seq_row0, seq_pos0, seq_nq)
    assert int(max_nq) >= 0
    q2 = _aligned(q)
    if out is None:
        out = torch.empty((R, H, D), dtype=q.dtype, device=dev)
    _check_out(out, (R, H, D), q.dtype, dev)
    _prefill(q2, kv, tables, seq_row0, seq_pos0, seq_nq, out, N, R, int(max_nq), W)
    return out


def paged_verify_attention_kv8(q: torch.Tensor, kv: KV8Pages, tables: torch.Tensor,
                               seq_lens: torch.Tensor) -> torch.Tensor:
    """paged_verify_attention over the 8-bit cache: q [B, m, H, D], the m last positions of each
    sequence; seq_lens [B] counts them. Row (b, j) sees seq_lens[b] - (m - 1 - j) tokens; one
    that sees none is NaN. Windows of one token are decode."""
    assert q.dim() == 4
    B, M, H, D = q.shape
    assert M >= 1, "verify window must be non-empty"
    if M == 1:
        return paged_decode_attention_kv8(q[:, 0], kv, tables, seq_lens)[:, None]
    _check_pages(kv)
    dev = q.device
    _on(dev, q, *kv, tables, seq_lens)
    _check_attention(q, kv)
    W = _check_tables(kv, B, tables, seq_lens)
    q2 = _aligned(q)
    out = torch.empty_like(q2)
    _prefill(q2, kv, tables, None, seq_lens, None, out, B, B * M, M, W)
    return out
