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

# (the stream's handle without a Stream object around it: a microsecond of a call's ten)
from torch._C import _cuda_getCurrentRawStream as _raw_stream

from acorninfer_amd._lib import check, dtype_code, lib, ptr, require_gpu

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


# The checks of a call take a few microseconds on the host, as long as a small launch takes on
# the GPU: they look at each tensor once and at nothing that a tensor property does not hold.
def _pool(kv: KV8Pages) -> tuple[int, int, int, int]:
    """(num_blocks, kv_heads, head_dim, page_size) of pages that are as they should be."""
    k, v, s = kv
    shape = k.shape
    assert len(shape) == 4 and shape == v.shape and shape[3] % GROUP == 0, \
        "tiles are [num_blocks, KV, P // 16, 16 * D]"
    NB, KV, G, n = shape
    assert s.shape == (NB, KV, G, 2 * GROUP), "scales are [num_blocks, KV, P // 16, 32]"
    assert k.dtype is v.dtype is s.dtype is torch.uint8 and k.is_contiguous() and \
        v.is_contiguous() and s.is_contiguous(), "pages are contiguous uint8"
    return NB, KV, n // GROUP, G * GROUP


def _device(first: torch.Tensor, *tensors: torch.Tensor) -> int:
    """The index of the one GPU that holds the tensors: a kernel launches on one device's stream
    and reaches every tensor by its pointer."""
    dev = first.get_device()
    for t in tensors:
        if t.get_device() != dev:
            require_gpu(first, *tensors)
            raise AssertionError(f"tensors on {first.device} and {t.device}")
    if dev < 0:
        require_gpu(first)
    return dev


def _call(name: str, dev: int, *args) -> None:
    """Launch on the current stream of device `dev`, with that device current."""
    fn = getattr(lib(), "acorn_" + name)
    if torch.cuda.current_device() == dev:
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        check(rc, name)


def _check_targets(pages: torch.Tensor, slots: torch.Tensor, rows: int) -> None:
    for t in (pages, slots):
        assert t.dtype is torch.int64 and t.shape == (rows,) and t.is_contiguous(), \
            "pages and slots are contiguous int64, one per row"


def _check_tables(N: int, tables: torch.Tensor, *meta: torch.Tensor) -> int:
    """Block tables and per-sequence metadata; the table's width (1 for an empty batch)."""
    for t in meta:
        assert t.dtype is torch.int32 and t.shape == (N,) and t.is_contiguous(), \
            "lengths and metadata are contiguous int32, one per sequence"
    assert tables.dtype is torch.int32 and tables.dim() == 2 and tables.is_contiguous(), \
        "tables are contiguous int32 [N, pages]"
    n, W = tables.shape
    assert n == N and (W >= 1 or N == 0), "tables must hold at least one page per sequence"
    return max(1, W)


def _check_out(out: torch.Tensor, shape: tuple, dtype: torch.dtype, dev: int) -> None:
    assert tuple(out.shape) == tuple(shape), f"out must be {tuple(shape)}, not {tuple(out.shape)}"
    assert out.dtype == dtype, f"out dtype {out.dtype} != {dtype}"
    assert out.get_device() == dev and out.is_contiguous() and out.data_ptr() % 16 == 0, \
        "out must be contiguous on the inputs' device, from a 16-byte boundary"


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [R, KV, D] as the kernel reads it: dims side by side, each lane's D / 16 values aligned."""
    size = x.element_size()
    step = min(16, x.shape[2] // 16 * size)
    rs, hs, ds = x.stride()
    if ds != 1 or x.data_ptr() % step or rs * size % step or hs * size % step:
        return x.clone(memory_format=torch.contiguous_format)
    return x


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """x contiguous from a 16-byte boundary (a view into a tensor may start anywhere)."""
    if not x.is_contiguous():
        x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def kv8_scatter(k: torch.Tensor, v: torch.Tensor, kv: KV8Pages, pages: torch.Tensor,
                slots: torch.Tensor) -> None:
    """Quantise rows k, v [R, KV, D] (fp32 / fp16 / bf16, any strides) into the cache at
    (pages[i], slots[i]) (int64). A target outside the pool is skipped, as in
    PagedKVCache.scatter_decode; two rows with one target leave it undefined."""
    NB, KV, D, P = _pool(kv)
    dev = _device(kv.k, kv.v, kv.scales, k, v, pages, slots)
    R = k.shape[0]
    assert k.shape == v.shape == (R, KV, D), \
        f"k is {tuple(k.shape)}, v {tuple(v.shape)}; the pool holds {KV} kv heads of {D}"
    assert k.dtype is v.dtype
    _check_targets(pages, slots, R)
    k, v = _rows(k), _rows(v)
    (ks, kh, _), (vs, vh, _) = k.stride(), v.stride()
    _call("kv8_scatter", dev, k.data_ptr(), v.data_ptr(), kv.k.data_ptr(), kv.v.data_ptr(),
          kv.scales.data_ptr(), pages.data_ptr(), slots.data_ptr(), R, KV, D, P, NB, ks, kh, vs, vh,
          dtype_code(k))


def kv8_gather(kv: KV8Pages, tables: torch.Tensor, seq_row0: torch.Tensor, seq_pos0: torch.Tensor,
               seq_nq: torch.Tensor, max_nq: int, rows: int, *,
               dtype: torch.dtype = torch.bfloat16,
               out: tuple[torch.Tensor, torch.Tensor] | None = None
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """The cache read back: k, v [rows, KV, D] of `dtype`, where row seq_row0[n] + j holds token
    seq_pos0[n] + j (j < seq_nq[n] <= max_nq) of the sequence with block table tables[n]. Rows
    that no sequence covers, or past their table row's pages, are not written."""
    NB, KV, D, P = _pool(kv)
    dev = _device(kv.k, kv.v, kv.scales, tables, seq_row0, seq_pos0, seq_nq)
    N = seq_row0.shape[0]
    W = _check_tables(N, tables, seq_row0, seq_pos0, seq_nq)
    R, max_nq = int(rows), int(max_nq)
    assert R >= 0 and max_nq >= 0
    if out is None:
        k = torch.empty((R, KV, D), dtype=dtype, device=kv.k.device)
        out = (k, torch.empty_like(k))
    else:
        for o in out:
            _check_out(o, (R, KV, D), dtype, dev)
    _call("kv8_gather", dev, kv.k.data_ptr(), kv.v.data_ptr(), kv.scales.data_ptr(),
          tables.data_ptr(), seq_row0.data_ptr(), seq_pos0.data_ptr(), seq_nq.data_ptr(),
          out[0].data_ptr(), out[1].data_ptr(), N, R, max_nq, KV, D, P, NB, W, dtype_code(out[0]))
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
    NB, KV, D, P = _pool(kv)
    dev = _device(kv.k, kv.v, kv.scales, qkv, pages, slots, positions, inv_freq, q_weight, k_weight)
    H = int(q_heads)
    dtype = q_weight.dtype
    shape = qkv.shape
    assert len(shape) in (2, 3) and shape[-1] == (H + 2 * KV) * D and H >= 1, \
        f"qkv rows hold {(H + 2 * KV) * D} values"
    planes = shape[0] if len(shape) == 3 else 0
    assert qkv.dtype is (torch.float32 if len(shape) == 3 else dtype), \
        "qkv is [S, R, width] fp32 or [R, width] of the weights' dtype"
    assert len(shape) == 2 or planes >= 1
    R = shape[-2]
    _check_targets(pages, slots, R)
    assert positions.shape == (R,) and positions.dtype is torch.int64 and positions.is_contiguous()
    assert inv_freq.shape == (D // 2,) and inv_freq.dtype is torch.float32 and inv_freq.is_contiguous()
    assert q_weight.shape == k_weight.shape == (D,) and k_weight.dtype is dtype
    qkv, qw, kw = _aligned(qkv), _aligned(q_weight), _aligned(k_weight)
    if out is None:
        out = torch.empty((R, H, D), dtype=dtype, device=qkv.device)
    else:
        _check_out(out, (R, H, D), dtype, dev)
    _call("qkv_epilogue_kv8", dev, qkv.data_ptr(), planes, out.data_ptr(), kv.k.data_ptr(),
          kv.v.data_ptr(), kv.scales.data_ptr(), pages.data_ptr(), slots.data_ptr(), R, H, KV, D, P,
          NB, qw.data_ptr(), kw.data_ptr(), float(eps), positions.data_ptr(), inv_freq.data_ptr(),
          dtype_code(out))
    return out


def kv8_splits(batch: int, kv_heads: int, max_pages: int, page_size: int) -> int:
    """Splits of the cache's length for paged_decode_attention_kv8 over block tables max_pages
    wide. The kernel runs splits of more than 16 groups of 16 tokens as workgroups of eight waves,
    of which a CU holds one, and shorter ones as one wave; more than one split takes a second
    launch (2 to 8 us). Measured on MI355X, 32 / 8 heads, tables as wide as the longest sequence,
    us, each line from one sweep (figures of other cards and runs differ by some 5%):
    - (sequence, kv head) pairs that fill the CUs, or short tables: one split (64 sequences of
      1024..8192 tokens 110, in 31 splits of one wave 116; one of 333 6.4, in 11 splits 7.3);
    - else as many as make one round of eight-wave workgroups (one sequence of 131000, 16 / 8
      heads: 32 splits 47.8, 64 49.8, 24 49.0; 16 of 4000: 2 splits 29.7, 3 33.5, 1 33.1),
    - but one-wave splits where those would be short (one of 4000: 63 splits 8.9, 16 12.7) or fill
      three quarters of the CUs or less (12 of 2000..8000: 31 splits 29, 2 36).
    The rule sees the table's width and not the lengths: splits grow with the table, and a sequence
    much longer than the others gets no more of them. 8 sequences of 2000..8000 take 22 us under a
    table of 7456 tokens and 48 under one of 131072; one of 100000 among 31 of 500..1500 takes 497
    (16-bit cache 167), where num_splits of the caller's choice may do better."""
    per = page_size // GROUP
    groups, pairs = max_pages * per, max(1, batch * kv_heads)
    if pairs >= MI355X_CUS or groups <= 32 or (groups <= 64 and pairs >= 64):
        return 1
    S = MI355X_CUS // pairs
    if groups > 16 * S and 4 * pairs * S > 3 * MI355X_CUS:
        return min(S, max_pages)
    unit = min(16, max(2, -(-groups // 64), -(-pairs * groups // 1024)))
    return -(-max_pages // -(-unit // per))


def kv8_workspace(batch: int, num_heads: int, head_dim: int, num_splits: int, device
                  ) -> tuple[torch.Tensor, torch.Tensor] | None:
    """The partials of num_splits splits (None for one)."""
    if num_splits <= 1:
        return None
    n = batch * num_heads * num_splits
    both = torch.empty(n * (head_dim + 2), dtype=torch.float32, device=device)
    return both[:n * head_dim], both[n * head_dim:]


def _check_attention(q: torch.Tensor, H: int, KV: int, D: int, P: int) -> None:
    assert q.shape[-1] == D and H >= KV and H % KV == 0, \
        f"q heads {tuple(q.shape[-2:])} over {KV} kv heads of {D}"
    if q.dtype not in (torch.bfloat16, torch.float16) or H // KV not in (1, 2, 4, 8):
        raise NotImplementedError(f"attention over the 8-bit cache: {q.dtype}, {H} / {KV} heads")


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
    NB, KV, D, P = _pool(kv)
    dev = _device(q, kv.k, kv.v, kv.scales, tables, seq_lens)
    assert q.dim() == 3
    B, H, _ = q.shape
    _check_attention(q, H, KV, D, P)
    W = _check_tables(B, tables, seq_lens)
    S = kv8_splits(B, KV, W, P) if num_splits is None else int(num_splits)
    assert S >= 1
    q = _aligned(q)
    if out is None:
        out = torch.empty_like(q)
    else:
        _check_out(out, (B, H, D), q.dtype, dev)
    ws = (None, None)
    if S > 1:
        ws = workspace
        if ws is None:
            ws = kv8_workspace(B, H, D, S, q.device)
        elif B:
            for t, n in ((ws[0], B * H * S * D), (ws[1], 2 * B * H * S)):
                assert t.dtype is torch.float32 and t.is_contiguous() and t.numel() >= n and \
                    t.get_device() == dev and t.data_ptr() % 16 == 0, \
                    "workspace: kv8_workspace of the same sizes"
    _call("paged_attention_kv8", dev, q.data_ptr(), kv.k.data_ptr(), kv.v.data_ptr(),
          kv.scales.data_ptr(), tables.data_ptr(), seq_lens.data_ptr(), out.data_ptr(), ptr(ws[0]),
          ptr(ws[1]), B, H, KV, D, P, NB, W, S, float(D ** -0.5), dtype_code(q))
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


def _prefill(dev, q, kv, pool, tables, row0, pos0, nq, out, N, R, max_nq, H, W) -> None:
    NB, KV, D, P = pool
    ws = prefill_workspace_kv8(N, R, max_nq, H, KV, D, P, W, q.device)
    _call("paged_prefill_attention_kv8", dev, q.data_ptr(), kv.k.data_ptr(), kv.v.data_ptr(),
          kv.scales.data_ptr(), tables.data_ptr(), ptr(row0), pos0.data_ptr(), ptr(nq),
          out.data_ptr(), N, R, max_nq, H, KV, D, P, NB, W, float(D ** -0.5), dtype_code(q), ptr(ws),
          0 if ws is None else ws.numel())


def paged_prefill_attention_kv8(q: torch.Tensor, kv: KV8Pages, tables: torch.Tensor,
                                seq_row0: torch.Tensor, seq_pos0: torch.Tensor,
                                seq_nq: torch.Tensor, max_nq: int, *,
                                out: torch.Tensor | None = None) -> torch.Tensor:
    """paged_prefill_attention over the 8-bit cache. q [R, H, D]: the prompt rows of N sequences,
    packed; row j of sequence n, q[seq_row0[n] + j] (j < seq_nq[n] <= max_nq), sits at position
    seq_pos0[n] + j and attends to the sequence's tokens 0 .. its own position, which are in the
    cache. Rows not covered by a sequence, or past their table row's pages, are left as they were
    in `out`."""
    pool = _pool(kv)
    dev = _device(q, kv.k, kv.v, kv.scales, tables, seq_row0, seq_pos0, seq_nq)
    assert q.dim() == 3
    R, H, D = q.shape
    _check_attention(q, H, *pool[1:])
    N = seq_row0.shape[0]
    W = _check_tables(N, tables, seq_row0, seq_pos0, seq_nq)
    assert int(max_nq) >= 0
    q = _aligned(q)
    if out is None:
        out = torch.empty_like(q)
    else:
        _check_out(out, (R, H, D), q.dtype, dev)
    _prefill(dev, q, kv, pool, tables, seq_row0, seq_pos0, seq_nq, out, N, R, int(max_nq), H, W)
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
    pool = _pool(kv)
    dev = _device(q, kv.k, kv.v, kv.scales, tables, seq_lens)
    _check_attention(q, H, *pool[1:])
    W = _check_tables(B, tables, seq_lens)
    q = _aligned(q)
    out = torch.empty_like(q)
    _prefill(dev, q, kv, pool, tables, None, seq_lens, None, out, B, B * M, M, H, W)
    return out
