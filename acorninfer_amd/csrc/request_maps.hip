// Block tables and slot maps from the lengths of requests, without the host:
//   acorn_block_tables  a flat list of blocks, ceil(length / P) to a request -> padded tables
//   acorn_slot_map      packed rows (counts[n] of request n, from token starts[n]) -> request,
//                       position, page, slot and length of every row
// Both are a prefix sum over the requests and then one write per entry. Every workgroup sums
// the requests before its own entries again: N values out of L2 cost less than a second launch.
// Latency: 64 requests, tables of 2000 pages, one row each: 3.1 + 2.8 us (0.5 MB); 23 requests,
// 8290 rows: 2.7 + 4.1.
#include <algorithm>

#include "common.h"

using namespace acorn;

namespace {

constexpr int kNT = 256, kWaves = kNT / kWave;

// v of the lane that the DPP control names, 0 where there is none or the row is masked out.
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t moved(int64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xF, true);
  return (int64_t)((uint64_t)hi << 32 | lo);
}
// Inclusive sums over the workgroup's threads, in order; *total the last. (Within a wave by DPP: rows of
// 16, then the last lane of a row to the next, of a half to the other.)
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* red, int64_t* total) {
  const int lane = threadIdx.x % kWave, wid = threadIdx.x / kWave;
  v += moved<0x111, 0xF>(v);
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);
  v += moved<0x143, 0xC>(v);
  __syncthreads();                             // (red may still be read from a call before)
  if (lane == kWave - 1) red[wid] = v;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int64_t r = red[w];
    if (w < wid) before += r;
    all += r;
  }
  *total = all;
  return before + v;
}

__device__ __forceinline__ int64_t pages_for(int32_t length, int shift) {
  return length > 0 ? ((int64_t)length + (1ll << shift) - 1) >> shift : 0;
}

// `rows` table rows to a workgroup, a part of their columns.
__global__ __launch_bounds__(kNT) void block_tables_kernel(
    const int32_t* __restrict__ blocks, int64_t n_blocks, const int32_t* __restrict__ lengths,
    int32_t* __restrict__ tables, int N, int width, int shift, int rows, int cols, int pad) {
  __shared__ int64_t red[kWaves];
  const int n0 = blockIdx.x * rows, n1 = min(n0 + rows, N);
  int64_t sum = 0, first = 0;
  for (int i = threadIdx.x; i < n0; i += kNT) sum += pages_for(lengths[i], shift);
  block_scan(sum, red, &first);
  const int c0 = blockIdx.y * cols, c1 = min(c0 + cols, width);
  for (int n = n0; n < n1; ++n) {
    const int64_t own = pages_for(lengths[n], shift);
    for (int c = c0 + threadIdx.x; c < c1; c += kNT) {
      const int64_t at = first + c;
      tables[(size_t)n * width + c] = c < own && at < n_blocks ? blocks[at] : pad;
    }
    first += own;
  }
}

constexpr int kPer = 4, kChunk = kNT * kPer;   // requests summed at a time

struct SlotMap {
  int32_t* seq;
  int64_t* positions;
  int64_t* pages;
  int64_t* slots;
  int32_t* lens;
  int32_t* row0;
};

// A row to a thread. Requests pass by kChunk at a time: their rows' ends in LDS, where each row
// looks for the request it belongs to. Workgroup 0 sees them all and writes row0.
__global__ __launch_bounds__(kNT) void slot_map_kernel(
    const int32_t* __restrict__ tables, const int32_t* __restrict__ starts,
    const int32_t* __restrict__ counts, const SlotMap o, int N, int64_t R, int width, int shift) {
  __shared__ int64_t red[kWaves], ends[kChunk];
  const int64_t row = (int64_t)blockIdx.x * kNT + threadIdx.x;
  const int64_t last = min((int64_t)(blockIdx.x + 1) * kNT, R);
  int64_t base = 0;
  for (int n0 = 0; n0 < N; n0 += kChunk) {
    if (blockIdx.x > 0 && base >= last) return;                // (the same for every thread)
    const int n = n0 + threadIdx.x * kPer;
    int64_t cnt[kPer], own = 0, total;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      cnt[i] = n + i < N ? max(counts[n + i], 0) : 0;
      own += cnt[i];
    }
    int64_t at = base + block_scan(own, red, &total) - own;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (blockIdx.x == 0 && n + i < N) o.row0[n + i] = (int32_t)min(at, (int64_t)INT32_MAX);
      at += cnt[i];
      ends[threadIdx.x * kPer + i] = at;
    }
    __syncthreads();
    if (row >= base && row < base + total && row < R) {
      int lo = 0, hi = min(kChunk, N - n0) - 1;                // the first request that ends past row
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (ends[mid] > row) hi = mid;
        else lo = mid + 1;
      }
      const int s = n0 + lo;
      const int64_t first = lo ? ends[lo - 1] : base;
      const int64_t pos = starts[s] + (row - first);
      const int64_t c = pos >> shift;
      o.seq[row] = s;
      o.positions[row] = pos;
      o.pages[row] = pos >= 0 && c < width ? tables[(size_t)s * width + c] : -1;
      o.slots[row] = pos & ((1 << shift) - 1);
      o.lens[row] = (int32_t)min(pos + 1, (int64_t)INT32_MAX);
    }
    base += total;
  }
}

int shift_of(int64_t page_size) {
  if (page_size < 1 || page_size > (1 << 30) || (page_size & (page_size - 1))) return -1;
  return __builtin_ctzll((unsigned long long)page_size);
}

}  // namespace

extern "C" int acorn_block_tables(const int32_t* blocks, int64_t n_blocks, const int32_t* lengths,
                                  int32_t* tables, int64_t N, int64_t width, int64_t page_size,
                                  int pad, void* stream) {
  const int shift = shift_of(page_size);
  if (shift < 0 || N < 0 || N > 0x3fffffff || width < 1 || width > 0x7fffffff || n_blocks < 0)
    return ACORN_ERR_SHAPE;
  if (N == 0) return ACORN_OK;
  if ((n_blocks && !blocks) || !lengths || !tables) return ACORN_ERR_VALUE;
  const int64_t rows = (N + 2047) / 2048, cols = 1024;
  if ((width + cols - 1) / cols > 65535) return ACORN_ERR_SHAPE;
  block_tables_kernel<<<dim3((unsigned)((N + rows - 1) / rows), (unsigned)((width + cols - 1) / cols)),
                        dim3(kNT), 0, (hipStream_t)stream>>>(blocks, n_blocks, lengths, tables,
                                                             (int)N, (int)width, shift, (int)rows,
                                                             (int)cols, pad);
  ACORN_LAUNCH_CHECK();
  return ACORN_OK;
}

extern "C" int acorn_slot_map(const int32_t* tables, const int32_t* starts, const int32_t* counts,
                              int32_t* seq, int64_t* positions, int64_t* pages, int64_t* slots,
                              int32_t* lens, int32_t* row0, int64_t N, int64_t R, int64_t width,
                              int64_t page_size, void* stream) {
  const int shift = shift_of(page_size);
  if (shift < 0 || N < 0 || N > 0x7fffffff - kChunk || R < 0 || R > 0x7fffffff || width < 1 ||
      width > 0x7fffffff)
    return ACORN_ERR_SHAPE;
  if (N == 0) return ACORN_OK;
  if (!tables || !starts || !counts || !row0) return ACORN_ERR_VALUE;
  if (R && (!seq || !positions || !pages || !slots || !lens)) return ACORN_ERR_VALUE;
  const SlotMap o = {seq, positions, pages, slots, lens, row0};
  slot_map_kernel<<<dim3((unsigned)std::max<int64_t>(1, (R + kNT - 1) / kNT)), dim3(kNT), 0,
                    (hipStream_t)stream>>>(tables, starts, counts, o, (int)N, R, (int)width, shift);
  ACORN_LAUNCH_CHECK();
  return ACORN_OK;
}
