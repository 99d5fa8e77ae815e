// Between two steps of a beam search, after its selection (beam_select.hip):
//   acorn_beam_advance  the next beams and the finished hypotheses of every group
//   acorn_beam_reorder  block tables and partly filled pages follow the beams
//   acorn_beam_trace    hypotheses out of the logs of tokens and parents
// All are short: a few hundred bytes, or copies of a page per layer, behind a chain of
// dependent loads.
#include <algorithm>
#include <cmath>

#include "common.h"

using namespace acorn;

namespace {

constexpr int kMaxBeams = 32, kMaxK = 64;
constexpr double kMaxPenalty = 64.0;             // ln of the largest length^penalty

__device__ __forceinline__ uint64_t lanes_below(int lane) { return (1ull << lane) - 1; }

struct BeamFields {
  float* scores;         // [G, W]
  int32_t* length;       // [G]
  int32_t* done;         // [G]
  int64_t* ids;          // [G, W]
  int32_t* position;     // [G, W]
  int32_t* parents;      // [G, W]
  float* fin_scores;     // [G, W]
  int32_t* fin_length;
  int32_t* fin_beam;
  int32_t* fin_token;
};

// One wave per group, a candidate to a lane; a group's old state is in registers before any of the
// new one is written, so that both may be the same memory. Latency: one round of loads, then some
// ballots and 2 W comparisons across lanes. 1 group of 4 beams 3.2 us, 64 of 16 4.6.
__global__ __launch_bounds__(kWave) void beam_advance_kernel(
    const BeamFields in, const BeamFields out, int32_t* token_log, int32_t* parent_log,
    const float* cand_score, const int32_t* cand_beam, const int64_t* cand_token,
    const int64_t* ends, const float* cand_low, float* low, int G, int W, int K, int T, int n_ends,
    double alpha, int early, int64_t pad) {
  const int g = blockIdx.x, lane = threadIdx.x;
  const size_t gw = (size_t)g * W;
  const bool beam = lane < W, cand = lane < K;
  const int l = beam ? lane : 0;
  const int t = in.length[g], old_done = in.done[g];
  const float score = in.scores[gw + l];
  const int position = in.position[gw + l];
  const float fin_score = in.fin_scores[gw + l];
  const int fin_length = in.fin_length[gw + l], fin_beam = in.fin_beam[gw + l],
            fin_token = in.fin_token[gw + l];
  const size_t ck = (size_t)g * K + (cand ? lane : 0);
  const float cs = cand_score[ck], cl = cand_low ? cand_low[ck] : 0.f;
  const int cb = cand_beam[ck];
  const int64_t ct = cand_token[ck];
  bool end = false;
  for (int i = 0; i < n_ends; ++i) end |= ct == ends[i];
  __syncthreads();

  if (old_done != 0 || t < 0 || t >= T) {                      // it stays as it is
    if (beam) {
      out.scores[gw + lane] = score;
      out.ids[gw + lane] = pad;
      out.position[gw + lane] = position;
      out.parents[gw + lane] = lane;
      out.fin_scores[gw + lane] = fin_score;
      out.fin_length[gw + lane] = fin_length;
      out.fin_beam[gw + lane] = fin_beam;
      out.fin_token[gw + lane] = fin_token;
    }
    if (lane == 0) {
      out.length[g] = t;
      out.done[g] = old_done;
    }
    return;
  }

  // the next beams: the first W candidates that go on
  const double sum = (double)cs + (double)cl;
  const bool valid = cand && sum > -INFINITY && cb >= 0 && cb < W;
  const bool goes = valid && !end;
  const uint64_t gm = __ballot(goes);
  const int slot = __popcll(gm & lanes_below(lane)), live = min(__popcll(gm), W);
  const size_t log = ((size_t)t * G + g) * W;
  auto put = [&](int i, float s, float rest, int64_t id, int parent) {
    out.scores[gw + i] = s;
    if (low) low[gw + i] = rest;
    out.ids[gw + i] = id;
    out.parents[gw + i] = parent;
    token_log[log + i] = (int32_t)id;
    parent_log[log + i] = parent;
  };
  if (goes && slot < W) put(slot, cs, cl, ct, cb);
  if (beam && lane >= live) put(lane, -INFINITY, 0.f, pad, lane);
  const double best = gm ? __shfl(sum, __ffsll((unsigned long long)gm) - 1) : -INFINITY;

  // the finished: the best W of those there were (lanes 0 .. W - 1, sorted) and those that end
  // now (lanes W .. 2 W - 1: candidates 0 .. W - 1), of equal ones the lower lane
  const double power = pow((double)(t + 1), alpha);
  const int from = lane >= W ? lane - W : 0;
  const bool took = __shfl((int)(valid && end), from) && lane >= W && lane < 2 * W;
  const float fresh = (float)(__shfl(sum, from) / power);
  const int fresh_beam = __shfl(cb, from), fresh_token = (int)__shfl((long long)ct, from);
  const float fs = beam ? fin_score : took ? fresh : -INFINITY;
  const int fl = beam ? fin_length : took ? t + 1 : 0;
  const int fb = beam ? fin_beam : took ? fresh_beam : 0;
  const int ft = beam ? fin_token : took ? fresh_token : 0;
  int rank = 0;
  for (int j = 0; j < 2 * W; ++j) {
    const float o = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(fs), j));
    rank += o > fs || (o == fs && j < lane);
  }
  const bool kept = lane < 2 * W && rank < W;
  if (kept) {
    out.fin_scores[gw + rank] = fs;
    out.fin_length[gw + rank] = fl;
    out.fin_beam[gw + rank] = fb;
    out.fin_token[gw + rank] = ft;
  }
  const uint64_t last = __ballot(kept && rank == W - 1);
  const int ll = __ffsll((unsigned long long)last) - 1;
  const float worst = __shfl(fs, max(ll, 0));
  const bool full = last && __shfl(fl, max(ll, 0)) > 0;
  if (beam) out.position[gw + lane] = position + 1;
  if (lane == 0) {
    const float reach = (float)(best / power);
    const bool stop = best == -INFINITY || t + 1 >= T || (full && (early || worst >= reach));
    out.length[g] = t + 1;
    out.done[g] = stop;
  }
}

// ---- the cache follows the beams --------------------------------------------------------------
// At n cached tokens the pages before column c = n / P are full: a beam's row takes its parent's,
// shared from now on. Column c is a page of the beam's own, filled by n % P tokens: the first
// child of a beam takes its page over, every further child a page of a beam without children, in
// order, with a copy of the tokens. So every page stays with one beam of its group, sources are
// pages that nothing is written to, and no page is needed that the group has not.

// Of lane l < W: the page that the next beam l holds at column c, and the one its tokens are in.
struct Plan {
  int to, from;
};
__device__ __forceinline__ Plan plan_pages(int parent, int page, int W, int lane) {
  bool first = lane < W, child = false;
  for (int j = 0; j < W; ++j) {
    const int pj = __builtin_amdgcn_readlane(parent, j);
    first &= !(j < lane && pj == parent);
    child |= pj == lane;
  }
  const uint64_t more = __ballot(lane < W && !first), spare = __ballot(lane < W && !child);
  const int from = __shfl(page, parent);
  // the r-th further child takes the page of the r-th beam without children
  const int r = __popcll(more & lanes_below(lane));
  uint64_t rest = spare;
  for (int i = 0; i < r; ++i) rest &= rest - 1;
  const int owner = rest ? __ffsll((unsigned long long)rest) - 1 : 0;
  const int other = __shfl(page, owner);
  return {first ? from : other, from};
}

__device__ __forceinline__ int parent_of(const int32_t* parents, size_t gw, int W, int lane) {
  const int l = lane < W ? lane : 0;
  const int p = parents[gw + l];
  return p >= 0 && p < W ? p : l;              // (a parent that there is not: the beam itself)
}

// The pools: pages of `bytes`, [layers, num_blocks] of them. Of a page whose first `fill` tokens are
// to be copied these are its first fill * row bytes (tokens one after another), or with `tiles` the
// groups of 16 tokens that hold one: of each kv head's P / 16 groups of 2^shift pieces of 16 bytes
// the first ones. An 8-bit cache's scale codes (2 pieces to a group) go with its V tiles.
struct Pools {
  uint8_t* k;
  uint8_t* v;
  uint8_t* scales;                                             // or none: no tiles
  int64_t bytes, num_blocks;
  int row, shift;
};

constexpr int kCopyNT = 256, kCopyUnroll = 4;
constexpr int64_t kCopyParts = 2048;                           // workgroups that a copy is divided into, if it has the units
constexpr int kCopyUnit = kCopyNT * kCopyUnroll;               // pieces of 16 bytes that are on their way together
typedef uint32_t bm_u32x4 __attribute__((ext_vector_type(4)));

// A workgroup per (layer and pool, group, part of the group's copies): every wave works the plan out,
// and the units of all copies are dealt to the parts, so that no workgroup is there for a beam that
// needs no copy. Bound by memory behind three dependent loads (length, page, tokens): 16 x 4 beams of
// a 16-bit cache through 36 layers (48 MB read and written) 11 us, 4.4 TB/s; 8 x 8 beams of an
// 8-bit one, pages of 32 (94 MB), 21, 4.5 TB/s; 1 x 4 beams 3.5. With a workgroup per beam, layer
// and pool 12.8, 25 and 3.3.
__global__ __launch_bounds__(kCopyNT) void beam_copy_kernel(
    const Pools pools, const int32_t* __restrict__ tables, const int32_t* __restrict__ lens,
    const int32_t* __restrict__ parents, int W, int P, int width) {
  const int g = blockIdx.y, layer = blockIdx.x >> 1;
  const bool second = blockIdx.x & 1;
  const int lane = threadIdx.x % kWave;
  const size_t gw = (size_t)g * W;
  const int n = lens[gw], fill = n % P, c = n / P;
  const int parent = parent_of(parents, gw, W, lane);
  if (n <= 0 || fill == 0 || c >= width) return;
  const int page = tables[(gw + (lane < W ? lane : 0)) * width + c];
  const Plan plan = plan_pages(parent, page, W, lane);
  const bool copy = lane < W && plan.to != plan.from && (uint32_t)plan.to < (uint32_t)pools.num_blocks &&
                    (uint32_t)plan.from < (uint32_t)pools.num_blocks;
  const uint64_t copies = __ballot(copy);
  const int rank = __popcll(copies & lanes_below(lane));
  const bool tiles = pools.scales != nullptr;
  const int groups = (fill + 15) / 16, of = P / 16;
  const int pieces = (int)((tiles ? pools.bytes : (int64_t)fill * pools.row) / 16);
  const int units = (pieces + kCopyUnit - 1) / kCopyUnit;
  uint8_t* pool = (second ? pools.v : pools.k) + (size_t)layer * pools.num_blocks * pools.bytes;
  for (int i = blockIdx.z; i < __popcll(copies) * units; i += gridDim.z) {
    const int from_lane = __ffsll((unsigned long long)__ballot(copy && rank == i / units)) - 1;
    const int64_t to = __builtin_amdgcn_readlane(plan.to, from_lane);
    const int64_t from = __builtin_amdgcn_readlane(plan.from, from_lane);
    const bm_u32x4* src = (const bm_u32x4*)(pool + from * pools.bytes);
    bm_u32x4* dst = (bm_u32x4*)(pool + to * pools.bytes);
    const int first = i % units * kCopyUnit + threadIdx.x;
    bm_u32x4 x[kCopyUnroll];
    bool on[kCopyUnroll];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u) {
      const int at = first + u * kCopyNT;
      on[u] = at < pieces && (!tiles || (at >> pools.shift & (of - 1)) < groups);
      x[u] = src[on[u] ? at : 0];
    }
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
      if (on[u]) dst[first + u * kCopyNT] = x[u];
    if (tiles && second && i % units == 0) {                   // the page's scale codes
      const int64_t codes = (pools.bytes >> pools.shift) * 2;  // 32 bytes to a group
      uint8_t* sc = pools.scales + (size_t)layer * pools.num_blocks * codes;
      for (int at = threadIdx.x; at < codes / 16; at += kCopyNT)
        if ((at >> 1 & (of - 1)) < groups)
          ((bm_u32x4*)(sc + to * codes))[at] = ((const bm_u32x4*)(sc + from * codes))[at];
    }
  }
}

// A thread per column, which reads the group's entries of it before it writes them; the wave that has
// the column with the partly filled pages works the plan out. A launch of its own, as every workgroup
// of the copy reads the pages that it replaces: 2.4 us for 1 group, 4.0 for 16 behind their copies
// (under the profiler; 3 of 14.0 in a graph).
constexpr int kTableNT = 256, kTableUnroll = 8;

__global__ __launch_bounds__(kTableNT) void beam_tables_kernel(int32_t* tables, const int32_t* lens,
                                                               const int32_t* parents, int W, int P,
                                                               int width) {
  __shared__ int32_t held[kMaxBeams][kTableNT];                // (each wave reads its own columns)
  const int g = blockIdx.y, lane = threadIdx.x % kWave, w0 = threadIdx.x - lane;
  const size_t gw = (size_t)g * W;
  const int first = blockIdx.x * kTableNT + w0, column = first + lane;
  const int n = max(lens[gw], 0), fill = n % P, c = n / P;
  const int parent = parent_of(parents, gw, W, lane);
  int32_t* t = tables + gw * width;
  for (int b = 0; b < W; b += kTableUnroll) {
    int32_t x[kTableUnroll];
#pragma unroll
    for (int i = 0; i < kTableUnroll; ++i)
      if (b + i < W) x[i] = (t + (size_t)(b + i) * width)[min(column, width - 1)];
#pragma unroll
    for (int i = 0; i < kTableUnroll; ++i)
      if (b + i < W) held[b + i][threadIdx.x] = x[i];
  }
  if (first > c) return;                                       // columns of the future
  __builtin_amdgcn_wave_barrier();
  int to = 0;
  if (fill && c < width && c < first + kWave)
    to = plan_pages(parent, held[lane < W ? lane : 0][w0 + c - first], W, lane).to;
  const bool mine = column < width && (column < c || (column == c && fill));
#pragma unroll 4
  for (int w = 0; w < W; ++w) {
    const int from = __builtin_amdgcn_readlane(parent, w), page = __builtin_amdgcn_readlane(to, w);
    if (mine && (column == c || from != w))
      (t + (size_t)w * width)[column] = column == c ? page : held[from][threadIdx.x];
  }
}

// ---- hypotheses -------------------------------------------------------------------------------
// out[g, m, t] = tokens[t, g, b_t] for t < steps[g, m], where b_{steps - 1} = beams[g, m] and
// b_{t - 1} = parents[t, g, b_t]; `pad` behind. T dependent steps, taken side by side: a wave's lanes
// are 64 / B stretches of L steps by B beams (B a power of 2, W of them used), 16 waves hold the T
// steps of a group. Every stretch is walked from each beam at its end: a map of beams. A
// hypothesis's beam at a stretch's end comes out of the maps of the stretches behind it (those
// of a wave composed by doubling), and the stretch is walked once more from there with the tokens.
// Up to four workgroups take a group: each makes all the maps and writes the tokens of a quarter of the
// waves (of consecutive ones, so that a SIMD has one each). 16 groups of 8 beams, 2048 steps: 16
// dependent steps, 16 more with the tokens, 12 us (16 with one workgroup, 73 with one stretch to a
// wave): instructions and exchanges between lanes of the CUs that have a group. 1 group of 4 beams,
// 100 steps: 4.2 us.
constexpr int kTraceWaves = 16;
constexpr int kPlaces = 256;                       // workgroups that run side by side
constexpr int kTile = 16;                          // steps whose rows are loaded together
// Stretches up to here are written as they come, others 16 tokens of a hypothesis at a time out of LDS:
// 4 groups of 4 beams, 256 steps (stretches of 1) 6.0 us and 7.4, 16 of 4, 2048 steps (8) 8.8 and
// 10.0; of stretches of 16 64 groups of 8 beams take 16.5 and 15.1, 128 groups 34 and 23.
constexpr int kDirect = 8;

template <bool DIRECT>
__global__ __launch_bounds__(kTraceWaves* kWave) void beam_trace_kernel(
    const int32_t* __restrict__ tokens, const int32_t* __restrict__ parents,
    const int32_t* __restrict__ steps, const int32_t* __restrict__ beams,
    int64_t* __restrict__ out, int T, int G, int W, int M, int L, int shift, int64_t pad) {
  // beam at a stretch's end -> before its first step; and through the wave's stretches behind it too
  __shared__ int8_t one[kTraceWaves * kWave], rest[kTraceWaves * kWave];
  __shared__ int8_t part[kMaxBeams];               // a hypothesis's beam before the stretch it ends in
  __shared__ int64_t stage[DIRECT ? 1 : kTraceWaves][kWave][kTile + 1];
  const int g = blockIdx.x, lane = threadIdx.x % kWave, wid = threadIdx.x / kWave;
  const int B = 1 << shift, S = kWave >> shift, j = lane >> shift, h = lane & (B - 1);
  const int own = lane - h;                        // the first lane of the stretch
  const int q = wid * S + j;                       // the stretch, steps a .. e - 1
  const int a = min((int64_t)q * L, (int64_t)T), e = min(a + L, T);
  auto inside = [&](int x) { return x >= 0 && x < W ? x : -1; };      // -1 ends a walk
  auto at = [&](int v, int beam) { return __shfl(v, own + max(beam, 0)); };
  auto hop = [&](int row, int cur) {
    const int next = at(row, cur);
    return cur < 0 ? -1 : inside(next);
  };
  // steps a + L - kTile (i + 1) .. of every stretch, one beam to a lane
  const uint32_t stride = (uint32_t)G * W;         // (below 2^31: the host's check)
  const int64_t column = (int64_t)g * W + min(h, W - 1);
  auto load = [&](const int32_t* from, int i, int (&x)[kTile]) {
    const int t0 = a + L - kTile * (i + 1);
#pragma unroll
    for (int o = kTile - 1; o >= 0; --o) {
      if (kTile * (i + 1) - o > L) break;          // (before every stretch)
      x[o] = from[column + (uint64_t)(uint32_t)min(t0 + o, T - 1) * stride];
    }
  };
  const int tiles = (L + kTile - 1) / kTile;
  // (a wave may have no steps, and the tokens are taken by one workgroup of the group)
  const bool some_steps = (int64_t)wid * S * L < T;
  const bool takes = some_steps && wid / (kTraceWaves / (int)gridDim.y) == (int)blockIdx.y;
  // where a stretch is one tile both passes' rows are loaded here, once
  int row[kTile], token[kTile];
  if (some_steps) load(parents, 0, row);
  if (takes) load(tokens, 0, token);
  int all = h < W ? h : -1;
  for (int h0 = 0; h0 < M; h0 += B) {
    const int m = h0 + h;
    const bool hyp = m < M;
    const int last = hyp ? min(max(steps[(size_t)g * M + m], 0), T) - 1 : -1;
    const int beam = hyp ? inside(beams[(size_t)g * M + m]) : -1;
    const int ends = last >= 0 ? last / L : -1;    // the stretch it ends in
    int mine = -1;
    const bool some = __ballot(q == ends) != 0;    // a hypothesis ends in one of the wave's stretches
    for (int i = 0; i < (some_steps && (h0 == 0 || some) ? tiles : 0); ++i) {
      if (tiles > 1) load(parents, i, row);
#pragma unroll
      for (int o = kTile - 1; o >= 0; --o) {
        if (kTile * (i + 1) - o > L) break;        // (before every stretch)
        const int t = a + L - kTile * (i + 1) + o;
        if (h0 == 0) {
          const int x = hop(row[o], all);
          if (t < e) all = x;
        }
        if (some) {
          if (t == last) mine = beam;              // (q == ends there)
          const int y = hop(row[o], mine);
          if (t < e) mine = y;
        }
      }
    }
    if (h0 == 0) {
      one[threadIdx.x] = (int8_t)all;
      for (int d = 1; d < S; d <<= 1) {            // this stretch after the d behind it
        const int v = __shfl(all, (lane + d * B) % kWave), x = at(all, v);
        if (j + d < S) all = v < 0 ? -1 : x;
      }
      rest[threadIdx.x] = (int8_t)all;
    }
    if (q == ends) part[h] = (int8_t)mine;
    __syncthreads();
    // the beam at this stretch's end
    int cur = -1;
    if (ends > q) {
      cur = part[h];
      auto follow = [&](const int8_t* map, int stretch) { cur = cur < 0 ? -1 : map[stretch * B + cur]; };
      const int w = ends / S, from = w == wid ? q + 1 : w * S;
      for (int i = ends - 1; i >= from; --i) follow(one, i);
      if (w != wid) {
        for (int i = w - 1; i > wid; --i) follow(rest, i * S);
        if (j + 1 < S) follow(rest, q + 1);
      }
    }
    __syncthreads();                               // (part is written again)
    for (int i = 0; i < (takes ? tiles : 0); ++i) {
      if (tiles > 1) {
        load(parents, i, row);
        load(tokens, i, token);
      }
#pragma unroll
      for (int o = kTile - 1; o >= 0; --o) {
        if (kTile * (i + 1) - o > L) break;
        const int t = a + L - kTile * (i + 1) + o;
        if (t == last) cur = beam;
        const int tok = at(token[o], cur);
        const int64_t value = cur < 0 || t > last ? pad : (int64_t)tok;
        if (!DIRECT)
          stage[wid][lane][o] = value;
        else if (hyp && t < e)
          out[((size_t)g * M + m) * T + t] = value;
        const int next = hop(row[o], cur);
        if (t < e && t <= last) cur = next;
      }
      if (DIRECT) continue;
      __builtin_amdgcn_wave_barrier();
      // kTile tokens of a lane side by side
      for (int r = 0; r < kWave * kTile; r += kWave) {
        const int of = (r + lane) / kTile, o = lane % kTile;
        const int a_of = min((int64_t)(wid * S + (of >> shift)) * L, (int64_t)T);
        const int t = a_of + L - kTile * (i + 1) + o, m_of = h0 + (of & (B - 1));
        if (m_of < M && t >= a_of && t < min(a_of + L, T))
          out[((size_t)g * M + m_of) * T + t] = stage[wid][of][o];
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

}  // namespace

extern "C" int acorn_beam_advance_low(const float* scores, const int32_t* length, const int32_t* done,
                                  const int32_t* position, const float* fin_scores,
                                  const int32_t* fin_length, const int32_t* fin_beam,
                                  const int32_t* fin_token, float* out_scores, int32_t* out_length,
                                  int32_t* out_done, int64_t* out_ids, int32_t* out_position,
                                  int32_t* out_parents, float* out_fin_scores,
                                  int32_t* out_fin_length, int32_t* out_fin_beam,
                                  int32_t* out_fin_token, int32_t* token_log, int32_t* parent_log,
                                  const float* cand_score, const int32_t* cand_beam,
                                  const int64_t* cand_token, const int64_t* ends,
                                  const float* cand_low, float* low, int64_t groups,
                                  int64_t beams, int64_t k, int64_t steps, int64_t n_ends,
                                  double length_penalty, int early_stopping, int64_t pad,
                                  void* stream) {
  if (groups < 0 || groups > 0x7fffffff || beams < 1 || k < 1 || steps < 1 || steps > 0x7fffffff ||
      n_ends < 0 || n_ends > 0x7fffffff)
    return ACORN_ERR_SHAPE;
  if (beams > kMaxBeams || k > kMaxK) return ACORN_ERR_UNSUPPORTED;
  if (groups == 0) return ACORN_OK;
  const void* all[] = {scores, length, done, position, fin_scores, fin_length, fin_beam, fin_token,
                       out_scores, out_length, out_done, out_ids, out_position, out_parents,
                       out_fin_scores, out_fin_length, out_fin_beam, out_fin_token, token_log,
                       parent_log, cand_score, cand_beam, cand_token};
  for (const void* p : all)
    if (!p) return ACORN_ERR_VALUE;
  // (steps^penalty as a factor that 32 bits hold, either way; NaN and infinities fail too)
  if ((n_ends && !ends) || !(fabs(length_penalty) * log((double)steps) <= kMaxPenalty) ||
      !(fabs(length_penalty) < INFINITY))
    return ACORN_ERR_VALUE;
  const BeamFields in = {(float*)scores, (int32_t*)length, (int32_t*)done, nullptr,
                         (int32_t*)position, nullptr, (float*)fin_scores, (int32_t*)fin_length,
                         (int32_t*)fin_beam, (int32_t*)fin_token};
  const BeamFields out = {out_scores, out_length, out_done, out_ids, out_position, out_parents,
                          out_fin_scores, out_fin_length, out_fin_beam, out_fin_token};
  beam_advance_kernel<<<dim3((unsigned)groups), dim3(kWave), 0, (hipStream_t)stream>>>(
      in, out, token_log, parent_log, cand_score, cand_beam, cand_token, ends, cand_low, low,
      (int)groups, (int)beams, (int)k, (int)steps, (int)n_ends, length_penalty, early_stopping, pad);
  ACORN_LAUNCH_CHECK();
  return ACORN_OK;
}

extern "C" int acorn_beam_advance(const float* scores, const int32_t* length, const int32_t* done,
                                  const int32_t* position, const float* fin_scores,
                                  const int32_t* fin_length, const int32_t* fin_beam,
                                  const int32_t* fin_token, float* out_scores, int32_t* out_length,
                                  int32_t* out_done, int64_t* out_ids, int32_t* out_position,
                                  int32_t* out_parents, float* out_fin_scores,
                                  int32_t* out_fin_length, int32_t* out_fin_beam,
                                  int32_t* out_fin_token, int32_t* token_log, int32_t* parent_log,
                                  const float* cand_score, const int32_t* cand_beam,
                                  const int64_t* cand_token, const int64_t* ends, int64_t groups,
                                  int64_t beams, int64_t k, int64_t steps, int64_t n_ends,
                                  double length_penalty, int early_stopping, int64_t pad,
                                  void* stream) {
  return acorn_beam_advance_low(scores, length, done, position, fin_scores, fin_length, fin_beam,
                                fin_token, out_scores, out_length, out_done, out_ids, out_position,
                                out_parents, out_fin_scores, out_fin_length, out_fin_beam,
                                out_fin_token, token_log, parent_log, cand_score, cand_beam,
                                cand_token, ends, nullptr, nullptr, groups, beams, k, steps, n_ends,
                                length_penalty, early_stopping, pad, stream);
}

extern "C" int acorn_beam_reorder(void* k_pool, void* v_pool, void* scale_pool, int32_t* tables,
                                  const int32_t* lens, const int32_t* parents, int64_t groups,
                                  int64_t beams, int64_t table_stride, int64_t layers,
                                  int64_t num_blocks, int64_t page_size, int64_t kv_heads,
                                  int64_t head_dim, int64_t elem_size, void* stream) {
  if (groups < 0 || groups > 65535 || beams < 1 || table_stride < 1 || layers < 1 || num_blocks < 1 ||
      num_blocks > 0x7fffffff || page_size < 1 || page_size > 65536 || kv_heads < 1 ||
      kv_heads > 65535 || head_dim < 1 || head_dim > 65536 || table_stride > 0x7fffffff / page_size)
    return ACORN_ERR_SHAPE;
  if (beams > kMaxBeams) return ACORN_ERR_UNSUPPORTED;
  if (groups * beams > 65535 || layers > 0x3fffffff) return ACORN_ERR_SHAPE;
  const bool tiles = scale_pool != nullptr;
  if (tiles && (page_size % 16 || (page_size & (page_size - 1)) || elem_size != 1)) return ACORN_ERR_SHAPE;
  if (tiles && head_dim != 64 && head_dim != 128) return ACORN_ERR_UNSUPPORTED;
  if (!tiles && elem_size != 2 && elem_size != 4) return ACORN_ERR_DTYPE;
  const int64_t row = kv_heads * head_dim * elem_size;         // a token's bytes
  if (row % 16 || row * page_size > 0x7fffffff) return ACORN_ERR_UNSUPPORTED;
  if (groups == 0) return ACORN_OK;
  if (!k_pool || !v_pool || !tables || !lens || !parents) return ACORN_ERR_VALUE;
  if ((uintptr_t)k_pool % 16 || (uintptr_t)v_pool % 16 || (uintptr_t)scale_pool % 16)
    return ACORN_ERR_VALUE;
  if (beams == 1) return ACORN_OK;
  const Pools pools = {(uint8_t*)k_pool, (uint8_t*)v_pool, (uint8_t*)scale_pool, row * page_size,
                       num_blocks, (int)row, tiles ? __builtin_ctzll((unsigned long long)head_dim) : 0};
  const int64_t most = (beams - 1) * ((pools.bytes / 16 + kCopyUnit - 1) / kCopyUnit);
  const int64_t parts = std::max<int64_t>(1, std::min(most, kCopyParts / (2 * layers * groups)));
  hipStream_t st = (hipStream_t)stream;
  beam_copy_kernel<<<dim3((unsigned)(2 * layers), (unsigned)groups, (unsigned)parts), dim3(kCopyNT), 0,
                     st>>>(pools, tables, lens, parents, (int)beams, (int)page_size,
                           (int)table_stride);
  ACORN_LAUNCH_CHECK();
  beam_tables_kernel<<<dim3((unsigned)((table_stride + kTableNT - 1) / kTableNT), (unsigned)groups),
                       dim3(kTableNT), 0, st>>>(tables, lens, parents, (int)beams, (int)page_size,
                                                (int)table_stride);
  ACORN_LAUNCH_CHECK();
  return ACORN_OK;
}

extern "C" int acorn_beam_trace(const int32_t* tokens, const int32_t* parents,
                                const int32_t* steps, const int32_t* beams, int64_t* out,
                                int64_t T, int64_t groups, int64_t W, int64_t M, int64_t pad,
                                void* stream) {
  if (T < 0 || T > 0x3fffffff || groups < 0 || groups > 0x7fffffff || W < 1 || M < 0 ||
      M > 0x7fffffff - kMaxBeams)
    return ACORN_ERR_SHAPE;
  if (W > kMaxBeams) return ACORN_ERR_UNSUPPORTED;
  if (groups * W > 0x7fffffff) return ACORN_ERR_SHAPE;
  if (T == 0 || groups == 0 || M == 0) return ACORN_OK;
  if (!tokens || !parents || !steps || !beams || !out) return ACORN_ERR_VALUE;
  int shift = 0;
  while ((1 << shift) < W) ++shift;
  const int64_t stretches = (int64_t)kTraceWaves * (kWave >> shift);
  // (where the chip has a place, a CU, for each of them: 128 groups of 8 beams, 2048 steps, 26 us with
  // one workgroup each, 23 with two, 37 with four)
  const unsigned parts = groups * 4 <= kPlaces ? 4 : groups * 2 <= kPlaces ? 2 : 1;
  const int L = (int)((T + stretches - 1) / stretches);
  (L <= kDirect ? beam_trace_kernel<true> : beam_trace_kernel<false>)<<<
      dim3((unsigned)groups, parts), dim3(kTraceWaves * kWave), 0, (hipStream_t)stream>>>(
      tokens, parents, steps, beams, out, (int)T, (int)groups, (int)W, (int)M, L, shift, pad);
  ACORN_LAUNCH_CHECK();
  return ACORN_OK;
}
