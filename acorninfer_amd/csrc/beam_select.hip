// Beam search's selection: of a group's W beams over a vocabulary of V tokens, the
// k best continuations by
//   s(w, v) = score[w] + x[w, v] - ln sum_u exp(x[w, u]),
// sorted, equal ones in order of w and then v.
//
// Two launches. beam_part_kernel reads the logits once: a workgroup takes a piece
// of one row and leaves the piece's maximum, its sum of exponentials and its k
// largest logits. Within a row the order of s is the order of x, so a piece needs
// neither the row's sum nor the beam's score. beam_join_kernel, one workgroup per
// group, joins a row's pieces, then the rows, by s in 64 bits: beams are compared
// through sums over the whole vocabulary, and 32 bits of s (2^-20 at 10) would tie
// or turn round what the logits tell apart.
//
// A value's key is its order-preserving image in 32 bits, then ~token: keys differ
// from one another, the larger is the better, and the k largest do not depend on
// the order they are met in. A wave keeps its best 64 sorted, one to a lane.
#include <algorithm>

#include "common.h"

using namespace acorn;

namespace {

typedef uint64_t u64;
typedef uint32_t bs_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kPartNT = 256, kPartWaves = kPartNT / kWave;
constexpr int kUnroll = 4;                     // 16-byte vectors of a lane in flight
constexpr int kMaxBeams = 32, kMaxK = 64;
constexpr float kLog2e = 1.4426950408889634f;

template <typename T> __device__ __forceinline__ float vec_elem(const bs_u32x4& w, int e);
template <> __device__ __forceinline__ float vec_elem<__bf16>(const bs_u32x4& w, int e) {
  return (e & 1) ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2]);
}
template <> __device__ __forceinline__ float vec_elem<_Float16>(const bs_u32x4& w, int e) {
  const uint32_t v = w[e / 2];
  return (float)__builtin_bit_cast(_Float16, (uint16_t)((e & 1) ? v >> 16 : v & 0xffffu));
}
template <> __device__ __forceinline__ float vec_elem<float>(const bs_u32x4& w, int e) {
  return __uint_as_float(w[e]);
}

// Ordered like the numbers, -0 and 0 alike (x + 0 is 0 for both).
__device__ __forceinline__ uint32_t order32(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float unorder32(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
__device__ __forceinline__ u64 order64(double x) {
  const u64 u = __builtin_bit_cast(u64, x + 0.0);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double unorder64(u64 k) {
  return __builtin_bit_cast(double, (k >> 63) ? (k & 0x7FFFFFFFFFFFFFFFull) : ~k);
}
__device__ __forceinline__ u64 key_of(float x, uint32_t token) {
  return (u64)order32(x) << 32 | (uint32_t)~token;
}

__device__ __forceinline__ uint32_t lane_xor(uint32_t v, int m) { return __shfl_xor(v, m); }
__device__ __forceinline__ u64 lane_xor(u64 v, int m) { return __shfl_xor((unsigned long long)v, m); }

// The lanes' values in falling order (a bitonic network whose blocks all fall).
template <typename U>
__device__ __forceinline__ U sort_wave(U v, int lane) {
#pragma unroll
  for (int size = 2; size <= kWave; size <<= 1) {
    const U o = lane_xor(v, size - 1);
    v = (lane & (size >> 1)) ? min(v, o) : max(v, o);
#pragma unroll
    for (int d = size >> 2; d > 0; d >>= 1) {
      const U p = lane_xor(v, d);
      v = (lane & d) ? min(v, p) : max(v, p);
    }
  }
  return v;
}
// The 64 best of two falling lists, falling. `other` comes reversed (lane i holds entry 63 - i).
__device__ __forceinline__ u64 merge_wave(u64 top, u64 other, int lane) {
  u64 v = max(top, other);
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) {
    const u64 p = lane_xor(v, d);
    v = (lane & d) ? min(v, p) : max(v, p);
  }
  return v;
}

// A row in vectors of 16 bytes from its first element, whatever that one's alignment (the loads
// are by element): what a lane adds up, and in which order, depends on the row's values alone, so
// that equal rows have equal sums. C pieces of `per` vectors.
template <typename T>
__global__ __launch_bounds__(kPartNT) void beam_part_kernel(
    const T* __restrict__ logits, int64_t row_stride, const float* __restrict__ scores, int V,
    int k, int per, u64* __restrict__ lists, float2* __restrict__ sums) {
  constexpr int E = 16 / sizeof(T);
  __shared__ u64 pend[kPartWaves][(E + 1) * kWave];
  __shared__ u64 tops[kPartWaves][kWave];
  __shared__ float wm[kPartWaves], ws[kPartWaves];
  const int row = blockIdx.y, piece = blockIdx.x, C = gridDim.x;
  const float score = scores[row];
  if (!(score > -INFINITY && score < INFINITY)) return;        // no such beam: nothing is read
  const T* p = logits + row * row_stride;
  const int tid = threadIdx.x, lane = tid % kWave, wid = tid / kWave;
  const int v0 = piece * per, v1 = min(v0 + per, (V + E - 1) / E);

  float m = -INFINITY, s = 0.f;
  u64 top = 0, thr = 0;                                        // thr: the list's k-th, 0 before it has k
  u64* buf = pend[wid];
  for (int t0 = v0 + wid * kWave; t0 < v1; t0 += kPartNT * kUnroll) {
    bs_u32x4 x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int j = t0 + u * kPartNT + lane, i0 = j * E;
      if (j < v1 && i0 <= V - E) {
        __builtin_memcpy(&x[u], p + i0, 16);
      } else {                                                 // the row's end, and past the piece
        T r[E];
#pragma unroll
        for (int e = 0; e < E; ++e) r[e] = j < v1 && i0 + e < V ? p[i0 + e] : (T)-INFINITY;
        __builtin_memcpy(&x[u], r, 16);
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) mx = fmaxf(mx, vec_elem<T>(x[u], e));
    // NaN and +inf reach s as NaN; -inf adds nothing
    const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
    s *= __builtin_amdgcn_exp2f((m - ref) * kLog2e);
    m = mn;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e)
        s += __builtin_amdgcn_exp2f((vec_elem<T>(x[u], e) - ref) * kLog2e);

    if (__ballot(order32(mx) >= (uint32_t)(thr >> 32)) == 0) continue;
    // what may enter the list; at first what reaches the k-th of the lanes' largest, as k do
    u64 least = thr + 1;
    if (thr == 0) least = max(least, (u64)__shfl(sort_wave(order32(mx), lane), k - 1) << 32);
    int n = 0;                                                 // pending
#pragma unroll 1
    for (int u = 0; u < kUnroll; ++u) {
      bs_u32x4 w = x[0];
#pragma unroll
      for (int i = 1; i < kUnroll; ++i) w = u == i ? x[i] : w;
      const int j = t0 + u * kPartNT + lane, i0 = j < v1 ? j * E : V;
      float vm = vec_elem<T>(w, 0);
#pragma unroll
      for (int e = 1; e < E; ++e) vm = fmaxf(vm, vec_elem<T>(w, e));
      if (__ballot(order32(vm) >= (uint32_t)(least >> 32)) != 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const u64 key = key_of(vec_elem<T>(w, e), i0 + e);
          const bool in = i0 + e < V && key >= least;
          const u64 mask = __ballot(in);
          if (in) buf[n + __popcll(mask & ((1ull << lane) - 1))] = key;
          n += __popcll(mask);
        }
      }
      while (n >= kWave || (n > 0 && u == kUnroll - 1)) {      // 64 of them into the list
        __builtin_amdgcn_wave_barrier();
        n -= kWave;
        const u64 v = n + lane >= 0 ? buf[n + lane] : 0;
        top = merge_wave(top, lane_xor(sort_wave(v, lane), kWave - 1), lane);
        thr = (u64)__shfl((unsigned long long)top, k - 1);
        least = max(least, thr + 1);
        __builtin_amdgcn_wave_barrier();
      }
    }
  }

  // the workgroup's list and sum
  const float mw = wave_max(m), refw = mw == -INFINITY ? 0.f : mw;
  const float sw = wave_sum(s * __builtin_amdgcn_exp2f((m - refw) * kLog2e));
  tops[wid][lane] = top;
  if (lane == 0) {
    wm[wid] = mw;
    ws[wid] = sw;
  }
  __syncthreads();
  if (wid != 0) return;
  float M = wm[0], S = ws[0];
#pragma unroll
  for (int w = 1; w < kPartWaves; ++w) {
    top = merge_wave(top, tops[w][kWave - 1 - lane], lane);
    const float n = fmaxf(M, wm[w]), r = n == -INFINITY ? 0.f : n;
    S = S * __builtin_amdgcn_exp2f((M - r) * kLog2e) + ws[w] * __builtin_amdgcn_exp2f((wm[w] - r) * kLog2e);
    M = n;
  }
  const int64_t at = (int64_t)row * C + piece;
  if (lane < k) lists[at * k + lane] = top;
  if (lane == 0) sums[at] = make_float2(M, S);
}

// An entry of the group's list: s as a key, then its place (beam * 64 + rank in the beam's list):
// the larger key first, of equal ones the lower place.
struct Entry {
  u64 key;
  uint32_t place;
};
__device__ __forceinline__ bool before(const Entry& a, const Entry& b) {
  return a.key > b.key || (a.key == b.key && a.place < b.place);
}
__device__ __forceinline__ Entry merge_entries(Entry top, Entry other, int lane) {
  Entry v = before(other, top) ? other : top;
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) {
    Entry o;
    o.key = lane_xor(v.key, d);
    o.place = __shfl_xor(v.place, d);
    const bool swap = (lane & d) ? before(v, o) : before(o, v);
    if (swap) v = o;
  }
  return v;
}

__global__ __launch_bounds__(1024) void beam_join_kernel(
    const u64* __restrict__ lists, const float2* __restrict__ sums,
    const float* __restrict__ scores, int W, int V, int k, int C, float* __restrict__ out_score,
    int32_t* __restrict__ out_beam, int64_t* __restrict__ out_token, int32_t* __restrict__ status) {
  __shared__ uint32_t tokens[kMaxBeams][kWave];
  __shared__ u64 keys[16][kWave];
  __shared__ uint32_t places[16][kWave];
  const int g = blockIdx.x, lane = threadIdx.x % kWave, wid = threadIdx.x / kWave;
  const int waves = blockDim.x / kWave;
  Entry best = {0, 0xFFFFFFFFu};
  for (int w = wid; w < W; w += waves) {
    const int64_t row = (int64_t)g * W + w;
    const float score = scores[row];
    bool bad = !(score < INFINITY), live = score > -INFINITY && !bad;
    double ref = 0.0, log_sum = 0.0;           // ln sum exp(x) = ref + log_sum
    u64 top = 0;
    if (live) {
      const float2* sp = sums + row * C;
      float M = -INFINITY;
      for (int c = lane; c < C; c += kWave) M = fmaxf(M, sp[c].x);
      M = wave_max(M);
      ref = M == -INFINITY ? 0.0 : (double)M;
      double S = 0.0;
      for (int c = lane; c < C; c += kWave) {
        const float2 ms = sp[c];
        S += (double)ms.y * exp2(((double)ms.x - ref) * (double)kLog2e);
      }
#pragma unroll
      for (int o = kWave / 2; o > 0; o >>= 1) S += __shfl_xor(S, o);
      if (!(S == S)) bad = true;
      live = !bad && M > -INFINITY;
      // (the pieces' exponentials are powers of 2 of x * kLog2e, which as a float is 1.3e-8 off)
      log_sum = log2(S) / (double)kLog2e;
    }
    if (live) {
      const u64* lp = lists + row * C * k;
      const int n = C * k;
      u64 thr = 0;
      for (int i = 0; i < n; i += kWave) {
        u64 v = i + lane < n ? lp[i + lane] : 0;
        if (__ballot(v > thr) == 0) continue;
        v = sort_wave(v, lane);
        top = merge_wave(top, lane_xor(v, kWave - 1), lane);
        thr = (u64)__shfl((unsigned long long)top, k - 1);
      }
    }
    Entry e = {0, (uint32_t)(w * kWave + lane)};
    if (live) {
      // (x - ref first: where logits are of the type's lowest value, their sum would swallow log_sum)
      if (top && lane < k)
        e.key = order64((double)score + (((double)unorder32((uint32_t)(top >> 32)) - ref) - log_sum));
      tokens[w][lane] = ~(uint32_t)top;
    } else {                                   // -inf: the first tokens
      if (lane < min(k, V)) e.key = order64(-INFINITY);
      tokens[w][lane] = lane;
    }
    if (lane == 0) status[row] = bad;
    Entry r;
    r.key = lane_xor(e.key, kWave - 1);
    r.place = __shfl_xor(e.place, kWave - 1);
    best = merge_entries(best, r, lane);
  }
  keys[wid][lane] = best.key;
  places[wid][lane] = best.place;
  __syncthreads();
  for (int half = 8; half > 0; half >>= 1) {
    if (wid < half && wid + half < waves) {
      const Entry r = {keys[wid + half][kWave - 1 - lane], places[wid + half][kWave - 1 - lane]};
      best = merge_entries(best, r, lane);
      keys[wid][lane] = best.key;
      places[wid][lane] = best.place;
    }
    __syncthreads();
  }
  if (wid == 0 && lane < k) {
    const int64_t o = (int64_t)g * k + lane;
    out_score[o] = (float)unorder64(best.key);
    out_beam[o] = (int32_t)(best.place / kWave);
    out_token[o] = (int64_t)tokens[best.place / kWave][best.place % kWave];
  }
}

// Pieces of a row and the vectors of one: enough workgroups for every CU several times over, and
// no piece below a workgroup's round of loads.
struct Pieces {
  int count, per;
};
Pieces pieces_of(int64_t rows, int64_t V, int elem) {
  const int64_t e = 16 / elem, vectors = (V + e - 1) / e;
  const int64_t least = kPartNT * kUnroll;
  const int64_t want = std::max<int64_t>(1, 1024 / std::max<int64_t>(rows, 1));
  const int64_t count = std::max<int64_t>(1, std::min(want, vectors / least));
  const int64_t per = (vectors + count - 1) / count;
  return {(int)((vectors + per - 1) / per), (int)per};
}

int sizes_ok(int64_t G, int64_t W, int64_t V, int64_t k) {
  if (G < 0 || W < 1 || V < 1 || k < 1 || V > 0x7fffffff - 65536 || G > 0x7fffffff) return ACORN_ERR_SHAPE;
  if (W > kMaxBeams || k > kMaxK) return ACORN_ERR_UNSUPPORTED;
  if (k > W * V || G * W > 65535) return ACORN_ERR_SHAPE;
  return ACORN_OK;
}

int elem_size(int dtype) { return dtype == ACORN_F32 ? 4 : 2; }

template <typename T>
void part(const void* logits, int64_t rs, const float* scores, int64_t rows, int64_t V, int64_t k,
          Pieces pc, void* ws, hipStream_t st) {
  u64* lists = (u64*)ws;
  float2* sums = (float2*)(lists + rows * pc.count * k);
  beam_part_kernel<T><<<dim3(pc.count, (unsigned)rows), dim3(kPartNT), 0, st>>>(
      (const T*)logits, rs, scores, (int)V, (int)k, pc.per, lists, sums);
}

}  // namespace

extern "C" int acorn_beam_select_workspace(int64_t groups, int64_t beams, int64_t vocab, int64_t k,
                                           int dtype, int64_t* bytes) {
  if (!bytes) return ACORN_ERR_VALUE;
  *bytes = 0;
  const int rc = sizes_ok(groups, beams, vocab, k);
  if (rc != ACORN_OK) return rc;
  if (dtype != ACORN_F32 && dtype != ACORN_F16 && dtype != ACORN_BF16) return ACORN_ERR_DTYPE;
  const int64_t rows = groups * beams;
  *bytes = rows * pieces_of(rows, vocab, elem_size(dtype)).count * (k + 1) * 8;
  return ACORN_OK;
}

extern "C" int acorn_beam_select(const void* logits, int64_t row_stride, const float* scores,
                                 int64_t groups, int64_t beams, int64_t vocab, int64_t k,
                                 float* out_score, int32_t* out_beam, int64_t* out_token,
                                 int32_t* status, void* ws, int64_t ws_bytes, int dtype,
                                 void* stream) {
  int64_t need = 0;
  const int rc = acorn_beam_select_workspace(groups, beams, vocab, k, dtype, &need);
  if (rc != ACORN_OK) return rc;
  if (groups == 0) return ACORN_OK;
  if (!logits || !scores || !out_score || !out_beam || !out_token || !status || !ws)
    return ACORN_ERR_VALUE;
  if (row_stride < 0 || ws_bytes < need || (uintptr_t)ws % 8 ||
      (uintptr_t)logits % (unsigned)elem_size(dtype))
    return ACORN_ERR_VALUE;
  hipStream_t st = (hipStream_t)stream;
  const int64_t rows = groups * beams;
  const Pieces pc = pieces_of(rows, vocab, elem_size(dtype));
  if (dtype == ACORN_F32) part<float>(logits, row_stride, scores, rows, vocab, k, pc, ws, st);
  if (dtype == ACORN_F16) part<_Float16>(logits, row_stride, scores, rows, vocab, k, pc, ws, st);
  if (dtype == ACORN_BF16) part<__bf16>(logits, row_stride, scores, rows, vocab, k, pc, ws, st);
  ACORN_LAUNCH_CHECK();
  const u64* lists = (const u64*)ws;
  const float2* sums = (const float2*)(lists + rows * pc.count * k);
  const unsigned waves = (unsigned)std::min<int64_t>(beams, 16);
  beam_join_kernel<<<dim3((unsigned)groups), dim3(waves * kWave), 0, st>>>(
      lists, sums, scores, (int)beams, (int)vocab, (int)k, pc.count, out_score, out_beam, out_token,
      status);
  ACORN_LAUNCH_CHECK();
  return ACORN_OK;
}
