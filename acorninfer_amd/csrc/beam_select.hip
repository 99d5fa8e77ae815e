// Beam search's selection: of a group's W beams over a vocabulary of V tokens, the
// k best continuations by
//   s(w, v) = score[w] + x[w, v] - ln sum_u exp(x[w, u]),
// sorted, equal ones in order of w and then v.
//
// Two launches. beam_part_kernel reads the logits once: a workgroup takes a piece of one
// row and leaves the piece's maximum, its sum of exponentials and its k largest logits,
// sorted. Within a row the order of s is the order of x, so a piece needs neither the
// row's sum nor the beam's score. beam_join_kernel, one workgroup per group, joins a
// row's pieces, then the rows, by s in 64 bits: beams are compared through sums over the
// whole vocabulary, and 32 bits of s (2^-20 at 10) would tie or turn round what the
// logits tell apart. A score may come and go in two words of 32 bits: a search adds up
// thousands of steps, and a sum rounded to 32 bits at each of them would be as coarse.
//
// A value's key is its order-preserving image in 32 bits, then ~token: keys differ
// from one another, the larger is the better, and the k largest do not depend on
// the order they are met in. Tokens at -inf are no candidates here: the join puts
// them behind the others where a row has too few.
//
// Rows of 151936 in bf16, from a graph: 1 row 7.8 us (k 2), 4 rows 8.4 (4 beams, k 8), 64 rows 13.4, 256
// rows 22.3 (8 beams, k 16: 23.5; 78 MB, 3.3 TB/s), 1024 rows 65 (4.8 TB/s). Few rows are latency: two
// launches, each with a chain of loads, a sort and a join. Of 256 rows' pieces, 19 us, the workgroups
// have their loads after 6 to 15.5 us, and each takes 3 more: threshold 0.7, queue 1.1, look 0.4, sort
// and write 0.9; that of the last ones has nothing beside it. Many rows are bound by VALU work (46
// instructions per vector of 8, 9 of them exponentials) beside the loads.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "common.h"

using namespace acorn;

namespace {

typedef uint64_t u64;
typedef uint32_t bs_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kPartNT = 256, kPartWaves = kPartNT / kWave;
constexpr int kMaxBeams = 32, kMaxK = 64;
constexpr int kHeld = 256;                     // a wave's candidates that are kept until they are sorted
constexpr int kQueue = 5 * kWave;              // a wave's vectors that may hold candidates
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHuge = 1e6f;                   // to here x log2 e as a float is off by less than 1 / 8
constexpr uint32_t kLowest = 0x007FFFFFu;      // order32 of -inf

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


// A vector as the compiler has not seen it: what it made of it before is not kept in registers.
__device__ __forceinline__ void forget(bs_u32x4& w) { asm volatile("" : "+v"(w)); }

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

// ---- across a wave ----------------------------------------------------------------------------
// The value of lane ^ D, D a power of two, without the LDS: DPP within rows of 16, else the
// swaps of rows and halves (of a value with itself: the even and the odd rows' in every lane).
template <int D>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v, int lane) {
  auto dpp = [](uint32_t x, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xF, 0xF, false);
  };
  if constexpr (D == 1) return dpp(v, std::integral_constant<int, 0xB1>{});        // quads 1 0 3 2
  else if constexpr (D == 2) return dpp(v, std::integral_constant<int, 0x4E>{});   // quads 2 3 0 1
  else if constexpr (D == 4)                                   // half rows mirrored, then quads
    return dpp(dpp(v, std::integral_constant<int, 0x141>{}), std::integral_constant<int, 0x1B>{});
  else if constexpr (D == 8) return dpp(v, std::integral_constant<int, 0x128>{});  // rows turned by 8
  else if constexpr (D == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return (lane & 16) ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (lane & 32) ? r[0] : r[1];
  }
}
template <int D>
__device__ __forceinline__ u64 lane_xor(u64 v, int lane) {
  return (u64)lane_xor<D>((uint32_t)(v >> 32), lane) << 32 | lane_xor<D>((uint32_t)v, lane);
}
template <typename U>
__device__ __forceinline__ U read_lane(U v, int lane);
template <>
__device__ __forceinline__ uint32_t read_lane(uint32_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
template <>
__device__ __forceinline__ u64 read_lane(u64 v, int lane) {
  return (u64)read_lane((uint32_t)(v >> 32), lane) << 32 | read_lane((uint32_t)v, lane);
}

// (of a condition, that is: __ballot makes an integer of it first)
__device__ __forceinline__ u64 ballot(bool c) { return __builtin_amdgcn_ballot_w64(c); }

__device__ __forceinline__ int lanes_before(u64 mask) {        // set bits below this lane's
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// One step of a bitonic network over the wave: of lanes that differ by D, the first keeps the
// larger value where `falls`, the smaller where not.
template <int D, typename U>
__device__ __forceinline__ U exchange(U v, int lane, bool falls) {
  const U o = lane_xor<D>(v, lane);
  const bool larger = ((lane & D) == 0) == falls;
  if constexpr (sizeof(U) == 4) return larger ? max(o, v) : min(o, v);   // (a swap to an operand)
  return (o > v) == larger ? o : v;
}
template <int D, typename U>
__device__ __forceinline__ U exchanges(U v, int lane, bool falls) {
  v = exchange<D>(v, lane, falls);
  if constexpr (D > 1) v = exchanges<D / 2>(v, lane, falls);
  return v;
}
// The lanes' values in rising order.
template <typename U>
__device__ __forceinline__ U sort_wave(U v, int lane) {
  v = exchanges<1>(v, lane, (lane & 2) != 0);
  v = exchanges<2>(v, lane, (lane & 4) != 0);
  v = exchanges<4>(v, lane, (lane & 8) != 0);
  v = exchanges<8>(v, lane, (lane & 16) != 0);
  v = exchanges<16>(v, lane, (lane & 32) != 0);
  return exchanges<32>(v, lane, false);
}
// The first n lanes' values in falling order, zeros (no larger than any) behind them: 10 exchanges for
// up to 16, 15 for up to 32.
template <typename U>
__device__ __forceinline__ U sort_first(U v, int lane, int n) {
  v = exchanges<1>(v, lane, (lane & 2) == 0);
  v = exchanges<2>(v, lane, (lane & 4) == 0);
  v = exchanges<4>(v, lane, (lane & 8) == 0);
  v = exchanges<8>(v, lane, n <= 16 || (lane & 16) == 0);
  if (n <= 16) return v;
  v = exchanges<16>(v, lane, n <= 32 || (lane & 32) == 0);
  if (n <= 32) return v;
  return exchanges<32>(v, lane, true);
}
// The value of lane 63 - lane.
template <typename U>
__device__ __forceinline__ U mirror(U v, int lane) {
  auto row = [](uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xF, 0xF, false);   // rows mirrored
  };
  if constexpr (sizeof(U) == 8)
    return (U)mirror((uint32_t)(v >> 32), lane) << 32 | mirror((uint32_t)v, lane);
  else
    return lane_xor<32>(lane_xor<16>(row(v), lane), lane);
}
// The 64 best of two falling lists, falling.
template <typename U>
__device__ __forceinline__ U merge_wave(U top, U other, int lane) {
  return exchanges<32>(max(top, mirror(other, lane)), lane, true);
}

// The sum, or another fold, over the wave, in every lane.
__device__ __forceinline__ uint32_t from_bits(uint32_t v, uint32_t) { return v; }
__device__ __forceinline__ uint32_t bits_of(uint32_t v) { return v; }
__device__ __forceinline__ float from_bits(uint32_t v, float) { return __uint_as_float(v); }
__device__ __forceinline__ double from_bits(u64 v, double) { return __builtin_bit_cast(double, v); }
__device__ __forceinline__ uint32_t bits_of(float v) { return __float_as_uint(v); }
__device__ __forceinline__ u64 bits_of(double v) { return __builtin_bit_cast(u64, v); }
template <int D = 32, typename F, typename Op>
__device__ __forceinline__ F over_lanes(F v, int lane, Op op) {
  v = op(v, from_bits(lane_xor<D>(bits_of(v), lane), v));
  if constexpr (D > 1) v = over_lanes<D / 2>(v, lane, op);
  return v;
}

// ---- pieces -----------------------------------------------------------------------------------
// A row in vectors of 16 bytes from its first element, whatever that one's alignment (the loads
// are by element): what a lane adds up, and in which order, depends on the row's values alone, so
// that equal rows have equal sums. Piece i takes vectors i * NV * kPartNT .. , NV to a lane, all
// of them on their way before the first is worked off.
//
// Candidates. `least`, which at least k values of the piece reach and few more do as a rule, comes
// from the lanes' maxima: the k-th largest of a wave's, or what k / 4 of each wave's reach. Vectors
// whose maximum reaches it (some 30 of a piece at k = 16) are queued in LDS and looked at one to a
// lane, and what is found is sorted by one wave (256 rows: 19 us; with the vectors of the lanes that
// reach it read again 23, with places counted instead of sorted 23; lists left unsorted make the
// join longer by more than the sort takes). Where a wave finds more than kHeld (values in
// order, or many alike), the k-th largest of those that were held takes its place: keys are
// different, so each time the ones held but k drop out.
struct Piece {
  float m, s;                                                  // the maximum, sum exp(x - m)
};

template <typename T, int NV>
__global__ __launch_bounds__(kPartNT, 4) void beam_part_kernel(
    const T* __restrict__ logits, int64_t row_stride, const float* __restrict__ scores, int V,
    int k, u64* __restrict__ lists, Piece* __restrict__ pieces) {
#pragma clang fp contract(off)
  constexpr int E = 16 / sizeof(T);
  __shared__ u64 held[kPartWaves][kHeld];
  __shared__ bs_u32x4 queue[kPartWaves][kQueue];
  __shared__ uint32_t first[kPartWaves][kQueue];               // their first tokens
  __shared__ float wave_m[kPartWaves], wave_s[kPartWaves];
  __shared__ uint32_t some[kPartWaves], most[kPartWaves];
  __shared__ int found[kPartWaves];
  __shared__ u64 limit;
  const int row = blockIdx.y, piece = blockIdx.x, C = gridDim.x;
  const float score = scores[row];
  if (!(score > -INFINITY && score < INFINITY)) return;        // no such beam: nothing is read
  const T* p = logits + row * row_stride;
  const int tid = threadIdx.x, lane = tid % kWave, wid = tid / kWave;
  const int full = V / E;                                      // the row's whole vectors
  const int p0 = piece * (NV * kPartNT);                       // the piece's first
  // this lane's vectors are p0 + tid + u * kPartNT; those past the row's whole ones read the last
  // of these
  const uint8_t* base = (const uint8_t*)(p + (int64_t)min(p0, max(full - 1, 0)) * E);
  const uint32_t last = (uint32_t)min(max(full - 1 - p0, 0), NV * kPartNT) * 16u;
  bs_u32x4 x[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u) x[u] = bs_u32x4{0u, 0u, 0u, 0u};
  if (full > 0) {
#pragma unroll
    for (int u = 0; u < NV; ++u)
      __builtin_memcpy(&x[u], base + min((uint32_t)(tid + u * kPartNT) * 16u, last), 16);
  }
  // the row's last elements, and nothing behind them
  auto ending = [&](int j) {
    T r[E];
#pragma unroll
    for (int e = 0; e < E; ++e) r[e] = (T)-INFINITY;
#pragma unroll
    for (int e = 0; e < E - 1; ++e)
      if (j == full && e < V % E) r[e] = p[(int64_t)full * E + e];
    bs_u32x4 w;
    __builtin_memcpy(&w, r, 16);
    return w;
  };
  if (p0 + NV * kPartNT > full) {                              // the row ends in this piece
    const bs_u32x4 none = ending(full + 1), rest = ending(full);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int j = p0 + tid + u * kPartNT;
      x[u] = j < full ? x[u] : j == full ? rest : none;
    }
  }

  // The lane's maximum m and s = sum exp(x - m), as powers of 2 of x log2 e - R, R the running
  // maximum's x log2 e as a float, so that one fma with one rounding makes the exponent. NaN and
  // +inf reach s as NaN, -inf adds nothing.
  // Beside a token that has nearly all of the probability the others are below half a unit in the
  // last place of s one by one: what an addition of a vector's sum rounds off is kept in `lost`.
  float m = -INFINITY, s = 0.f, lost = 0.f, R = -kHuge * kLog2e;
  float vmax[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    forget(x[u]);
    float vm = vec_elem<T>(x[u], 0);
#pragma unroll
    for (int e = 1; e < E; ++e) vm = fmaxf(vm, vec_elem<T>(x[u], e));
    vmax[u] = vm;
    m = fmaxf(m, vm);
    const float Rn = fmaxf(m, -kHuge) * kLog2e;
    const float scale = __builtin_amdgcn_exp2f(R - Rn);
    R = Rn;
    float t = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      t += __builtin_amdgcn_exp2f(__builtin_fmaf(vec_elem<T>(x[u], e), kLog2e, -R));
    s *= scale;
    const float sum = s + t;
    lost = lost * scale + (t - (sum - s));         // (exact where s >= t, as it soon is)
    s = sum;
    // (a vector is worked off while the ones behind it are on their way; its sum stays here)
    asm volatile("" : "+v"(s), "+v"(lost));
    __builtin_amdgcn_sched_barrier(0);
  }
  s = (s + lost) * __builtin_amdgcn_exp2f(-__builtin_fmaf(fmaxf(m, -kHuge), kLog2e, -R));
  if (ballot(fabsf(m) >= kHuge && m > -INFINITY) != 0) {     // (x log2 e is too coarse there)
    const float ref = m == -INFINITY ? 0.f : m;
    s = 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      forget(x[u]);
#pragma unroll
      for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f((vec_elem<T>(x[u], e) - ref) * kLog2e);
    }
  }

  const uint32_t rising = sort_wave(order32(m), lane);
  const float mw = over_lanes(m, lane, [](float a, float b) { return fmaxf(a, b); });
  const float refw = mw == -INFINITY ? 0.f : mw;
  const float sw = over_lanes(s * __builtin_amdgcn_exp2f((m - refw) * kLog2e), lane,
                              [](float a, float b) { return a + b; });
  // (read where all lanes are active: in a branch of one, what the others' values come from may be
  // computed for that one alone)
  const uint32_t part_k = read_lane(rising, kWave - (k + kPartWaves - 1) / kPartWaves);
  const uint32_t wave_k = read_lane(rising, kWave - k);
  if (lane == 0) {
    wave_m[wid] = mw;
    wave_s[wid] = sw;
    some[wid] = part_k;
    most[wid] = wave_k;
  }
  __syncthreads();
  u64 least = (u64)max(max(min(min(some[0], some[1]), min(some[2], some[3])),
                           max(max(most[0], most[1]), max(most[2], most[3]))), kLowest + 1) << 32;

  const int64_t at = (int64_t)row * C + piece;
  for (;;) {
    const float floor = unorder32((uint32_t)(least >> 32));
    int n = 0;                                                 // found by this wave
    // all vectors, or where the queue does not hold them as many at a time as fit for certain
    constexpr int kTurn = kQueue / kWave;
    uint32_t turn = ~0u;
    for (;;) {
      int q = 0;                                               // queued
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        if (NV > kTurn && !(turn >> u & 1)) continue;
        const bool any = vmax[u] >= floor;
        const u64 mask = ballot(any);
        if (mask == 0) continue;
        const int i = q + lanes_before(mask);
        if (any && (NV <= kTurn || i < kQueue)) {
          queue[wid][i] = x[u];
          first[wid][i] = (uint32_t)(p0 + tid + u * kPartNT) * E;
        }
        q += __popcll(mask);
      }
      if (NV > kTurn && q > kQueue) {
        turn = (1u << kTurn) - 1;
        continue;
      }
      __builtin_amdgcn_wave_barrier();
      // an element to a lane
      const uint8_t* values = (const uint8_t*)queue[wid];
#pragma unroll 1
      for (int i0 = 0; i0 < q * E; i0 += kWave) {
        const int i = i0 + lane, j = min(i, q * E - 1);
        T value;
        __builtin_memcpy(&value, values + j * sizeof(T), sizeof(T));
        const u64 key = key_of((float)value, first[wid][j / E] + j % E);
        const bool in = i < q * E && key >= least;
        const u64 mask = ballot(in);
        const int to = n + lanes_before(mask);
        if (in && to < kHeld) held[wid][to] = key;
        n += __popcll(mask);
      }
      __builtin_amdgcn_wave_barrier();
      if (NV <= kTurn || turn >> (NV - 1)) break;
      turn <<= kTurn;
    }
    if (lane == 0) found[wid] = n;
    __syncthreads();
    int end[kPartWaves];                                       // of the waves' candidates in a row
    bool more = false;
#pragma unroll
    for (int w = 0; w < kPartWaves; ++w) {
      more |= found[w] > kHeld;
      end[w] = (w ? end[w - 1] : 0) + min(found[w], kHeld);
    }
    u64 top = 0;
    if (wid == 0) {
#pragma unroll 1
      for (int i = 0; i < end[kPartWaves - 1]; i += kWave) {
        const int j = i + lane;
        int w = 0, from = j;
#pragma unroll
        for (int c = 0; c < kPartWaves - 1; ++c)
          if (j >= end[c]) w = c + 1, from = j - end[c];
        const u64 v = j < end[kPartWaves - 1] ? held[w][from] : 0;
        if (ballot(v > read_lane(top, k - 1)) == 0) continue;
        const u64 batch = sort_first(v, lane, end[kPartWaves - 1] - i);
        top = i == 0 ? batch : merge_wave(top, batch, lane);
      }
      const u64 kth = read_lane(top, k - 1);
      if (lane == 0) limit = kth;
    }
    if (!more) {
      if (wid == 0 && lane < k) lists[at * k + lane] = top;
      break;
    }
    __syncthreads();
    least = limit;
    __syncthreads();                                           // (before found is written again)
  }
  if (tid == kPartNT - 1) {
    float M = wave_m[0], S = wave_s[0];
#pragma unroll
    for (int w = 1; w < kPartWaves; ++w) {
      const float n = fmaxf(M, wave_m[w]), r = n == -INFINITY ? 0.f : n;
      S = S * __builtin_amdgcn_exp2f((M - r) * kLog2e) +
          wave_s[w] * __builtin_amdgcn_exp2f((wave_m[w] - r) * kLog2e);
      M = n;
    }
    pieces[at] = Piece{M, S};
  }
}

// ---- the join ---------------------------------------------------------------------------------
constexpr int kJoinWaves = 16;
constexpr int kAhead = 5;                      // loads of a lane in flight

// An entry of the group's list: s as a key, then its place (beam * 64 + rank in the beam's list): the
// larger key first, of equal ones the lower place.
struct Entry {
  u64 key;
  uint32_t place;
};
__device__ __forceinline__ bool comes_before(const Entry& a, const Entry& b) {
  return a.key > b.key || (a.key == b.key && a.place < b.place);
}
__device__ __forceinline__ Entry entry_of(const u64 (*keys)[kMaxK], int w, int k, int i) {
  return i < k ? Entry{keys[w][i], (uint32_t)(w * kWave + i)} : Entry{0, 0xFFFFFFFFu};
}
template <int D>
__device__ __forceinline__ Entry exchange_entries(const Entry& v, int lane, bool ordered) {
  const Entry o = {lane_xor<D>(v.key, lane), lane_xor<D>(v.place, lane)};
  const Entry r = comes_before(o, v) == (((lane & D) == 0) == ordered) ? o : v;
  if constexpr (D > 1) return exchange_entries<D / 2>(r, lane, ordered);
  return r;
}
// The 64 first of a list in order and one in the opposite order, in order.
__device__ __forceinline__ Entry merge_entries(const Entry& a, const Entry& b, int lane) {
  return exchange_entries<32>(comes_before(b, a) ? b : a, lane, true);
}

// ln s to 1e-12 for normal s > 0 (2^31 pieces of sums past any need): s = 2^e f with f between
// sqrt(1/2) and sqrt(2), ln f = 2 atanh t = 2 (t + t^3/3 + ... ), t = (f - 1) / (f + 1), |t| < 0.172: the
// term of t^15 is below 5e-13. The library's log2 holds every size to the last place: 0.2 us more of
// the launch's 4, in code that is cold.
__device__ __forceinline__ double ln64(double s) {
  double f = __builtin_amdgcn_frexp_mant(s);                   // 1/2 .. 1
  int e = __builtin_amdgcn_frexp_exp(s);
  const bool low = f < 0.70710678118654752;
  f = low ? f + f : f;
  e -= low;
  const double d = f + 1.0;
  double r = __builtin_amdgcn_rcp(d);                          // (two steps of Newton's)
  r = r * __builtin_fma(-d, r, 2.0);
  r = r * __builtin_fma(-d, r, 2.0);
  const double t = (f - 1.0) * r, u = t * t;
  double p = 1.0 / 13.0;
  p = __builtin_fma(p, u, 1.0 / 11.0);
  p = __builtin_fma(p, u, 1.0 / 9.0);
  p = __builtin_fma(p, u, 1.0 / 7.0);
  p = __builtin_fma(p, u, 1.0 / 5.0);
  p = __builtin_fma(p, u, 1.0 / 3.0);
  p = __builtin_fma(p, u, 1.0);
  return __builtin_fma((double)e, 0.69314718055994531, (t + t) * p);
}

// A wave per row (or two): the sum of its pieces, and its k best out of their lists, sorted; then the
// rows' lists are merged pair by pair. (Finding every entry's place by halving in the other rows'
// lists is W^2 log k reads of LDS: as fast for 4 beams, 1 us more for 8, 11 more for 32.)
// TWO: scores come or go in two words (a branch on the pointers at run time: 0.1 to 0.2 us).
template <bool TWO>
__global__ __launch_bounds__(kJoinWaves* kWave) void beam_join_kernel(
    const u64* __restrict__ lists, const Piece* __restrict__ pieces,
    const float* __restrict__ scores, const float* __restrict__ low, int W, int V, int k, int C,
    float* __restrict__ out_score, float* __restrict__ out_low, int32_t* __restrict__ out_beam,
    int64_t* __restrict__ out_token, int32_t* __restrict__ status) {
  __shared__ uint32_t tokens[kMaxBeams][kMaxK];
  __shared__ u64 keys[kMaxBeams][kMaxK];                       // s, 0: no entry
  __shared__ u64 reach[kJoinWaves][(kAhead + 1) * kWave];      // of a row's entries, those that may count
  __shared__ u64 pair_key[kJoinWaves][kWave];
  __shared__ uint32_t pair_place[kJoinWaves][kWave];
  const int g = blockIdx.x, lane = threadIdx.x % kWave, wid = threadIdx.x / kWave;
  const int waves = blockDim.x / kWave;
  for (int w = wid; w < W; w += waves) {
    const int64_t row = (int64_t)g * W + w;
    const Piece* pc = pieces + row * C;
    const u64* lp = lists + row * C * k;
    const int total = C * k;
    double score = (double)scores[row];
    if (TWO && low) score += (double)low[row];
    // (the first loads together: what they find of a row that was not read is not used)
    const Piece b = pc[min(lane, C - 1)];
    const uint32_t head = (uint32_t)(lp[(int64_t)min(lane, C - 1) * k] >> 32);
    u64 ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ahead[i] = lp[min(i * kWave + lane, total - 1)];
    bool bad = !(score < INFINITY), live = score > -INFINITY && !bad;
    double ref = 0.0, log_sum = 0.0;           // ln sum exp(x) = ref + log_sum
    u64 top = 0;
    if (live) {
      float M = lane < C ? b.m : -INFINITY;
      for (int c = lane + kWave; c < C; c += kWave) M = fmaxf(M, pc[c].m);
      M = over_lanes(M, lane, [](float a, float b) { return fmaxf(a, b); });
      ref = M == -INFINITY ? 0.0 : (double)M;
      double S = 0.0;
      for (int c = lane; c < C; c += kWave) {
        const Piece e = c < kWave ? b : pc[c];
        S += (double)e.s * exp2(((double)e.m - ref) * (double)kLog2e);
      }
      S = over_lanes(S, lane, [](double a, double b) { return a + b; });
      if (!(S == S)) bad = true;
      live = !bad && M > -INFINITY;
      // (the pieces' exponentials are powers of 2 of x * kLog2e, which as a float is 1.3e-8 off: what
      // is left of that is 1.3e-8 times the row's entropy, 1e-7)
      log_sum = ln64(S) * (1.0 / (0.69314718055994531 * (double)kLog2e));
    }
    if (live) {
      // lists begin with their largest: at least k entries reach the k-th of (the first 64 of) those
      const uint32_t reaches = C < k ? 0u : read_lane(sort_wave(lane < C ? head : 0u, lane), kWave - k);
      const u64 least = max((u64)reaches << 32, (u64)1);
      u64* buf = reach[wid];
      int n = 0;
      bool empty = true;
#pragma unroll 1
      for (int i0 = 0; i0 < total; i0 += kAhead * kWave) {
        const bool rest = i0 + kAhead * kWave >= total;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const int i = i0 + a * kWave + lane;
          const bool in = i < total && ahead[a] >= least;
          const u64 mask = ballot(in);
          if (in) buf[n + lanes_before(mask)] = ahead[a];
          n += __popcll(mask);
          ahead[a] = lp[min(i + kAhead * kWave, total - 1)];
        }
#pragma unroll 1
        while (n >= kWave || (n > 0 && rest)) {                // 64 of them into the list
          __builtin_amdgcn_wave_barrier();
          const int from = max(n - kWave, 0), some = n - from;
          const u64 batch = sort_first(lane < some ? buf[from + lane] : (u64)0, lane, some);
          top = empty ? batch : merge_wave(top, batch, lane);
          empty = false;
          n = from;
          __builtin_amdgcn_wave_barrier();
        }
      }
    }
    const int have = live ? min(__popcll(ballot(top != 0)), k) : 0;
    uint32_t token = ~(uint32_t)top;
    u64 key = 0;
    if (lane < have)
      // (x - ref first: where logits are of the type's lowest value, their sum would swallow log_sum)
      key = order64(score + (((double)unorder32((uint32_t)(top >> 32)) - ref) - log_sum));
    if (lane < k) {
      keys[w][lane] = key;
      tokens[w][lane] = token;
    }
    __builtin_amdgcn_wave_barrier();
    if (lane >= have && lane < k) {
      // behind the row's tokens above -inf (all of them are here, if they are fewer than k): the
      // lowest others, at -inf: past as many as lie at or below them
      token = lane - have;
      for (bool moved = have > 0; moved;) {
        uint32_t t = lane - have;
        for (int j = 0; j < have; ++j) t += tokens[w][j] <= token;
        moved = t != token;
        token = t;
      }
      keys[w][lane] = lane < V ? order64(-INFINITY) : 0;
      tokens[w][lane] = token;
    }
    if (lane == 0) status[row] = bad;
  }
  __syncthreads();
  // a wave takes as many lists as fit into its lanes, every second one turned round, and merges them
  // in pairs; then the waves' lists pair by pair
  const int size = k <= 8 ? 8 : k <= 16 ? 16 : k <= 32 ? 32 : kWave, per = kWave / size;
  const int parts = (W + per - 1) / per, most = min(W, per) * size;
  Entry best = {0, 0xFFFFFFFFu};
  if (wid < parts) {
    const int w = wid * per + lane / size, i = lane % size;
    if (w < W) best = entry_of(keys, w, k, (w & 1) && size < kWave ? size - 1 - i : i);
    if (size <= 8 && most > 8) best = exchange_entries<8>(best, lane, (lane & 16) == 0);
    if (size <= 16 && most > 16) best = exchange_entries<16>(best, lane, (lane & 32) == 0);
    if (size <= 32 && most > 32) best = exchange_entries<32>(best, lane, true);
    if (wid + waves < parts)                                   // (more than 16 lists of more than 32)
      best = merge_entries(best, entry_of(keys, wid + waves, k, kWave - 1 - lane), lane);
  }
  const int lists_left = min(parts, waves);
  for (int half = lists_left > 1 ? 1 << (31 - __builtin_clz(lists_left - 1)) : 0; half > 0; half >>= 1) {
    pair_key[wid][lane] = best.key;
    pair_place[wid][lane] = best.place;
    __syncthreads();
    if (wid < half && wid + half < lists_left)
      best = merge_entries(best, Entry{pair_key[wid + half][kWave - 1 - lane],
                                       pair_place[wid + half][kWave - 1 - lane]}, lane);
    __syncthreads();
  }
  if (wid == 0 && lane < k) {
    const int64_t at = (int64_t)g * k + lane;
    const double s = unorder64(best.key);
    out_score[at] = (float)s;
    if (TWO && out_low) out_low[at] = fabs(s) <= FLT_MAX ? (float)(s - (double)(float)s) : 0.f;
    out_beam[at] = (int32_t)(best.place / kWave);
    out_token[at] = (int64_t)tokens[best.place / kWave][best.place % kWave];
  }
}

// Vectors of a lane and pieces of a row: the shortest pieces with which a batch has at most 1024
// workgroups, as many as the chip has places for (four to a CU), so that it runs in one round, each with
// one sort; the longest where none gives so few. Rows of 151936 in bf16, 4 beams, k 8, us with 2 / 5 /
// 10 / 19 vectors: 16 rows 10.0 / 9.3 / 10.8 / 11.8, 32 11.9 / 10.5 / 11.1 / 12.2, 64 15.9 / 13.3 / 13.4 /
// 14.3, 128 22.5 / 17.0 / 16.8 / 16.9, 256 35.6 / 23.7 / 22.8 / 22.5, 1024 126 / 75 / 66 / 64. 19 vectors
// is the most that 128 registers hold beside their maxima (20 spill: 1 us more for 256 rows).
// The rule does not count a piece's vectors behind the row's end, which are worked off like the others.
// Past 1024 rows of a short vocabulary most of the longest piece is such: 2048 rows of 500 17.2 / 19.6 /
// 24.2 / 31.3, of 3000 17.8 / 19.7 / 24.0 / 31.2, of 8000 23.8 / 20.4 / 24.6 / 31.8; 1025 rows of 8000
// 25.1 / 22.3 / 25.3 / 30.2 (1024, which take 5: 19.9); 512 rows of 50257 28.4 / 20.2 / 20.1 / 22.2.
struct Pieces {
  int count, nv;
};
Pieces pieces_of(int64_t rows, int64_t V, int elem) {
  const int64_t e = 16 / elem, vectors = (V + e - 1) / e;
  Pieces pc = {0, 0};
  for (int nv : {2, 5, 10, 19}) {
    pc = {(int)((vectors + nv * kPartNT - 1) / (nv * kPartNT)), nv};
    if (pc.count * rows <= 1024) break;
  }
  return pc;
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
          Pieces pc, u64* lists, Piece* pieces, hipStream_t st) {
  auto kfn = pc.nv == 2   ? beam_part_kernel<T, 2>
             : pc.nv == 5  ? beam_part_kernel<T, 5>
             : pc.nv == 10 ? beam_part_kernel<T, 10>
                           : beam_part_kernel<T, 19>;
  kfn<<<dim3(pc.count, (unsigned)rows), dim3(kPartNT), 0, st>>>(
      (const T*)logits, rs, scores, (int)V, (int)k, lists, pieces);
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
  *bytes = rows * pieces_of(rows, vocab, elem_size(dtype)).count *
           (k * (int64_t)sizeof(u64) + (int64_t)sizeof(Piece));
  return ACORN_OK;
}

extern "C" int acorn_beam_select_low(const void* logits, int64_t row_stride, const float* scores,
                                     const float* low, int64_t groups, int64_t beams, int64_t vocab,
                                     int64_t k, float* out_score, float* out_low, int32_t* out_beam,
                                     int64_t* out_token, int32_t* status, void* ws,
                                     int64_t ws_bytes, int dtype, void* stream) {
  int64_t need = 0;
  const int rc = acorn_beam_select_workspace(groups, beams, vocab, k, dtype, &need);
  if (rc != ACORN_OK) return rc;
  if (groups == 0) return ACORN_OK;
  if (!logits || !scores || !out_score || !out_beam || !out_token || !status || !ws)
    return ACORN_ERR_VALUE;
  if (row_stride < 0 || ws_bytes < need || (uintptr_t)ws % 16 ||
      (uintptr_t)logits % (unsigned)elem_size(dtype))
    return ACORN_ERR_VALUE;
  hipStream_t st = (hipStream_t)stream;
  const int64_t rows = groups * beams;
  const Pieces pc = pieces_of(rows, vocab, elem_size(dtype));
  Piece* pieces = (Piece*)ws;
  u64* lists = (u64*)(pieces + rows * pc.count);
  if (dtype == ACORN_F32) part<float>(logits, row_stride, scores, rows, vocab, k, pc, lists, pieces, st);
  if (dtype == ACORN_F16) part<_Float16>(logits, row_stride, scores, rows, vocab, k, pc, lists, pieces, st);
  if (dtype == ACORN_BF16) part<__bf16>(logits, row_stride, scores, rows, vocab, k, pc, lists, pieces, st);
  ACORN_LAUNCH_CHECK();
  const unsigned waves = (unsigned)std::min<int64_t>(beams, kJoinWaves);
  (low || out_low ? beam_join_kernel<true> : beam_join_kernel<false>)<<<dim3((unsigned)groups),
                                                                      dim3(waves * kWave), 0, st>>>(
      lists, pieces, scores, low, (int)beams, (int)vocab, (int)k, pc.count, out_score, out_low,
      out_beam, out_token, status);
  ACORN_LAUNCH_CHECK();
  return ACORN_OK;
}

extern "C" int acorn_beam_select(const void* logits, int64_t row_stride, const float* scores,
                                 int64_t groups, int64_t beams, int64_t vocab, int64_t k,
                                 float* out_score, int32_t* out_beam, int64_t* out_token,
                                 int32_t* status, void* ws, int64_t ws_bytes, int dtype,
                                 void* stream) {
  return acorn_beam_select_low(logits, row_stride, scores, nullptr, groups, beams, vocab, k, out_score,
                               nullptr, out_beam, out_token, status, ws, ws_bytes, dtype, stream);
}
