// Beam search's selection: of a group's W beams over a vocabulary of V tokens, the
// k best continuations by
//   s(w, v) = score[w] + x[w, v] - ln sum_u exp(x[w, u]),
// sorted, equal ones in order of w and then v.
//
// Two launches. beam_part_kernel reads the logits once: a workgroup holds a piece of one
// row in registers and leaves the piece's maximum, its sum of exponentials and its k
// largest logits. Within a row the order of s is the order of x, so a piece needs
// neither the row's sum nor the beam's score. beam_join_kernel, one workgroup per
// group, joins a row's pieces, then the rows, by s in 64 bits: beams are compared
// through sums over the whole vocabulary, and 32 bits of s (2^-20 at 10) would tie
// or turn round what the logits tell apart.
//
// A value's key is its order-preserving image in 32 bits, then ~token: keys differ
// from one another, the larger is the better, and the k largest do not depend on
// the order they are met in. Tokens at -inf are no candidates here: the join puts
// them behind the others where a row has too few.
#include <algorithm>
#include <type_traits>

#include "common.h"

using namespace acorn;

namespace {

typedef uint64_t u64;
typedef uint32_t bs_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kPartNT = 256, kPartWaves = kPartNT / kWave;
constexpr int kMaxBeams = 32, kMaxK = 64;
constexpr int kHeld = 1024;                    // candidates of a piece that are kept before they are sorted
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

// ---- lists across a wave ----------------------------------------------------------------------
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

// An entry of a group's list: s as a key, then its place (beam * 64 + rank in the beam's list): the
// larger key first, of equal ones the lower place.
struct Entry {
  u64 key;
  uint32_t place;
};
template <int D>
__device__ __forceinline__ Entry lane_xor(const Entry& e, int lane) {
  return {lane_xor<D>(e.key, lane), lane_xor<D>(e.place, lane)};
}
__device__ __forceinline__ bool before(uint32_t a, uint32_t b) { return a > b; }
__device__ __forceinline__ bool before(u64 a, u64 b) { return a > b; }
__device__ __forceinline__ bool before(const Entry& a, const Entry& b) {
  return a.key > b.key || (a.key == b.key && a.place < b.place);
}

// One step of a bitonic network over the wave: of lanes that differ by D, the first keeps the
// better value where `falls`, the worse where not.
template <int D, typename U>
__device__ __forceinline__ U exchange(const U& v, int lane, bool falls) {
  const U o = lane_xor<D>(v, lane);
  const bool better = ((lane & D) == 0) == falls;
  return before(o, v) == better ? o : v;
}
template <int D, typename U>
__device__ __forceinline__ U exchanges(U v, int lane, bool falls) {
  v = exchange<D>(v, lane, falls);
  if constexpr (D > 1) v = exchanges<D / 2>(v, lane, falls);
  return v;
}
// The lanes' values in falling order, or in rising order.
template <bool FALLS, typename U>
__device__ __forceinline__ U sort_wave(U v, int lane) {
  v = exchanges<1>(v, lane, ((lane & 2) == 0) == FALLS);
  v = exchanges<2>(v, lane, ((lane & 4) == 0) == FALLS);
  v = exchanges<4>(v, lane, ((lane & 8) == 0) == FALLS);
  v = exchanges<8>(v, lane, ((lane & 16) == 0) == FALLS);
  v = exchanges<16>(v, lane, ((lane & 32) == 0) == FALLS);
  return exchanges<32>(v, lane, FALLS);
}
// The 64 best of a falling list and a rising one, falling.
template <typename U>
__device__ __forceinline__ U merge_wave(const U& top, const U& other, int lane) {
  return exchanges<32>(before(other, top) ? other : top, lane, true);
}

// The sum, or another fold, over the wave, in every lane.
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
// that equal rows have equal sums. Piece i takes vectors i * NV * kPartNT .. , NV to a lane.
//
// The k largest: at least k values of the piece reach the k-th largest of the lanes' own maxima,
// few more do as a rule, and these are gathered in LDS and sorted by one wave. Where more than
// kHeld reach it (values in order, or many alike), the k-th of those that were gathered takes its
// place: keys are different, so each time the gathered ones but k drop out.
template <typename T, int NV>
__global__ __launch_bounds__(kPartNT, 4) void beam_part_kernel(
    const T* __restrict__ logits, int64_t row_stride, const float* __restrict__ scores, int V,
    int k, u64* __restrict__ lists, float2* __restrict__ sums) {
#pragma clang fp contract(off)
  constexpr int E = 16 / sizeof(T);
  __shared__ u64 held[kHeld];
  __shared__ uint32_t maxima[kPartWaves][kWave];
  __shared__ float wave_m[kPartWaves], wave_s[kPartWaves];
  __shared__ u64 limit;
  __shared__ int count;
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
  const uint32_t last = (uint32_t)max(full - 1 - p0, 0) * 16u;
  bs_u32x4 x[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u) x[u] = bs_u32x4{0u, 0u, 0u, 0u};
  if (full > 0) {
#pragma unroll
    for (int u = 0; u < NV; ++u)
      __builtin_memcpy(&x[u], base + min((uint32_t)(tid + u * kPartNT) * 16u, last), 16);
  }
  if (p0 + NV * kPartNT > full) {                              // the row ends in this piece
    T r[E];
#pragma unroll
    for (int e = 0; e < E; ++e) r[e] = (T)-INFINITY;
    bs_u32x4 none, rest;
    __builtin_memcpy(&none, r, 16);
#pragma unroll
    for (int e = 0; e < E - 1; ++e)
      if (e < V % E) r[e] = p[(int64_t)full * E + e];
    __builtin_memcpy(&rest, r, 16);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int j = p0 + tid + u * kPartNT;
      x[u] = j < full ? x[u] : j == full ? rest : none;
    }
  }
  if (tid == 0) count = 0;

  // The lane's maximum m and s = sum exp(x - m), as powers of 2 of x log2 e - R, R the running
  // maximum's x log2 e as a float, so that one fma with one rounding makes the exponent. NaN and
  // +inf reach s as NaN, -inf adds nothing.
  float m = -INFINITY, s = 0.f, R = -kHuge * kLog2e;
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
    s *= __builtin_amdgcn_exp2f(R - Rn);
    R = Rn;
#pragma unroll
    for (int e = 0; e < E; ++e)
      s += __builtin_amdgcn_exp2f(__builtin_fmaf(vec_elem<T>(x[u], e), kLog2e, -R));
    // (a vector is worked off while the ones behind it are on their way; its sum stays here)
    asm volatile("" : "+v"(s));
    __builtin_amdgcn_sched_barrier(0);
  }
  s *= __builtin_amdgcn_exp2f(-__builtin_fmaf(fmaxf(m, -kHuge), kLog2e, -R));
  if (__ballot(fabsf(m) >= kHuge && m > -INFINITY) != 0) {     // (x log2 e is too coarse there)
    const float ref = m == -INFINITY ? 0.f : m;
    s = 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f((vec_elem<T>(x[u], e) - ref) * kLog2e);
  }
  const uint32_t sorted = sort_wave<true>(order32(m), lane);
  maxima[wid][lane] = sorted;
  const float mw = unorder32(read_lane(sorted, 0)), refw = mw == -INFINITY ? 0.f : mw;
  const float sw = over_lanes(s * __builtin_amdgcn_exp2f((m - refw) * kLog2e), lane,
                              [](float a, float b) { return a + b; });
  if (lane == 0) {
    wave_m[wid] = mw;
    wave_s[wid] = sw;
  }
  __syncthreads();
  uint32_t all = maxima[0][lane];
#pragma unroll
  for (int w = 1; w < kPartWaves; ++w) all = merge_wave(all, maxima[w][kWave - 1 - lane], lane);
  u64 least = (u64)max(read_lane(all, k - 1), kLowest + 1) << 32;

  u64 top = 0;
  for (;;) {
    int at0 = p0 + tid;
    asm volatile("" : "+v"(at0));
    const float floor = unorder32((uint32_t)(least >> 32));
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      if (__ballot(vmax[u] >= floor) == 0) continue;
      forget(x[u]);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float f = vec_elem<T>(x[u], e);
        if (f >= floor) {
          const u64 key = key_of(f, (at0 + u * kPartNT) * E + e);
          if (key >= least) {
            const int at = atomicAdd(&count, 1);
            if (at < kHeld) held[at] = key;
          }
        }
      }
    }
    __syncthreads();
    const int n = count;
    if (wid == 0) {
      top = 0;
      for (int i = 0; i < min(n, kHeld); i += kWave) {
        const u64 v = i + lane < min(n, kHeld) ? held[i + lane] : 0;
        if (__ballot(v > read_lane(top, k - 1)) == 0) continue;
        top = i == 0 ? sort_wave<true>(v, lane) : merge_wave(top, sort_wave<false>(v, lane), lane);
      }
      if (lane == 0) {
        limit = read_lane(top, k - 1);
        count = 0;
      }
    }
    if (n <= kHeld) break;
    __syncthreads();
    least = limit;
    __syncthreads();                                           // (count is 0 for all)
  }
  if (wid != 0) return;
  const int64_t at = (int64_t)row * C + piece;
  if (lane < k) lists[at * k + lane] = top;
  if (lane == 0) {
    float M = wave_m[0], S = wave_s[0];
#pragma unroll
    for (int w = 1; w < kPartWaves; ++w) {
      const float n = fmaxf(M, wave_m[w]), r = n == -INFINITY ? 0.f : n;
      S = S * __builtin_amdgcn_exp2f((M - r) * kLog2e) +
          wave_s[w] * __builtin_amdgcn_exp2f((wave_m[w] - r) * kLog2e);
      M = n;
    }
    sums[at] = make_float2(M, S);
  }
}

// ---- the join ---------------------------------------------------------------------------------
constexpr int kJoinWaves = 16, kAhead = 4;

// A wave per row: the sum of its pieces, and its k best out of their lists. Then wave 0 takes the
// group's best of the rows'.
__global__ __launch_bounds__(kJoinWaves* kWave) void beam_join_kernel(
    const u64* __restrict__ lists, const float2* __restrict__ sums,
    const float* __restrict__ scores, int W, int V, int k, int C, float* __restrict__ out_score,
    int32_t* __restrict__ out_beam, int64_t* __restrict__ out_token, int32_t* __restrict__ status) {
  __shared__ uint32_t tokens[kMaxBeams][kWave];
  __shared__ u64 keys[kMaxBeams][kWave];
  __shared__ u64 reach[kJoinWaves][(kAhead + 1) * kWave];      // of a row's entries, those that may count
  const int g = blockIdx.x, lane = threadIdx.x % kWave, wid = threadIdx.x / kWave;
  const int waves = blockDim.x / kWave;
  for (int w = wid; w < W; w += waves) {
    const int64_t row = (int64_t)g * W + w;
    const float score = scores[row];
    // (the first loads together: what they find of a row that was not read is not used)
    const float2* sp = sums + row * C;
    const u64* lp = lists + row * C * k;
    const int total = C * k;
    const float2 ms0 = sp[min(lane, C - 1)];
    const uint32_t head = (uint32_t)(lp[(int64_t)min(lane, C - 1) * k] >> 32);
    u64 ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ahead[i] = lp[min(i * kWave + lane, total - 1)];
    bool bad = !(score < INFINITY), live = score > -INFINITY && !bad;
    double ref = 0.0, log_sum = 0.0;           // ln sum exp(x) = ref + log_sum
    u64 top = 0;
    if (live) {
      float M = lane < C ? ms0.x : -INFINITY;
      for (int c = lane + kWave; c < C; c += kWave) M = fmaxf(M, sp[c].x);
      M = over_lanes(M, lane, [](float a, float b) { return fmaxf(a, b); });
      ref = M == -INFINITY ? 0.0 : (double)M;
      double S = 0.0;
      for (int c = lane; c < C; c += kWave) {
        const float2 ms = c < kWave ? ms0 : sp[c];
        S += (double)ms.y * exp2(((double)ms.x - ref) * (double)kLog2e);
      }
      S = over_lanes(S, lane, [](double a, double b) { return a + b; });
      if (!(S == S)) bad = true;
      live = !bad && M > -INFINITY;
      // (the pieces' exponentials are powers of 2 of x * kLog2e, which as a float is 1.3e-8 off)
      log_sum = log2(S) / (double)kLog2e;
    }
    if (live) {
      // lists begin with their largest: at least k entries reach the k-th of (the first 64 of) those
      const uint32_t reaches = sort_wave<true>(lane < C ? head : 0u, lane);
      const u64 least = max((u64)read_lane(reaches, k - 1) << 32, (u64)1);
      u64* buf = reach[wid];
      int n = 0;
      auto flush = [&]() {
        __builtin_amdgcn_wave_barrier();
        n -= kWave;
        const u64 v = n + lane >= 0 ? buf[n + lane] : 0;
        n = max(n, 0);
        __builtin_amdgcn_wave_barrier();
        top = merge_wave(top, sort_wave<false>(v, lane), lane);
      };
      for (int i0 = 0; i0 < total; i0 += kAhead * kWave) {
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const int i = i0 + a * kWave + lane;
          const bool in = i < total && ahead[a] >= least;
          const u64 mask = __ballot(in);
          if (in) buf[n + __popcll(mask & ((1ull << lane) - 1))] = ahead[a];
          n += __popcll(mask);
          ahead[a] = lp[min(i + kAhead * kWave, total - 1)];
        }
        while (n >= kWave) flush();
      }
      if (n > 0) flush();
    }
    // behind the row's tokens above -inf (all of them are in the list, if there are fewer than k):
    // the lowest others, at -inf
    const uint32_t token = ~(uint32_t)top;
    const int have = live ? __popcll(__ballot(top != 0)) : 0;
    u64 key = 0;
    uint32_t shown = token;
    if (lane < have) {
      // (x - ref first: where logits are of the type's lowest value, their sum would swallow log_sum)
      key = order64((double)score + (((double)unorder32((uint32_t)(top >> 32)) - ref) - log_sum));
    } else {
      key = order64(-INFINITY);
      shown = lane - have;
    }
    if (have > 0 && have < min(k, V)) {
      const uint32_t rising = sort_wave<false>(lane < have ? token : 0xFFFFFFFFu, lane);
      for (int i = 0; i < have; ++i) shown += lane >= have && read_lane(rising, i) <= shown;
    }
    keys[w][lane] = lane < min(k, V) ? key : 0;
    tokens[w][lane] = shown;
    if (lane == 0) status[row] = bad;
  }
  __syncthreads();
  if (wid != 0) return;
  Entry best = {0, 0xFFFFFFFFu};
  for (int i = 0; i < W * k; i += kWave) {
    const int at = i + lane, w = at / k, r = at % k;
    const bool on = at < W * k;
    Entry e = {on ? keys[w][r] : 0, on ? (uint32_t)(w * kWave + r) : 0xFFFFFFFFu};
    const Entry last = {read_lane(best.key, k - 1), read_lane(best.place, k - 1)};
    if (__ballot(before(e, last)) == 0) continue;
    best = i == 0 ? sort_wave<true>(e, lane) : merge_wave(best, sort_wave<false>(e, lane), lane);
  }
  if (lane < k) {
    const int64_t o = (int64_t)g * k + lane;
    out_score[o] = (float)unorder64(best.key);
    out_beam[o] = (int32_t)(best.place / kWave);
    out_token[o] = (int64_t)tokens[best.place / kWave][best.place % kWave];
  }
}

// Vectors of a lane and pieces of a row: the longest pieces that still make workgroups for every
// place of the chip (four to a CU), so that a batch runs in one round.
struct Pieces {
  int count, nv;
};
Pieces pieces_of(int64_t rows, int64_t V, int elem) {
  const int64_t e = 16 / elem, vectors = (V + e - 1) / e;
  Pieces pc = {0, 0};
  for (int nv : {2, 5, 10, 20}) {
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
          Pieces pc, void* ws, hipStream_t st) {
  u64* lists = (u64*)ws;
  float2* sums = (float2*)(lists + rows * pc.count * k);
  auto kfn = pc.nv == 2   ? beam_part_kernel<T, 2>
             : pc.nv == 5  ? beam_part_kernel<T, 5>
             : pc.nv == 10 ? beam_part_kernel<T, 10>
                           : beam_part_kernel<T, 20>;
  kfn<<<dim3(pc.count, (unsigned)rows), dim3(kPartNT), 0, st>>>((const T*)logits, rs, scores, (int)V,
                                                                (int)k, lists, sums);
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
  const unsigned waves = (unsigned)std::min<int64_t>(beams, kJoinWaves);
  beam_join_kernel<<<dim3((unsigned)groups), dim3(waves * kWave), 0, st>>>(
      lists, sums, scores, (int)beams, (int)vocab, (int)k, pc.count, out_score, out_beam, out_token,
      status);
  ACORN_LAUNCH_CHECK();
  return ACORN_OK;
}
