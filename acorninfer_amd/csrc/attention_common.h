// What the attention kernels over the paged caches share (paged_attention.hip:
// the 16-bit cache; kv8_attention.hip: the 8-bit one): MFMA and packing helpers,
// the merge kernels of split launches, the rows and the key split of a prefill
// launch. Everything has internal linkage: each file holds its own kernels.
#pragma once
#include <algorithm>
#include <type_traits>

#include "common.h"

using namespace acorn;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kCUs = 256;   // MI355X compute units

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

constexpr float kMaxSlack = 8.0f;

template <typename T>
__device__ __forceinline__ f32x4_t mfma16x16x32(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                    __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                   __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ f32x4_t mfma16x16x16(u32x2_t a, u32x2_t b, f32x4_t c) {
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, a),
                                                      __builtin_bit_cast(s16x4_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, a),
                                                  __builtin_bit_cast(f16x4_t, b), c, 0, 0, 0);
}

// Two values already on T's grid, packed lo | hi << 16.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const T a = (T)lo, b = (T)hi;
  return (uint32_t)__builtin_bit_cast(uint16_t, a) |
         ((uint32_t)__builtin_bit_cast(uint16_t, b) << 16);
}

// Two floats rounded to T's grid, packed lo | hi << 16; sum gains the two
// rounded values (lo first).
template <typename T>
__device__ __forceinline__ uint32_t pack_sum(float lo, float hi, float& sum) {
  if constexpr (std::is_same<T, __bf16>::value) {
    const uint32_t u = pack_bf16x2(lo, hi);
    sum += bf16_lo(u);
    sum += bf16_hi(u);
    return u;
  } else {
    const float a = round_to<T>(lo), b = round_to<T>(hi);
    sum += a;
    sum += b;
    return pack2<T>(a, b);
  }
}

// pack_sum with the two rounded values added by one dot product with (1, 1).
template <typename T>
__device__ __forceinline__ uint32_t pack_dot(float lo, float hi, float& sum) {
  if constexpr (std::is_same<T, __bf16>::value) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const uint32_t u = pack_bf16x2(lo, hi);
    sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, u),
                                          __builtin_bit_cast(bf16x2_t, 0x3F803F80u), sum, false);
    return u;
  } else {
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    const uint32_t u = pack2<T>(lo, hi);
    sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, u),
                                 __builtin_bit_cast(f16x2_t, 0x3C003C00u), sum, false);
    return u;
  }
}

// Phase 2: merge the partials of one (b, h) with the common max.
// Only sequences that used more than one split have partials; the kernels
// above wrote the others' output directly.
//
// One workgroup of kCombineWaves waves per (b, h), built so that one round
// trip to memory suffices for up to kWave splits: the length, every split's
// (m, l) (lane s) and each wave's share of the partial rows (s = wave,
// wave + kCombineWaves, ...) are all requested before any of them is used;
// slots past the sequence's split count are masked by selection, so stale
// workspace contents never reach the sums. The waves' sums are added in LDS
// in a fixed order.
constexpr int kCombineWaves = 4;

// NORM: the MFMA kernel's partials, each split's normalised output acc / l in
// fp16 (weight w_s l_s); else fp32 unnormalised acc (weight w_s).
template <typename T, int D, bool NORM>
__global__ __launch_bounds__(kCombineWaves * kWave) void paged_attn_combine_kernel(
    const float* __restrict__ ws_acc, const float* __restrict__ ws_m,
    const float* __restrict__ ws_l, T* __restrict__ out, const int32_t* __restrict__ lens,
    int H, int P, int table_stride, int S) {
  constexpr int DL = (D + kWave - 1) / kWave;        // dims per lane
  constexpr int SPW = kWave / kCombineWaves;         // slots per wave per round
  __shared__ float part[kCombineWaves][D];
  const size_t row = blockIdx.x;
  const int wid = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int d0 = lane * DL;
  const float* m = ws_m + row * S;
  const float* l = ws_l + row * S;
  const float* src = ws_acc + row * S * D;
  const _Float16* srch = (const _Float16*)ws_acc + row * S * D;
  const int pps = (table_stride + S - 1) / S;
  float a[DL];
#pragma unroll
  for (int i = 0; i < DL; ++i) a[i] = 0.f;
  float M = -INFINITY, lsum = 0.f;
  // the length as a vector load (a VGPR index), so that it is in flight with
  // the partial rows instead of a scalar round trip ahead of them
  int bi = (int)(row / H);
  asm volatile("" : "+v"(bi));
  const int lraw = lens[bi];
  int nsb = 0;
  for (int s0 = 0; s0 < S; s0 += kWave) {
    // ---- requests: (m, l) of slots s0 + lane, this wave's rows ----
    // Slots past S re-read slot S-1 and dims past D re-read dim D-1
    // (unconditional loads keep the wait counts static); every use below is
    // masked by s < nsb <= S.
    const float ml = m[min(s0 + lane, S - 1)];
    const float ll = l[min(s0 + lane, S - 1)];
    float x[SPW][DL];
#pragma unroll
    for (int k = 0; k < SPW; ++k) {
      const int s = min(s0 + wid + kCombineWaves * k, S - 1);
#pragma unroll
      for (int i = 0; i < DL; ++i) {
        const size_t e = (size_t)s * D + min(d0 + i, D - 1);
        x[k][i] = NORM ? (float)srch[e] : src[e];
      }
    }
    // The empty asm pins the requests (with the length above) ahead of the
    // early exit; otherwise they sink below it and cost a second round trip.
    asm volatile("" ::"v"(ml), "v"(ll), "v"(lraw));
#pragma unroll
    for (int k = 0; k < SPW; ++k)
#pragma unroll
      for (int i = 0; i < DL; ++i) asm volatile("" ::"v"(x[k][i]));
    // ---- use ----
    const int L = min(max(__builtin_amdgcn_readfirstlane(lraw), 0), table_stride * P);
    nsb = ((L + P - 1) / P + pps - 1) / pps;         // <= S
    if (nsb <= 1) return;                            // uniform over the workgroup
    const bool used = s0 + lane < nsb;
    const float mv = used ? ml : -INFINITY;
    const float Mr = wave_max(mv);                   // finite when s0 < nsb
    if (s0 >= nsb) break;
    const float Mn = fmaxf(M, Mr);
    const float scale_old = exp2f(M - Mn);           // 0 on the first round
    const float wl = used ? exp2f(ml - Mn) : 0.f;
    lsum = lsum * scale_old + wave_sum(used ? wl * ll : 0.f);
#pragma unroll
    for (int i = 0; i < DL; ++i) a[i] *= scale_old;
    M = Mn;
#pragma unroll
    for (int k = 0; k < SPW; ++k) {
      const int s = s0 + wid + kCombineWaves * k;
      const float w = __shfl(NORM ? wl * ll : wl, wid + kCombineWaves * k);
      if (s < nsb) {
#pragma unroll
        for (int i = 0; i < DL; ++i) a[i] += w * x[k][i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < DL; ++i)
    if (d0 + i < D) part[wid][d0 + i] = a[i];
  __syncthreads();
  const float inv = 1.0f / lsum;
  for (int d = threadIdx.x; d < D; d += kCombineWaves * kWave) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kCombineWaves; ++w) t += part[w][d];
    out[row * D + d] = from_f32<T>(t * inv);
  }
}

// One sequence of a prefill launch: its first q row, that row's position and
// its rows. WIN (no seq_nq): every sequence is a window of max_nq rows at row
// n max_nq and seq_pos0 holds its length, the window included, taken as at most
// `cap`, the tokens its table row has pages for, as K3 takes it. (A template
// parameter and not a test: one more min in the kernel of the prefill chunks
// cost 8192 causal tokens 35 of 700 us.) Rows past q's R rows (or past max_nq)
// are not served, so bad metadata cannot reach past q / out.
struct PrefillSeq {
  int row0, pos0, nq;
};
template <bool WIN>
__device__ __forceinline__ PrefillSeq prefill_seq(const int32_t* row0, const int32_t* pos0,
                                                  const int32_t* nq, int n, int R, int max_nq,
                                                  int cap) {
  PrefillSeq s;
  if constexpr (WIN) {
    s = {n * max_nq, min(max(pos0[n], 0), cap) - max_nq, max_nq};
  } else {
    s = {row0[n], pos0[n], nq[n]};
    if (s.row0 < 0 || s.pos0 < 0) s.nq = 0;
  }
  s.nq = min(min(s.nq, max_nq), R - s.row0);
  return s;
}

// Where the fp32 partials of row j of sequence n lie in a run's plane: by packed
// q row, or by (n, j) where q has many rows that no sequence covers, whichever
// plane is the smaller.
__host__ __device__ __forceinline__ int64_t prefill_slots(int64_t N, int64_t R, int64_t max_nq) {
  return R < N * max_nq ? R : N * max_nq;
}
__device__ __forceinline__ int64_t prefill_slot(int64_t N, int64_t R, int64_t max_nq, int n,
                                                int row0, int j) {
  return R < N * max_nq ? (int64_t)row0 + j : n * max_nq + j;
}

constexpr int kPrefillChunk = 64;   // keys staged per barrier (32: 3% slower at 8192 tokens)

// Merge of a split tile's partials: one group of D / 4 lanes per (row, head),
// four dims per lane; tiles of one run were written by the kernel itself.
constexpr int kPrefillCombineNT = 256;
// CAP: rows at positions past their table row's `cap` tokens are not served.
template <typename T, int D, bool WIN, bool CAP = false>
__global__ __launch_bounds__(kPrefillCombineNT) void paged_prefill_combine_kernel(
    const float* __restrict__ ws, const int32_t* __restrict__ seq_row0,
    const int32_t* __restrict__ seq_pos0, const int32_t* __restrict__ seq_nq, T* __restrict__ out,
    int R, int H, int max_nq, int S, int cps, int WQ, int cap) {
  constexpr int LPP = D / 4;
  const int n = blockIdx.y;
  const int pair = (int)(blockIdx.x * (kPrefillCombineNT / LPP)) + threadIdx.x / LPP;
  const int j = pair / H, h = pair % H, d0 = 4 * (threadIdx.x % LPP);
  PrefillSeq sq = prefill_seq<WIN>(seq_row0, seq_pos0, seq_nq, n, R, max_nq, cap);
  if (CAP) sq.nq = min(sq.nq, cap - sq.pos0);
  if (j >= sq.nq) return;
  const int L = sq.pos0 + min(j / WQ * WQ + WQ, sq.nq);
  const int total = (L + kPrefillChunk - 1) / kPrefillChunk;
  if (total <= cps) return;
  // (rows placed past their table row's pages have more runs than the S planned
  // from the table: those past S were not launched and have no partials)
  const int ns = min((total + cps - 1) / cps, S);
  const size_t slots = (size_t)prefill_slots(gridDim.y, R, max_nq) * H;
  const size_t slot = (size_t)prefill_slot(gridDim.y, R, max_nq, n, sq.row0, j) * H + h;
  const float2* ml = (const float2*)(ws + (size_t)S * slots * D) + slot;
  const float* src = ws + slot * D + d0;
  float M = -INFINITY;
  for (int s = 0; s < ns; ++s) M = fmaxf(M, ml[s * slots].x);
  f32x4_t a = {0.f, 0.f, 0.f, 0.f};
  float lsum = 0.f;
  constexpr int U = 4;                           // runs requested together
  for (int s0 = 0; s0 < ns; s0 += U) {
    f32x4_t x[U];
    float2 mls[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t s = (size_t)min(s0 + u, ns - 1);
      x[u] = *(const f32x4_t*)(src + s * slots * D);
      mls[u] = ml[s * slots];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u >= ns) continue;
      const float w = M == -INFINITY ? 0.f : exp2f(mls[u].x - M);
      lsum += w * mls[u].y;
      a += w * x[u];
    }
  }
  const float inv = 1.0f / lsum;
  const u32x2_t w = {pack2<T>(a[0] * inv, a[1] * inv), pack2<T>(a[2] * inv, a[3] * inv)};
  *(u32x2_t*)(out + ((size_t)(sq.row0 + j) * H + h) * D + d0) = w;
}

// The key split of a prefill launch: S runs of cps chunks per query tile (S ==
// 1: none) and the 16-query blocks per wave.
struct PrefillPlan {
  int qw = 2, S = 1, cps = 1;
  int64_t ws_bytes = 0;
};
// The tiles alone (R rows in all, a partly filled tile per sequence) leave
// CUs idle: split towards two workgroups per CU, the most that fit their LDS,
// three where sequences may differ in length (a short one's runs end early). A
// run costs its rows' fp32 partials, written and read: small next to a window's
// keys, about five chunks' time for a full tile, so runs keep kWindowMinRun
// chunks, kPrefillMinRun, or kPrefillBusyRun once half the CUs have a tile.
// Everything here was measured with the 16-bit cache's kernel; the 8-bit cache's
// takes the same plan, of which only single launches were timed.
// Measured, one split / this rule (us), 32 / 8 heads: 5 rows over 8000 tokens
// 157 / 27, 64 rows 213 / 39, 150 rows 216 / 63, 520 rows 227 / 150, 800 rows
// 236 / 193.
constexpr int64_t kWindowMinRun = 4, kPrefillMinRun = 6, kPrefillBusyRun = 16;
constexpr int64_t kPrefillMaxRuns = 64;
PrefillPlan prefill_plan(int64_t N, int64_t R, int64_t max_nq, int64_t H, int64_t KV, int64_t D,
                         int64_t P, int64_t table_stride) {
  PrefillPlan p;
  const int64_t rep = H / KV;
  const int64_t qg = rep >= 4 ? 1 : 4 / rep;
  if (max_nq <= 16 * qg) p.qw = 1;
  const int64_t wq = 16 * p.qw * qg;
  const int64_t tiles = std::min(N * ((max_nq + wq - 1) / wq), (R + wq - 1) / wq + N / 2);
  const int64_t base = std::max<int64_t>(1, tiles * KV);
  const int64_t chunks = (table_stride * P + kPrefillChunk - 1) / kPrefillChunk;
  const int64_t min_run = p.qw == 1 ? kWindowMinRun
                          : base >= kCUs / 2 ? kPrefillBusyRun
                                             : kPrefillMinRun;
  const int64_t target = p.qw == 2 && N > 1 ? 3 * kCUs : 2 * kCUs;
  const int64_t S = std::min(std::min((target + base / 2) / base, (chunks + min_run - 1) / min_run),
                             kPrefillMaxRuns);
  if (S <= 1) return p;
  const int64_t cps = (chunks + S - 1) / S, runs = (chunks + cps - 1) / cps;
  // ... and only where that is faster: rounds of resident workgroups times their
  // chunks, after and before, in chunks' time (1.8 us), of which the merge launch
  // takes 3 and 10 MB of partials, written and read, one. Of 1706 launches swept
  // (1..8 sequences of 5..1150 rows over 0..8000 tokens, four head counts), 251 were
  // slower split than not without this (5 x 520 rows over 1500, 16 / 8 heads, 94 us
  // against 77; 3 x 800 over 700, 32 / 8, 64 against 44), 19 with it.
  const int64_t slots = rep >= 8 ? kCUs : 2 * kCUs;    // eight-wave workgroups: one per CU
  const int64_t before = chunks * ((base + slots - 1) / slots);
  const int64_t after = cps * ((runs * base + slots - 1) / slots) + 3 +
                        runs * prefill_slots(N, R, max_nq) * H * (D + 2) * 8 / 10000000;
  if (runs <= 1 || after > before) return p;
  p.cps = (int)cps;
  p.S = (int)runs;
  // (S tiles KV stays below 4 / 3 of the target and a tile has at most 256 rows
  // of heads, so the partials take at most 1024 x 256 x (D + 2) floats, 136 MB)
  p.ws_bytes = p.S * prefill_slots(N, R, max_nq) * H * (D + 2) * 4;
  return p;
}

}  // namespace
