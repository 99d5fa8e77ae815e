// Attention over the 8-bit paged KV cache (format and layout: kv8.h):
//   acorn_paged_attention_kv8          one new token per sequence, split over
//                                      the cache's length and joined
//   acorn_paged_prefill_attention_kv8  packed prompt rows, causal
// Both turn bytes into bf16 / fp16 and use the 16-bit MFMAs with fp32 sums. The
// conversion is exact within the type's range: fp16 (K, and V of prompt attention)
// rounds what lies below 2^-14 to steps of 2^-24. The fp8 MFMAs would take the bytes
// as they lie, with q in two or three e4m3 terms, but add their products to fewer
// bits: measured against 64 bits 1.6e-5 of the sum of magnitudes for normal numbers,
// 2.8e-4 where one in sixteen is a hundred times larger, 2e-8 with the bf16 MFMA.
#include <algorithm>
#include <type_traits>

#include "attention_common.h"
#include "kv8.h"

using namespace acorn;

namespace {

// Two floats rounded to T, lo in the low half: one instruction for either type.
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  typedef T t2 __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 f = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, t2));
}

// ---------------------------------------------------------------------------
// Decode. A workgroup of NWV waves serves one (split, kv head, sequence); its
// waves divide the split's groups of 16 tokens. Per step of two groups, with
// lane = 16 r + c:
//  * S^T = K q^T on v_mfma_f32_16x16x32: A = K (row = token c), from the tile's
//    pieces as they are loaded, 8 conversions of two bytes per MFMA pair; a
//    token's scale goes into its conversions. B = q^T (column = head c; columns
//    past REP repeat the last head). Register i of lane (r, c) then holds the
//    score of head c for token 4 r + i.
//  * online softmax in that layout, the maximum moved only by scores that
//    exceed it by more than kMaxSlack. p goes through the MFMAs as two bf16 terms, p
//    cut to bf16 and the rest, and l sums p itself: as near to 64 bits as the
//    result's own rounding lets it be, and free beside the loads (with one term the
//    error of a result is 1.4 times that rounding's). V's bytes become bf16 for it, in
//    fp16 too: exactly, and p has no least step (one fp16 term lost the weight of
//    tokens 17.5 below the largest score, and half of it at 17).
//  * O^T += V^T P^T on v_mfma_f32_16x16x32: B = the p of lane (r, c) as they
//    stand (tokens 4 r .. 4 r + 3 of both groups); A = V^T, from the E dims of
//    those tokens that the lane has loaded and converted, transposed by v_perm.
// The wave's block ids are fetched one step ahead of their tiles, DEPTH steps
// of tiles are in flight. Loads are unconditional (wait counts stay static):
// those past the wave's last group read one line of it.
// Bound by memory: 64 sequences of 1024..8192 tokens, 32 / 8 heads, 105 us, 5.4
// TB/s; one of 131000, 16 / 8 heads, 48.7 us, 5.5 TB/s (a large copy: 4.8). In one
// sweep, where the first took 111 (another card): with default instead of non-temporal loads 120, three
// steps in flight 111, four waves per workgroup 109 to 117 by splits, 128 registers for four
// waves per SIMD 185.
template <typename T, int D, int REP, int NWV, int DEPTH>
__global__ __launch_bounds__(NWV * kWave, 2) void kv8_decode_kernel(
    const T* __restrict__ q, const uint8_t* __restrict__ k_tiles,
    const uint8_t* __restrict__ v_tiles, const uint8_t* __restrict__ scales,
    const int32_t* __restrict__ tables, const int32_t* __restrict__ lens, T* __restrict__ out,
    float* __restrict__ ws_acc, float* __restrict__ ws_m, float* __restrict__ ws_l, int H, int KV,
    int P, int num_blocks, int table_stride, int S, float scale_log2) {
  constexpr int E = D / 16;                    // dims per lane of V = MFMAs per P V
  constexpr int KP = D / 64;                   // 16-byte pieces per lane and tile, K or V
  constexpr int KB = D / 32;                   // q.k MFMAs per group
  __shared__ __align__(16) float sacc[NWV == 1 ? 1 : NWV][REP][D];
  __shared__ float sm[NWV][REP], sl[NWV][REP];

  const int kvh = blockIdx.x, sp = blockIdx.y, b = blockIdx.z;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int r = lane >> 4, c = lane & 15;
  const int gshift = __builtin_ctz(P) - 4;     // groups per block, as a shift

  const int L = min(max(lens[b], 0), table_stride * P);
  const int groups = (L + kKv8Group - 1) / kKv8Group;
  const int npages = (L + P - 1) / P;
  const int pps = (table_stride + S - 1) / S;                 // pages per split
  const int nsb = max(1, (npages + pps - 1) / pps);           // splits this sequence uses
  if (sp >= nsb) return;                                      // uniform over the workgroup
  const int wg0 = (sp * pps) << gshift, wg1 = min(wg0 + (pps << gshift), groups);
  // this wave's groups, in pairs
  const int per = ((wg1 - wg0 + NWV - 1) / NWV + 1) & ~1;
  const int g0 = min(wg0 + wid * per, wg1), g1 = min(g0 + per, wg1);
  const int glast = max(g1 - 1, 0);
  const int32_t* trow = tables + (size_t)b * table_stride;

  u32x4_t qb[KB];
  const T* qp = q + ((size_t)b * H + kvh * REP + min(c, REP - 1)) * D;
#pragma unroll
  for (int j = 0; j < KB; ++j)
    qb[j] = *(const u32x4_t*)(qp + 64 * (j / 2) + 16 * r + 8 * (j % 2));

  auto block_of = [&](int g) -> size_t {       // of group g, clamped to the wave's last and the pool
    const unsigned pg = (unsigned)trow[min(min(g, glast) >> gshift, table_stride - 1)];
    return pg < (unsigned)num_blocks ? pg : 0u;
  };
  struct Step {
    u32x4_t k[2][KP], v[2][KP];
    uint32_t ks[2], vs[2];
  };
  auto load = [&](int g, const size_t (&blk)[2], Step& s) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int gc = min(g + u, glast);
      const size_t tile = ((blk[u] * KV + kvh) << gshift) + (gc & ((1 << gshift) - 1));
      const uint32_t off = g + u <= glast ? lane * 16 : 0;
      const uint8_t* kb = k_tiles + tile * (16 * D);
      const uint8_t* vb = v_tiles + tile * (16 * D);
      const uint8_t* sb = scales + tile * 32;
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        s.k[u][i] = load_nt((const u32x4_t*)(kb + off + 1024 * i));
        s.v[u][i] = load_nt((const u32x4_t*)(vb + off + 1024 * i));
      }
      s.ks[u] = sb[c];
      s.vs[u] = *(const uint32_t*)(sb + 16 + 4 * r);
    }
  };
  // m starts at the least finite number: scores of -inf (a product past 32 bits) have no weight
  // also where a wave begins with them
  float m = -__FLT_MAX__, l = 0.f;
  f32x4_t acc[E];
#pragma unroll
  for (int j = 0; j < E; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  auto consume = [&](int g, Step& s) {
    f32x4_t sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      const float f = kv8_scale(s.ks[u]);
#pragma unroll
      for (int j = 0; j < KB; ++j)
        sc[u] = mfma16x16x32<T>(kv8_cvt8<T>(s.k[u][j / 2][2 * (j % 2)], s.k[u][j / 2][2 * (j % 2) + 1], f),
                                qb[j], sc[u]);
    }
    float x[8];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * u + i] = sc[u][i] * scale_log2;
    if (kKv8Group * (g + 2) > L || g + 2 > g1) {
      // tokens past the sequence, or past the wave's groups: no weight, and V bytes and
      // codes of 0 (a block may hold anything there)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (g + u >= g1 || kKv8Group * (g + u) + 4 * r + i >= L) {
            x[4 * u + i] = -INFINITY;
#pragma unroll
            for (int w = 0; w < E / 4; ++w) {
              const int at = E / 4 * i + w;
              s.v[u][at / 4][at % 4] = 0u;
            }
            s.vs[u] &= ~(0xFFu << (8 * i));
          }
    }
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, x[i]);
    if (__builtin_amdgcn_ballot_w64(mx > m + kMaxSlack) != 0) {
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float mn = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int j = 0; j < E; ++j) acc[j] *= alpha;
    }
    u32x4_t pb, pr;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p0 = __builtin_amdgcn_exp2f(x[2 * i] - m), p1 = __builtin_amdgcn_exp2f(x[2 * i + 1] - m);
      const uint32_t b0 = __float_as_uint(p0), b1 = __float_as_uint(p1);
      pb[i] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
      pr[i] = pack_pair<__bf16>(p0 - __uint_as_float(b0 & 0xffff0000u),
                                p1 - __uint_as_float(b1 & 0xffff0000u));
      l += p0 + p1;
    }
    // V: token i of group u, E dims in E / 2 words
    uint32_t vt[2][4][E / 2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float f[4] = {kv8_scale_of<0>(s.vs[u]), kv8_scale_of<1>(s.vs[u]),
                          kv8_scale_of<2>(s.vs[u]), kv8_scale_of<3>(s.vs[u])};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < E / 4; ++w) {
          const int at = E / 4 * i + w;
          vt[u][i][2 * w] = kv8_cvt2<__bf16, false>(s.v[u][at / 4][at % 4], f[i]);
          vt[u][i][2 * w + 1] = kv8_cvt2<__bf16, true>(s.v[u][at / 4][at % 4], f[i]);
        }
    }
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
      const u32x4_t va = {__builtin_amdgcn_perm(vt[0][1][j / 2], vt[0][0][j / 2], sel),
                          __builtin_amdgcn_perm(vt[0][3][j / 2], vt[0][2][j / 2], sel),
                          __builtin_amdgcn_perm(vt[1][1][j / 2], vt[1][0][j / 2], sel),
                          __builtin_amdgcn_perm(vt[1][3][j / 2], vt[1][2][j / 2], sel)};
      acc[j] = mfma16x16x32<__bf16>(va, pb, acc[j]);
      acc[j] = mfma16x16x32<__bf16>(va, pr, acc[j]);
    }
  };

  if (g0 < g1) {
    Step st[DEPTH];
    size_t blk[2];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      blk[0] = block_of(g0 + 2 * i);
      blk[1] = block_of(g0 + 2 * i + 1);
      load(g0 + 2 * i, blk, st[i]);
    }
    blk[0] = block_of(g0 + 2 * DEPTH);
    blk[1] = block_of(g0 + 2 * DEPTH + 1);
    bool more = true;
    for (int g = g0; more; g += 2 * DEPTH) {
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) {
        if (more) {
          const int gi = g + 2 * i;
          consume(gi, st[i]);
          load(gi + 2 * DEPTH, blk, st[i]);
          blk[0] = block_of(gi + 2 * DEPTH + 2);
          blk[1] = block_of(gi + 2 * DEPTH + 3);
          more = gi + 2 < g1;
        }
      }
    }
  }
  // l: each lane summed its own tokens; add the four lane rows of a head
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  // register i of accumulator j of lane (r, c) holds dim E (4 r + i) + j of head c
  if constexpr (NWV == 1) {
    if (c < REP) {
      const size_t orow = (size_t)b * H + kvh * REP + c;
      if (nsb == 1) {
        const float inv = 1.0f / l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w[E / 2];
#pragma unroll
          for (int j = 0; j < E / 2; ++j)
            w[j] = pack_pair<T>(acc[2 * j][i] * inv, acc[2 * j + 1][i] * inv);
          __builtin_memcpy(__builtin_assume_aligned(out + orow * D + E * (4 * r + i), 2 * E), w, sizeof(w));
        }
      } else {
        const size_t slot = orow * S + sp;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f[E];
#pragma unroll
          for (int j = 0; j < E; ++j) f[j] = acc[j][i];
          __builtin_memcpy(__builtin_assume_aligned(ws_acc + slot * D + E * (4 * r + i), 16), f, sizeof(f));
        }
        if (r == 0) {
          ws_m[slot] = m;
          ws_l[slot] = l;
        }
      }
    }
    return;
  }
  if (c < REP) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[E];
#pragma unroll
      for (int j = 0; j < E; ++j) f[j] = acc[j][i];
      __builtin_memcpy(__builtin_assume_aligned(&sacc[wid][c][E * (4 * r + i)], 16), f, sizeof(f));
    }
    if (r == 0) {
      sm[wid][c] = m;
      sl[wid][c] = l;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < REP * D; e += NWV * kWave) {
    const int h = e / D, d = e % D;
    // (a wave that saw a NaN score keeps m of its other scores and has l and acc NaN)
    float M = sm[0][h];
#pragma unroll
    for (int w = 1; w < NWV; ++w) M = fmaxf(M, sm[w][h]);
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < NWV; ++w) {
      // a wave without tokens has l = acc = 0
      const float f = __builtin_amdgcn_exp2f(sm[w][h] - M);
      num += f * sacc[w][h][d];
      den += f * sl[w][h];
    }
    const size_t orow = (size_t)b * H + kvh * REP + h;
    if (nsb == 1) {
      out[orow * D + d] = from_f32<T>(num / den);
    } else {
      const size_t slot = orow * S + sp;
      ws_acc[slot * D + d] = num;
      if (d == 0) {
        ws_m[slot] = M;
        ws_l[slot] = den;
      }
    }
  }
}

struct DecodeArgs {
  const void *q, *kt, *vt, *sc;
  const int32_t *tables, *lens;
  void* out;
  float *ws_acc, *ws_ml;
  int64_t B, H, KV, P, num_blocks, table_stride, S;
  float scale;
  hipStream_t st;
};

// Splits of at most this many groups of 16 tokens run as one wave, longer ones
// as eight (the split rule and what it measured: ops/kv8.py).
constexpr int64_t kOneWaveGroups = 16;
constexpr int kWaves = 8;
// LDS that a one-wave workgroup asks for without using it, so that a CU holds eight of
// them (two per SIMD) and not twelve: 12 sequences of 2000..8000 tokens 29 us against 32,
// 22 of them 48 against 52; 16, 23 and 26 KB 1 to 2 us slower.
constexpr size_t kOneWaveLds = 20 * 1024;

template <typename T, int D, int REP>
int launch_decode(const DecodeArgs& a) {
  const int64_t pps = (a.table_stride + a.S - 1) / a.S;
  const bool one = a.S > 1 && pps * (a.P / kKv8Group) <= kOneWaveGroups;
  float* ws_m = a.ws_ml;
  float* ws_l = a.ws_ml ? a.ws_ml + a.B * a.H * a.S : nullptr;
  auto kfn = one ? kv8_decode_kernel<T, D, REP, 1, 2> : kv8_decode_kernel<T, D, REP, kWaves, 2>;
  kfn<<<dim3((unsigned)a.KV, (unsigned)a.S, (unsigned)a.B), dim3((one ? 1 : kWaves) * kWave),
        one ? kOneWaveLds : 0, a.st>>>(
      (const T*)a.q, (const uint8_t*)a.kt, (const uint8_t*)a.vt, (const uint8_t*)a.sc, a.tables,
      a.lens, (T*)a.out, a.ws_acc, ws_m, ws_l, (int)a.H, (int)a.KV, (int)a.P, (int)a.num_blocks,
      (int)a.table_stride, (int)a.S, a.scale * kLog2e);
  ACORN_LAUNCH_CHECK();
  if (a.S > 1) {
    paged_attn_combine_kernel<T, D, false>
        <<<dim3((unsigned)(a.B * a.H)), dim3(kCombineWaves * kWave), 0, a.st>>>(
            a.ws_acc, ws_m, ws_l, (T*)a.out, a.lens, (int)a.H, (int)a.P, (int)a.table_stride,
            (int)a.S);
    ACORN_LAUNCH_CHECK();
  }
  return ACORN_OK;
}

template <typename T, int D>
int decode_rep(const DecodeArgs& a) {
  switch (a.H / a.KV) {
    case 1: return launch_decode<T, D, 1>(a);
    case 2: return launch_decode<T, D, 2>(a);
    case 4: return launch_decode<T, D, 4>(a);
    case 8: return launch_decode<T, D, 8>(a);
  }
  return ACORN_ERR_UNSUPPORTED;
}

// ---------------------------------------------------------------------------
// Prefill: query-tiled flash attention, causal. A workgroup serves the REP q heads
// of a kv head for WQ query tokens, wave (head, group) QW blocks of 16 of them; it
// walks the keys in steps of 32. Per step and query block, as in decode but with 16
// queries of one head as the MFMA's columns: S^T = K Q^T, the online softmax per
// query column (the maximum moved only by scores that exceed it by kMaxSlack, the
// scale inside the exp2 argument), O^T += V^T P^T. The sum of a query's P is what an
// MFMA with ones in place of V^T adds up.
//
// Bytes become T once per workgroup, on their way into LDS (rows padded by 32
// bytes: neither the score operand's reads nor the transposing ds_read_b64_tr_b16
// of V conflict). A step's MFMAs (544 cycles of a SIMD at QW = 2, D = 128) and VALU
// instructions (about 600: 16 exponentials of 16 cycles among some 100) take as long
// as each other, so they have to run at the same time: an iteration holds three
// steps' work without dependences between them, the probabilities of step s, the score
// MFMAs of step s + 1 and the P V MFMAs of step s - 1, while K of step s + 2 and V of
// step s move from registers into LDS. K and V have two LDS buffers each, with one
// barrier per step. 8192 causal tokens, 32 / 8 heads: 510 to 540 us on different cards
// (1.08 to 1.02 PFLOP/s; a large library product reaches 1.21). Where it took 521: the
// steps' parts one after another 772; P V of step s - 1 ahead of the scores, V held in
// registers over the barrier, 569; fixed orders of MFMA and VALU instructions
// (scheduling groups) and wave priorities around the MFMAs 530 to 600.
//
// P is rounded to T once (a second term would double the P V MFMAs, which already take
// as long as the VALU work), and the sum of a query's P is that of the rounded values. In
// fp16 P is held times 2^7, so that the slack's 2^8 ends at 2^15 and the type's least
// step lies 2^-31 below the largest weight (before, 2^-24: 0.4% of the weight of tokens 10
// below the largest score was lost, all of it 17.5 below); a smaller slack under a
// larger factor moves the maximum more often (8192 causal tokens in fp16 515 us without
// the factor, 519 with it, a slack of 4 2% more, of 0 15%).
//
// Masked scores are set to -inf whatever they are, and V bytes are finite, so a row
// that holds NaN reaches only the queries that see it; V rows past the last key are
// taken as 0. Steps before the workgroup's first query need no mask.
// Windows take P in two bf16 terms and V in bf16, in fp16 too, as decode does: a row
// of a window is as near to 64 bits as the same row through decode (one term 1.4
// times as far). 8 windows of 5 rows over 1024..8192 tokens 36 -> 39 us in bf16, 37
// -> 41 in fp16; the sums of P on the VALU instead of by an MFMA of ones: no change.
// SPLIT, WIN, partials and merge: as in paged_attention.hip. The kv head is the
// grid's fastest index: workgroups are dealt to the 8 XCDs round robin, so with a
// multiple of 8 kv heads a head's keys stay in one XCD's L2.
template <typename T, int D, int REP, int QG, int QW, bool SPLIT, bool WIN>
__global__ __launch_bounds__(REP * QG * kWave, 2) void kv8_prefill_kernel(
    const T* __restrict__ q, const uint8_t* __restrict__ k_tiles,
    const uint8_t* __restrict__ v_tiles, const uint8_t* __restrict__ scales,
    const int32_t* __restrict__ tables, const int32_t* __restrict__ seq_row0,
    const int32_t* __restrict__ seq_pos0, const int32_t* __restrict__ seq_nq, T* __restrict__ out,
    int R, int H, int KV, int P, int num_blocks, int table_stride, float scale_log2, int max_nq,
    int S, int cps, float* __restrict__ ws, int cap) {
  constexpr int NT = REP * QG * kWave;           // threads
  constexpr int KB = D / 32, E = D / 16, TP = 16 / E;
  constexpr int PITCH = 2 * D + 32;              // bytes per staged row
  constexpr int KC = 32;                         // keys per step
  constexpr int WQ = QG * QW * 16;               // query rows per workgroup
  constexpr int PCS = KC / kKv8Group * D;        // 16-byte pieces per step, K or V
  constexpr bool TWO = WIN;                      // P in two bf16 terms, V in bf16
  using VT = std::conditional_t<TWO, __bf16, T>;
  // P in fp16 is held times 2^kShift, at most 2^(kShift + kMaxSlack) = 2^15
  constexpr bool F16P = std::is_same<VT, _Float16>::value;
  constexpr float kShift = F16P ? 15.f - kMaxSlack : 0.f;
  constexpr int PPT = (2 * PCS + NT - 1) / NT;   // pieces per thread per step
  static_assert((2 * PCS) % NT == 0 || 2 * PCS < NT, "whole pieces per thread");
  __shared__ __align__(16) uint8_t ks[2][KC * PITCH], vs[2][KC * PITCH];
  const int kvh = blockIdx.x % KV, n = blockIdx.y;
  const int tid = threadIdx.x;
  const int wid = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lane = tid % kWave;
  const int r = lane >> 4, c = lane & 15;
  const int hq = wid % REP, sub = wid / REP;
  const int h = kvh * REP + hq;
  const PrefillSeq sq = prefill_seq<WIN>(seq_row0, seq_pos0, seq_nq, n, R, max_nq, cap);
  // (rows placed past their table row's pages are not served)
  const int pos0 = sq.pos0, row0 = sq.row0, nq = WIN ? sq.nq : min(sq.nq, cap - pos0);
  const int by = (int)((gridDim.x - 1 - blockIdx.x) / KV);      // longest tiles first
  const int tile_q = SPLIT ? by / S : by;
  const int wg_j0 = tile_q * WQ;
  if (wg_j0 >= nq) return;                                      // uniform over the workgroup
  const int j0 = wg_j0 + sub * QW * 16;                         // this wave's first query row
  const int nvalid = max(0, min(QW * 16, nq - j0));             // 0: the wave only stages
  const int L = pos0 + min(wg_j0 + WQ, nq);                     // keys of the workgroup's last query
  const int total = (L + kPrefillChunk - 1) / kPrefillChunk;
  const int sp = SPLIT ? by % S : 0;
  const int cb = SPLIT ? sp * cps : 0;
  if (cb >= total) {                             // uniform over the workgroup
    // a window's tile before its sequence's first token sees no key
    if (WIN && total <= 0 && sp == 0) {
#pragma unroll
      for (int qw = 0; qw < QW; ++qw)
        if (16 * qw + c < nvalid) {
          T* o = out + ((size_t)(row0 + j0 + 16 * qw + c) * H + h) * D + 4 * r;
#pragma unroll
          for (int jj = 0; jj < E; ++jj)
            *(u32x2_t*)(o + 16 * jj) = u32x2_t{pack_pair<T>(NAN, NAN), pack_pair<T>(NAN, NAN)};
        }
    }
    return;
  }
  // this workgroup's steps [s0, s1); those before sm need no mask
  constexpr int SPC = kPrefillChunk / KC;
  const int steps = (L + KC - 1) / KC;
  const int s0 = cb * SPC, s1 = SPLIT ? min((cb + cps) * SPC, steps) : steps;
  const int sm = min(max((pos0 + wg_j0 + 1) / KC, s0), s1);
  const int32_t* trow = tables + (size_t)n * table_stride;
  const int gshift = __builtin_ctz(P) - 4;
  const int glast = (L - 1) / kKv8Group;

  // the queries: block qw's column c is query row j0 + 16 qw + c (clamped)
  u32x4_t qb[QW][KB];
  int pc[QW];
#pragma unroll
  for (int qw = 0; qw < QW; ++qw) {
    const int jc = min(16 * qw + c, max(nvalid - 1, 0));
    pc[qw] = pos0 + j0 + jc;
    const size_t qrow = (size_t)(row0 + min(j0 + jc, nq - 1));
#pragma unroll
    for (int jb = 0; jb < KB; ++jb)
      qb[qw][jb] = *(const u32x4_t*)(q + (qrow * H + h) * D + 32 * jb + 8 * r);
  }

  // Staging. Piece x = i NT + tid of a step: K's for x < PCS, V's from there; piece x % D
  // of tile x / D. K: dims 16 (x % D / 16) .. of token x % 16. V: the E dims of TP tokens
  // (kv8.h). A wave's pieces are of one kind and one tile (D and PCS are multiples of
  // 64), so the block ids are scalar loads. An iteration stages K of the step after V's.
  struct Piece {
    u32x4_t v;
    uint32_t code;
  };
  Piece stage[PPT];
  size_t tl[PPT];
  const bool stages = 2 * PCS >= NT || wid * kWave < 2 * PCS;
  auto first = [&](int i) { return i * NT + wid * kWave; };     // the wave's first piece
  auto of_k = [&](int i) { return (i + 1) * NT <= PCS || (i * NT < PCS && first(i) < PCS); };
  auto find = [&](int i, int step) -> size_t {
    const int g = min(2 * step + (first(i) % PCS) / D, glast);
    const unsigned pg = (unsigned)trow[min(g >> gshift, table_stride - 1)];
    const size_t blk = pg < (unsigned)num_blocks ? pg : 0u;
    return ((blk * KV + kvh) << gshift) + (g & ((1 << gshift) - 1));
  };
  auto load = [&](int i, size_t tile, Piece& pc_) {
    const int p = first(i) % D + lane;           // piece of the tile
    const uint8_t* src = (of_k(i) ? k_tiles : v_tiles) + tile * (16 * D);
    const uint8_t* sb = scales + tile * 32;
    pc_.v = *(const u32x4_t*)(src + p * 16);
    if (of_k(i)) {
      pc_.code = sb[p % 16];
    } else if constexpr (TP == 2) {
      pc_.code = *(const uint16_t*)(sb + 16 + 4 * (p % 64 / 16) + 2 * (p / 64));
    } else {
      pc_.code = *(const uint32_t*)(sb + 16 + 4 * (p / 16));
    }
  };
  auto store = [&](int i, Piece& pc_, int step, int buf, auto tail) {      // the pieces of `step`
    const int p = first(i) % D + lane;
    const int t0 = (first(i) % PCS) / D * kKv8Group;            // the tile's first row
    if (of_k(i)) {
      const float f = kv8_scale(pc_.code);
      uint8_t* dst = ks[buf] + (t0 + p % 16) * PITCH + p / 16 * 32;
      *(u32x4_t*)dst = kv8_cvt8<T>(pc_.v[0], pc_.v[1], f);
      *(u32x4_t*)(dst + 16) = kv8_cvt8<T>(pc_.v[2], pc_.v[3], f);
    } else {
      const int t = t0 + 4 * (p % 64 / 16) + TP * (p / 64);
      uint8_t* dst = vs[buf] + t * PITCH + p % 16 * (2 * E);
      if constexpr (decltype(tail)::value) {     // rows past the last key
#pragma unroll
        for (int j = 0; j < TP; ++j)
#pragma unroll
          for (int w = 0; w < E / 4; ++w)
            pc_.v[E / 4 * j + w] = step * KC + t + j < L ? pc_.v[E / 4 * j + w] : 0u;
      }
#pragma unroll
      for (int j = 0; j < TP; ++j) {
        const float f = kv8_scale_finite(pc_.code >> (8 * j) & 0xFFu);
        if constexpr (TP == 2)
          *(u32x4_t*)(dst + j * PITCH) = kv8_cvt8<VT>(pc_.v[2 * j], pc_.v[2 * j + 1], f);
        else
          *(u32x2_t*)(dst + j * PITCH) =
              u32x2_t{kv8_cvt2<VT, false>(pc_.v[j], f), kv8_cvt2<VT, true>(pc_.v[j], f)};
      }
    }
  };
  // the step that piece i belongs to in iteration s
  auto step_of = [&](int i, int s) { return of_k(i) ? s + 2 : s; };

  float m[QW], nm[QW];                           // nm: -m (0 while m is -inf), plus kShift
  f32x4_t acc[QW][E], accl[QW], sc[QW][2];
  u32x4_t va[E], pb[QW], pr[TWO ? QW : 1];       // pr: the second term
  const uint32_t one2 = std::is_same<VT, __bf16>::value ? 0x3F803F80u : 0x3C003C00u;
  const u32x4_t ones = {one2, one2, one2, one2};
#pragma unroll
  for (int qw = 0; qw < QW; ++qw) {
    m[qw] = -INFINITY;
    nm[qw] = 0.f;
    accl[qw] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    pb[qw] = u32x4_t{0u, 0u, 0u, 0u};
    if constexpr (TWO) pr[qw] = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
    for (int jj = 0; jj < E; ++jj) acc[qw][jj] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t vlane = (uint32_t)((4 * r + (c >> 2)) * PITCH + 8 * (c & 3));

  auto pv_of = [&](const u32x4_t* p) {
#pragma unroll
    for (int jj = 0; jj < E; ++jj)
#pragma unroll
      for (int qw = 0; qw < QW; ++qw) acc[qw][jj] = mfma16x16x32<VT>(va[jj], p[qw], acc[qw][jj]);
#pragma unroll
    for (int qw = 0; qw < QW; ++qw) accl[qw] = mfma16x16x32<VT>(ones, p[qw], accl[qw]);
  };
  auto pv = [&]() {
    pv_of(pb);
    if constexpr (TWO) pv_of(pr);
  };
  u32x4_t kf[2][KB];
  auto read_k = [&](int step) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int jb = 0; jb < KB; ++jb)
        kf[hh][jb] = *(const u32x4_t*)(ks[step & 1] + (16 * hh + c) * PITCH + 2 * (32 * jb + 8 * r));
  };
  auto scores = [&]() {
#pragma unroll
    for (int qw = 0; qw < QW; ++qw) sc[qw][0] = sc[qw][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int jb = 0; jb < KB; ++jb)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int qw = 0; qw < QW; ++qw) sc[qw][hh] = mfma16x16x32<T>(kf[hh][jb], qb[qw][jb], sc[qw][hh]);
  };
  auto read_v = [&](int step) {
    typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;
    const __attribute__((address_space(3))) uint8_t* vl =
        (const __attribute__((address_space(3))) uint8_t*)vs[step & 1] + vlane;
#pragma unroll
    for (int jj = 0; jj < E; ++jj) {
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vl + 32 * jj));
      const s16x4_t hi =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vl + 16 * PITCH + 32 * jj));
      const u32x2_t l2 = __builtin_bit_cast(u32x2_t, lo), h2 = __builtin_bit_cast(u32x2_t, hi);
      va[jj] = u32x4_t{l2[0], l2[1], h2[0], h2[1]};
    }
  };
  // the scores of `step` (raw; lane (r, c) holds keys 4 r .. 4 r + 3 of each half for query
  // c of a block), masked, and the maxima. A move of the maximum by 2^-alpha applies to
  // the sums one iteration later, once the P V that is still due has been added to them.
  float alpha[QW];
#pragma unroll
  for (int qw = 0; qw < QW; ++qw) alpha[qw] = 1.f;
  bool moved = false;                            // uniform
  auto settle = [&](int step, auto masked) {
    if (__builtin_expect(moved, 0)) {
#pragma unroll
      for (int qw = 0; qw < QW; ++qw) {
        accl[qw] *= alpha[qw];
#pragma unroll
        for (int jj = 0; jj < E; ++jj) acc[qw][jj] *= alpha[qw];
      }
    }
    if constexpr (decltype(masked)::value) {
#pragma unroll
      for (int qw = 0; qw < QW; ++qw)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (step * KC + 16 * hh + 4 * r + i > pc[qw]) sc[qw][hh][i] = -INFINITY;
    }
    float mx[QW];
    bool up = false;
#pragma unroll
    for (int qw = 0; qw < QW; ++qw) {
      mx[qw] = sc[qw][0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx[qw] = fmaxf(mx[qw], sc[qw][i / 4][i % 4]);
      mx[qw] *= scale_log2;                      // scale_log2 > 0
      up |= mx[qw] > m[qw] + kMaxSlack;
    }
    moved = __builtin_amdgcn_ballot_w64(up) != 0;
    if (__builtin_expect(moved, 0)) {
#pragma unroll
      for (int qw = 0; qw < QW; ++qw) {
        float x = fmaxf(mx[qw], __shfl_xor(mx[qw], 16));
        x = fmaxf(x, __shfl_xor(x, 32));
        const float mn = fmaxf(m[qw], x);
        // (a query that has seen no key yet keeps -inf: alpha 0, p = exp2(-inf))
        const float neg = mn == -INFINITY ? 0.f : -mn;
        alpha[qw] = __builtin_amdgcn_exp2f(m[qw] + neg);
        nm[qw] = F16P ? neg + kShift : neg;
        m[qw] = mn;
      }
    }
  };

  // prologue, one round trip to memory: K of steps s0 and s0 + 1 staged, the pieces of
  // iteration s0 (K of s0 + 2, V of s0) in flight; as V of step s0 - 1, which the first
  // iteration multiplies by P = 0, that of s0
  {
    Piece ka[PPT], kb[PPT];
#pragma unroll
    for (int i = 0; i < PPT; ++i)
      if (stages) {
        if (of_k(i)) {
          load(i, find(i, s0), ka[i]);
          load(i, find(i, s0 + 1), kb[i]);
        }
        load(i, find(i, step_of(i, s0)), stage[i]);
      }
#pragma unroll
    for (int i = 0; i < PPT; ++i)
      if (stages) {
        tl[i] = find(i, step_of(i, s0 + 1));
        if (of_k(i)) {
          store(i, ka[i], s0, s0 & 1, std::true_type{});
          store(i, kb[i], s0 + 1, (s0 + 1) & 1, std::true_type{});
        } else {
          store(i, stage[i], s0, (s0 - 1) & 1, std::true_type{});
        }
      }
  }
  __syncthreads();
  read_k(s0);
  scores();
  if (s0 < sm) settle(s0, std::false_type{});
  else settle(s0, std::true_type{});
  __syncthreads();

  auto iteration = [&](int s, auto masked) {
    read_k(s + 1);
    u32x4_t pn[QW], rn[TWO ? QW : 1];
#pragma unroll
    for (int qw = 0; qw < QW; ++qw)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(
            __builtin_fmaf(sc[qw][i / 2][2 * (i % 2)], scale_log2, nm[qw]));
        const float p1 = __builtin_amdgcn_exp2f(
            __builtin_fmaf(sc[qw][i / 2][2 * (i % 2) + 1], scale_log2, nm[qw]));
        if constexpr (TWO) {
          const uint32_t b0 = __float_as_uint(p0), b1 = __float_as_uint(p1);
          pn[qw][i] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
          rn[qw][i] = pack_pair<__bf16>(p0 - __uint_as_float(b0 & 0xffff0000u),
                                        p1 - __uint_as_float(b1 & 0xffff0000u));
        } else {
          pn[qw][i] = pack_pair<T>(p0, p1);
        }
      }
    scores();
    read_v(s - 1);
    pv();
#pragma unroll
    for (int qw = 0; qw < QW; ++qw) {
      pb[qw] = pn[qw];
      if constexpr (TWO) pr[qw] = rn[qw];
    }
#pragma unroll
    for (int i = 0; i < PPT; ++i)
      if (stages) {
        store(i, stage[i], step_of(i, s), s & 1, masked);
        load(i, tl[i], stage[i]);                // of iteration s + 1
        tl[i] = find(i, step_of(i, s + 2));
      }
    // (without this the probabilities' work, next needed in the iteration to come, would sink
    // behind settle's branch, away from the MFMAs)
#pragma unroll
    for (int qw = 0; qw < QW; ++qw) {
      asm volatile("" : "+v"(pb[qw]));
      if constexpr (TWO) asm volatile("" : "+v"(pr[qw]));
    }
    settle(s + 1, masked);
    __syncthreads();
  };
  for (int s = s0; s < sm - 1; ++s) iteration(s, std::false_type{});
  for (int s = max(sm - 1, s0); s < s1; ++s) iteration(s, std::true_type{});
  if (nvalid == 0) return;
  read_v(s1 - 1);
  pv();
  if (moved) {
#pragma unroll
    for (int qw = 0; qw < QW; ++qw) {
      accl[qw] *= alpha[qw];
#pragma unroll
      for (int jj = 0; jj < E; ++jj) acc[qw][jj] *= alpha[qw];
    }
  }
  if (SPLIT && total > cps) {                    // one run of several: its fp32 partial
    const size_t slots = (size_t)prefill_slots(gridDim.y, R, max_nq) * H;
    float2* ml = (float2*)(ws + (size_t)S * slots * D);
#pragma unroll
    for (int qw = 0; qw < QW; ++qw)
      if (16 * qw + c < nvalid) {
        const size_t slot = (size_t)sp * slots +
                            (size_t)prefill_slot(gridDim.y, R, max_nq, n, row0, j0 + 16 * qw + c) * H + h;
#pragma unroll
        for (int jj = 0; jj < E; ++jj)
          *(f32x4_t*)(ws + slot * D + 16 * jj + 4 * r) = acc[qw][jj];
        if (r == 0) ml[slot] = make_float2(m[qw], accl[qw][0]);
      }
    return;
  }
  // lane (r, c) of block qw holds dims 16 jj + 4 r + i of query column 16 qw + c
#pragma unroll
  for (int qw = 0; qw < QW; ++qw)
    if (16 * qw + c < nvalid) {
      const size_t orow = (size_t)(row0 + j0 + 16 * qw + c) * H + h;
      const float inv = 1.0f / accl[qw][0];
#pragma unroll
      for (int jj = 0; jj < E; ++jj) {
        const u32x2_t w = {pack_pair<T>(acc[qw][jj][0] * inv, acc[qw][jj][1] * inv),
                           pack_pair<T>(acc[qw][jj][2] * inv, acc[qw][jj][3] * inv)};
        *(u32x2_t*)(out + orow * D + 16 * jj + 4 * r) = w;
      }
    }
}

struct PrefillArgs {
  const void *q, *kt, *vt, *sc;
  const int32_t *tables, *row0, *pos0, *nq;
  void* out;
  int64_t N, R, max_nq, H, KV, P, num_blocks, table_stride;
  float scale;
  PrefillPlan plan;
  float* ws;
  hipStream_t st;
};

template <typename T, int D, int REP, int QW, bool SPLIT, bool WIN>
int launch_prefill(const PrefillArgs& a) {
  constexpr int QG = REP >= 4 ? 1 : 4 / REP;
  constexpr int WQ = 16 * QW * QG;
  const int64_t tiles = (a.max_nq + WQ - 1) / WQ;
  const int S = SPLIT ? a.plan.S : 1;
  const int cap = (int)std::min<int64_t>(a.table_stride * a.P, 0x7fffffff);
  if (tiles * S > 0x7fffffff / a.KV) return ACORN_ERR_SHAPE;
  kv8_prefill_kernel<T, D, REP, QG, QW, SPLIT, WIN>
      <<<dim3((unsigned)(a.KV * tiles * S), (unsigned)a.N), dim3(REP * QG * kWave), 0,
         a.st>>>((const T*)a.q, (const uint8_t*)a.kt, (const uint8_t*)a.vt, (const uint8_t*)a.sc,
                 a.tables, a.row0, a.pos0, a.nq, (T*)a.out, (int)a.R, (int)a.H, (int)a.KV,
                 (int)a.P, (int)a.num_blocks, (int)a.table_stride, a.scale * kLog2e,
                 (int)a.max_nq, S, a.plan.cps, a.ws, cap);
  ACORN_LAUNCH_CHECK();
  if (SPLIT) {
    constexpr int pairs = kPrefillCombineNT / (D / 4);
    paged_prefill_combine_kernel<T, D, WIN, !WIN>
        <<<dim3((unsigned)((a.max_nq * a.H + pairs - 1) / pairs), (unsigned)a.N),
           dim3(kPrefillCombineNT), 0, a.st>>>(a.ws, a.row0, a.pos0, a.nq, (T*)a.out, (int)a.R,
                                               (int)a.H, (int)a.max_nq, S, a.plan.cps, WQ, cap);
    ACORN_LAUNCH_CHECK();
  }
  return ACORN_OK;
}

template <typename T, int D, int REP, bool WIN>
int prefill_form(const PrefillArgs& a) {
  if (a.plan.S > 1)
    return a.plan.qw == 1 ? launch_prefill<T, D, REP, 1, true, WIN>(a)
                          : launch_prefill<T, D, REP, 2, true, WIN>(a);
  return a.plan.qw == 1 ? launch_prefill<T, D, REP, 1, false, WIN>(a)
                        : launch_prefill<T, D, REP, 2, false, WIN>(a);
}

template <typename T, int D>
int prefill_rep(const PrefillArgs& a) {
  switch (a.H / a.KV) {
#define ACORN_REP(n) \
  case n: return a.nq ? prefill_form<T, D, n, false>(a) : prefill_form<T, D, n, true>(a);
    ACORN_REP(1)
    ACORN_REP(2)
    ACORN_REP(4)
    ACORN_REP(8)
#undef ACORN_REP
  }
  return ACORN_ERR_UNSUPPORTED;
}

int attn_shape(int64_t N, int64_t H, int64_t KV, int64_t D, int64_t P, int64_t num_blocks,
               int64_t table_stride) {
  if (N < 0 || N > 65535 || H <= 0 || KV <= 0 || KV > 65535 || H % KV != 0 || D <= 0 || P <= 0 ||
      num_blocks <= 0 || num_blocks > 0x7fffffff || table_stride < 1)
    return ACORN_ERR_SHAPE;
  if ((P & (P - 1)) != 0 || P % kKv8Group != 0 || P > 65536 || table_stride > 0x7fffffff / P - 8)
    return ACORN_ERR_SHAPE;
  const int64_t rep = H / KV;
  if ((D != 64 && D != 128) || !(rep == 1 || rep == 2 || rep == 4 || rep == 8))
    return ACORN_ERR_UNSUPPORTED;
  return ACORN_OK;
}

bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p % 16) return false;
  return true;
}

}  // namespace

extern "C" int acorn_paged_attention_kv8(const void* q, const void* k_tiles, const void* v_tiles,
                                         const void* scales, const int32_t* tables,
                                         const int32_t* seq_lens, void* out, float* ws_acc,
                                         float* ws_ml, int64_t B, int64_t H, int64_t KV, int64_t D,
                                         int64_t P, int64_t num_blocks, int64_t table_stride,
                                         int64_t num_splits, float scale, int dtype,
                                         void* stream) {
  const int rc = attn_shape(B, H, KV, D, P, num_blocks, table_stride);
  if (rc != ACORN_OK) return rc;
  if (num_splits < 1 || num_splits > 65535) return ACORN_ERR_SHAPE;
  if (B == 0) return ACORN_OK;
  if (!q || !k_tiles || !v_tiles || !scales || !tables || !seq_lens || !out) return ACORN_ERR_VALUE;
  if (num_splits > 1 && (!ws_acc || !ws_ml)) return ACORN_ERR_VALUE;
  if (!aligned16({q, k_tiles, v_tiles, scales, out, ws_acc})) return ACORN_ERR_VALUE;
  const DecodeArgs a{q,  k_tiles, v_tiles, scales, tables,       seq_lens,   out,   ws_acc, ws_ml,
                     B,  H,       KV,      P,      num_blocks,   table_stride, num_splits, scale,
                     (hipStream_t)stream};
  switch (dtype) {
    case ACORN_F16: return D == 64 ? decode_rep<_Float16, 64>(a) : decode_rep<_Float16, 128>(a);
    case ACORN_BF16: return D == 64 ? decode_rep<__bf16, 64>(a) : decode_rep<__bf16, 128>(a);
  }
  return ACORN_ERR_DTYPE;
}

extern "C" int acorn_paged_prefill_workspace_kv8(int64_t N, int64_t R, int64_t max_nq, int64_t H,
                                                 int64_t KV, int64_t D, int64_t P,
                                                 int64_t table_stride, int64_t* bytes) {
  const int rc = attn_shape(N, H, KV, D, P, 1, table_stride);
  if (rc != ACORN_OK) return rc;
  if (R < 0 || max_nq < 0 || R > 0x7fffffff || max_nq > 0x7fffffff) return ACORN_ERR_SHAPE;
  if (!bytes) return ACORN_ERR_VALUE;
  *bytes = N == 0 || R == 0 || max_nq == 0
               ? 0
               : prefill_plan(N, R, std::min(max_nq, R), H, KV, D, P, table_stride).ws_bytes;
  return ACORN_OK;
}

extern "C" int acorn_paged_prefill_attention_kv8(
    const void* q, const void* k_tiles, const void* v_tiles, const void* scales,
    const int32_t* tables, const int32_t* seq_row0, const int32_t* seq_pos0,
    const int32_t* seq_nq, void* out, int64_t N, int64_t R, int64_t max_nq, int64_t H, int64_t KV,
    int64_t D, int64_t P, int64_t num_blocks, int64_t table_stride, float scale, int dtype,
    void* ws, int64_t ws_bytes, void* stream) {
  const int rc = attn_shape(N, H, KV, D, P, num_blocks, table_stride);
  if (rc != ACORN_OK) return rc;
  if (R < 0 || max_nq < 0 || R > 0x7fffffff || max_nq > 0x7fffffff) return ACORN_ERR_SHAPE;
  if (N == 0 || R == 0 || max_nq == 0) return ACORN_OK;
  if (!q || !k_tiles || !v_tiles || !scales || !tables || !seq_pos0 || !out || !seq_row0 != !seq_nq)
    return ACORN_ERR_VALUE;
  if (!seq_nq && R != N * max_nq) return ACORN_ERR_SHAPE;
  // (the maxima are those of the scores before the factor, and -inf masks stay so behind it)
  if (!(scale > 0.f && scale * kLog2e <= __FLT_MAX__)) return ACORN_ERR_VALUE;
  if (!aligned16({q, k_tiles, v_tiles, scales, out, ws})) return ACORN_ERR_VALUE;
  max_nq = std::min(max_nq, R);                // a bound far above the rows there are costs nothing
  PrefillArgs a{q, k_tiles, v_tiles, scales, tables, seq_row0, seq_pos0, seq_nq, out, N, R, max_nq,
                H, KV, P, num_blocks, table_stride, scale,
                prefill_plan(N, R, max_nq, H, KV, D, P, table_stride), (float*)ws,
                (hipStream_t)stream};
  if (!ws || ws_bytes < a.plan.ws_bytes) a.plan.S = 1;   // nothing is split
  switch (dtype) {
    case ACORN_F16: return D == 64 ? prefill_rep<_Float16, 64>(a) : prefill_rep<_Float16, 128>(a);
    case ACORN_BF16: return D == 64 ? prefill_rep<__bf16, 64>(a) : prefill_rep<__bf16, 128>(a);
  }
  return ACORN_ERR_DTYPE;
}
