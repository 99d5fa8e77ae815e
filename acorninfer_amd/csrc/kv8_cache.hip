// The 8-bit paged KV cache (format and layout: kv8.h) written and read back:
//   acorn_kv8_scatter       rows of k and v into the cache
//   acorn_qkv_epilogue_kv8  the qkv projection's output -> q, and k, v into the cache
//   acorn_kv8_gather        rows of sequences out of it
// All three are bound by memory: per (token, kv head) D values of k and of v on
// one side and 2 D + 2 bytes on the other. 8 kv heads of 128: 7013 tokens written from
// fp16 9.4 us, 4.6 TB/s; 28535 tokens read into bf16 29.7 us, 5.9 TB/s; 8 tokens
// written, or 333 read, 3 us, the latency of a launch and two dependent loads.
#include <algorithm>
#include <type_traits>

#include "kv8.h"

using namespace acorn;

namespace {

constexpr int kNT = 256;

// E consecutive values as floats; p is aligned for E values of T.
template <typename T, int E>
__device__ __forceinline__ void load_row(const T* p, float (&f)[E]) {
  T r[E];
  __builtin_memcpy(r, __builtin_assume_aligned(p, E * sizeof(T) < 16 ? E * sizeof(T) : 16), sizeof(r));
#pragma unroll
  for (int i = 0; i < E; ++i) f[i] = to_f32(r[i]);
}

// 16 lanes per (row, head), the workgroup 16 rows of one head: consecutive tokens, as a
// rule one tile, whose lines one L2 then completes.
template <typename T, int D>
__global__ __launch_bounds__(kNT) void kv8_scatter_kernel(
    const T* __restrict__ k, const T* __restrict__ v, uint8_t* __restrict__ k_tiles,
    uint8_t* __restrict__ v_tiles, uint8_t* __restrict__ scales,
    const int64_t* __restrict__ pages, const int64_t* __restrict__ slots, int64_t rows, int KV,
    int P, int64_t num_blocks, int64_t k_rs, int64_t k_hs, int64_t v_rs, int64_t v_hs) {
  constexpr int E = D / 16;
  const int c = threadIdx.x & 15;
  const int64_t row = (int64_t)blockIdx.x * (kNT / 16) + (threadIdx.x >> 4);
  const int h = blockIdx.y;
  const int64_t rc = min(row, rows - 1);
  const uint64_t page = (uint64_t)pages[rc], slot = (uint64_t)slots[rc];
  float kf[E], vf[E];
  load_row<T, E>(k + rc * k_rs + h * k_hs + E * c, kf);
  load_row<T, E>(v + rc * v_rs + h * v_hs + E * c, vf);
  // a (page, slot) outside the pool is dropped rather than written
  const bool on = row < rows && page < (uint64_t)num_blocks && slot < (uint64_t)P;
  const size_t tile = (page * KV + h) * (P / kKv8Group) + slot / kKv8Group;
  kv8_store_row<D, std::is_same<T, _Float16>::value>(k_tiles, v_tiles, scales, on ? tile : 0,
                                                     (int)(slot % kKv8Group), on, c, kf, vf);
}

// The rows of a gather: sequence n's tokens pos0 .. pos0 + nq - 1 are rows row0 ..
// of the result. One workgroup per (group of 16 tokens, kv head, sequence): D
// threads take the K tile's pieces, D the V tile's. K: eight threads hold a
// token's pieces (dims 16 p ..), so that a wave reads whole lines of the tile
// and writes eight whole rows.
template <typename T, int D>
__global__ __launch_bounds__(2 * D) void kv8_gather_kernel(
    const uint8_t* __restrict__ k_tiles, const uint8_t* __restrict__ v_tiles,
    const uint8_t* __restrict__ scales, const int32_t* __restrict__ tables,
    const int32_t* __restrict__ seq_row0, const int32_t* __restrict__ seq_pos0,
    const int32_t* __restrict__ seq_nq, T* __restrict__ k_out, T* __restrict__ v_out, int R,
    int max_nq, int KV, int P, int num_blocks, int table_stride) {
  constexpr int E = D / 16, TP = 16 / E, PK = D / 16;
  const int n = blockIdx.z, h = blockIdx.y;
  const int row0 = seq_row0[n], pos0 = seq_pos0[n];
  if (row0 < 0 || pos0 < 0) return;
  const int nq = min(min(seq_nq[n], max_nq), R - row0);
  const int g = pos0 / kKv8Group + blockIdx.x;                  // group of the sequence
  // (rows placed past their table row's pages have nothing to be read from)
  if ((int64_t)g * kKv8Group >= (int64_t)pos0 + nq || g / (P / kKv8Group) >= table_stride) return;
  const unsigned pg = (unsigned)tables[(size_t)n * table_stride + g / (P / kKv8Group)];
  const size_t block = pg < (unsigned)num_blocks ? pg : 0u;
  const size_t tile = (block * KV + h) * (P / kKv8Group) + g % (P / kKv8Group);
  auto out_row = [&](int t) -> int {                            // row of token t of the group, or -1
    const int j = g * kKv8Group + t - pos0;
    return j >= 0 && j < nq ? row0 + j : -1;
  };
  // two bytes of w (at 2 H) as values of the result, in 32 bits: one rounding at the end
  auto emit = [&](T* dst, uint32_t w, float s) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    dst[0] = from_f32<T>(a[0] * s);
    dst[1] = from_f32<T>(a[1] * s);
    dst[2] = from_f32<T>(b[0] * s);
    dst[3] = from_f32<T>(b[1] * s);
  };
  if (threadIdx.x < D) {
    const int t = threadIdx.x / PK, p = threadIdx.x % PK;
    const kv8_u32x4 w = *(const kv8_u32x4*)(k_tiles + tile * (16 * D) + p * 256 + t * 16);
    const float s = kv8_scale(scales[tile * 32 + t]);
    const int row = out_row(t);
    if (row < 0) return;
    T o[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) emit(o + 4 * i, w[i], s);
    __builtin_memcpy(__builtin_assume_aligned(k_out + ((size_t)row * KV + h) * D + 16 * p, 16), o,
                     sizeof(o));
  } else {
    const int q = threadIdx.x - D;                              // piece of the V tile
    const int i = q / 64, r = q % 64 / 16, c = q % 16;
    const kv8_u32x4 w = *(const kv8_u32x4*)(v_tiles + tile * (16 * D) + q * 16);
#pragma unroll
    for (int j = 0; j < TP; ++j) {
      const int t = 4 * r + TP * i + j;
      const float s = kv8_scale(scales[tile * 32 + 16 + t]);
      const int row = out_row(t);
      if (row < 0) continue;
      T o[E];
#pragma unroll
      for (int x = 0; x < E / 4; ++x) emit(o + 4 * x, w[E / 4 * j + x], s);
      __builtin_memcpy(
          __builtin_assume_aligned(v_out + ((size_t)row * KV + h) * D + E * c, E * sizeof(T) < 16 ? E * sizeof(T) : 16),
          o, sizeof(o));
    }
  }
}

// Sum over the 16 lanes of a row; every lane receives it.
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

// cos and sin of pos * f, within two units of the last place of 32 bits: the product
// (exact in 64 bits) reduced to a quarter turn there (Cody and Waite), the rest in two
// floats. The angle as a float would be off by up to 2^-12 at 8192 tokens, and k, which
// is quantised from 32 bits, would fall on the other side of a border 2^-12 / 2^-4 as often.
__device__ __forceinline__ void angle(int64_t pos, float f, float& c, float& s) {
  const double a = (double)pos * (double)f;
  const double n = __builtin_rint(a * 0.63661977236758134308);           // 2 / pi
  const double r = __builtin_fma(n, -6.1232339957367660e-17,             // pi / 2 in two parts
                                 __builtin_fma(n, -1.5707963267948966, a));
  const float rh = (float)r, rl = (float)(r - (double)rh);
  const float c0 = cosf(rh), s0 = sinf(rh);
  const float cr = c0 - s0 * rl, sr = s0 + c0 * rl;
  const int q = (int)((int64_t)n & 3);
  c = q & 1 ? sr : cr;
  s = q & 1 ? cr : sr;
  if (q == 1 || q == 2) c = -c;
  if (q >= 2) s = -s;
}

// The qkv projection's output of a token (H q heads, KV k heads, KV v heads of D
// values: S fp32 planes that are added in order, or one plane of T) to
//   q: per-head RMSNorm and RoPE, rounded to T once, and
//   k (the same) and v, quantised into the cache from their 32-bit values.
// Nothing is rounded to T on the way, unlike in qkv_epilogue_kernel, which
// follows the roundings of a 16-bit cache's path: here k would be rounded twice.
// One workgroup per (token, part of its heads): 16 lanes per head, E dims each;
// a lane's rotation partner, D / 2 dims away, is 8 lanes away. The angles are
// the same for every head: the first D / 2 threads compute them into LDS while
// the first heads are on their way; after that a head is loaded while the one before
// it is worked on. 5164 tokens in bf16, 32 / 8 heads: 27 us, 4.3 TB/s (a large copy:
// 4.8); without the prefetch and with the angles once per 16 heads 32.8, with tokens
// dealt to the XCDs one by one 29.2. 8 tokens, three planes: 4.4 us, latency.
template <typename T, typename PT, int D>
__global__ __launch_bounds__(kNT) void qkv_epilogue_kv8_kernel(
    const PT* __restrict__ part, int nsplit, T* __restrict__ q_out, uint8_t* __restrict__ k_tiles,
    uint8_t* __restrict__ v_tiles, uint8_t* __restrict__ scales,
    const int64_t* __restrict__ pages, const int64_t* __restrict__ slots, int64_t batch, int H,
    int KV, int P, int64_t num_blocks, const T* __restrict__ q_w, const T* __restrict__ k_w,
    float eps, const int64_t* __restrict__ pos, const float* __restrict__ inv_freq, int units_per_wg) {
  constexpr int E = D / 16, HALF = D / 2, PER = kNT / 16;
  __shared__ __align__(16) float cs[HALF], sn[HALF];
  // Workgroups are dealt to the 8 XCDs round robin: 16 consecutive tokens, as a rule one
  // tile's, to one of them, so that its L2 completes the tile's lines before they are written
  // back (a token's pieces are 8 or 16 bytes of a line).
  const unsigned bx = blockIdx.x, run = bx & ~127u;
  const int64_t b = run + 128 <= gridDim.x ? run + (bx % 8) * 16 + bx % 128 / 8 : bx;
  const int c = threadIdx.x & 15;
  const size_t width = (size_t)(H + 2 * KV) * D, plane = (size_t)batch * width;
  // units: the H q heads, then the KV kv heads (k and v)
  const int u0 = blockIdx.y * units_per_wg, u1 = min(u0 + units_per_wg, H + KV);
  auto sum = [&](int head, float (&x)[E]) {
    const PT* src = part + (size_t)b * width + (size_t)head * D + E * c;
    load_row<PT, E>(src, x);
    for (int s = 1; s < nsplit; ++s) {
      float y[E];
      load_row<PT, E>(src + s * plane, y);
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] += y[i];
    }
  };
  auto fetch = [&](int un, float (&x)[E], float (&v)[E]) {
    const int u = min(un, u1 - 1);                 // (lanes without a unit repeat the last)
    sum(u, x);
    if (u >= H) sum(u + KV, v);
  };
  float x[E], v[E], xn[E], vn[E];
  int un = u0 + (int)(threadIdx.x >> 4);
  fetch(un, x, v);
  const uint64_t page = (uint64_t)pages[b], slot = (uint64_t)slots[b];
  float wq[E], wk[E];
  load_row<T, E>(q_w + E * c, wq);
  load_row<T, E>(k_w + E * c, wk);
  if (threadIdx.x < HALF) angle(pos[b], inv_freq[threadIdx.x], cs[threadIdx.x], sn[threadIdx.x]);
  __syncthreads();
  float co[E], si[E];                              // of this lane's dims: y = x cos +- partner sin
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int d = (E * c) % HALF + i;
    co[i] = cs[d];
    si[i] = c < 8 ? -sn[d] : sn[d];
  }
  auto norm_rope = [&](float (&y)[E], const float (&w)[E]) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) ss += y[i] * y[i];
    const float inv = 1.0f / sqrtf(row_sum(ss) / (float)D + eps);
#pragma unroll
    for (int i = 0; i < E; ++i) y[i] = y[i] * inv * w[i];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float z = __shfl_xor(y[i], 8);
      y[i] = y[i] * co[i] + z * si[i];
    }
  };
  for (int ub = u0; ub < u1; ub += PER) {
    if (ub + PER < u1) fetch(un + PER, xn, vn);
    const int u = min(un, u1 - 1);
    if (u < H) {
      norm_rope(x, wq);
      if (un < u1) {
        T o[E];
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = from_f32<T>(x[i]);
        __builtin_memcpy(__builtin_assume_aligned(q_out + ((size_t)b * H + u) * D + E * c,
                                                  E * sizeof(T)), o, sizeof(o));
      }
    } else {
      norm_rope(x, wk);
      const int kvh = u - H;
      // a (page, slot) outside the pool is dropped rather than written
      const bool on = un < u1 && page < (uint64_t)num_blocks && slot < (uint64_t)P;
      const size_t tile = (page * KV + kvh) * (P / kKv8Group) + slot / kKv8Group;
      kv8_store_row<D, std::is_same<T, _Float16>::value>(k_tiles, v_tiles, scales, on ? tile : 0,
                                                         (int)(slot % kKv8Group), on, c, x, v);
    }
    un += PER;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      x[i] = xn[i];
      v[i] = vn[i];
    }
  }
}

// Token rows from which a workgroup takes all heads of its token (the angles once):
// enough workgroups for every CU several times over.
constexpr int64_t kRowsPerWorkgroup = 1024;

int pool_shape(int64_t KV, int64_t D, int64_t P, int64_t num_blocks) {
  if (KV <= 0 || KV > 65535 || D <= 0 || P <= 0 || num_blocks <= 0 || num_blocks > 0x7fffffff)
    return ACORN_ERR_SHAPE;
  if ((P & (P - 1)) != 0 || P % kKv8Group != 0 || P > 65536) return ACORN_ERR_SHAPE;
  if (D != 64 && D != 128) return ACORN_ERR_UNSUPPORTED;
  return ACORN_OK;
}

template <typename T>
int scatter(const void* k, const void* v, void* kt, void* vt, void* sc, const int64_t* pages,
            const int64_t* slots, int64_t rows, int64_t KV, int64_t D, int64_t P, int64_t NB,
            int64_t k_rs, int64_t k_hs, int64_t v_rs, int64_t v_hs, hipStream_t st) {
  // rows are read D / 16 values at a time
  const uintptr_t align = std::min<uintptr_t>(16, (uintptr_t)(D / 16) * sizeof(T));
  const auto off = [&](const void* p, int64_t rs, int64_t hs) {
    return (uintptr_t)p % align || (uintptr_t)(rs * (int64_t)sizeof(T)) % align ||
           (uintptr_t)(hs * (int64_t)sizeof(T)) % align;
  };
  if (off(k, k_rs, k_hs) || off(v, v_rs, v_hs)) return ACORN_ERR_VALUE;
  const dim3 grid((unsigned)((rows + kNT / 16 - 1) / (kNT / 16)), (unsigned)KV);
  auto kfn = D == 128 ? kv8_scatter_kernel<T, 128> : kv8_scatter_kernel<T, 64>;
  kfn<<<grid, dim3(kNT), 0, st>>>((const T*)k, (const T*)v, (uint8_t*)kt, (uint8_t*)vt,
                                  (uint8_t*)sc, pages, slots, rows, (int)KV, (int)P, NB, k_rs,
                                  k_hs, v_rs, v_hs);
  ACORN_LAUNCH_CHECK();
  return ACORN_OK;
}

template <typename T>
int gather(const void* kt, const void* vt, const void* sc, const int32_t* tables,
           const int32_t* row0, const int32_t* pos0, const int32_t* nq, void* ko, void* vo,
           int64_t N, int64_t R, int64_t max_nq, int64_t KV, int64_t D, int64_t P, int64_t NB,
           int64_t ts, hipStream_t st) {
  // a run of max_nq tokens touches at most this many groups
  const dim3 grid((unsigned)((max_nq + 2 * kKv8Group - 2) / kKv8Group), (unsigned)KV, (unsigned)N);
  auto kfn = D == 128 ? kv8_gather_kernel<T, 128> : kv8_gather_kernel<T, 64>;
  kfn<<<grid, dim3((unsigned)(2 * D)), 0, st>>>(
      (const uint8_t*)kt, (const uint8_t*)vt, (const uint8_t*)sc, tables, row0, pos0, nq, (T*)ko,
      (T*)vo, (int)R, (int)max_nq, (int)KV, (int)P, (int)NB, (int)ts);
  ACORN_LAUNCH_CHECK();
  return ACORN_OK;
}

template <typename T, typename PT>
int epilogue(const void* part, int64_t nsplit, void* q_out, void* kt, void* vt, void* sc,
             const int64_t* pages, const int64_t* slots, int64_t batch, int64_t H, int64_t KV,
             int64_t D, int64_t P, int64_t NB, const void* qw, const void* kw, float eps,
             const int64_t* pos, const float* inv_freq, hipStream_t st) {
  const int64_t units = H + KV;
  const int64_t per = batch >= kRowsPerWorkgroup ? units : kNT / 16;
  const dim3 grid((unsigned)batch, (unsigned)((units + per - 1) / per));
  auto kfn = D == 128 ? qkv_epilogue_kv8_kernel<T, PT, 128> : qkv_epilogue_kv8_kernel<T, PT, 64>;
  kfn<<<grid, dim3(kNT), 0, st>>>((const PT*)part, (int)std::max<int64_t>(nsplit, 1), (T*)q_out,
                                  (uint8_t*)kt, (uint8_t*)vt, (uint8_t*)sc, pages, slots, batch,
                                  (int)H, (int)KV, (int)P, NB, (const T*)qw, (const T*)kw, eps,
                                  pos, inv_freq, (int)per);
  ACORN_LAUNCH_CHECK();
  return ACORN_OK;
}

bool tiles_ok(const void* kt, const void* vt, const void* sc) {
  return (uintptr_t)kt % 16 == 0 && (uintptr_t)vt % 16 == 0 && (uintptr_t)sc % 16 == 0;
}

}  // namespace

extern "C" int acorn_kv8_scatter(const void* k, const void* v, void* k_tiles, void* v_tiles,
                                 void* scales, const int64_t* pages, const int64_t* slots,
                                 int64_t rows, int64_t kv_heads, int64_t head_dim,
                                 int64_t page_size, int64_t num_blocks, int64_t k_row_stride,
                                 int64_t k_head_stride, int64_t v_row_stride,
                                 int64_t v_head_stride, int dtype, void* stream) {
  const int rc = pool_shape(kv_heads, head_dim, page_size, num_blocks);
  if (rc != ACORN_OK) return rc;
  if (rows < 0 || rows > 0x7fffffff) return ACORN_ERR_SHAPE;
  if (rows == 0) return ACORN_OK;
  if (!k || !v || !k_tiles || !v_tiles || !scales || !pages || !slots) return ACORN_ERR_VALUE;
  if (!tiles_ok(k_tiles, v_tiles, scales)) return ACORN_ERR_VALUE;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case ACORN_F32: return scatter<float>(k, v, k_tiles, v_tiles, scales, pages, slots, rows, kv_heads, head_dim, page_size, num_blocks, k_row_stride, k_head_stride, v_row_stride, v_head_stride, st);
    case ACORN_F16: return scatter<_Float16>(k, v, k_tiles, v_tiles, scales, pages, slots, rows, kv_heads, head_dim, page_size, num_blocks, k_row_stride, k_head_stride, v_row_stride, v_head_stride, st);
    case ACORN_BF16: return scatter<__bf16>(k, v, k_tiles, v_tiles, scales, pages, slots, rows, kv_heads, head_dim, page_size, num_blocks, k_row_stride, k_head_stride, v_row_stride, v_head_stride, st);
  }
  return ACORN_ERR_DTYPE;
}

extern "C" int acorn_kv8_gather(const void* k_tiles, const void* v_tiles, const void* scales,
                                const int32_t* tables, const int32_t* seq_row0,
                                const int32_t* seq_pos0, const int32_t* seq_nq, void* k_out,
                                void* v_out, int64_t N, int64_t R, int64_t max_nq,
                                int64_t kv_heads, int64_t head_dim, int64_t page_size,
                                int64_t num_blocks, int64_t table_stride, int dtype,
                                void* stream) {
  const int rc = pool_shape(kv_heads, head_dim, page_size, num_blocks);
  if (rc != ACORN_OK) return rc;
  if (N < 0 || N > 65535 || R < 0 || R > 0x7fffffff || max_nq < 0 || max_nq > 0x7fffffff - 32 ||
      table_stride < 1 || table_stride > 0x7fffffff / page_size)
    return ACORN_ERR_SHAPE;
  if (N == 0 || R == 0 || max_nq == 0) return ACORN_OK;
  if (!k_tiles || !v_tiles || !scales || !tables || !seq_row0 || !seq_pos0 || !seq_nq || !k_out ||
      !v_out)
    return ACORN_ERR_VALUE;
  if (!tiles_ok(k_tiles, v_tiles, scales) || (uintptr_t)k_out % 16 || (uintptr_t)v_out % 16)
    return ACORN_ERR_VALUE;
  max_nq = std::min(max_nq, R);                // a bound far above the rows there are costs nothing
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case ACORN_F32: return gather<float>(k_tiles, v_tiles, scales, tables, seq_row0, seq_pos0, seq_nq, k_out, v_out, N, R, max_nq, kv_heads, head_dim, page_size, num_blocks, table_stride, st);
    case ACORN_F16: return gather<_Float16>(k_tiles, v_tiles, scales, tables, seq_row0, seq_pos0, seq_nq, k_out, v_out, N, R, max_nq, kv_heads, head_dim, page_size, num_blocks, table_stride, st);
    case ACORN_BF16: return gather<__bf16>(k_tiles, v_tiles, scales, tables, seq_row0, seq_pos0, seq_nq, k_out, v_out, N, R, max_nq, kv_heads, head_dim, page_size, num_blocks, table_stride, st);
  }
  return ACORN_ERR_DTYPE;
}

extern "C" int acorn_qkv_epilogue_kv8(const void* part, int64_t nsplit, void* q_out,
                                      void* k_tiles, void* v_tiles, void* scales,
                                      const int64_t* pages, const int64_t* slots, int64_t batch,
                                      int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                      int64_t page_size, int64_t num_blocks, const void* q_w,
                                      const void* k_w, float eps, const int64_t* positions,
                                      const float* inv_freq, int dtype, void* stream) {
  const int rc = pool_shape(kv_heads, head_dim, page_size, num_blocks);
  if (rc != ACORN_OK) return rc;
  if (batch < 0 || batch > 0x7fffffff || q_heads <= 0 || q_heads > 65535 || nsplit < 0 ||
      nsplit > 0x7fffffff)
    return ACORN_ERR_SHAPE;
  if (batch == 0) return ACORN_OK;
  if (!part || !q_out || !k_tiles || !v_tiles || !scales || !pages || !slots || !q_w || !k_w ||
      !positions || !inv_freq)
    return ACORN_ERR_VALUE;
  if (!tiles_ok(k_tiles, v_tiles, scales) || (uintptr_t)part % 16 || (uintptr_t)q_out % 16 ||
      (uintptr_t)q_w % 16 || (uintptr_t)k_w % 16)
    return ACORN_ERR_VALUE;
  hipStream_t st = (hipStream_t)stream;
#define ACORN_EPI_ARGS                                                                          \
  part, nsplit, q_out, k_tiles, v_tiles, scales, pages, slots, batch, q_heads, kv_heads, head_dim, \
      page_size, num_blocks, q_w, k_w, eps, positions, inv_freq, st
  switch (dtype) {
    case ACORN_F16: return nsplit ? epilogue<_Float16, float>(ACORN_EPI_ARGS) : epilogue<_Float16, _Float16>(ACORN_EPI_ARGS);
    case ACORN_BF16: return nsplit ? epilogue<__bf16, float>(ACORN_EPI_ARGS) : epilogue<__bf16, __bf16>(ACORN_EPI_ARGS);
  }
#undef ACORN_EPI_ARGS
  return ACORN_ERR_DTYPE;
}
