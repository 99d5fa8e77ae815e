// The 8-bit paged KV cache: its layout and number format, shared by the kernels
// that write and read it (kv8_cache.hip) and attend over it (kv8_attention.hip).
//
// Format. A row x (the D values of one token and kv head, of k or of v) is held
// as D bytes and one scale code. With amax = max |x_d| and e the least integer,
// -126 at least, for which amax <= 448 * 2^e:
//   code = e + 127,  byte_d = e4m3(x_d * 2^-e) (nearest, ties to even),
// and a byte stands for e4m3 * 2^(code - 127). The scale is a power of two, so
// the division is exact and a row's bytes do not depend on who computes them;
// e4m3 being a float format, a finer scale would gain nothing but part of a
// bit of range (2^15 of normal numbers below amax), and a scale per row can be
// applied by the conversions, whose scale operand is a power of two. A code of
// 0 (memory never written) stands for 0 together with bytes of 0.
// A (token, head) whose k or v holds an infinity or NaN is held as NaN: both
// codes 255, bytes 0. So the bytes of v are finite whatever was written, a
// probability of 0 removes a row that a query must not see, and a query that
// sees such a row gets NaN through its score.
// What is held stays finite when it is read: the largest number is 240 * 2^120
// (the next of the grid, 2^128, is neither an fp32 nor a bf16), of fp16 rows
// 240 * 2^8 = 61440 (65536 is not an fp16); greater magnitudes are held as it.
//
// Layout. A block holds P tokens (a multiple of 16) in groups of 16; per (block,
// kv head, group) one K tile and one V tile of 16 D bytes, and 32 bytes of
// codes: 16 of k, 16 of v. Tiles are 16-byte pieces in the order the lanes of a
// wave take them for v_mfma_f32_16x16x32, lane = 16 r + c, so that every load
// is one line after another with no lane exchange for K:
//   K: piece (d / 16) * 16 + t: 16 dims of token t. Lane (r, c) takes pieces
//      16 r + c and, for D = 128, 64 + 16 r + c: 8 dims each of the A operands
//      (row = token c).
//   V: with E = D / 16 dims and TP = 16 / E tokens to a piece, piece
//      (t % 4 / TP) * 64 + (t / 4) * 16 + d / E: tokens TP to a piece, E dims
//      each. Lane (r, c) takes dims E c .. of tokens 4 r .. 4 r + 3: the rows
//      that a 16x16 transpose in registers turns into V^T operands. Two
//      dimensions of one token stay side by side, so that a conversion of two
//      bytes has one scale.
#pragma once
#include "common.h"

namespace acorn {

typedef uint32_t kv8_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t kv8_u32x2 __attribute__((ext_vector_type(2)));

constexpr int kKv8Group = 16;                      // tokens of a tile
constexpr float kKv8Max = 240.f * 0x1p120f, kKv8MaxF16 = 240.f * 0x1p8f;    // the largest numbers

// Byte of (token t of the group, dim d) in a K tile and in a V tile.
template <int D>
__device__ __forceinline__ int kv8_k_byte(int t, int d) {
  return (d >> 4) * 256 + t * 16 + (d & 15);
}
template <int D>
__device__ __forceinline__ int kv8_v_byte(int t, int d) {
  constexpr int E = D / 16, TP = 16 / E;
  return (t % 4 / TP) * 1024 + (16 * (t / 4) + d / E) * 16 + t % TP * E + d % E;
}

// 2^(code - 127); 0 for code 0, an infinity for 255.
__device__ __forceinline__ float kv8_scale(uint32_t code) { return __uint_as_float(code << 23); }
// The scale code at byte i of four.
template <int I>
__device__ __forceinline__ float kv8_scale_of(uint32_t codes) {
  return __uint_as_float((I < 3 ? codes << (23 - 8 * I) : codes >> 1) & 0x7F800000u);
}
// ... for rows that a query may have to leave out (255: 2^127; the bytes are 0).
__device__ __forceinline__ float kv8_scale_finite(uint32_t code) {
  return __uint_as_float(min(code, 254u) << 23);
}

// Bytes 2 H and 2 H + 1 of w as two values of T, times the scale (of which the
// exponent is used).
template <typename T, bool H>
__device__ __forceinline__ uint32_t kv8_cvt2(uint32_t w, float scale);
template <>
__device__ __forceinline__ uint32_t kv8_cvt2<__bf16, false>(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}
template <>
__device__ __forceinline__ uint32_t kv8_cvt2<__bf16, true>(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true));
}
template <>
__device__ __forceinline__ uint32_t kv8_cvt2<_Float16, false>(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
}
template <>
__device__ __forceinline__ uint32_t kv8_cvt2<_Float16, true>(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true));
}
// Eight bytes as eight values of T.
template <typename T>
__device__ __forceinline__ kv8_u32x4 kv8_cvt8(uint32_t lo, uint32_t hi, float scale) {
  return kv8_u32x4{kv8_cvt2<T, false>(lo, scale), kv8_cvt2<T, true>(lo, scale),
                   kv8_cvt2<T, false>(hi, scale), kv8_cvt2<T, true>(hi, scale)};
}

// The largest over the 16 lanes of a row (DPP rotations within the row).
__device__ __forceinline__ uint32_t kv8_row_max(uint32_t v) {
  auto ror = [](uint32_t x, auto n) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + decltype(n)::value, 0xF, 0xF,
                                                 false);
  };
  v = max(v, ror(v, std::integral_constant<int, 8>{}));
  v = max(v, ror(v, std::integral_constant<int, 4>{}));
  v = max(v, ror(v, std::integral_constant<int, 2>{}));
  v = max(v, ror(v, std::integral_constant<int, 1>{}));
  return v;
}

// Writes one (token, kv head) of the cache: the 16 lanes of a row hold E = D / 16
// dims each of k and of v, dims E c .. . `tile` is the tile's number, t the
// token in it; `on` false writes nothing (every lane takes part in the row's
// maxima all the same). SAT: an fp16 cache.
template <int D, bool SAT>
__device__ __forceinline__ void kv8_store_row(uint8_t* k_tiles, uint8_t* v_tiles, uint8_t* scales,
                                              size_t tile, int t, bool on, int c,
                                              const float (&k)[D / 16], const float (&v)[D / 16]) {
  constexpr int E = D / 16;
  const float* x[2] = {k, v};
  uint32_t top[2] = {0, 0};                        // |x| as bits: ordered like the numbers
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int i = 0; i < E; ++i) top[a] = max(top[a], __float_as_uint(x[a][i]) & 0x7FFFFFFFu);
  top[0] = kv8_row_max(top[0]);
  top[1] = kv8_row_max(top[1]);
  const bool nan = max(top[0], top[1]) >= 0x7F800000u;
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    // (a constant: with the limit in registers the qkv epilogue passes 96 of them, which
    // takes a fifth of its waves and costs 5164 tokens 5 us)
    constexpr float kMax = SAT ? kKv8MaxF16 : kKv8Max;
    const uint32_t m = min(top[a], __float_as_uint(kMax));
    // 448 = 1.75 * 2^8
    uint32_t code = (uint32_t)max((int)(m >> 23) - 8 + ((m & 0x7FFFFFu) > 0x600000u ? 1 : 0), 1);
    const float inv = __uint_as_float((254u - code) << 23);      // 2^-e, e + 127 = code <= 247
    uint32_t w[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = __builtin_amdgcn_fmed3f(x[a][4 * i + j], -kMax, kMax) * inv;
      int b = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      b = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], b, true);
      w[i] = nan ? 0u : (uint32_t)b;
    }
    if (nan) code = 255u;
    if (on) {
      const int off = a == 0 ? kv8_k_byte<D>(t, E * c) : kv8_v_byte<D>(t, E * c);
      uint8_t* dst = (a == 0 ? k_tiles : v_tiles) + tile * (16 * D) + off;
      __builtin_memcpy(__builtin_assume_aligned(dst, E), w, E);
      if (c == 0) scales[tile * 32 + 16 * a + t] = (uint8_t)code;
    }
  }
}

}  // namespace acorn
