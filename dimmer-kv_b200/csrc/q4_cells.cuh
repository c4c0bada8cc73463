// q4_cells.cuh — layout of the paged 4-bit cache.
//
// One page of one KV head holds 64 tokens: [key codes][value codes][headers], one contiguous block of kBytes that a
// single bulk copy fetches. The codes lie in the order in which the lanes of an m16n8k16 product (lane = 4 * g + t)
// hold its first operand, so that a lane gets its share of the operand with one 16-byte (head_dim 128) or 8-byte
// (64) shared-memory load and unpacks it with masks alone:
//
//   keys: a token's D / 2 bytes are 4 pieces, one per t; piece t holds, per group of 64 dimensions, the 16
//     dimensions gr * 64 + t * 16 .. + 15 in two words, nibble n of word w = dimension t * 16 + 8 w + n.
//     Masks 0x000f000f and 0x00f000f0 (of the word and of the word >> 8) give the pairs (n, n + 4).
//   values: two tokens (2p, 2p + 1) share D bytes in 8 pieces, one per g; piece g holds, per group, the 8 dimensions
//     gr * 64 + g * 8 .. in two words of 4 dimensions, the even token in a word's low half, the odd one in its high
//     half, so the same masks give (even token, odd token) pairs, which is how the second product contracts over
//     tokens. The piece's place is rotated by the pair, (g + 2 p) % 8 for D = 128, and (g + 4 (p / 2 % 2)) % 8 for
//     64: lanes t = 0..3 read four pairs at once, a multiple of 64 bytes apart, and would share banks otherwise.
//   headers: float16 (scale, low) of a token's key groups, then of its value groups: one load per token.
//
// Quantising: eight lanes hold a group of 64 dimensions, eight each; minimum and maximum are three shuffles, a
// lane's eight key codes are exactly one word of the key cell, its value codes the halves of two words of the pair's.
// The code is the nearest whole number to the true quotient (x - low) / scale, not to its float32 rounding: the
// float32 quotient, off by less than 2^-18, decides unless it lies within 2^-16 of a half; then the border
// low + (c + 1/2) * scale, which float64 holds exactly (two float16 numbers, exponents -25 .. 15, and 5 bits),
// is compared with x. So the codes do not depend on how a device rounds a division.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/dimmer_kv.h"

namespace dkv {
namespace q4 {

constexpr int kPage = DKV_PAGE_TOKENS;
constexpr int kGroup = 64;
constexpr float kCellMax = 32768.f;  // largest magnitude a cell holds: low + 15 * scale stays finite in float16

template <int D>
struct Cells {
  static_assert(D == 64 || D == 128, "head_dim");
  static constexpr int kGroups = D / kGroup;
  static constexpr int kKeyCodes = 0;
  static constexpr int kValueCodes = kPage * D / 2;
  static constexpr int kHeads = 2 * kValueCodes;
  static constexpr int kHeadBytes = kGroups * 8;  // of a token
  static constexpr int kBytes = kHeads + kPage * kHeadBytes;

  // Byte of the 8 key codes of dimensions 8 * j .. + 7 (one word, nibble n = dimension 8 j + n) of token r.
  static __device__ __forceinline__ int key_word(int r, int j) {
    const int gr = j >> 3, t = (j & 7) >> 1, w = j & 1;
    return kKeyCodes + r * (D / 2) + t * (D / 8) + gr * 8 + w * 4;
  }
  static __device__ __forceinline__ int value_piece(int pair, int g) {
    const int at = D == 128 ? (g + 2 * pair) & 7 : (g + 4 * ((pair >> 1) & 1)) & 7;
    return kValueCodes + pair * D + at * (D / 8);
  }
  // Byte of the two words that hold dimensions 8 * j .. + 7 of the two tokens of `pair`.
  static __device__ __forceinline__ int value_words(int pair, int j) {
    return value_piece(pair, j & 7) + (j >> 3) * 8;
  }
  static __device__ __forceinline__ int key_head(int r, int gr) { return kHeads + r * kHeadBytes + gr * 4; }
  static __device__ __forceinline__ int value_head(int r, int gr) { return key_head(r, kGroups + gr); }
};

template <bool F16>
__device__ __forceinline__ float from16(uint16_t v) {
  return F16 ? __half2float(__ushort_as_half(v)) : __bfloat162float(__ushort_as_bfloat16(v));
}
template <bool F16>
__device__ __forceinline__ uint16_t to16(float v) {
  return F16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// Nearest whole number of 0..15 to (x - low) / scale, ties to even; inv = 1 / scale to float32 accuracy.
__device__ __forceinline__ uint32_t code_of(float x, float low, float scale, float inv) {
  const float q = __fmul_rn(__fsub_rn(x, low), inv);
  float c = rintf(q);
  const float below = floorf(q);
  if (fabsf(q - below - 0.5f) < 0x1p-16f && q > -1.f && q < 16.f) {
    const double border = static_cast<double>(low) + (static_cast<double>(below) + 0.5) * static_cast<double>(scale);
    const double xd = static_cast<double>(x);
    const bool up = xd > border || (xd == border && (static_cast<int>(below) & 1));
    c = up ? below + 1.f : below;
  }
  return static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f));
}

struct Cell8 {
  uint32_t codes;  // nibble e: element e of the lane's eight
  uint16_t scale, low;
  bool fits;       // the lane's elements are finite and within kCellMax
};

// The lane's eight elements of a group that this lane and the 7 beside it hold (all of a warp's lanes call it).
template <bool F16>
__device__ __forceinline__ Cell8 quantise8(const uint4& raw) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = from16<F16>(static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1))));
  float lo = x[0], hi = x[0];
  Cell8 c;
  c.fits = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
    c.fits = c.fits && fabsf(x[e]) <= kCellMax;  // false for a NaN
  }
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
  }
  const __half low_h = __float2half_rn(lo);
  const float low = __half2float(low_h);
  const __half scale_h = __float2half_rn(__fdiv_rn(__fsub_rn(hi, low), 15.f));
  const float scale = __half2float(scale_h);
  const float inv = scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f;
  c.codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) c.codes |= code_of(x[e], low, scale, inv) << (4 * e);
  if (!(scale > 0.f)) c.codes = 0;
  c.scale = __half_as_ushort(scale_h);
  c.low = __half_as_ushort(low_h);
  return c;
}

// The j-th eight dimensions of token r of a page, written into it (in shared or in global memory).
template <int D>
__device__ __forceinline__ void store_key8(uint8_t* page, int r, int j, const Cell8& c) {
  *reinterpret_cast<uint32_t*>(page + Cells<D>::key_word(r, j)) = c.codes;
  if (j % 8 == 0)
    *reinterpret_cast<uint32_t*>(page + Cells<D>::key_head(r, j / 8)) =
        static_cast<uint32_t>(c.scale) | static_cast<uint32_t>(c.low) << 16;
}
template <int D>
__device__ __forceinline__ void store_value8(uint8_t* page, int r, int j, const Cell8& c) {
  uint8_t* w = page + Cells<D>::value_words(r >> 1, j) + 2 * (r & 1);
  *reinterpret_cast<uint16_t*>(w) = static_cast<uint16_t>(c.codes);
  *reinterpret_cast<uint16_t*>(w + 4) = static_cast<uint16_t>(c.codes >> 16);
  if (j % 8 == 0)
    *reinterpret_cast<uint32_t*>(page + Cells<D>::value_head(r, j / 8)) =
        static_cast<uint32_t>(c.scale) | static_cast<uint32_t>(c.low) << 16;
}

}  // namespace q4
}  // namespace dkv
