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
// Quantising: 8 / H lanes hold a group of 64 dimensions, 8 H each (H 16-byte loads); minimum and maximum are a shuffle
// or two, eight key codes are exactly one word of the key cell, eight value codes the halves of two words of the pair's.
// The code is the nearest whole number to the true quotient (x - low) / scale, ties to even, not to a float32
// rounding of it: the float32 quotient, by the hardware's reciprocal off by less than 2^-18, decides unless it lies
// within 2^-16 of a half; then the border low + (c + 1/2) * scale, which float64 holds exactly (two float16 numbers,
// exponents -25 .. 15, and 5 bits), is compared with x. So the codes do not depend on how a device divides.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/dimmer_kv.h"
#include "dkv_ptx.cuh"
#include "dkv_serving.h"

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

// Codes of a lane whose quotients go beyond 0 .. 15 or come close to a border between two codes: rare.
template <bool F16>
static __device__ __noinline__ uint32_t codes_with_care(uint4 raw, float low, float scale, float part) {
  uint32_t codes = 0;
#pragma unroll 1
  for (int e = 0; e < 8; ++e) {
    const uint32_t pair = (e >> 1) == 0 ? raw.x : (e >> 1) == 1 ? raw.y : (e >> 1) == 2 ? raw.z : raw.w;
    const float x = from16<F16>(static_cast<uint16_t>(pair >> (16 * (e & 1))));
    const float q = fminf(fmaxf(__fmul_rn(__fsub_rn(x, low), part), 0.f), 15.f);
    const float below = floorf(q);
    uint32_t code = static_cast<uint32_t>(rintf(q));
    if (fabsf(q - below - 0.5f) < 0x1p-15f) {
      const double border = static_cast<double>(low) + (static_cast<double>(below) + 0.5) * static_cast<double>(scale);
      const double xd = static_cast<double>(x);
      const bool up = xd > border || (xd == border && (static_cast<int>(below) & 1));
      code = static_cast<uint32_t>(up ? below + 1.f : below);
    }
    codes |= code << (4 * e);
  }
  return codes;
}

template <int H>
struct CellPart {
  uint32_t codes[H];  // of the lane's eights of elements, nibble e: element e
  uint16_t scale, low;
  bool fits;          // the group is finite and within kCellMax
};

template <bool F16, bool MAX>
__device__ __forceinline__ uint32_t extreme2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (F16) {
    if constexpr (MAX) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  } else {
    if constexpr (MAX) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  }
  return r;
}

// The lane's 8 H elements of a group that this lane and those beside it hold (all of a warp's lanes call it).
template <bool F16, int H>
__device__ __forceinline__ CellPart<H> quantise(const uint4 (&raw)[H]) {
  uint32_t w[4 * H];
#pragma unroll
  for (int h = 0; h < H; ++h) w[4 * h] = raw[h].x, w[4 * h + 1] = raw[h].y, w[4 * h + 2] = raw[h].z, w[4 * h + 3] = raw[h].w;
  uint32_t least = w[0], most = w[0];
#pragma unroll
  for (int e = 1; e < 4 * H; ++e) {
    least = extreme2<F16, false>(least, w[e]);
    most = extreme2<F16, true>(most, w[e]);
  }
#pragma unroll
  for (int d = 1; d < 8 / H; d <<= 1) {
    least = extreme2<F16, false>(least, __shfl_xor_sync(0xffffffffu, least, d));
    most = extreme2<F16, true>(most, __shfl_xor_sync(0xffffffffu, most, d));
  }
  least = extreme2<F16, false>(least, least >> 16);
  most = extreme2<F16, true>(most, most >> 16);
  const float lo = from16<F16>(static_cast<uint16_t>(least)), hi = from16<F16>(static_cast<uint16_t>(most));
  CellPart<H> c;
  c.fits = lo >= -kCellMax && hi <= kCellMax;  // false for a NaN
  const __half low_h = __float2half_rn(lo);
  const float low = __half2float(low_h);
  // low's rounding may lie above every element (a bfloat16 group of next to nothing): +0 then, never a scale with a sign
  const __half scale_h = __float2half_rn(__fdiv_rn(fmaxf(__fsub_rn(hi, low), 0.f), 15.f));
  const float scale = __half2float(scale_h);
  float part;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(part) : "f"(scale));
  part = scale > 0.f ? part : 0.f;
  constexpr float kWhole = 12582912.f;  // 1.5 * 2^23: what is added to it becomes a whole number
  const uint64_t low2 = f32x2_pack(__float_as_uint(-low), __float_as_uint(-low));
  const uint64_t part2 = f32x2_pack(__float_as_uint(part), __float_as_uint(part));
  const uint64_t whole2 = f32x2_pack(__float_as_uint(kWhole), __float_as_uint(kWhole));
  const uint64_t minus2 = f32x2_pack(0xbf800000u, 0xbf800000u);
  const bool inside = (lo - low) * part > -0.49f && (hi - low) * part < 15.49f;  // false where low's rounding is coarse
#pragma unroll
  for (int h = 0; h < H; ++h) {
    uint32_t codes = 0;
    float off = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t u = w[4 * h + e];
      const float x0 = from16<F16>(static_cast<uint16_t>(u)), x1 = from16<F16>(static_cast<uint16_t>(u >> 16));
      const uint64_t d = add_f32x2(f32x2_pack(__float_as_uint(x0), __float_as_uint(x1)), low2);
      const uint64_t m = fma_f32x2(d, part2, whole2);
      const uint64_t r = fma_f32x2(d, part2, fma_f32x2(m, minus2, whole2));  // quotient - code
      off = fmaxf(off, fmaxf(fabsf(__uint_as_float(static_cast<uint32_t>(r))), fabsf(__uint_as_float(static_cast<uint32_t>(r >> 32)))));
      codes += (static_cast<uint32_t>(m) << (8 * e)) + (static_cast<uint32_t>(m >> 32) << (8 * e + 4));
    }
    c.codes[h] = codes - 0x4b400000u * 0x11111111u;  // the constant's own bits under the codes
    if (!inside || off > 0.5f - 0x1p-16f) c.codes[h] = codes_with_care<F16>(raw[h], low, scale, part);
  }
  c.scale = __half_as_ushort(scale_h);
  c.low = __half_as_ushort(low_h);
  return c;
}

// The j-th 8 H dimensions of token r of a page, written into it (in shared or in global memory).
template <int D, int H>
__device__ __forceinline__ void store_key(uint8_t* page, int r, int j, const CellPart<H>& c) {
#pragma unroll
  for (int h = 0; h < H; h += 2)
    *reinterpret_cast<uint2*>(page + Cells<D>::key_word(r, H * j + h)) = make_uint2(c.codes[h], c.codes[h + 1]);
  if (j % (8 / H) == 0)
    *reinterpret_cast<uint32_t*>(page + Cells<D>::key_head(r, j / (8 / H))) =
        static_cast<uint32_t>(c.scale) | static_cast<uint32_t>(c.low) << 16;
}
template <int D, int H>
__device__ __forceinline__ void store_value_head(uint8_t* page, int r, int j, const CellPart<H>& c) {
  if (j % (8 / H) == 0)
    *reinterpret_cast<uint32_t*>(page + Cells<D>::value_head(r, j / (8 / H))) =
        static_cast<uint32_t>(c.scale) | static_cast<uint32_t>(c.low) << 16;
}
template <int D, int H>
__device__ __forceinline__ void store_value(uint8_t* page, int r, int j, const CellPart<H>& c) {
#pragma unroll
  for (int h = 0; h < H; ++h) {
    uint8_t* w = page + Cells<D>::value_words(r >> 1, H * j + h) + 2 * (r & 1);
    *reinterpret_cast<uint16_t*>(w) = static_cast<uint16_t>(c.codes[h]);
    *reinterpret_cast<uint16_t*>(w + 4) = static_cast<uint16_t>(c.codes[h] >> 16);
  }
  store_value_head<D>(page, r, j, c);
}

}  // namespace q4
}  // namespace dkv
