// q4_cells.cuh — layout of the paged 4-bit cache.
//
// One page of one KV head holds 64 tokens: [key codes][key headers][value codes][value headers], one contiguous
// block of page_bytes() that a single bulk copy fetches. The codes lie in the order in which the lanes of an
// m16n8k16 product (lane = 4 * g + t) hold its first operand, so that a lane gets its share of the operand
// with one 16-byte (head_dim 128) or 8-byte (64) shared-memory load and unpacks it with masks alone:
//
//   keys: a token's D / 2 bytes are 4 pieces, one per t; piece t holds, per group of 64 dimensions, the 16
//     dimensions gr * 64 + t * 16 .. + 15 in two words, nibble n of word w = dimension t * 16 + 8 w + n.
//     Masks 0x000f000f and 0x00f000f0 (of the word and of the word >> 8) give the pairs (n, n + 4).
//   values: two tokens (2p, 2p + 1) share D bytes in 8 pieces, one per g, of the D / 8 dimensions g * D / 8 ..;
//     word i of a piece holds 4 dimensions, the even token in its low half, the odd one in its high half, so
//     the same masks give (even token, odd token) pairs, which is how the second product contracts over tokens.
//     The piece's place is rotated by the pair, (g + 2 p) % 8 for D = 128, and (g + 4 (p / 2 % 2)) % 8 for 64:
//     lanes t = 0..3 read four pairs at once, a multiple of 64 bytes apart, and would share banks otherwise.
//   headers: float16 (scale, low) per key token and group; (scale even, scale odd, low even, low odd) per value
//     pair and group.
#pragma once
#include <cstdint>

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
  static constexpr int kKeyHeads = kPage * D / 2;
  static constexpr int kValueCodes = kKeyHeads + kPage * kGroups * 4;
  static constexpr int kValueHeads = kValueCodes + kPage * D / 2;
  static constexpr int kBytes = kValueHeads + kPage * kGroups * 4;

  // Byte of the 8 key codes of dimensions 8 * j .. + 7 (one word, nibble n = dimension 8 j + n) of token r.
  static __device__ __forceinline__ int key_word(int r, int j) {
    const int gr = j >> 3, t = (j & 7) >> 1, w = j & 1;
    return kKeyCodes + r * (D / 2) + t * (D / 8) + gr * 8 + w * 4;
  }
  static __device__ __forceinline__ int key_head(int r, int gr) { return kKeyHeads + (r * kGroups + gr) * 4; }

  static __device__ __forceinline__ int value_piece(int pair, int g) {
    const int at = D == 128 ? (g + 2 * pair) & 7 : (g + 4 * ((pair >> 1) & 1)) & 7;
    return kValueCodes + pair * D + at * (D / 8);
  }
  // Byte of the word that holds dimensions 4 * j .. + 3 of the two tokens of `pair`.
  static __device__ __forceinline__ int value_word(int pair, int j) {
    return value_piece(pair, j / (D / 32)) + (j % (D / 32)) * 4;
  }
  static __device__ __forceinline__ int value_head(int pair, int gr) {
    return kValueHeads + (pair * kGroups + gr) * 8;
  }
};

}  // namespace q4
}  // namespace dkv
