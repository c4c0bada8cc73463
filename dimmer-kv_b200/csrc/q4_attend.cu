// q4_attend.cu — causal attention of new tokens' queries over the paged 4-bit cache (dkv_q4_attend), and the new
// tokens' cells with it.
//
// With k_d = low_g + scale_g * c_d (g = d / 64, the token's own scales and lows), a score splits into
//   q . k = sum_g scale_g * (sum_{d in g} q_d c_d) + sum_g low_g * (sum_{d in g} q_d),
// and a weighted value likewise into
//   sum_j p_j v_jd = sum_j (p_j scale_jg) c_jd + sum_j p_j low_jg:
// both products run over the codes themselves, which float16 holds exactly, the low terms in float32. The query enters
// as float16 times a power of two of its row (exact but for what is below 2^-38 of the row's largest), so a score is
// good to float32. p * scale enters as float16 of 2^7 * exp(score - m) * scale / 2^k, with m within 2^8 of the running
// maximum and 2^k one to four times the largest scale of the head so far, of either group: one rounding of 2^-11 at
// most where p * scale is above 2^-19 of the largest, so that sums over a long context of small probabilities do not
// vanish; below that float16 has fewer bits, and a term is off by up to 2^-26 of that largest scale (a step's half,
// 2^-25, times a code of 15). So a group whose scales are a 2^12th of its neighbour's, or of an earlier token's, keeps
// its bits for probabilities down to 2^-7, and no fewer than 7 of them down to 2^-11. For float16 outputs, whose own step
// is as small as the rounding, the factor enters as two float16 numbers (the rounded one and what it lacks). Four
// conversations of 4K to 16K tokens: bfloat16 outputs are off by 1.75e-3 of their size, 1.68e-3 in float32 arithmetic
// and rounded once, float16 ones by 2.1e-4, as there.
//
// q4_decode_kernel: few query rows per KV head (one token, or a short draft). Bound by the cells' bytes, and close to it
// by unpacking them (the integer pipe runs at half rate). The pages of all (conversation, KV head, row chunk) units
// form one line, cut into equal pieces, one per WARP, so that any mix of lengths, heads and conversations fills the
// GPU evenly; a unit that several warps share leaves partial (m, l, O) in the workspace, which the join
// kernels put together. A page of one KV head is one contiguous block: each warp keeps a ring of bulk copies of its own and meets no
// other warp. It contracts tokens as the 16 rows of m16n8k16 and query rows as its 8 columns (3 or 4 heads that share a
// KV head are the rule), S^T = C Q^T, then O^T = C^T P^T; P^T in the layout of the second product is one 8 x 8
// transpose per 8 tokens (movmatrix). A code pair of a word is a float16 pair after ONE mask: the 4 bits are a
// subnormal c * 2^-24 (or 16 times that from the odd nibbles, against q / 16 in the first product, and divided out at
// the end in the second). The warp that owns a new token's page quantises the token itself, into the page's copy and
// into the cache.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "q4_attend.cuh"

namespace dkv {
namespace {

using namespace q4;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// x += u, y += w, as one packed addition.
__device__ __forceinline__ void add2(float& x, float& y, float u, float w) {
  const uint64_t r = add_f32x2(f32x2_pack(__float_as_uint(x), __float_as_uint(y)),
                               f32x2_pack(__float_as_uint(u), __float_as_uint(w)));
  x = __uint_as_float(static_cast<uint32_t>(r));
  y = __uint_as_float(static_cast<uint32_t>(r >> 32));
}

// Transpose of an 8 x 8 matrix of 16-bit elements held one pair per lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ int warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }

// How a warp holds its query rows: NT tiles of 8 columns, two columns per lane; or, NT = 0, up to 4 rows, each on the
// even column of a pair, so that a lane has one row to do the softmax of and the odd column takes what the rounding of
// the row's probabilities lacks.
template <int D, int NT>
struct Decode {
  using C = Cells<D>;
  static constexpr bool kPair = NT == 0;
  static constexpr int kTilesN = kPair ? 1 : NT;
  static constexpr int kCols = kPair ? 1 : 2;    // of a lane, per tile
  static constexpr int kRows = kPair ? 4 : 8 * NT;
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kTiles = NT <= 1 ? 2 : 1;  // of 16 tokens at a time, for the latencies to overlap
  // Two or three tiles need the registers of two CTAs per SM: with three, spilled, 16 rows of heads of 64 over 9 contexts of
  // 0 to 8K take 29.5 us against 27.6, 20 rows 42 against 33.
  static constexpr int kBlocksPerSm = NT >= 2 ? 2 : 3;
  static constexpr int kWarpBytes = kStages * C::kBytes;
  static constexpr int kBars = kWarps * kWarpBytes;
  static constexpr int kBytes = kBars + kWarps * kStages * 8;
  // The row of column c of tile nt that lane t = 0..3 has.
  static __device__ __forceinline__ int row(int nt, int t, int c) { return kPair ? t : nt * 8 + 2 * t + c; }
};

// A unit's query rows as the second operand, and the factors of their scores.
template <int D, int NT>
struct Query {
  using S = Decode<D, NT>;
  static constexpr int kGroups = Cells<D>::kGroups;
  uint32_t frag[D / 16][S::kTilesN][2];
  float factor[S::kTilesN][S::kCols], sum[S::kTilesN][S::kCols][kGroups];
  int limit[S::kTilesN][S::kCols];  // tokens below it are seen (0: no row)
};
// The rows as they lie in memory: a lane has 16 dimensions of each group of the row of column g.
template <int D, int NT>
struct RawQuery {
  uint4 v[Decode<D, NT>::kTilesN][Cells<D>::kGroups][2];
};

template <int D, int NT>
__device__ __forceinline__ void fetch_query(const dkv_q4_attend_args& a, int seq, int head, int row0, int share, int fresh,
                                            RawQuery<D, NT>& raw) {
  using S = Decode<D, NT>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < S::kTilesN; ++nt) {
    const int r = row0 + (S::kPair ? g >> 1 : nt * 8 + g), i = r / share;
    const bool real = r < a.q_len * share && i < fresh && !(S::kPair && (g & 1));
    const uint16_t* src = static_cast<const uint16_t*>(a.query) + seq * a.q_stride[0] +
                          (head * share + r - i * share) * a.q_stride[1] + i * a.q_stride[2] + t * 16;
#pragma unroll
    for (int gr = 0; gr < Cells<D>::kGroups; ++gr)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        raw.v[nt][gr][h] = real ? *reinterpret_cast<const uint4*>(src + gr * 64 + h * 8) : make_uint4(0u, 0u, 0u, 0u);
  }
}

template <int D, int NT, bool F16>
__device__ __forceinline__ void make_query(const dkv_q4_attend_args& a, int row0, int share, int start, int fresh,
                                           const RawQuery<D, NT>& raw, Query<D, NT>& q) {
  using S = Decode<D, NT>;
  constexpr int kGroups = Cells<D>::kGroups;
  const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < S::kTilesN; ++nt) {
    float x[kGroups][16];
    float big = 0.f, sum[kGroups];
#pragma unroll
    for (int gr = 0; gr < kGroups; ++gr) {
      sum[gr] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 u = raw.v[nt][gr][h];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = from16<F16>(static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1))));
          x[gr][h * 8 + e] = v;
          big = fmaxf(big, fabsf(v));
          sum[gr] += v;
        }
      }
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], d);
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
    // A power of two brings the row's largest element to [2^13, 2^14): float16 then holds what is above 2^-38 of it.
    const int ex = (__float_as_uint(big) >> 23) & 255;
    const float up = __uint_as_float(static_cast<uint32_t>(min(254, max(1, 267 - ex))) << 23);
#pragma unroll
    for (int gr = 0; gr < kGroups; ++gr)
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          const float f = odd ? up * 0.0625f : up;
          const float* v = &x[gr][8 * w + odd];
          q.frag[gr * 4 + w * 2 + odd][nt][0] = pack_half2(v[0] * f, v[4] * f);
          q.frag[gr * 4 + w * 2 + odd][nt][1] = pack_half2(v[2] * f, v[6] * f);
        }
    const float scale = a.scaling * kLog2e;
    const float fac = scale * (16777216.f / up);
#pragma unroll
    for (int c = 0; c < S::kCols; ++c) {
      const int from = (2 * t + c) * 4;  // a lane of the column's row
      q.factor[nt][c] = __shfl_sync(0xffffffffu, fac, from);
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) q.sum[nt][c][gr] = __shfl_sync(0xffffffffu, sum[gr] * scale, from);
      const int r = row0 + S::row(nt, t, c), i = r / share;
      q.limit[nt][c] = (r < a.q_len * share && i < fresh) ? start + i + 1 : 0;
    }
  }
}

// Running softmax of a unit: per column (query row) the reference -(m - kBias), the sums of p and of p * low, and O^T
// over the codes in units of 2^k * 2^-24 (even dimensions) or 2^-20 (odd ones).
template <int D, int NT>
struct State {
  using S = Decode<D, NT>;
  float o[D / 16][S::kTilesN][2 * S::kCols];  // [column] of dimension row g, then of g + 8
  float l[S::kTilesN][S::kCols], neg[S::kTilesN][S::kCols], low[S::kTilesN][S::kCols][Cells<D>::kGroups];
  float unit;      // 2^-k
  uint32_t cap;    // 2^k as float16 bits: no scale so far is above it
  uint32_t known;  // bit kCols nt + c: the column has a reference
  bool open;       // some column has none yet (warp-uniform)
};

// Before a page's tokens: the unit for their value scales (tokens from `seen` on are not looked at).
template <int D, int NT>
__device__ __forceinline__ void fit_unit(const uint8_t* page, int base, int seen, State<D, NT>& st) {
  using C = Cells<D>;
  using S = Decode<D, NT>;
  const int lane = threadIdx.x & 31;
  uint32_t most = 0;  // scales are not negative: ordered as their bits (but for the sign that a zero may have)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = lane + 32 * h;
    const uint8_t* hp = page + C::value_head(r, 0);
    uint32_t top;
    if constexpr (C::kGroups == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(hp);
      top = max(u.x & 0x7fffu, u.y & 0x7fffu);
    } else {
      top = *reinterpret_cast<const uint32_t*>(hp) & 0x7fffu;
    }
    if (base + r < seen) most = max(most, top);
  }
  if (!__any_sync(0xffffffffu, most > st.cap)) return;
  most = __reduce_max_sync(0xffffffffu, most);
  // a power of two at least twice the largest scale, so that it seldom has to move
  const int ex = (__float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(most)))) >> 23) & 255;
  const float unit = __uint_as_float(static_cast<uint32_t>(252 - ex) << 23);
  st.cap = __half_as_ushort(__float2half_rn(1.f / unit));
  const float shrink = unit / st.unit;
  st.unit = unit;
#pragma unroll
  for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
    for (int nt = 0; nt < S::kTilesN; ++nt)
#pragma unroll
      for (int e = 0; e < 2 * S::kCols; ++e) st.o[mt][nt][e] *= shrink;
}

// 16 * TT tokens of a page in shared memory (rows 16 * tile ..), the first of them token `base` of the conversation.
// EDGE: some row does not see some of them.
template <int D, int NT, int TT, bool F16, bool EDGE>
__device__ __forceinline__ void attend(const uint8_t* page, int tile, int base, int seen, const Query<D, NT>& q,
                                       State<D, NT>& st) {
  using C = Cells<D>;
  using S = Decode<D, NT>;
  constexpr int kGroups = C::kGroups, kN = S::kTilesN, kCols = S::kCols;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float p[TT][kN][2][kCols];  // [tokens g, g + 8][column]
  __half2 vhead[TT][2][kGroups];
  bool rise = EDGE || st.open;
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
    // ---- scores of tokens g and g + 8
    const int row = (tile + tt) * 16 + g;
    float acc[kGroups][kN][4];
    const uint8_t* kr = page + C::kKeyCodes + row * (D / 2) + t * (D / 8);
    uint32_t x[2 * kGroups], y[2 * kGroups];
    if constexpr (D == 128) {
      const uint4 u = *reinterpret_cast<const uint4*>(kr), v = *reinterpret_cast<const uint4*>(kr + 8 * (D / 2));
      x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
      y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(kr), v = *reinterpret_cast<const uint2*>(kr + 8 * (D / 2));
      x[0] = u.x, x[1] = u.y;
      y[0] = v.x, y[1] = v.y;
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) {
        const uint32_t u = x[gr * 2 + w], v = y[gr * 2 + w], u8 = u >> 8, v8 = v >> 8;
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          const uint32_t mask = odd ? 0x00f000f0u : 0x000f000fu;
#pragma unroll
          for (int nt = 0; nt < kN; ++nt) {
            const uint32_t* b = q.frag[gr * 4 + w * 2 + odd][nt];
            if (w == 0 && odd == 0) mma16816_first(acc[gr][nt], u & mask, v & mask, u8 & mask, v8 & mask, b[0], b[1]);
            else mma16816(acc[gr][nt], u & mask, v & mask, u8 & mask, v8 & mask, b[0], b[1]);
          }
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t hd[2 * kGroups];
      const uint8_t* hp = page + C::kHeads + (row + 8 * h) * C::kHeadBytes;
      if constexpr (kGroups == 2) {
        const uint4 u = *reinterpret_cast<const uint4*>(hp);
        hd[0] = u.x, hd[1] = u.y, hd[2] = u.z, hd[3] = u.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(hp);
        hd[0] = u.x, hd[1] = u.y;
      }
      const bool gone = EDGE && base + tt * 16 + g + 8 * h >= seen;
      float ks[kGroups], kl[kGroups];
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) {
        const float2 f = __half22float2(as_half2(hd[gr]));
        ks[gr] = f.x;
        kl[gr] = f.y;
        // tokens that no row sees may never have been written: no NaN of theirs into the sums
        vhead[tt][h][gr] = as_half2(gone ? 0u : hd[kGroups + gr]);
      }
#pragma unroll
      for (int nt = 0; nt < kN; ++nt)
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          float dot = ks[0] * acc[0][nt][2 * h + c];
          float s = fmaf(kl[0], q.sum[nt][c][0], st.neg[nt][c]);
          if constexpr (kGroups == 2) {
            dot = fmaf(ks[1], acc[1][nt][2 * h + c], dot);
            s = fmaf(kl[1], q.sum[nt][c][1], s);
          }
          s = fmaf(dot, q.factor[nt][c], s);
          if constexpr (EDGE) {
            if (base + tt * 16 + g + 8 * h >= q.limit[nt][c]) s = -INFINITY;
          }
          p[tt][nt][h][c] = s;
          rise = rise || s > kBias + kSlack;
        }
    }
  }
  if (__any_sync(0xffffffffu, rise)) {
    // ---- a score above the reference's slack, or a column without a reference: references move up to the columns'
    // maxima, and what is summed so far scales down
    bool open = false;
#pragma unroll
    for (int nt = 0; nt < kN; ++nt) {
      float f[kCols];
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        float top = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) top = fmaxf(top, fmaxf(p[tt][nt][0][c], p[tt][nt][1][c]));
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        // a column's first tokens set the reference wherever they are; later ones raise it, and only from beyond the
        // slack, so that a row's result does not depend on the rows beside it
        const uint32_t bit = 1u << (kCols * nt + c);
        const bool first = (st.known & bit) == 0, none = first && top == -INFINITY;
        const float move = none ? 0.f : first || top > kBias + kSlack ? top - kBias : 0.f;
        st.known |= none ? 0u : bit;
        f[c] = first ? 0.f : exp2_fast(-move);
        st.neg[nt][c] -= move;
        st.l[nt][c] *= f[c];
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) st.low[nt][c][gr] *= f[c];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
          p[tt][nt][0][c] -= move;
          p[tt][nt][1][c] -= move;
        }
        open = open || none;
      }
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int e = 0; e < 2 * kCols; ++e) st.o[mt][nt][e] *= f[e % kCols];
    }
    st.open = __any_sync(0xffffffffu, open);
  }
  // Second operands: with a column per row what a float16 rounding lacks takes products of its own, with a pair of
  // columns it is the second column's.
  constexpr bool kMore = F16 && !S::kPair;
  uint32_t pf[TT][kGroups][kN][2], pr[kMore ? TT : 1][kGroups][kN][2], v[TT][2][D / 32];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float vs[kGroups], vl[kGroups];
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) {
        const float2 f = __half22float2(vhead[tt][h][gr]);
        vs[gr] = f.x * st.unit;
        vl[gr] = f.y;
      }
#pragma unroll
      for (int nt = 0; nt < kN; ++nt) {
        float e[kCols];
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          e[c] = exp2_fast(p[tt][nt][h][c]);
          st.l[nt][c] += e[c];
#pragma unroll
          for (int gr = 0; gr < kGroups; ++gr) st.low[nt][c][gr] = fmaf(e[c], vl[gr], st.low[nt][c][gr]);
        }
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) {
          const float w0 = e[0] * vs[gr];
          if constexpr (S::kPair) {
            uint32_t hi = pack_half2(w0, 0.f);
            if constexpr (F16) hi = pack_half2(w0, w0 - __low2float(as_half2(hi)));
            pf[tt][gr][nt][h] = transpose8(hi);
          } else {
            const float w1 = e[kCols - 1] * vs[gr];
            const uint32_t hi = pack_half2(w0, w1);
            pf[tt][gr][nt][h] = transpose8(hi);
            if constexpr (kMore) {
              const float2 back = __half22float2(as_half2(hi));
              pr[tt][gr][nt][h] = transpose8(pack_half2(w0 - back.x, w1 - back.y));
            }
          }
        }
      }
    }
    // ---- values: token pairs t and t + 4 of the 16
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t* vr = page + C::value_piece((tile + tt) * 8 + t + 4 * h, g);
      if constexpr (D == 128) {
        const uint4 u = *reinterpret_cast<const uint4*>(vr);
        v[tt][h][0] = u.x, v[tt][h][1] = u.y, v[tt][h][2] = u.z, v[tt][h][3] = u.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(vr);
        v[tt][h][0] = u.x, v[tt][h][1] = u.y;
      }
    }
  }
  // The products of these tokens on their own, then added to O by the float32 units: the tensor core cuts a sum where
  // it does not round it, and the codes are not negative, so a long chain of its sums would drift (by 4e-5 over 10000
  // tokens, as much as 1e-3 of outputs that average to little).
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int nt = 0; nt < kN; ++nt) {
        float sum[4];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
          const uint32_t u = b ? v[tt][0][i] >> 8 : v[tt][0][i], w = b ? v[tt][1][i] >> 8 : v[tt][1][i];
          const uint32_t u0 = u & 0x000f000fu, u1 = u & 0x00f000f0u, w0 = w & 0x000f000fu, w1 = w & 0x00f000f0u;
          const uint32_t* hi = pf[tt][i >> 1][nt];
          if (tt == 0) mma16816_first(sum, u0, u1, w0, w1, hi[0], hi[1]);
          else mma16816(sum, u0, u1, w0, w1, hi[0], hi[1]);
          if constexpr (kMore) mma16816(sum, u0, u1, w0, w1, pr[tt][i >> 1][nt][0], pr[tt][i >> 1][nt][1]);
        }
        float* o = st.o[i * 2 + b][nt];
        if constexpr (S::kPair) {
          if constexpr (F16) add2(sum[0], sum[2], sum[1], sum[3]);
          add2(o[0], o[1], sum[0], sum[2]);
        } else {
          add2(o[0], o[1], sum[0], sum[1]);
          add2(o[2], o[3], sum[2], sum[3]);
        }
      }
}

// The new tokens of a page (tokens first .. last of the conversation), quantised by the warp into the page's copy in
// shared memory and into the cache: whatever the copy caught of them is overwritten. Tokens without a slot (of a plan that
// failed) stay out, as in dkv_q4_append: their places are those of an earlier plan's.
template <int D, bool F16>
__device__ __noinline__ void store_new(const dkv_q4_attend_args& a, int seq, int head, int start, int first, int last,
                                       uint8_t* copy, uint8_t* cell) {
  constexpr int kLanes = D / 16, kPer = 32 / (2 * kLanes);  // lanes of a row; tokens (key and value row) at a time
  const int lane = threadIdx.x & 31;
  const int j = lane % kLanes, is_value = (lane / kLanes) & 1, sub = lane / (2 * kLanes);
  const int64_t* sd = is_value ? a.v_stride : a.k_stride;
  const uint16_t* src = static_cast<const uint16_t*>(is_value ? a.value : a.key) + seq * sd[0] + head * sd[1] + j * 16;
  const int32_t* slots = a.slots + static_cast<int64_t>(seq) * a.q_len - start;
  for (int tok = first; tok < last; tok += kPer) {
    const int mine = tok + sub;
    int slot = -1;
    uint4 raw[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
    if (mine < last) {  // under way together
      slot = slots[mine];
      const uint4* from = reinterpret_cast<const uint4*>(src + (mine - start) * sd[2]);
      raw[0] = from[0], raw[1] = from[1];
    }
    const q4::CellPart<2> c = q4::quantise<F16>(raw);
    if (slot >= 0) {
      if (!c.fits) record_error(a.status, kSiteQ4Rows + kErrCellRange);
      const int r = mine % q4::kPage;
      if (is_value) {
        q4::store_value<D>(copy, r, j, c);
        q4::store_value<D>(cell, r, j, c);
      } else {
        q4::store_key<D>(copy, r, j, c);
        q4::store_key<D>(cell, r, j, c);
      }
    }
  }
  __syncwarp();
  fence_async_shared();  // the next bulk copy into this place comes after these writes
}

template <int D, int NT, bool F16>
__global__ void __launch_bounds__(kThreads, (Decode<D, NT>::kBlocksPerSm))
q4_decode_kernel(const __grid_constant__ dkv_q4_attend_args a, int chunks, int workers, int append) {
  using C = Cells<D>;
  using S = Decode<D, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = warp_id();
  const int g = lane >> 2, t = lane & 3;
  const int share = a.n_q_heads / a.n_kv_heads;
  const int rows = min(S::kRows, a.q_len * share);
  uint8_t* ring = smem + warp * S::kWarpBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars) + warp * S::kStages;
  if (lane == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  const int failed = status_at_entry(a.status);
  const int worker = warp * gridDim.x + blockIdx.x;  // neighbours in the line on different SMs
  const int units = a.n_kv_heads * chunks;  // of a conversation
  // Pages of the 32 conversations from `base` on, one per lane; the first 32 are kept for the search below.
  auto lane_pages = [&](int base) { return base + lane < a.n_seq ? pages_of(tokens_of(a, base + lane)) : 0; };
  const int kept = lane_pages(0);
  int64_t all = warp_sum(kept);
  for (int base = 32; base < a.n_seq; base += 32) all += warp_sum(lane_pages(base));
  const Deal deal(all * units, workers);
  if (__any_sync(0xffffffffu, failed != 0)) return;
  if (worker >= deal.workers) return;
  const int64_t begin = deal.begin(worker), end = deal.begin(worker + 1);

  // the conversation of the first page
  int seq = 0;
  int64_t seq_at = 0;  // its first place in the line
  for (int base = 0; base < a.n_seq; base += 32) {
    const int own = base == 0 ? kept : lane_pages(base);
    int incl = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, seq_at + static_cast<int64_t>(incl) * units > begin);
    if (past) {
      const int first = __ffs(past) - 1;
      seq = base + first;
      seq_at += static_cast<int64_t>(__shfl_sync(0xffffffffu, incl - own, first)) * units;
      break;
    }
    seq_at += static_cast<int64_t>(__shfl_sync(0xffffffffu, incl, 31)) * units;
  }

  uint32_t copies = 0;  // issued by this warp so far: stage copies % kStages, phase copies / kStages
  int64_t at = begin;
  while (at < end) {
    // ---- one unit's segment
    int tokens = tokens_of(a, seq);
    while (tokens == 0) tokens = tokens_of(a, ++seq);
    const int n_pages = pages_of(tokens);
    const int64_t off = at - seq_at;
    const int unit = static_cast<int>(divide<true>(off, n_pages));
    const int64_t unit_at = seq_at + static_cast<int64_t>(unit) * n_pages;
    const int p0 = static_cast<int>(at - unit_at);
    const int p1 = static_cast<int>(min(static_cast<int64_t>(n_pages), end - unit_at));
    const int head = unit / chunks, row0 = (unit - head * chunks) * S::kRows;
    const int start = a.starts[seq], fresh = min(tokens - start, a.q_len);
    const int last_i = min((min(row0 + S::kRows, a.q_len * share) - 1) / share, fresh - 1);
    const int seen = row0 / share < fresh ? start + last_i + 1 : 0;
    const int full_below = start + row0 / share + 1;  // tokens below it are seen by every row
    if (lane == 0)
      record_unit(unit_record(a, workers, rows, static_cast<int64_t>(seq) * units + unit), worker, at != begin, p0 == 0,
                  p1 == n_pages);
    const int32_t* table = a.blocks + static_cast<int64_t>(seq) * a.max_blocks;
    const int64_t page_stride = static_cast<int64_t>(a.n_kv_heads) * C::kBytes;
    uint8_t* cells = a.cells + static_cast<int64_t>(head) * C::kBytes;

    // The pages' places, one per lane, 32 at a time, the next 32 on their way.
    int ids_at = p0, ids = p0 + lane < p1 ? table[p0 + lane] : 0, ids_next = p0 + 32 + lane < p1 ? table[p0 + 32 + lane] : 0;
    RawQuery<D, NT> raw;
    fetch_query<D, NT>(a, seq, head, row0, share, fresh, raw);  // ahead of the pages, which would keep it waiting
    auto page_id = [&](int p) {
      if (p >= ids_at + 32) {
        ids_at += 32;
        ids = ids_next;
        ids_next = ids_at + 32 + lane < p1 ? table[ids_at + 32 + lane] : 0;
      }
      const int id = __shfl_sync(0xffffffffu, ids, p - ids_at);
      if (static_cast<unsigned>(id) < static_cast<unsigned>(a.n_pages)) return id;
      record_error(a.status, kSiteQ4Attend + kErrBadDescriptor);
      return -1;
    };
    const uint32_t copies0 = copies;  // page p is copy copies0 + p - p0
    auto fetch = [&](int p) {
      const int id = max(page_id(p), 0);  // a page that is none is recorded, and one that exists read in its place
      const uint32_t stage = copies % S::kStages;
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[stage], C::kBytes);
        bulk_load(ring + stage * C::kBytes, cells + id * page_stride, C::kBytes, &full[stage]);
      }
      ++copies;
    };
    const int pe = min(p1, pages_of(seen));  // what follows is seen by no row of this chunk
    __syncwarp();
    for (int p = p0; p < min(pe, p0 + S::kStages); ++p) fetch(p);

    Query<D, NT> q;
    make_query<D, NT, F16>(a, row0, share, start, fresh, raw, q);
    State<D, NT> st;
    st.open = true;
    st.known = 0;
    st.unit = 1.f;
    st.cap = 0;
#pragma unroll
    for (int nt = 0; nt < S::kTilesN; ++nt) {
#pragma unroll
      for (int c = 0; c < S::kCols; ++c) {
        st.l[nt][c] = st.neg[nt][c] = 0.f;
#pragma unroll
        for (int gr = 0; gr < C::kGroups; ++gr) st.low[nt][c][gr] = 0.f;
      }
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int e = 0; e < 2 * S::kCols; ++e) st.o[mt][nt][e] = 0.f;
    }

    bool ok = true;
    for (int p = p0; p < pe; ++p) {
      const uint32_t n = copies0 + (p - p0), stage = n % S::kStages;
      ok = warp_wait(&full[stage], (n / S::kStages) & 1, a.status, kSiteQ4Attend + kErrWaitCodes, nullptr);
      if (!ok) break;
      uint8_t* page = ring + stage * C::kBytes;
      const int base = p * q4::kPage;
      if (append && base + q4::kPage > start) {
        const int id = table[p];
        if (id >= 0 && id < a.n_pages)
          store_new<D, F16>(a, seq, head, start, max(start, base), min(start + fresh, base + q4::kPage), page,
                            cells + id * page_stride);
      }
      fit_unit<D, NT>(page, base, seen, st);
      if (base + q4::kPage <= full_below) {
        for (int tile = 0; tile < q4::kPage / 16; tile += S::kTiles)
          attend<D, NT, S::kTiles, F16, false>(page, tile, base + tile * 16, seen, q, st);
      } else {
        for (int tile = 0; tile < q4::kPage / 16 && base + tile * 16 < seen; ++tile)
          attend<D, NT, 1, F16, true>(page, tile, base + tile * 16, seen, q, st);
      }
      __syncwarp();
      if (p + S::kStages < pe) fetch(p + S::kStages);
    }
    if (!ok) {
      // leave with no copy of this warp in flight
      for (uint32_t n = copies - min(copies, static_cast<uint32_t>(S::kStages)); n < copies; ++n)
        warp_wait(&full[n % S::kStages], (n / S::kStages) & 1, a.status, kSiteQ4Attend + kErrWaitDrain, nullptr);
      return;
    }

    // ---- the segment's result
    const bool whole = p0 == 0 && p1 == n_pages;
    float* slot = a.workspace + (worker * 2 + (at == begin ? 0 : 1)) * slot_floats(rows, D);
    const float even = 0x1p24f / st.unit, odd = 0x1p20f / st.unit;
#pragma unroll
    for (int nt = 0; nt < S::kTilesN; ++nt)
#pragma unroll
      for (int c = 0; c < S::kCols; ++c) {
        float sum = st.l[nt][c], low[C::kGroups];
#pragma unroll
        for (int gr = 0; gr < C::kGroups; ++gr) low[gr] = st.low[nt][c][gr];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          sum += __shfl_xor_sync(0xffffffffu, sum, d);
#pragma unroll
          for (int gr = 0; gr < C::kGroups; ++gr) low[gr] += __shfl_xor_sync(0xffffffffu, low[gr], d);
        }
        const int col = S::row(nt, t, c), r = row0 + col, i = r / share;
        if (r >= a.q_len * share || i >= fresh) continue;  // the joins write the zeros behind the new tokens
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        const int64_t to =
            ((static_cast<int64_t>(seq) * a.q_len + i) * a.n_q_heads + head * share + r - i * share) * D + g * 8;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          const float y0 = fmaf(st.o[2 * k][nt][c], even, low[k >> 1]), y1 = fmaf(st.o[2 * k][nt][c + S::kCols], odd, low[k >> 1]);
          const float y2 = fmaf(st.o[2 * k + 1][nt][c], even, low[k >> 1]),
                      y3 = fmaf(st.o[2 * k + 1][nt][c + S::kCols], odd, low[k >> 1]);
          const int dim = (k >> 1) * 64 + (k & 1) * 4;
          if (whole) store_out4<F16>(a, to + dim, y0 * inv, y1 * inv, y2 * inv, y3 * inv);
          else *reinterpret_cast<float4*>(slot + col * D + g * 8 + dim) = make_float4(y0, y1, y2, y3);
        }
        if (!whole && g == 0) *reinterpret_cast<float2*>(slot + rows * D + col * 4) = make_float2(st.neg[nt][c], sum);
      }
    at = unit_at + p1;
    if (at == seq_at + static_cast<int64_t>(units) * n_pages) {
      seq_at = at;
      ++seq;
    }
  }
}

// The joins write the rows of the units that several workers share, and the zeros of the rows behind the new tokens.
struct JoinRow {
  int seq, head, r, i;
  int64_t to;  // where the row's output begins
  __device__ __forceinline__ JoinRow(const dkv_q4_attend_args& a, int id, int share, int d) {
    const int rows = a.q_len * share;
    const int line = id / rows;
    r = id - line * rows;
    seq = line / a.n_kv_heads;
    head = line - seq * a.n_kv_heads;
    i = r / share;
    to = ((static_cast<int64_t>(seq) * a.q_len + i) * a.n_q_heads + head * share + r - i * share) * d;
  }
};

// Many rows, of few pieces each: a warp per row.
constexpr int kJoinWarps = 8;
template <int D, int NT, bool F16>
__global__ void __launch_bounds__(kJoinWarps * 32)
q4_join_rows_kernel(const __grid_constant__ dkv_q4_attend_args a, int chunks, int workers) {
  constexpr int kRows = Decode<D, NT>::kRows;
  const int share = a.n_q_heads / a.n_kv_heads, rows = a.q_len * share, units = a.n_kv_heads * chunks;
  const int id = blockIdx.x * kJoinWarps + warp_id();
  if (id >= rows * a.n_kv_heads * a.n_seq) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const JoinRow row(a, id, share, D);
  const int tokens = tokens_of(a, row.seq), held = min(kRows, rows), chunk = row.r / kRows;
  const bool real = tokens > 0 && row.i < min(tokens - a.starts[row.seq], a.q_len);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // what is above does not depend on the main kernel
  const int2 by = *unit_record(a, workers, held, static_cast<int64_t>(row.seq) * units + row.head * chunks + chunk);
  const int failed = status_at_entry(a.status);
  float sum[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) sum[e] = 0.f;
  if (real && !__any_sync(0xffffffffu, failed != 0)) {
    const Pieces pieces(a, by, workers, held, D);
    if (pieces.n == 1) return;  // one worker had the whole unit
    // all of 32 pieces' loads under way, the first eight with their factors': 125.6 us where 64 conversations took 127.9
    join_row<D, -1, 24, 8>(pieces, held, row.r - chunk * kRows, sum);
  }
  store_row<D, F16>(a, row.to, sum);
}

// Few rows, of many pieces: a CTA per row and 32 dimensions; the pieces' factors first, then 8 lanes of 4 dimensions in
// kSlices slices over the pieces, with nothing that one load has to wait for another.
constexpr int kPartThreads = 256;
constexpr int kFactors = 512;  // pieces whose factors are held at a time
template <int D, int NT, bool F16>
__global__ void __launch_bounds__(kPartThreads)
q4_join_parts_kernel(const __grid_constant__ dkv_q4_attend_args a, int chunks, int workers) {
  constexpr int kRows = Decode<D, NT>::kRows, kParts = D / 32, kSlices = kPartThreads / 8;
  __shared__ float4 part[kPartThreads / 32][8];
  __shared__ float factor[kFactors];
  __shared__ float warp_ref[kPartThreads / 32], warp_den[kPartThreads / 32];
  const int share = a.n_q_heads / a.n_kv_heads, rows = min(kRows, a.q_len * share), units = a.n_kv_heads * chunks;
  const JoinRow row(a, blockIdx.x / kParts, share, D);
  const int tid = threadIdx.x, slice = tid / 8, dim = (blockIdx.x % kParts) * 32 + (tid % 8) * 4;
  const int tokens = tokens_of(a, row.seq), chunk = row.r / kRows, col = row.r - chunk * kRows;
  const bool real = tokens > 0 && row.i < min(tokens - a.starts[row.seq], a.q_len);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // what is above does not depend on the main kernel
  const int2 by = *unit_record(a, workers, rows, static_cast<int64_t>(row.seq) * units + row.head * chunks + chunk);
  // That one may have set the status word while others of its warps finished: the CTA's one answer.
  if (cta_failed_at_entry(a.status) || !real) {
    if (slice == 0) store_out4<F16>(a, row.to + dim, 0.f, 0.f, 0.f, 0.f);
    return;
  }
  const Pieces pieces(a, by, workers, rows, D);
  if (pieces.n == 1) return;  // one worker had the whole unit
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  float den = 0.f, ref = INFINITY;  // sums are relative to 2^-ref; the smallest ref is the largest maximum
  for (int base = 0; base < pieces.n; base += kFactors) {
    const int m = min(kFactors, pieces.n - base);
    float mine[kFactors / kPartThreads], weight[kFactors / kPartThreads];
    float low = INFINITY;
#pragma unroll
    for (int k = 0; k < kFactors / kPartThreads; ++k) {
      const int w = k * kPartThreads + tid;
      const float2 s = w < m ? *reinterpret_cast<const float2*>(pieces.slot(base + w) + rows * D + col * 4) : make_float2(0.f, 0.f);
      mine[k] = s.y == 0.f ? INFINITY : s.x;  // a piece that saw no token of this row
      weight[k] = s.y;
      low = fminf(low, mine[k]);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, d));
    if ((tid & 31) == 0) warp_ref[tid >> 5] = low;
    __syncthreads();
    float now = ref;
#pragma unroll
    for (int k = 0; k < kPartThreads / 32; ++k) now = fminf(now, warp_ref[k]);
    float add = 0.f;
#pragma unroll
    for (int k = 0; k < kFactors / kPartThreads; ++k) {
      const int w = k * kPartThreads + tid;
      const float f = mine[k] == INFINITY ? 0.f : exp2_fast(now - mine[k]);
      if (w < m) factor[w] = f;
      add = fmaf(weight[k], f, add);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) add += __shfl_xor_sync(0xffffffffu, add, d);
    if ((tid & 31) == 0) warp_den[tid >> 5] = add;
    __syncthreads();
    const float keep = ref == INFINITY ? 0.f : exp2_fast(now - ref);
    den *= keep;
#pragma unroll
    for (int k = 0; k < kPartThreads / 32; ++k) den += warp_den[k];
    sum.x *= keep, sum.y *= keep, sum.z *= keep, sum.w *= keep;
    ref = now;
#pragma unroll 8
    for (int w = slice; w < m; w += kSlices) {
      const float4 o = *reinterpret_cast<const float4*>(pieces.slot(base + w) + col * D + dim);
      const float f = factor[w];
      sum.x = fmaf(o.x, f, sum.x);
      sum.y = fmaf(o.y, f, sum.y);
      sum.z = fmaf(o.z, f, sum.z);
      sum.w = fmaf(o.w, f, sum.w);
    }
    __syncthreads();
  }
  // the slices' sums: four of a warp's by shuffles, the warps' through shared memory
#pragma unroll
  for (int d = 8; d < 32; d <<= 1) {
    sum.x += __shfl_xor_sync(0xffffffffu, sum.x, d);
    sum.y += __shfl_xor_sync(0xffffffffu, sum.y, d);
    sum.z += __shfl_xor_sync(0xffffffffu, sum.z, d);
    sum.w += __shfl_xor_sync(0xffffffffu, sum.w, d);
  }
  if ((tid & 31) < 8) part[tid >> 5][tid & 7] = sum;
  __syncthreads();
  if (slice != 0) return;
#pragma unroll
  for (int k = 1; k < kPartThreads / 32; ++k) {
    const float4 o = part[k][tid];
    sum.x += o.x, sum.y += o.y, sum.z += o.z, sum.w += o.w;
  }
  const float inv = den != 0.f ? 1.f / den : 0.f;
  store_out4<F16>(a, row.to + dim, sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
}

// NT of q4_decode_kernel, and the query rows that a warp then holds.
int tiles_of(const dkv_q4_attend_args& a) {
  const int rows = rows_of(a);
  // 17 to 24 rows of heads of 64 go through the pages once, in three tiles (a third one of 128 leaves no registers).
  return rows <= 4 ? 0 : rows <= 8 ? 1 : rows > 16 && rows <= 24 && a.head_dim == 64 ? 3 : 2;
}
int held_rows(int nt) { return nt == 0 ? 4 : 8 * nt; }

int64_t floats_of(const dkv_q4_attend_args& a) {
  const int rows = rows_of(a), most = held_rows(tiles_of(a)), held = rows < most ? rows : most;
  const int64_t units = static_cast<int64_t>(a.n_seq) * a.n_kv_heads * ((rows + most - 1) / most);
  return 2 * static_cast<int64_t>(device_sms() * 3 * kWarps) * slot_floats(held, a.head_dim) + 2 * units;
}

template <int D, int NT, bool F16>
int launch_decode(const dkv_q4_attend_args& a, int append, cudaStream_t stream) {
  const int rows = rows_of(a), held = held_rows(NT), chunks = (rows + held - 1) / held;
  if (static_cast<int64_t>(a.n_kv_heads) > 65535) return DKV_ERR_CONFIG;
  // At most one worker per page that there can be.
  const int64_t pages = static_cast<int64_t>((a.len_bound + q4::kPage - 1) / q4::kPage) * a.n_seq * a.n_kv_heads * chunks;
  const int most = device_sms() * Decode<D, NT>::kBlocksPerSm;
  const int ctas = pages < most ? (pages < 1 ? 1 : static_cast<int>(pages)) : most;
  const int workers = ctas * kWarps;
  auto kernel = q4_decode_kernel<D, NT, F16>;
  constexpr int bytes = Decode<D, NT>::kBytes;
  static std::atomic<uint64_t> done{0};
  if (!allow_shared(kernel, bytes, done)) return DKV_ERR_CUDA;
  kernel<<<ctas, kThreads, bytes, stream>>>(a, chunks, workers, append);
  if (cudaGetLastError() != cudaSuccess) return DKV_ERR_CUDA;
  // Many rows have few pieces each and a warp does for one; of few rows each has the pieces of many workers. 24 heads of
  // 128 over 4K-16K tokens: 64 conversations 127 us with a warp per row, 156 with CTAs; 16: 48 and 52; 8: 38 and 34.
  const int64_t joins = static_cast<int64_t>(rows) * a.n_kv_heads * a.n_seq;
  const bool many = joins >= 256;
  const int64_t grid = many ? (joins + kJoinWarps - 1) / kJoinWarps : joins * (D / 32);
  if (joins * (D / 32) > INT32_MAX) return DKV_ERR_CONFIG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(many ? kJoinWarps * 32 : kPartThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto join = many ? q4_join_rows_kernel<D, NT, F16> : q4_join_parts_kernel<D, NT, F16>;
  return cudaLaunchKernelEx(&cfg, join, a, chunks, workers) == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
}

int check_sizes(const dkv_q4_attend_args* a) {
  if (a->n_pages < 1 || a->max_blocks < 1 || a->n_seq < 0 || a->q_len < 0 || a->n_kv_heads < 1 || a->n_q_heads < 1 ||
      a->n_q_heads % a->n_kv_heads != 0)
    return DKV_ERR_ARGS;
  if (a->head_dim != 64 && a->head_dim != 128) return DKV_ERR_CONFIG;
  if (static_cast<int64_t>(a->n_pages) * q4::kPage > INT32_MAX ||
      static_cast<int64_t>(a->max_blocks) * q4::kPage > INT32_MAX || a->n_seq > 8192 || a->n_kv_heads > 65535 ||
      static_cast<int64_t>(a->q_len) * a->n_q_heads > INT32_MAX / 2)
    return DKV_ERR_CONFIG;
  return DKV_OK;
}

}  // namespace
}  // namespace dkv

extern "C" {

int64_t dkv_q4_attend_floats(const dkv_q4_attend_args* a) {
  if (a == nullptr || dkv::check_sizes(a) != DKV_OK) return -1;
  if (a->n_seq == 0 || a->q_len == 0) return 0;
  return dkv::q4::prefill_takes(*a) ? dkv::q4::prefill_floats(*a) : dkv::floats_of(*a);
}

int dkv_q4_attend(const dkv_q4_attend_args* a, void* stream) {
  if (a == nullptr || a->cells == nullptr || a->blocks == nullptr || a->lengths == nullptr || a->starts == nullptr ||
      a->status == nullptr)
    return DKV_ERR_ARGS;
  const int rc = dkv::check_sizes(a);
  if (rc != DKV_OK) return rc;
  if (a->n_seq == 0 || a->q_len == 0) return DKV_OK;  // tensors without an element have no address
  if (a->query == nullptr || a->out == nullptr) return DKV_ERR_ARGS;
  if ((a->key == nullptr) != (a->value == nullptr) || (a->key != nullptr && a->slots == nullptr)) return DKV_ERR_ARGS;
  if (reinterpret_cast<uintptr_t>(a->cells) % 16 || reinterpret_cast<uintptr_t>(a->query) % 16 ||
      reinterpret_cast<uintptr_t>(a->key) % 16 || reinterpret_cast<uintptr_t>(a->value) % 16 ||
      reinterpret_cast<uintptr_t>(a->out) % 16 || reinterpret_cast<uintptr_t>(a->workspace) % 16)
    return DKV_ERR_ARGS;
  for (int k = 0; k < 3; ++k)
    if (a->q_stride[k] % 8 || (a->key != nullptr && (a->k_stride[k] % 8 || a->v_stride[k] % 8))) return DKV_ERR_ARGS;
  if (a->workspace == nullptr || a->workspace_floats < dkv_q4_attend_floats(a)) return DKV_ERR_SCRATCH;
  const bool prefill = dkv::q4::prefill_takes(*a);
  const int nt = dkv::tiles_of(*a);
  int append = a->key != nullptr;
  if (append && (prefill || dkv::q4::rows_of(*a) > dkv::held_rows(nt))) {
    // Several row chunks read a new token's page: it has to be there before the first of them.
    dkv_q4_rows_args r = {};
    r.cells = a->cells;
    r.n_pages = a->n_pages, r.n_kv_heads = a->n_kv_heads, r.head_dim = a->head_dim, r.fp16 = a->fp16;
    r.slots = a->slots;
    r.n_seq = a->n_seq, r.q_len = a->q_len;
    r.key = const_cast<void*>(a->key), r.value = const_cast<void*>(a->value);
    for (int k = 0; k < 3; ++k) r.k_stride[k] = a->k_stride[k], r.v_stride[k] = a->v_stride[k];
    r.status = a->status;
    const int done = dkv_q4_append(&r, stream);
    if (done != DKV_OK) return done;
    append = 0;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (prefill) return dkv::q4::run_prefill(*a, a->key != nullptr, st);
#define DKV_Q4_DECODE(D, NT) \
  (a->fp16 ? dkv::launch_decode<D, NT, true>(*a, append, st) : dkv::launch_decode<D, NT, false>(*a, append, st))
  if (a->head_dim == 128) return nt == 0 ? DKV_Q4_DECODE(128, 0) : nt == 1 ? DKV_Q4_DECODE(128, 1) : DKV_Q4_DECODE(128, 2);
  return nt == 0 ? DKV_Q4_DECODE(64, 0) : nt == 1 ? DKV_Q4_DECODE(64, 1) : nt == 2 ? DKV_Q4_DECODE(64, 2) : DKV_Q4_DECODE(64, 3);
#undef DKV_Q4_DECODE
}

}  // extern "C"
