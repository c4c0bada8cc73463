// q4_attend.cu — causal attention of new tokens' queries over the paged 4-bit cache (dkv_q4_attend), and the new
// tokens' cells with it.
//
// With key value k_d = low_g + scale_g * c_d (g = d / 64), a score splits into
//   q . k = sum_g scale_g * (sum_{d in g} q_d c_d) + sum_g low_g * (sum_{d in g} q_d):
// the product runs over the codes themselves, which float16 holds exactly, and the key's rounding is the
// cache's alone. Values enter as float16(low + scale * c), one rounding of at most 2^-11 relative; probabilities
// as float16 of 2^7 * exp(score - m) with m within 2^8 of the running maximum, so that a token down to 2^-21 of the
// largest keeps 11 bits (sums over a long context of small probabilities do not vanish). For float16 outputs, whose
// own step is as small, a probability enters as two float16 numbers (the rounded one and what it lacks).
//
// q4_decode_kernel: few query rows per KV head (one token, or a short draft). Bound by the cells' bytes. The pages of
// all (conversation, KV head, row chunk) units form one line, cut into equal pieces, one per WARP, so that any mix
// of lengths, heads and conversations fills the GPU evenly; a unit that several warps share leaves partial
// (m, l, O) in the workspace, which q4_combine_kernel joins. A page of one KV head is one contiguous block: each warp
// keeps a ring of bulk copies of its own and meets no other warp. It contracts tokens as the 16 rows of m16n8k16
// and query rows as its 8 columns (3 or 4 heads that share a KV head are the rule), S^T = C Q^T, then O^T = V^T P^T;
// P^T in the layout of the second product is one 8 x 8 transpose per 8 tokens (movmatrix). A code pair of a word is a
// float16 pair after ONE mask: the 4 bits are a subnormal c * 2^-24 (or 16 times that, from the odd nibbles,
// against q / 16), and the power of two goes into the score's factor. The warp that owns a new token's page
// quantises the token itself, into the page's copy and into the cache.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dkv_ptx.cuh"
#include "q4_cells.cuh"

namespace dkv {
namespace {

using q4::Cells;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBias = 7.f;    // probabilities are scaled by 2^7
constexpr float kSlack = 8.f;   // the reference maximum may lag by 2^8: 2^(7 + 8) < 65504

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 matrix of 16-bit elements held one pair per lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) { return as_u32(__floats2half2_rn(lo, hi)); }

// How the pages of all units are dealt to the workers (warps): worker w takes the pages
// [total * w / workers, total * (w + 1) / workers) of the line (conversation, KV head, row chunk, page).
struct Deal {
  int64_t total;
  int workers;
  __device__ __forceinline__ int64_t begin(int w) const { return total * w / workers; }
  __device__ __forceinline__ int owner(int64_t x) const { return static_cast<int>(((x + 1) * workers - 1) / total); }
};

// Tokens that conversation s attends over (0 if it has no new token).
__device__ __forceinline__ int tokens_of(const dkv_q4_attend_args& a, int s) {
  const int start = a.starts[s], len = min(a.lengths[s], a.max_blocks * q4::kPage);
  return start >= 0 && len > start ? len : 0;
}
__device__ __forceinline__ int pages_of(int tokens) { return (tokens + q4::kPage - 1) / q4::kPage; }

__device__ __forceinline__ int warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }

// One warp: pages of all conversations, and of those before `seq`.
__device__ __forceinline__ int64_t count_pages(const dkv_q4_attend_args& a, int seq, int64_t& before) {
  int64_t total = 0;
  before = 0;
  for (int base = 0; base < a.n_seq; base += 32) {
    const int s = base + (threadIdx.x & 31);
    const int p = s < a.n_seq ? pages_of(tokens_of(a, s)) : 0;
    total += warp_sum(p);
    before += warp_sum(s < seq ? p : 0);
  }
  return total;
}

template <int D, int NT>
struct Decode {
  using C = Cells<D>;
  static constexpr int kRows = 8 * NT;
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kBlocksPerSm = D == 128 && NT == 2 ? 2 : 3;  // two accumulators of 128 need the registers
  static constexpr int kWarpBytes = kStages * C::kBytes;
  static constexpr int kBars = kWarps * kWarpBytes;
  static constexpr int kBytes = kBars + kWarps * kStages * 8;
};

// A unit's query rows as the second operand, and the factors of their scores.
template <int D, int NT>
struct Query {
  static constexpr int kGroups = Cells<D>::kGroups;
  uint32_t frag[D / 16][NT][2];
  float factor[NT][2], sum[NT][2][kGroups];
  int limit[NT][2];  // tokens below it are seen (0: no row)
};

template <int D, int NT, bool F16>
__device__ __forceinline__ void load_query(const dkv_q4_attend_args& a, int seq, int head, int row0, int share, int start,
                                           int fresh, Query<D, NT>& q) {
  constexpr int kGroups = Cells<D>::kGroups;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = row0 + nt * 8 + g;
    const int i = r / share;
    const bool real = r < a.q_len * share && i < fresh;
    float x[kGroups][16];
    float big = 0.f, sum[kGroups];
#pragma unroll
    for (int gr = 0; gr < kGroups; ++gr) {
      uint4 raw[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
      if (real) {
        const uint16_t* src = static_cast<const uint16_t*>(a.query) + seq * a.q_stride[0] +
                              (head * share + r - i * share) * a.q_stride[1] + i * a.q_stride[2] + gr * 64 + t * 16;
        raw[0] = *reinterpret_cast<const uint4*>(src);
        raw[1] = *reinterpret_cast<const uint4*>(src + 8);
      }
      sum[gr] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w[4] = {raw[h].x, raw[h].y, raw[h].z, raw[h].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = q4::from16<F16>(static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1))));
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
    for (int c = 0; c < 2; ++c) {
      const int from = (2 * t + c) * 4;
      q.factor[nt][c] = __shfl_sync(0xffffffffu, fac, from);
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) q.sum[nt][c][gr] = __shfl_sync(0xffffffffu, sum[gr] * scale, from);
      const int rc = row0 + nt * 8 + 2 * t + c, ic = rc / share;
      q.limit[nt][c] = (rc < a.q_len * share && ic < fresh) ? start + ic + 1 : 0;
    }
  }
}

// Running softmax of a unit: per column (query row) the reference -(m - kBias), the sum, and O^T.
template <int D, int NT>
struct State {
  float o[D / 16][NT][4];
  float l[NT][2], neg[NT][2];
  uint32_t known;  // bit 2 nt + c: the column has a reference
  bool open;       // some column has none yet (warp-uniform)
};

// 16 tokens of a page in shared memory (rows tile * 16 ..), the first of them token `base` of the conversation. EDGE:
// some row does not see some of the 16.
template <int D, int NT, bool F16, bool EDGE>
__device__ __forceinline__ void attend16(const uint8_t* page, int tile, int base, int seen, const Query<D, NT>& q,
                                         State<D, NT>& st) {
  using C = Cells<D>;
  constexpr int kGroups = C::kGroups;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // ---- scores: rows g and g + 8
  float acc[kGroups][NT][4];
  {
    const uint8_t* kr = page + C::kKeyCodes + (tile * 16 + g) * (D / 2) + t * (D / 8);
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
    for (int gr = 0; gr < kGroups; ++gr) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[gr][nt][e] = 0.f;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t u = x[gr * 2 + w], v = y[gr * 2 + w], u8 = u >> 8, v8 = v >> 8;
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          const uint32_t mask = odd ? 0x00f000f0u : 0x000f000fu;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816(acc[gr][nt], u & mask, v & mask, u8 & mask, v8 & mask, q.frag[gr * 4 + w * 2 + odd][nt][0],
                     q.frag[gr * 4 + w * 2 + odd][nt][1]);
        }
      }
    }
  }
  float ks[2][kGroups], kl[2][kGroups];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int gr = 0; gr < kGroups; ++gr) {
      const float2 f = __half22float2(
          as_half2(*reinterpret_cast<const uint32_t*>(page + C::key_head(tile * 16 + g + 8 * h, gr))));
      ks[h][gr] = f.x;
      kl[h][gr] = f.y;
    }
  float p[NT][4];
  bool rise = EDGE || st.open;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int h = e >> 1, c = e & 1;
      float dot = ks[h][0] * acc[0][nt][e];
      float s = fmaf(kl[h][0], q.sum[nt][c][0], st.neg[nt][c]);
      if constexpr (kGroups == 2) {
        dot = fmaf(ks[h][1], acc[1][nt][e], dot);
        s = fmaf(kl[h][1], q.sum[nt][c][1], s);
      }
      s = fmaf(dot, q.factor[nt][c], s);
      if constexpr (EDGE) {
        if (base + g + 8 * h >= q.limit[nt][c]) s = -INFINITY;
      }
      p[nt][e] = s;
      rise = rise || s > kBias + kSlack;
    }
  if (__any_sync(0xffffffffu, rise)) {
    // ---- a score above the reference's slack, or a column without a reference: references move up to the columns'
    // maxima, and what is summed so far scales down
    bool open = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float f[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = fmaxf(p[nt][c], p[nt][c + 2]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        // a column's first tokens set the reference wherever they are; later ones only raise it
        const uint32_t bit = 1u << (2 * nt + c);
        const bool first = (st.known & bit) == 0, none = first && top == -INFINITY;
        const float move = none ? 0.f : first ? top - kBias : fmaxf(top - kBias, 0.f);
        st.known |= none ? 0u : bit;
        f[c] = first ? 0.f : exp2_fast(-move);
        st.neg[nt][c] -= move;
        st.l[nt][c] *= f[c];
        p[nt][c] -= move;
        p[nt][c + 2] -= move;
        open = open || none;
      }
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) st.o[mt][nt][e] *= f[e & 1];
    }
    st.open = __any_sync(0xffffffffu, open);
  }
  uint32_t pf[NT][2], pr[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      p[nt][e] = exp2_fast(p[nt][e]);
      st.l[nt][e & 1] += p[nt][e];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t hi = pack_half2(p[nt][2 * h], p[nt][2 * h + 1]);
      pf[nt][h] = transpose8(hi);
      if constexpr (F16) {
        const float2 back = __half22float2(as_half2(hi));
        pr[nt][h] = transpose8(pack_half2(p[nt][2 * h] - back.x, p[nt][2 * h + 1] - back.y));
      }
    }
  }
  // ---- values: token pairs t and t + 4 of the 16
  uint32_t v[2][D / 32];
  __half2 vs[2], vl[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int pair = tile * 8 + t + 4 * h;
    const uint8_t* vr = page + C::value_piece(pair, g);
    if constexpr (D == 128) {
      const uint4 u = *reinterpret_cast<const uint4*>(vr);
      v[h][0] = u.x, v[h][1] = u.y, v[h][2] = u.z, v[h][3] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(vr);
      v[h][0] = u.x, v[h][1] = u.y;
    }
    uint2 hd = *reinterpret_cast<const uint2*>(page + C::value_head(pair, kGroups == 2 ? g >> 2 : 0));
    if constexpr (EDGE) {
      // tokens that no row sees may never have been written: no NaN of theirs into the sums
      const int tok = base + 2 * (t + 4 * h);
      const uint32_t keep = (tok < seen ? 0x0000ffffu : 0u) | (tok + 1 < seen ? 0xffff0000u : 0u);
      hd.x &= keep;
      hd.y &= keep;
    }
    vs[h] = as_half2(hd.x);
    vl[h] = as_half2(hd.y);
  }
  const __half2 k1024 = as_half2(0x64006400u), k16th = as_half2(0x2c002c00u), k64 = as_half2(0xd400d400u);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint32_t x[2][2];  // [tokens t / t + 4][dimension 2 b, 2 b + 1]
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w = b ? v[h][i] >> 8 : v[h][i];
        // 1024 + c and 1024 + 16 c, both exact; then c, then the value with its one rounding
        const __half2 even = __hsub2(as_half2((w & 0x000f000fu) | 0x64006400u), k1024);
        const __half2 odd = __hfma2(as_half2((w & 0x00f000f0u) | 0x64006400u), k16th, k64);
        x[h][0] = as_u32(__hfma2(even, vs[h], vl[h]));
        x[h][1] = as_u32(__hfma2(odd, vs[h], vl[h]));
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma16816(st.o[i * 2 + b][nt], x[0][0], x[0][1], x[1][0], x[1][1], pf[nt][0], pf[nt][1]);
        if constexpr (F16) mma16816(st.o[i * 2 + b][nt], x[0][0], x[0][1], x[1][0], x[1][1], pr[nt][0], pr[nt][1]);
      }
    }
  }
}

// The new tokens of a page (tokens first .. last of the conversation), quantised by the warp into the page's copy in
// shared memory and into the cache: whatever the copy caught of them is overwritten.
template <int D, bool F16>
__device__ __noinline__ void store_new(const dkv_q4_attend_args& a, int seq, int head, int start, int first, int last,
                                       uint8_t* copy, uint8_t* cell) {
  constexpr int kLanes = D / 8, kPer = 32 / (2 * kLanes);  // lanes of a row; tokens (key and value row) at a time
  const int lane = threadIdx.x & 31;
  const int j = lane % kLanes, is_value = (lane / kLanes) & 1, sub = lane / (2 * kLanes);
  const int64_t* sd = is_value ? a.v_stride : a.k_stride;
  const uint16_t* src = static_cast<const uint16_t*>(is_value ? a.value : a.key) + seq * sd[0] + head * sd[1] + j * 8;
  for (int tok = first; tok < last; tok += kPer) {
    const int mine = tok + sub;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (mine < last) raw = *reinterpret_cast<const uint4*>(src + (mine - start) * sd[2]);
    const q4::Cell8 c = q4::quantise8<F16>(raw);
    if (!c.fits) record_error(a.status, kSiteQ4Rows + kErrCellRange);
    if (mine < last) {
      const int r = mine % q4::kPage;
      if (is_value) {
        q4::store_value8<D>(copy, r, j, c);
        q4::store_value8<D>(cell, r, j, c);
      } else {
        q4::store_key8<D>(copy, r, j, c);
        q4::store_key8<D>(cell, r, j, c);
      }
    }
  }
  __syncwarp();
  fence_async_shared();  // the next bulk copy into this place comes after these writes
}

template <bool F16>
__device__ __forceinline__ void store_out4(const dkv_q4_attend_args& a, int64_t at, float x, float y, float z, float w) {
  if (a.out_f32)
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(x, y, z, w);
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
        make_uint2(static_cast<uint32_t>(q4::to16<F16>(x)) | static_cast<uint32_t>(q4::to16<F16>(y)) << 16,
                   static_cast<uint32_t>(q4::to16<F16>(z)) | static_cast<uint32_t>(q4::to16<F16>(w)) << 16);
}

// A partial result in the workspace: per slot (two per worker) [rows][D] of O, then [rows][2] of (m, l).
__host__ __device__ __forceinline__ int64_t slot_floats(int rows, int d) { return static_cast<int64_t>(rows) * (d + 4); }

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
  int64_t unused;
  const int units = a.n_kv_heads * chunks;  // of a conversation
  const Deal deal = {count_pages(a, 0, unused) * units, workers};
  if (__any_sync(0xffffffffu, failed != 0)) return;
  const int64_t begin = deal.begin(worker), end = deal.begin(worker + 1);
  if (begin >= end) return;

  // the conversation of the first page
  int seq = 0;
  int64_t seq_at = 0;  // its first place in the line
  for (int base = 0;; base += 32) {
    const int s = base + lane;
    int64_t incl = s < a.n_seq ? static_cast<int64_t>(pages_of(tokens_of(a, s))) * units : 0;
    const int64_t own = incl;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, seq_at + incl > begin);
    if (past) {
      const int first = __ffs(past) - 1;
      seq = base + first;
      seq_at += __shfl_sync(0xffffffffu, incl - own, first);
      break;
    }
    seq_at += __shfl_sync(0xffffffffu, incl, 31);
    if (base + 32 >= a.n_seq) return;  // not reached: begin lies on the line
  }

  uint32_t copies = 0;  // issued by this warp so far: stage copies % kStages, phase copies / kStages
  int64_t at = begin;
  while (at < end) {
    // ---- one unit's segment
    int tokens = tokens_of(a, seq);
    while (tokens == 0) tokens = tokens_of(a, ++seq);
    const int n_pages = pages_of(tokens);
    const int unit = static_cast<int>((at - seq_at) / n_pages);
    const int64_t unit_at = seq_at + static_cast<int64_t>(unit) * n_pages;
    const int p0 = static_cast<int>(at - unit_at);
    const int p1 = static_cast<int>(min(static_cast<int64_t>(n_pages), end - unit_at));
    const int head = unit / chunks, row0 = (unit - head * chunks) * S::kRows;
    const int start = a.starts[seq], fresh = min(tokens - start, a.q_len);
    const int last_i = min((min(row0 + S::kRows, a.q_len * share) - 1) / share, fresh - 1);
    const int seen = row0 / share < fresh ? start + last_i + 1 : 0;
    const int full_below = start + row0 / share + 1;  // tokens below it are seen by every row
    const int32_t* table = a.blocks + static_cast<int64_t>(seq) * a.max_blocks;
    const int64_t page_stride = static_cast<int64_t>(a.n_kv_heads) * C::kBytes;
    uint8_t* cells = a.cells + static_cast<int64_t>(head) * C::kBytes;

    int ids = 0, ids_at = p0 - 32;
    auto page_id = [&](int p) {
      if (p >= ids_at + 32) {
        ids_at = p;
        ids = p + lane < p1 ? table[p + lane] : 0;
        if (static_cast<unsigned>(ids) >= static_cast<unsigned>(a.n_pages)) {
          record_error(a.status, kSiteQ4Attend + kErrBadDescriptor);
          ids = -1;
        }
      }
      return __shfl_sync(0xffffffffu, ids, p - ids_at);
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
    load_query<D, NT, F16>(a, seq, head, row0, share, start, fresh, q);
    State<D, NT> st;
    st.open = true;
    st.known = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      st.l[nt][0] = st.l[nt][1] = st.neg[nt][0] = st.neg[nt][1] = 0.f;
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) st.o[mt][nt][e] = 0.f;
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
      if (base + q4::kPage <= full_below) {
#pragma unroll 2
        for (int tile = 0; tile < q4::kPage / 16; ++tile)
          attend16<D, NT, F16, false>(page, tile, base + tile * 16, seen, q, st);
      } else {
        for (int tile = 0; tile < q4::kPage / 16 && base + tile * 16 < seen; ++tile)
          attend16<D, NT, F16, true>(page, tile, base + tile * 16, seen, q, st);
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
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = st.l[nt][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const int col = nt * 8 + 2 * t + c, r = row0 + col, i = r / share;
        if (r >= a.q_len * share || i >= fresh) continue;  // q4_combine_kernel writes the zeros behind the new tokens
        if (whole) {
          const float inv = sum != 0.f ? 1.f / sum : 0.f;
          const int64_t to =
              ((static_cast<int64_t>(seq) * a.q_len + i) * a.n_q_heads + head * share + r - i * share) * D + g * (D / 8);
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
            store_out4<F16>(a, to + k * 4, st.o[2 * k][nt][c] * inv, st.o[2 * k][nt][c + 2] * inv,
                            st.o[2 * k + 1][nt][c] * inv, st.o[2 * k + 1][nt][c + 2] * inv);
        } else {
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
            *reinterpret_cast<float4*>(slot + col * D + g * (D / 8) + k * 4) =
                make_float4(st.o[2 * k][nt][c], st.o[2 * k][nt][c + 2], st.o[2 * k + 1][nt][c], st.o[2 * k + 1][nt][c + 2]);
          if (g == 0) {
            slot[rows * D + col * 4] = st.neg[nt][c];
            slot[rows * D + col * 4 + 1] = sum;
          }
        }
      }
    at = unit_at + p1;
    if (at == seq_at + static_cast<int64_t>(units) * n_pages) {
      seq_at = at;
      ++seq;
    }
  }
}

// Joins the partial results of the units that several workers share, and writes the zeros of the rows behind the new
// tokens. One CTA per (query row of a KV head, KV head, conversation): D / 4 lanes of 4 dimensions, in kSlices
// slices over the unit's workers.
constexpr int kCombineThreads = 256;
template <int D, int NT, bool F16>
__global__ void __launch_bounds__(kCombineThreads)
q4_combine_kernel(const __grid_constant__ dkv_q4_attend_args a, int chunks, int workers) {
  constexpr int kLanes = D / 4, kSlices = kCombineThreads / kLanes;
  __shared__ int64_t line[2];
  __shared__ float4 part[kSlices][kLanes];
  __shared__ float2 stat[kSlices];
  const int share = a.n_q_heads / a.n_kv_heads;
  const int rows = min(8 * NT, a.q_len * share);
  const int r = blockIdx.x, head = blockIdx.y, seq = blockIdx.z;
  const int chunk = r / (8 * NT), col = r - chunk * 8 * NT, i = r / share;
  const int x = threadIdx.x % kLanes, slice = threadIdx.x / kLanes;
  const int tokens = tokens_of(a, seq), n_pages = pages_of(tokens);
  const int fresh = tokens == 0 ? 0 : min(tokens - a.starts[seq], a.q_len);
  if (threadIdx.x < 32) {
    int64_t before;
    const int64_t all = count_pages(a, seq, before);
    if (threadIdx.x == 0) line[0] = all, line[1] = before;
  }
  __syncthreads();
  const int units = a.n_kv_heads * chunks;
  const Deal deal = {line[0] * units, workers};
  const int64_t to = ((static_cast<int64_t>(seq) * a.q_len + i) * a.n_q_heads + head * share + r - i * share) * D + x * 4;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (i >= fresh || status_at_entry(a.status) != 0) {
    if (slice == 0) store_out4<F16>(a, to, 0.f, 0.f, 0.f, 0.f);
    return;
  }
  const int64_t unit_at = line[1] * units + static_cast<int64_t>(head * chunks + chunk) * n_pages;
  const int w0 = deal.owner(unit_at), w1 = deal.owner(unit_at + n_pages - 1);
  if (w0 == w1) return;  // one worker had the whole unit
  const int64_t stride = slot_floats(rows, D);
  const int second = deal.begin(w0) < unit_at ? 1 : 0;  // the unit is the last segment of w0, the first of the others
  // x2^-neg is what a slot's sums are relative to: the smallest neg is the largest reference
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  float den = 0.f, ref = INFINITY;
  for (int w = w0 + slice; w <= w1; w += kSlices) {
    if (deal.begin(w) == deal.begin(w + 1)) continue;  // fewer pages than workers
    const float* slot = a.workspace + (2 * w + (w == w0 ? second : 0)) * stride;
    const float2 s = *reinterpret_cast<const float2*>(slot + rows * D + col * 4);
    const float4 o = *reinterpret_cast<const float4*>(slot + col * D + x * 4);
    if (s.y == 0.f) continue;  // it saw no token of this row
    const float now = fminf(ref, s.x);
    const float keep = ref == INFINITY ? 0.f : exp2_fast(now - ref), add = exp2_fast(now - s.x);
    sum.x = fmaf(o.x, add, sum.x * keep);
    sum.y = fmaf(o.y, add, sum.y * keep);
    sum.z = fmaf(o.z, add, sum.z * keep);
    sum.w = fmaf(o.w, add, sum.w * keep);
    den = fmaf(s.y, add, den * keep);
    ref = now;
  }
  part[slice][x] = sum;
  if (x == 0) stat[slice] = make_float2(ref, den);
  __syncthreads();
  if (slice != 0) return;
  float top = INFINITY;
#pragma unroll
  for (int k = 0; k < kSlices; ++k) top = fminf(top, stat[k].x);
  sum = make_float4(0.f, 0.f, 0.f, 0.f);
  den = 0.f;
#pragma unroll
  for (int k = 0; k < kSlices; ++k) {
    const float f = stat[k].x == INFINITY ? 0.f : exp2_fast(top - stat[k].x);
    sum.x = fmaf(part[k][x].x, f, sum.x);
    sum.y = fmaf(part[k][x].y, f, sum.y);
    sum.z = fmaf(part[k][x].z, f, sum.z);
    sum.w = fmaf(part[k][x].w, f, sum.w);
    den = fmaf(stat[k].y, f, den);
  }
  const float inv = den != 0.f ? 1.f / den : 0.f;
  store_out4<F16>(a, to, sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

int rows_of(const dkv_q4_attend_args& a) { return a.q_len * (a.n_q_heads / a.n_kv_heads); }
int tiles_of(const dkv_q4_attend_args& a) { return rows_of(a) <= 8 ? 1 : 2; }  // of 8 query rows that a warp holds

int64_t floats_of(const dkv_q4_attend_args& a) {
  const int rows = rows_of(a), held = rows < 8 * tiles_of(a) ? rows : 8 * tiles_of(a);
  return 2 * static_cast<int64_t>(sm_count() * 3 * kWarps) * slot_floats(held, a.head_dim);
}

template <int D, int NT, bool F16>
int launch_decode(const dkv_q4_attend_args& a, int append, cudaStream_t stream) {
  const int rows = rows_of(a), chunks = (rows + 8 * NT - 1) / (8 * NT);
  if (static_cast<int64_t>(a.n_kv_heads) > 65535) return DKV_ERR_CONFIG;
  // At most one worker per page that there can be.
  const int64_t pages = static_cast<int64_t>((a.len_bound + q4::kPage - 1) / q4::kPage) * a.n_seq * a.n_kv_heads * chunks;
  const int most = sm_count() * Decode<D, NT>::kBlocksPerSm;
  const int ctas = pages < most ? (pages < 1 ? 1 : static_cast<int>(pages)) : most;
  const int workers = ctas * kWarps;
  auto kernel = q4_decode_kernel<D, NT, F16>;
  constexpr int bytes = Decode<D, NT>::kBytes;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return DKV_ERR_CUDA;
  kernel<<<ctas, kThreads, bytes, stream>>>(a, chunks, workers, append);
  if (cudaGetLastError() != cudaSuccess) return DKV_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows, a.n_kv_heads, a.n_seq);
  cfg.blockDim = dim3(kCombineThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, q4_combine_kernel<D, NT, F16>, a, chunks, workers) == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
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
  return a->n_seq == 0 || a->q_len == 0 ? 0 : dkv::floats_of(*a);
}

int dkv_q4_attend(const dkv_q4_attend_args* a, void* stream) {
  if (a == nullptr || a->cells == nullptr || a->blocks == nullptr || a->lengths == nullptr || a->starts == nullptr ||
      a->query == nullptr || a->out == nullptr || a->status == nullptr)
    return DKV_ERR_ARGS;
  const int rc = dkv::check_sizes(a);
  if (rc != DKV_OK) return rc;
  if ((a->key == nullptr) != (a->value == nullptr) || (a->key != nullptr && a->slots == nullptr)) return DKV_ERR_ARGS;
  if (reinterpret_cast<uintptr_t>(a->cells) % 16 || reinterpret_cast<uintptr_t>(a->query) % 16 ||
      reinterpret_cast<uintptr_t>(a->key) % 16 || reinterpret_cast<uintptr_t>(a->value) % 16 ||
      reinterpret_cast<uintptr_t>(a->out) % 16 || reinterpret_cast<uintptr_t>(a->workspace) % 16)
    return DKV_ERR_ARGS;
  for (int k = 0; k < 3; ++k)
    if (a->q_stride[k] % 8 || (a->key != nullptr && (a->k_stride[k] % 8 || a->v_stride[k] % 8))) return DKV_ERR_ARGS;
  if (a->n_seq == 0 || a->q_len == 0) return DKV_OK;
  if (a->workspace == nullptr || a->workspace_floats < dkv::floats_of(*a)) return DKV_ERR_SCRATCH;
  const int nt = dkv::tiles_of(*a);
  int append = a->key != nullptr;
  if (append && dkv::rows_of(*a) > 8 * nt) {
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
#define DKV_Q4_DECODE(D, NT) \
  (a->fp16 ? dkv::launch_decode<D, NT, true>(*a, append, st) : dkv::launch_decode<D, NT, false>(*a, append, st))
  if (a->head_dim == 128) return nt == 1 ? DKV_Q4_DECODE(128, 1) : DKV_Q4_DECODE(128, 2);
  return nt == 1 ? DKV_Q4_DECODE(64, 1) : DKV_Q4_DECODE(64, 2);
#undef DKV_Q4_DECODE
}

}  // extern "C"
