// q4_attend.cu — causal attention of new tokens' queries over the paged 4-bit cache (dkv_q4_attend).
//
// With key value k_d = low_g + scale_g * c_d (g = d / 64), a score splits into
//   q . k = sum_g scale_g * (sum_{d in g} q_d c_d) + sum_g low_g * (sum_{d in g} q_d):
// the product runs over the codes themselves, which float16 holds exactly, and the key's rounding is the
// cache's alone. Values enter as float16(low + scale * c), one rounding of at most 2^-11 relative; probabilities
// as float16 of 2^7 * exp(score - m) with m within 2^8 of the running maximum, so that a token down to 2^-21 of the
// largest keeps 11 bits (sums over a long context of small probabilities do not vanish).
//
// q4_decode_kernel: few query rows per KV head (one token, or a short draft). Bound by the cells' bytes. A page of
// one KV head is one contiguous block: one bulk copy by a producer warp into a ring, four warps take 16 tokens
// of it each. A warp contracts tokens as the 16 rows of m16n8k16 and query rows as its 8 columns (few rows are the
// rule: 3 or 4 heads share a KV head), S^T = C Q^T, then O^T = V^T P^T; P^T in the layout of the second product is
// one 8 x 8 transpose per 8 tokens (movmatrix). A code pair of a word is a float16 pair after ONE mask: the 4 bits
// are a subnormal c * 2^-24 (or 16 times that, from the odd nibbles, against q / 16), and the power of two goes
// into the score's factor. The CTAs of a cluster share one (conversation, KV head, row chunk): pages dealt in turn,
// partial (m, l, O) merged over distributed shared memory, so one launch does it all and needs no workspace.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dkv_ptx.cuh"
#include "q4_cells.cuh"

namespace dkv {
namespace {

using q4::Cells;
constexpr int kWarps = 4;                        // consumer warps: 16 tokens of a page each
constexpr int kDecodeThreads = (kWarps + 1) * 32;
constexpr int kStages = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBias = 7.f;                     // probabilities are scaled by 2^7
constexpr float kSlack = 8.f;                    // the reference maximum may lag by 2^8: 2^(7 + 8) < 65504

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

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }

template <bool F16>
__device__ __forceinline__ float load16(uint16_t v) {
  return F16 ? __half2float(__ushort_as_half(v)) : __bfloat162float(__ushort_as_bfloat16(v));
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int D, int NT>
struct DecodeShared {
  static constexpr int kRows = 8 * NT;
  static constexpr int kRing = kStages * Cells<D>::kBytes;
  static constexpr int kMerge = kWarps * kRows * D * 4;
  static constexpr int kBody = kRing > kMerge ? kRing : kMerge;  // the ring, then the warps' O
  static constexpr int kStats = kBody;                           // [kWarps + 1][kRows][2] m, l; the last: the CTA's
  static constexpr int kBars = kStats + (kWarps + 1) * kRows * 8;
  static constexpr int kBytes = kBars + 2 * kStages * 8;
};

template <int D, int NT, bool F16>
__global__ void __launch_bounds__(kDecodeThreads)
q4_decode_kernel(const dkv_q4_attend_args a, int chunks) {
  using C = Cells<D>;
  using S = DecodeShared<D, NT>;
  constexpr int kRows = S::kRows;
  constexpr int kGroups = C::kGroups;
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* empty = full + kStages;
  float* stats = reinterpret_cast<float*>(smem + S::kStats);

  const int splits = gridDim.x, rank = blockIdx.x;
  const int head = blockIdx.y / chunks, row0 = (blockIdx.y - head * chunks) * kRows, seq = blockIdx.z;
  const int share = a.n_q_heads / a.n_kv_heads;
  const int lane = threadIdx.x & 31, warp = warp_id();
  const int g = lane >> 2, t = lane & 3;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
    fence_barrier_init();
  }
  // A CTA that finds the status word set takes no pages, but stays for the cluster's merge.
  const bool failed = cta_failed_at_entry(a.status);

  const int start = max(a.starts[seq], 0);
  const int len = min(a.lengths[seq], a.max_blocks * q4::kPage);
  const int fresh = min(len - start, a.q_len);
  // Tokens that the last row of the chunk sees (0: no row of it is a new token's).
  const int last_i = min((min(row0 + kRows, a.q_len * share) - 1) / share, fresh - 1);
  const int seen = (failed || row0 / share >= fresh) ? 0 : start + last_i + 1;
  const int n_pages = (seen + q4::kPage - 1) / q4::kPage;
  const int mine = n_pages > rank ? (n_pages - rank + splits - 1) / splits : 0;

  float o[D / 16][NT][4];
  float l[NT][2], m[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      l[nt][c] = 0.f;
      m[nt][c] = -INFINITY;
    }
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[mt][nt][e] = 0.f;
  }

  if (warp == kWarps) {
    // ---- producer: one bulk copy per page
    const int32_t* row = a.blocks + static_cast<int64_t>(seq) * a.max_blocks;
    const int64_t page_stride = static_cast<int64_t>(a.n_kv_heads) * C::kBytes;
    int ids = 0, issued = 0;
    for (int k = 0; k < mine; ++k) {
      if ((k & 31) == 0) ids = k + lane < mine ? row[rank + (k + lane) * splits] : 0;
      int page = __shfl_sync(0xffffffffu, ids, k & 31);
      if (page < 0 || page >= a.n_pages) {  // recorded, and a page that exists read in its place
        if (lane == 0) record_error(a.status, kSiteQ4Attend + kErrBadDescriptor);
        page = 0;
      }
      const int stage = k % kStages;
      if (k >= kStages && !warp_wait(&empty[stage], ((k / kStages) - 1) & 1, a.status, kSiteQ4Attend + kErrWaitEmpty, nullptr))
        break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[stage], C::kBytes);
        bulk_load(smem + stage * C::kBytes, a.cells + page * page_stride + static_cast<int64_t>(head) * C::kBytes,
                  C::kBytes, &full[stage]);
      }
      __syncwarp();
      issued = k + 1;
    }
    // No copy of this CTA is in flight when it leaves, also when a consumer has given up.
    for (int k = max(0, issued - kStages); k < issued; ++k)
      warp_wait(&full[k % kStages], (k / kStages) & 1, a.status, kSiteQ4Attend + kErrWaitDrain, nullptr);
  } else if (mine > 0) {
    // ---- the query as the second operand, its sums per group, and the score's factors
    uint32_t qf[D / 16][NT][2];
    float factor[NT][2], qsum[NT][2][kGroups];
    int limit[NT][2];
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
            const float v = load16<F16>(static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1))));
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
            qf[gr * 4 + w * 2 + odd][nt][0] = pack_half2(v[0] * f, v[4] * f);
            qf[gr * 4 + w * 2 + odd][nt][1] = pack_half2(v[2] * f, v[6] * f);
          }
      const float scale = a.scaling * kLog2e;
      const float fac = scale * (16777216.f / up);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = (2 * t + c) * 4;
        factor[nt][c] = __shfl_sync(0xffffffffu, fac, from);
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) qsum[nt][c][gr] = __shfl_sync(0xffffffffu, sum[gr] * scale, from);
        const int rc = row0 + nt * 8 + 2 * t + c, ic = rc / share;
        limit[nt][c] = (rc < a.q_len * share && ic < fresh) ? start + ic + 1 : 0;
      }
    }
    const int full_below = start + row0 / share + 1;  // tokens below this are seen by every row of the chunk

    for (int k = 0; k < mine; ++k) {
      const int stage = k % kStages;
      if (!warp_wait(&full[stage], (k / kStages) & 1, a.status, kSiteQ4Attend + kErrWaitCodes, nullptr)) break;
      const uint8_t* page = smem + stage * C::kBytes;
      const int base = (rank + k * splits) * q4::kPage + warp * 16;  // first token of this warp's 16
      if (base < seen) {
        // ---- scores of 16 tokens: rows g and g + 8
        float acc[kGroups][NT][4];
        {
          const uint8_t* kr = page + C::kKeyCodes + (warp * 16 + g) * (D / 2) + t * (D / 8);
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
                  mma16816(acc[gr][nt], u & mask, v & mask, u8 & mask, v8 & mask, qf[gr * 4 + w * 2 + odd][nt][0],
                           qf[gr * 4 + w * 2 + odd][nt][1]);
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
                as_half2(*reinterpret_cast<const uint32_t*>(page + C::key_head(warp * 16 + g + 8 * h, gr))));
            ks[h][gr] = f.x;
            kl[h][gr] = f.y;
          }
        const bool edge = base + 16 > full_below;  // some row does not see some token
        float p[NT][4];
        bool rise = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int h = e >> 1, c = e & 1;
            float dot = 0.f, off = 0.f;
#pragma unroll
            for (int gr = 0; gr < kGroups; ++gr) {
              dot = fmaf(ks[h][gr], acc[gr][nt][e], dot);
              off = fmaf(kl[h][gr], qsum[nt][c][gr], off);
            }
            float s = fmaf(dot, factor[nt][c], off);
            if (edge && base + g + 8 * h >= limit[nt][c]) s = -INFINITY;
            p[nt][e] = s;
            rise = rise || s > m[nt][c] + kSlack;
          }
        if (__any_sync(0xffffffffu, rise)) {
          // ---- a score above the reference maximum's slack: new maxima, and what is summed so far scaled down
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float f[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float top = fmaxf(p[nt][c], p[nt][c + 2]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
              top = fmaxf(top, m[nt][c]);
              f[c] = top > m[nt][c] ? exp2_fast(m[nt][c] - top) : 1.f;
              m[nt][c] = top;
              l[nt][c] *= f[c];
            }
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[mt][nt][e] *= f[e & 1];
          }
        }
        uint32_t pf[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float ref = m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1] - kBias;
            p[nt][e] = exp2_fast(p[nt][e] - ref);
            l[nt][e & 1] += p[nt][e];
          }
          pf[nt][0] = transpose8(pack_half2(p[nt][0], p[nt][1]));
          pf[nt][1] = transpose8(pack_half2(p[nt][2], p[nt][3]));
        }
        // ---- values: token pairs t and t + 4 of the 16
        uint32_t v[2][D / 32];
        __half2 vs[2], vl[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int pair = warp * 8 + t + 4 * h;
          const uint8_t* vr = page + C::value_piece(pair, g);
          if constexpr (D == 128) {
            const uint4 u = *reinterpret_cast<const uint4*>(vr);
            v[h][0] = u.x, v[h][1] = u.y, v[h][2] = u.z, v[h][3] = u.w;
          } else {
            const uint2 u = *reinterpret_cast<const uint2*>(vr);
            v[h][0] = u.x, v[h][1] = u.y;
          }
          uint2 hd = *reinterpret_cast<const uint2*>(page + C::value_head(pair, kGroups == 2 ? g >> 2 : 0));
          if (base + 16 > seen) {
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
            for (int nt = 0; nt < NT; ++nt)
              mma16816(o[i * 2 + b][nt], x[0][0], x[0][1], x[1][0], x[1][1], pf[nt][0], pf[nt][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
    }
  }
  __syncwarp();
  __syncthreads();  // the ring is free

  // ---- merge of the warps, then of the cluster
  float* body = reinterpret_cast<float*>(smem);
  if (warp < kWarps) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[nt][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const int col = nt * 8 + 2 * t + c;
        if (g == 0) {
          stats[(warp * kRows + col) * 2] = m[nt][c];
          stats[(warp * kRows + col) * 2 + 1] = sum;
        }
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
          *reinterpret_cast<float4*>(body + (warp * kRows + col) * D + g * (D / 8) + i * 4) =
              make_float4(o[2 * i][nt][c], o[2 * i][nt][c + 2], o[2 * i + 1][nt][c], o[2 * i + 1][nt][c + 2]);
      }
  }
  __syncthreads();
  float* mine_stats = stats + kWarps * kRows * 2;
  for (int e = threadIdx.x; e < kRows * D; e += kDecodeThreads) {
    const int col = e / D;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stats[(w * kRows + col) * 2]);
    float sum = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = stats[(w * kRows + col) * 2];
      const float f = mw == -INFINITY ? 0.f : exp2_fast(mw - top);
      sum = fmaf(f, body[w * kRows * D + e], sum);
      den = fmaf(f, stats[(w * kRows + col) * 2 + 1], den);
    }
    body[e] = sum;
    if (e % D == 0) {
      mine_stats[col * 2] = top;
      mine_stats[col * 2 + 1] = den;
    }
  }
  const int rows_here = min(kRows, a.q_len * share - row0);
  __syncwarp();
  if (splits > 1) cluster_sync_all();
  else __syncthreads();
  const uint32_t body_s = smem_u32(body), stats_s = smem_u32(mine_stats);
  for (int e = threadIdx.x + rank * kDecodeThreads; e < rows_here * D; e += kDecodeThreads * splits) {
    const int col = e / D;
    float sum, den;
    if (splits == 1) {
      sum = body[e];
      den = mine_stats[col * 2 + 1];
    } else {
      float top = -INFINITY;
      sum = den = 0.f;
      for (int c = 0; c < splits; ++c) {
        const float mc = ld_cluster_f32(mapa_shared(stats_s + col * 8, c));
        const float f_new = mc > top ? exp2_fast(top - mc) : 1.f;  // of what is summed so far
        const float f_c = mc > top ? 1.f : mc == -INFINITY ? 0.f : exp2_fast(mc - top);
        top = fmaxf(top, mc);
        sum = fmaf(f_c, ld_cluster_f32(mapa_shared(body_s + e * 4, c)), sum * f_new);
        den = fmaf(f_c, ld_cluster_f32(mapa_shared(stats_s + col * 8 + 4, c)), den * f_new);
      }
    }
    const int r = row0 + col, i = r / share;
    const float y = den != 0.f && i < fresh ? sum / den : 0.f;  // a row behind the last new token is zero
    const int64_t at = ((static_cast<int64_t>(seq) * a.q_len + i) * a.n_q_heads + head * share + r - i * share) * D + e % D;
    if (a.out_f32)
      static_cast<float*>(a.out)[at] = y;
    else if (F16)
      static_cast<__half*>(a.out)[at] = __float2half_rn(y);
    else
      static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
  }
  __syncwarp();
  if (splits > 1) cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

template <int D, int NT, bool F16>
int launch_decode(const dkv_q4_attend_args& a, int splits, int chunks, cudaStream_t stream) {
  auto kernel = q4_decode_kernel<D, NT, F16>;
  constexpr int bytes = DecodeShared<D, NT>::kBytes;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return DKV_ERR_CUDA;
  if (splits > 8 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return DKV_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits, a.n_kv_heads * chunks, a.n_seq);
  cfg.blockDim = dim3(kDecodeThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, chunks) == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
}

}  // namespace
}  // namespace dkv

extern "C" int dkv_q4_attend(const dkv_q4_attend_args* a, void* stream) {
  if (a == nullptr || a->cells == nullptr || a->blocks == nullptr || a->lengths == nullptr || a->starts == nullptr ||
      a->query == nullptr || a->out == nullptr || a->status == nullptr)
    return DKV_ERR_ARGS;
  if (a->n_pages < 1 || a->max_blocks < 1 || a->n_seq < 0 || a->q_len < 0 || a->n_kv_heads < 1 || a->n_q_heads < 1 ||
      a->n_q_heads % a->n_kv_heads != 0)
    return DKV_ERR_ARGS;
  if (a->head_dim != 64 && a->head_dim != 128) return DKV_ERR_CONFIG;
  if (reinterpret_cast<uintptr_t>(a->cells) % 16 || reinterpret_cast<uintptr_t>(a->query) % 16) return DKV_ERR_ARGS;
  for (int k = 0; k < 3; ++k)
    if (a->q_stride[k] % 8) return DKV_ERR_ARGS;
  if (static_cast<int64_t>(a->n_pages) * dkv::q4::kPage > INT32_MAX ||
      static_cast<int64_t>(a->max_blocks) * dkv::q4::kPage > INT32_MAX || a->n_seq > 65535)
    return DKV_ERR_CONFIG;
  if (a->n_seq == 0 || a->q_len == 0) return DKV_OK;
  const int64_t rows = static_cast<int64_t>(a->q_len) * (a->n_q_heads / a->n_kv_heads);
  const int nt = rows <= 8 ? 1 : 2;
  const int64_t chunks = (rows + 8 * nt - 1) / (8 * nt);
  if (chunks * a->n_kv_heads > 65535) return DKV_ERR_CONFIG;
  // CTAs of a cluster: enough of them in all to fill the GPU several times over, none without a page.
  const int64_t units = static_cast<int64_t>(a->n_seq) * a->n_kv_heads * chunks;
  const int pages = (a->len_bound + dkv::q4::kPage - 1) / dkv::q4::kPage;
  int splits = 1;
  while (splits < 16 && units * splits < 148 * 6 && splits * 2 <= pages) splits *= 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int c = static_cast<int>(chunks);
#define DKV_Q4_DECODE(D, NT) \
  (a->fp16 ? dkv::launch_decode<D, NT, true>(*a, splits, c, st) : dkv::launch_decode<D, NT, false>(*a, splits, c, st))
  if (a->head_dim == 128) return nt == 1 ? DKV_Q4_DECODE(128, 1) : DKV_Q4_DECODE(128, 2);
  return nt == 1 ? DKV_Q4_DECODE(64, 1) : DKV_Q4_DECODE(64, 2);
#undef DKV_Q4_DECODE
}
