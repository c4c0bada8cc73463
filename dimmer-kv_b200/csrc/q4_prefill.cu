// q4_prefill.cu — causal attention over the paged 4-bit cache for many query rows per KV head (a question, a prompt's
// chunk): dkv_q4_attend's matrix-product form, on tcgen05.
//
// A CTA has two tiles of 128 query rows (the rows of a KV head's query heads, token after token), which use the same
// unpacked keys and values, and two buffers of scores for each: a step is one page, 64 tokens, and a tile's next scores
// are made while the softmax of the last is under way. At head_dim 128 a step of both tiles takes at least 1024 cycles of
// the SM's exponential units, 1024 of its tensor core and about 1300 of its shared memory's bandwidth (of that of
// float16 caches, below, 2048 and 2500); measured are 2300 for bfloat16, where the softmax's latencies, two warps
// to a scheduler, are the bound, and 3100 for float16, where the products are. Steps of twice as many tokens with one
// buffer, of fewer and wider products, took 5500 and 8000.
//
//   warps 0-3, 4-7   softmax of the first and the second tile, one row per thread: scores from TMEM, probabilities
//                    back into TMEM (over the scores they come from), where the second product takes them
//   warps 8-15       unpack a page, four threads per token: the keys into a float16 tile with the 128-byte swizzle, the
//                    values into one whose rows are those of the second product's contraction
//   warps 16, 17     issue the products of a tile each (per step the next Q K, then P V; one warp for both tiles, which
//                    waits for each in turn, took 299 us where two take 224)
//   warp 18          issues the copies of the pages
//
// TMEM: two score buffers of 64 columns and an output per tile, 512 columns. The rows' references (running maxima) lag by
// up to 2^8, so that outputs are scaled down in TMEM (once the products on them are complete) only when a row's maximum
// has grown past that.
//
// Keys and values are rounded to float16 (2^-11 at most of each), probabilities likewise. For float16 caches, whose
// outputs show that, what the rounding of keys lacks forms a second tile, and what that of probabilities lacks a second
// operand beside the first (each 32 columns of scores become 16 of either), that go through second products. The values
// stay one float16 number: a key's rounding moves its token's weight in every dimension alike, those of the values are of
// either sign and independent, and their sum shows less (the chunk below is off by 2.8e-4 of its values, 2.1e-4 in float32
// arithmetic and rounded once), for a third product of the tensor core's bound that is already doubled.
//
// The steps of all (conversation, KV head, 256-row block) units form one line that is cut evenly over one CTA per
// SM; blocks that several CTAs share leave partial results in the workspace, which q4_prefill_combine_kernel joins.
//
// 24 / 8 heads of 128: 4 x 512 tokens over 2K to 8K, float16, 203 us with the store and the joins, 64 tokens over 32K,
// bfloat16, 61 us.
#include "q4_attend.cuh"

namespace dkv {
namespace q4 {
namespace {

constexpr int kStep = kPage;         // tokens of a step
constexpr int kRows = 128;           // query rows of a tile
constexpr int kBlock = 2 * kRows;    // of a unit
constexpr int kSoftWarps = 8;

constexpr int kUnpackWarps = 8;
constexpr int kMmaWarp = kSoftWarps + kUnpackWarps, kCopyWarp = kMmaWarp + 2;
constexpr int kThreads = (kMmaWarp + 4) * 32;  // whole warpgroups: registers are dealt to these
// Registers per thread: 96 at launch (5 warpgroups, 480 in all), then 2 x 128 + 2 x 72 + 80 = 480.
constexpr int kSoftRegs = 128, kUnpackRegs = 72, kIssueRegs = 80;

template <int D, bool F16>
struct Shared {
  using C = Cells<D>;
  static constexpr int kQPart = kRows * 128, kPart = kStep * 128;  // 64 dimensions of 128 rows, of 64 tokens, in float16
  static constexpr int kQTile = D / 64 * kQPart, kTile = D / 64 * kPart;
  static constexpr int kRawStages = 4, kStages = 2;
  static constexpr int kQ = 0;                        // two tiles
  static constexpr int kK = kQ + 2 * kQTile;          // kStages of each
  static constexpr int kV = kK + kStages * kTile;
  static constexpr int kKLow = kV + kStages * kTile;  // what the rounding of keys lacks (float16 caches)
  static constexpr int kRaw = kKLow + (F16 ? kStages * kTile : 0);
  static constexpr int kBars = kRaw + kRawStages * C::kBytes;
  static constexpr int kNumBars = 2 * kRawStages + 4 * kStages + 2 + 4 + 4 + 2 + 2 + 2;
  static constexpr int kBytes = kBars + kNumBars * 8 + 16;
  static constexpr int kAlloc = kBytes + 1024;        // the tiles begin on a 1024-byte boundary
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// After tmem_ld_wait: no use of the registers may be scheduled before it.
__device__ __forceinline__ void tmem_fence32(uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] * B[smem]: A's rows are TMEM lanes, two float16 of the contraction per 32-bit column.
__device__ __forceinline__ void mma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// One lane of a warp whose lanes are together, the same one every time; a branch on it keeps the warp's uniform registers,
// in which tcgen05 takes its operands, where one on the lane's number moves every operand there again.
__device__ __forceinline__ bool elect_lane() {
  uint32_t lead;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}\n" : "=r"(lead));
  return lead != 0;
}

// ---------------------------------------------------------------- the line of steps
struct Seq {
  int start, fresh, rows, blocks;  // rows: new tokens' rows of a KV head
};
__device__ __forceinline__ Seq seq_of(const dkv_q4_attend_args& a, int s, int share) {
  Seq q;
  const int tokens = tokens_of(a, s);
  q.start = a.starts[s];
  q.fresh = tokens == 0 ? 0 : min(tokens - q.start, a.q_len);
  q.rows = q.fresh * share;
  q.blocks = (q.rows + kBlock - 1) / kBlock;
  return q;
}
// Tokens that the rows of block b see, and steps to go through them.
__device__ __forceinline__ int seen_by(const Seq& q, int b, int share) {
  return q.start + min(((b + 1) * kBlock - 1) / share, q.fresh - 1) + 1;
}
__device__ __forceinline__ int steps_of(const Seq& q, int b, int share) {
  return (seen_by(q, b, share) + kStep - 1) / kStep;
}
__device__ __forceinline__ int64_t seq_steps(const Seq& q, int share) {  // of one KV head
  int64_t n = 0;
  for (int b = 0; b < q.blocks; ++b) n += steps_of(q, b, share);
  return n;
}

__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

int slot_rows_of(const dkv_q4_attend_args& a) { return rows_of(a) < kBlock ? rows_of(a) : kBlock; }

__device__ __forceinline__ int64_t unit_of(const dkv_q4_attend_args& a, int seq, int head, int block) {
  const int blocks = (a.q_len * (a.n_q_heads / a.n_kv_heads) + kBlock - 1) / kBlock;
  return (static_cast<int64_t>(seq) * a.n_kv_heads + head) * blocks + block;
}

// Where a CTA's piece of the line begins and ends, and the step of `begin`.
struct Start {
  int64_t begin, end;
  Seq q;
  int seq, head, block, first;
};
// One warp, all lanes alike: 64-bit divisions and two rounds of loads, of which every role's warp would take its share of
// the SM's time.
__device__ __forceinline__ Start find_start(const dkv_q4_attend_args& a, int share, int workers) {
  const int lane = threadIdx.x & 31;
  auto steps_at = [&](int s) { return s < a.n_seq ? seq_steps(seq_of(a, s, share), share) * a.n_kv_heads : 0; };
  const int64_t own0 = steps_at(lane);  // the first 32 conversations'
  int64_t total = warp_sum64(own0);
  for (int base = 32; base < a.n_seq; base += 32) total += warp_sum64(steps_at(base + lane));
  const DealOf<false> deal(total, workers);
  Start at = {};
  if (static_cast<int>(blockIdx.x) >= deal.workers) return at;
  at.begin = deal.begin(blockIdx.x);
  at.end = deal.begin(blockIdx.x + 1);
  int64_t line = 0;
  for (int base = 0; base < a.n_seq; base += 32) {  // the conversation of `begin`
    const int64_t own = base == 0 ? own0 : steps_at(base + lane);
    int64_t incl = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, line + incl > at.begin);
    if (past) {
      const int l = __ffs(past) - 1;
      at.seq = base + l;
      at.q = seq_of(a, at.seq, share);
      int64_t rest = at.begin - line - __shfl_sync(0xffffffffu, incl - own, l);
      const int64_t per_head = seq_steps(at.q, share);
      at.head = static_cast<int>(divide<false>(rest, per_head));
      rest -= at.head * per_head;
      while (rest >= steps_of(at.q, at.block, share)) rest -= steps_of(at.q, at.block++, share);
      at.first = static_cast<int>(rest);
      return at;
    }
    line += __shfl_sync(0xffffffffu, incl, 31);
  }
  at.end = at.begin;  // not reached: begin lies on the line
  return at;
}

// A CTA's piece of the line, unit by unit. Every warp goes through it on its own (all lanes alike).
struct Walk {
  const dkv_q4_attend_args& a;
  int share;
  int64_t at, end;      // places left
  int seq, head, block;
  Seq q;
  int first, last, steps;  // this unit's steps [first, last) of `steps`
  bool opened;

  __device__ __forceinline__ Walk(const dkv_q4_attend_args& a_, int share_, const Start& s)
      : a(a_), share(share_), at(s.begin), end(s.end), q(s.q), seq(s.seq), head(s.head), block(s.block), first(s.first),
        opened(false) {}
  // The next unit; false behind the last.
  __device__ __forceinline__ bool next() {
    if (opened) {
      first = 0;
      if (++block == q.blocks) {
        block = 0;
        if (++head == a.n_kv_heads) {
          head = 0;
          if (at < end) {
            do q = seq_of(a, ++seq, share);
            while (q.blocks == 0);
          }
        }
      }
    }
    opened = true;
    if (at >= end) return false;
    steps = steps_of(q, block, share);
    last = static_cast<int>(min(static_cast<int64_t>(steps), first + (end - at)));
    at += last - first;
    return true;
  }
  __device__ __forceinline__ bool whole() const { return first == 0 && last == steps; }
  __device__ __forceinline__ bool two() const { return q.rows - block * kBlock > kRows; }  // the second tile has rows
};

// ---------------------------------------------------------------- unpacking
__device__ __forceinline__ uint64_t wide2(__half2 h) {
  const float2 f = __half22float2(h);
  return f32x2_pack(__float_as_uint(f.x), __float_as_uint(f.y));
}
// What the float16 pair h lacks to x.
__device__ __forceinline__ uint32_t lack2(uint64_t x, __half2 h) {
  const uint64_t d = fma_f32x2(wide2(h), f32x2_pack(0xbf800000u, 0xbf800000u), x);
  return pack_half2(__uint_as_float(static_cast<uint32_t>(d)), __uint_as_float(static_cast<uint32_t>(d >> 32)));
}
// By the exponent's bits: a nibble n in the low bits of the float16 0x6400 makes 1024 + n, four bits higher 1024 + 16 n.
// Eight codes (nibbles of w) to eight float16 values scale * c + low in the order 0 4 1 5 2 6 3 7, each rounded once; with
// LOW also what the rounding lacks.
template <bool LOW>
__device__ __forceinline__ uint4 unpack8(uint32_t w, __half2 scale, __half2 low, uint4& lack) {
  const __half2 k1024 = as_half2(0x64006400u), k16th = as_half2(0x2c002c00u), k64 = as_half2(0xd400d400u);
  uint32_t v[4], r[4];
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const uint32_t u = b ? w >> 8 : w;
    const __half2 even = __hsub2(as_half2((u & 0x000f000fu) | 0x64006400u), k1024);
    const __half2 odd = __hfma2(as_half2((u & 0x00f000f0u) | 0x64006400u), k16th, k64);
    const __half2 x = __hfma2(even, scale, low), y = __hfma2(odd, scale, low);
    v[2 * b] = as_u32(x);
    v[2 * b + 1] = as_u32(y);
    if constexpr (LOW) {
      const uint32_t s = __float_as_uint(__low2float(scale)), l = __float_as_uint(__low2float(low));
      const uint64_t s2 = f32x2_pack(s, s), l2 = f32x2_pack(l, l);
      r[2 * b] = lack2(fma_f32x2(wide2(even), s2, l2), x);
      r[2 * b + 1] = lack2(fma_f32x2(wide2(odd), s2, l2), y);
    }
  }
  if constexpr (LOW) lack = make_uint4(r[0], r[1], r[2], r[3]);
  return make_uint4(v[0], v[1], v[2], v[3]);
}
// Place p of a chunk of 8 holds dimension kOrder[p].
__device__ constexpr int kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 1)
q4_prefill_kernel(const __grid_constant__ dkv_q4_attend_args a, int workers, int slot_rows) {
  using S = Shared<D, F16>;
  using C = Cells<D>;
  constexpr int kGroups = C::kGroups;
  extern __shared__ uint8_t smem_raw[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint8_t* smem = smem_raw + (1024 - smem_u32(smem_raw) % 1024) % 1024;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* raw_full = bars;                     // bulk copies of a step's pages
  uint64_t* raw_free = raw_full + S::kRawStages; // unpacked
  uint64_t* k_full = raw_free + S::kRawStages;   // [kStages] each
  uint64_t* v_full = k_full + S::kStages;
  uint64_t* k_free = v_full + S::kStages;        // products that read the tile are complete
  uint64_t* v_free = k_free + S::kStages;
  uint64_t* q_full = v_free + S::kStages;        // [2], by tile
  uint64_t* s_full = q_full + 2;                 // [tile][buffer]: scores complete
  uint64_t* p_full = s_full + 4;                 // [tile][buffer]: probabilities in TMEM
  uint64_t* o_done = p_full + 4;                 // [tile]: a step's product on the output complete
  uint64_t* o_full = o_done + 2;                 // [tile]: a unit's output complete
  uint64_t* drain = o_full + 2;                  // [tile]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + S::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = threadIdx.x & 31;
  const int share = a.n_q_heads / a.n_kv_heads;
  __shared__ Start start;
  if (warp == 1) {
    const Start at = find_start(a, share, workers);
    if (lane == 0) start = at;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kRawStages; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_free[i], kUnpackWarps);
    }
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&k_full[i], kUnpackWarps);
      mbar_init(&v_full[i], kUnpackWarps);
      mbar_init(&k_free[i], 2);
      mbar_init(&v_free[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_full[i], 1);
      mbar_init(&drain[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the new tokens' cells; what is above reads lengths alone
  const bool failed = cta_failed_at_entry(a.status);  // a barrier of the CTA
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int64_t begin = start.begin, end = failed ? begin : start.end;
  // scores of tile i, buffer b: columns 128 i + 64 b .. (its probabilities in their place); outputs: columns 256 + 128 i ..
  if (begin < end) {
    // Every warp of the warpgroups gives or takes its registers at the head of its role (the compiler allots the roles'
    // code by that), the two without a role as well.
    if (warp < kSoftWarps) {
      setmaxnreg_inc<kSoftRegs>();
      Walk walk(a, share, start);
      // ------------------------------------------------------------ softmax
      const int tile = warp >> 2, row_in_tile = (warp & 3) * 32 + lane;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t o_at = tmem + lanes + 256 + tile * 128;
      uint32_t count = 0, units = 0;  // this tile's steps and units so far
      bool ok = true;
      int64_t place = begin;
      while (ok && walk.next()) {
        const int64_t unit_begin = place;
        place += walk.last - walk.first;
        if (threadIdx.x == 0)
          record_unit(unit_record(a, workers, slot_rows, unit_of(a, walk.seq, walk.head, walk.block)), blockIdx.x,
                      unit_begin != begin, walk.first == 0, walk.last == walk.steps);
        if (tile == 1 && !walk.two()) continue;
        const Seq& q = walk.q;
        const int row0 = walk.block * kBlock + tile * kRows, r = row0 + row_in_tile, i = r / share;
        const bool real = r < q.rows;
        // ---- the row into shared memory, by a power of two that brings its largest element to [2^13, 2^14)
        float factor;
        {
          // (rows behind the last load the first element's, and count as zeros)
          const int64_t src =
              real ? walk.seq * a.q_stride[0] + (walk.head * share + r - i * share) * a.q_stride[1] + i * a.q_stride[2] : 0;
          const unsigned reals = __ballot_sync(0xffffffffu, real);
          uint8_t* own = smem + S::kQ + tile * S::kQTile;
          uint4 raw[D / 8];
          constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;  // lanes that load a row, rows of a load: all under way at once
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            const int from = c * kAtOnce + lane / kLanes;
            const int64_t at = __shfl_sync(0xffffffffu, src, from);
            raw[c] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.query) + at + lane % kLanes * 8);
          }
          __syncwarp();
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            const int from = c * kAtOnce + lane / kLanes, chunk = lane % kLanes;
            *reinterpret_cast<uint4*>(own + (chunk >> 3) * S::kQPart + sw128_offset(row_in_tile - lane + from, chunk & 7)) =
                (reals >> from) & 1u ? raw[c] : make_uint4(0u, 0u, 0u, 0u);
          }
          __syncwarp();
          // (rolled: the code runs once per unit, and comes from L2 when it does)
          uint32_t most = 0;
#pragma unroll 4
          for (int c = 0; c < D / 8; ++c) {
            const uint4 w = *reinterpret_cast<const uint4*>(own + (c >> 3) * S::kQPart + sw128_offset(row_in_tile, c & 7));
            most = extreme2<F16, true>(most, w.x & 0x7fff7fffu);
            most = extreme2<F16, true>(most, w.y & 0x7fff7fffu);
            most = extreme2<F16, true>(most, w.z & 0x7fff7fffu);
            most = extreme2<F16, true>(most, w.w & 0x7fff7fffu);
          }
          const float big = fmaxf(from16<F16>(static_cast<uint16_t>(most)), from16<F16>(static_cast<uint16_t>(most >> 16)));
          const int ex = (__float_as_uint(big) >> 23) & 255;
          const uint32_t e_up = static_cast<uint32_t>(min(253, max(1, 267 - ex)));
          const float up = __uint_as_float(e_up << 23), down = __uint_as_float((254u - e_up) << 23);  // 2^n and 2^-n
          // a negative scaling goes into the query, so that the largest product is the largest score
          const float f = a.scaling < 0.f ? -up : up;
          factor = fabsf(a.scaling) * kLog2e * down;
          factor = factor < 0x1p-126f ? 0x1p-126f : factor;  // above zero, for what is hidden is infinity times it
#pragma unroll 4
          for (int c = 0; c < D / 8; ++c) {
            uint4& at = *reinterpret_cast<uint4*>(own + (c >> 3) * S::kQPart + sw128_offset(row_in_tile, c & 7));
            const uint32_t w[4] = {at.x, at.y, at.z, at.w};
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = from16<F16>(static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)))) * f;
            at = make_uint4(pack_half2(x[0], x[4]), pack_half2(x[1], x[5]), pack_half2(x[2], x[6]), pack_half2(x[3], x[7]));
          }
          fence_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[tile]);
        }
        const int limit = real ? q.start + i + 1 : 0;
        const int full_below = q.start + row0 / share + 1;  // tokens below it are seen by every row of the tile
        const uint64_t f2 = f32x2_pack(__float_as_uint(factor), __float_as_uint(factor));
        float ref = 0.f;
        uint64_t l2 = 0;     // two sums, of the even and the odd tokens
        bool known = false;  // the row has a reference
        for (int t = walk.first; t < walk.last && ok; ++t, ++count) {
          const int bar = tile * 2 + (count & 1);
          const uint32_t s_at = tmem + lanes + bar * 64;
          ok = warp_wait(&s_full[bar], (count >> 1) & 1, a.status, kSiteQ4Attend + kErrWaitAccum, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const int base = t * kStep;
          const bool edge = base + kStep > full_below;
          uint32_t s[kStep / 32][32];
#pragma unroll
          for (int c = 0; c < kStep / 32; ++c) tmem_ld32(s_at + c * 32, s[c]);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < kStep / 32; ++c) tmem_fence32(s[c]);
          if (edge) {
            const int n = limit - base;
#pragma unroll
            for (int e = 0; e < kStep; ++e) s[e / 32][e % 32] = e < n ? s[e / 32][e % 32] : 0xff800000u;  // -infinity; the factor is positive
          }
          const uint64_t o2 = f32x2_pack(__float_as_uint(kBias - ref), __float_as_uint(kBias - ref));
          float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < kStep; e += 2) {
            uint32_t &s0 = s[e / 32][e % 32], &s1 = s[e / 32][e % 32 + 1];
            const uint64_t x = fma_f32x2(f32x2_pack(s0, s1), f2, o2);
            s0 = static_cast<uint32_t>(x);
            s1 = static_cast<uint32_t>(x >> 32);
            float& top = tops[e / 2 % 4];
            top = fmaxf(top, fmaxf(__uint_as_float(s0), __uint_as_float(s1)));
          }
          const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
          const bool raise = known ? top > kBias + kSlack : top > -INFINITY;
          if (__any_sync(0xffffffffu, raise)) {
            // ---- a row's first tokens set its reference, a maximum beyond the slack moves it: by a whole number, so that
            // what is scaled down for it (the output so far) loses nothing
            const float up = raise ? ceilf(top - kBias) : 0.f;
            const float down = !raise ? 1.f : known ? exp2_fast(-up) : 0.f;
            ref += up;
            known = known || raise;
            l2 = mul_f32x2(l2, f32x2_pack(__float_as_uint(down), __float_as_uint(down)));
#pragma unroll
            for (int e = 0; e < kStep; ++e) s[e / 32][e % 32] = __float_as_uint(__uint_as_float(s[e / 32][e % 32]) - up);
            if (t > walk.first) {
              // these scores came after the product of the step before the last, so one phase at most is open
              ok = ok && warp_wait(&o_done[tile], (count - 1) & 1, a.status, kSiteQ4Attend + kErrWaitAccum, abort_flag);
              tc_fence_after();
#pragma unroll 1
              for (int k = 0; k < D / 16; ++k) {
                uint32_t x[16];
                tmem_ld16(o_at + k * 16, x);
                tmem_ld_wait();
                tmem_reg_fence(x);
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * down);
                tmem_st16(o_at + k * 16, x);
              }
            }
          }
          // 32 scores become 16 columns of probabilities (and 16 of what their rounding lacks) in their place
#pragma unroll
          for (int c = 0; c < kStep / 32; ++c) {
            uint32_t p[16], lack[F16 ? 16 : 1];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float e0 = exp2_fast(__uint_as_float(s[c][2 * e])), e1 = exp2_fast(__uint_as_float(s[c][2 * e + 1]));
              const uint64_t both = f32x2_pack(__float_as_uint(e0), __float_as_uint(e1));
              l2 = add_f32x2(l2, both);
              p[e] = pack_half2(e0, e1);
              if constexpr (F16) lack[e] = lack2(both, as_half2(p[e]));
            }
            tmem_st16(s_at + c * 32, p);
            if constexpr (F16) tmem_st16(s_at + c * 32 + 16, lack);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[bar]);
        }
        if (!ok) break;
        ok = warp_wait(&o_full[tile], units++ & 1, a.status, kSiteQ4Attend + kErrWaitAccum, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const float l = f32x2_sum(l2);
        const bool whole = walk.whole();
        const float inv = !whole ? 1.f : l != 0.f ? 1.f / l : 0.f;
        const int64_t to = ((static_cast<int64_t>(walk.seq) * a.q_len + i) * a.n_q_heads + walk.head * share + r - i * share) * D;
        const int row = tile * kRows + row_in_tile;  // of the block
        float* slot = a.workspace + (2 * static_cast<int64_t>(blockIdx.x) + (unit_begin == begin ? 0 : 1)) * slot_floats(slot_rows, D);
        const unsigned reals = __ballot_sync(0xffffffffu, real);
        // 32 dimensions of the warp's 32 rows at a time through shared memory (the tile's queries are done with), so that
        // eight lanes write a row's 128 bytes
        float* box = reinterpret_cast<float*>(smem + S::kQ + tile * S::kQTile) + (warp & 3) * 1024;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t x[32];
          __syncwarp();
          tmem_ld32(o_at + c * 32, x);
          tmem_ld_wait();
          tmem_fence32(x);
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[kOrder[e]] = __uint_as_float(x[h * 8 + e]) * inv;
            *reinterpret_cast<float4*>(box + lane * 32 + ((2 * h) ^ (lane & 7)) * 4) = make_float4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<float4*>(box + lane * 32 + ((2 * h + 1) ^ (lane & 7)) * 4) = make_float4(y[4], y[5], y[6], y[7]);
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int from = k * 4 + (lane >> 3), dim = c * 32 + (lane & 7) * 4;  // the row's lane, the dimension
            const float4 v = *reinterpret_cast<const float4*>(box + from * 32 + ((lane & 7) ^ (from & 7)) * 4);
            const int64_t at = __shfl_sync(0xffffffffu, to, from);
            if ((reals >> from) & 1u) {
              if (whole) store_out4<F16>(a, at + dim, v.x, v.y, v.z, v.w);
              else *reinterpret_cast<float4*>(slot + (row - lane + from) * D + dim) = v;
            }
          }
        }
        fence_async_shared();  // the next unit's queries come after these
        if (!whole && real) *reinterpret_cast<float2*>(slot + slot_rows * D + row * 4) = make_float2(ref, l);
        tc_fence_before();
      }
      if (!ok) *abort_flag = 1;
    } else if (warp < kMmaWarp) {
      // ------------------------------------------------------------ unpacking
      setmaxnreg_dec<kUnpackRegs>();
      Walk walk(a, share, start);
      const int r = threadIdx.x % kStep, part = (threadIdx.x / kStep) & 3;  // the token of the page, which quarter of it
      // The one of the token's four pieces of key codes that this thread takes, so that the lanes of a load, and those of a
      // store into the swizzled tile, lie on different banks: rows 2 i and 2 i + 1 (4 i .. 4 i + 3 of 64 dimensions, where
      // the piece i itself does) take part ^ f(i), with f(i) and f(i) ^ i both permutations of 0 .. 3.
      const int i2 = (r >> 1) & 3;
      const int piece = part ^ (D == 128 ? i2 >> 1 | ((i2 ^ i2 >> 1) & 1) << 1 : (r >> 2) & 3);
      uint32_t iter = 0;
      bool ok = true;
      auto load = [&](uint32_t (&w)[D / 32], const uint8_t* src) {
        if constexpr (D == 128) {
          const uint4 u = *reinterpret_cast<const uint4*>(src);
          w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(src);
          w[0] = u.x, w[1] = u.y;
        }
      };
      auto wait = [&](uint64_t* bar, uint32_t parity, int err) {
        ok = ok && warp_wait(bar, parity, a.status, kSiteQ4Attend + err, abort_flag);
        return ok;
      };
      while (ok && walk.next()) {
        const int seen = seen_by(walk.q, walk.block, share);
        for (int t = walk.first; t < walk.last; ++t, ++iter) {
          const uint32_t raw = iter % S::kRawStages, stage = iter % S::kStages, turn = iter / S::kStages;
          wait(&raw_full[raw], (iter / S::kRawStages) & 1, kErrWaitCodes);
          if (turn > 0) wait(&k_free[stage], (turn - 1) & 1, kErrWaitEmpty);
          if (!ok) break;
          const uint8_t* page = smem + S::kRaw + raw * C::kBytes;
          // a token that no row sees may never have been written: zeros, no NaN of its
          const bool there = t * kStep + r < seen;
          uint32_t heads[2 * kGroups];  // (scale, low) of the key's groups, of the value's
          load(heads, page + C::key_head(r, 0));
#pragma unroll
          for (int e = 0; e < 2 * kGroups; ++e) heads[e] = there ? heads[e] : 0u;
          {
            uint32_t w[D / 32];
            load(w, page + C::kKeyCodes + r * (D / 2) + piece * (D / 8));
#pragma unroll
            for (int gr = 0; gr < kGroups; ++gr) {
              const __half2 h = as_half2(heads[gr]);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint4 lack;
                const uint4 x = unpack8<F16>(w[2 * gr + e], __low2half2(h), __high2half2(h), lack);
                const uint32_t to = stage * S::kTile + gr * S::kPart + sw128_offset(r, piece * 2 + e);
                *reinterpret_cast<uint4*>(smem + S::kK + to) = x;
                if constexpr (F16) *reinterpret_cast<uint4*>(smem + S::kKLow + to) = lack;
              }
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&k_full[stage]);
          }
          if (turn > 0 && !wait(&v_free[stage], (turn - 1) & 1, kErrWaitEmpty)) break;
          // two of the pair's eight pieces, this token's halves of them
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int g = 2 * part + k;
            uint32_t w[D / 32];
            load(w, page + C::value_piece(r >> 1, g));
#pragma unroll
            for (int gr = 0; gr < kGroups; ++gr) {
              const __half2 h = as_half2(heads[kGroups + gr]);
              uint4 none;
              *reinterpret_cast<uint4*>(smem + S::kV + stage * S::kTile + gr * S::kPart + sw128_offset(r, g)) =
                  unpack8<false>(__byte_perm(w[2 * gr], w[2 * gr + 1], r & 1 ? 0x7632 : 0x5410), __low2half2(h), __high2half2(h), none);
            }
          }
          fence_async_shared();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&v_full[stage]);
            mbar_arrive(&raw_free[raw]);
          }
        }
      }
      if (!ok) *abort_flag = 1;
    } else if (warp == kCopyWarp) {
      setmaxnreg_dec<kIssueRegs>();
      Walk walk(a, share, start);
      // ------------------------------------------------------------ copies of the pages, ahead of the unpacking
      const int64_t page_stride = static_cast<int64_t>(a.n_kv_heads) * C::kBytes;
      uint32_t issued = 0;
      bool ok = true;
      while (ok && walk.next()) {
        const int n_pages = pages_of(seen_by(walk.q, walk.block, share));
        const int32_t* table = a.blocks + static_cast<int64_t>(walk.seq) * a.max_blocks;
        const uint8_t* cells = a.cells + static_cast<int64_t>(walk.head) * C::kBytes;
        int ids = 0, ids_at = walk.first - 32;
        for (int t = walk.first; t < walk.last && ok; ++t, ++issued) {
          if (t >= ids_at + 32) {  // the next 32 pages' places, one per lane
            ids_at = t;
            ids = t + lane < n_pages ? table[t + lane] : 0;
            if (static_cast<unsigned>(ids) >= static_cast<unsigned>(a.n_pages)) {
              record_error(a.status, kSiteQ4Attend + kErrBadDescriptor);
              ids = 0;  // recorded, and a page that exists read in its place
            }
          }
          const int id = __shfl_sync(0xffffffffu, ids, t - ids_at);
          const uint32_t raw = issued % S::kRawStages;
          if (issued >= S::kRawStages)
            ok = warp_wait(&raw_free[raw], ((issued / S::kRawStages) - 1) & 1, a.status, kSiteQ4Attend + kErrWaitEmpty, abort_flag);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&raw_full[raw], C::kBytes);
            bulk_load(smem + S::kRaw + raw * C::kBytes, cells + id * page_stride, C::kBytes, &raw_full[raw]);
          }
          __syncwarp();
        }
      }
      if (!ok) *abort_flag = 1;
      // No copy is in flight when the CTA leaves.
      for (uint32_t n = issued - min(issued, static_cast<uint32_t>(S::kRawStages)); n < issued; ++n)
        warp_wait(&raw_full[n % S::kRawStages], (n / S::kRawStages) & 1, a.status, kSiteQ4Attend + kErrWaitDrain, nullptr);
    } else if (warp > kCopyWarp) {
      setmaxnreg_dec<kIssueRegs>();
    } else {
      setmaxnreg_dec<kIssueRegs>();
      Walk walk(a, share, start);
      // ------------------------------------------------------------ products
      constexpr uint32_t kQk = idesc_f16(kRows, kStep, false, false, false);
      constexpr uint32_t kPv = idesc_f16(kRows, D, false, false, true);
      const int tile = warp - kMmaWarp;
      const uint32_t q_at = smem_u32(smem + S::kQ + tile * S::kQTile), k_at = smem_u32(smem + S::kK), v_at = smem_u32(smem + S::kV);
      const uint32_t s_at = __shfl_sync(0xffffffffu, tmem, 0) + tile * 128, o_at = s_at + 256;
      uint32_t iter = 0, made = 0, used = 0, units = 0;  // steps, of them with scores made, probabilities used
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, int err) {
        ok = ok && warp_wait(bar, parity, a.status, kSiteQ4Attend + err, abort_flag);
        return ok;
      };
      // Scores go where the product of two steps before had its probabilities, as an operand in TMEM. Products are ordered
      // among themselves only where accumulator and shape are the same, so that one's completion is waited for: the last
      // that the warp has issued, before every step, so that no more than one phase of its barrier is ever open.
      auto last_product = [&](bool mine) { return !mine || used == 0 || wait(&o_done[tile], (used - 1) & 1, kErrWaitAccum); };
      // Q K of step `step` (a dimension step of 16 is 32 bytes further in a row, one of 64 the next part).
      auto scores = [&](uint32_t step, bool mine) {
        const uint32_t stage = step % S::kStages;
        if (!wait(&k_full[stage], (step / S::kStages) & 1, kErrWaitA)) return;
        tc_fence_after();
        const uint32_t bar = made & 1;
        const uint64_t q_desc = smem_desc_sw128(q_at, 16, 1024), k_desc = smem_desc_sw128(k_at + stage * S::kTile, 16, 1024);
        if (elect_lane()) {
          if (mine) {
#pragma unroll
            for (int k = 0; k < (F16 ? 2 : 1) * D / 16; ++k) {
              const int part = k / (D / 16), gr = k / 4 % kGroups, at = 2 * (k % 4);
              mma_f16(s_at + bar * 64, q_desc + gr * (S::kQPart / 16) + at,
                      k_desc + part * ((S::kKLow - S::kK) / 16) + gr * (S::kPart / 16) + at, kQk, k > 0);
            }
            mma_commit(&s_full[tile * 2 + bar]);
          }
          mma_commit(&k_free[stage]);
        }
        __syncwarp();
        made += mine;
      };
      bool more = walk.next();
      while (ok && more) {
        const bool mine = tile == 0 || walk.two();
        const int n = __shfl_sync(0xffffffffu, walk.last - walk.first, 0);
        if (mine) wait(&q_full[tile], units++ & 1, kErrWaitA);
        if (ok && last_product(mine)) scores(iter, mine);
        for (int t = 0; t < n && ok; ++t, ++iter) {
          if (last_product(mine) && t + 1 < n) scores(iter + 1, mine);
          const uint32_t stage = iter % S::kStages, bar = used & 1;
          if (mine && !wait(&p_full[tile * 2 + bar], (used >> 1) & 1, kErrWaitA)) break;
          if (!wait(&v_full[stage], (iter / S::kStages) & 1, kErrWaitA)) break;
          tc_fence_after();
          const uint64_t v_desc = smem_desc_sw128(v_at + stage * S::kTile, S::kPart, 1024);
          if (elect_lane()) {
            if (mine) {  // P V; 16 tokens are 2048 bytes further
#pragma unroll
              for (int k = 0; k < (F16 ? 2 : 1) * kStep / 16; ++k) {
                const int part = k / (kStep / 16), at = k % (kStep / 16);
                mma_f16_ta(o_at, s_at + bar * 64 + part * 16 + (at >> 1) * 32 + (at & 1) * 8, v_desc + 128 * at, kPv, t > 0 || k > 0);
              }
              mma_commit(&o_done[tile]);
              if (t + 1 == n) mma_commit(&o_full[tile]);
            }
            mma_commit(&v_free[stage]);
          }
          __syncwarp();
          used += mine;
        }
        more = walk.next();
      }
      if (!ok) *abort_flag = 1;
      // Every product is complete before TMEM is given back.
      if (elect_lane()) mma_commit(&drain[tile]);
      __syncwarp();
      warp_wait(&drain[tile], 0, a.status, kSiteQ4Attend + kErrWaitDrain, nullptr);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// Joins the blocks that several CTAs share and writes the zeros of the rows behind the new tokens: cta_rows (which divides
// kBlock) rows of one block per CTA. A row of many pieces, as few long contexts leave them, has a warp that takes the pieces'
// factors in its lanes; of few pieces, a warp takes kAtOnce rows together, with all of their loads under way (the
// 49152 rows of 4 x 512 tokens of 24 heads of 128, in two or three pieces: 15 us, one row after another 20).
constexpr int kCombineWarps = 8, kAtOnce = 4, kFewPieces = 4;
template <int D, bool F16>
__global__ void __launch_bounds__(kCombineWarps * 32)
q4_prefill_combine_kernel(const __grid_constant__ dkv_q4_attend_args a, int workers, int slot_rows, int cta_rows) {
  const int share = a.n_q_heads / a.n_kv_heads;
  const int head = blockIdx.y, seq = blockIdx.z, warp = warp_id(), lane = threadIdx.x & 31;
  const Seq q = seq_of(a, seq, share);
  const int rows = a.q_len * share, r0 = blockIdx.x * cta_rows, block = r0 / kBlock;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const bool failed = cta_failed_at_entry(a.status);
  Pieces pieces = {};
  if (r0 < q.rows && !failed)
    pieces = Pieces(a, *unit_record(a, workers, slot_rows, unit_of(a, seq, head, block)), workers, slot_rows, D);
  constexpr int kPer = D / 32;
  const int end = min(r0 + cta_rows, rows);  // of the CTA
  auto place = [&](int r) {
    const int i = r / share;
    return ((static_cast<int64_t>(seq) * a.q_len + i) * a.n_q_heads + head * share + r - i * share) * D;
  };
  const float zeros[kPer] = {};
  for (int r = max(r0, failed ? 0 : q.rows) + warp; r < end; r += kCombineWarps) store_row<D, F16>(a, place(r), zeros);
  if (pieces.n <= 1) return;  // one CTA had the whole block, or it has no row
  const int last = min(end, q.rows);
  if (pieces.n > kFewPieces) {
    for (int r = r0 + warp; r < last; r += kCombineWarps) {
      float sum[kPer];
      join_row<D, 1, 16, 0>(pieces, slot_rows, r - block * kBlock, sum);
      store_row<D, F16>(a, place(r), sum);
    }
    return;
  }
  for (int first = r0 + warp * kAtOnce; first < last; first += kCombineWarps * kAtOnce) {
    float o[kFewPieces][kAtOnce][kPer];
    float2 s[kFewPieces][kAtOnce];
#pragma unroll
    for (int w = 0; w < kFewPieces; ++w)
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const float* slot = pieces.slot(min(w, pieces.n - 1));
        const int row = min(first + k, last - 1) - block * kBlock;
        if (w < pieces.n) {
          load_row<kPer>(slot + row * D + lane * kPer, o[w][k]);
          s[w][k] = *reinterpret_cast<const float2*>(slot + slot_rows * D + row * 4);
        } else {
          for (float& x : o[w][k]) x = 0.f;
          s[w][k] = make_float2(0.f, 0.f);
        }
      }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      float ref = -INFINITY, den = 0.f, sum[kPer] = {};
#pragma unroll
      for (int w = 0; w < kFewPieces; ++w) ref = s[w][k].y == 0.f ? ref : fmaxf(ref, s[w][k].x);
#pragma unroll
      for (int w = 0; w < kFewPieces; ++w) {
        // a piece that saw no token of this row has no say
        const float f = s[w][k].y == 0.f ? 0.f : exp2_fast(s[w][k].x - ref);
        den = fmaf(s[w][k].y, f, den);
#pragma unroll
        for (int e = 0; e < kPer; ++e) sum[e] = fmaf(o[w][k][e], f, sum[e]);
      }
      const float inv = den != 0.f ? 1.f / den : 0.f;
#pragma unroll
      for (int e = 0; e < kPer; ++e) sum[e] *= inv;
      if (first + k < last) store_row<D, F16>(a, place(first + k), sum);
    }
  }
}

template <int D, bool F16>
int launch_prefill(const dkv_q4_attend_args& a, bool appended, cudaStream_t stream) {
  auto kernel = q4_prefill_kernel<D, F16>;
  static std::atomic<uint64_t> done{0};
  if (!allow_shared(kernel, Shared<D, F16>::kAlloc, done)) return DKV_ERR_CUDA;
  const int workers = device_sms(), slot_rows = slot_rows_of(a);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(workers);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Shared<D, F16>::kAlloc;
  cfg.stream = stream;
  cfg.attrs = attr;
  // Right behind the kernel that stores the new tokens, which writes nothing that is read before the wait for it; behind
  // any other, whose writes are not known, in its turn.
  cfg.numAttrs = appended ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, a, workers, slot_rows) != cudaSuccess) return DKV_ERR_CUDA;
  // Few rows: a warp each, for the joins of a long context are long; many: several each, in about one wave of CTAs.
  const int64_t rows = static_cast<int64_t>(rows_of(a)) * a.n_kv_heads * a.n_seq;
  const int cta_rows = rows <= workers * 8 * kCombineWarps ? kCombineWarps : 8 * kCombineWarps;
  cfg.gridDim = dim3((rows_of(a) + cta_rows - 1) / cta_rows, a.n_kv_heads, a.n_seq);
  cfg.blockDim = dim3(kCombineWarps * 32);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, q4_prefill_combine_kernel<D, F16>, a, workers, slot_rows, cta_rows) == cudaSuccess
             ? DKV_OK
             : DKV_ERR_CUDA;
}

}  // namespace

// Up to 64 rows q4_decode_kernel, which takes 16 at a time, is the faster one: over 4 contexts of 3K to 9K tokens, 24 / 8
// heads of 128, bf16, 48 rows take 47 us there and 50 here, 63 rows 50 and 47 (64 rows of heads of 64: 41 and 42, 84: 45
// and 39); over 32 such contexts 48 rows 174 and 215.
bool prefill_takes(const dkv_q4_attend_args& a) { return rows_of(a) > 64; }

int64_t prefill_floats(const dkv_q4_attend_args& a) {
  const int64_t units = static_cast<int64_t>(a.n_seq) * a.n_kv_heads * ((rows_of(a) + kBlock - 1) / kBlock);
  return 2 * static_cast<int64_t>(device_sms()) * slot_floats(slot_rows_of(a), a.head_dim) + 2 * units;
}

int run_prefill(const dkv_q4_attend_args& a, bool appended, cudaStream_t stream) {
  if (a.head_dim == 128)
    return a.fp16 ? launch_prefill<128, true>(a, appended, stream) : launch_prefill<128, false>(a, appended, stream);
  return a.fp16 ? launch_prefill<64, true>(a, appended, stream) : launch_prefill<64, false>(a, appended, stream);
}

}  // namespace q4
}  // namespace dkv
