// dak_attention_kv4.cu - decode attention over the 4-bit paged KV cache
// (dak_kv4.cuh), whose pages lie in HBM or in pinned host memory.
//
// One query token per sequence: o = softmax(scaling q K^T) V over the first
// seq_lens[b] tokens, K and V being scale * code + zero.  A row is one
// (sequence, KV head, block of up to 8 query heads); its tokens are cut into
// chunks of 64, and the chunks of all rows are dealt out to the CTAs that the GPU
// holds at once, whatever the lengths (Q4Deal): a CTA takes a piece of one row, or a
// range over several rows, which it walks over row by row; its four warps take
// every fourth chunk, with copies running ahead across rows.  A row that spans CTAs
// is merged by log-sum-exp.  Scores are kept in base 2; a sequence of no tokens
// gives zeros.
//
// A warp has two chunks in flight, each a bulk copy per page (one contiguous slab
// with K and V of a head).  For 16 tokens and up to 8 heads:
//   S^T [16 tokens x 8 heads] = K Q^T, scale and zero of the token applied to the
//     FP32 scores;
//   O^T [128 dims x 8 heads] += V^T P^T, with the token's scale multiplied into P
//     and its zero added to O as sum_t p_t zero_t per chunk.
// Codes never become floating-point values of their own: they enter the MMAs as
// float16 subnormals, K's one by one, of V the even codes and the whole bytes (even
// + 16 odd, units of 2^-24), which a mask or a byte permutation each give; V's odd
// dims are the difference, at the end (masks and shifts for each nibble took 1 to
// 3% longer; K has no such form, because even - odd / 16 of a query does not fit
// float16).  P is float16, in units of each chunk's largest products (see
// "Statistics" below): for bfloat16 outputs in one term (2^-11 relative, an eighth
// of the output's own rounding), for float16 outputs in two, because one made the
// output up to 1.9 times less exact than its rounding and two do not show.  One unit
// for all chunks and groups, from the largest score and the largest scale, was 1.5%
// (float16 3%, groups of 32 6%) faster and lost V's codes where large scales had
// small weights.
//
// Bound, at 32 x 16384 tokens of 8 KV heads (570 MB, 89 us at the measured copy
// rate): 113 us in bfloat16 and 119 us in float16 in a graph of twelve calls, 126 us
// in bfloat16 over many calls back to back, when power limits the clocks.  The
// copies alone take 91 us; the rest is arithmetic that two warps per scheduler do
// not quite hide (4.4 cycles per instruction and warp, 870 instructions per chunk).
// Plain bulk copies replaced tensor copies with a 64-byte swizzle: bank conflicts
// cost less than the 64-byte rows did, and host pages come 15% faster (46 GB/s).
#include <cfloat>
#include <cstring>
#include <type_traits>

#include "dak_common.cuh"
#include "dak_host.h"
#include "dak_kv4.cuh"

namespace dak {
namespace {

// Two CTAs of four warps per SM: two warps for each of its four schedulers, with
// all the registers that they can use.  Three warps per scheduler with 168
// registers each, as two CTAs of six warps, took 10 to 30% longer, and five warps
// a CTA, which the schedulers cannot share evenly, 20%.
constexpr int kQ4Warps = 4;
constexpr int kQ4Threads = 32 * kQ4Warps;
constexpr int kQ4PerSm = 2;
constexpr int kQ4Heads = 8;    // query heads per CTA: the MMA's N
constexpr int kQ4Chunk = 64;   // tokens a warp takes at a time
constexpr int kQ4Stages = 2;   // chunks in flight per warp
constexpr int kQ4MergeBatch = 6;  // pieces of a row read at once
constexpr int kQ4Slack = 8;      // see Q4Deal
constexpr int kQ4RowChunks = 8;  // rows up to this long are not split while the GPU holds them all

struct AttnQ4Params {
  Kv4Cache c;
  const uint16_t *query;
  long long q_stride_b, q_stride_h;
  uint16_t *out;
  long long o_stride_b, o_stride_h;
  const int32_t *seq_lens;
  float *scratch;     // 2 slots per CTA: outputs (kQ4Frags float4 each), then (m, l) of the heads
  int32_t *counters;  // [rows]: the CTA that finishes a split row last merges it (nullptr: merge kernel)
  int num_q_heads, group, block_heads, head_blocks;  // group: query heads per KV head
  int max_seq_len;
  int ctas, by_row;  // by_row: CTA i takes row i whatever the lengths; there is no scratch
  float scale_log2;                                  // scaling * log2(e)
  int pdl;
};

// Shared memory of a CTA: per warp a ring of chunks, a block of outputs and its
// statistics; barriers.
template <int NG>
struct Q4Smem {
  static constexpr uint32_t stage = 2 * kQ4Chunk * (64 + 4 * NG);
  static constexpr uint32_t o_off = kQ4Warps * kQ4Stages * stage;               // [warps][heads][128]
  static constexpr uint32_t m_off = o_off + kQ4Warps * kQ4Heads * kKv4Dim * 4;  // [warps][heads]
  static constexpr uint32_t l_off = m_off + kQ4Warps * kQ4Heads * 4;
  static constexpr uint32_t bar_off = l_off + kQ4Warps * kQ4Heads * 4;
  static constexpr uint32_t flag_off = bar_off + kQ4Warps * kQ4Stages * 8;   // abort, abort of the drain, last
  static constexpr uint32_t bytes = flag_off + 16;
  static_assert(kQ4PerSm * (bytes + 1024) <= 228 * 1024, "CTAs per SM");
};

// The (scale, zero) words of one token, one per group.
template <int NG> __device__ __forceinline__ void load_pairs(const uint8_t *a, uint32_t (&w)[NG]) {
  if constexpr (NG == 1) {
    w[0] = *reinterpret_cast<const uint32_t *>(a);
  } else if constexpr (NG == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(a);
    w[0] = v.x;
    w[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4 *>(a);
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 half2_of(uint32_t w) { return __half22float2(*reinterpret_cast<__half2 *>(&w)); }
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// D += A (16x16, row) * B (16x8, col), float16 in, FP32 accumulators.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// The transpose of an 8x8 matrix of 16-bit elements spread over the warp.
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Two FP32 products, or products and sums, in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 a, b, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mul.rn.f32x2 d, a, b; mov.b64 {%0, %1}, d;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{.reg .b64 a, b, c, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7}; fma.rn.f32x2 d, a, b, c; "
      "mov.b64 {%0, %1}, d;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// The FP32 number whose upper half is in the lower (e = 0) or upper half of w.
__device__ __forceinline__ float ref_of(uint32_t w, int e) { return __uint_as_float(e ? w & 0xFFFF0000u : w << 16); }

// Outputs are added up and kept in scratch in the MMA's own layout, 256 float4 of
// a row: number i holds, for c = i % 4, g = i / 4 % 8 and t = i / 32, dims d, d + 1
// of heads 2c and 2c + 1 as (d, 2c), (d, 2c + 1), (d + 1, 2c), (d + 1, 2c + 1), d
// being frag_dim.  Every step is then linear in the thread.
constexpr int kQ4Frags = kQ4Heads * kKv4Dim / 4;
static_assert(kQ4Frags == 2 * kQ4Threads, "a thread merges two of a row's float4s");
template <int NG> __device__ __forceinline__ int frag_dim(int t, int g) {
  const int q = t >> 1;
  return (NG == 1 ? 16 * g + 4 * q : NG == 2 ? 64 * (q >> 1) + 8 * g + 4 * (q & 1) : 32 * q + 4 * g) + 2 * (t & 1);
}

// Writes float4 i of a row's output over its denominators; zeros where no weight
// was summed.
template <typename T, int NG>
__device__ __forceinline__ void store_frag(const AttnQ4Params &p, int b, int h0, int nh, int i, float4 v, float den0,
                                           float den1) {
  const int h = 2 * (i & 3);
  uint16_t *to = p.out + b * p.o_stride_b + (h0 + h) * p.o_stride_h + frag_dim<NG>(i >> 5, (i >> 2) & 7);
  const float r0 = den0 == 0.f ? 0.f : 1.f / den0, r1 = den1 == 0.f ? 0.f : 1.f / den1;
  if (h < nh) *reinterpret_cast<uint32_t *>(to) = Elem<T>::pack2(v.x * r0, v.z * r0);
  if (h + 1 < nh) *reinterpret_cast<uint32_t *>(to + p.o_stride_h) = Elem<T>::pack2(v.y * r1, v.w * r1);
}

__device__ __forceinline__ int seq_of(const AttnQ4Params &p, int b) {
  return max(0, min(p.seq_lens[b], p.max_seq_len));
}
__device__ __forceinline__ int chunks_of(int seq) { return (seq + kQ4Chunk - 1) / kQ4Chunk; }

// How the chunks are dealt out: rows are cut into pieces of `size` chunks, a piece
// for each CTA (whole), or ranges of `size` chunks of all rows, end to end, a range
// for each CTA.
//
// Merging a row costs the CTA that does it about 0.1 us per piece, and four chunks,
// one per warp, take 1.5 us: a row of n chunks is best cut into about sqrt(3 n)
// pieces, which matters where one or two rows are all there is (one row of 131072
// tokens: 57 us in 293 pieces, 27 in 79).  A range with chunks of two rows takes
// longer than one of a single row, by the first row's end and warps without a chunk
// there: pieces of up to kQ4Slack chunks more are taken before ranges.  Side by side,
// 24 ragged sequences of up to 6001 tokens: 12.3 us, 19.7 in ranges; 16 of up to
// 20000: 16 and 30; 32 x 16384 of one KV head: 23.3 and 24.9.
struct Q4Deal {
  int size;
  bool whole;
  int ctas;   // with work
  int total;  // chunks
};
// ceil(n / size), for up to 2^20 pieces (here at most p.ctas), in a fraction of a
// division's latency: the rounded quotient is at most two too small.
__device__ __forceinline__ int pieces_of(int n, int size, float rcp) {
  const uint32_t k = (uint32_t)(n * rcp), at = k * size;
  return (int)(k + (at < (uint32_t)n) + (at + size < (uint32_t)n));
}
__device__ __forceinline__ float rcp_of(int size) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"((float)size));
  return r;
}
__device__ __forceinline__ float sqrt_of(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// n32: chunks of sequence lane_id(); all lanes get the answer.
__device__ __forceinline__ Q4Deal q4_deal(const AttnQ4Params &p, int n32) {
  constexpr int kBlocks = 3;  // of 32 sequences behind the first whose lengths stay in registers
  const int lane = lane_id(), R = p.c.kv_heads * p.head_blocks;
  int total = n32, longest = n32, more[kBlocks] = {0, 0, 0};
  if (p.c.rows > 32) {
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const int b = 32 * (i + 1) + lane;
      more[i] = b < p.c.rows ? chunks_of(seq_of(p, b)) : 0;
      total += more[i];
      longest = max(longest, more[i]);
    }
    for (int b = 32 * (kBlocks + 1) + lane; b < p.c.rows; b += 32) {
      const int n = chunks_of(seq_of(p, b));
      total += n;
      longest = max(longest, n);
    }
  }
  total = __reduce_add_sync(0xffffffffu, total) * R;
  longest = __reduce_max_sync(0xffffffffu, longest);
  Q4Deal d;
  d.total = total;
  d.size = max(max((int)(((uint32_t)total + p.ctas - 1) / p.ctas), kQ4Warps), (int)sqrt_of(longest * (1.f / 3.f)));
  d.whole = true;
  const int least = (d.size + kQ4Warps - 1) / kQ4Warps * kQ4Warps;
  for (int size = least; size <= least + kQ4Slack; size += kQ4Warps) {
    const float rcp = rcp_of(size);
    int pieces = pieces_of(n32, size, rcp);
    if (p.c.rows > 32) {
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) pieces += pieces_of(more[i], size, rcp);
      for (int b = 32 * (kBlocks + 1) + lane; b < p.c.rows; b += 32) pieces += pieces_of(chunks_of(seq_of(p, b)), size, rcp);
    }
    d.ctas = __reduce_add_sync(0xffffffffu, pieces) * R;
    if (d.ctas <= p.ctas) {
      d.size = size;
      return d;
    }
  }
  d.whole = false;
  d.ctas = (int)(((uint32_t)total + d.size - 1) / d.size);
  return d;
}

// Merges a row from its pieces in the scratch, in order.  They were left by CTA
// `first` and those after it, as their first segments (slot 2 i of CTA i), or, if the
// row begins within `first`'s range (late), as its last (slot 2 i + 1).
template <typename T, int NG>
__device__ __forceinline__ void merge_row(const AttnQ4Params &p, int b, int h0, int nh, int first, int pieces, bool late) {
  const float4 *po = reinterpret_cast<const float4 *>(p.scratch);
  const float4 *pm = po + 2ll * p.ctas * kQ4Frags;  // (m, l) of two heads
  auto slot = [&](int i) { return 2ll * (first + i) + (late && i == 0 ? 1 : 0); };
  const int k = threadIdx.x;  // this thread's float4s, of the same two heads: k and k + kQ4Threads
  float m0 = -FLT_MAX, m1 = -FLT_MAX, l0 = 0.f, l1 = 0.f;
  float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int i0 = 0; i0 < pieces; i0 += kQ4MergeBatch) {
    float4 ml[kQ4MergeBatch], v[kQ4MergeBatch][2];  // all in flight at once
#pragma unroll
    for (int i = 0; i < kQ4MergeBatch; ++i) {
      const bool in = i0 + i < pieces;
      const long long at = slot(in ? i0 + i : i0);
      ml[i] = __ldcg(pm + at * (kQ4Heads / 2) + (k & 3));
      if (!in) ml[i] = make_float4(-FLT_MAX, 0.f, -FLT_MAX, 0.f);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        v[i][j] = __ldcg(po + at * kQ4Frags + k + j * kQ4Threads);
        if (!in) v[i][j] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    float n0 = m0, n1 = m1;
#pragma unroll
    for (int i = 0; i < kQ4MergeBatch; ++i) n0 = fmaxf(n0, ml[i].x), n1 = fmaxf(n1, ml[i].z);
    const float a0 = ex2(m0 - n0), a1 = ex2(m1 - n1);
    m0 = n0, m1 = n1;
    l0 *= a0, l1 *= a1;
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[j] = make_float4(acc[j].x * a0, acc[j].y * a1, acc[j].z * a0, acc[j].w * a1);
#pragma unroll
    for (int i = 0; i < kQ4MergeBatch; ++i) {
      const float c0 = ex2(ml[i].x - m0), c1 = ex2(ml[i].z - m1);
      l0 = fmaf(ml[i].y, c0, l0);
      l1 = fmaf(ml[i].w, c1, l1);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        acc[j].x = fmaf(v[i][j].x, c0, acc[j].x);
        acc[j].y = fmaf(v[i][j].y, c1, acc[j].y);
        acc[j].z = fmaf(v[i][j].z, c0, acc[j].z);
        acc[j].w = fmaf(v[i][j].w, c1, acc[j].w);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) store_frag<T, NG>(p, b, h0, nh, k + j * kQ4Threads, acc[j], l0, l1);
}

template <typename T, int NG, int P>
__global__ void __launch_bounds__(kQ4Threads, kQ4PerSm) attn_q4_kernel(const __grid_constant__ AttnQ4Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  using S = Q4Smem<NG>;
  constexpr int W = kQ4Warps;
  // The weights of a float16 output are split into two float16 terms.
  constexpr bool kTwoTerms = std::is_same<T, __half>::value;
  const uint32_t sbase = smem_u32(smem);
  const int warp = warp_id(), lane = lane_id();
  const int g = lane >> 2, cq = lane & 3;  // fragment row, column pair
  constexpr int ppc = kQ4Chunk / P;        // pages per chunk
  constexpr uint32_t half = kv4_half_bytes(P, NG), slab = 2 * half;
  const uint32_t bar0 = sbase + S::bar_off + warp * kQ4Stages * 8;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + S::flag_off);
  const WaitCtx wc{abort_flag, p.c.status};
  if (threadIdx.x == 0) {
    for (int s = 0; s < W * kQ4Stages; ++s) mbar_init(sbase + S::bar_off + 8 * s, 1);
    abort_flag[0] = abort_flag[1] = 0;  // [1]: of the wait for copies in flight
    fence_mbar_init();
  }
  pdl_enter(p.pdl);
  __syncthreads();

  // This CTA's range of chunks [lo, hi) and the row (b0, r0) that it begins in,
  // whose chunks begin at `begin`.
  const int R = p.c.kv_heads * p.head_blocks;
  int lo, hi, begin, b0, r0, seq0;
  int per = 0;                // chunks of a range; 0: the CTA has a piece of one row,
  int first = 0, pieces = 1;  // of so many, the first of which CTA `first` has
  const float4 nothing = make_float4(0.f, 0.f, 0.f, 0.f);
  auto zero_rows = [&]() {  // sequences of no tokens belong to no CTA
    for (int b = blockIdx.x; b < p.c.rows; b += p.ctas)
      if (seq_of(p, b) == 0)
        for (int h = 0; h < p.num_q_heads; h += kQ4Heads)
          for (int k = threadIdx.x; k < kQ4Frags; k += kQ4Threads)
            store_frag<T, NG>(p, b, h, p.num_q_heads - h, k, nothing, 0.f, 0.f);
  };
  if (p.by_row) {
    b0 = blockIdx.x / R;
    r0 = blockIdx.x - b0 * R;
    lo = begin = 0;
    seq0 = seq_of(p, b0);
    hi = chunks_of(seq0);
    if (hi == 0) {
      const int hb = r0 % p.head_blocks;
      for (int k = threadIdx.x; k < kQ4Frags; k += kQ4Threads)
        store_frag<T, NG>(p, b0, r0 / p.head_blocks * p.group + hb * p.block_heads,
                          min(p.block_heads, p.group - hb * p.block_heads), k, nothing, 0.f, 0.f);
      return;
    }
  } else {
    // Lengths of 32 sequences, one per lane; most batches have no more.
    int seqs = lane < p.c.rows ? seq_of(p, lane) : 0;
    int n32 = chunks_of(seqs);
    const Q4Deal deal = q4_deal(p, n32);
    if ((int)blockIdx.x >= deal.ctas) {
      zero_rows();
      return;
    }
    // The row in which unit `from` lies, a unit being a piece or a chunk.
    const int from = deal.whole ? blockIdx.x : blockIdx.x * deal.size;
    int before = 0;  // units of the sequences before this block of 32
    for (int base = 0;; base += 32) {
      if (base > 0) {
        seqs = base + lane < p.c.rows ? seq_of(p, base + lane) : 0;
        n32 = chunks_of(seqs);
      }
      const int units = deal.whole ? pieces_of(n32, deal.size, rcp_of(deal.size)) : n32;
      int incl = units * R;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, x);
        if (lane >= x) incl += v;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, before + incl > from);
      if (past) {
        const int l0 = __ffs(past) - 1, row_units = __shfl_sync(0xffffffffu, units, l0);
        const int seq_begin = before + __shfl_sync(0xffffffffu, incl, l0) - row_units * R;
        b0 = base + l0;
        r0 = (from - seq_begin) / row_units;
        begin = seq_begin + r0 * row_units;
        seq0 = __shfl_sync(0xffffffffu, seqs, l0);
        pieces = row_units;
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (deal.whole) {
      first = begin;
      lo = (from - begin) * deal.size;
      begin = 0;
      hi = min(chunks_of(seq0), lo + deal.size);
    } else {
      per = deal.size;
      lo = from;
      hi = lo + min(per, deal.total - lo);
    }
  }

  // Word w (0..3) of a K row that this lane multiplies, 8 dims each: all the
  // words of one group meet in the same MMA steps.
  auto k_word = [&](int w) {
    return NG == 1 ? 4 * cq + w : NG == 2 ? 8 * (w >> 1) + 2 * cq + (w & 1) : 4 * w + cq;
  };
  // Query words of head g of a row, as they are; used when the row's turn comes.
  uint4 qraw[4];
  auto heads_of = [&](int r, int &h0, int &nh) {
    const int hb = r % p.head_blocks;
    h0 = r / p.head_blocks * p.group + hb * p.block_heads;
    nh = min(p.block_heads, p.group - hb * p.block_heads);
  };
  auto fetch_query = [&](int b, int r) {
    int h0, nh;
    heads_of(r, h0, nh);
#pragma unroll
    for (int w = 0; w < 4; ++w)
      qraw[w] = g < nh ? *reinterpret_cast<const uint4 *>(p.query + b * p.q_stride_b + (h0 + g) * p.q_stride_h + 8 * k_word(w))
                       : make_uint4(0u, 0u, 0u, 0u);
  };
  fetch_query(b0, r0);

  // Copies, ahead of the arithmetic: this warp takes chunks lo + warp, + 4, ...
  // The position (row, table entries) of the copy after next is worked out while
  // the chunks in flight are multiplied.
  const uint64_t pol = l2_policy_evict_first();
  int at = lo + warp, at_b = b0, at_r = r0, at_begin = begin, at_pages = (seq0 + P - 1) / P;
  int at_end = begin + chunks_of(seq0);
  const int32_t *at_row = p.c.table + b0 * p.c.table_stride + lane;
  uint32_t head_off = (uint32_t)(r0 / p.head_blocks) * slab;
  int entry = 0, pages = 0, issued = 0;
  auto locate = [&]() {
    if (at >= hi) return;
    while (at >= at_end) {
      at_begin = at_end;
      if (++at_r == R) {
        at_r = 0;
        int seq;
        do {
          seq = seq_of(p, ++at_b);
        } while (seq == 0);  // there is one: the range goes on
        at_pages = (seq + P - 1) / P;
        at_row = p.c.table + at_b * p.c.table_stride + lane;
      }
      at_end = at_begin + (at_pages + ppc - 1) / ppc;
      head_off = (uint32_t)(at_r / p.head_blocks) * slab;
    }
    const int first = (at - at_begin) * ppc;
    pages = min(ppc, at_pages - first);
    entry = lane < pages ? at_row[first] : 0;
  };
  auto issue = [&]() {
    const int s = issued % kQ4Stages;
    uint8_t *to = smem + (warp * kQ4Stages + s) * S::stage;
    const int tier = entry < 0 ? 1 : 0;
    const uint32_t page = entry < 0 ? ~entry : entry;  // -1 - v is ~v
    const bool good = lane < pages && page < p.c.pages[tier];
    const uint32_t which = __ballot_sync(0xffffffffu, good);
    if (lane == 0) mbar_arrive_expect_tx(bar0 + 8 * s, __popc(which) * slab);
    __syncwarp();
    if (good)
      bulk_load(smem_u32(to) + lane * slab, p.c.pool[tier] + page * p.c.page_bytes + head_off, slab, bar0 + 8 * s, pol);
    if (__popc(which) < pages) {  // an entry outside its pool: zeros
      if (lane == 0) atomicCAS(p.c.status, 0, DAK_ERR_INVALID_ARG);
      for (int i = 0; i < pages; ++i)
        if (!(which >> i & 1u))
          for (int v = lane; v < slab / 16; v += 32) reinterpret_cast<uint4 *>(to + i * slab)[v] = make_uint4(0u, 0u, 0u, 0u);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the stage's next fill is a copy
    }
    __syncwarp();
    ++issued;
    at += W;
    locate();
  };
  locate();
  for (int j = 0; j < kQ4Stages; ++j)
    if (at < hi) issue();
  if (!p.by_row) zero_rows();

  // Scores.  A query is scaled by a power of two so that its largest value lies
  // between 2^13 and 2^14; float16 then holds the others exactly down to 2^-23 of it
  // (bfloat16's too), and smaller ones to 2^-34 of it.  Products and sums are FP32.
  // Integer MMAs over whole bytes, the query in 16 and 20 bits, were 2% faster with one
  // group, no faster with two, and lost the bits of all other channels where one was
  // far larger.
  uint32_t qf[8][2];
  float qs[2][NG], f[2];  // q summed over each group (for the zeros' share); raw scores to base 2
  auto ready_query = [&]() {
    float x[4][8], mx = 0.f, bad = 0.f, sum[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) sum[n] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t u[4] = {qraw[w].x, qraw[w].y, qraw[w].z, qraw[w].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 y = Elem<T>::to_float2(u[e]);
        x[w][2 * e] = y.x;
        x[w][2 * e + 1] = y.y;
        mx = max3(mx, fabsf(y.x), fabsf(y.y));
        bad += y.x * 0.f + y.y * 0.f;  // NaN for a query that is not finite
      }
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    bad += __shfl_xor_sync(0xffffffffu, bad, 1);
    bad += __shfl_xor_sync(0xffffffffu, bad, 2);
    const int k = mx > 0.f ? min(127, 13 - ((int)(__float_as_uint(mx) >> 23) - 127)) : 0;  // -114 (finite q) to 127
    // A negative scaling turns the query over, so that a larger raw score is
    // always a larger score.
    const float up = copysignf(__uint_as_float((uint32_t)(127 + k) << 23), p.scale_log2);
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float a = x[w][2 * h] * up, c = x[w][2 * h + 4] * up;
        const float d = x[w][2 * h + 1] * up, e = x[w][2 * h + 5] * up;
        qf[2 * w + h][0] = pack_half2(a, c);
        qf[2 * w + h][1] = pack_half2(d * 0.0625f, e * 0.0625f);
        sum[w * NG / 4] += ((a + c) + (d + e)) * 0x1p-24f;
      }
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 1);
      sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 2);
    }
    // Back to the scores: |scaling| x 2^(24 - k), in two steps because the power alone
    // may lie beyond FP32.  Above 2^100, raw scores that differ at all (by 2^-34 or more)
    // leave one weight: a larger factor changes nothing, and scores stay finite.
    const int up1 = (24 - k) / 2, up2 = 24 - k - up1;
    float fh = fabsf(p.scale_log2) * __uint_as_float((uint32_t)(127 + up1) << 23) * __uint_as_float((uint32_t)(127 + up2) << 23);
    fh = (fh > 0x1p100f ? 0x1p100f : fh) + bad + p.scale_log2 * 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // lane 4h holds head h
      const int src = 4 * (2 * cq + e);
      f[e] = __shfl_sync(0xffffffffu, fh, src);
#pragma unroll
      for (int n = 0; n < NG; ++n) qs[e][n] = __shfl_sync(0xffffffffu, sum[n], src);
    }
  };

  // V: this lane takes 4 dims at a time (piece x) of tokens 2 cq, 2 cq + 1 (and 8
  // on).  Odd columns read the second token first, so that a warp's rows are even
  // and odd ones and use all banks; the byte selectors put the pair back in order.
  const uint32_t flip = cq & 1;
  const uint32_t sel_lo = flip ? 0x1054u : 0x5410u, sel_hi = flip ? 0x3276u : 0x7632u;
  const uint32_t sel_g = (g & 1) ? sel_hi : sel_lo;

  // Statistics: weights are 2^(score - m), m being the largest score so far.  What
  // float16 has to hold is weight x scale, and the largest product need not be that
  // of the largest score or of the largest scale, so P and O have a unit of their
  // own, per head and group (ref: two heads' FP32 powers of two, upper halves): each
  // chunk takes the exponent of its largest product (several groups: of the largest
  // sum over a lane's 8 tokens, one instruction less), so that products are below 2
  // and those above 2^-14 keep all of their bits.  The unit falls as well as rises,
  // and O with it, exactly; it stays at 2^-104 of the largest weight or above so that
  // FP32 holds O (2^16 x 255 x 2^-24 per token, over 2^23 tokens).
  constexpr uint32_t kRefMin = (127 - 104) << 7 | (127 - 104) << 23;
  float o[8][4], m[2], l[2];
  uint32_t ref[NG];

  // One chunk of `valid` tokens in the stage at `st`.
  auto chunk = [&](const uint8_t *st, int valid, auto full_c) {
    constexpr bool kFull = decltype(full_c)::value;
    // Where tile t's code rows begin (V: + half), and the pairs of token g + 8r.
    auto rows_at = [](int t) { return (uint32_t)((16 * t) / P * slab + (16 * t) % P * 64); };
    auto pairs_at = [&](int t, int r) {
      return (uint32_t)((16 * t) / P * slab + P * 64 + ((16 * t) % P + g + 8 * r) * (4 * NG));
    };
    float y[4][4];  // raw scores: tile, {token g, g + 8} x {head 2 cq, 2 cq + 1}
    float mx[2] = {-INFINITY, -INFINITY};
    // V's (scale, zero) words of token g + 8r of tile t.  Several groups' are read
    // again where they are needed, which costs less than the registers would.
    auto load_vp = [&](int t, int r, uint32_t(&vp)[NG]) {
      load_pairs<NG>(st + half + pairs_at(t, r), vp);
#pragma unroll
      for (int n = 0; n < NG; ++n)
        if (!kFull && t * 16 + 8 * r + g >= valid) vp[n] = 0u;  // anything may lie behind the last token
    };
    auto forget = [] {
      if (NG > 1) asm volatile("" ::: "memory");
    };
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (!kFull && t * 16 >= valid) continue;
      // S^T = K Q^T
      uint32_t w0[4], w1[4];  // tokens g and g + 8
      if constexpr (NG == 1) {
        const uint8_t *a = st + rows_at(t) + g * 64 + 16 * cq;
        const uint4 u = *reinterpret_cast<const uint4 *>(a), v = *reinterpret_cast<const uint4 *>(a + 512);
        w0[0] = u.x, w0[1] = u.y, w0[2] = u.z, w0[3] = u.w;
        w1[0] = v.x, w1[1] = v.y, w1[2] = v.z, w1[3] = v.w;
      } else if constexpr (NG == 2) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint8_t *a = st + rows_at(t) + g * 64 + 32 * n + 8 * cq;
          const uint2 u = *reinterpret_cast<const uint2 *>(a), v = *reinterpret_cast<const uint2 *>(a + 512);
          w0[2 * n] = u.x, w0[2 * n + 1] = u.y;
          w1[2 * n] = v.x, w1[2 * n + 1] = v.y;
        }
      } else {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint8_t *a = st + rows_at(t) + g * 64 + 16 * n + 4 * cq;
          w0[n] = *reinterpret_cast<const uint32_t *>(a);
          w1[n] = *reinterpret_cast<const uint32_t *>(a + 512);
        }
      }
      uint32_t kp[2][NG];
#pragma unroll
      for (int r = 0; r < 2; ++r) load_pairs<NG>(st + pairs_at(t, r), kp[r]);
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        // A nibble at bits 0-3 of a half word is the subnormal code * 2^-24, at bits
        // 4-7 code * 2^-20 (its q is / 16).
#pragma unroll
        for (int w = n * 4 / NG; w < (n + 1) * 4 / NG; ++w) {
          mma_f16(acc, w0[w] & 0x000F000Fu, w1[w] & 0x000F000Fu, w0[w] & 0x00F000F0u, w1[w] & 0x00F000F0u, qf[2 * w][0],
                  qf[2 * w][1]);
          const uint32_t s0 = __byte_perm(w0[w], 0u, 0x4341u), s1 = __byte_perm(w1[w], 0u, 0x4341u);
          mma_f16(acc, s0 & 0x000F000Fu, s1 & 0x000F000Fu, s0 & 0x00F000F0u, s1 & 0x00F000F0u, qf[2 * w + 1][0],
                  qf[2 * w + 1][1]);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float2 sz = half2_of(kp[r][n]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float zq = n == 0 ? sz.y * qs[e][n] : fmaf(sz.y, qs[e][n], y[t][2 * r + e]);
            y[t][2 * r + e] = fmaf(sz.x, acc[2 * r + e], zq);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (kFull) {
          mx[e] = max3(mx[e], y[t][e], y[t][2 + e]);
        } else {
          if (t * 16 + g < valid) mx[e] = fmaxf(mx[e], y[t][e]);
          if (t * 16 + 8 + g < valid) mx[e] = fmaxf(mx[e], y[t][2 + e]);
        }
      }
    }
    float alpha[2];
    float2 zs[2][NG], top[2][NG];  // of the tokens g and g + 8 of all tiles
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x <= 16; x <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], x));
      const float mn = fmaxf(m[e], mx[e] * f[e]);
      alpha[e] = ex2(m[e] - mn);
      m[e] = mn;
      l[e] *= alpha[e];
#pragma unroll
      for (int n = 0; n < NG; ++n) zs[e][n] = top[e][n] = make_float2(0.f, 0.f);
    }
    // Weights, the zeros' share of the output, sum_t p_t zero_t per group, and the
    // largest product.  One group's products take the weights' place.
    forget();
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (!kFull && t * 16 >= valid) continue;
      uint32_t vp[2][NG];
      load_vp(t, 0, vp[0]);
      load_vp(t, 1, vp[1]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float w[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          w[r] = ex2(fmaf(y[t][2 * r + e], f[e], -m[e]));
          if (!kFull && t * 16 + 8 * r + g >= valid) w[r] = 0.f;
          l[e] += w[r];
        }
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const float2 v0 = half2_of(vp[0][n]), v1 = half2_of(vp[1][n]), ww = make_float2(w[0], w[1]);
          zs[e][n] = fma2(ww, make_float2(v0.y, v1.y), zs[e][n]);
          if (NG == 1) {
            const float2 a = mul2(ww, make_float2(v0.x, v1.x));
            top[e][n].x = max3(top[e][n].x, a.x, a.y);
            y[t][e] = a.x, y[t][2 + e] = a.y;
          } else {
            top[e][n] = fma2(ww, make_float2(v0.x, v1.x), top[e][n]);
          }
        }
        if (NG > 1) y[t][e] = w[0], y[t][2 + e] = w[1];
      }
    }
    forget();
    // This chunk's units, and O from the last chunk's to them.
    float up[2][NG], beta[2][NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      uint32_t now = __byte_perm(__float_as_uint(top[0][n].x + top[0][n].y), __float_as_uint(top[1][n].x + top[1][n].y), 0x7632u);
#pragma unroll
      for (int x = 4; x <= 16; x <<= 1) now = max_u16x2(now, __shfl_xor_sync(0xffffffffu, now, x));
      now = max_u16x2(now & 0x7F807F80u, kRefMin);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        up[e][n] = __uint_as_float(0x7F000000u - (e ? now & 0xFFFF0000u : now << 16));
        beta[e][n] = alpha[e] * (ref_of(ref[n], e) * up[e][n]);
      }
      ref[n] = now;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        zs[e][n].x += zs[e][n].y;
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) zs[e][n].x += __shfl_xor_sync(0xffffffffu, zs[e][n].x, x);
      }
    // O rows: even dims in units of 2^-24, and the sum of an even dim and 16 times the
    // odd one beside it.  Adding the zeros' share chunk by chunk keeps O centred, so
    // nothing cancels at the end.
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const float2 even = make_float2(zs[0][n].x * (up[0][n] * 0x1p-24f), zs[1][n].x * (up[1][n] * 0x1p-24f));
      const float2 odd = make_float2(even.x * 17, even.y * 17), old = make_float2(beta[0][n], beta[1][n]);
#pragma unroll
      for (int t = 8 * n / NG; t < 8 * (n + 1) / NG; ++t) {
        const float2 a = fma2(make_float2(o[t][0], o[t][1]), old, even), c = fma2(make_float2(o[t][2], o[t][3]), old, odd);
        o[t][0] = a.x, o[t][1] = a.y, o[t][2] = c.x, o[t][3] = c.y;
      }
    }
    // O^T += V^T P^T
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (!kFull && t * 16 >= valid) continue;
      uint32_t bf[NG][2];
      [[maybe_unused]] uint32_t bl[NG][2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        uint32_t vp[NG];
        if (NG > 1) load_vp(t, r, vp);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          float a = y[t][2 * r] * up[0][n], c = y[t][2 * r + 1] * up[1][n];
          if (NG > 1) {
            const float s = half2_of(vp[n]).x;
            a *= s;
            c *= s;
          }
          const uint32_t hi = pack_half2(a, c);
          bf[n][r] = movmatrix(hi);
          if constexpr (kTwoTerms) {
            const float2 back = half2_of(hi);
            bl[n][r] = movmatrix(pack_half2(a - back.x, c - back.y));
          }
        }
      }
      // Token pairs (2 cq, + 1) and (2 cq + 8, + 9): 4 pieces of 4 dims of each.
      uint32_t x[2][4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint8_t *a = st + half + rows_at(t) + (2 * cq + flip + 8 * r) * 64;
        const uint8_t *c = st + half + rows_at(t) + (2 * cq + 1 - flip + 8 * r) * 64;
        if constexpr (NG == 1) {
          const uint2 u = *reinterpret_cast<const uint2 *>(a + 8 * g), v = *reinterpret_cast<const uint2 *>(c + 8 * g);
          x[r][0] = __byte_perm(u.x, v.x, sel_lo);
          x[r][1] = __byte_perm(u.x, v.x, sel_hi);
          x[r][2] = __byte_perm(u.y, v.y, sel_lo);
          x[r][3] = __byte_perm(u.y, v.y, sel_hi);
        } else if constexpr (NG == 2) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const uint32_t u = *reinterpret_cast<const uint32_t *>(a + 32 * n + 4 * g);
            const uint32_t v = *reinterpret_cast<const uint32_t *>(c + 32 * n + 4 * g);
            x[r][2 * n] = __byte_perm(u, v, sel_lo);
            x[r][2 * n + 1] = __byte_perm(u, v, sel_hi);
          }
        } else {
#pragma unroll
          for (int n = 0; n < 4; ++n)
            x[r][n] = __byte_perm(*reinterpret_cast<const uint32_t *>(a + 16 * n + 4 * (g >> 1)),
                                  *reinterpret_cast<const uint32_t *>(c + 16 * n + 4 * (g >> 1)), sel_g);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = q * NG / 4;
        // Bytes 0 and 2 (even code + 16 odd), then bytes 1 and 3; their even codes.
        const uint32_t b0 = x[0][q] & 0x00FF00FFu, b1 = x[1][q] & 0x00FF00FFu;
        const uint32_t c0 = __byte_perm(x[0][q], 0u, 0x4341u), c1 = __byte_perm(x[1][q], 0u, 0x4341u);
        const uint32_t e0 = x[0][q] & 0x000F000Fu, e1 = x[1][q] & 0x000F000Fu;
        const uint32_t f0 = c0 & 0x000F000Fu, f1 = c1 & 0x000F000Fu;
        mma_f16(o[2 * q], e0, b0, e1, b1, bf[n][0], bf[n][1]);
        mma_f16(o[2 * q + 1], f0, c0, f1, c1, bf[n][0], bf[n][1]);
        if constexpr (kTwoTerms) {
          mma_f16(o[2 * q], e0, b0, e1, b1, bl[n][0], bl[n][1]);
          mma_f16(o[2 * q + 1], f0, c0, f1, c1, bl[n][0], bl[n][1]);
        }
      }
    }
  };

  float *sm_m = reinterpret_cast<float *>(smem + S::m_off), *sm_l = reinterpret_cast<float *>(smem + S::l_off);
  float4 *sm_o = reinterpret_cast<float4 *>(smem + S::o_off);
  int done = 0, dead_at = -1;  // chunks taken; the chunk whose copy never came
  int b = b0, r = r0, seq = seq0, n = chunks_of(seq0);
  for (int s0 = lo; s0 < hi;) {
    // The segment [s0, s1) of row (b, r), whose chunks begin at `begin`.
    const int s1 = min(hi, begin + n);
    int h0, nh;
    heads_of(r, h0, nh);
    ready_query();
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[t][e] = 0.f;
    m[0] = m[1] = -FLT_MAX;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int x = 0; x < NG; ++x) ref[x] = kRefMin;
    for (; lo + warp + W * done < s1; ++done) {
      const int id = lo + warp + W * done, s = done % kQ4Stages;
      const uint32_t parity = (done / kQ4Stages) & 1;
      const bool ok = dead_at < 0 && (mbar_try_wait(bar0 + 8 * s, parity) || mbar_wait<false>(bar0 + 8 * s, parity, wc));
      if (!__all_sync(0xffffffffu, ok)) {  // give up, but keep to the barriers below
        if (dead_at < 0) dead_at = done;
        continue;
      }
      const uint8_t *st = smem + (warp * kQ4Stages + s) * S::stage;
      const int valid = min(kQ4Chunk, seq - (id - begin) * kQ4Chunk);
      if (valid == kQ4Chunk)
        chunk(st, valid, std::true_type{});
      else
        chunk(st, valid, std::false_type{});
      __syncwarp();
      if (at < hi) issue();
    }

    // The row after this one, and its query.
    const bool whole = s0 == begin && s1 == begin + n;
    const int row_b = b, row_r = r;
    bool late = false;
    if (per > 0) {
      first = begin / per;
      pieces = (begin + n - 1) / per - first + 1;
      late = first * per < begin;
    }
    if (s1 < hi) {
      begin = s1;
      if (++r == R) {
        r = 0;
        do {
          seq = seq_of(p, ++b);
        } while (seq == 0);  // there is one: the range goes on
        n = chunks_of(seq);
      }
      fetch_query(b, r);
    }

    // Add up the warps: statistics first, then each warp's share (zero from a warp
    // that had no chunk).
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x <= 16; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
      if (g == 0) {
        sm_m[warp * kQ4Heads + 2 * cq + e] = m[e];
        sm_l[warp * kQ4Heads + 2 * cq + e] = l[e];
      }
    }
    __syncthreads();
    float gm[2], share[2];  // heads 2 cq, 2 cq + 1
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      gm[e] = sm_m[2 * cq + e];
#pragma unroll
      for (int w = 1; w < W; ++w) gm[e] = fmaxf(gm[e], sm_m[w * kQ4Heads + 2 * cq + e]);
      share[e] = ex2(m[e] - gm[e]);
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      // The unit first: it may be small and O large, and its product with the share below FP32.
      const float c0 = ref_of(ref[t * NG / 8], 0) * 0x1p24f, c1 = ref_of(ref[t * NG / 8], 1) * 0x1p24f;
      sm_o[warp * kQ4Frags + t * 32 + lane] =
          make_float4(o[t][0] * c0 * share[0], o[t][1] * c1 * share[1], (o[t][2] - o[t][0]) * (c0 * 0.0625f) * share[0],
                      (o[t][3] - o[t][1]) * (c1 * 0.0625f) * share[1]);
    }
    __syncthreads();
    float den[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int w = 0; w < W; ++w)
        den[e] = fmaf(sm_l[w * kQ4Heads + 2 * cq + e], ex2(sm_m[w * kQ4Heads + 2 * cq + e] - gm[e]), den[e]);
    // The output, or a piece of it; a thread's float4s are all of heads 2 cq and + 1.
    const long long slot = 2ll * blockIdx.x + (s0 == lo ? 0 : 1);
#pragma unroll
    for (int k = threadIdx.x; k < kQ4Frags; k += kQ4Threads) {
      float4 v = sm_o[k];
#pragma unroll
      for (int w = 1; w < W; ++w) {
        const float4 u = sm_o[w * kQ4Frags + k];
        v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
      }
      if (whole)
        store_frag<T, NG>(p, row_b, h0, nh, k, v, den[0], den[1]);
      else
        __stcg(reinterpret_cast<float4 *>(p.scratch) + slot * kQ4Frags + k, v);
    }
    if (!whole && threadIdx.x < 4)
      __stcg(reinterpret_cast<float4 *>(p.scratch) + 2ll * p.ctas * kQ4Frags + slot * (kQ4Heads / 2) + cq,
             make_float4(gm[0], den[0], gm[1], den[1]));
    if (!whole && p.counters) {
      // The CTA that finishes the row last merges it and resets the counter.
      int *last = reinterpret_cast<int *>(smem + S::flag_off + 8);
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        int32_t *counter = p.counters + (long long)row_b * R + row_r;
        *last = atomicAdd(counter, 1) == pieces - 1;
        if (*last) *counter = 0;
      }
      __syncthreads();
      if (*last) {
        __threadfence();
        merge_row<T, NG>(p, row_b, h0, nh, first, pieces, late);
      }
    }
    __syncthreads();  // statistics and outputs are free again
    s0 = s1;
  }
  if (dead_at >= 0 && lane == 0) {
    // Copies still in flight land before the CTA leaves (bounded again).
    const WaitCtx drain{reinterpret_cast<volatile int *>(smem + S::flag_off + 4), p.c.status};
    for (int k = dead_at; k < issued; ++k) mbar_wait<false>(bar0 + 8 * (k % kQ4Stages), (k / kQ4Stages) & 1, drain);
  }
}

// The merge as a launch of its own, one CTA per row.
template <typename T, int NG>
__global__ void __launch_bounds__(kQ4Threads) attn_q4_merge_kernel(const __grid_constant__ AttnQ4Params p) {
  pdl_enter(p.pdl);
  const int R = p.c.kv_heads * p.head_blocks;
  const int b = blockIdx.x / R, r = blockIdx.x - b * R;
  const Q4Deal deal = q4_deal(p, lane_id() < p.c.rows ? chunks_of(seq_of(p, lane_id())) : 0);
  auto units = [&](int i) {
    const int n = chunks_of(seq_of(p, i));
    return deal.whole ? pieces_of(n, deal.size, rcp_of(deal.size)) : n;
  };
  int first = 0;
  for (int i = lane_id(); i < b; i += 32) first += units(i);
  int pieces = units(b);
  first = __reduce_add_sync(0xffffffffu, first) * R + r * pieces;
  bool late = false;
  if (!deal.whole && pieces > 0) {
    const int begin = first;
    first = begin / deal.size;
    pieces = (begin + pieces - 1) / deal.size - first + 1;
    late = first * deal.size < begin;
  }
  if (pieces < 2) return;  // written already
  const int hb = r % p.head_blocks;
  merge_row<T, NG>(p, b, r / p.head_blocks * p.group + hb * p.block_heads, min(p.block_heads, p.group - hb * p.block_heads),
                   first, pieces, late);
}

template <typename T, int NG, int P>
cudaError_t launch_attn(const AttnQ4Params &p, int rows, cudaStream_t s) {
  auto kern = attn_q4_kernel<T, NG, P>;
  cudaError_t e = prepare_kernel_attributes(reinterpret_cast<const void *>(kern));
  if (e != cudaSuccess) return e;
  e = launch_ex(kern, dim3(p.ctas), dim3(kQ4Threads), Q4Smem<NG>::bytes, s, 1, p.pdl != 0, p);
  if (e != cudaSuccess || p.by_row || p.counters) return e;
  return launch_ex(attn_q4_merge_kernel<T, NG>, dim3(rows), dim3(kQ4Threads), 0, s, 1, p.pdl != 0, p);
}

template <typename T, int NG>
cudaError_t launch_attn_g(const AttnQ4Params &p, int rows, cudaStream_t s) {
  switch (p.c.page_size) {
    case 16: return launch_attn<T, NG, 16>(p, rows, s);
    case 32: return launch_attn<T, NG, 32>(p, rows, s);
    default: return launch_attn<T, NG, 64>(p, rows, s);
  }
}

template <typename T>
cudaError_t launch_attn_t(const AttnQ4Params &p, int rows, cudaStream_t s) {
  switch (p.c.ng) {
    case 1: return launch_attn_g<T, 1>(p, rows, s);
    case 2: return launch_attn_g<T, 2>(p, rows, s);
    default: return launch_attn_g<T, 4>(p, rows, s);
  }
}

// How a call is dealt out.  Rows that fit the GPU at once and are short are not
// split: a merge would cost more than it gives.  Else there are as many CTAs as
// the GPU holds at once, or as there can be warps with a chunk.
struct Q4Plan {
  long long rows;
  int ctas, by_row;
  long long scratch_floats;
};

Q4Plan q4_plan(const dak_kv4_cache *c, int num_q_heads, int max_seq_len) {
  Q4Plan plan;
  const int group = num_q_heads / c->kv_heads;
  plan.rows = (long long)c->batch * c->kv_heads * ((group + kQ4Heads - 1) / kQ4Heads);
  const long long chunks = ((long long)max_seq_len + kQ4Chunk - 1) / kQ4Chunk;
  const int resident = device_sms() * kQ4PerSm;
  plan.by_row = plan.rows <= resident && chunks <= kQ4RowChunks;
  plan.ctas = plan.by_row ? (int)plan.rows
                          : (int)std::min<long long>(resident, plan.rows * ((chunks + kQ4Warps - 1) / kQ4Warps));
  plan.scratch_floats = plan.by_row ? 0 : 2ll * plan.ctas * kQ4Heads * (kKv4Dim + 2);
  return plan;
}

}  // namespace
}  // namespace dak

extern "C" int dak_attn_decode_paged_q4(const dak_kv4_cache *cache, const dak_attn_q4_args *a, void *stream) {
  using namespace dak;
  if (!a) return fail(DAK_ERR_INVALID_ARG, "args is null");
  int st = kv4_check(cache);
  if (st) return st;
  if (a->dtype != DAK_DTYPE_F16 && a->dtype != DAK_DTYPE_BF16)
    return fail(DAK_ERR_UNSUPPORTED, "attention supports float16 and bfloat16 only");
  if (a->num_q_heads <= 0 || a->num_q_heads % cache->kv_heads)
    return fail(DAK_ERR_INVALID_ARG, "num_q_heads must be a positive multiple of kv_heads");
  if (a->max_seq_len <= 0 || (int64_t)cache->max_pages * cache->page_size < a->max_seq_len)
    return fail(DAK_ERR_INVALID_ARG, "max_seq_len must be positive and within the block table's pages");
  if (a->max_seq_len > 0x7fffffff - kQ4Chunk) return fail(DAK_ERR_UNSUPPORTED, "max_seq_len is too large for one launch");
  if (!a->query || !a->out || !a->seq_lens) return fail(DAK_ERR_INVALID_ARG, "query, out and seq_lens are required");
  if (a->q_stride_b % 8 || a->q_stride_h % 8 || a->o_stride_b % 8 || a->o_stride_h % 8 ||
      ((reinterpret_cast<uintptr_t>(a->query) | reinterpret_cast<uintptr_t>(a->out) |
        reinterpret_cast<uintptr_t>(a->scratch)) & 15u))
    return fail(DAK_ERR_ALIGNMENT, "query, out and scratch must be 16-byte aligned, strides multiples of 8 elements");
  const BlockGrid q = {a->query, cache->batch, 2 * a->q_stride_b, a->num_q_heads, 2 * a->q_stride_h, 2 * kKv4Dim};
  const BlockGrid out = {a->out, cache->batch, 2 * a->o_stride_b, a->num_q_heads, 2 * a->o_stride_h, 2 * kKv4Dim};
  if (overlaps_itself(out)) return fail(DAK_ERR_INVALID_ARG, "heads of out overlap");
  const bool in_place = a->query == a->out && (cache->batch == 1 || a->q_stride_b == a->o_stride_b) &&
                        (a->num_q_heads == 1 || a->q_stride_h == a->o_stride_h);
  if (!in_place && overlap(q, out)) return fail(DAK_ERR_INVALID_ARG, "out overlaps the query without being it");
  const Q4Plan plan = q4_plan(cache, a->num_q_heads, a->max_seq_len);
  if (plan.rows > 0x7fffffffll / (((int64_t)a->max_seq_len + kQ4Chunk - 1) / kQ4Chunk))
    return fail(DAK_ERR_UNSUPPORTED, "batch x heads x max_seq_len is too large for one launch");
  if (plan.scratch_floats > 0 && (!a->scratch || a->scratch_floats < plan.scratch_floats))
    return fail(DAK_ERR_INVALID_ARG, "attention needs %lld floats of scratch", (long long)plan.scratch_floats);
  const void *ptrs[5] = {a->query, a->out, a->seq_lens, plan.by_row ? nullptr : a->scratch,
                         plan.by_row ? nullptr : a->merge_counters};
  for (const void *q : ptrs)
    if (q && (st = check_gpu_accessible(q, "attention buffer"))) return st;
  AttnQ4Params p;
  std::memset(&p, 0, sizeof(p));
  if ((st = kv4_view(cache, &p.c))) return st;
  p.query = static_cast<const uint16_t *>(a->query);
  p.q_stride_b = a->q_stride_b;
  p.q_stride_h = a->q_stride_h;
  p.out = static_cast<uint16_t *>(a->out);
  p.o_stride_b = a->o_stride_b;
  p.o_stride_h = a->o_stride_h;
  p.seq_lens = a->seq_lens;
  p.scratch = plan.by_row ? nullptr : a->scratch;
  p.counters = plan.by_row ? nullptr : a->merge_counters;
  p.num_q_heads = a->num_q_heads;
  p.group = a->num_q_heads / cache->kv_heads;
  p.head_blocks = (p.group + kQ4Heads - 1) / kQ4Heads;
  p.block_heads = (p.group + p.head_blocks - 1) / p.head_blocks;
  p.max_seq_len = a->max_seq_len;
  p.ctas = plan.ctas;
  p.by_row = plan.by_row;
  p.scale_log2 = a->scaling * 1.4426950408889634f;
  p.pdl = decode_pdl_enabled() ? 1 : 0;
  auto s = static_cast<cudaStream_t>(stream);
  const int rows = (int)plan.rows;
  return cuda_status(a->dtype == DAK_DTYPE_F16 ? launch_attn_t<__half>(p, rows, s) : launch_attn_t<__nv_bfloat16>(p, rows, s),
                     "4-bit attention launch");
}

extern "C" int64_t dak_attn_q4_scratch(const dak_kv4_cache *cache, int num_q_heads, int max_seq_len) {
  using namespace dak;
  if (kv4_check(cache) || num_q_heads <= 0 || num_q_heads % cache->kv_heads || max_seq_len <= 0) return -1;
  return q4_plan(cache, num_q_heads, max_seq_len).scratch_floats;
}
