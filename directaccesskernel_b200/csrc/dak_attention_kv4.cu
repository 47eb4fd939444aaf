// dak_attention_kv4.cu - decode attention over the 4-bit paged KV cache
// (dak_kv4.cuh), whose pages lie in HBM or in pinned host memory.
//
// One query token per sequence: o = softmax(scaling q K^T) V over the first
// seq_lens[b] tokens, K and V being scale * code + zero.  One CTA per
// (sequence, KV head, block of up to 8 query heads, split of the tokens); the
// splits' (o, m, l) are merged with log-sum-exp.  Scores are kept in base 2.
// A sequence of no tokens gives zeros.
#include <cudaTypedefs.h>

#include <cfloat>
#include <cstring>
#include <type_traits>

#include "dak_common.cuh"
#include "dak_host.h"
#include "dak_kv4.cuh"

namespace dak {
namespace {

constexpr int kQ4Warps = 4;
constexpr int kQ4Threads = kQ4Warps * 32;
constexpr int kQ4Heads = 8;    // query heads per CTA: the MMA's N
constexpr int kQ4Chunk = 64;   // tokens a warp takes at a time
constexpr int kQ4Stages = 2;   // chunks in flight per warp

struct alignas(64) AttnQ4Params {
  CUtensorMap map[2];  // device, host pool: dims {64 bytes, slab rows, pages x heads}
  Kv4Cache c;
  const uint16_t *query;
  long long q_stride_b, q_stride_h;
  uint16_t *out;
  long long o_stride_b, o_stride_h;
  const int32_t *seq_lens;
  float *partial_o, *partial_ml;
  int32_t *counters;
  int num_q_heads, group, block_heads, head_blocks;  // group: query heads per KV head
  int max_seq_len, split_size, num_splits;
  float scale_log2;                                  // scaling * log2(e)
  int pdl;
};

// Shared memory of a CTA: per warp a ring of chunks, then barriers and the
// warps' softmax statistics.  After the last chunk a warp's ring holds its
// partial outputs.
template <int NG>
struct Q4Smem {
  static constexpr uint32_t stage = 2 * kQ4Chunk * (64 + 4 * NG);
  static constexpr uint32_t bar_off = kQ4Warps * kQ4Stages * stage;
  static constexpr uint32_t m_off = bar_off + kQ4Warps * kQ4Stages * 8;  // [warps][heads]
  static constexpr uint32_t l_off = m_off + kQ4Warps * kQ4Heads * 4;
  static constexpr uint32_t flag_off = l_off + kQ4Warps * kQ4Heads * 4;
  static constexpr uint32_t bytes = flag_off + 16 + 512;  // 512: alignment
  static_assert(stage % 512 == 0 && kQ4Stages * stage >= kQ4Heads * kKv4Dim * 4, "a ring must hold a partial output");
};

__device__ __forceinline__ void tma_load_slab(uint32_t dst, const CUtensorMap *map, int slab, uint32_t bar,
                                              uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%2, %2, %3}], [%4], %5;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(slab), "r"(bar), "l"(policy)
      : "memory");
}

// Where the 64-byte TMA swizzle put byte `lb` (below 64) of the row `row` rows
// after offset C of a stage (C a multiple of 64, the stage 512-byte aligned):
// bits 4-5 are xored with bits 7-8.  C is a constant at every call, so what
// depends on the lane is the same few values for all tiles.
__device__ __forceinline__ uint32_t swz(uint32_t C, uint32_t row, uint32_t lb) {
  return C + row * 64 + (lb ^ ((((C >> 7) + ((row + ((C >> 6) & 1u)) >> 1)) & 3u) << 4));
}

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
// The transpose of an 8x8 matrix of 16-bit elements spread over the warp.
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// floor(log2 s) of a float16 s >= 0 given by its bits; -24 (its smallest
// exponent) for 0.
__device__ __forceinline__ float exponent_of(uint32_t bits) {
  const float s = __half2float(__ushort_as_half((unsigned short)bits));
  return fmaxf((float)((int)(__float_as_uint(s) >> 23) - 127), -24.f);
}

// Splits that hold tokens of a sequence (at least one, which writes the zeros of
// an empty sequence).
__device__ __forceinline__ int live_splits(const AttnQ4Params &p, int seq) {
  return max(1, (seq + p.split_size - 1) / p.split_size);
}

// Log-sum-exp merge of a block of heads' split partials by 128 threads, in split
// order: first each warp forms the maximum and denominator of two heads, then
// thread d sums dim d of every head.
template <typename T>
__device__ __forceinline__ void merge_q4(const AttnQ4Params &p, int b, int h0, int nh, int splits, float *sm) {
  const long long base = ((long long)b * p.num_q_heads + h0) * p.num_splits;
  for (int h = warp_id(); h < nh; h += kQ4Warps) {
    const float2 *ml = reinterpret_cast<const float2 *>(p.partial_ml) + base + (long long)h * p.num_splits;
    float gm = -FLT_MAX, den = 0.f;
    for (int s = lane_id(); s < splits; s += 32) gm = fmaxf(gm, __ldcg(ml + s).x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, x));
    for (int s = lane_id(); s < splits; s += 32) {
      const float2 v = __ldcg(ml + s);
      den = fmaf(v.y, ex2(v.x - gm), den);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) den += __shfl_xor_sync(0xffffffffu, den, x);
    if (lane_id() == 0) {
      sm[h] = gm;
      sm[kQ4Heads + h] = den;
    }
  }
  __syncthreads();
  const int d = threadIdx.x;
  for (int h = 0; h < nh; ++h) {
    const long long at = base + (long long)h * p.num_splits;
    const float gm = sm[h], den = sm[kQ4Heads + h];
    float acc = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s)
      acc = fmaf(__ldcg(p.partial_o + (at + s) * kKv4Dim + d), ex2(__ldcg(p.partial_ml + (at + s) * 2) - gm), acc);
    p.out[b * p.o_stride_b + (h0 + h) * p.o_stride_h + d] = Elem<T>::from_float(den == 0.f ? 0.f : acc / den);
  }
}

template <typename T, int NG, int P>
__global__ void __launch_bounds__(kQ4Threads, NG == 4 ? 2 : 3) attn_q4_kernel(const __grid_constant__ AttnQ4Params p) {
  extern __shared__ uint8_t smem_raw[];
  using S = Q4Smem<NG>;
  // The weights of a float16 output are split into two float16 terms.
  constexpr bool kTwoTerms = std::is_same<T, __half>::value;
  uint8_t *smem = smem_raw + ((512u - (smem_u32(smem_raw) & 511u)) & 511u);
  const uint32_t sbase = smem_u32(smem);
  pdl_enter(p.pdl);
  const int warp = warp_id(), lane = lane_id();
  const int g = lane >> 2, cq = lane & 3;  // fragment row, column pair
  int i = blockIdx.x;
  const int split = i % p.num_splits;
  i /= p.num_splits;
  const int hb = i % p.head_blocks;
  i /= p.head_blocks;
  const int kvh = i % p.c.kv_heads;
  const int b = i / p.c.kv_heads;
  const int seq = max(0, min(p.seq_lens[b], p.max_seq_len));
  const int splits = live_splits(p, seq);
  if (split >= splits) return;
  const int h0 = kvh * p.group + hb * p.block_heads;
  const int nh = min(p.block_heads, p.group - hb * p.block_heads);
  const int t0 = split * p.split_size, t1 = min(seq, t0 + p.split_size);
  const int chunks = (t1 - t0 + kQ4Chunk - 1) / kQ4Chunk;
  const int mine = chunks > warp ? (chunks - warp + kQ4Warps - 1) / kQ4Warps : 0;  // this warp's chunks
  constexpr int ppc = kQ4Chunk / P;  // pages per chunk
  constexpr uint32_t half = kv4_half_bytes(P, NG), slab = 2 * half;

  const uint32_t ring = sbase + warp * kQ4Stages * S::stage;
  const uint32_t bar0 = sbase + S::bar_off + warp * kQ4Stages * 8;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + S::flag_off);
  const WaitCtx wc{abort_flag, p.c.status};
  if (threadIdx.x == 0) {
    for (int s = 0; s < kQ4Warps * kQ4Stages; ++s) mbar_init(sbase + S::bar_off + 8 * s, 1);
    abort_flag[0] = abort_flag[1] = 0;  // [1]: of the wait for copies in flight
    fence_mbar_init();
  }
  __syncthreads();

  // Block-table entries: lane l holds entry l of a window of 32 / ppc chunks, and
  // the window after it is already on its way.
  constexpr int per_win = 32 / ppc;
  const int32_t *row = p.c.table + (long long)b * p.c.table_stride;
  const int last_page = (t1 - 1) / P;
  auto window = [&](int first) {  // entries of chunks first .. of this warp
    const int j = first + lane / ppc;
    const int page = (t0 + (warp + j * kQ4Warps) * kQ4Chunk) / P + lane % ppc;
    return j < mine && page <= last_page ? row[page] : 0;
  };
  int cur = window(0), nxt = window(per_win);
  const uint64_t pol = l2_policy_evict_first();
  auto issue = [&](int j) {  // chunk j of this warp into its stage
    if (j % per_win == 0 && j > 0) {
      cur = nxt;
      nxt = window(j + per_win);
    }
    const int entry = __shfl_sync(0xffffffffu, cur, (j % per_win) * ppc + lane % ppc);
    const int first = t0 + (warp + j * kQ4Warps) * kQ4Chunk;
    const int pages = min(ppc, last_page - first / P + 1);
    const int s = j % kQ4Stages;
    if (lane == 0) mbar_arrive_expect_tx(bar0 + 8 * s, pages * slab);
    __syncwarp();
    if (lane < pages) {
      const int tier = entry < 0 ? 1 : 0;
      long long page = entry < 0 ? -1ll - entry : entry;
      if (page >= p.c.pages[tier]) {  // the copy starts past the map's end and reads zeros
        atomicCAS(p.c.status, 0, DAK_ERR_INVALID_ARG);
        page = max(1ll, p.c.pages[tier]);
      }
      tma_load_slab(ring + s * S::stage + lane * slab, &p.map[tier], (int)(page * p.c.kv_heads + kvh), bar0 + 8 * s, pol);
    }
    __syncwarp();
  };
  const int ahead = min(mine, kQ4Stages);
  for (int j = 0; j < ahead; ++j) issue(j);

  // Word w (0..3) of a K row that this lane multiplies, 8 dims each: all the
  // words of one group meet in the same MMA steps.
  auto k_word = [&](int w) {
    return NG == 1 ? 4 * cq + w : NG == 2 ? 8 * (w >> 1) + 2 * cq + (w & 1) : 4 * w + cq;
  };
  // Query of head g: scaled by a power of two to below 2^14 and to float16 (the
  // values that float16 cannot hold are 2^-38 of the largest), and summed
  // over each group for the zeros' share.
  uint32_t qf[8][2];
  float qs[2][NG], f[2];
  {
    float x[4][8], mx = 0.f, sum[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) sum[n] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (g < nh)
        v = *reinterpret_cast<const uint4 *>(p.query + b * p.q_stride_b + (h0 + g) * p.q_stride_h + 8 * k_word(w));
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 y = Elem<T>::to_float2(u[e]);
        x[w][2 * e] = y.x;
        x[w][2 * e + 1] = y.y;
        mx = fmaxf(mx, fmaxf(fabsf(y.x), fabsf(y.y)));
      }
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const int k = mx > 0.f ? max(-100, min(100, 13 - ((int)(__float_as_uint(mx) >> 23) - 127))) : 0;
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
        sum[w * NG / 4] += (a + c) + (d + e);
      }
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 1);
      sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 2);
    }
    const float fh = fabsf(p.scale_log2) * __uint_as_float((uint32_t)(127 + 24 - k) << 23);
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // lane 4h holds head h
      const int src = 4 * (2 * cq + e);
      f[e] = __shfl_sync(0xffffffffu, fh, src);
#pragma unroll
      for (int n = 0; n < NG; ++n) qs[e][n] = __shfl_sync(0xffffffffu, sum[n], src) * 0x1p-24f;
    }
  }

  // V: this lane takes 4 dims at a time (piece x) of tokens 2 cq, 2 cq + 1 (and 8
  // on).  Odd columns read the second token first, which spreads a warp's reads
  // over all banks; the byte selectors put the pair back in order.
  const uint32_t flip = cq & 1;
  const uint32_t sel_lo = flip ? 0x1054u : 0x5410u, sel_hi = flip ? 0x3276u : 0x7632u;
  const uint32_t sel_g = (g & 1) ? sel_hi : sel_lo;

  // Statistics: weights are 2^(score - m).  m is the largest score so far plus E,
  // the exponent of the warp's largest V scale so far, so that weight x scale is
  // below 2 and float16 holds it whatever V's magnitude.
  float o[8][4], m[2] = {-FLT_MAX, -FLT_MAX}, l[2] = {0.f, 0.f}, E = -24.f;
  uint32_t s_max = 0u;
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[t][e] = 0.f;

  // One chunk of `valid` tokens in the stage at `st`.
  auto chunk = [&](const uint8_t *st, int valid, auto full_c) {
    constexpr bool kFull = decltype(full_c)::value;
    // Offset of tile t's first code row (V: + half) and of its pairs of token g + 8r.
    auto rows_at = [](int t) { return (uint32_t)((16 * t) / P * slab + (16 * t) % P * 64); };
    auto pairs_at = [&](int t, int r) {
      const uint32_t c = (16 * t) / P * slab + P * 64 + (16 * t) % P * (4 * NG);
      return NG == 4 ? swz(c + 128 * r, g >> 2, 16 * (g & 3)) : NG == 2 ? swz(c + 64 * r, 0, 8 * g) : swz(c, 0, 4 * g + 32 * r);
    };
    auto vpairs_at = [&](int t, int r) {
      const uint32_t c = (16 * t) / P * slab + half + P * 64 + (16 * t) % P * (4 * NG);
      return NG == 4 ? swz(c + 128 * r, g >> 2, 16 * (g & 3)) : NG == 2 ? swz(c + 64 * r, 0, 8 * g) : swz(c, 0, 4 * g + 32 * r);
    };
    float y[4][4];  // raw scores: tile, {token g, g + 8} x {head 2 cq, 2 cq + 1}
    float mx[2] = {-INFINITY, -INFINITY};
    uint32_t vp[4][2][NG];
    __half2 vmax = __float2half2_rn(0.f);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (!kFull && t * 16 >= valid) continue;
      // S^T = K Q^T with the codes as they are: a nibble at bits 0-3 of a half word
      // is the subnormal code * 2^-24, at bits 4-7 code * 2^-20 (its q is / 16).
      uint32_t w0[4], w1[4];  // tokens g and g + 8
      if constexpr (NG == 1) {
        const uint8_t *a = st + swz(rows_at(t), g, 16 * cq);
        const uint4 u = *reinterpret_cast<const uint4 *>(a), v = *reinterpret_cast<const uint4 *>(a + 512);
        w0[0] = u.x, w0[1] = u.y, w0[2] = u.z, w0[3] = u.w;
        w1[0] = v.x, w1[1] = v.y, w1[2] = v.z, w1[3] = v.w;
      } else if constexpr (NG == 2) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint8_t *a = st + swz(rows_at(t), g, 32 * n + 8 * cq);
          const uint2 u = *reinterpret_cast<const uint2 *>(a), v = *reinterpret_cast<const uint2 *>(a + 512);
          w0[2 * n] = u.x, w0[2 * n + 1] = u.y;
          w1[2 * n] = v.x, w1[2 * n + 1] = v.y;
        }
      } else {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint8_t *a = st + swz(rows_at(t), g, 16 * n + 4 * cq);
          w0[n] = *reinterpret_cast<const uint32_t *>(a);
          w1[n] = *reinterpret_cast<const uint32_t *>(a + 512);
        }
      }
      uint32_t kp[2][NG];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        load_pairs<NG>(st + pairs_at(t, r), kp[r]);
        load_pairs<NG>(st + vpairs_at(t, r), vp[t][r]);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          if (!kFull && t * 16 + 8 * r + g >= valid) vp[t][r][n] = 0u;  // anything may lie behind the last token
          vmax = __hmax2(vmax, *reinterpret_cast<const __half2 *>(&vp[t][r][n]));
        }
      }
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = n * 4 / NG; w < (n + 1) * 4 / NG; ++w) {
          mma_f16(acc, w0[w] & 0x000F000Fu, w1[w] & 0x000F000Fu, w0[w] & 0x00F000F0u, w1[w] & 0x00F000F0u, qf[2 * w][0],
                  qf[2 * w][1]);
          const uint32_t s0 = w0[w] >> 8, s1 = w1[w] >> 8;
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
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (kFull || t * 16 + 8 * r + g < valid) mx[e] = fmaxf(mx[e], y[t][2 * r + e]);
    }
    // A larger V scale than any before raises E (rarely, after the first chunks).
    const uint32_t sm = __reduce_max_sync(0xffffffffu, *reinterpret_cast<const uint32_t *>(&vmax) & 0xffffu);
    float rise = 0.f;
    if (sm > s_max) {
      s_max = sm;
      const float en = fmaxf(E, exponent_of(sm));
      rise = en - E;
      E = en;
    }
    float alpha[2], zs[2][NG];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x <= 16; x <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], x));
      const float mn = fmaxf(m[e] + rise, fmaf(mx[e], f[e], E));
      alpha[e] = ex2(m[e] - mn);
      m[e] = mn;
      l[e] *= alpha[e];
#pragma unroll
      for (int n = 0; n < NG; ++n) zs[e][n] = 0.f;
    }
    // Weights, and the zeros' share of the output: sum_t p_t zero_t per group.
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (!kFull && t * 16 >= valid) continue;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float w = ex2(fmaf(y[t][2 * r + e], f[e], -m[e]));
          if (!kFull && t * 16 + 8 * r + g >= valid) w = 0.f;
          y[t][2 * r + e] = w;
          l[e] += w;
#pragma unroll
          for (int n = 0; n < NG; ++n) zs[e][n] = fmaf(w, half2_of(vp[t][r][n]).y, zs[e][n]);
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) zs[e][n] += __shfl_xor_sync(0xffffffffu, zs[e][n], x);
    // O rows: even dims count codes * 2^-24, odd dims * 2^-20.  Adding the zeros'
    // share chunk by chunk keeps O centred, so nothing cancels at the end.
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const float even = zs[e][n] * 0x1p-24f, odd = zs[e][n] * 0x1p-20f;
#pragma unroll
        for (int t = 8 * n / NG; t < 8 * (n + 1) / NG; ++t) {
          o[t][e] = fmaf(o[t][e], alpha[e], even);
          o[t][2 + e] = fmaf(o[t][2 + e], alpha[e], odd);
        }
      }
    // O^T += V^T P^T
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (!kFull && t * 16 >= valid) continue;
      uint32_t bf[NG][2];
      [[maybe_unused]] uint32_t bl[NG][2];
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float s = half2_of(vp[t][r][n]).x;
          const float a = y[t][2 * r] * s, c = y[t][2 * r + 1] * s;
          const uint32_t hi = pack_half2(a, c);
          bf[n][r] = movmatrix(hi);
          if constexpr (kTwoTerms) {
            const float2 back = half2_of(hi);
            bl[n][r] = movmatrix(pack_half2(a - back.x, c - back.y));
          }
        }
      uint32_t x[2][4];  // token pairs (2 cq, +1) and (2 cq + 8, +9): 4 pieces of 4 dims
      const uint32_t row0 = 2 * cq + flip, row1 = 2 * cq + 1 - flip;
      const uint32_t vc = rows_at(t) + half;
      if constexpr (NG == 1) {
        const uint8_t *a = st + swz(vc, row0, 8 * g), *c = st + swz(vc, row1, 8 * g);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint2 u = *reinterpret_cast<const uint2 *>(a + 512 * r), v = *reinterpret_cast<const uint2 *>(c + 512 * r);
          x[r][0] = __byte_perm(u.x, v.x, sel_lo);
          x[r][1] = __byte_perm(u.x, v.x, sel_hi);
          x[r][2] = __byte_perm(u.y, v.y, sel_lo);
          x[r][3] = __byte_perm(u.y, v.y, sel_hi);
        }
      } else if constexpr (NG == 2) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint8_t *a = st + swz(vc, row0, 32 * n + 4 * g), *c = st + swz(vc, row1, 32 * n + 4 * g);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t u = *reinterpret_cast<const uint32_t *>(a + 512 * r);
            const uint32_t v = *reinterpret_cast<const uint32_t *>(c + 512 * r);
            x[r][2 * n] = __byte_perm(u, v, sel_lo);
            x[r][2 * n + 1] = __byte_perm(u, v, sel_hi);
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint8_t *a = st + swz(vc, row0, 16 * n + 4 * (g >> 1)), *c = st + swz(vc, row1, 16 * n + 4 * (g >> 1));
#pragma unroll
          for (int r = 0; r < 2; ++r)
            x[r][n] = __byte_perm(*reinterpret_cast<const uint32_t *>(a + 512 * r),
                                  *reinterpret_cast<const uint32_t *>(c + 512 * r), sel_g);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = q * NG / 4;
        const uint32_t s0 = x[0][q] >> 8, s1 = x[1][q] >> 8;
        mma_f16(o[2 * q], x[0][q] & 0x000F000Fu, x[0][q] & 0x00F000F0u, x[1][q] & 0x000F000Fu, x[1][q] & 0x00F000F0u,
                bf[n][0], bf[n][1]);
        mma_f16(o[2 * q + 1], s0 & 0x000F000Fu, s0 & 0x00F000F0u, s1 & 0x000F000Fu, s1 & 0x00F000F0u, bf[n][0], bf[n][1]);
        if constexpr (kTwoTerms) {
          mma_f16(o[2 * q], x[0][q] & 0x000F000Fu, x[0][q] & 0x00F000F0u, x[1][q] & 0x000F000Fu, x[1][q] & 0x00F000F0u,
                  bl[n][0], bl[n][1]);
          mma_f16(o[2 * q + 1], s0 & 0x000F000Fu, s0 & 0x00F000F0u, s1 & 0x000F000Fu, s1 & 0x00F000F0u, bl[n][0],
                  bl[n][1]);
        }
      }
    }
  };

  bool ok = true;
  for (int j = 0; j < mine; ++j) {
    const int s = j % kQ4Stages;
    ok = mbar_wait<false>(bar0 + 8 * s, (j / kQ4Stages) & 1, wc);
    if (!__all_sync(0xffffffffu, ok)) {
      // Gave up: let this warp's copies land (bounded again), then leave.
      if (lane == 0) {
        const WaitCtx drain{reinterpret_cast<volatile int *>(smem + S::flag_off + 4), p.c.status};
        for (int k = j; k < min(mine, j + kQ4Stages); ++k)
          mbar_wait<false>(bar0 + 8 * (k % kQ4Stages), (k / kQ4Stages) & 1, drain);
      }
      __syncwarp();
      break;
    }
    const uint8_t *st = smem + (warp * kQ4Stages + s) * S::stage;
    const int valid = min(kQ4Chunk, t1 - (t0 + (warp + j * kQ4Warps) * kQ4Chunk));
    if (valid == kQ4Chunk)
      chunk(st, valid, std::true_type{});
    else
      chunk(st, valid, std::false_type{});
    __syncwarp();
    if (j + kQ4Stages < mine) issue(j + kQ4Stages);
  }

  // Merge the warps: each leaves (m, l, o) of its heads, o in its own ring.
  float *sm_m = reinterpret_cast<float *>(smem + S::m_off), *sm_l = reinterpret_cast<float *>(smem + S::l_off);
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int x = 4; x <= 16; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
  float *ring_f = reinterpret_cast<float *>(smem + warp * kQ4Stages * S::stage);  // [head][dim]
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int h = 2 * cq + e;
    if (h >= nh) continue;
    if (g == 0) {
      sm_m[warp * kQ4Heads + h] = m[e];
      sm_l[warp * kQ4Heads + h] = l[e];
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const int q = t >> 1;
      const int d = (NG == 1 ? 16 * g + 4 * q : NG == 2 ? 64 * (q >> 1) + 8 * g + 4 * (q & 1) : 32 * q + 4 * g) + 2 * (t & 1);
      *reinterpret_cast<float2 *>(ring_f + h * kKv4Dim + d) = make_float2(o[t][e] * 0x1p24f, o[t][2 + e] * 0x1p20f);
    }
  }
  __syncthreads();
  const int d = threadIdx.x;
  for (int h = 0; h < nh; ++h) {
    float gm = -FLT_MAX;
#pragma unroll
    for (int w = 0; w < kQ4Warps; ++w) gm = fmaxf(gm, sm_m[w * kQ4Heads + h]);
    float den = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kQ4Warps; ++w) {
      const float c = ex2(sm_m[w * kQ4Heads + h] - gm);
      den = fmaf(sm_l[w * kQ4Heads + h], c, den);
      acc = fmaf(reinterpret_cast<const float *>(smem + w * kQ4Stages * S::stage)[h * kKv4Dim + d], c, acc);
    }
    if (splits == 1) {
      p.out[b * p.o_stride_b + (h0 + h) * p.o_stride_h + d] = Elem<T>::from_float(den == 0.f ? 0.f : acc / den);
    } else {
      const long long at = ((long long)b * p.num_q_heads + h0 + h) * p.num_splits + split;
      p.partial_o[at * kKv4Dim + d] = acc;
      if (d == 0) {
        p.partial_ml[at * 2] = gm;
        p.partial_ml[at * 2 + 1] = den;
      }
    }
  }
  if (splits > 1 && p.counters) {
    // The split that finishes last merges all of them and resets the counter.
    int *last = reinterpret_cast<int *>(smem + S::flag_off + 8);
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      int32_t *counter = p.counters + blockIdx.x / p.num_splits;
      *last = atomicAdd(counter, 1) == splits - 1;
      if (*last) *counter = 0;
    }
    __syncthreads();
    if (*last) {
      __threadfence();
      merge_q4<T>(p, b, h0, nh, splits, sm_m);
    }
  }
}

// The merge as a launch of its own, one CTA per block of heads.
template <typename T>
__global__ void __launch_bounds__(kQ4Threads) attn_q4_merge_kernel(const __grid_constant__ AttnQ4Params p) {
  __shared__ float sm[2 * kQ4Heads];
  pdl_enter(p.pdl);
  int i = blockIdx.x;
  const int hb = i % p.head_blocks;
  i /= p.head_blocks;
  const int kvh = i % p.c.kv_heads;
  const int b = i / p.c.kv_heads;
  const int splits = live_splits(p, max(0, min(p.seq_lens[b], p.max_seq_len)));
  if (splits == 1) return;  // written already
  merge_q4<T>(p, b, kvh * p.group + hb * p.block_heads, min(p.block_heads, p.group - hb * p.block_heads), splits, sm);
}

template <typename T, int NG, int P>
cudaError_t launch_attn(const AttnQ4Params &p, long long grid, cudaStream_t s) {
  auto kern = attn_q4_kernel<T, NG, P>;
  cudaError_t e = prepare_kernel_attributes(reinterpret_cast<const void *>(kern));
  if (e != cudaSuccess) return e;
  e = launch_ex(kern, dim3((unsigned)grid), dim3(kQ4Threads), Q4Smem<NG>::bytes, s, 1, p.pdl != 0, p);
  if (e != cudaSuccess || p.num_splits == 1 || p.counters) return e;
  return launch_ex(attn_q4_merge_kernel<T>, dim3((unsigned)(grid / p.num_splits)), dim3(kQ4Threads), 0, s, 1, p.pdl != 0, p);
}

template <typename T, int NG>
cudaError_t launch_attn_g(const AttnQ4Params &p, long long grid, cudaStream_t s) {
  switch (p.c.page_size) {
    case 16: return launch_attn<T, NG, 16>(p, grid, s);
    case 32: return launch_attn<T, NG, 32>(p, grid, s);
    default: return launch_attn<T, NG, 64>(p, grid, s);
  }
}

template <typename T>
cudaError_t launch_attn_t(const AttnQ4Params &p, long long grid, cudaStream_t s) {
  switch (p.c.ng) {
    case 1: return launch_attn_g<T, 1>(p, grid, s);
    case 2: return launch_attn_g<T, 2>(p, grid, s);
    default: return launch_attn_g<T, 4>(p, grid, s);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) ==
                        cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ok ? ptr : nullptr);
  }();
  return fn;
}

// Map of a pool as slabs of 64-byte rows, one box per slab, stored with the
// 64-byte swizzle.
int slab_map(CUtensorMap *out, const Kv4Cache &c, int tier) {
  const int from = c.pool[tier] ? tier : 1 - tier;  // an absent tier: one page that no entry reaches
  const long long pages = c.pool[tier] ? c.pages[tier] : 1;
  const long long slabs = pages * c.kv_heads;
  if (slabs + c.kv_heads > 0x7fffffffll) return fail(DAK_ERR_UNSUPPORTED, "pages x kv_heads of a pool must stay below 2^31");
  auto fn = tensor_map_encoder();
  if (!fn) return fail(DAK_ERR_DRIVER, "cuTensorMapEncodeTiled entry point unavailable");
  const cuuint64_t dims[3] = {64, (cuuint64_t)c.slab_bytes / 64, (cuuint64_t)slabs};
  const cuuint64_t strides[2] = {64, (cuuint64_t)c.slab_bytes};
  const cuuint32_t box[3] = {64, (cuuint32_t)c.slab_bytes / 64, 1};
  const cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, c.pool[from], dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(DAK_ERR_DRIVER, "cuTensorMapEncodeTiled (4-bit KV) failed with %d", (int)r);
  return DAK_OK;
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
  if (a->split_size <= 0 || a->split_size % 64)
    return fail(DAK_ERR_INVALID_ARG, "split_size must be a positive multiple of 64");
  if (!a->query || !a->out || !a->seq_lens) return fail(DAK_ERR_INVALID_ARG, "query, out and seq_lens are required");
  if (a->q_stride_b % 8 || a->q_stride_h % 8 || (reinterpret_cast<uintptr_t>(a->query) & 15u))
    return fail(DAK_ERR_ALIGNMENT, "query must be 16-byte aligned, its strides multiples of 8 elements");
  const int splits = (int)(((long long)a->max_seq_len + a->split_size - 1) / a->split_size);
  if (splits > 1 && (!a->partial_o || !a->partial_ml))
    return fail(DAK_ERR_INVALID_ARG, "partial_o and partial_ml scratch are required when max_seq_len > split_size");
  const void *ptrs[6] = {a->query, a->out, a->seq_lens, splits > 1 ? a->partial_o : nullptr,
                         splits > 1 ? a->partial_ml : nullptr, splits > 1 ? a->merge_counters : nullptr};
  for (const void *q : ptrs)
    if (q && (st = check_gpu_accessible(q, "attention buffer"))) return st;
  AttnQ4Params p;
  std::memset(&p, 0, sizeof(p));
  if ((st = kv4_view(cache, &p.c))) return st;
  for (int tier = 0; tier < 2; ++tier)
    if ((st = slab_map(&p.map[tier], p.c, tier))) return st;
  p.query = static_cast<const uint16_t *>(a->query);
  p.q_stride_b = a->q_stride_b;
  p.q_stride_h = a->q_stride_h;
  p.out = static_cast<uint16_t *>(a->out);
  p.o_stride_b = a->o_stride_b;
  p.o_stride_h = a->o_stride_h;
  p.seq_lens = a->seq_lens;
  p.partial_o = a->partial_o;
  p.partial_ml = a->partial_ml;
  p.counters = splits > 1 ? a->merge_counters : nullptr;
  p.num_q_heads = a->num_q_heads;
  p.group = a->num_q_heads / cache->kv_heads;
  p.head_blocks = (p.group + kQ4Heads - 1) / kQ4Heads;
  p.block_heads = (p.group + p.head_blocks - 1) / p.head_blocks;
  p.max_seq_len = a->max_seq_len;
  p.split_size = a->split_size;
  p.num_splits = splits;
  p.scale_log2 = a->scaling * 1.4426950408889634f;
  p.pdl = decode_pdl_enabled() ? 1 : 0;
  const long long grid = (long long)cache->batch * cache->kv_heads * p.head_blocks * splits;
  if (grid > 0x7fffffffll) return fail(DAK_ERR_UNSUPPORTED, "too many splits for one launch; raise split_size");
  auto s = static_cast<cudaStream_t>(stream);
  return cuda_status(a->dtype == DAK_DTYPE_F16 ? launch_attn_t<__half>(p, grid, s) : launch_attn_t<__nv_bfloat16>(p, grid, s),
                     "4-bit attention launch");
}
