// dak_attention_kv4.cu - decode attention over the 4-bit paged KV cache
// (dak_kv4.cuh), whose pages lie in HBM or in pinned host memory.
//
// One query token per sequence: o = softmax(scaling q K^T) V over the first
// seq_lens[b] tokens, K and V being scale * code + zero.  One CTA per
// (sequence, KV head, block of up to 8 query heads, split of the tokens); the
// splits' (o, m, l) are merged with log-sum-exp.  Scores are kept in base 2.
// A sequence of no tokens gives zeros.
#include <cfloat>
#include <cstring>

#include "dak_common.cuh"
#include "dak_host.h"
#include "dak_kv4.cuh"

namespace dak {
namespace {

constexpr int kQ4Warps = 4;
constexpr int kQ4Threads = kQ4Warps * 32;
constexpr int kQ4Heads = 8;  // query heads per CTA

struct AttnQ4Params {
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

// Sum of the splits' partials of one query head at dim d, in split order.
template <typename T>
__device__ __forceinline__ void merge_q4(const AttnQ4Params &p, int b, int hq, int d) {
  const long long base = ((long long)b * p.num_q_heads + hq) * p.num_splits;
  float gm = -FLT_MAX;
  for (int s = 0; s < p.num_splits; ++s) gm = fmaxf(gm, __ldcg(p.partial_ml + (base + s) * 2));
  float den = 0.f, acc = 0.f;
  for (int s = 0; s < p.num_splits; ++s) {
    const float c = exp2f(__ldcg(p.partial_ml + (base + s) * 2) - gm);  // an empty split has l = 0 and o = 0
    den = fmaf(__ldcg(p.partial_ml + (base + s) * 2 + 1), c, den);
    acc = fmaf(__ldcg(p.partial_o + (base + s) * kKv4Dim + d), c, acc);
  }
  p.out[b * p.o_stride_b + hq * p.o_stride_h + d] = Elem<T>::from_float(den == 0.f ? 0.f : acc / den);
}

template <typename T, int NG>
__global__ void __launch_bounds__(kQ4Threads) attn_q4_kernel(const __grid_constant__ AttnQ4Params p) {
  __shared__ float sm_m[kQ4Warps][kQ4Heads], sm_l[kQ4Warps][kQ4Heads], sm_o[kQ4Warps][kQ4Heads][kKv4Dim];
  __shared__ int last;
  pdl_enter(p.pdl);
  const int warp = warp_id(), lane = lane_id();
  int i = blockIdx.x;
  const int split = i % p.num_splits;
  i /= p.num_splits;
  const int hb = i % p.head_blocks;
  i /= p.head_blocks;
  const int kvh = i % p.c.kv_heads;
  const int b = i / p.c.kv_heads;
  const int h0 = kvh * p.group + hb * p.block_heads;
  const int nh = min(p.block_heads, p.group - hb * p.block_heads);
  const int seq = min(p.seq_lens[b], p.max_seq_len);
  const int t0 = split * p.split_size, t1 = min(seq, t0 + p.split_size);
  const int P = p.c.page_size, half = kv4_half_bytes(P, NG);

  // Lane owns dims 4 lane .. +3, in group lane / (32 / NG).
  float q[kQ4Heads][4], o[kQ4Heads][4], m[kQ4Heads], l[kQ4Heads];
#pragma unroll
  for (int h = 0; h < kQ4Heads; ++h) {
    m[h] = -FLT_MAX;
    l[h] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[h][e] = 0.f;
      q[h][e] = h < nh ? Elem<T>::to_float(p.query[b * p.q_stride_b + (h0 + h) * p.q_stride_h + 4 * lane + e]) : 0.f;
    }
  }
  for (int t = t0 + warp; t < t1; t += kQ4Warps) {
    int tier = 0;
    const uint8_t *slab = kv4_page(p.c, b, t / P, &tier);
    float k[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
    if (!slab) {
      if (lane == 0) atomicCAS(p.c.status, 0, DAK_ERR_INVALID_ARG);  // reads zeros
    } else {
      slab += (long long)kvh * p.c.slab_bytes;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint8_t *part = slab + kv * half;
        const uint32_t w = *reinterpret_cast<const uint16_t *>(part + (t % P) * 64 + 2 * lane);
        const __half2 sz = *reinterpret_cast<const __half2 *>(part + P * 64 + ((t % P) * NG + lane / (32 / NG)) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          (kv ? v : k)[e] = fmaf(__low2float(sz), (float)((w >> (4 * e)) & 15u), __high2float(sz));
      }
    }
#pragma unroll
    for (int h = 0; h < kQ4Heads; ++h) {
      float s = q[h][0] * k[0] + q[h][1] * k[1] + q[h][2] * k[2] + q[h][3] * k[3];
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= p.scale_log2;
      const float mn = fmaxf(m[h], s);
      const float a = exp2f(m[h] - mn), w = exp2f(s - mn);
      m[h] = mn;
      l[h] = l[h] * a + w;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[h][e] = fmaf(w, v[e], o[h][e] * a);
    }
  }
#pragma unroll
  for (int h = 0; h < kQ4Heads; ++h) {
    if (lane == 0) {
      sm_m[warp][h] = m[h];
      sm_l[warp][h] = l[h];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sm_o[warp][h][4 * lane + e] = o[h][e];
  }
  __syncthreads();
  const int d = threadIdx.x;
  for (int h = 0; h < nh; ++h) {
    float gm = -FLT_MAX;
    for (int w = 0; w < kQ4Warps; ++w) gm = fmaxf(gm, sm_m[w][h]);
    float den = 0.f, acc = 0.f;
    for (int w = 0; w < kQ4Warps; ++w) {
      const float c = exp2f(sm_m[w][h] - gm);
      den = fmaf(sm_l[w][h], c, den);
      acc = fmaf(sm_o[w][h][d], c, acc);
    }
    if (p.num_splits == 1) {
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
  if (p.num_splits > 1 && p.counters) {
    // The split that finishes last merges all of them and resets the counter.
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      int32_t *counter = p.counters + blockIdx.x / p.num_splits;
      last = atomicAdd(counter, 1) == p.num_splits - 1;
      if (last) *counter = 0;
    }
    __syncthreads();
    if (last) {
      __threadfence();
      for (int h = 0; h < nh; ++h) merge_q4<T>(p, b, h0 + h, d);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kKv4Dim) attn_q4_merge_kernel(const __grid_constant__ AttnQ4Params p) {
  pdl_enter(p.pdl);
  merge_q4<T>(p, blockIdx.x / p.num_q_heads, blockIdx.x % p.num_q_heads, threadIdx.x);
}

template <typename T, int NG>
cudaError_t launch_attn(const AttnQ4Params &p, long long grid, cudaStream_t s) {
  cudaError_t e = launch_ex(attn_q4_kernel<T, NG>, dim3((unsigned)grid), dim3(kQ4Threads), 0, s, 1, p.pdl != 0, p);
  if (e != cudaSuccess || p.num_splits == 1 || p.counters) return e;
  return launch_ex(attn_q4_merge_kernel<T>, dim3((unsigned)(p.c.rows * p.num_q_heads)), dim3(kKv4Dim), 0, s, 1, p.pdl != 0,
                   p);
}

template <typename T>
cudaError_t launch_attn_t(const AttnQ4Params &p, long long grid, cudaStream_t s) {
  switch (p.c.ng) {
    case 1: return launch_attn<T, 1>(p, grid, s);
    case 2: return launch_attn<T, 2>(p, grid, s);
    default: return launch_attn<T, 4>(p, grid, s);
  }
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
