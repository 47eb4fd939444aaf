// dak_kv4.cu - writing and reading the 4-bit paged KV cache (dak_kv4.cuh).
//
// Append, for each token: q heads are rotated into q_out; k heads are rotated
// and v heads taken as they are, and each head's 128 values become 4-bit codes,
// group by group (32, 64 or 128 dims):
//   zero  = fp16(min), scale = fp16((max - min) / 15)   (saturated at +-65504)
//   code  = clamp(rint((x - zero) * (1 / scale)), 0, 15) (0 when scale is 0)
// from the rounded zero and scale, in FP32 from the rotated FP32 values: k is
// not rounded to 16 bits first.  A NaN takes no part in min and max and becomes code
// 0; a group of nothing else has zero and scale 0.  Read-back: value = scale * code + zero, one
// rounding to the 16-bit type.
//
// Both are bound by memory.  Eight lanes own a (token, head) row, 16 dims each
// (two 16-byte loads, one 8-byte code store), so a group's minimum and maximum
// are 1, 2 or 3 shuffles away; a warp takes the same head of four neighbouring
// tokens, whose code rows are neighbours in the page.  The append's CTA takes
// four tokens and up to 48 heads of each: four bulk copies bring them into shared
// memory, all in flight at once, while the threads work out the tokens' angles,
// one each; their pages are looked up behind the angles and the q heads.  With few
// heads it takes 8 or 16 tokens, each four with its share of the warps: the start-up
// is the larger part of a small CTA.
//
// The instructions count nearly as much as the bytes (249 per head of four tokens,
// 0.6 of the issue slots, before a q head's angles were kept in registers).  Append
// of 16384 tokens, 32 + 16 heads in bfloat16, groups of 32 (358 MB): 59 us, 6.1 TB/s,
// 0.94 of the measured copy rate (75 us before that, 64 us with the pages looked up
// first); of 4099 tokens 20 us; of 65536 tokens, 8 + 2 heads 58 us (109 us with four
// tokens per CTA); of 32 tokens 3.4 us.  CTAs that walk over tiles of 8 heads with
// four in flight took a quarter longer (97 us): they wait at each four tokens for
// positions and pages.  Five or six CTAs per SM with fewer registers, or fewer heads
// per CTA, took 10 to 30% longer.
//
// Read-back of 65536 tokens x 8 heads, groups of 128 (340 MB): 58 us, 5.9 TB/s, 0.91
// (63 us with four rows in flight per thread and four CTAs per SM, 75 with one row);
// of 257 tokens 2.3 us.
#include <cstring>

#include "dak_host.h"
#include "dak_kv4.cuh"
#include "dak_rotary.cuh"

namespace dak {

int kv4_check(const dak_kv4_cache *a) {
  if (!a) return fail(DAK_ERR_INVALID_ARG, "cache is null");
  if (a->page_size != 16 && a->page_size != 32 && a->page_size != 64)
    return fail(DAK_ERR_UNSUPPORTED, "page_size must be 16, 32 or 64");
  if (a->group != 32 && a->group != 64 && a->group != 128)
    return fail(DAK_ERR_UNSUPPORTED, "group must be 32, 64 or 128");
  if (a->batch <= 0 || a->kv_heads <= 0 || a->max_pages <= 0)
    return fail(DAK_ERR_INVALID_ARG, "batch, kv_heads and max_pages must be positive");
  if (a->kv_heads > 65535) return fail(DAK_ERR_UNSUPPORTED, "at most 65535 KV heads");
  if (a->table_stride < a->max_pages) return fail(DAK_ERR_INVALID_ARG, "table_stride below max_pages");
  if (!a->block_table) return fail(DAK_ERR_INVALID_ARG, "block_table is required");
  if (a->dev_pages < 0 || a->host_pages < 0 || (a->dev_pages > 0) != (a->pool_dev != nullptr) ||
      (a->host_pages > 0) != (a->pool_host != nullptr))
    return fail(DAK_ERR_INVALID_ARG, "each tier needs a pool and a positive page count, or neither");
  if (a->dev_pages == 0 && a->host_pages == 0) return fail(DAK_ERR_INVALID_ARG, "no KV pool given");
  if ((reinterpret_cast<uintptr_t>(a->pool_dev) | reinterpret_cast<uintptr_t>(a->pool_host)) & 15u)
    return fail(DAK_ERR_ALIGNMENT, "KV pools must be 16-byte aligned");
  return DAK_OK;
}

int kv4_view(const dak_kv4_cache *a, Kv4Cache *out) {
  const void *ptrs[3] = {a->pool_dev, a->pool_host, a->block_table};
  for (const void *q : ptrs) {
    if (!q) continue;
    int st = check_gpu_accessible(q, "KV buffer");
    if (st) return st;
  }
  Kv4Cache &c = *out;
  std::memset(&c, 0, sizeof(c));
  c.pool[0] = static_cast<uint8_t *>(a->pool_dev);
  c.pool[1] = static_cast<uint8_t *>(a->pool_host);
  c.pages[0] = a->dev_pages;
  c.pages[1] = a->host_pages;
  c.ng = kKv4Dim / a->group;
  c.slab_bytes = 2 * kv4_half_bytes(a->page_size, c.ng);
  c.page_bytes = (long long)c.slab_bytes * a->kv_heads;
  c.table = a->block_table;
  c.table_stride = a->table_stride;
  c.max_pages = a->max_pages;
  c.rows = a->batch;
  c.kv_heads = a->kv_heads;
  c.page_size = a->page_size;
  c.page_log2 = a->page_size == 16 ? 4 : a->page_size == 32 ? 5 : 6;
  c.status = device_status_word();
  if (!c.status) return fail(DAK_ERR_CUDA, "no device status word");
  return DAK_OK;
}

namespace {

constexpr int kKv4Threads = 256;
constexpr int kKv4Warps = kKv4Threads / 32;
constexpr int kAppendHeads = 48;            // of four tokens of an append's CTA, at most: 48 KB of shared memory
constexpr int kAppendTokens = 16;           // of an append's CTA, at most
constexpr long long kAppendFull = 148 * 4;  // CTAs that the GPU holds at once
constexpr long long kAppendCtas = 148 * 6;  // an append's CTAs, where its tokens alone give fewer
constexpr long long kReadWarps = 9472;      // a read's warps, likewise
constexpr int kReadRows = 8;                // of a token on one warp of a read, at most
constexpr int kBatch = 2;                   // rows a reading thread has in flight

struct AppendParams {
  Kv4Cache c;
  const uint16_t *qkv;
  long long ld;
  const int32_t *positions, *seq_index;
  const float *inv_freq;
  float scale;
  uint16_t *q_out;
  int tokens, q_heads, rotary_dim, interleaved, units;
  int slice;   // heads (q, then k, then v) per CTA
  int groups;  // 1, 2 or 4 groups of four tokens per CTA, each with its share of the warps
  int pdl;
};

__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Codes of a lane's 16 values and, in the group's first lane, the (scale, zero)
// pair, from the group's minimum and maximum over the lanes that share it.
template <int NG>
__device__ __forceinline__ void kv4_quantise(const float (&x)[16], int lane8, uint8_t *codes, uint8_t *pairs) {
  float mn = fminf(x[0], x[1]), mx = fmaxf(x[0], x[1]);  // a NaN gives way to any number
#pragma unroll
  for (int i = 2; i < 16; i += 2) {
    mn = min3(mn, x[i], x[i + 1]);
    mx = max3(mx, x[i], x[i + 1]);
  }
#pragma unroll
  for (int m = 1; m < 8 / NG; m <<= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, m));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, m));
  }
  const float lo = mn == mn ? fminf(fmaxf(mn, -65504.f), 65504.f) : 0.f;  // nothing but NaN: zeros
  const __half z = __float2half_rn(lo);
  const __half s = __float2half_rn(fminf(fmaxf(__fdiv_rn(mx - mn, 15.f), 0.f), 65504.f));
  const float zf = __half2float(z), sf = __half2float(s);
  const float inv = sf > 0.f ? __frcp_rn(sf) : 0.f;
  // Added to 1.5 x 2^23 a number is rounded to an integer in the sum's low bits, by
  // an addition instead of rint and a conversion, which run at a quarter of its rate
  // (2 to 6% of the kernel's time).  The upper bits of eight sums, shifted, add up to
  // a constant.
  constexpr float kBig = 12582912.f;
  constexpr uint32_t kBits = 0x4B400000u;
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    w[j] = 0u - kBits * 0x11111111u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float n = fminf(fmaxf(__fadd_rn(__fmul_rn(x[8 * j + i] - zf, inv), kBig), kBig), kBig + 15.f);  // NaN: 0
      w[j] += __float_as_uint(n) << (4 * i);
    }
  }
  if (codes) {
    *reinterpret_cast<uint2 *>(codes + lane8 * 8) = make_uint2(w[0], w[1]);
    if (lane8 % (8 / NG) == 0)
      reinterpret_cast<uint32_t *>(pairs)[lane8 / (8 / NG)] =
          (uint32_t)__half_as_ushort(s) | ((uint32_t)__half_as_ushort(z) << 16);
  }
}

struct AppendSmem {
  uint8_t *page[kAppendTokens];
  uint64_t bar;
  int tier[kAppendTokens];
  int abort_flag[2];  // [1]: of the second wait
};

// G groups of four tokens, one for each G-th of the warps; a head of the four at a
// time per warp: q heads are rotated, k heads rotated and packed, v heads packed.
template <typename T, int NG, int G>
__global__ void __launch_bounds__(kKv4Threads, 4) kv4_append_kernel(const __grid_constant__ AppendParams p) {
  extern __shared__ __align__(128) uint8_t rows_s[];  // [tokens][slice][128] 16-bit, then angles, then the rest
  constexpr int ct = 4 * G;                           // tokens of the CTA
  const int stride = rope_stride(p.rotary_dim);
  float *tab = reinterpret_cast<float *>(rows_s + ct * p.slice * kKv4Dim * 2);
  AppendSmem &sm = *reinterpret_cast<AppendSmem *>(tab + 2 * ct * stride);
  pdl_enter(p.pdl);
  const int t0 = blockIdx.x * ct, nt = min(ct, p.tokens - t0);
  // A warp takes every warps-th head of four of the tokens.
  constexpr int warps = kKv4Warps / G;
  const int lane8 = lane_id() & 7, sub = warp_id() / warps * 4 + (lane_id() >> 3);
  const bool live = sub < nt;
  const int t = t0 + (live ? sub : 0);  // idle lanes stay for the shuffles
  const int P = p.c.page_size, Hkv = p.c.kv_heads;
  const int h0 = blockIdx.y * p.slice, h_end = min(p.q_heads + 2 * Hkv, h0 + p.slice);
  const uint32_t bar_a = smem_u32(&sm.bar), token_bytes = (h_end - h0) * kKv4Dim * 2;
  const WaitCtx wc{&sm.abort_flag[0], p.c.status};
  if (threadIdx.x == 0) {
    sm.abort_flag[0] = sm.abort_flag[1] = 0;
    mbar_init(bar_a, 1);
    fence_mbar_init();
    mbar_arrive_expect_tx(bar_a, nt * token_bytes);
    const uint64_t pol = l2_policy_evict_first();
    for (int i = 0; i < nt; ++i)
      bulk_load(smem_u32(rows_s) + i * token_bytes, p.qkv + (long long)(t0 + i) * p.ld + h0 * kKv4Dim, token_bytes, bar_a, pol);
  }
  // The page look-up (position, then table entry) runs behind the angles and the q
  // heads; its result is wanted for k and v.
  bool in = false;
  int entry = 0;
  if (threadIdx.x < nt) {
    const int seq = p.seq_index ? p.seq_index[t0 + threadIdx.x] : t0 + (int)threadIdx.x;
    const int page = p.positions[t0 + threadIdx.x] >> p.c.page_log2;
    in = kv4_in_table(p.c, seq, page);
    if (in) entry = p.c.table[(long long)seq * p.c.table_stride + page];
  }
  rope_table(tab, p.positions + t0, nt, ct, p.inv_freq, p.rotary_dim, p.scale);
  __syncthreads();
  const float *cos_row = tab + (live ? sub : 0) * stride, *sin_row = cos_row + ct * stride;
  const int slot = p.positions[t] & (P - 1);
  const int half = kv4_half_bytes(P, NG);
  const int R = p.rotary_dim, part = R / 16;  // vectors between the partners of the half layout
  const uint8_t *row = rows_s + (live ? sub : 0) * token_bytes;
  const bool ok = mbar_wait<false>(bar_a, 0, wc);

  // q: a unit at a time, its angles in registers for all of the warp's heads.
  constexpr int row_vecs = kKv4Dim / 8;
  const uint4 *vecs = reinterpret_cast<const uint4 *>(row);
  int h = h0 + warp_id() % warps;
  const int q_end = ok ? min(h_end, p.q_heads) : h, k_end = min(h_end, p.q_heads + Hkv);
  for (int u = live ? lane8 : p.units; u < p.units; u += 8) {
    const RopeUnit unit = rope_unit(u, R, p.interleaved);
    float c[8], s[8];
    rope_unit_angles(unit, cos_row, sin_row, c, s);
    uint4 *dst = reinterpret_cast<uint4 *>(p.q_out) + ((long long)t * p.q_heads + h) * row_vecs;
    const uint4 *src = vecs + (h - h0) * row_vecs;
    for (int i = h; i < q_end; i += warps) {
      rope_unit_apply<T>(unit, p.interleaved, src[unit.v0], src[unit.v1 >= 0 ? unit.v1 : unit.v0], c, s, dst);
      src += warps * row_vecs;
      dst += warps * row_vecs;
    }
  }
  if (h < q_end) h += (q_end - h + warps - 1) / warps * warps;
  // k and v: 16 dims a lane.
  if (threadIdx.x < nt) {
    int tier = 0;
    uint8_t *page = in ? kv4_page_of(p.c, entry, &tier) : nullptr;
    if (!page) atomicCAS(p.c.status, 0, DAK_ERR_INVALID_ARG);
    sm.page[threadIdx.x] = page;
    sm.tier[threadIdx.x] = tier;
  }
  __syncthreads();
  if (!ok) {  // gave up: let the copies land (bounded again), then leave
    mbar_wait<false>(bar_a, 0, WaitCtx{&sm.abort_flag[1], p.c.status});
    return;
  }
  uint8_t *page = live ? sm.page[sub] : nullptr;
  uint8_t *codes = page ? page + slot * 64 : nullptr, *pairs = page ? page + P * 64 + slot * 4 * NG : nullptr;
  auto store = [&](const float(&x)[16], long long at) {
    kv4_quantise<NG>(x, lane8, page ? codes + at : nullptr, pairs + at);
  };
  for (; h < k_end; h += warps) {
    const uint4 *src = vecs + (h - h0) * row_vecs;
    float x[16];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float y[8];
      const int v = lane8 * 2 + k;
      unpack8<T>(src[v], y);
      if (!p.interleaved && v < 2 * part) {
        float z[8], c[8], s[8];
        unpack8<T>(src[v < part ? v + part : v - part], z);  // each lane keeps its own side of the pairs
        const int f = 8 * (v < part ? v : v - part);
        load4(cos_row + f, c), load4(cos_row + f + 4, c + 4);
        load4(sin_row + f, s), load4(sin_row + f + 4, s + 4);
        const float sign = v < part ? -1.f : 1.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = fmaf(y[i], c[i], z[i] * (s[i] * sign));
      } else if (p.interleaved && v * 8 < R) {
        float c[4], s[4];
        load4(cos_row + 4 * v, c);
        load4(sin_row + 4 * v, s);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (v * 8 + 2 * i < R) rope_turn(y[2 * i], y[2 * i + 1], c[i], s[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[8 * k + i] = y[i];
    }
    store(x, (long long)(h - p.q_heads) * p.c.slab_bytes);
  }
  for (; h < h_end; h += warps) {
    const uint4 *src = vecs + (h - h0) * row_vecs + 2 * lane8;
    float x[16], y[8];
    unpack8<T>(src[0], y);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i];
    unpack8<T>(src[1], y);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[8 + i] = y[i];
    store(x, (long long)(h - p.q_heads - Hkv) * p.c.slab_bytes + half);
  }
  // Host pages are read back over the host link by the next kernels of the
  // stream; make the writes visible system-wide before this grid completes.
  if (live && sm.tier[sub] == 1) __threadfence_system();
}

struct ReadParams {
  Kv4Cache c;
  const int32_t *positions, *seq_index;
  uint16_t *out[2];  // k, v: [tokens, kv_heads, 128]
  int tokens, groups, pdl;
};

template <typename T, int NG>
__global__ void __launch_bounds__(kKv4Threads, 5) kv4_read_kernel(const __grid_constant__ ReadParams p) {
  pdl_enter(p.pdl);
  const long long w = (long long)blockIdx.x * kKv4Warps + warp_id();
  const int g = (int)(w % p.groups);
  const int lane8 = lane_id() & 7;
  const long long t = (w / p.groups) * 4 + (lane_id() >> 3);
  if (t >= p.tokens) return;
  const int P = p.c.page_size;
  const int pos = p.positions[t];
  int tier = 0;
  const uint8_t *page =
      pos < 0 ? nullptr : kv4_page(p.c, p.seq_index ? p.seq_index[t] : (int)t, pos >> p.c.page_log2, &tier);
  if (!page && lane8 == 0) atomicCAS(p.c.status, 0, DAK_ERR_INVALID_ARG);
  const int half = kv4_half_bytes(P, NG), items = 2 * p.c.kv_heads;  // K rows of all heads, then V rows
  const int code_at = (pos & (P - 1)) * 64 + lane8 * 8;
  const int pair_at = P * 64 + ((pos & (P - 1)) * NG + lane8 / (8 / NG)) * 4;
  for (int i0 = g; i0 < items; i0 += kBatch * p.groups) {
    uint2 codes[kBatch];
    uint32_t pair[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k * p.groups;
      codes[k] = make_uint2(0u, 0u);
      pair[k] = 0u;
      if (i < items && page) {
        const int isv = i >= p.c.kv_heads;
        const uint8_t *slab = page + (long long)(i - isv * p.c.kv_heads) * p.c.slab_bytes + isv * half;
        codes[k] = __ldcs(reinterpret_cast<const uint2 *>(slab + code_at));
        pair[k] = *reinterpret_cast<const uint32_t *>(slab + pair_at);
      }
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k * p.groups;
      if (i >= items) break;
      const int isv = i >= p.c.kv_heads;
      const float s = __half2float(__ushort_as_half((unsigned short)(pair[k] & 0xffffu)));
      const float z = __half2float(__ushort_as_half((unsigned short)(pair[k] >> 16)));
      uint4 *dst = reinterpret_cast<uint4 *>(p.out[isv] + (t * p.c.kv_heads + (i - isv * p.c.kv_heads)) * kKv4Dim) + lane8 * 2;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const uint32_t word = v ? codes[k].y : codes[k].x;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf(s, (float)((word >> (4 * e)) & 15u), z);
        __stcs(dst + v, pack8<T>(x));
      }
    }
  }
}

template <typename T, int NG, int G>
cudaError_t launch_append_t(const AppendParams &p, dim3 grid, cudaStream_t s) {
  auto kern = kv4_append_kernel<T, NG, G>;
  const cudaError_t e = prepare_kernel_attributes(reinterpret_cast<const void *>(kern));
  const size_t smem = 4 * G * (p.slice * kKv4Dim * 2 + 2 * rope_stride(p.rotary_dim) * sizeof(float)) + sizeof(AppendSmem);
  return e != cudaSuccess ? e : launch_ex(kern, grid, dim3(kKv4Threads), smem, s, 1, p.pdl != 0, p);
}

template <typename T, int NG>
cudaError_t launch_append_g(const AppendParams &p, dim3 grid, cudaStream_t s) {
  return p.groups == 1   ? launch_append_t<T, NG, 1>(p, grid, s)
         : p.groups == 2 ? launch_append_t<T, NG, 2>(p, grid, s)
                         : launch_append_t<T, NG, 4>(p, grid, s);
}

template <typename T>
cudaError_t launch_append(const AppendParams &p, dim3 grid, cudaStream_t s) {
  switch (p.c.ng) {
    case 1: return launch_append_g<T, 1>(p, grid, s);
    case 2: return launch_append_g<T, 2>(p, grid, s);
    default: return launch_append_g<T, 4>(p, grid, s);
  }
}

template <typename T>
cudaError_t launch_read(const ReadParams &p, unsigned grid, cudaStream_t s) {
  switch (p.c.ng) {
    case 1: return launch_ex(kv4_read_kernel<T, 1>, dim3(grid), dim3(kKv4Threads), 0, s, 1, p.pdl != 0, p);
    case 2: return launch_ex(kv4_read_kernel<T, 2>, dim3(grid), dim3(kKv4Threads), 0, s, 1, p.pdl != 0, p);
    default: return launch_ex(kv4_read_kernel<T, 4>, dim3(grid), dim3(kKv4Threads), 0, s, 1, p.pdl != 0, p);
  }
}

int check_tokens(int tokens, const int32_t *positions, const int32_t *seq_index, int batch) {
  if (tokens < 0) return fail(DAK_ERR_INVALID_ARG, "tokens must not be negative");
  if (!positions) return fail(DAK_ERR_INVALID_ARG, "positions is required");
  if (!seq_index && tokens != batch)
    return fail(DAK_ERR_INVALID_ARG, "without seq_index there is one token per sequence (%d tokens, %d sequences)", tokens,
                batch);
  return DAK_OK;
}

}  // namespace
}  // namespace dak

extern "C" int dak_rope_kv_append_q4(const dak_kv4_cache *cache, const dak_kv4_append_args *a, void *stream) {
  using namespace dak;
  if (!a) return fail(DAK_ERR_INVALID_ARG, "args is null");
  int st = kv4_check(cache);
  if (st) return st;
  if (a->dtype != DAK_DTYPE_F16 && a->dtype != DAK_DTYPE_BF16)
    return fail(DAK_ERR_UNSUPPORTED, "the 4-bit append takes float16 and bfloat16");
  if ((st = check_tokens(a->tokens, a->positions, a->seq_index, cache->batch))) return st;
  if (a->q_heads < 0 || !a->qkv || (a->q_heads > 0 && !a->q_out))
    return fail(DAK_ERR_INVALID_ARG, "qkv and, with q heads, q_out are required");
  if (a->ld < ((int64_t)a->q_heads + 2ll * cache->kv_heads) * kKv4Dim)
    return fail(DAK_ERR_INVALID_ARG, "qkv row stride below (q_heads + 2 kv_heads) x 128");
  if (a->ld % 8 || ((reinterpret_cast<uintptr_t>(a->qkv) | reinterpret_cast<uintptr_t>(a->q_out)) & 15u))
    return fail(DAK_ERR_ALIGNMENT, "qkv and q_out must be 16-byte aligned, the row stride a multiple of 8 elements");
  if ((st = check_rotary_dim(a->rotary_dim, kKv4Dim, a->interleaved))) return st;
  if (a->rotary_dim > 0 && !a->inv_freq) return fail(DAK_ERR_INVALID_ARG, "inv_freq is required to rotate");
  const int64_t row = ((int64_t)a->q_heads + 2ll * cache->kv_heads) * kKv4Dim * 2;
  if (a->q_heads > 0 && overlap({a->qkv, a->tokens, 2 * a->ld, 1, 0, row},
                                {a->q_out, a->tokens > 0, 0, 1, 0, 2ll * a->tokens * a->q_heads * kKv4Dim}))
    return fail(DAK_ERR_INVALID_ARG, "q_out must not overlap qkv");
  const void *ptrs[5] = {a->qkv, a->q_heads > 0 ? a->q_out : nullptr, a->rotary_dim > 0 ? a->inv_freq : nullptr,
                         a->positions, a->seq_index};
  for (const void *q : ptrs)
    if (q && (st = check_gpu_accessible(q, "append buffer"))) return st;
  AppendParams p;
  std::memset(&p, 0, sizeof(p));
  if ((st = kv4_view(cache, &p.c))) return st;
  if (a->tokens == 0) return DAK_OK;
  p.qkv = static_cast<const uint16_t *>(a->qkv);
  p.ld = a->ld;
  p.positions = a->positions;
  p.seq_index = a->seq_index;
  p.inv_freq = a->inv_freq;
  p.scale = a->rope_scale;
  p.q_out = static_cast<uint16_t *>(a->q_out);
  p.tokens = a->tokens;
  p.q_heads = a->q_heads;
  p.rotary_dim = a->rotary_dim;
  p.interleaved = a->interleaved != 0;
  p.units = rope_units(kKv4Dim, a->rotary_dim, p.interleaved);
  const long long quads = (a->tokens + 3ll) / 4;
  p.pdl = decode_pdl_enabled() ? 1 : 0;
  // All heads of four tokens on one CTA, or on as many as keep the GPU busy, down
  // to one head per warp.
  const long long heads = a->q_heads + 2ll * cache->kv_heads;
  const long long slices = std::max((heads + kAppendHeads - 1) / kAppendHeads,
                                    std::min((heads + kKv4Warps - 1) / kKv4Warps, kAppendCtas / quads));
  if (heads > 65535ll * kKv4Warps) return fail(DAK_ERR_UNSUPPORTED, "too many heads");
  p.slice = (int)(slices == 1 ? heads : ((heads + slices - 1) / slices + kKv4Warps - 1) / kKv4Warps * kKv4Warps);
  // Few heads of many tokens: more tokens per CTA, each of which starts up once, as
  // far as the shared memory of 48 heads goes and half the GPU still gets a CTA.  8 + 2
  // heads of 2500 tokens: 5.8 us, 7.3 without; of 65536: 58 and 109.
  p.groups = 1;
  while (4 * p.groups < kAppendTokens && 2 * p.groups * p.slice <= kAppendHeads && heads <= p.slice &&
         quads >= p.groups * kAppendFull)
    p.groups *= 2;
  const dim3 grid((unsigned)((quads + p.groups - 1) / p.groups), (unsigned)((heads + p.slice - 1) / p.slice));
  auto s = static_cast<cudaStream_t>(stream);
  return cuda_status(a->dtype == DAK_DTYPE_F16 ? launch_append<__half>(p, grid, s)
                                               : launch_append<__nv_bfloat16>(p, grid, s),
                     "4-bit append launch");
}

extern "C" int dak_kv_read_q4(const dak_kv4_cache *cache, const int32_t *positions, const int32_t *seq_index, void *k_out,
                              void *v_out, int tokens, int dtype, void *stream) {
  using namespace dak;
  int st = kv4_check(cache);
  if (st) return st;
  if (dtype != DAK_DTYPE_F16 && dtype != DAK_DTYPE_BF16)
    return fail(DAK_ERR_UNSUPPORTED, "the 4-bit cache is read to float16 and bfloat16");
  if ((st = check_tokens(tokens, positions, seq_index, cache->batch))) return st;
  if (!k_out || !v_out) return fail(DAK_ERR_INVALID_ARG, "k_out and v_out are required");
  const int64_t bytes = 2ll * tokens * cache->kv_heads * kKv4Dim;
  if (k_out == v_out || overlap({k_out, 1, 0, 1, 0, bytes}, {v_out, 1, 0, 1, 0, bytes}))
    return fail(DAK_ERR_INVALID_ARG, "k_out and v_out must not overlap");
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15u)
    return fail(DAK_ERR_ALIGNMENT, "k_out and v_out must be 16-byte aligned");
  const void *ptrs[4] = {k_out, v_out, positions, seq_index};
  for (const void *q : ptrs)
    if (q && (st = check_gpu_accessible(q, "read buffer"))) return st;
  ReadParams p;
  std::memset(&p, 0, sizeof(p));
  if ((st = kv4_view(cache, &p.c))) return st;
  if (tokens == 0) return DAK_OK;
  p.positions = positions;
  p.seq_index = seq_index;
  p.out[0] = static_cast<uint16_t *>(k_out);
  p.out[1] = static_cast<uint16_t *>(v_out);
  p.tokens = tokens;
  const long long quads = (tokens + 3ll) / 4;
  // One row per warp until the GPU is full, then more, up to eight: a warp that took
  // all 16 rows of 8 heads wrote to so many places that HBM slowed down (65536 tokens:
  // 57 us with 8 rows per warp, 62 with 16 or 4).
  const long long rows = 2ll * cache->kv_heads;
  p.groups = (int)std::max((rows + kReadRows - 1) / kReadRows, std::min(rows, kReadWarps / quads));
  p.pdl = decode_pdl_enabled() ? 1 : 0;
  const long long grid = (quads * p.groups + kKv4Warps - 1) / kKv4Warps;
  if (grid > 0x7fffffffll) return fail(DAK_ERR_UNSUPPORTED, "too many tokens for one launch");
  auto s = static_cast<cudaStream_t>(stream);
  return cuda_status(dtype == DAK_DTYPE_F16 ? launch_read<__half>(p, (unsigned)grid, s)
                                            : launch_read<__nv_bfloat16>(p, (unsigned)grid, s),
                     "4-bit read launch");
}
