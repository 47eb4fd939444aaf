// dak_kv4.cu - writing and reading the 4-bit paged KV cache (dak_kv4.cuh).
//
// Append, for each token: q heads are rotated into q_out; k heads are rotated
// and v heads taken as they are, and each head's 128 values become 4-bit codes,
// group by group (32, 64 or 128 dims):
//   zero  = fp16(min), scale = fp16((max - min) / 15)   (saturated at +-65504)
//   code  = clamp(rint((x - zero) * (1 / scale)), 0, 15) (0 when scale is 0)
// from the rounded zero and scale, in FP32 from the rotated FP32 values: k is
// not rounded to 16 bits first.  Read-back: value = scale * code + zero, one
// rounding to the 16-bit type.
//
// Both are bound by memory.  Eight lanes own a (token, head) row, 16 dims each
// (two 16-byte loads, one 8-byte code store), so a group's minimum and maximum
// are 1, 2 or 3 shuffles away; a warp takes the same head of four neighbouring
// tokens, whose code rows are neighbours in the page.  The append's CTA takes
// four tokens and up to 48 heads of each: four bulk copies bring them into shared
// memory, all in flight at once, while the threads work out the tokens' angles,
// one each, and look up their pages.
//
// Append of 16384 tokens, 32 + 16 heads in bfloat16, groups of 32 (358 MB): 71 us,
// 5.0 TB/s, 0.79 of the measured copy rate; of 4099 tokens 24 us (38 us when each
// thread fetched its heads itself and worked out their angles); of 32 tokens
// 3.1 us.  Read-back of 65536 tokens x 8 heads, groups of 128 (340 MB): 62 us,
// 5.5 TB/s, 0.85 (75 us with one row in flight per thread).
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
constexpr int kAppendHeads = 48;            // of an append's CTA, at most: 48 KB of shared memory
constexpr long long kAppendCtas = 148 * 6;  // an append's CTAs, where its tokens alone give fewer
constexpr int kReadWarps = 9472;            // a read's warps, likewise
constexpr int kBatch = 4;                   // rows a reading thread has in flight

struct AppendParams {
  Kv4Cache c;
  const uint16_t *qkv;
  long long ld;
  const int32_t *positions, *seq_index;
  const float *inv_freq;
  float scale;
  uint16_t *q_out;
  int tokens, q_heads, rotary_dim, interleaved, units;
  int slice;  // heads (q, then k, then v) per CTA
  int pdl;
};

// Codes of a lane's 16 values and, in the group's first lane, the (scale, zero)
// pair, from the group's minimum and maximum over the lanes that share it.
template <int NG>
__device__ __forceinline__ void kv4_quantise(const float (&x)[16], int lane8, uint8_t *codes, uint8_t *pairs) {
  float mn = x[0], mx = x[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) {
    mn = fminf(mn, x[i]);  // a NaN gives way to any number
    mx = fmaxf(mx, x[i]);
  }
#pragma unroll
  for (int m = 1; m < 8 / NG; m <<= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, m));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, m));
  }
  const __half z = __float2half_rn(fminf(fmaxf(mn, -65504.f), 65504.f));
  const __half s = __float2half_rn(fminf(fmaxf(__fdiv_rn(mx - mn, 15.f), 0.f), 65504.f));
  const float zf = __half2float(z), sf = __half2float(s);
  const float inv = sf > 0.f ? __frcp_rn(sf) : 0.f;
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float n = fminf(fmaxf(rintf((x[i] - zf) * inv), 0.f), 15.f);  // NaN: 0
    w[i >> 3] |= (uint32_t)n << (4 * (i & 7));
  }
  if (codes) {
    *reinterpret_cast<uint2 *>(codes + lane8 * 8) = make_uint2(w[0], w[1]);
    if (lane8 % (8 / NG) == 0)
      reinterpret_cast<uint32_t *>(pairs)[lane8 / (8 / NG)] =
          (uint32_t)__half_as_ushort(s) | ((uint32_t)__half_as_ushort(z) << 16);
  }
}

struct AppendSmem {
  alignas(16) float tab[2 * 4 * kKv4Dim / 2];  // angles of the four tokens
  uint8_t *page[4];
  uint64_t bar;
  int tier[4];
  int abort_flag[2];  // [1]: of the second wait
};

// A head of the four tokens at a time per warp: q heads are rotated, k heads
// rotated and packed, v heads packed.
template <typename T, int NG>
__global__ void __launch_bounds__(kKv4Threads, 4) kv4_append_kernel(const __grid_constant__ AppendParams p) {
  extern __shared__ __align__(128) uint8_t rows_s[];  // [tokens][slice][128] 16-bit, then the rest
  AppendSmem &sm = *reinterpret_cast<AppendSmem *>(rows_s + 4 * p.slice * kKv4Dim * 2);
  pdl_enter(p.pdl);
  const int t0 = blockIdx.x * 4, nt = min(4, p.tokens - t0);
  const int lane8 = lane_id() & 7, sub = lane_id() >> 3;
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
  if (threadIdx.x < nt) {
    const int pos = p.positions[t0 + threadIdx.x];
    int tier = 0;
    uint8_t *page = pos < 0 ? nullptr
                            : kv4_page(p.c, p.seq_index ? p.seq_index[t0 + threadIdx.x] : t0 + (int)threadIdx.x,
                                       pos >> p.c.page_log2, &tier);
    if (!page) atomicCAS(p.c.status, 0, DAK_ERR_INVALID_ARG);
    sm.page[threadIdx.x] = page;
    sm.tier[threadIdx.x] = tier;
  }
  const int stride = rope_stride(p.rotary_dim);
  rope_table(sm.tab, p.positions + t0, nt, 4, p.inv_freq, p.rotary_dim, p.scale);
  __syncthreads();
  const float *cos_row = sm.tab + (live ? sub : 0) * stride, *sin_row = cos_row + 4 * stride;
  const int slot = p.positions[t] & (P - 1);
  uint8_t *page = live ? sm.page[sub] : nullptr;
  const int half = kv4_half_bytes(P, NG);
  const int R = p.rotary_dim, part = R / 16;  // vectors between the partners of the half layout
  const uint8_t *row = rows_s + (live ? sub : 0) * token_bytes;
  if (!mbar_wait<false>(bar_a, 0, wc)) {  // gave up: let the copies land (bounded again), then leave
    mbar_wait<false>(bar_a, 0, WaitCtx{&sm.abort_flag[1], p.c.status});
    return;
  }

  for (int h = h0 + warp_id(); h < h_end; h += kKv4Warps) {
    const uint4 *src = reinterpret_cast<const uint4 *>(row + (h - h0) * kKv4Dim * 2);
    if (h < p.q_heads) {
      if (!live) continue;
      uint4 *dst = reinterpret_cast<uint4 *>(p.q_out + ((long long)t * p.q_heads + h) * kKv4Dim);
      for (int u = lane8; u < p.units; u += 8) {
        const RopeUnit unit = rope_unit(u, R, p.interleaved);
        float c[8], s[8];
        rope_unit_angles(unit, cos_row, sin_row, c, s);
        rope_unit_apply<T>(unit, p.interleaved, src[unit.v0], src[unit.v1 >= 0 ? unit.v1 : unit.v0], c, s, dst);
      }
      continue;
    }
    const int isv = h >= p.q_heads + Hkv ? 1 : 0;
    float x[16];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float y[8];
      const int v = lane8 * 2 + k;
      unpack8<T>(src[v], y);
      if (!isv && !p.interleaved && v < 2 * part) {
        float z[8], c[8], s[8];
        unpack8<T>(src[v < part ? v + part : v - part], z);  // each lane keeps its own side of the pairs
        const int f = 8 * (v < part ? v : v - part);
        load4(cos_row + f, c), load4(cos_row + f + 4, c + 4);
        load4(sin_row + f, s), load4(sin_row + f + 4, s + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = fmaf(y[i], c[i], z[i] * (v < part ? -s[i] : s[i]));
      } else if (!isv && p.interleaved && v * 8 < R) {
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
    uint8_t *slab = page ? page + (long long)(h - p.q_heads - isv * Hkv) * p.c.slab_bytes + isv * half : nullptr;
    kv4_quantise<NG>(x, lane8, slab ? slab + slot * 64 : nullptr, slab ? slab + P * 64 + slot * 4 * NG : nullptr);
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
__global__ void __launch_bounds__(kKv4Threads) kv4_read_kernel(const __grid_constant__ ReadParams p) {
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

template <typename T, int NG>
cudaError_t launch_append_g(const AppendParams &p, dim3 grid, cudaStream_t s) {
  auto kern = kv4_append_kernel<T, NG>;
  const cudaError_t e = prepare_kernel_attributes(reinterpret_cast<const void *>(kern));
  return e != cudaSuccess ? e : launch_ex(kern, grid, dim3(kKv4Threads), 4 * p.slice * kKv4Dim * 2 + sizeof(AppendSmem), s, 1, p.pdl != 0, p);
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
  p.slice = (int)(((heads + slices - 1) / slices + kKv4Warps - 1) / kKv4Warps * kKv4Warps);
  const dim3 grid((unsigned)quads, (unsigned)((heads + p.slice - 1) / p.slice));
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
  if (k_out == v_out) return fail(DAK_ERR_INVALID_ARG, "k_out and v_out must not overlap");
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
  // One row per warp until the GPU is full, then more.
  p.groups = (int)std::min<long long>(2ll * cache->kv_heads, std::max<long long>(1, kReadWarps / quads));
  p.pdl = decode_pdl_enabled() ? 1 : 0;
  const long long grid = (quads * p.groups + kKv4Warps - 1) / kKv4Warps;
  if (grid > 0x7fffffffll) return fail(DAK_ERR_UNSUPPORTED, "too many tokens for one launch");
  auto s = static_cast<cudaStream_t>(stream);
  return cuda_status(dtype == DAK_DTYPE_F16 ? launch_read<__half>(p, (unsigned)grid, s)
                                            : launch_read<__nv_bfloat16>(p, (unsigned)grid, s),
                     "4-bit read launch");
}
