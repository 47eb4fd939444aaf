// dak_rotary.cu - rotary positions of the heads of any number of tokens: half
// or interleaved pairs, all or part of the head, frequencies and attention
// factor as the model's scaling gives them.
//
// Bound by memory: each 16-byte vector is read once and written once.  A CTA
// takes up to four tokens and puts the cosines and sines of their angles into
// shared memory, one angle per thread.  A thread then owns one unit
// (dak_rotary.cuh) of one of the tokens, keeps its angles in registers and walks
// over heads, four at a time so that eight loads are in flight; the first are on
// their way while the angles are worked out.
//
// 8192 tokens x 40 heads of 128 in bfloat16 (168 MB): 28.6 us, 5.9 TB/s, 0.91 of
// the measured copy rate; 45 us with every thread working out its own eight FP64
// angles.  8 tokens: 2.1 us, a launch's latency.
#include "dak_host.h"
#include "dak_rotary.cuh"

namespace dak {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryBatch = 4;
constexpr int kRotaryTokens = 4;              // per CTA, while their angles number at most 256
constexpr long long kRotaryTarget = 148 * 4;  // CTAs that fill the GPU

struct RotaryParams {
  const uint16_t *x;
  uint16_t *out;
  long long xt, xh, ot, oh;  // token and head strides, elements
  const int32_t *positions;
  const float *inv_freq;
  float scale;
  int tokens, heads, units;
  int cta_tokens, cta_heads;  // per CTA
  int lanes;                  // heads of a token that the CTA's threads take at once
  int rotary_dim, interleaved, pdl;
};

template <typename T>
__global__ void __launch_bounds__(kRotaryThreads, 3) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ __align__(16) float tab[];
  pdl_enter(p.pdl);
  const int t0 = blockIdx.x * p.cta_tokens, nt = min(p.cta_tokens, p.tokens - t0);
  const int h_end = min(p.heads, (int)(blockIdx.y + 1) * p.cta_heads);
  const int row = threadIdx.x / p.units, tok = row % p.cta_tokens;
  const RopeUnit unit = rope_unit(threadIdx.x - row * p.units, p.rotary_dim, p.interleaved);
  int h = blockIdx.y * p.cta_heads + row / p.cta_tokens;
  if (tok >= nt || row >= p.lanes * p.cta_tokens) h = h_end;  // no unit for this thread
  const uint4 *src = reinterpret_cast<const uint4 *>(p.x + (t0 + tok) * p.xt);
  uint4 *dst = reinterpret_cast<uint4 *>(p.out + (t0 + tok) * p.ot);
  const long long src_h = p.xh / 8, dst_h = p.oh / 8;
  uint4 a[kRotaryBatch], b[kRotaryBatch];
  auto load = [&](int h) {
#pragma unroll
    for (int k = 0; k < kRotaryBatch; ++k) {
      if (h + k * p.lanes >= h_end) break;
      a[k] = src[(h + k * p.lanes) * src_h + unit.v0];
      if (unit.v1 >= 0) b[k] = src[(h + k * p.lanes) * src_h + unit.v1];
    }
  };
  load(h);
  rope_table(tab, p.positions + t0, nt, p.cta_tokens, p.inv_freq, p.rotary_dim, p.scale);
  __syncthreads();
  const int stride = rope_stride(p.rotary_dim);
  float c[8], s[8];
  rope_unit_angles(unit, tab + tok * stride, tab + (p.cta_tokens + tok) * stride, c, s);
  while (h < h_end) {
#pragma unroll
    for (int k = 0; k < kRotaryBatch; ++k) {
      if (h + k * p.lanes >= h_end) break;
      rope_unit_apply<T>(unit, p.interleaved, a[k], b[k], c, s, dst + (h + k * p.lanes) * dst_h);
    }
    h += kRotaryBatch * p.lanes;
    load(h);
  }
}

}  // namespace
}  // namespace dak

extern "C" int dak_rotary(const dak_rotary_args *r, void *stream) {
  using namespace dak;
  if (!r) return fail(DAK_ERR_INVALID_ARG, "args is null");
  if (r->dtype != DAK_DTYPE_F16 && r->dtype != DAK_DTYPE_BF16)
    return fail(DAK_ERR_UNSUPPORTED, "rotary supports float16 and bfloat16");
  if (r->tokens < 0 || r->heads <= 0 || r->head_dim <= 0 || r->head_dim > 1024)
    return fail(DAK_ERR_INVALID_ARG, "rotary: tokens must not be negative, heads positive, head_dim 1..1024");
  if (r->head_dim % 8) return fail(DAK_ERR_ALIGNMENT, "rotary: head_dim must be a multiple of 8");
  int st = check_rotary_dim(r->rotary_dim, r->head_dim, r->interleaved);
  if (st) return st;
  if (!r->x || !r->out || !r->positions || !r->inv_freq)
    return fail(DAK_ERR_INVALID_ARG, "rotary: x, out, positions and inv_freq are required");
  if (r->x_stride_t % 8 || r->x_stride_h % 8 || r->o_stride_t % 8 || r->o_stride_h % 8 ||
      ((reinterpret_cast<uintptr_t>(r->x) | reinterpret_cast<uintptr_t>(r->out)) & 15u))
    return fail(DAK_ERR_ALIGNMENT, "rotary: x and out must be 16-byte aligned, strides multiples of 8 elements");
  const BlockGrid x = {r->x, r->tokens, 2 * r->x_stride_t, r->heads, 2 * r->x_stride_h, 2 * r->head_dim};
  const BlockGrid out = {r->out, r->tokens, 2 * r->o_stride_t, r->heads, 2 * r->o_stride_h, 2 * r->head_dim};
  if (overlaps_itself(out)) return fail(DAK_ERR_INVALID_ARG, "rotary: heads of out overlap");
  const bool in_place = r->x == r->out && (r->tokens <= 1 || r->x_stride_t == r->o_stride_t) &&
                        (r->heads <= 1 || r->x_stride_h == r->o_stride_h);
  if (!in_place && overlap(x, out)) return fail(DAK_ERR_INVALID_ARG, "rotary: out overlaps x without being x");
  const void *ptrs[4] = {r->x, r->out, r->positions, r->inv_freq};
  for (const void *q : ptrs)
    if ((st = check_gpu_accessible(q, "rotary buffer"))) return st;
  if (r->tokens == 0) return DAK_OK;
  RotaryParams p = {};
  p.x = static_cast<const uint16_t *>(r->x);
  p.out = static_cast<uint16_t *>(r->out);
  p.xt = r->x_stride_t;
  p.xh = r->x_stride_h;
  p.ot = r->o_stride_t;
  p.oh = r->o_stride_h;
  p.positions = r->positions;
  p.inv_freq = r->inv_freq;
  p.scale = r->rope_scale;
  p.tokens = r->tokens;
  p.heads = r->heads;
  p.units = rope_units(r->head_dim, r->rotary_dim, r->interleaved != 0);
  p.rotary_dim = r->rotary_dim;
  p.interleaved = r->interleaved != 0;
  p.pdl = decode_pdl_enabled() ? 1 : 0;
  const int stride = rope_stride(r->rotary_dim), rows = kRotaryThreads / p.units;
  // Four tokens share a CTA where there are enough to fill the GPU.
  p.cta_tokens = 1;
  while (p.cta_tokens < kRotaryTokens && 2 * p.cta_tokens * stride <= kRotaryThreads && 2 * p.cta_tokens <= rows &&
         r->tokens >= 2 * p.cta_tokens * kRotaryTarget)
    p.cta_tokens *= 2;
  p.lanes = rows / p.cta_tokens;
  const long long tiles = ((long long)r->tokens + p.cta_tokens - 1) / p.cta_tokens;
  // Few tokens: their heads on several CTAs, down to one unit per thread.
  const long long slices = std::max(1ll, kRotaryTarget / tiles);
  p.cta_heads = (int)std::max<long long>(std::min(p.lanes, r->heads), (r->heads + slices - 1) / slices);
  const dim3 grid((unsigned)tiles, (unsigned)((r->heads + p.cta_heads - 1) / p.cta_heads));
  if (grid.y > 65535u) return fail(DAK_ERR_UNSUPPORTED, "rotary: too many heads for one launch");
  const size_t smem = 2u * p.cta_tokens * stride * sizeof(float);
  auto s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      r->dtype == DAK_DTYPE_F16
          ? launch_ex(rotary_kernel<__half>, grid, dim3(kRotaryThreads), smem, s, 1, p.pdl != 0, p)
          : launch_ex(rotary_kernel<__nv_bfloat16>, grid, dim3(kRotaryThreads), smem, s, 1, p.pdl != 0, p);
  return cuda_status(e, "rotary launch");
}

namespace dak {
int check_rotary_dim(int rotary_dim, int head_dim, int interleaved) {
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2)
    return fail(DAK_ERR_INVALID_ARG, "rotary_dim must be even and at most head_dim");
  if (!interleaved && rotary_dim % 16)
    return fail(DAK_ERR_UNSUPPORTED, "rotary_dim must be a multiple of 16 in the half layout");
  return DAK_OK;
}
}  // namespace dak
