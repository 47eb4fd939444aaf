// dak_rotary.cu - rotary positions of the heads of any number of tokens: half
// or interleaved pairs, all or part of the head, frequencies and attention
// factor as the model's scaling gives them.
//
// Bound by memory: each 16-byte vector is read once and written once.  One
// thread owns one unit (dak_rotary.cuh) of a token and walks over heads, four at
// a time so that eight loads are in flight, and the FP64 angles and sincospif are
// paid once per unit and head group, not per head.
#include "dak_host.h"
#include "dak_rotary.cuh"

namespace dak {
namespace {

constexpr int kRotaryThreads = 256;
constexpr long long kRotaryTarget = 200000;  // threads that fill the GPU

struct RotaryParams {
  const uint16_t *x;
  uint16_t *out;
  long long xt, xh, ot, oh;  // token and head strides, elements
  const int32_t *positions;
  const float *inv_freq;
  float scale;
  int tokens, heads, units, groups;  // groups: head groups; group g owns heads g, g + groups, ...
  int rotary_dim, interleaved, pdl;
};

template <typename T>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  pdl_enter(p.pdl);
  const long long i = (long long)blockIdx.x * kRotaryThreads + threadIdx.x;
  const long long row = i / p.units;
  const int u = (int)(i - row * p.units);
  const int t = (int)(row / p.groups);
  const int g = (int)(row - (long long)t * p.groups);
  if (t >= p.tokens) return;
  const RopeUnit unit = rope_unit(u, p.rotary_dim, p.interleaved);
  float c[8], s[8];
  rope_unit_angles(unit, p.positions[t], p.inv_freq, p.scale, c, s);
  constexpr int kBatch = 4;
  for (int h0 = g; h0 < p.heads; h0 += kBatch * p.groups) {
    uint4 a[kBatch], b[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int h = h0 + k * p.groups;
      if (h >= p.heads) break;
      const uint4 *src = reinterpret_cast<const uint4 *>(p.x + t * p.xt + h * p.xh);
      a[k] = src[unit.v0];
      b[k] = unit.v1 >= 0 ? src[unit.v1] : a[k];
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int h = h0 + k * p.groups;
      if (h >= p.heads) break;
      rope_unit_apply<T>(unit, p.interleaved, a[k], b[k], c, s, reinterpret_cast<uint4 *>(p.out + t * p.ot + h * p.oh));
    }
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
  // One head per thread until the GPU's threads are all taken, then more heads
  // per thread.
  const long long per_group = (long long)r->tokens * p.units;
  p.groups = (int)std::min<long long>(r->heads, std::max<long long>(1, kRotaryTarget / per_group));
  p.rotary_dim = r->rotary_dim;
  p.interleaved = r->interleaved != 0;
  p.pdl = decode_pdl_enabled() ? 1 : 0;
  const long long blocks = (per_group * p.groups + kRotaryThreads - 1) / kRotaryThreads;
  if (blocks > 0x7fffffffll) return fail(DAK_ERR_UNSUPPORTED, "rotary: too many tokens for one launch");
  auto s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      r->dtype == DAK_DTYPE_F16
          ? launch_ex(rotary_kernel<__half>, dim3((unsigned)blocks), dim3(kRotaryThreads), 0, s, 1, p.pdl != 0, p)
          : launch_ex(rotary_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(kRotaryThreads), 0, s, 1, p.pdl != 0, p);
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
