// dak_rotary.cu - rotary positions of the heads of any number of tokens: half
// or interleaved pairs, all or part of the head, frequencies and attention
// factor as the model's scaling gives them.
//
// Bound by memory: each 16-byte vector is read once and written once.  One
// thread owns one unit (dak_rotary.cuh) of a token and walks over heads, so the
// FP64 angle and sincospif are paid once per unit and head group, not per head.
#include "dak_host.h"
#include "dak_rotary.cuh"

namespace dak {
namespace {

constexpr int kRotaryThreads = 256;

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
  for (int h = g; h < p.heads; h += p.groups) {
    const uint4 *src = reinterpret_cast<const uint4 *>(p.x + t * p.xt + h * p.xh);
    uint4 *dst = reinterpret_cast<uint4 *>(p.out + t * p.ot + h * p.oh);
    const uint4 a = src[unit.v0];
    const uint4 b = unit.v1 >= 0 ? src[unit.v1] : a;
    rope_unit_apply<T>(unit, p.interleaved, a, b, c, s, dst);
  }
}

}  // namespace
}  // namespace dak

extern "C" int dak_rotary(const void *x, int64_t x_stride_t, int64_t x_stride_h, const int32_t *positions,
                          const float *inv_freq, float rope_scale, int interleaved, void *out, int64_t o_stride_t,
                          int64_t o_stride_h, int tokens, int heads, int head_dim, int rotary_dim, int dtype,
                          void *stream) {
  using namespace dak;
  if (dtype != DAK_DTYPE_F16 && dtype != DAK_DTYPE_BF16)
    return fail(DAK_ERR_UNSUPPORTED, "rotary supports float16 and bfloat16");
  if (tokens < 0 || heads <= 0 || head_dim <= 0 || head_dim > 1024)
    return fail(DAK_ERR_INVALID_ARG, "rotary: tokens must not be negative, heads positive, head_dim 1..1024");
  if (head_dim % 8) return fail(DAK_ERR_ALIGNMENT, "rotary: head_dim must be a multiple of 8");
  int st = check_rotary_dim(rotary_dim, head_dim, interleaved);
  if (st) return st;
  if (!x || !out || !positions || !inv_freq)
    return fail(DAK_ERR_INVALID_ARG, "rotary: x, out, positions and inv_freq are required");
  if (x_stride_t % 8 || x_stride_h % 8 || o_stride_t % 8 || o_stride_h % 8 ||
      ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15u))
    return fail(DAK_ERR_ALIGNMENT, "rotary: x and out must be 16-byte aligned, strides multiples of 8 elements");
  const void *ptrs[4] = {x, out, positions, inv_freq};
  for (const void *q : ptrs)
    if ((st = check_gpu_accessible(q, "rotary buffer"))) return st;
  if (tokens == 0) return DAK_OK;
  RotaryParams p = {};
  p.x = static_cast<const uint16_t *>(x);
  p.out = static_cast<uint16_t *>(out);
  p.xt = x_stride_t;
  p.xh = x_stride_h;
  p.ot = o_stride_t;
  p.oh = o_stride_h;
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.scale = rope_scale;
  p.tokens = tokens;
  p.heads = heads;
  p.units = rope_units(head_dim, rotary_dim, interleaved != 0);
  // One head per thread until the GPU's threads are all taken, then more heads
  // per thread.
  const long long per_group = (long long)tokens * p.units;
  p.groups = (int)std::min<long long>(heads, std::max<long long>(1, 600000 / per_group));
  p.rotary_dim = rotary_dim;
  p.interleaved = interleaved != 0;
  p.pdl = decode_pdl_enabled() ? 1 : 0;
  const long long blocks = (per_group * p.groups + kRotaryThreads - 1) / kRotaryThreads;
  if (blocks > 0x7fffffffll) return fail(DAK_ERR_UNSUPPORTED, "rotary: too many tokens for one launch");
  auto s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      dtype == DAK_DTYPE_F16
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
