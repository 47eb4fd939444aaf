// dak_rotary.cuh - rotary positions of 8-dim vectors, shared by the stand-alone
// rotary kernel and the 4-bit KV append.
//
// The first R dims of a head are rotated in pairs by the angle
// position * inv_freq[i]: half layout pairs (i, i + R/2), interleaved layout
// pairs (2i, 2i + 1); both outputs are scaled by the attention factor a:
//   y1 = a (x1 cos t - x2 sin t),  y2 = a (x2 cos t + x1 sin t).
// Angles of far positions lose bits in FP32 (at position 131072 and frequency 1
// the product's last bit is 1/128 rad), so the turn count is formed in FP64, its
// whole turns are dropped there, and only the remaining half turns in [-1, 1]
// go to FP32 and sincospif: the angle is good to about 1e-7 rad at any int32
// position.  The rotation is FP32; callers round once.
#pragma once

#include "dak_common.cuh"

namespace dak {

__device__ __forceinline__ void rope_cos_sin(int pos, float inv_freq, float scale, float &c, float &s) {
  const double turns = (double)pos * ((double)inv_freq * 0.15915494309189535);  // 1 / (2 pi)
  sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
  c *= scale;
  s *= scale;
}

__device__ __forceinline__ void rope_turn(float &x1, float &x2, float c, float s) {
  const float y1 = fmaf(x1, c, -(x2 * s));
  x2 = fmaf(x2, c, x1 * s);
  x1 = y1;
}

// 8 values of a 16-byte vector in FP32, and back (one rounding each).
template <typename T> __device__ __forceinline__ void unpack8(const uint4 &v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem<T>::to_float2(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T> __device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(Elem<T>::pack2(x[0], x[1]), Elem<T>::pack2(x[2], x[3]), Elem<T>::pack2(x[4], x[5]),
                    Elem<T>::pack2(x[6], x[7]));
}

// One unit of work on a row (a head) of `head_dim` dims, R of them rotated: a
// pair of vectors (half layout), one vector of 4 pairs (interleaved), or one
// vector that passes through.
struct RopeUnit {
  int v0, v1;   // vectors of 8 dims; v1 < 0: one vector
  int pairs;    // rotated pairs: 8 (half), 0..4 (interleaved), 0 (passes through)
  int freq0;    // frequency of the first pair
};

__host__ __device__ __forceinline__ int rope_units(int head_dim, int rotary_dim, int interleaved) {
  return interleaved ? head_dim / 8 : head_dim / 8 - rotary_dim / 16;
}

__device__ __forceinline__ RopeUnit rope_unit(int u, int rotary_dim, int interleaved) {
  RopeUnit r;
  if (interleaved) {
    r.v0 = u;
    r.v1 = -1;
    r.pairs = max(0, min(4, rotary_dim / 2 - 4 * u));
    r.freq0 = 4 * u;
  } else {
    const int half = rotary_dim / 16;
    const bool pair = u < half;
    r.v0 = pair ? u : u + half;
    r.v1 = pair ? u + half : -1;
    r.pairs = pair ? 8 : 0;
    r.freq0 = 8 * u;
  }
  return r;
}

// The angles of `tokens` tokens for a whole CTA, each worked out once: cosines
// [tokens][stride], then sines, in shared memory.  stride is rotary_dim / 2
// rounded up to 8 so that 4 neighbours are one aligned load.
__host__ __device__ __forceinline__ int rope_stride(int rotary_dim) { return (rotary_dim / 2 + 7) / 8 * 8; }

__device__ __forceinline__ void rope_table(float *tab, const int32_t *positions, int tokens, int max_tokens,
                                           const float *inv_freq, int rotary_dim, float scale) {
  const int stride = rope_stride(rotary_dim), half = rotary_dim / 2;
  for (int i = threadIdx.x; i < tokens * stride; i += blockDim.x) {
    const int t = i / stride, f = i - t * stride;
    float c = 1.f, s = 0.f;
    if (f < half) rope_cos_sin(positions[t], inv_freq[f], scale, c, s);
    tab[i] = c;
    tab[max_tokens * stride + i] = s;
  }
}

__device__ __forceinline__ void load4(const float *from, float *to) {
  const float4 v = *reinterpret_cast<const float4 *>(from);
  to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
}

// cos and sin of a unit's pairs from a token's row of the table.
__device__ __forceinline__ void rope_unit_angles(const RopeUnit &u, const float *cos_row, const float *sin_row, float (&c)[8],
                                                 float (&s)[8]) {
  if (u.pairs > 0) {
    load4(cos_row + u.freq0, c);
    load4(sin_row + u.freq0, s);
  }
  if (u.pairs > 4) {
    load4(cos_row + u.freq0 + 4, c + 4);
    load4(sin_row + u.freq0 + 4, s + 4);
  }
}

// Rotates a unit of a row from src to dst (which may be the same row).
template <typename T>
__device__ __forceinline__ void rope_unit_apply(const RopeUnit &u, int interleaved, uint4 a, uint4 b,
                                                const float (&c)[8], const float (&s)[8], uint4 *dst) {
  float x[8];
  unpack8<T>(a, x);
  if (u.v1 >= 0) {
    float y[8];
    unpack8<T>(b, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) rope_turn(x[i], y[i], c[i], s[i]);
    dst[u.v0] = pack8<T>(x);
    dst[u.v1] = pack8<T>(y);
  } else {
    if (interleaved) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < u.pairs) rope_turn(x[2 * i], x[2 * i + 1], c[i], s[i]);
    }
    dst[u.v0] = u.pairs > 0 ? pack8<T>(x) : a;
  }
}

}  // namespace dak
