// What turns a head by its token's angles (rotary.hip, kv_append.hip): the bits are the same wherever it is done.
#pragma once

#include "fmoba_common.h"

namespace fmoba {

// cosine and sine of pair j's angle at token t
__device__ __forceinline__ float2 turn_of(const fmoba_rotary_args &a, int64_t t, int j) {
  int axis = 0, end = a.sections[0];
  while (axis + 1 < a.axes && j >= end) end += a.sections[++axis];
  const int64_t at = axis * a.pos_axis_stride + t;
  const double pos = a.positions_64 ? (double)reinterpret_cast<const int64_t *>(a.positions)[at] : (double)reinterpret_cast<const int32_t *>(a.positions)[at];
  const double turns = pos * (exp2(a.log2_base * (-2.0 * j / a.rotary_dim)) * 0.15915494309189533577);
  float s, c;
  sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
  return make_float2(c, a.inverse ? -s : s);
}
// one rounding of a product and one of the sum, whatever the code around them
__device__ __forceinline__ float turned_x(float x, float y, float2 c) { return __builtin_fmaf(x, c.x, -(y * c.y)); }
__device__ __forceinline__ float turned_y(float x, float y, float2 c) { return __builtin_fmaf(x, c.y, y * c.x); }

// W: features of a vector, 8, or 4 where half of rotary_dim is no multiple of 8
template <typename T, int W, bool INTERLEAVED>
__device__ __forceinline__ void rotate_piece(const uint16_t *src, uint16_t *dst, const float2 *cs, int piece, int half) {
  constexpr int NW = W / 2;  // 32-bit words of a vector
  typedef uint32_t vec __attribute__((ext_vector_type(NW)));
  auto value = [](uint32_t w, int i) { return elem_to_float<T>((uint16_t)(w >> (16 * i))); };
  if constexpr (INTERLEAVED) {
    vec x = *reinterpret_cast<const vec *>(src + piece * W);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const float2 c = cs[piece * NW + i];
      const float a = value(x[i], 0), b = value(x[i], 1);
      x[i] = pack2<T>(turned_x(a, b, c), turned_y(a, b, c));
    }
    *reinterpret_cast<vec *>(dst + piece * W) = x;
  } else {
    vec x = *reinterpret_cast<const vec *>(src + piece * W), y = *reinterpret_cast<const vec *>(src + half + piece * W);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const float2 c0 = cs[piece * W + 2 * i], c1 = cs[piece * W + 2 * i + 1];
      const float a0 = value(x[i], 0), a1 = value(x[i], 1), b0 = value(y[i], 0), b1 = value(y[i], 1);
      x[i] = pack2<T>(turned_x(a0, b0, c0), turned_x(a1, b1, c1));
      y[i] = pack2<T>(turned_y(a0, b0, c0), turned_y(a1, b1, c1));
    }
    *reinterpret_cast<vec *>(dst + piece * W) = x;
    *reinterpret_cast<vec *>(dst + half + piece * W) = y;
  }
}

// checks of a call, with or without a place for the turned keys; 0 if all is well
int check_rotary_args(const fmoba_rotary_args *a, bool k_out);

}  // namespace fmoba
