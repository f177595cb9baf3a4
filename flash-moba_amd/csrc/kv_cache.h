// What the kernels of the paged 8-bit cache share: the two formats, and the checks of its description.
#pragma once

#include "fmoba_common.h"

namespace fmoba {

// E4M3 and INT8 as types for templates.
//   unpack4: four values of a 32-bit word in units of their scale, exact in 32 bits
//   pack4:   four values in units of their scale, rounded to nearest (ties to even), cut off at the largest; int8 holds a NaN as 0.  SURE: no NaN among them
struct HeldE4M3 {
  static constexpr int kFormat = FMOBA_CACHE_E4M3;
  static __device__ __forceinline__ void unpack4(uint32_t w, float (&f)[4]) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    f[0] = lo[0], f[1] = lo[1], f[2] = hi[0], f[3] = hi[1];
#else
    (void)w, (void)f;
#endif
  }
  // four values as two words of two 16-bit elements, exact
  template <typename T>
  static __device__ __forceinline__ void widen4(uint32_t w, uint32_t &lo, uint32_t &hi) {
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (std::is_same<T, bf16_t>::value) {
      const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.f, true);
      __builtin_memcpy(&lo, &a, 4);
      __builtin_memcpy(&hi, &b, 4);
    } else {
      const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, true);
      __builtin_memcpy(&lo, &a, 4);
      __builtin_memcpy(&hi, &b, 4);
    }
#else
    (void)w, (void)lo, (void)hi;
#endif
  }
  // whether any of four values is NaN (all bits but the sign set)
  static __device__ __forceinline__ bool any_nan4(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0u; }
  // the values with zeros for NaNs
  static __device__ __forceinline__ uint32_t without_nan4(uint32_t w) {
    const uint32_t nan = (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;  // 1 in the bytes that are
    return w & ~(nan * 255u);
  }
  template <bool SURE>
  static __device__ __forceinline__ float limit(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
    const float y = __builtin_amdgcn_fmed3f(x, -448.f, 448.f);
    return !SURE && x != x ? x : y;
#else
    return x;
#endif
  }
  template <bool SURE = false>
  static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
#if defined(__HIP_DEVICE_COMPILE__)
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(limit<SURE>(a), limit<SURE>(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(limit<SURE>(c), limit<SURE>(d), w, true);
#else
    (void)a, (void)b, (void)c, (void)d;
    return 0;
#endif
  }
  // exponent of the least power of two s with amax <= 448 s, amax = m 2^x, 1 <= m < 2: 448 = 1.75 * 2^8
  static __device__ __forceinline__ int scale_exponent(float m, int x) { return x - 8 + (m > 1.75f ? 1 : 0); }
};
struct HeldInt8 {
  static constexpr int kFormat = FMOBA_CACHE_INT8;
  static __device__ __forceinline__ void unpack4(uint32_t w, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i));
  }
  template <typename T>
  static __device__ __forceinline__ void widen4(uint32_t w, uint32_t &lo, uint32_t &hi) {
    float f[4];
    unpack4(w, f);
    lo = pack2<T>(f[0], f[1]);
    hi = pack2<T>(f[2], f[3]);
  }
  static __device__ __forceinline__ bool any_nan4(uint32_t) { return false; }
  static __device__ __forceinline__ uint32_t without_nan4(uint32_t w) { return w; }
  // 1.5 * 2^23 + x, |x| <= 127: the sum's unit is 1, so it is rounded to a whole number, whose low byte is x's
  template <bool SURE>
  static __device__ __forceinline__ uint32_t pack1(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
    const float y = __builtin_amdgcn_fmed3f(x, -127.f, 127.f);
    return __float_as_uint((!SURE && x != x ? 0.f : y) + 12582912.f);
#else
    return (void)x, 0;
#endif
  }
  template <bool SURE = false>
  static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
#if defined(__HIP_DEVICE_COMPILE__)
    const uint32_t lo = __builtin_amdgcn_perm(pack1<SURE>(b), pack1<SURE>(a), 0x0c0c0400u), hi = __builtin_amdgcn_perm(pack1<SURE>(d), pack1<SURE>(c), 0x04000c0cu);
    return lo | hi;
#else
    return (void)a, (void)b, (void)c, (void)d, 0;
#endif
  }
  // 127 = 1.984375 * 2^6
  static __device__ __forceinline__ int scale_exponent(float m, int x) { return x - 6 + (m > 1.984375f ? 1 : 0); }
};
constexpr int kLeastScale = -64, kLargestScale = 64;  // exponents
template <typename H>
__device__ __forceinline__ float scale_of(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = amax < 1e-30f ? kLeastScale : H::scale_exponent(__uint_as_float((u & 0x7fffffu) | 0x3f800000u), (int)(u >> 23) - 127);
  return __uint_as_float((uint32_t)(min(max(e, kLeastScale), kLargestScale) + 127) << 23);
}

#define FMOBA_CHECK_CACHE(c)                                                                                                                            \
  do {                                                                                                                                                  \
    FMOBA_REQUIRE((c).dtype == FMOBA_DTYPE_F16 || (c).dtype == FMOBA_DTYPE_BF16, "FlashMoBA only supports fp16 and bf16 data types");                   \
    FMOBA_REQUIRE((c).format == FMOBA_CACHE_E4M3 || (c).format == FMOBA_CACHE_INT8, "cache: values are held as e4m3 or int8");                          \
    FMOBA_REQUIRE((c).page_size >= 64 && (c).page_size <= 1024 && (c).page_size % 64 == 0, "cache: page_size must be a multiple of 64 up to 1024");     \
    FMOBA_REQUIRE((c).head_dim >= 16 && (c).head_dim <= 256 && (c).head_dim % 16 == 0, "cache: head_size must be a multiple of 16 up to 256");          \
    FMOBA_REQUIRE((c).num_pages >= 0 && (c).heads_k >= 1 && (c).heads_k <= 65535, "cache: negative number of pages, or no or too many heads");          \
    FMOBA_REQUIRE((c).num_pages == 0 || ((c).k && (c).v && (c).k_scale && (c).v_scale && (c).k_mean), "cache: null pointer");                           \
    FMOBA_REQUIRE((((c).k_page_stride | (c).k_head_stride | (c).k_token_stride | (c).v_page_stride | (c).v_head_stride | (c).v_token_stride) & 15) == 0, \
                  "cache: strides must be multiples of 16 elements");                                                                                   \
    FMOBA_REQUIRE((((uintptr_t)(c).k | (uintptr_t)(c).v | (uintptr_t)(c).k_mean) & 15) == 0, "cache: k, v and k_mean must be 16-byte aligned");         \
  } while (0)

}  // namespace fmoba
