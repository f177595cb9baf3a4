// New keys and values rounded into the pages of an 8-bit cache: a workgroup takes the tokens that one page receives, for one key head, of K or of V.
//   s = 2^ceil(log2(amax / M)), M = 448 or 127;  held = rne(x / s);  the sum of the page's keys and their mean beside it.
// A power of two leaves nothing to round in x / s and held * s, and a page whose scale grows (a later token is larger) loses by its second rounding
// no more than it would have by one at the larger scale, half a step each.
//
// Bound by memory: two bytes read and one written per feature.  The scale needs the largest value of the page's new rows before any can be
// written: they stay in registers in between where a thread has up to kKept pieces (pages of 128 tokens and heads of 128), and are read again from the
// caches beyond.  14272 tokens, 8 heads of 128, pages of 64: 23.0 us, 88 MB at 3.8 TB/s.  (30.6 with a comparison, a choice and a rounding of its own for every element: the
// vector unit had half of the time.  So magnitudes are compared as whole numbers, two at a time, and only a thread that sees an infinity or a NaN looks at each;
// and a value is rounded to int8 by one addition.  Held to 64 registers, for eight waves a SIMD instead of seven, it spills: 25.0.)
// A decode step brings one row per page: there it is a launch and three dependent loads (5.4 us, 16 requests).
#include "kv_cache.h"
#include "rotary.h"

#include <algorithm>

namespace fmoba {

constexpr int kAppendThreads = 256;
constexpr int kKept = 8;

template <typename T>
constexpr uint32_t kInfBits = std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u;

// The largest magnitude's bits of a thread's pieces: without their signs, the bits of two elements are ordered as their values are (NaNs above all).
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
template <typename T>
__device__ __forceinline__ uint32_t largest_bits(const Pack8 (&x)[kKept]) {
  u16x2 most = {0, 0};
#pragma unroll
  for (int i = 0; i < kKept; ++i) {
    uint32_t w[4];
    __builtin_memcpy(w, &x[i], 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t abs = w[j] & 0x7fff7fffu;
      u16x2 two;
      __builtin_memcpy(&two, &abs, 4);
      most = __builtin_elementwise_max(most, two);
    }
  }
  return max((uint32_t)most.x, (uint32_t)most.y);
}

template <typename T, typename H, bool SURE>
__device__ __forceinline__ uint2 pack_row(const Pack8 &x, float inv) {
  float f[8];
  unpack8<T>(x, f);
  uint2 w;
  w.x = H::template pack4<SURE>(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
  w.y = H::template pack4<SURE>(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
  return w;
}

// TURN: the keys are turned by their positions first, as fmoba_rotary does, and workgroups behind the others turn the queries, one a token.  Of a serving step of 16 requests, 32 over
// 8 heads of 128, it spares a launch: 35.7 instead of 38.3 us.
constexpr int kTurnRows = FMOBA_TURN_ROWS;  // new tokens of a sequence, at most: their angles lie in LDS, once for every head
struct NoTurn {};
template <typename T>
__device__ __forceinline__ void turn_piece(const fmoba_rotary_args &r, const uint16_t *src, uint16_t *dst, const float2 *cs, int piece, int turned) {
  if (piece >= turned) {
    const int e = r.rotary_dim + (piece - turned) * 8;
    *reinterpret_cast<Pack8 *>(dst + e) = ld_global16(src + e);
  } else if (r.interleaved) {
    rotate_piece<T, 8, true>(src, dst, cs, piece, r.rotary_dim / 2);
  } else if (r.rotary_dim % 16 == 0) {
    rotate_piece<T, 8, false>(src, dst, cs, piece, r.rotary_dim / 2);
  } else {
    rotate_piece<T, 4, false>(src, dst, cs, piece, r.rotary_dim / 2);
  }
}

template <typename T, typename H, bool TURN>
__global__ __launch_bounds__(kAppendThreads) void cache_append_kernel(fmoba_cache_append_args a, std::conditional_t<TURN, fmoba_rotary_args, NoTurn> turn) {
  __shared__ __align__(16) float sSum[kAppendThreads * 8];
  __shared__ float sMax[kAppendThreads / 64];
  __shared__ __align__(16) uint16_t sRows[TURN ? kTurnRows * 256 : 8];
  const fmoba_kv_cache &c = a.cache;
  const int b = blockIdx.y, tid = threadIdx.x, P = c.page_size, D = c.head_dim;
  const bool is_k = (blockIdx.x & 1) == 0;
  const int nth = (int)(blockIdx.x >> 1) / c.heads_k, hk = (int)(blockIdx.x >> 1) - nth * c.heads_k;  // (the heads of a token side by side: its row is read at one time)
  const int row0 = min(max(a.cu_seqlens[b], 0), a.total_new), row1 = min(max(a.cu_seqlens[b + 1], row0), a.total_new);
  int pairs = 0, turned = 0, pieces = 0;  // of a head
  if constexpr (TURN) {
    pairs = turn.rotary_dim / 2;
    turned = turn.interleaved ? turn.rotary_dim / 8 : turn.rotary_dim % 16 == 0 ? pairs / 8 : pairs / 4;
    pieces = turned + (D - turn.rotary_dim) / 8;
    float2 *angles = reinterpret_cast<float2 *>(sSum);
    const int nq = min(a.max_seqlen_new, a.total_new), t = row0 + (int)blockIdx.x - ((int)gridDim.x - nq);
    if (t >= row0) {
      if (t >= row1) return;
      if (tid < pairs) angles[tid] = turn_of(turn, t, tid);
      __syncthreads();
      for (int i = tid; i < turn.heads * pieces; i += kAppendThreads) {
        const int h = i / pieces;
        turn_piece<T>(turn, reinterpret_cast<const uint16_t *>(turn.q) + (int64_t)t * turn.q_row_stride + (int64_t)h * turn.q_head_stride,
                      reinterpret_cast<uint16_t *>(turn.q_out) + (int64_t)t * turn.qo_row_stride + (int64_t)h * turn.qo_head_stride, angles, i - h * pieces, turned);
      }
      return;
    }
  }
  const int end = a.seqlens_k[b], start = end - (row1 - row0);
  const int slot = max(start, 0) / P + nth;
  if (slot >= a.max_pages || (int64_t)slot * P >= end) return;
  const int lo = max(start, slot * P), hi = min(min((int64_t)end, (int64_t)slot * P + P), TURN ? (int64_t)lo + kTurnRows : INT64_MAX);  // the new tokens of the page
  if (lo >= hi) return;
  const int old = lo - slot * P;  // tokens that it has already
  const int page = a.block_table[(int64_t)b * a.table_stride + slot];  // (looked at when the first rows are on their way)

  const int lanes = D / 8, rows = kAppendThreads / lanes;  // threads of a row (8 features each), rows of a pass
  const int r = tid / lanes, e = (tid - r * lanes) * 8;
  const bool works = r < rows;
  const int64_t src_stride = is_k ? a.k_row_stride : a.v_row_stride;
  const uint16_t *src = reinterpret_cast<const uint16_t *>(is_k ? a.k : a.v) + (int64_t)(row0 + (lo - start)) * src_stride + (int64_t)hk * (is_k ? a.k_head_stride : a.v_head_stride) + e;
  // ---- the largest finite magnitude, and the sums of the features ----
  const int n = hi - lo;
  if constexpr (TURN) {
    if (is_k) {
      float2 *angles = reinterpret_cast<float2 *>(sSum);
      for (int i = tid; i < n * pairs; i += kAppendThreads) angles[i] = turn_of(turn, row0 + (lo - start) + i / pairs, i % pairs);
      __syncthreads();
      for (int i = tid; i < n * pieces; i += kAppendThreads) {
        const int row = i / pieces;
        turn_piece<T>(turn, src - e + (int64_t)row * src_stride, sRows + row * D, angles + row * pairs, i - row * pieces, turned);
      }
      __syncthreads();  // (the angles' place is the sums' from here on)
    }
  }
  Pack8 x[kKept];
  bool sure = true;  // all of this thread's values are finite
  float amax = 0.f, sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto load = [&](int i0) {
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
      const int row = i0 + i * rows + r;
      if (TURN && is_k)
        x[i] = works && row < n ? *reinterpret_cast<const Pack8 *>(sRows + row * D + e) : zero_pack8();
      else
        x[i] = works && row < n ? ld_global16(src + (int64_t)row * src_stride) : zero_pack8();
    }
  };
  const int at_once = rows * kKept;  // rows that the whole workgroup keeps
  load(0);
  if (page < 0 || page >= c.num_pages) return;
  const int64_t at = (int64_t)page * c.heads_k + hk;
  const int64_t dst_stride = is_k ? c.k_token_stride : c.v_token_stride;
  uint8_t *held = reinterpret_cast<uint8_t *>(is_k ? c.k : c.v) + (int64_t)page * (is_k ? c.k_page_stride : c.v_page_stride) + (int64_t)hk * (is_k ? c.k_head_stride : c.v_head_stride) + e;
  float *scale_at = (is_k ? c.k_scale : c.v_scale) + at;
  const float was = old > 0 ? *scale_at : 0.f;
  for (int i0 = 0; i0 < n; i0 += at_once) {
    if (i0 > 0) load(i0);
    const uint32_t most = largest_bits<T>(x);
    if (most < kInfBits<T>) {
      T value;
      const uint16_t bits = (uint16_t)most;
      __builtin_memcpy(&value, &bits, 2);
      amax = fmaxf(amax, (float)value);
    } else {  // (an infinity or a NaN among them: the largest of the others)
      sure = false;
#pragma unroll
      for (int i = 0; i < kKept; ++i) {
        float f[8];
        unpack8<T>(x[i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fabsf(f[j]) < INFINITY ? fmaxf(amax, fabsf(f[j])) : amax;
      }
    }
    if (is_k)
#pragma unroll
      for (int i = 0; i < kKept; ++i) {
        float f[8];
        unpack8<T>(x[i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += f[j];
      }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
  if ((tid & 63) == 0) sMax[tid >> 6] = amax;
  if (is_k && works) {
#pragma unroll
    for (int j = 0; j < 8; ++j) sSum[r * D + e + j] = sum[j];
  }
  __syncthreads();
  amax = fmaxf(fmaxf(sMax[0], sMax[1]), fmaxf(sMax[2], sMax[3]));
  const float scale = old > 0 ? fmaxf(scale_of<H>(amax), was) : scale_of<H>(amax);
  if (tid == 0) {
    *scale_at = scale;
    if (is_k && old == 0 && c.weight != nullptr) c.weight[at] = 0;
  }

  // ---- what the page has, at its new scale ----
  if (scale > was && old > 0 && works) {
    const float ratio = was / scale;
    for (int row = r; row < old; row += rows) {
      uint2 *p = reinterpret_cast<uint2 *>(held + (int64_t)row * dst_stride);
      uint2 w = *p;
      float f[4], g[4];
      H::unpack4(w.x, f);
      H::unpack4(w.y, g);
      w.x = H::pack4(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
      w.y = H::pack4(g[0] * ratio, g[1] * ratio, g[2] * ratio, g[3] * ratio);
      *p = w;
    }
  }
  // ---- the new rows ----
  const float inv = 1.f / scale;
  for (int i0 = 0; i0 < n; i0 += at_once) {
    if (n > at_once) load(i0);
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
      const int row = i0 + i * rows + r;
      if (!works || row >= n) continue;
      const uint2 w = sure ? pack_row<T, H, true>(x[i], inv) : pack_row<T, H, false>(x[i], inv);
      *reinterpret_cast<uint2 *>(held + (int64_t)(old + row) * dst_stride) = w;
    }
  }
  if (is_k && tid < D) {
    float s = 0.f;
    for (int i = 0; i < rows; ++i) s += sSum[i * D + tid];
    float *k_sum = c.k_sum + at * D + tid;
    if (old > 0) s += *k_sum;
    *k_sum = s;
    reinterpret_cast<uint16_t *>(c.k_mean)[at * D + tid] = float_to_elem_bits<T>(s / (float)(old + n));
  }
}

// turn: the positions, or null
static int append(const fmoba_cache_append_args *a, const fmoba_rotary_args *turn, hipStream_t s) {
  FMOBA_REQUIRE(a != nullptr, "cache_append: null args");
  FMOBA_CHECK_CACHE(a->cache);
  FMOBA_REQUIRE(a->batch >= 1 && a->batch <= 65535 && a->total_new >= 0 && a->max_seqlen_new >= 0 && a->max_pages >= 0, "cache_append: sizes must not be negative, batch at most 65535");
  if (a->total_new == 0 || a->max_seqlen_new == 0 || ((a->max_pages == 0 || a->cache.num_pages == 0) && turn == nullptr)) return 0;
  const bool pages = a->max_pages > 0 && a->cache.num_pages > 0;
  FMOBA_REQUIRE(a->k && a->v && a->cu_seqlens && a->seqlens_k && (!pages || (a->block_table && a->cache.k_sum)), "cache_append: null pointer");
  FMOBA_REQUIRE(a->k_row_stride % 8 == 0 && a->k_head_stride % 8 == 0 && a->v_row_stride % 8 == 0 && a->v_head_stride % 8 == 0, "cache_append: strides must be multiples of 8 elements");
  FMOBA_REQUIRE((((uintptr_t)a->k | (uintptr_t)a->v) % 16) == 0, "cache_append: k and v must be 16-byte aligned");
  // the pages that max_seqlen_new tokens can touch, K and V apart
  const int64_t most = std::min<int64_t>(a->max_seqlen_new, a->total_new);
  const int64_t touched = pages ? std::min<int64_t>(ceil_div64(most, a->cache.page_size) + 1, a->max_pages) : 0;
  const int64_t groups = 2 * touched * a->cache.heads_k + (turn ? most : 0);
  FMOBA_REQUIRE(groups * kAppendThreads <= UINT32_MAX, "cache_append: too many tokens of a sequence for the launch grid");
  const dim3 grid((uint32_t)groups, a->batch), block(kAppendThreads);
  const bool bf16 = a->cache.dtype == FMOBA_DTYPE_BF16, e4m3 = a->cache.format == FMOBA_CACHE_E4M3;
  if (turn) {
    auto kern = bf16 ? (e4m3 ? cache_append_kernel<bf16_t, HeldE4M3, true> : cache_append_kernel<bf16_t, HeldInt8, true>)
                     : (e4m3 ? cache_append_kernel<f16_t, HeldE4M3, true> : cache_append_kernel<f16_t, HeldInt8, true>);
    hipLaunchKernelGGL(kern, grid, block, 0, s, *a, *turn);
  } else {
    auto kern = bf16 ? (e4m3 ? cache_append_kernel<bf16_t, HeldE4M3, false> : cache_append_kernel<bf16_t, HeldInt8, false>)
                     : (e4m3 ? cache_append_kernel<f16_t, HeldE4M3, false> : cache_append_kernel<f16_t, HeldInt8, false>);
    hipLaunchKernelGGL(kern, grid, block, 0, s, *a, NoTurn{});
  }
  FMOBA_LAUNCH_CHECK("cache_append_kernel");
  return 0;
}

}  // namespace fmoba

extern "C" int fmoba_cache_append(const fmoba_cache_append_args *a, void *stream) { return fmoba::append(a, nullptr, (hipStream_t)stream); }

extern "C" int fmoba_cache_append_turned(const fmoba_cache_append_args *a, const fmoba_rotary_args *turn, void *stream) {
  using namespace fmoba;
  FMOBA_REQUIRE(a != nullptr && turn != nullptr, "cache_append: null args");
  if (int rc = check_rotary_args(turn, false)) return rc;
  FMOBA_REQUIRE(turn->total == a->total_new && turn->heads_k == a->cache.heads_k && turn->head_dim == a->cache.head_dim && turn->dtype == a->cache.dtype && turn->k == a->k &&
                    turn->k_row_stride == a->k_row_stride && turn->k_head_stride == a->k_head_stride,
                "cache_append: the keys to turn are not the keys to append");
  FMOBA_REQUIRE(a->max_seqlen_new <= kTurnRows, "cache_append: positions for up to %d new tokens of a sequence", kTurnRows);
  return append(a, turn, (hipStream_t)stream);
}
