// Rotary positions with several axes: pair j of the first rotary_dim features of a head is turned by the angle
//   theta = positions[axis of j][token] * base^(-2 j / rotary_dim),
//   (x, y) -> (x cos - y sin, x sin + y cos);   backward (inverse): by -theta.
// Pairs are (j, j + rotary_dim / 2), or (2 j, 2 j + 1) interleaved; the axes have consecutive runs of pairs; features behind rotary_dim are copied.
//
// Bound by memory: every feature of q and k is read once and written once.  The angles of a token are the same for all of its heads, so a
// workgroup takes whole tokens, as many as give each of its threads an angle, and keeps their cosines and sines in LDS.  An angle is formed in
// 64 bits as a number of turns and reduced there (positions reach 2^31; in 32 bits position 262144 would be off by 0.01 radians), sine and cosine of the rest
// are taken in 32 bits.  24571 tokens, 16 and 16 heads of 128, there and back: 150 us, 0.8 GB at 5.4 TB/s; one token of each of 16 requests: 5.4 us.
#include "rotary.h"

#include <algorithm>

namespace fmoba {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryPairs = 128;  // of a head, at most (rotary_dim <= 256)

template <typename T, int W, bool INTERLEAVED>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(fmoba_rotary_args a, int tokens) {  // tokens: of a workgroup
  __shared__ float2 sTurn[kRotaryThreads];
  const int tid = threadIdx.x, pairs = a.rotary_dim / 2;
  const int64_t t0 = (int64_t)blockIdx.x * tokens;
  const int nt = (int)min((int64_t)tokens, a.total - t0);
  for (int i = tid; i < nt * pairs; i += kRotaryThreads) {
    const int t = i / pairs, j = i - t * pairs;
    sTurn[i] = turn_of(a, t0 + t, j);
  }
  __syncthreads();
  const int turned = INTERLEAVED ? a.rotary_dim / W : pairs / W, copied = (a.head_dim - a.rotary_dim) / 8;
  const int pieces = turned + copied, heads = a.heads + a.heads_k, items = nt * heads * pieces;
  for (int i = tid; i < items; i += kRotaryThreads) {
    const int r = i / pieces, piece = i - r * pieces;
    const int t = r / heads, h = r - t * heads;
    const bool is_q = h < a.heads;
    const int64_t row = t0 + t, head = is_q ? h : h - a.heads;
    const uint16_t *src = reinterpret_cast<const uint16_t *>(is_q ? a.q : a.k) + row * (is_q ? a.q_row_stride : a.k_row_stride) + head * (is_q ? a.q_head_stride : a.k_head_stride);
    uint16_t *dst = reinterpret_cast<uint16_t *>(is_q ? a.q_out : a.k_out) + row * (is_q ? a.qo_row_stride : a.ko_row_stride) + head * (is_q ? a.qo_head_stride : a.ko_head_stride);
    if (piece < turned) {
      rotate_piece<T, W, INTERLEAVED>(src, dst, sTurn + t * pairs, piece, pairs);
    } else {
      const int e = a.rotary_dim + (piece - turned) * 8;
      *reinterpret_cast<Pack8 *>(dst + e) = ld_global16(src + e);
    }
  }
}

// of a workgroup: a thread an angle; fewer where that leaves less than two workgroups per compute unit
static int rotary_tokens(const fmoba_rotary_args &a) {
  int tokens = std::max(1, kRotaryThreads / (a.rotary_dim / 2));
  while (tokens > 1 && a.total / tokens < 512) tokens /= 2;
  return tokens;
}
template <typename T>
static void launch_rotary(const fmoba_rotary_args &a, hipStream_t s) {
  const int tokens = rotary_tokens(a);
  const dim3 grid((uint32_t)ceil_div64(a.total, tokens)), block(kRotaryThreads);
  if (a.interleaved)
    hipLaunchKernelGGL((rotary_kernel<T, 8, true>), grid, block, 0, s, a, tokens);
  else if (a.rotary_dim % 16 == 0)
    hipLaunchKernelGGL((rotary_kernel<T, 8, false>), grid, block, 0, s, a, tokens);
  else
    hipLaunchKernelGGL((rotary_kernel<T, 4, false>), grid, block, 0, s, a, tokens);
}

int check_rotary_args(const fmoba_rotary_args *a, bool k_out) {
  FMOBA_REQUIRE(a != nullptr, "rotary: null args");
  FMOBA_REQUIRE(a->dtype == FMOBA_DTYPE_F16 || a->dtype == FMOBA_DTYPE_BF16, "FlashMoBA only supports fp16 and bf16 data types");
  FMOBA_REQUIRE(a->total >= 0 && a->total <= INT32_MAX && a->heads >= 0 && a->heads_k >= 0 && a->heads + a->heads_k >= 1 && a->heads <= 65535 && a->heads_k <= 65535,
                "rotary: numbers of tokens and heads must be positive and below 2^31 and 65536");
  FMOBA_REQUIRE(a->head_dim >= 8 && a->head_dim <= 256 && a->head_dim % 8 == 0, "head_size must be a multiple of 8 up to 256");
  FMOBA_REQUIRE(a->rotary_dim >= 8 && a->rotary_dim <= a->head_dim && a->rotary_dim % 8 == 0, "rotary_dim must be a multiple of 8 up to the head size");
  FMOBA_REQUIRE(a->axes >= 1 && a->axes <= FMOBA_ROTARY_AXES, "rotary: 1 to %d axes", FMOBA_ROTARY_AXES);
  int64_t pairs = 0;
  for (int i = 0; i < a->axes; ++i) {
    FMOBA_REQUIRE(a->sections[i] >= 0, "rotary: a section is negative");
    pairs += a->sections[i];
  }
  FMOBA_REQUIRE(pairs == a->rotary_dim / 2, "rotary: the sections have %lld pairs, rotary_dim has %d", (long long)pairs, a->rotary_dim / 2);
  FMOBA_REQUIRE(a->log2_base >= 0.0 && a->log2_base <= 1024.0, "rotary: base must be a number from 1 on");
  if (a->total == 0) return 0;
  FMOBA_REQUIRE(ceil_div64(a->total, rotary_tokens(*a)) * kRotaryThreads <= UINT32_MAX, "rotary: too many tokens for the launch grid");
  FMOBA_REQUIRE(a->positions && (a->heads == 0 || (a->q && a->q_out)) && (a->heads_k == 0 || (a->k && (a->k_out || !k_out))), "rotary: null pointer");
  FMOBA_REQUIRE(a->q_row_stride % 8 == 0 && a->q_head_stride % 8 == 0 && a->k_row_stride % 8 == 0 && a->k_head_stride % 8 == 0 && a->qo_row_stride % 8 == 0 &&
                    a->qo_head_stride % 8 == 0 && a->ko_row_stride % 8 == 0 && a->ko_head_stride % 8 == 0,
                "rotary: strides must be multiples of 8 elements");
  FMOBA_REQUIRE((((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->q_out | (uintptr_t)a->k_out) % 16) == 0, "rotary: q and k must be 16-byte aligned");
  return 0;
}

}  // namespace fmoba

extern "C" int fmoba_rotary(const fmoba_rotary_args *a, void *stream) {
  using namespace fmoba;
  if (int rc = check_rotary_args(a, true)) return rc;
  if (a->total == 0) return 0;
  if (a->dtype == FMOBA_DTYPE_BF16)
    launch_rotary<bf16_t>(*a, (hipStream_t)stream);
  else
    launch_rotary<f16_t>(*a, (hipStream_t)stream);
  FMOBA_LAUNCH_CHECK("rotary_kernel");
  return 0;
}
