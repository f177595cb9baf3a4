// What the forms of the attention over the paged 8-bit cache share (kv_attn.hip, kv_attn_columns.hip): the call, where a row lies, the order of scores.
#pragma once

#include "kv_cache.h"

namespace fmoba {

struct CacheAttn {
  fmoba_cache_attn_args a;
  uint32_t *key_hi, *key_lo;  // [(row, head)][page of the table]: order keys of the scores, 0: no candidate
  int32_t cols;               // pages of a sequence, at most
};

// position of a row, the sequence and its table
struct RowPlace {
  int b, row, pos;  // pos < 0: the row sees nothing
};
__device__ __forceinline__ RowPlace find_row(const fmoba_cache_attn_args &a, int t) {
  const int lane = threadIdx.x & 63;
  int b = 0;  // sequences that end at or before the row (empty ones included) come first
  for (int b0 = 0; b0 < a.batch; b0 += 64) b += __popcll(__ballot(b0 + lane < a.batch && a.cu_seqlens_q[b0 + lane + 1] <= t));
  RowPlace r{b, 0, -1};
  if (b >= a.batch) return r;
  const int q0 = a.cu_seqlens_q[b];
  r.row = t - q0;
  r.pos = q0 < 0 || r.row < 0 || r.row >= a.max_seqlen_q ? -1 : a.seqlens_k[b] - (a.cu_seqlens_q[b + 1] - t);
  return r;
}

// the same by a single lane (rows of a wave that differ)
__device__ __forceinline__ RowPlace find_row_lane(const fmoba_cache_attn_args &a, int t) {
  int lo = 0, hi = a.batch;  // the first sequence that ends behind the row
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_seqlens_q[mid + 1] <= t)
      lo = mid + 1;
    else
      hi = mid;
  }
  RowPlace r{lo, 0, -1};
  if (lo >= a.batch) return r;
  const int q0 = a.cu_seqlens_q[lo];
  r.row = t - q0;
  r.pos = q0 < 0 || r.row < 0 || r.row >= a.max_seqlen_q ? -1 : a.seqlens_k[lo] - (a.cu_seqlens_q[lo + 1] - t);
  return r;
}

// order of a score among the candidates of a row: larger is better, 0 is none
__device__ __forceinline__ uint64_t score_key(double s) {
  if (!(s > -INFINITY)) return 0ull;
  const uint64_t u = (uint64_t)__double_as_longlong(s + 0.0);  // (-0 is 0)
  return (u >> 63) ? ~u : u | (1ull << 63);
}

// ------------------------------------------------------------------------------------
// The best `want` of n candidates, by one wave: take(candidate, upper half of its key, place) for each, in any order, by the lane that holds it; returns how many.  hi(i) and lo(i)
// are the halves of candidate i's key, id(i) decides between equal keys (the larger).  The upper halves decide but for ties: the largest cut that leaves
// `want` of them at or above it is found bit by bit, a count is a ballot; of those that share the cut the lower halves decide.
// The upper halves are in registers for up to 64 NJ candidates, NJ = 0: asked for each time.
// ------------------------------------------------------------------------------------
template <int NJ, typename Hi, typename Lo, typename Id, typename Take>
__device__ __forceinline__ int pick_best(int n, int want, int lane, Hi hi, Lo lo, Id id, Take take) {
  if (want <= 0 || n <= 0) return 0;
  const int places = NJ > 0 ? NJ : (n + 63) / 64;
  uint32_t reg[NJ > 0 ? NJ : 1];
  if constexpr (NJ > 0) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) reg[j] = j * 64 + lane < n ? hi(j * 64 + lane) : 0u;
  }
  auto each = [&](auto &&f) {  // f(candidate, its upper half), all lanes at once
    if constexpr (NJ > 0) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) f(j * 64 + lane, reg[j]);
    } else {
      for (int j = 0; j < places; ++j) f(j * 64 + lane, j * 64 + lane < n ? hi(j * 64 + lane) : 0u);
    }
  };
  auto count_ge = [&](uint32_t v) {
    int m = 0;
    each([&](int, uint32_t k) { m += __popcll(__ballot(k >= v)); });
    return m;
  };
  uint32_t cut = 1u;
  int n_cut = count_ge(1u);
  if (n_cut > want) {
    cut = 0u;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t trial = cut | (1u << bit);
      const int m = count_ge(trial);
      if (m >= want) cut = trial, n_cut = m;
      if (m == want) break;
    }
  }
  const bool tie = n_cut > want;
  int total = 0;
  each([&](int c, uint32_t k) {
    const bool in = tie ? k > cut : k >= cut;
    const unsigned long long m = __ballot(in);
    if (in) take(c, k, total + __popcll(m & ((1ull << lane) - 1ull)));
    total += __popcll(m);
  });
  uint64_t below = ~0ull;
  for (; tie && total < want; ++total) {  // the best of those that share the cut, one by one
    uint64_t best = 0ull;  // lower half + 1 | id: of 64 bits the upper 33 and the lower 31 (ids are pages of a table)
    int mine = -1;
    each([&](int c, uint32_t k) {
      if (k != cut) return;
      const uint64_t x = ((uint64_t)lo(c) + 1) << 31 | (uint32_t)id(c);
      if (x < below && x > best) best = x, mine = c;
    });
    uint64_t top = best;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const uint64_t y = __shfl_xor(top, o, 64);
      top = y > top ? y : top;
    }
    if (mine >= 0 && best == top) take(mine, cut, total);  // (ids differ: one lane)
    below = top;
  }
  return total;
}

// the form for many rows
constexpr int kColumnCols = 32768;  // pages of a table, at most (a word of bits for each in LDS, and its number in a score)
size_t column_workspace_bytes(const fmoba_cache_attn_args &a, int cols);
bool column_grid_fits(const fmoba_cache_attn_args &a, int cols);
int run_cache_columns(const CacheAttn &c, hipStream_t s);

}  // namespace fmoba
