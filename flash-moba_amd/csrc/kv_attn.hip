// Gated attention over the paged 8-bit cache.
//   score[row, page] = q . k_mean[page]     for the pages before the row's own, in 64 bits: two roundings of a score in 32 bits
//                                           would let the order of a sum decide which page a row reads
//   out = sum_j p_j v_j s_v[page of j] / sum_j p_j,   p_j = exp(scale s_k[page of j] (q . k_j) - m)
// The scale of a page is the same for all of its keys and multiplies a whole score or weight, never a feature.
#include "kv_attn.h"

#include <algorithm>

namespace fmoba {

// ------------------------------------------------------------------------------------
// Scores of up to eight (row, head of the group) pairs against 64 pages: four lanes share a page's mean, a quarter of the features each.  The pairs' queries
// lie in LDS as doubles.  A decode step reads every mean once and is bound by latency: the lengths, then the queries and the table, then the means, each once
// and all of a lane's loads together.  Many rows are bound by the 64-bit products.
// ------------------------------------------------------------------------------------
constexpr int kScorePages = 64, kScorePairs = 8;
template <typename T, int HD>
__global__ __launch_bounds__(256) void cache_scores_kernel(CacheAttn p) {
  __shared__ double sQ[kScorePairs * HD];
  const fmoba_cache_attn_args &a = p.a;
  const int D = a.cache.head_dim, P = a.cache.page_size, G = a.heads / a.cache.heads_k, tid = threadIdx.x;
  const int b = blockIdx.z / a.cache.heads_k, hk = blockIdx.z - b * a.cache.heads_k;
  const int c = blockIdx.x * kScorePages + (tid >> 2), part = tid & 3;
  const int page = c < p.cols - 1 ? a.block_table[(int64_t)b * a.table_stride + c] : -1;
  const int q0 = a.cu_seqlens_q[b], q1 = a.cu_seqlens_q[b + 1], len = a.seqlens_k[b];
  const int R = min(q1, a.total_q) - q0, pair0 = blockIdx.y * kScorePairs;
  const int npairs = (int)min((int64_t)kScorePairs, (int64_t)R * G - pair0);
  if (q0 < 0 || npairs <= 0) return;
  const int last_pos = len - (q1 - q0) + (pair0 + npairs - 1) / G;  // pairs: row by row, a row's heads one after the other
  const int npages = last_pos < 0 ? 0 : min(last_pos / P, p.cols - 1);  // that any of the rows can select beside its own
  if ((int)blockIdx.x * kScorePages >= npages) return;
  const bool there = c < npages && page >= 0 && page < a.cache.num_pages;
  const uint16_t *mean = reinterpret_cast<const uint16_t *>(a.cache.k_mean) + ((int64_t)(there ? page : 0) * a.cache.heads_k + hk) * D;
  constexpr int NP = HD / 32;
  Pack8 x[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) x[i] = there && i * 32 + part * 8 < D ? ld_global16(mean + i * 32 + part * 8) : zero_pack8();
  for (int i = tid; i < npairs * HD; i += 256) {
    const int r = i / HD, e = i % HD, pair = pair0 + r;
    const int row = q0 + pair / G, h = hk * G + pair % G;
    sQ[i] = e < D ? (double)elem_to_float<T>(reinterpret_cast<const uint16_t *>(a.q)[(int64_t)row * a.q_row_stride + (int64_t)h * a.q_head_stride + e]) : 0.0;
  }
  __syncthreads();
  constexpr int RC = HD > 128 ? 1 : 2;  // pairs at a time: all of them read ahead do not fit the registers
#pragma unroll 1
  for (int r0 = 0; r0 < npairs; r0 += RC) {
    double s[RC];
#pragma unroll
    for (int r = 0; r < RC; ++r) s[r] = 0.0;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      float f[8];
      unpack8<T>(x[i], f);
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int r = 0; r < RC; ++r) s[r] = fma((double)f[j], sQ[min(r0 + r, npairs - 1) * HD + i * 32 + part * 8 + j], s[r]);
    }
#pragma unroll
    for (int r = 0; r < RC; ++r) {
      s[r] += __shfl_xor(s[r], 1, 64);
      s[r] += __shfl_xor(s[r], 2, 64);
      if (part == 0 && c < npages && r0 + r < npairs) {
        const int pair = pair0 + r0 + r;
        const int64_t at = ((int64_t)(q0 + pair / G) * a.heads + hk * G + pair % G) * p.cols + c;
        const uint64_t key = there ? score_key(s[r]) : 0ull;
        p.key_hi[at] = (uint32_t)(key >> 32);
        p.key_lo[at] = (uint32_t)key;
      }
    }
  }
}

// ------------------------------------------------------------------------------------
// One workgroup per (row, head): eight waves take the units of 64 keys of its pages side by side and merge in LDS.  16 bytes (features) a lane and load,
// LPR lanes a key.  Every key and value that a row reads is read once (from the L2 again where heads of a group choose alike): 16 rows of 16 sequences with 512 to 32768 tokens, 32
// over 8 heads of 128, 8 pages of 128: 22.7 us, 106 MB at 4.7 TB/s.  With fewer rows than compute units it is a chain: scores, choice, pages, merge (four rows of up to 262144
// tokens, 16 heads of 64: 30 us on 64 units; sixteen waves instead of eight took 28.5 there and 14.5 instead of 12.7 for four of 8192, 32 heads).
// ------------------------------------------------------------------------------------
constexpr int kUnitKeys = 64;
constexpr int kRowWaves = 8;  // of a workgroup: two of them share a compute unit
static_assert(kRowWaves == 8, "64 groups of candidates: eight threads each");
// Candidates of a row that its workgroup scores itself, at most.  Rows score for themselves what the heads of a group could share, from the L2, and spare a launch
// that everything waits for: one row of each of 16 sequences, 32 over 8 heads, 1024 pages 33.5 instead of 44.0 us, of one 18.7 and 18.8; 2048 pages, 16 heads of 64, 16
// sequences 30.2 and 42.3, four 25.3 and 25.1, one 21.8 and 19.2.
constexpr int kOwnScores = 2048;
// Rows share pages where there are kColumnRowsLeast (row, head) pairs or more and a page is selected by kVisitsOwn of them on average, or by kVisits if the scores are a
// launch of their own; else the form for many rows takes longer, for its three launches and for pages that few rows visit.  Visits of a page, us of the form for many rows and of this
// one, heads of 128, 8 pages of 128 a row: 16 sequences of 2048 tokens, 16 heads, 4 rows each 2: 93, 34; 8 rows 4: 94, 63; 16 rows 8: 97, 119; of 32768 tokens, 32 over 8
// heads, 32 rows 4: 624, 525; of 8192 8 rows 4: 172, 124; 16 rows 8: 180, 236; a sequence of 100000 tokens 64 rows 2.6: 145, 104; 128 rows 5.2: 160, 193; 256 rows 10: 169, 367;
// with its own launch for the scores, four sequences of 300000, 32 rows 0.4: 1072, 391; 128 rows 1.7: 1436, 1466.  One row of each of 64
// sequences, 32 heads over one, of 2048 tokens 16: 41, 64; of 8192 4: 97, 77.  Few pairs, 1536: 16 over 2 heads, 384 visits: 51, 48; 1024, 32 over 8 heads, 64: 29, 34; 2048, 16 heads, 64: 30, 63.
// (Averages over the sequences of a call: one with a few long parts of prompts and many single rows takes the row form.)
constexpr int kColumnRowsLeast = 2048, kVisitsOwn = 5, kVisits = 2;
constexpr int kPickAlone = 256;  // candidates that one wave chooses from (by the groups' cut 128 of them took 2 us longer)
constexpr int kPickList = 512;  // candidates that are left when the cut of the groups is known, beyond which all are looked through again
constexpr int kUnitsWithWeight = 1024;  // units of a row, at most: 64 pages of 1024 keys

// the largest of 8 consecutive lanes, in all of them
__device__ __forceinline__ uint32_t max_lanes8(uint32_t x) {
#if defined(__HIP_DEVICE_COMPILE__)
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, true));   // quad_perm 1 0 3 2
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, true));   // quad_perm 2 3 0 1
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, true));  // row_half_mirror
#endif
  return x;
}

// lane permutations on the vector unit: CTRL of update_dpp
template <int CTRL>
__device__ __forceinline__ float dpp_f(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
#else
  return x;
#endif
}
// sum over the LPR (4, 8 or 16) consecutive lanes of a key, in all of them
template <int LPR>
__device__ __forceinline__ float sum_key_lanes(float x) {
  x += dpp_f<0xb1>(x);   // quad_perm 1 0 3 2
  x += dpp_f<0x4e>(x);   // quad_perm 2 3 0 1
  if constexpr (LPR >= 8) x += dpp_f<0x141>(x);   // row_half_mirror
  if constexpr (LPR >= 16) x += dpp_f<0x140>(x);  // row_mirror
  return x;
}
// sum and maximum over the lanes of equal features: every LPR-th
template <int LPR>
__device__ __forceinline__ float sum_keys(float x) {
  if constexpr (LPR == 4) x += dpp_f<0x124>(x);  // row_ror 4
  if constexpr (LPR <= 8) x += dpp_f<0x128>(x);  // row_ror 8
  return sum_rows4_f(x);
}
template <int LPR>
__device__ __forceinline__ float max_keys(float x) {
  if constexpr (LPR == 4) x = fmaxf(x, dpp_f<0x124>(x));
  if constexpr (LPR <= 8) x = fmaxf(x, dpp_f<0x128>(x));
  return max_rows4_f(x);
}

// The scores of one row against its nc candidates by a whole workgroup: four lanes a page, 16 pages a wave, two of them in flight.
template <typename T, int HD>
__device__ __forceinline__ void score_row(const fmoba_cache_attn_args &a, int t, int h, int hk, int nc, const int32_t *table, uint32_t *key_hi, uint32_t *key_lo) {
  constexpr int NP = HD / 32, TURN = kRowWaves * 16;
  const int D = a.cache.head_dim, tid = threadIdx.x, part = tid & 3;
  const uint16_t *src = reinterpret_cast<const uint16_t *>(a.q) + (int64_t)t * a.q_row_stride + (int64_t)h * a.q_head_stride + part * 8;
  Pack8 q[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) q[i] = i * 32 + part * 8 < D ? ld_global16(src + i * 32) : zero_pack8();
  int page[2], page_next[2];
  auto ask_pages = [&](int c0) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int c = c0 + u * TURN + (tid >> 2);
      page_next[u] = c < nc ? table[c] : -1;
    }
  };
  ask_pages(0);
  for (int c0 = 0; c0 < nc; c0 += 2 * TURN) {
    Pack8 x[2][NP];
    page[0] = page_next[0], page[1] = page_next[1];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bool there = page[u] >= 0 && page[u] < a.cache.num_pages;
      const uint16_t *mean = reinterpret_cast<const uint16_t *>(a.cache.k_mean) + ((int64_t)(there ? page[u] : 0) * a.cache.heads_k + hk) * D + part * 8;
#pragma unroll
      for (int i = 0; i < NP; ++i) x[u][i] = there && i * 32 + part * 8 < D ? ld_global16(mean + i * 32) : zero_pack8();
    }
    ask_pages(c0 + 2 * TURN);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      double s = 0.0;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        float f[8], g[8];
        unpack8<T>(x[u][i], f);
        unpack8<T>(q[i], g);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fma((double)f[j], (double)g[j], s);
      }
      s += __shfl_xor(s, 1, 64);
      s += __shfl_xor(s, 2, 64);
      const int c = c0 + u * TURN + (tid >> 2);
      if (part == 0 && c < nc) {
        const uint64_t key = page[u] >= 0 && page[u] < a.cache.num_pages ? score_key(s) : 0ull;
        key_hi[c] = (uint32_t)(key >> 32);
        key_lo[c] = (uint32_t)key;
      }
    }
  }
}

// SCORES: the workgroup scores its row's candidates itself, as cache_scores_kernel does, into LDS.
template <typename T, typename H, int HD, bool WEIGHT, bool SCORES>
__global__ __launch_bounds__(64 * kRowWaves, HD > 128 ? 2 : 4) void cache_attn_row_kernel(CacheAttn p) {
  constexpr int LPR = HD / 16, KPI = 64 / LPR, NW = kRowWaves, NIN = kUnitKeys / KPI;
  const fmoba_cache_attn_args &a = p.a;
  __shared__ int sChosen[64], sCount, sPages[64];
  __shared__ float sScaleK[64], sScaleV[64];
  __shared__ uint32_t sTop[64], sCut, sKeyHi[SCORES ? kOwnScores : 1], sKeyLo[SCORES ? kOwnScores : 1];
  __shared__ int sPage[kPickList], sFound[NW];
  __shared__ float sAcc[NW][HD], sM[NW], sL[NW];
  __shared__ float sUnitM[WEIGHT ? kUnitsWithWeight : 1], sUnitL[WEIGHT ? kUnitsWithWeight : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t = blockIdx.x / a.heads, i = blockIdx.x - t * a.heads;
  const int h = a.heads % 8 == 0 ? (i & 7) * (a.heads >> 3) + (i >> 3) : i;  // heads of a group on one XCD
  const RowPlace at = find_row(a, t);
  uint16_t *out = reinterpret_cast<uint16_t *>(a.out) + (int64_t)t * a.o_row_stride + (int64_t)h * a.o_head_stride;
  const int D = a.cache.head_dim, P = a.cache.page_size;
  const int hk = h / (a.heads / a.cache.heads_k);
  const int own = at.pos >= 0 ? at.pos / P : 0, kend = at.pos + 1;
  const int32_t *table = a.block_table + (int64_t)(at.b < a.batch ? at.b : 0) * a.table_stride;
  // ---- the pages of the row ----
  const int64_t keys = ((int64_t)t * a.heads + h) * p.cols;
  const uint32_t *key_hi = SCORES ? sKeyHi : p.key_hi + keys, *key_lo = SCORES ? sKeyLo : p.key_lo + keys;
  const int nc = at.pos >= 0 ? min(own, p.cols - 1) : 0;  // (a sequence longer than max_seqlen_k: what lies behind is not looked at)
  const int want = a.topk - 1;
  if constexpr (SCORES) {
    if (want > 0 && nc > 0) {
      score_row<T, HD>(a, t, h, hk, nc, table, sKeyHi, sKeyLo);
      __syncthreads();
    }
  }
  int picked = 0;
  if (nc <= kPickAlone) {  // one wave, while the others ask for the query
    if (wave == 0)
      picked = pick_best<kPickAlone / 64>(nc, want, lane, [&](int c) { return key_hi[c]; }, [&](int c) { return key_lo[c]; }, [](int c) { return c; }, [&](int c, uint32_t, int at) { sChosen[at] = c; });
  } else if (want > 0) {
    // The candidates are 64 groups.  The want-th largest of the groups' largest keys is no larger than the want-th largest of all, so those at or above it are
    // enough to choose from: a few more than are wanted.
    uint32_t top = 0u;
    for (int c = tid; c < nc; c += 64 * NW) top = max(top, key_hi[c]);
    top = max_lanes8(top);
    if (lane % 8 == 0) sTop[tid / 8] = top;
    __syncthreads();
    if (wave == 0) {
      const uint32_t mine = sTop[lane];
      int at_least = 0;
      for (int i = 0; i < 64; ++i) at_least += (uint32_t)__builtin_amdgcn_readlane((int)mine, i) >= mine ? 1 : 0;
      uint32_t cut = max(at_least >= want ? mine : 1u, 1u);
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) cut = max(cut, (uint32_t)__shfl_xor((int)cut, o, 64));
      if (lane == 0) sCut = cut;
    }
    __syncthreads();
    const uint32_t cut = sCut;
    int found = 0;
    for (int c0 = wave * 64; c0 < nc; c0 += 64 * NW) found += __popcll(__ballot(c0 + lane < nc && key_hi[min(c0 + lane, nc - 1)] >= cut));
    if (lane == 0) sFound[wave] = found;
    __syncthreads();
    int place = 0, m = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      place += w < wave ? sFound[w] : 0;
      m += sFound[w];
    }
    for (int c0 = wave * 64; c0 < nc; c0 += 64 * NW) {
      const int c = c0 + lane;
      const bool in = c < nc && key_hi[min(c, nc - 1)] >= cut;
      const unsigned long long mask = __ballot(in);
      const int i = place + __popcll(mask & ((1ull << lane) - 1ull));
      if (in && i < kPickList) sPage[i] = c;
      place += __popcll(mask);
    }
    __syncthreads();
    if (wave == 0) {
      if (m <= 64) {  // one a lane: its rank among them
        const int c = lane < m ? sPage[lane] : 0;
        const uint32_t hi = lane < m ? key_hi[c] : 0u, lo = key_lo[c];
        int rank = 0;
        for (int i = 0; i < m; ++i) {
          const uint32_t h = (uint32_t)__builtin_amdgcn_readlane((int)hi, i), l = (uint32_t)__builtin_amdgcn_readlane((int)lo, i);
          const int o = __builtin_amdgcn_readlane(c, i);
          rank += h > hi || (h == hi && (l > lo || (l == lo && o > c))) ? 1 : 0;
        }
        const bool in = hi != 0u && rank < want;
        if (in) sChosen[rank] = c;
        picked = __popcll(__ballot(in));
      } else if (m <= kPickList) {
        picked = pick_best<kPickList / 64>(
            m, want, lane, [&](int i) { return key_hi[sPage[i]]; }, [&](int i) { return key_lo[sPage[i]]; }, [&](int i) { return sPage[i]; },
            [&](int i, uint32_t, int at) { sChosen[at] = sPage[i]; });
      } else {
        picked = pick_best<0>(
            nc, want, lane, [&](int c) { return key_hi[c]; }, [&](int c) { return key_lo[c]; }, [](int c) { return c; }, [&](int c, uint32_t, int at) { sChosen[at] = c; });
      }
    }
  }
  if (wave == 0) {
    const int page = at.pos >= 0 && own < p.cols ? table[own] : -1;
    const bool has_own = page >= 0 && page < a.cache.num_pages;
    if (lane == 0) {
      if (has_own) sChosen[picked] = own;
      sCount = picked + (has_own ? 1 : 0);
    }
  }
  const int e = (lane % LPR) * 16, ec = min(e, D - 16);
  float q[16];
  {
    const uint16_t *src = reinterpret_cast<const uint16_t *>(a.q) + (int64_t)t * a.q_row_stride + (int64_t)h * a.q_head_stride + ec;
    float lo[8], hi[8];
    unpack8<T>(ld_global16(src), lo);
    unpack8<T>(ld_global16(src + 8), hi);
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = e < D ? lo[j] : 0.f, q[8 + j] = e < D ? hi[j] : 0.f;
  }
  __syncthreads();
  if (tid < sCount) {  // where the pages lie, and their scales
    const int64_t page = table[sChosen[tid]];
    const bool there = page >= 0 && page < a.cache.num_pages;  // (it was when it was scored)
    sPages[tid] = there ? (int)page : -1;
    sScaleK[tid] = there ? a.cache.k_scale[page * a.cache.heads_k + hk] : 0.f;
    sScaleV[tid] = there ? a.cache.v_scale[page * a.cache.heads_k + hk] : 0.f;
  }
  __syncthreads();
  const int upc = P / kUnitKeys, nunit = sCount * upc;
  const float scale_log2 = a.softmax_scale * 1.4426950408889634f;
  float m = -INFINITY, l = 0.f, acc[16];  // l and acc: over this lane's keys (every KPI-th)
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = 0.f;
  for (int u = wave; u < nunit; u += NW) {
    const int n_page = u / upc, c = sChosen[n_page], in_page = (u - n_page * upc) * kUnitKeys;
    const int64_t page = sPages[n_page];
    if (c * P + in_page >= kend || page < 0) {
      if (WEIGHT && lane == 0) sUnitM[u] = -INFINITY, sUnitL[u] = 0.f;
      continue;
    }
    const uint8_t *kg = reinterpret_cast<const uint8_t *>(a.cache.k) + page * a.cache.k_page_stride + (int64_t)hk * a.cache.k_head_stride + ec;
    const uint8_t *vg = reinterpret_cast<const uint8_t *>(a.cache.v) + page * a.cache.v_page_stride + (int64_t)hk * a.cache.v_head_stride + ec;
    const float ks = sScaleK[n_page] * scale_log2, vs = sScaleV[n_page];
    const int r0 = in_page + lane / LPR, last = kend - 1 - c * P;  // keys behind the row's own are copies of it: what lies there may be anything
    Pack8 kx[NIN], vx[NIN];
#pragma unroll
    for (int n = 0; n < NIN; ++n) kx[n] = ld_global16(kg + (int64_t)min(r0 + n * KPI, last) * a.cache.k_token_stride);
#pragma unroll
    for (int n = 0; n < NIN; ++n) vx[n] = ld_global16(vg + (int64_t)min(r0 + n * KPI, last) * a.cache.v_token_stride);
    float s[NIN], mu = -INFINITY;
#pragma unroll
    for (int n = 0; n < NIN; ++n) {
      float d = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float f[4];
        H::unpack4(kx[n].w[w], f);
#pragma unroll
        for (int j = 0; j < 4; ++j) d = fmaf(q[4 * w + j], f[j], d);
      }
      d = sum_key_lanes<LPR>(d) * ks;
      s[n] = r0 + n * KPI <= last ? d : -INFINITY;
      mu = fmaxf(mu, s[n]);
    }
    mu = max_keys<LPR>(mu);
    const float mn = fmaxf(m, mu), mref = mn == -INFINITY ? 0.f : mn;
    const float resc = __builtin_amdgcn_exp2f(m - mref);
    m = mn;
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] *= resc;
    float lu = 0.f;
#pragma unroll
    for (int n = 0; n < NIN; ++n) {
      const float pn = __builtin_amdgcn_exp2f(s[n] - mref), pv = pn * vs;
      lu += pn;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float f[4];
        H::unpack4(vx[n].w[w], f);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[4 * w + j] = fmaf(pv, f[j], acc[4 * w + j]);
      }
    }
    l = fmaf(l, resc, lu);
    if constexpr (WEIGHT) {
      lu = sum_keys<LPR>(lu);
      if (lane == 0) sUnitM[u] = mref, sUnitL[u] = lu;
    }
  }
  l = sum_keys<LPR>(l);
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = sum_keys<LPR>(acc[j]);
  if (lane < LPR) {
#pragma unroll
    for (int j = 0; j < 16; ++j) sAcc[wave][e + j] = acc[j];
  }
  if (lane == 0) sM[wave] = m, sL[wave] = l;
  __syncthreads();
  if (wave * 64 >= max(HD, WEIGHT ? nunit : 0)) return;
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < NW; ++w) M = fmaxf(M, sM[w]);
  const float Mref = M == -INFINITY ? 0.f : M;
  float L = 0.f, o = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const float f = __builtin_amdgcn_exp2f(sM[w] - Mref);
    L = fmaf(f, sL[w], L);
    if (tid < HD) o = fmaf(f, sAcc[w][tid], o);
  }
  const bool empty = L == 0.f;  // no key (a NaN among the scores stays one)
  if (tid < D) out[tid] = float_to_elem_bits<T>(empty ? 0.f : o / L);
  if (tid == 0) a.softmax_lse[(int64_t)h * a.total_q + t] = empty ? INFINITY : (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f;
  if constexpr (WEIGHT) {
    for (int u = tid; u < nunit; u += 64 * NW) {
      const float part = __builtin_amdgcn_exp2f(sUnitM[u] - Mref) * sUnitL[u] / L;  // (a unit past the row: 0)
      if (part > 0.f) atomicAdd(reinterpret_cast<unsigned long long *>(a.cache.weight) + (int64_t)sPages[u / upc] * a.cache.heads_k + hk, (unsigned long long)rintf(part * 4294967296.f));
    }
  }
}

// pages of a sequence, at most
static int call_cols(const fmoba_cache_attn_args &a) {
  return a.max_seqlen_k > 0 && a.max_pages > 0 && a.cache.num_pages > 0 ? std::min(ceil_div(a.max_seqlen_k, a.cache.page_size), a.max_pages) : 0;
}
// whether the rows' workgroups score their pages themselves
static bool own_scores(int cols) { return cols - 1 <= kOwnScores; }
// whether the row form's launches fit their grids
static int64_t score_turns(const fmoba_cache_attn_args &a) { return ceil_div64((int64_t)std::min(a.max_seqlen_q, a.total_q) * (a.heads / a.cache.heads_k), kScorePairs); }
static bool has_scores(const fmoba_cache_attn_args &a, int cols) { return !own_scores(cols) && cols > 1 && a.topk > 1 && a.max_seqlen_q > 0; }
static bool rows_grid_fits(const fmoba_cache_attn_args &a) { return (int64_t)a.total_q * a.heads * 64 * kRowWaves <= UINT32_MAX; }
static bool scores_grid_fits(const fmoba_cache_attn_args &a, int cols) {
  return !has_scores(a, cols) || (score_turns(a) <= 65535 && (int64_t)a.batch * a.cache.heads_k <= 65535);
}
// Whether rows share the pages that they select (kv_attn_columns.hip), or every (row, head) reads its own; where the launch grid has no room for the one, the other.
static bool many_rows(const fmoba_cache_attn_args &a, int cols) {
  if (cols <= 0 || cols > kColumnCols || a.max_seqlen_q <= 0) return false;  // (no row of any sequence, rows that are padding: nothing to launch but what writes their outputs)
  const int64_t rows = (int64_t)a.total_q * a.heads;
  const bool shared = rows >= kColumnRowsLeast && rows * std::min(a.topk, cols) >= (own_scores(cols) ? kVisitsOwn : kVisits) * (int64_t)a.batch * a.cache.heads_k * cols;
  const bool alone_fits = rows_grid_fits(a) && scores_grid_fits(a, cols), shared_fits = column_grid_fits(a, cols);
  return shared ? shared_fits || !alone_fits : shared_fits && !alone_fits;
}

template <typename T, typename H, bool WEIGHT>
static void launch_rows(const CacheAttn &p, hipStream_t s) {
  const int D = p.a.cache.head_dim;
  const bool own = own_scores(p.cols);
  auto kern = D <= 64    ? (own ? cache_attn_row_kernel<T, H, 64, WEIGHT, true> : cache_attn_row_kernel<T, H, 64, WEIGHT, false>)
              : D <= 128 ? (own ? cache_attn_row_kernel<T, H, 128, WEIGHT, true> : cache_attn_row_kernel<T, H, 128, WEIGHT, false>)
                         : (own ? cache_attn_row_kernel<T, H, 256, WEIGHT, true> : cache_attn_row_kernel<T, H, 256, WEIGHT, false>);
  hipLaunchKernelGGL(kern, dim3((uint32_t)p.a.total_q * p.a.heads), dim3(64 * kRowWaves), 0, s, p);
}

template <typename T, int HD>
static void launch_scores(const CacheAttn &p, hipStream_t s) {
  const fmoba_cache_attn_args &a = p.a;
  const dim3 grid(ceil_div(p.cols - 1, kScorePages), (uint32_t)score_turns(a), (uint32_t)(a.batch * a.cache.heads_k));
  hipLaunchKernelGGL((cache_scores_kernel<T, HD>), grid, dim3(256), 0, s, p);
}

template <typename T>
static int run_cache_attn(const CacheAttn &p, hipStream_t s) {
  const fmoba_cache_attn_args &a = p.a;
  const int D = a.cache.head_dim;
  if (many_rows(a, p.cols)) return run_cache_columns(p, s);
  if (has_scores(a, p.cols)) {
    D <= 64 ? launch_scores<T, 64>(p, s) : D <= 128 ? launch_scores<T, 128>(p, s) : launch_scores<T, 256>(p, s);
    FMOBA_LAUNCH_CHECK("cache_scores_kernel");
  }
  if (a.cache.format == FMOBA_CACHE_E4M3)
    a.add_weight ? launch_rows<T, HeldE4M3, true>(p, s) : launch_rows<T, HeldE4M3, false>(p, s);
  else
    a.add_weight ? launch_rows<T, HeldInt8, true>(p, s) : launch_rows<T, HeldInt8, false>(p, s);
  FMOBA_LAUNCH_CHECK("cache_attn_row_kernel");
  return 0;
}

}  // namespace fmoba

extern "C" size_t fmoba_cache_attn_workspace_bytes(const fmoba_cache_attn_args *a) {
  using namespace fmoba;
  if (a == nullptr || a->total_q <= 0 || a->heads <= 0 || a->cache.heads_k <= 0 || a->cache.page_size <= 0) return 0;
  const int cols = call_cols(*a);
  if (cols == 0) return 0;
  if (many_rows(*a, cols)) return column_workspace_bytes(*a, cols);
  return own_scores(cols) ? 0 : (size_t)a->total_q * a->heads * cols * 8;
}

extern "C" int fmoba_cache_attn_check(const fmoba_cache_attn_args *a) {
  using namespace fmoba;
  FMOBA_REQUIRE(a != nullptr, "cache_attn: null args");
  FMOBA_CHECK_CACHE(a->cache);
  FMOBA_REQUIRE(a->batch >= 1 && a->batch <= 65535 && a->total_q >= 0 && a->max_seqlen_q >= 0 && a->max_seqlen_k >= 0 && a->max_pages >= 0, "cache_attn: sizes must not be negative, batch at most 65535");
  FMOBA_REQUIRE(a->heads >= 1 && a->heads <= 65535 && a->heads % a->cache.heads_k == 0, "#heads in key/value must divide #heads in query");
  FMOBA_REQUIRE(a->topk >= 1 && a->topk <= 64, "moba_topk must be in [1, 64]");
  FMOBA_REQUIRE((int64_t)a->total_q * a->heads <= INT32_MAX, "cache_attn: too many rows times heads for the launch grid");
  FMOBA_REQUIRE(!a->add_weight || a->cache.weight || a->cache.num_pages == 0, "cache_attn: the cache keeps no weight");
  if (a->total_q == 0) return 0;
  FMOBA_REQUIRE(a->q && a->out && a->softmax_lse && a->cu_seqlens_q && a->seqlens_k && (a->block_table || a->max_pages == 0), "cache_attn: null pointer");
  FMOBA_REQUIRE(a->q_row_stride % 8 == 0 && a->q_head_stride % 8 == 0 && a->o_row_stride % 8 == 0 && a->o_head_stride % 8 == 0, "cache_attn: strides must be multiples of 8 elements");
  FMOBA_REQUIRE((((uintptr_t)a->q | (uintptr_t)a->out) % 16) == 0, "cache_attn: q and out must be 16-byte aligned");
  const size_t need = fmoba_cache_attn_workspace_bytes(a);
  FMOBA_REQUIRE(a->workspace_bytes >= need && (a->workspace || need == 0) && (uintptr_t)a->workspace % 256 == 0, "cache_attn: workspace too small (%zu < %zu) or not 256-byte aligned", a->workspace_bytes, need);
  const int cols = call_cols(*a);
  if (many_rows(*a, cols)) {
    FMOBA_REQUIRE(column_grid_fits(*a, cols), "cache_attn: too many rows, or sequences times pages for the launch grid");
  } else {
    FMOBA_REQUIRE(rows_grid_fits(*a), "cache_attn: too many rows times heads for the launch grid");
    FMOBA_REQUIRE(scores_grid_fits(*a, cols), "cache_attn: too many rows, or sequences times heads, for the launch grid");
  }
  return 0;
}

extern "C" int fmoba_cache_attn(const fmoba_cache_attn_args *a, void *stream) {
  using namespace fmoba;
  if (int rc = fmoba_cache_attn_check(a)) return rc;
  if (a->total_q == 0) return 0;
  CacheAttn p{};
  p.a = *a;
  p.cols = call_cols(*a);
  p.key_hi = reinterpret_cast<uint32_t *>(a->workspace);
  p.key_lo = p.key_hi + (size_t)a->total_q * a->heads * p.cols;
  return a->cache.dtype == FMOBA_DTYPE_BF16 ? run_cache_attn<bf16_t>(p, (hipStream_t)stream) : run_cache_attn<f16_t>(p, (hipStream_t)stream);
}
