// Gated attention over the paged 8-bit cache.
//   score[row, page] = q . k_mean[page]     for the pages before the row's own, in 64 bits: two roundings of a score in 32 bits
//                                           would let the order of a sum decide which page a row reads
//   out = sum_j p_j v_j s_v[page of j] / sum_j p_j,   p_j = exp(scale s_k[page of j] (q . k_j) - m)
// The scale of a page is the same for all of its keys and multiplies a whole score or weight, never a feature.
#include "kv_cache.h"

#include <algorithm>

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

// order of a score among the candidates of a row: larger is better, 0 is none
__device__ __forceinline__ uint64_t score_key(double s) {
  if (!(s > -INFINITY)) return 0ull;
  const uint64_t u = (uint64_t)__double_as_longlong(s + 0.0);  // (-0 is 0)
  return (u >> 63) ? ~u : u | (1ull << 63);
}

// ------------------------------------------------------------------------------------
// Scores of kScoreRows (row, head of the group) pairs against 64 pages: four lanes share a page's mean, a quarter of the features each.  The pairs' queries
// lie in LDS as doubles.  Decode steps read every mean once: memory; many rows are bound by the 64-bit products.
// ------------------------------------------------------------------------------------
constexpr int kScoreRows = 8, kScorePages = 64;
template <typename T>
__global__ __launch_bounds__(256) void cache_scores_kernel(CacheAttn p) {
  extern __shared__ double sQ[];  // [kScoreRows][D]
  const fmoba_cache_attn_args &a = p.a;
  const int D = a.cache.head_dim, P = a.cache.page_size, G = a.heads / a.cache.heads_k, tid = threadIdx.x;
  const int b = blockIdx.z / a.cache.heads_k, hk = blockIdx.z - b * a.cache.heads_k;
  const int q0 = a.cu_seqlens_q[b], R = min(a.cu_seqlens_q[b + 1], a.total_q) - q0, pair0 = blockIdx.y * kScoreRows, c0 = blockIdx.x * kScorePages;
  const int npairs = min((int64_t)kScoreRows, (int64_t)R * G - pair0);
  if (q0 < 0 || npairs <= 0) return;
  const int last_pos = a.seqlens_k[b] - (a.cu_seqlens_q[b + 1] - q0) + (pair0 + npairs - 1) / G;  // pairs: row by row, a row's heads one after the other
  const int npages = last_pos < 0 ? 0 : min(last_pos / P, p.cols - 1);  // that any of the rows can select beside its own
  if (c0 >= npages) return;
  for (int i = tid; i < kScoreRows * D; i += 256) {
    const int r = i / D, e = i - r * D, pair = pair0 + min(r, npairs - 1);
    const int row = q0 + pair / G, h = hk * G + pair % G;
    sQ[i] = (double)elem_to_float<T>(reinterpret_cast<const uint16_t *>(a.q)[(int64_t)row * a.q_row_stride + (int64_t)h * a.q_head_stride + e]);
  }
  __syncthreads();
  const int c = c0 + (tid >> 2), part = tid & 3;
  const int page = c < npages ? a.block_table[(int64_t)b * a.table_stride + c] : -1;
  const bool there = page >= 0 && page < a.cache.num_pages;
  const uint16_t *mean = reinterpret_cast<const uint16_t *>(a.cache.k_mean) + ((int64_t)(there ? page : 0) * a.cache.heads_k + hk) * D;
  double acc[kScoreRows];
#pragma unroll
  for (int r = 0; r < kScoreRows; ++r) acc[r] = 0.0;
  for (int e = part * 8; e < D; e += 32) {
    float f[8];
    unpack8<T>(there ? ld_global16(mean + e) : zero_pack8(), f);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int r = 0; r < kScoreRows; ++r) acc[r] = fma((double)f[j], sQ[r * D + e + j], acc[r]);
  }
#pragma unroll
  for (int r = 0; r < kScoreRows; ++r) {
    double s = acc[r];
    s += __shfl_xor(s, 1, 64);
    s += __shfl_xor(s, 2, 64);
    if (part == 0 && c < npages && r < npairs) {
      const int pair = pair0 + r;
      const int64_t at = ((int64_t)(q0 + pair / G) * a.heads + hk * G + pair % G) * p.cols + c;
      const uint64_t key = there ? score_key(s) : 0ull;
      p.key_hi[at] = (uint32_t)(key >> 32);
      p.key_lo[at] = (uint32_t)key;
    }
  }
}

// ------------------------------------------------------------------------------------
// The best `want` of a row's nc candidates, by one wave, into `chosen` (any order); returns how many.  The upper halves of the keys decide but for ties: the
// largest cut that leaves `want` of them at or above it is found bit by bit, a count is a ballot; of those that share the cut the lower halves
// decide, then the later page.  `hi` in registers for up to 256 candidates, else in LDS or, from kPickLds on, where the scores are.
// ------------------------------------------------------------------------------------
constexpr int kPickLds = 4096;
template <int NJ>
__device__ __forceinline__ int pick_pages(const uint32_t *key_hi, const uint32_t *key_lo, int nc, int want, int lane, uint32_t *keys, int *chosen) {
  if (want <= 0 || nc <= 0) return 0;
  const int places = NJ > 0 ? NJ : (nc + 63) / 64;
  const bool in_lds = NJ == 0 && nc <= kPickLds;
  uint32_t reg[NJ > 0 ? NJ : 1];
  if constexpr (NJ > 0) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) reg[j] = j * 64 + lane < nc ? key_hi[j * 64 + lane] : 0u;
  } else if (in_lds) {
    for (int j = 0; j < places; ++j) keys[j * 64 + lane] = j * 64 + lane < nc ? key_hi[j * 64 + lane] : 0u;
  }
  auto each = [&](auto &&f) {  // f(candidate, its upper half), all lanes at once
    if constexpr (NJ > 0) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) f(j * 64 + lane, reg[j]);
    } else {
      for (int j = 0; j < places; ++j) {
        const int c = j * 64 + lane;
        f(c, in_lds ? keys[c] : c < nc ? key_hi[c] : 0u);  // (its own lane wrote it)
      }
    }
  };
  auto count_ge = [&](uint32_t v) {
    int n = 0;
    each([&](int, uint32_t k) { n += __popcll(__ballot(k >= v)); });
    return n;
  };
  const int all = count_ge(1u);
  uint32_t cut = 1u;
  int n_cut = all;
  if (all > want) {
    cut = 0u;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t trial = cut | (1u << bit);
      const int n = count_ge(trial);
      if (n >= want) cut = trial, n_cut = n;
      if (n == want) break;
    }
  }
  const bool tie = n_cut > want;
  int total = 0;
  each([&](int c, uint32_t k) {
    const unsigned long long m = __ballot(tie ? k > cut : k >= cut);
    if ((m >> lane) & 1ull) chosen[total + __popcll(m & ((1ull << lane) - 1ull))] = c;
    total += __popcll(m);
  });
  for (uint64_t below = ~0ull; tie && total < want; ++total) {  // the best of those that share the cut, one by one
    uint64_t best = 0ull;
    each([&](int c, uint32_t k) {
      if (k != cut) return;
      const uint64_t x = (uint64_t)key_lo[c] << 32 | (uint32_t)(c + 1);
      if (x < below && x > best) best = x;
    });
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const uint64_t y = __shfl_xor(best, o, 64);
      best = y > best ? y : best;
    }
    if (lane == 0) chosen[total] = (int)(uint32_t)best - 1;
    below = best;
  }
  return total;
}

// ------------------------------------------------------------------------------------
// One workgroup per (row, head): eight waves take the units of 64 keys of its pages side by side and merge in LDS.  16 bytes (features) a lane and load,
// LPR lanes a key.
// ------------------------------------------------------------------------------------
constexpr int kRowWaves = 8, kUnitKeys = 64;
constexpr int kUnitsWithWeight = 1024;  // units of a row, at most: 64 pages of 1024 keys

template <int LPR>
__device__ __forceinline__ float sum_key_lanes(float x) {  // over the LPR consecutive lanes of a key
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}

template <typename T, typename H, int HD, bool WEIGHT>
__global__ __launch_bounds__(64 * kRowWaves, 2) void cache_attn_row_kernel(CacheAttn p) {
  constexpr int LPR = HD / 16, KPI = 64 / LPR, NIN = kUnitKeys / KPI;
  const fmoba_cache_attn_args &a = p.a;
  __shared__ int sChosen[64], sCount;
  __shared__ uint32_t sKeys[kPickLds];
  __shared__ float sAcc[kRowWaves][HD], sM[kRowWaves], sL[kRowWaves];
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
  if (wave == 0) {
    int n = 0;
    if (at.pos >= 0) {
      const int64_t keys = ((int64_t)t * a.heads + h) * p.cols;
      const int nc = min(own, p.cols - 1);  // (a sequence longer than max_seqlen_k: what lies behind is not looked at)
      n = nc <= 256 ? pick_pages<4>(p.key_hi + keys, p.key_lo + keys, nc, a.topk - 1, lane, sKeys, sChosen)
                    : pick_pages<0>(p.key_hi + keys, p.key_lo + keys, nc, a.topk - 1, lane, sKeys, sChosen);
      const int page = own < p.cols ? table[own] : -1;
      if (page >= 0 && page < a.cache.num_pages) {
        if (lane == 0) sChosen[n] = own;
        ++n;
      }
    }
    if (lane == 0) sCount = n;
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
  const int upc = P / kUnitKeys, nunit = sCount * upc;
  const float scale_log2 = a.softmax_scale * 1.4426950408889634f;
  float m = -INFINITY, l = 0.f, acc[16];  // l and acc: over this lane's keys (every KPI-th)
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = 0.f;
  for (int u = wave; u < nunit; u += kRowWaves) {
    const int c = sChosen[u / upc], in_page = (u % upc) * kUnitKeys, key0 = c * P + in_page;
    const int64_t page = table[c];
    if (key0 >= kend || page < 0 || page >= a.cache.num_pages) {  // (only pages of the cache are chosen, unless another stream changes the table meanwhile)
      if (WEIGHT && lane == 0) sUnitM[u] = -INFINITY, sUnitL[u] = 0.f;
      continue;
    }
    const uint8_t *kg = reinterpret_cast<const uint8_t *>(a.cache.k) + page * a.cache.k_page_stride + (int64_t)hk * a.cache.k_head_stride + ec;
    const uint8_t *vg = reinterpret_cast<const uint8_t *>(a.cache.v) + page * a.cache.v_page_stride + (int64_t)hk * a.cache.v_head_stride + ec;
    const float ks = a.cache.k_scale[page * a.cache.heads_k + hk] * scale_log2, vs = a.cache.v_scale[page * a.cache.heads_k + hk];
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
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1) mu = fmaxf(mu, __shfl_xor(mu, o, 64));
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
#pragma unroll
      for (int o = LPR; o < 64; o <<= 1) lu += __shfl_xor(lu, o, 64);
      if (lane == 0) sUnitM[u] = mref, sUnitL[u] = lu;
    }
  }
#pragma unroll
  for (int o = LPR; o < 64; o <<= 1) {
    l += __shfl_xor(l, o, 64);
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] += __shfl_xor(acc[j], o, 64);
  }
  if (lane < LPR) {
#pragma unroll
    for (int j = 0; j < 16; ++j) sAcc[wave][e + j] = acc[j];
  }
  if (lane == 0) sM[wave] = m, sL[wave] = l;
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) M = fmaxf(M, sM[w]);
  const float Mref = M == -INFINITY ? 0.f : M;
  float L = 0.f, o = 0.f;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    const float f = __builtin_amdgcn_exp2f(sM[w] - Mref);
    L = fmaf(f, sL[w], L);
    if (tid < HD) o = fmaf(f, sAcc[w][tid], o);
  }
  const bool empty = L == 0.f;  // no key (a NaN among the scores stays one)
  if (tid < D) out[tid] = float_to_elem_bits<T>(empty ? 0.f : o / L);
  if (tid == 0) a.softmax_lse[(int64_t)h * a.total_q + t] = empty ? INFINITY : (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f;
  if constexpr (WEIGHT) {
    for (int u = tid; u < nunit; u += 64 * kRowWaves) {
      const float part = __builtin_amdgcn_exp2f(sUnitM[u] - Mref) * sUnitL[u] / L;  // (a unit past the row: 0)
      if (part > 0.f) atomicAdd(reinterpret_cast<unsigned long long *>(a.cache.weight) + (int64_t)table[sChosen[u / upc]] * a.cache.heads_k + hk, (unsigned long long)rintf(part * 4294967296.f));
    }
  }
}

template <typename T, typename H, bool WEIGHT>
static void launch_rows(const CacheAttn &p, hipStream_t s) {
  const dim3 grid((uint32_t)p.a.total_q * p.a.heads), block(64 * kRowWaves);
  if (p.a.cache.head_dim <= 64)
    hipLaunchKernelGGL((cache_attn_row_kernel<T, H, 64, WEIGHT>), grid, block, 0, s, p);
  else if (p.a.cache.head_dim <= 128)
    hipLaunchKernelGGL((cache_attn_row_kernel<T, H, 128, WEIGHT>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((cache_attn_row_kernel<T, H, 256, WEIGHT>), grid, block, 0, s, p);
}

template <typename T>
static int run_cache_attn(const CacheAttn &p, hipStream_t s) {
  const fmoba_cache_attn_args &a = p.a;
  const int D = a.cache.head_dim;
  if (p.cols > 1 && a.topk > 1) {
    const int64_t pairs = (int64_t)a.max_seqlen_q * (a.heads / a.cache.heads_k);
    const dim3 grid(ceil_div(p.cols - 1, kScorePages), (uint32_t)ceil_div64(pairs, kScoreRows), (uint32_t)a.batch * a.cache.heads_k);
    FMOBA_REQUIRE(grid.y <= 65535 && (int64_t)a.batch * a.cache.heads_k <= 65535, "cache_attn: too many rows, or sequences times heads, for the launch grid");
    hipLaunchKernelGGL((cache_scores_kernel<T>), grid, dim3(256), (size_t)kScoreRows * D * 8, s, p);
    FMOBA_LAUNCH_CHECK("cache_scores_kernel");
  }
  if (a.cache.format == FMOBA_CACHE_E4M3)
    a.add_weight ? launch_rows<T, HeldE4M3, true>(p, s) : launch_rows<T, HeldE4M3, false>(p, s);
  else
    a.add_weight ? launch_rows<T, HeldInt8, true>(p, s) : launch_rows<T, HeldInt8, false>(p, s);
  FMOBA_LAUNCH_CHECK("cache_attn_row_kernel");
  return 0;
}

static int cache_cols(const fmoba_cache_attn_args &a) { return std::min(ceil_div(a.max_seqlen_k, a.cache.page_size), a.max_pages); }

}  // namespace fmoba

extern "C" size_t fmoba_cache_attn_workspace_bytes(const fmoba_cache_attn_args *a) {
  using namespace fmoba;
  if (a == nullptr || a->total_q <= 0 || a->heads <= 0 || a->max_seqlen_k <= 0 || a->max_pages <= 0 || a->cache.page_size <= 0) return 0;
  return (size_t)a->total_q * a->heads * cache_cols(*a) * 8;
}

extern "C" int fmoba_cache_attn(const fmoba_cache_attn_args *a, void *stream) {
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
  CacheAttn p{};
  p.a = *a;
  p.cols = a->max_seqlen_k > 0 && a->max_pages > 0 && a->cache.num_pages > 0 ? cache_cols(*a) : 0;
  p.key_hi = reinterpret_cast<uint32_t *>(a->workspace);
  p.key_lo = p.key_hi + (size_t)a->total_q * a->heads * p.cols;
  return a->cache.dtype == FMOBA_DTYPE_BF16 ? run_cache_attn<bf16_t>(p, (hipStream_t)stream) : run_cache_attn<f16_t>(p, (hipStream_t)stream);
}
