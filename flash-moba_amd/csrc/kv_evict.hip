// Which pages of a sequence stay when it may keep `keep` of them: the first `sink`, the last `recent`, and of the others those with the most attention
// weight (64-bit integers, so that a sum over heads has no order, and of equals the first).  One workgroup per sequence.
//
// Bound by latency: 8 heads_k bytes per page are gathered once; the cut is found byte by byte from the highest one that any of them has set, with a histogram in
// LDS, and it ends as soon as what is left of a byte's bin is taken as a whole.  The pages kept and the pages let go are written in order by two running counts.
#include "fmoba_common.h"

namespace fmoba {

constexpr int kEvictThreads = 1024;
constexpr int kEvictPages = 8192;  // pages of a sequence whose weights are kept in LDS (64 KB); beyond, in the workspace

// number of set flags among threads before this one, and of the workgroup in `total`; two barriers
__device__ __forceinline__ int block_rank(bool flag, int *counts, int &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned long long m = __ballot(flag);
  __syncthreads();
  if (lane == 0) counts[wave] = __popcll(m);
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kEvictThreads / 64; ++w) {
    before += w < wave ? counts[w] : 0;
    total += counts[w];
  }
  return before + __popcll(m & ((1ull << lane) - 1ull));
}

__global__ __launch_bounds__(kEvictThreads) void cache_evict_kernel(fmoba_cache_evict_args a) {
  __shared__ uint64_t sKeys[kEvictPages];
  __shared__ int sHist[256], sCounts[kEvictThreads / 64];
  __shared__ uint64_t sCut;
  __shared__ unsigned long long sTop;
  __shared__ int sLeft, sDone;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int len = max(a.seqlens_k[b], 0);
  const int n = min((int)(((int64_t)len + a.page_size - 1) / a.page_size), a.max_pages);
  const int32_t *table = a.block_table + (int64_t)b * a.table_stride;
  int32_t *kept_out = a.new_table + (int64_t)b * a.max_pages, *freed_out = a.freed + (int64_t)b * a.max_pages;
  const int first = min(a.sink, n), last = max(n - a.recent, first);  // pages [first, last) may go
  const int choose = n > a.keep ? a.keep - first - (n - last) : last - first;  // of which so many stay (keep >= sink + recent)
  if (choose >= last - first) {
    for (int i = tid; i < a.max_pages; i += kEvictThreads) {
      kept_out[i] = i < n ? table[i] : -1;
      freed_out[i] = -1;
    }
    if (tid == 0) a.new_seqlens[b] = a.seqlens_k[b], a.num_freed[b] = 0;
    return;
  }
  uint64_t *keys = n <= kEvictPages ? sKeys : reinterpret_cast<uint64_t *>(a.workspace) + (int64_t)b * a.max_pages;
  if (tid == 0) sTop = 0ull, sDone = 0, sCut = 0ull, sLeft = choose;
  __syncthreads();
  unsigned long long any = 0ull;
  for (int i = first + tid; i < last; i += kEvictThreads) {
    const int page = table[i];
    int64_t w = 0;
    if (page >= 0 && page < a.num_pages)
      for (int h = 0; h < a.heads_k; ++h) w += a.weight[(int64_t)page * a.heads_k + h];
    const uint64_t key = (uint64_t)(w > 0 ? w : 0);  // (weights are not negative)
    keys[i] = key;
    any |= key;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) any |= __shfl_xor(any, o, 64);
  if ((tid & 63) == 0) atomicOr(&sTop, any);
  __syncthreads();
  // ---- the cut: keys above it stay, and sLeft of those equal to it under `mask` ----
  const int bits = 64 - __clzll((long long)sTop);  // (0 if no page has any weight)
  uint64_t mask = 0ull;
  for (int shift = (bits + 7) / 8 * 8 - 8; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kEvictThreads) sHist[i] = 0;
    __syncthreads();
    const uint64_t cut = sCut;
    for (int i = first + tid; i < last; i += kEvictThreads) {
      const uint64_t key = keys[i];
      if ((key & mask) == cut) atomicAdd(&sHist[(key >> shift) & 255], 1);
    }
    __syncthreads();
    mask |= 255ull << shift;
    if (tid < 64) {  // bins from the top, four per lane
      int c[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = sHist[255 - (tid * 4 + j)], sum += c[j];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(upto, o, 64);
        upto += tid >= o ? up : 0;
      }
      int above = upto - sum;
      const int left = sLeft;
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (above < left && above + c[j] >= left) {  // (one lane and bin: left >= 1, the bins hold more than that)
          sCut = cut | (uint64_t)(255 - (tid * 4 + j)) << shift;
          sLeft = left - above;
          sDone = above + c[j] == left;
        }
        above += c[j];
      }
    }
    __syncthreads();
    if (choose == 0 || sDone) break;
  }
  const uint64_t cut = sCut;
  const int equal = sLeft;
  // ---- both lists in order ----
  int nkept = 0, ngone = 0, nequal = 0;
  for (int i0 = 0; i0 < n; i0 += kEvictThreads) {
    const int i = i0 + tid;
    const bool there = i < n, may_go = there && i >= first && i < last;
    const uint64_t key = may_go ? keys[i] & mask : 0ull;
    const bool eq = may_go && choose > 0 && key == cut;
    int total;
    const int eq_rank = nequal + block_rank(eq, sCounts, total);
    nequal += total;
    const bool keep = there && (!may_go || (choose > 0 && (key > cut || (eq && eq_rank < equal))));
    const int at = nkept + block_rank(keep, sCounts, total);
    const int kept_now = total;
    const int gone_at = ngone + (i - i0) - (at - nkept);
    if (there) {
      if (keep)
        kept_out[at] = table[i];
      else
        freed_out[gone_at] = table[i];
    }
    ngone += min(kEvictThreads, n - i0) - kept_now;
    nkept += kept_now;
  }
  for (int i = tid; i < a.max_pages; i += kEvictThreads) {
    if (i >= nkept) kept_out[i] = -1;
    if (i >= ngone) freed_out[i] = -1;
  }
  if (tid == 0) {
    a.new_seqlens[b] = a.seqlens_k[b] - ngone * a.page_size;
    a.num_freed[b] = ngone;
  }
}

}  // namespace fmoba

extern "C" size_t fmoba_cache_evict_workspace_bytes(int32_t batch, int32_t max_pages) {
  return batch > 0 && max_pages > fmoba::kEvictPages ? (size_t)batch * (size_t)max_pages * 8 : 0;
}

extern "C" int fmoba_cache_evict(const fmoba_cache_evict_args *a, void *stream) {
  using namespace fmoba;
  FMOBA_REQUIRE(a != nullptr, "cache_evict: null args");
  FMOBA_REQUIRE(a->batch >= 1 && a->max_pages >= 0 && a->num_pages >= 0 && a->heads_k >= 1, "cache_evict: sizes must not be negative, batch and heads positive");
  FMOBA_REQUIRE(a->page_size >= 1, "cache_evict: page_size must be positive");
  FMOBA_REQUIRE(a->sink >= 0 && a->recent >= 1, "cache_evict: sink pages must not be negative, and the page that is being filled stays (recent pages at least 1)");
  FMOBA_REQUIRE((int64_t)a->keep >= (int64_t)a->sink + a->recent, "cache_evict: fewer pages to keep than sink and recent pages");
  FMOBA_REQUIRE(a->seqlens_k && a->new_seqlens && a->num_freed && (a->max_pages == 0 || (a->block_table && a->new_table && a->freed)), "cache_evict: null pointer");
  FMOBA_REQUIRE(a->weight || a->num_pages == 0, "cache_evict: null pointer");
  const size_t need = fmoba_cache_evict_workspace_bytes(a->batch, a->max_pages);
  FMOBA_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need && (uintptr_t)a->workspace % 8 == 0), "cache_evict: workspace too small (%zu < %zu)", a->workspace_bytes, need);
  hipLaunchKernelGGL(cache_evict_kernel, dim3(a->batch), dim3(kEvictThreads), 0, (hipStream_t)stream, *a);
  FMOBA_LAUNCH_CHECK("cache_evict_kernel");
  return 0;
}
