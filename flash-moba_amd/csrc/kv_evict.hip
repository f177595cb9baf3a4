// Which pages of a sequence stay when it may keep `keep` of them: the first `sink`, the last `recent`, and of the others those with the most attention
// weight (64-bit integers, so that a sum over heads has no order, and of equals the first).  One workgroup per sequence.
//
// Bound by latency: 8 heads_k bytes per page are gathered once.  One histogram of the weights in bins of a 32nd of a power of two says in which bin the cut
// lies; of the few weights there the last one to stay is the one of the right rank, or, if they are many, is found byte by byte.  The pages kept and the pages
// let go are written in order, every wave a stretch of the table.  16 tables of up to 768 pages 9.3 us, 64 of up to 4096 22.6 (34 with one workgroup for all of a table's
// sums, and byte by byte from the first bit on).
#include "fmoba_common.h"

namespace fmoba {

constexpr int kEvictThreads = 1024;
constexpr int kEvictPages = 8192;  // pages of a sequence whose weights are kept in LDS (64 KB); beyond, in the workspace
// Pages of a table that the sequence's workgroup sums itself; with more a launch before it does.  us alone and with the launch, 16 tables of 8 heads: 512 pages 9.1, 10.4; 1024 11.2, 11.7; 2048
// 16.4, 13.7; 4096 26.8, 18.5.
constexpr int kEvictAlone = 1024;

// Bin of a key: the place of its highest bit and the five bits behind it (a key below 32 is its own bin), so that the bins of weights of any size hold alike.
constexpr int kEvictBins = 32 * 60;
__device__ __forceinline__ int weight_bin(uint64_t key) {
  if (key < 32) return (int)key;
  const int e = 63 - __clzll((long long)key);  // 5 .. 62
  return (e - 4) * 32 + (int)((key >> (e - 5)) & 31);
}

// Sum of a page's weights over heads, by LP lanes next to each other (a power of two, up to the number of heads); kAtOnce of their pages on their way together.
// done(i, key) by one of the lanes, for pages i0, i0 + turn, .. below `last`.
constexpr int kAtOnce = 8;
template <int LP, typename PageAt, typename Done>
__device__ __forceinline__ void sum_weights(const fmoba_cache_evict_args &a, int i0, int turn, int last, int part, PageAt page_at, Done done) {
  for (; i0 < last; i0 += turn * kAtOnce) {
    int64_t w[kAtOnce];
    int page[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int i = i0 + u * turn;
      page[u] = i < last ? page_at(i) : -1;
      if (page[u] >= a.num_pages) page[u] = -1;
      w[u] = page[u] >= 0 ? a.weight[(int64_t)page[u] * a.heads_k + part] : 0;
    }
    for (int h = part + LP; h < a.heads_k; h += LP)
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) w[u] += page[u] >= 0 ? a.weight[(int64_t)page[u] * a.heads_k + h] : 0;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
#pragma unroll
      for (int o = 1; o < LP; o <<= 1) w[u] += __shfl_xor(w[u], o, 64);
      const int i = i0 + u * turn;
      if (part == 0 && i < last) done(i, (uint64_t)(w[u] > 0 ? w[u] : 0));  // (weights are not negative)
    }
  }
}

// The sums of long tables, by the whole device: one compute unit has too few lines on their way (4096 pages of 64 bytes each take it 25 us).
template <int LP>
__global__ __launch_bounds__(256) void cache_evict_sums_kernel(fmoba_cache_evict_args a) {
  constexpr int TURN = 256 / LP;
  const int b = blockIdx.y, len = max(a.seqlens_k[b], 0), i0 = blockIdx.x * TURN * kAtOnce;
  const int n = min((int)(((int64_t)len + a.page_size - 1) / a.page_size), a.max_pages);
  if (n <= a.keep || i0 >= n) return;
  const int32_t *table = a.block_table + (int64_t)b * a.table_stride;
  uint64_t *keys = reinterpret_cast<uint64_t *>(a.workspace) + (int64_t)b * a.max_pages;
  sum_weights<LP>(a, i0 + (int)threadIdx.x / LP, TURN, min(i0 + TURN * kAtOnce, n), threadIdx.x % LP, [&](int i) { return table[i]; }, [&](int i, uint64_t key) { keys[i] = key; });
}

// SUMS: the sums are in the workspace
template <int LP, bool SUMS>
__global__ __launch_bounds__(kEvictThreads) void cache_evict_kernel(fmoba_cache_evict_args a) {
  __shared__ uint64_t sKeys[kEvictPages];
  __shared__ int32_t sPages[kEvictPages];
  constexpr int WAVES = kEvictThreads / 64, LIST = 64;
  __shared__ int sHist[kEvictBins], sCounts[WAVES], sKept[WAVES], sList[LIST];
  __shared__ uint64_t sCut;
  __shared__ int sBin, sLeft, sInBin, sListed, sDone;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
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
  const bool near = n <= kEvictPages;
  for (int i = tid; i < kEvictBins; i += kEvictThreads) sHist[i] = 0;
  if (tid == 0) sListed = 0, sDone = 0;
  if (near)
    for (int i = tid; i < n; i += kEvictThreads) sPages[i] = table[i];
  __syncthreads();
  auto page_at = [&](int i) { return near ? sPages[i] : table[i]; };
  if constexpr (SUMS) {
    const uint64_t *sums = reinterpret_cast<const uint64_t *>(a.workspace) + (int64_t)b * a.max_pages;
    for (int i = first + tid; i < last; i += kEvictThreads) {
      const uint64_t key = sums[i];
      if (near) keys[i] = key;
      atomicAdd(&sHist[weight_bin(key)], 1);
    }
  } else {
    sum_weights<LP>(a, first + tid / LP, kEvictThreads / LP, last, tid % LP, page_at, [&](int i, uint64_t key) {
      keys[i] = key;
      atomicAdd(&sHist[weight_bin(key)], 1);
    });
  }
  __syncthreads();
  // ---- the bin of the cut: `choose` weights lie in it and above ----
  uint64_t mask = 0ull, cut = 0ull;  // keys that are above `cut` under `mask` stay, and `equal` of those that are the same
  int equal = choose;
  if (choose > 0) {
    int in_two = 0, bin = 0, c[2] = {0, 0};
    bin = kEvictBins - 1 - 2 * tid;  // bins from the highest down, two a thread
    if (bin > 0) c[0] = sHist[bin], c[1] = sHist[bin - 1], in_two = c[0] + c[1];
    int upto = in_two;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(upto, o, 64);
      upto += lane >= o ? up : 0;
    }
    if (lane == 63) sCounts[wave] = upto;
    __syncthreads();
    int above = upto - in_two;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) above += w < wave ? sCounts[w] : 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (above < choose && above + c[j] >= choose) sBin = bin - j, sLeft = choose - above, sInBin = c[j];  // (one thread)
      above += c[j];
    }
    __syncthreads();
    const int at = sBin, e = at / 32 + 4;
    int low = 0;  // bits below the bin's
    if (at < 32)
      mask = ~0ull, cut = (uint64_t)at;
    else
      low = e - 5, mask = ~0ull << low, cut = (uint64_t)(32 + at % 32) << low;
    equal = sLeft;
    if (low > 0 && equal < sInBin) {
      if (sInBin <= LIST) {  // the page of the right rank: by weight, of equals the first
        for (int i = first + tid; i < last; i += kEvictThreads)
          if ((keys[i] & mask) == cut) sList[atomicAdd(&sListed, 1)] = i;
        __syncthreads();
        if (wave == 0) {
          const int m = sInBin, i = lane < m ? sList[lane] : 0;
          const uint64_t key = lane < m ? keys[i] : 0ull;
          int rank = 0, larger = 0;
          for (int j = 0; j < m; ++j) {
            const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), j) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)key, j);
            larger += other > key ? 1 : 0;
            rank += other > key || (other == key && __builtin_amdgcn_readlane(i, j) < i) ? 1 : 0;
          }
          if (lane < m && rank == equal - 1) sCut = key, sLeft = equal - larger;  // (the last one to stay: one lane)
        }
        __syncthreads();
        mask = ~0ull, cut = sCut, equal = sLeft;
      } else {
        for (int shift = (low + 7) / 8 * 8 - 8; shift >= 0; shift -= 8) {  // byte by byte (the highest may have bits of the bin: they agree)
          for (int i = tid; i < 256; i += kEvictThreads) sHist[i] = 0;
          __syncthreads();
          for (int i = first + tid; i < last; i += kEvictThreads) {
            const uint64_t key = keys[i];
            if ((key & mask) == cut) atomicAdd(&sHist[(key >> shift) & 255], 1);
          }
          __syncthreads();
          if (wave == 0) {  // bins from the top, four per lane
            int d[4], sum = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = sHist[255 - (lane * 4 + j)], sum += d[j];
            int so_far = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
              const int up = __shfl_up(so_far, o, 64);
              so_far += lane >= o ? up : 0;
            }
            int over = so_far - sum;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (over < equal && over + d[j] >= equal) {  // (one lane and bin: the bins hold `equal` or more)
                sBin = 255 - (lane * 4 + j);
                sLeft = equal - over;
                sDone = over + d[j] == equal;
              }
              over += d[j];
            }
          }
          __syncthreads();
          mask |= 255ull << shift;
          cut = (cut & ~(255ull << shift)) | (uint64_t)sBin << shift;
          equal = sLeft;
          if (sDone) break;
        }
      }
    }
  }
  // ---- both lists in order: a stretch of the table a wave ----
  const int stretch = ((n + WAVES - 1) / WAVES + 63) / 64 * 64, s0 = wave * stretch, s1 = min(s0 + stretch, n);
  auto stays = [&](int i) { return i < n && (i < first || i >= last || (choose > 0 && (keys[i] & mask) > cut)); };
  auto at_cut = [&](int i) { return i >= first && i < last && choose > 0 && (keys[i] & mask) == cut; };
  int staying = 0, equals = 0;
  for (int i0 = s0; i0 < s1; i0 += 64) {
    staying += __popcll(__ballot(stays(i0 + lane)));
    equals += __popcll(__ballot(at_cut(i0 + lane)));
  }
  if (lane == 0) sKept[wave] = staying, sCounts[wave] = equals;
  __syncthreads();
  int nkept = 0, eq_before = 0, kept_all = 0, eq_all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w == wave) nkept = kept_all, eq_before = eq_all;
    kept_all += sKept[w] + min(max(equal - eq_all, 0), sCounts[w]);  // (the first `equal` of them)
    eq_all += sCounts[w];
  }
  for (int i0 = s0; i0 < s1; i0 += 64) {
    const int i = i0 + lane;
    const unsigned long long eq = __ballot(at_cut(i)), before = (1ull << lane) - 1ull;
    const bool keep = stays(i) || (((eq >> lane) & 1ull) && eq_before + __popcll(eq & before) < equal);
    const unsigned long long kept = __ballot(keep);
    const int to = nkept + __popcll(kept & before);
    if (i < n) {
      if (keep)
        kept_out[to] = page_at(i);
      else
        freed_out[i - to] = page_at(i);
    }
    nkept += __popcll(kept);
    eq_before += __popcll(eq);
  }
  const int gone = n - kept_all;
  for (int i = tid; i < a.max_pages; i += kEvictThreads) {
    if (i >= kept_all) kept_out[i] = -1;
    if (i >= gone) freed_out[i] = -1;
  }
  if (tid == 0) {
    a.new_seqlens[b] = a.seqlens_k[b] - gone * a.page_size;
    a.num_freed[b] = gone;
  }
}

}  // namespace fmoba

extern "C" size_t fmoba_cache_evict_workspace_bytes(int32_t batch, int32_t max_pages) {
  return batch > 0 && max_pages > fmoba::kEvictAlone ? (size_t)batch * (size_t)max_pages * 8 : 0;
}

extern "C" int fmoba_cache_evict(const fmoba_cache_evict_args *a, void *stream) {
  using namespace fmoba;
  FMOBA_REQUIRE(a != nullptr, "cache_evict: null args");
  FMOBA_REQUIRE(a->batch >= 1 && a->batch <= 65535 && a->max_pages >= 0 && a->num_pages >= 0 && a->heads_k >= 1, "cache_evict: sizes must not be negative, batch and heads positive");
  FMOBA_REQUIRE(a->page_size >= 1, "cache_evict: page_size must be positive");
  FMOBA_REQUIRE(a->sink >= 0 && a->recent >= 1, "cache_evict: sink pages must not be negative, and the page that is being filled stays (recent pages at least 1)");
  FMOBA_REQUIRE((int64_t)a->keep >= (int64_t)a->sink + a->recent, "cache_evict: fewer pages to keep than sink and recent pages");
  FMOBA_REQUIRE(a->seqlens_k && a->new_seqlens && a->num_freed && (a->max_pages == 0 || (a->block_table && a->new_table && a->freed)), "cache_evict: null pointer");
  FMOBA_REQUIRE(a->weight || a->num_pages == 0, "cache_evict: null pointer");
  const size_t need = fmoba_cache_evict_workspace_bytes(a->batch, a->max_pages);
  FMOBA_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need && (uintptr_t)a->workspace % 8 == 0), "cache_evict: workspace too small (%zu < %zu)", a->workspace_bytes, need);
  auto launch = [&](auto lanes) {
    constexpr int LP = decltype(lanes)::value;
    const hipStream_t s = (hipStream_t)stream;
    if (need > 0) {
      hipLaunchKernelGGL((cache_evict_sums_kernel<LP>), dim3(ceil_div(a->max_pages, 256 / LP * kAtOnce), a->batch), dim3(256), 0, s, *a);
      hipLaunchKernelGGL((cache_evict_kernel<LP, true>), dim3(a->batch), dim3(kEvictThreads), 0, s, *a);
    } else {
      hipLaunchKernelGGL((cache_evict_kernel<LP, false>), dim3(a->batch), dim3(kEvictThreads), 0, s, *a);
    }
  };
  if (a->heads_k >= 8)
    launch(std::integral_constant<int, 8>{});
  else if (a->heads_k >= 4)
    launch(std::integral_constant<int, 4>{});
  else if (a->heads_k >= 2)
    launch(std::integral_constant<int, 2>{});
  else
    launch(std::integral_constant<int, 1>{});
  FMOBA_LAUNCH_CHECK("cache_evict_kernel");
  return 0;
}
