// Gated attention over the paged 8-bit cache for many rows (parts of prompts, whole prompts): three launches.
//   gate     32 rows of a head: scores by matrix products in 32 bits, the best pages of every row; a row whose cut lies closer than the error of such a score
//            decides again in 64 bits.  Leaves the pages of every row, and for every page a word with one bit per row.
//   columns  a page of a key head and the rows that selected it, read from these words, 32 to a wave: S^T = K Q^T, softmax over the page, O^T = V^T P^T.
//            A page is brought into LDS once for all of them, widened to 16 bits, exactly; its scales multiply scores and the result of a visit.
//            Every visit leaves its output over the page and the logarithm of its sum.
//   combine  adds a row's visits.
// The weights of a visit go to the second product as two fp16 numbers each (split_weights).  Its output is summed in 32 bits and left in 16-bit whole numbers, 32767 for the largest of
// its features: at most 2^-16 of that is lost, a quarter of what fp16 would lose of most features.  Features far below the largest lose more of themselves, but a
// page's values are eight bits of one scale to begin with.
#include "kv_attn.h"

#include <algorithm>

namespace fmoba {

constexpr int kTileRows = 32;  // rows of a head that share a word of bits

constexpr int kNanPart = -32768;

struct ColumnPlan {
  CacheAttn c;
  int32_t *sel;      // [(row, head)][topk4]: pages, -1 behind them
  uint32_t *bits;    // [key head][block of 32 rows][head of the group][page]: a bit for each of the rows
  float *scores;     // [workgroup of the gate][32 rows][half of the wave][slot], where LDS does not hold them
  float2 *head;      // [(row, head)][slots]: log2 of a visit's sum of weights, and what its output has to be multiplied by
  uint16_t *part;    // [(row, head)][slots][head_dim]: that output, int16; kNanPart is a NaN
  int32_t topk4;     // topk, rounded up to a multiple of four
  int32_t steps;     // a page's, each a column of its own with step_keys keys (or 1)
  int32_t step_keys;
  int32_t slots;     // visits of a row, at most: pages times steps
  int32_t blocks;    // blocks of 32 rows, all sequences (block_of)
  int32_t row_blocks;  // of a sequence, at most
  int32_t gates;     // workgroups of the gate, where LDS does not hold their scores
  int32_t tiles;     // words of a page in a sequence, at most: its blocks times the heads of a group
  int32_t parts;     // workgroups of a page
};

// The first block of a sequence: those of a sequence of n rows from q0 on are ceil(n / 32) <= floor((q0 + n) / 32) - floor(q0 / 32) + 1.
__device__ __forceinline__ int64_t block_of(int q0, int b) { return q0 / kTileRows + b; }

// ------------------------------------------------------------------------------------
// gate: a workgroup takes 32 rows of a head, its waves a quarter of the pages each.  Scores^T = means q^T, so that a lane has half of a row's scores (the other half of the wave the others), 16 of a
// product's 32 pages.  A score gives its lowest bits up for the page's number; eight groups of a lane's scores are known by their largest, and the best
// are taken off one by one: the largest of eight, whose group is then looked through again.  About 60 instructions for one page of 32 rows, where counting
// scores above a cut (a ballot per 64 scores and bit) takes 30 for one bit of one row: 29 instead of 142 us, 8191 tokens, 16 heads, 64 pages.
// Bound by latency: 2825 rows of three sequences, 32 heads, up to 258 pages take 58 us, of which a workgroup spends a fifth on its queries' way, two fifths on the scores and a third on the
// best (the other waves wait); LDS has room for three of them a compute unit.  Page numbers a tile ahead and means fetched 64 bytes of a row at a time changed nothing.
// ------------------------------------------------------------------------------------
constexpr int kGateCols = 1024;   // pages whose scores of 32 rows LDS holds (135 KB); beyond, in the workspace (258 pages, whole calls: 94 us in LDS, 156 in the workspace)
// Bytes of the workspace for them, about: of a whole number of workgroups a compute unit (1 of tables of 32768 pages, 15 of 2048).  409 workgroups instead of 256, 1024 rows, 16 heads, 20000
// pages: 3710 and 3210 us; 1677, 2048 rows, 5000 pages: 1086, a workgroup for each of the 2048 blocks 1140.
constexpr int64_t kGateScores = int64_t(1) << 30;
constexpr int kGateGroups = 8;

// row . mean of a page in 64 bits, by 16 lanes (four pages a wave)
template <typename T>
__device__ __forceinline__ double row16_dot(const uint16_t *q, const uint16_t *mean, int D, int lane) {
  double s = 0.0;
  for (int e = (lane & 15) * 8; e < D; e += 128) {
    float f[8], g[8];
    unpack8<T>(ld_global16(q + e), f);
    unpack8<T>(ld_global16(mean + e), g);
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fma((double)f[j], (double)g[j], s);
  }
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  return s;
}
template <typename T>
__device__ __forceinline__ double lane_dot(const uint16_t *q, const uint16_t *mean, int D) {
  double s = 0.0;
  for (int e = 0; e < D; ++e) s = fma((double)elem_to_float<T>(q[e]), (double)elem_to_float<T>(mean[e]), s);
  return s;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
  return x;
}
// sum of the squares of eight elements, added to s
template <typename T>
__device__ __forceinline__ float add_squares(const Pack8 &x, float s) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef T pair_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    pair_t v;
    __builtin_memcpy(&v, &x.w[w], 4);
    if constexpr (std::is_same<T, bf16_t>::value)
      s = __builtin_amdgcn_fdot2_f32_bf16(v, v, s, false);
    else
      s = __builtin_amdgcn_fdot2(v, v, s, false);
  }
#endif
  return s;
}
// where a lane keeps the score of page c of its row: tile of 32 pages, 16 of them in each half of the wave
__device__ __forceinline__ int gate_half(int c) { return (c >> 2) & 1; }
__device__ __forceinline__ int gate_slot(int c) { return (c >> 5) * 16 + ((c >> 3) & 3) * 4 + (c & 3); }
__host__ __device__ __forceinline__ int gate_stride(int cols) { return (cols + 31) / 32 * 16 + 4; }  // floats of a lane (four more: 16 lanes' reads of 16 bytes meet all banks once)

static int64_t gate_score_bytes(int cols) { return (int64_t)kTileRows * 2 * gate_stride(cols) * 4; }
// 32 rows of a head: block rb of sequence b.  scores: (without LDS) a place for them that is no other workgroup's
template <typename T, int HD, bool LDS>
__device__ __forceinline__ void gate_block(const ColumnPlan &p, int page_bits, int rb, int h, int b, float *scores) {
  constexpr int KS = HD / 16;
  __shared__ float sTop[kGateGroups][64], sMean2[4], sLow[kTileRows];
  __shared__ int sPicked[kTileRows], sCandidate[4][64];
  __shared__ uint32_t sUnsure, sAll;
  extern __shared__ __align__(16) float gate_smem[];  // (LDS) the scores, [row][half][slot]; then the bits of every page
  const fmoba_cache_attn_args &a = p.c.a;
  const int D = a.cache.head_dim, P = a.cache.page_size, G = a.heads / a.cache.heads_k;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5, li = lane & 31;
  const int hk = h / G, cols = p.c.cols;
  const int q0 = a.cu_seqlens_q[b], q1 = a.cu_seqlens_q[b + 1], len = a.seqlens_k[b];
  const int R = min(min(q1, a.total_q) - q0, a.max_seqlen_q), row0 = rb * kTileRows;
  if (q0 < 0 || row0 >= R) return;
  const int shift = len - (q1 - q0);  // position of row 0
  const int rows = min(kTileRows, R - row0), last = shift + row0 + rows - 1;
  const int npages = min((int)(((int64_t)max(len, 0) + P - 1) / P), cols);                 // of the sequence
  const int nscore = last < 0 || a.topk <= 1 ? 0 : min(last / P, cols - 1);                // that any of the rows can select beside its own
  const int32_t *table = a.block_table + (int64_t)b * a.table_stride;
  const int stride = gate_stride(cols);
  if (LDS) scores = gate_smem;
  uint32_t *sBits = reinterpret_cast<uint32_t *>(gate_smem + (LDS ? kTileRows * 2 * stride : 0));
  float *mine = scores + (li * 2 + hh) * stride;
  const uint16_t *qh = reinterpret_cast<const uint16_t *>(a.q) + (int64_t)(q0 + row0) * a.q_row_stride + (int64_t)h * a.q_head_stride;
  const uint16_t *means = reinterpret_cast<const uint16_t *>(a.cache.k_mean) + (int64_t)hk * D;
  const int64_t mean_stride = (int64_t)a.cache.heads_k * D;
  const int nw = blockDim.x >> 6;
  for (int i = tid; i < npages; i += blockDim.x) sBits[i] = 0u;
  // this lane's row (both halves have it), its own page and the candidates before it
  const int pos = li < rows ? shift + row0 + li : -1;
  const int own = pos >= 0 ? pos / P : -1, n_row = own < 0 ? 0 : min(own, nscore), want = min(a.topk - 1, n_row);
  const int own_page = own >= 0 && own < cols ? table[own] : -1;
  int32_t *sel = p.sel + ((int64_t)(q0 + row0 + min(li, rows - 1)) * a.heads + h) * p.topk4;

  // ---- scores ----
  const int tiles = (nscore + 31) / 32, per_group = (tiles + kGateGroups - 1) / kGateGroups;
  const uint32_t number = (1u << page_bits) - 1u;
  float top[kGateGroups], q2 = 0.f, mean2 = 0.f;
  uint32_t q_bits = 0u;  // 0: a row of zeros
  if (nscore > 0) {
    Pack8 q[KS], k[KS];
    bool there = false;
    auto load = [&](int tile) {
      const int c = tile * 32 + li, page = tile < tiles && c < nscore ? table[c] : -1;
      there = page >= 0 && page < a.cache.num_pages;
      const uint16_t *mean = means + (int64_t)(there ? page : 0) * mean_stride + hh * 8;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) k[ks] = there && ks * 16 + hh * 8 < D ? ld_global16(mean + ks * 16) : zero_pack8();
    };
    load(wave * per_group);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int e = ks * 16 + hh * 8;
      q[ks] = e < D ? ld_global16(qh + (int64_t)min(li, rows - 1) * a.q_row_stride + e) : zero_pack8();
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q2 = add_squares<T>(q[ks], q2);
    q2 = sum_xor32_f(q2);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q_bits |= (q[ks].w[0] | q[ks].w[1] | q[ks].w[2] | q[ks].w[3]) & 0x7fff7fffu;
    q_bits |= (uint32_t)__shfl_xor((int)q_bits, 32, 64);
    for (int g = wave; g < kGateGroups; g += nw) {  // the groups of a wave
      const int end = min((g + 1) * per_group, tiles);
      float best = -INFINITY;
      for (int tile = g * per_group; tile < end; ++tile) {
        f32x16 acc;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = 0.f;
        float k2 = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) acc = mfma32<T>(k[ks], q[ks], acc);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) k2 = add_squares<T>(k[ks], k2);
        mean2 = fmaxf(mean2, sum_xor32_f(k2));
        const uint32_t valid = (uint32_t)__ballot(there);  // (both halves ask for the same pages)
        load(tile + 1 < end ? tile + 1 : (g + nw) * per_group);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f32x4 v;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int in_tile = 8 * j + 4 * hh + i, c = tile * 32 + in_tile;
            const float s = __uint_as_float((__float_as_uint(acc[4 * j + i]) & ~number) | (uint32_t)c);
            v[i] = c < n_row && ((valid >> in_tile) & 1u) ? s : NAN;  // (a NaN is never the largest)
            best = fmaxf(best, v[i]);
          }
          *reinterpret_cast<f32x4 *>(mine + tile * 16 + 4 * j) = v;
        }
      }
      sTop[g][lane] = best;
    }
    mean2 = wave_max(mean2);
    if (lane == 0) sMean2[wave] = mean2;
  }
  __syncthreads();
  auto set_bit = [&](int c, int r) { atomicOr(&sBits[c], 1u << r); };

  // ---- the best, one by one, by the first wave ----
  if (wave == 0) {
    float err = 0.f;
    // A score of D products in 32 bits, in whatever order and with whatever is cut off between the steps of the matrix unit, is off by less than D 2^-23 of
    // |q| |mean| (and these by less than 2^-10): scores further apart than twice that are in the order of 64 bits.  What is too small for 32 bits is lost beside that: up to 2^-126 of an
    // element, a product and a sum, whatever of it the matrix unit keeps, and of the whole where the page's number is in its place; of a square up to that of the least normal element.
    if (nscore > 0) {
      for (int w = 0; w < nw; ++w) mean2 = fmaxf(mean2, sMean2[w]);
      const float lost = (float)(D + 1) * 0x1p-126f, lost2 = std::is_same<T, bf16_t>::value ? lost : (float)D * 0x1p-28f;
      const float q_size = sqrtf(q2 + lost2), mean_size = sqrtf(mean2 + lost2);
      err = (float)D * (1.192092896e-7f * 1.002f) * q_size * mean_size + 2.f * lost * (1.f + q_size + mean_size);
    }
#pragma unroll
    for (int g = 0; g < kGateGroups; ++g) top[g] = nscore > 0 ? sTop[g][lane] : -INFINITY;
    int picked = 0;
    float in = INFINITY, out = -INFINITY;  // the last one taken, and the best that was not
    int steps = want;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) steps = max(steps, __shfl_xor(steps, o, 64));
    for (int i = 0; i <= steps && nscore > 0; ++i) {
      float best = top[0];
#pragma unroll
      for (int g = 1; g < kGateGroups; ++g) best = fmaxf(best, top[g]);
      best = max_xor32_f(best);
      const bool any = best > -INFINITY;
      if (any && i < want) {
        const int c = (int)(__float_as_uint(best) & number), tile = c >> 5;
        in = best;
        ++picked;
        if (hh == 0) {
          sel[i] = c;
          set_bit(c, li);
        }
        if (gate_half(c) == hh) {
          mine[gate_slot(c)] = -INFINITY;  // taken
          const int g = tile / per_group;
          float m = -INFINITY;
          for (int s = g * per_group; s < min((g + 1) * per_group, tiles); ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const f32x4 v = *reinterpret_cast<const f32x4 *>(mine + s * 16 + 4 * j);
#pragma unroll
              for (int k = 0; k < 4; ++k) m = fmaxf(m, v[k]);
            }
#pragma unroll
          for (int k = 0; k < kGateGroups; ++k) top[k] = k == g ? m : top[k];
        }
      } else if (any && i == want) {
        out = best;
      }
    }
    // Rows whose cut is too close for 32 bits.  (The page's number in a score: less than 2^(page_bits - 23) of it.  The scores of a row of zeros are equal, and of them the
    // later pages came first.)
    const float near = 2.f * err + ldexpf(2.f * fmaxf(fabsf(in), fabsf(out)), page_bits - 23);
    const bool sized = err < 1e30f;  // (else sizes overflow, or are no numbers: all pages decide in 64 bits)
    const bool unsure = li < rows && want > 0 && (!sized || (out > -INFINITY && q_bits != 0u && !(in - out > near)));
    if (hh == 0) sPicked[li] = picked, sLow[li] = in - near;
    const uint32_t unsure_rows = (uint32_t)__ballot(unsure), all_rows = (uint32_t)__ballot(!sized);
    if (lane == 0) sUnsure = unsure_rows, sAll = all_rows;
  }
  __syncthreads();

  // ---- these in 64 bits, by all waves: of the pages taken and those that the errors could bring before them, the best ----
  int nth = 0;
  for (uint32_t todo = sUnsure; todo; todo &= todo - 1u, ++nth) {
    if (nth % nw != wave) continue;
    const int r = __ffs((int)todo) - 1, n = __builtin_amdgcn_readlane(n_row, r), most = __builtin_amdgcn_readlane(want, r);
    const bool all = (sAll >> r) & 1u;
    const float low = sLow[r];
    float *rs = scores + r * 2 * stride;
    int32_t *rsel = p.sel + ((int64_t)(q0 + row0 + r) * a.heads + h) * p.topk4;
    const uint16_t *qr = qh + (int64_t)r * a.q_row_stride;
    auto at = [&](int c) { return rs + gate_half(c) * stride + gate_slot(c); };
    auto score64 = [&](int page) { return score_key(row16_dot<T>(qr, means + (int64_t)page * mean_stride, D, lane)); };
    int m = 0, got;
    for (int c0 = 0; c0 < n; c0 += 64) {
      const int c = c0 + lane;
      const float s = c < n ? *at(c) : NAN;
      const bool taken = s == -INFINITY, decides = taken || s >= low;
      const unsigned long long mask = __ballot(decides);
      const int place = m + __popcll(mask & ((1ull << lane) - 1ull));
      if (decides && place < 64) sCandidate[wave][place] = c;
      if (taken) atomicAnd(&sBits[c], ~(1u << r));
      m += __popcll(mask);
    }
    wave_lds_fence();
    if (m <= 64 && !all) {  // one a lane
      const int c = lane < m ? sCandidate[wave][lane] : 0, page = table[c];
      uint64_t key = 0ull;
      for (int i = 0; i < m; i += 4) {  // 16 lanes a product
        const uint64_t x = score64(__shfl(page, min(i + (lane >> 4), m - 1), 64));
        const uint64_t y = __shfl(x, (lane & 3) * 16, 64);
        if ((lane >> 2) == (i >> 2)) key = y;
      }
      if (lane >= m) key = 0ull;
      int rank = 0;
      for (int i = 0; i < m; ++i) {
        const uint64_t other = __shfl(key, i, 64);
        rank += other > key || (other == key && __builtin_amdgcn_readlane(c, i) > c) ? 1 : 0;
      }
      const bool chosen = key != 0ull && rank < most;
      const unsigned long long mask = __ballot(chosen);
      if (chosen) {
        rsel[__popcll(mask & ((1ull << lane) - 1ull))] = c;
        set_bit(c, r);
      }
      got = __popcll(mask);
    } else {
      for (int c0 = 0; c0 < n; c0 += 64) {
        const int c = c0 + lane, page = c < n ? table[c] : -1;
        const float s = c < n ? *at(c) : NAN;
        const bool decides = page >= 0 && page < a.cache.num_pages && (all || s == -INFINITY || s >= low);
        uint32_t key = 0u;
        for (unsigned long long left = __ballot(decides); left;) {  // four at a time
          int l = -1;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int next = left ? (int)__ffsll(left) - 1 : l;
            if (lane >> 4 >= u) l = next;
            left &= left - 1ull;
          }
          const uint64_t x = score64(__shfl(page, l, 64));
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int to = __builtin_amdgcn_readlane(l, u * 16);
            const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), u * 16);
            if (lane == to) key = hi;
          }
        }
        if (c < n) *at(c) = __uint_as_float(key);  // its own lane reads it below
      }
      got = pick_best<0>(
          n, most, lane, [&](int c) { return __float_as_uint(*at(c)); }, [&](int c) { return (uint32_t)score_key(lane_dot<T>(qr, means + (int64_t)table[c] * mean_stride, D)); },
          [](int c) { return c; },
          [&](int c, uint32_t, int i) {
            rsel[i] = c;
            set_bit(c, r);
          });
    }
    if (lane == 0) sPicked[r] = got;
  }
  __syncthreads();
  if (wave == 0 && hh == 0 && li < rows) {
    int picked = sPicked[li];
    if (own_page >= 0 && own_page < a.cache.num_pages) {
      sel[picked++] = own;
      set_bit(own, li);
    }
    for (int i = picked; i < p.topk4; ++i) sel[i] = -1;
  }
  __syncthreads();
  uint32_t *bits = p.bits + (((int64_t)hk * p.blocks + block_of(q0, b) + rb) * G + (h - hk * G)) * cols;
  for (int i = tid; i < npages; i += blockDim.x) bits[i] = sBits[i];
}

// A workgroup a block where LDS holds its scores; else as many workgroups as the device runs at a time, each with a place in the workspace that its blocks share one after the other: for
// rows of a long prompt, all of whose scores together are rows times pages.  Every other head's blocks come from the last on, so that a workgroup has early and late ones.
template <typename T, int HD, bool LDS>
__global__ __launch_bounds__(256) void cache_gate_kernel(ColumnPlan p, int page_bits) {
  if constexpr (LDS) {
    gate_block<T, HD, true>(p, page_bits, blockIdx.x, blockIdx.y, blockIdx.z, nullptr);
  } else {
    const int heads = p.c.a.heads;
    const int64_t all = (int64_t)p.row_blocks * heads * p.c.a.batch;
    float *scores = p.scores + (int64_t)blockIdx.x * kTileRows * 2 * gate_stride(p.c.cols);
    for (int64_t i = blockIdx.x; i < all; i += gridDim.x) {
      const int64_t nth = i / p.row_blocks;  // head of a sequence
      const int rb = (int)(i - nth * p.row_blocks), b = (int)(nth / heads), h = (int)(nth - (int64_t)b * heads);
      if (i != blockIdx.x) __syncthreads();  // (what the block before has in LDS and in the workspace is read)
      gate_block<T, HD, false>(p, page_bits, nth & 1 ? p.row_blocks - 1 - rb : rb, h, b, scores);
    }
  }
}

// ------------------------------------------------------------------------------------
// columns: a workgroup of four waves keeps a page in LDS and takes 128 of its rows a turn, what a turn needs of memory on its way during the one before.  2825 rows of three sequences of 9216 to 33000
// tokens, 32 over 8 heads of 128: 171 us, 402 MB at 2.4 TB/s; 8191 rows, 16 heads: 167 us, 0.41 PFLOP/s.  Bound by latency: products and softmax of a turn would take a third of what it does; with one product a
// weight (155 and 147 us), 16 of a workgroup's 33 thousand clocks (1.9 turns a page) were gone before its first product, on lengths and table, words of bits and the page, the rows, one
// after the other, and two waves a SIMD (256 registers) hide little of it.  (Two pages a workgroup, the second one's bytes on their way during the first one's last turn, in the registers of the
// rows, then: 185 and 206.)
// ------------------------------------------------------------------------------------
constexpr int kColumnRows = 128;  // of a turn: 32 a wave
constexpr int kColumnWords = 128;  // words of bits that are spread out at a time: 32 a wave
constexpr int kColumnList = kColumnRows + kColumnWords * 32;
constexpr int kColumnPart = 2048;  // words of a workgroup, at most: an entry of its list has 16 bits

// two numbers of [-1, 1] as int16, rounded to nearest
__device__ __forceinline__ uint32_t pack_part(float x, float y) {
  uint32_t w = 0u;
#if defined(__HIP_DEVICE_COMPILE__)
  const auto two = __builtin_amdgcn_cvt_pknorm_i16(x, y);
  __builtin_memcpy(&w, &two, 4);
#endif
  return w;
}

// Weights are formed as 2^15 of themselves and go to the second product as two fp16 numbers each, the second what the first cuts off: what is lost is 2^-20 of a weight, or 2^-39
// of the largest.  (As one fp16 number, 2^-11 of a weight, outputs in fp16 were 1.3 times as far from 64 bits as their own rounding; it costs 6 %.  The remainder by one mixed
// multiply-add instead of a conversion and a subtraction: the registers spill, no time gained.)
constexpr float kWeightBits = 15.f, kOneWeight = 1.f / 32768.f;
__device__ __forceinline__ void split_weights(float x, float y, uint32_t &two, uint32_t &rest) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto cut = __builtin_amdgcn_cvt_pkrtz(x, y);
  const auto left = __builtin_amdgcn_cvt_pkrtz(x - (float)cut[0], y - (float)cut[1]);
  __builtin_memcpy(&two, &cut, 4);
  __builtin_memcpy(&rest, &left, 4);
#else
  (void)x, (void)y, (void)two, (void)rest;
#endif
}

// ONE: the column is one step of KT keys, which LDS holds
template <typename T, typename H, int HD, int KT, bool ONE>  // KT: keys of a softmax step
__global__ __launch_bounds__(256, HD > 128 ? 1 : 2) void cache_columns_kernel(ColumnPlan p, int held) {  // held: keys of a page that LDS holds at a time
  constexpr int KS = HD / 16, DT = HD / 32, ST = KT / 32, ROW = HD * 2;  // (LDS rows of exactly HD elements, their pieces swizzled: tile_swz)
  extern __shared__ __align__(1024) uint8_t column_smem[];
  __shared__ uint16_t sList[kColumnList];
  __shared__ int sFound[4], sNan;
  const fmoba_cache_attn_args &a = p.c.a;
  const int D = a.cache.head_dim, P = a.cache.page_size, G = a.heads / a.cache.heads_k, cols = p.c.cols;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5, li = lane & 31;
  const PairItem item = xcd_pair_item(blockIdx.x, a.batch * a.cache.heads_k, cols * p.steps * p.parts);
  const int b = item.pair / a.cache.heads_k, hk = item.pair - b * a.cache.heads_k, nth = item.idx / p.parts, part = item.idx - nth * p.parts;
  const int c = nth / p.steps, step = nth - c * p.steps, key0 = ONE ? step * KT : 0;  // page of the table, and the first of its keys that are this column's
  const int q0 = a.cu_seqlens_q[b], q1 = a.cu_seqlens_q[b + 1], len = a.seqlens_k[b], page = a.block_table[(int64_t)b * a.table_stride + c];  // (asked for together)
  const int R = min(min(q1, a.total_q) - q0, a.max_seqlen_q);
  if (q0 < 0 || R <= 0 || (int64_t)c * P + key0 >= len || page < 0 || page >= a.cache.num_pages) return;
  const int shift = len - (q1 - q0), G_tiles = (R + kTileRows - 1) / kTileRows * G;
  // the words of rows that can see the page, shared out evenly
  const int first = max(c * P + key0 - shift, 0) / kTileRows * G;
  const int each = ((G_tiles - first + p.parts - 1) / p.parts + 7) / 8 * 8;
  const int w0 = first + part * each, w1 = min(w0 + each, G_tiles);
  if (w0 >= w1) return;
  const int keys = min(ONE ? KT : P, len - c * P - key0);  // that are there
  const uint32_t *bits = p.bits + ((int64_t)hk * p.blocks + block_of(q0, b)) * G * cols + c;
  const uint8_t *kg = reinterpret_cast<const uint8_t *>(a.cache.k) + (int64_t)page * a.cache.k_page_stride + (int64_t)hk * a.cache.k_head_stride + (int64_t)key0 * a.cache.k_token_stride;
  const uint8_t *vg = reinterpret_cast<const uint8_t *>(a.cache.v) + (int64_t)page * a.cache.v_page_stride + (int64_t)hk * a.cache.v_head_stride + (int64_t)key0 * a.cache.v_token_stride;
  const int my_word = wave * 32 + li;
  uint32_t word = hh == 0 && w0 + my_word < w1 ? bits[(int64_t)(w0 + my_word) * cols] : 0u;  // (those of the next turn of words, always)
  // the scale of a score, its sign with q (the largest product is the largest score), and not 0 (times which a masked product would be no number)
  const float scale_log2 = a.softmax_scale * 1.4426950408889634f, scale_abs = fabsf(scale_log2) * a.cache.k_scale[(int64_t)page * a.cache.heads_k + hk];
  const float k_scale = scale_abs < 1e-30f ? 1e-30f : scale_abs;
  const uint32_t q_sign = scale_log2 < 0.f ? 0x80008000u : 0u;
  const float v_scale = a.cache.v_scale[(int64_t)page * a.cache.heads_k + hk];
  if (tid == 0) sNan = 0;

  const uint32_t k_base = (uint32_t)(uintptr_t)to_lds(column_smem), v_base = k_base + (uint32_t)(held * ROW);
  // keys [k0, k0 + held) of the page, widened; features past D and keys that are not there are zeros, and so are NaNs among the values (they count below)
  constexpr int PIECES = HD / 16, AT_ONCE = 4;  // 16-byte pieces of a row; of K and of V that a thread has on their way at a time (a page of one step: all of its)
  Pack8 kx[AT_ONCE], vx[AT_ONCE];
  auto stage_ask = [&](int k0, int i0) {
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = i0 + u * 256, r = i / PIECES, e = (i % PIECES) * 16;
      const bool there = i < held * PIECES && k0 + r < keys && e < D;
      kx[u] = there ? ld_global16(kg + (int64_t)(k0 + r) * a.cache.k_token_stride + e) : zero_pack8();
      vx[u] = there ? ld_global16(vg + (int64_t)(k0 + r) * a.cache.v_token_stride + e) : zero_pack8();
    }
  };
  auto stage_put = [&](int i0) {
    bool nan = false;
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = i0 + u * 256, r = i / PIECES, piece = (i % PIECES) * 2;
      if (i >= held * PIECES) continue;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        u32x4_t ko, vo;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t lo, hi, vw = vx[u].w[half * 2 + w];
          H::template widen4<T>(kx[u].w[half * 2 + w], lo, hi);
          ko[2 * w] = lo, ko[2 * w + 1] = hi;
          if (H::any_nan4(vw)) nan = true, vw = H::without_nan4(vw);
          H::template widen4<f16_t>(vw, lo, hi);
          vo[2 * w] = lo, vo[2 * w + 1] = hi;
        }
        const uint32_t at = (uint32_t)(r * ROW + ((piece + half) ^ tile_swz<HD>(r)) * 16);
        lds_write_vec(k_base + at, ko);
        lds_write_vec(v_base + at, vo);
      }
    }
    if (nan) sNan = 1;
  };
  auto stage = [&](int k0) {
    for (int i0 = tid; i0 < held * PIECES; i0 += 256 * AT_ONCE) {
      stage_ask(k0, i0);
      stage_put(i0);
    }
  };
  // where this lane's operands lie: of K row li, its pieces; of V four features of a row of four, and the row eight further down
  uint32_t k_at[KS], v_lo[DT], v_hi[DT];
  {
    const uint32_t k0 = (uint32_t)(li * ROW + (tile_frag_piece<HD>(hh, 0) ^ tile_swz<HD>(li)) * 16);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k_at[ks] = k_base + tile_frag_addr<HD>(k0, ks);
    const int i = lane & 15, r = 4 * hh + (i >> 2);
    const uint32_t v0 = (uint32_t)(r * ROW + (((li >> 4) * 2 + ((i & 3) >> 1)) ^ tile_swz<HD>(r)) * 16 + (i & 1) * 8);
#pragma unroll
    for (int d = 0; d < DT; ++d) v_lo[d] = v_base + tile_tr_addr<HD>(v0, d), v_hi[d] = v_base + tile_tr_addr8<HD>(v0, d);
  }

  // the value of the lane of this half with lane % 32 = lane % 16, or 16 + lane % 16
  auto of_pair = [&](int64_t x, bool odd) {
    const UPair lo = swap16((uint32_t)x), hi = swap16((uint32_t)((uint64_t)x >> 32));
    return (int64_t)((uint64_t)(odd ? hi.b : hi.a) << 32 | (odd ? lo.b : lo.a));
  };
  // What a turn of 128 entries of the list needs of memory: the rows' queries, four lanes 64 bytes of a row at a time, each lane of entries lane % 16 and
  // 16 + lane % 16 (q_rows_load), and the first of their pages, among which the visit's place is.  Asked for while the turn before is under way, once its
  // products with the keys are done (the registers of its queries are free then).
  Pack8 q[KS];
  int4 pages[2];
  int row = 0, g = 0;
  int64_t rowhead = (int64_t)q0 * a.heads + hk * G;
  auto ask = [&](int from, int count) {
    const int entry = sList[from + min(wave * 32 + li, count - 1)], w = w0 + (entry >> 5), rb = w / G;
    g = w - rb * G, row = rb * kTileRows + (entry & 31);
    rowhead = (int64_t)(q0 + row) * a.heads + hk * G + g;
    const int64_t qr = (int64_t)(q0 + row) * a.q_row_stride + (int64_t)(hk * G + g) * a.q_head_stride;
    const uint16_t *even = reinterpret_cast<const uint16_t *>(a.q) + of_pair(qr, false), *odd = reinterpret_cast<const uint16_t *>(a.q) + of_pair(qr, true);
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const int e = min((4 * i + (lane >> 4)) * 8, D - 8);  // (features past D: zeroed by the exchange)
      q[2 * i] = ld_global16(even + e);
      q[2 * i + 1] = ld_global16(odd + e);
    }
    const int4 *sel = reinterpret_cast<const int4 *>(p.sel + rowhead * p.topk4);
    pages[0] = sel[0], pages[1] = sel[p.topk4 > 4 ? 1 : 0];
  };
  auto place = [&]() {  // of the visit among the row's
    auto among = [&](const int4 &s, int i, int slot) { return s.x == c ? i : s.y == c ? i + 1 : s.z == c ? i + 2 : s.w == c ? i + 3 : slot; };
    int slot = among(pages[0], 0, among(pages[1], 4, 0));
    const int4 *sel = reinterpret_cast<const int4 *>(p.sel + rowhead * p.topk4);
    for (int i = 8; i < p.topk4; i += 4) slot = among(sel[i >> 2], i, slot);
    return slot;
  };
  // What was asked for, taken over before anything is stored: a wait for loads is one for the stores in front of them too.
  int64_t at_next = 0;
  int lim_next = 0;
  auto take_over = [&]() {
    q_rows_arrange<HD>(q, hh, D);
    if (q_sign != 0u) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i) q[ks].w[i] ^= q_sign;
    }
    at_next = rowhead * p.slots + place() * p.steps + step;
    lim_next = shift + row - c * P - key0;  // last key that the row sees (of its own page's later steps none, and the combine looks at none)
  };
  // one turn: `count` entries of the list, which were asked for and taken over; then those of the next turn, `next` from `from_next` on
  auto turn = [&](int count, int from_next, int next) {
    if (ONE && wave * 32 >= count) return;  // (a last turn: nothing follows)
    const bool there = wave * 32 + li < count;
    const int lim = lim_next;
    const int64_t at = at_next;
    f32x16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    for (int k0 = 0; k0 < (ONE ? 1 : keys); k0 += held) {
      if (!ONE && held < P) {
        __syncthreads();
        stage(k0);
        __syncthreads();
      }
      for (int s0 = 0; s0 < (ONE ? 1 : held) && k0 + s0 < keys; s0 += KT) {
        if (!ONE && __ballot(there && lim >= k0 + s0) == 0ull) continue;
        const uint32_t off = (uint32_t)(s0 * ROW);
        f32x16 s[ST];
#pragma unroll
        for (int t = 0; t < ST; ++t) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[t][i] = 0.f;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) s[t] = mfma32<T>(lds_read16(k_at[ks] + off + (uint32_t)(t * 32 * ROW)), q[ks], s[t]);
        }
        if (ONE && next > 0) ask(from_next, next);
        const int left = lim - k0 - s0;  // last visible key of this step
        float mx = -INFINITY;
        if (__ballot(left < KT - 1) != 0ull) {
#pragma unroll
          for (int t = 0; t < ST; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][i] = t * 32 + acc_row(i, hh) <= left ? s[t][i] : -INFINITY;
        }
#pragma unroll
        for (int t = 0; t < ST; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
        mx = max_xor32_f(mx) * k_scale;
        const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
        if (!ONE && k0 + s0 > 0) {
          const float resc = __builtin_amdgcn_exp2f(m - ref);
          l *= resc;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= resc;
        }
        m = mn;
        const float base = kWeightBits - ref;
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < ST; ++t)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            Pack8 pk, rest;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
              const float x = __builtin_amdgcn_exp2f(fmaf(s[t][8 * u + i], k_scale, base)), y = __builtin_amdgcn_exp2f(fmaf(s[t][8 * u + i + 1], k_scale, base));
              sum += x + y;
              split_weights(x, y, pk.w[i >> 1], rest.w[i >> 1]);
            }
            const uint32_t rows = off + (uint32_t)((t * 32 + 16 * u) * ROW);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              const Pack8 vt = lds_tr8(v_lo[d] + rows, v_hi[d] + rows);
              o[d] = mfma32<f16_t>(vt, pk, o[d]);
              o[d] = mfma32<f16_t>(vt, rest, o[d]);
            }
          }
        l += sum_xor32_f(sum);
      }
    }
    if (ONE && next > 0) take_over();
    uint16_t *dst = p.part + at * D;
    float most = 1e-36f;  // (a NaN is none; smaller sums are nothing beside the others')
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(o[d][i]));
    most = max_xor32_f(most);
    const float inv = l == 0.f ? 0.f : 1.f / l, norm = __builtin_amdgcn_rcpf(most);
    if (there && hh == 0) p.head[at] = make_float2(l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l * kOneWeight), v_scale * (inv * most * (1.f / 32767.f)));
    {
      // Features 8 j + 4 hh .. of both halves to eight of one lane, then to four lanes with 64 bytes of a row, as the queries were loaded: stores of 16 bytes of 64
      // rows at a time take the caches a cycle for each.
      uint16_t *even = p.part + of_pair(at * D, false), *odd = p.part + of_pair(at * D, true);
      const bool even_there = wave * 32 + (lane & 15) < count, odd_there = wave * 32 + 16 + (lane & 15) < count;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        uint32_t x[4], y[4];  // pieces 4 d + hh and 4 d + 2 + hh of row li
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) (j < 2 ? x : y)[(j & 1) * 2 + i] = pack_part(o[d][4 * j + 2 * i] * norm, o[d][4 * j + 2 * i + 1] * norm);
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const auto r = __builtin_amdgcn_permlane32_swap(x[i], x[2 + i], false, false), s = __builtin_amdgcn_permlane32_swap(y[i], y[2 + i], false, false);
          x[i] = r[0], x[2 + i] = r[1], y[i] = s[0], y[2 + i] = s[1];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const auto r = __builtin_amdgcn_permlane16_swap(x[i], y[i], false, false);
          x[i] = r[0], y[i] = r[1];
        }
#endif
        const int e = d * 32 + ((lane >> 4 & 1) * 2 + hh) * 8;
        if (e < D && even_there) *reinterpret_cast<Pack8 *>(even + e) = Pack8{{x[0], x[1], x[2], x[3]}};
        if (e < D && odd_there) *reinterpret_cast<Pack8 *>(odd + e) = Pack8{{y[0], y[1], y[2], y[3]}};
      }
    }
    // NaNs among the values of the page: a row that sees one has it in that feature
    if (H::kFormat == FMOBA_CACHE_E4M3 && sNan != 0) {
      wait_all_loads();  // (the stores above, which other lanes made)
      if (there) {
        const int last = min(lim, keys - 1);
        for (int e = hh; e < D; e += 2)
          for (int k = 0; k <= last; ++k)
            if ((vg[(int64_t)k * a.cache.v_token_stride + e] & 0x7f) == 0x7f) dst[e] = (uint16_t)kNanPart;
      }
    }
  };

  // the bits of kColumnWords words from wb on, spread out behind the `have` entries that the list has; returns how many it has then
  auto spread = [&](int wb, int have) {
    uint32_t x = word;
    const int n = __popc(x);
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int before = __shfl_up(upto, o, 32);
      upto += li >= o ? before : 0;
    }
    if (lane == 31) sFound[wave] = upto;
    const int next = wb + kColumnWords + my_word;
    word = hh == 0 && next < w1 ? bits[(int64_t)next * cols] : 0u;
    __syncthreads();
    int at = have + upto - n, count = have;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      at += w < wave ? sFound[w] : 0;
      count += sFound[w];
    }
    while (x) {
      sList[at++] = (uint16_t)((wb - w0 + my_word) << 5 | (__ffs(x) - 1));
      x &= x - 1u;
    }
    __syncthreads();
    return count;
  };
  if (!ONE && held >= P) {
    __syncthreads();  // (sNan is cleared before any wave sets it: the others have a barrier of their own before they store)
    stage(0);
  }
  if (ONE) stage_ask(0, tid);
  int wb = w0, count = spread(w0, 0);
  if (ONE && (count >= kColumnRows || wb + kColumnWords >= w1) && count > 0) ask(0, min(kColumnRows, count));
  if (ONE) {
    stage_put(tid);
    take_over();  // (of nothing, if there is no turn yet)
  }
  __syncthreads();
  while (true) {
    const bool end = wb + kColumnWords >= w1;
    int from = 0;
    auto turn_at = [&](int f) { return count - f >= kColumnRows || end ? min(kColumnRows, count - f) : 0; };  // entries of the turn that begins there
    for (int now = turn_at(0), then; now > 0; now = then) {
      then = turn_at(from + kColumnRows);
      if (!ONE) {
        ask(from, now);
        take_over();
      }
      turn(now, from + kColumnRows, then);
      from += kColumnRows;
    }
    if (end) return;
    const int have = max(count - from, 0);  // entries that wait
    __syncthreads();
    if (from > 0 && have > 0) {
      const uint16_t moved = tid < have ? sList[from + tid] : (uint16_t)0;
      __syncthreads();
      if (tid < have) sList[tid] = moved;
    }
    wb += kColumnWords;
    count = spread(wb, have);
    if (ONE && (count >= kColumnRows || wb + kColumnWords >= w1) && count > 0) {
      ask(0, min(kColumnRows, count));
      take_over();
    }
  }
}

// ------------------------------------------------------------------------------------
// combine: LPR lanes a (row, head), eight features each.  Bound by memory: two bytes a feature and visit (2825 rows, 32 heads of 128, 8 pages a row: 40 us, 206 MB at
// 5.1 TB/s; 46 with as many registers as the compiler takes, for five waves a SIMD instead of six; with weights, or heads of 64, the smaller number spills).
// ------------------------------------------------------------------------------------
// WEIGHT: what pages receive is added up in LDS for the rows of the workgroup first (integers, so in no order): rows next to each other choose alike, and
// atomics on few addresses of memory are slow (a million of them 180 us).
constexpr int kCombineCols = 2048, kCombineSlots = 64;
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
template <typename T, int LPR, bool WEIGHT>
__global__ __launch_bounds__(256, !WEIGHT && LPR == 16 ? 6 : 4) void cache_combine_kernel(ColumnPlan p, int rows) {  // rows: of a workgroup
  constexpr int AT_ONCE = 8;  // parts asked for together
  __shared__ unsigned long long sWeight[WEIGHT ? kCombineCols : 1];
  const fmoba_cache_attn_args &a = p.c.a;
  const int tid = threadIdx.x, lane = tid & 63, li = lane % LPR, group = lane - li, D = a.cache.head_dim, P = a.cache.page_size, h = blockIdx.y, t0 = blockIdx.x * rows;
  const int hk = h / (a.heads / a.cache.heads_k), cols = min(p.c.cols, kCombineCols);
  const int b0 = WEIGHT ? find_row_lane(a, t0).b : 0;
  const uint32_t per_step = (65535u + (uint32_t)p.steps) / (uint32_t)p.steps;  // s / steps = s per_step >> 16 for s below 64 and up to 16 steps
  auto receive = [&](int b, int c, unsigned long long x) {
    const int page = a.block_table[(int64_t)b * a.table_stride + c];
    if (page >= 0 && page < a.cache.num_pages) atomicAdd(reinterpret_cast<unsigned long long *>(a.cache.weight) + (int64_t)page * a.cache.heads_k + hk, x);
  };
  if constexpr (WEIGHT) {
    for (int i = tid; i < cols; i += 256) sWeight[i] = 0ull;
    __syncthreads();
  }
  for (int t = t0 + tid / LPR; t < min(t0 + rows, a.total_q); t += 256 / LPR) {
    const int64_t rowhead = (int64_t)t * a.heads + h;
    const int32_t *sel = p.sel + rowhead * p.topk4;
    const float2 *head = p.head + rowhead * p.slots;
    const uint16_t *part = p.part + rowhead * p.slots * D;
    const RowPlace at = find_row_lane(a, t);
    // visit s of the row: its page (or -1), the logarithm of its weights' sum (-inf if there is none) and its output's factor
    auto visit = [&](int s, int &c, float2 &x) {
      const int nth = (int)((uint32_t)s * per_step >> 16), page = s < p.slots && at.pos >= 0 ? sel[nth] : -1;
      c = page >= 0 && at.pos - page * P >= (s - nth * p.steps) * p.step_keys ? page : -1;  // (its own page is a row's last, and has the steps up to its place)
      x = c >= 0 ? head[s] : make_float2(-INFINITY, 0.f);
    };
    // They fill the slots from the first on, LPR of them at a time, one a lane; most rows have no more, and are asked for once.
    int c_first, n = 0;
    float2 x_first;
    float m = -INFINITY, l = 0.f;
    visit(li, c_first, x_first);
#pragma unroll 1
    for (int s0 = 0; s0 < p.slots; s0 += LPR) {
      int c = c_first;
      float2 x = x_first;
      if (s0 > 0) visit(s0 + li, c, x);
      m = x.x > m ? x.x : m;
      n += c >= 0 ? 1 : 0;
    }
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64)), n += __shfl_xor(n, o, 64);
    const float ref = m == -INFINITY ? 0.f : m;
    const int e = li * 8;
    float acc[8];
    i16x2 least = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.f;
#pragma unroll 1
    for (int s0 = 0; s0 < p.slots; s0 += LPR) {
      int c = c_first;
      float2 x_head = x_first;
      if (s0 > 0) visit(s0 + li, c, x_head);
      const float w = __builtin_amdgcn_exp2f(x_head.x - ref), vs = w * x_head.y;
      l += w;
#pragma unroll 1
      for (int i0 = 0; i0 < LPR && s0 + i0 < p.slots; i0 += AT_ONCE) {
        Pack8 x[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          const int s = s0 + i0 + i;
          x[i] = s < n && e < D ? ld_stream16(part + (int64_t)s * D + e) : zero_pack8();
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          const float of_visit = __shfl(vs, group + i0 + i, 64), wv = s0 + i0 + i < n ? of_visit : 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            i16x2 two;
            __builtin_memcpy(&two, &x[i].w[k], 4);
            least = __builtin_elementwise_min(least, two);
            acc[2 * k] = fmaf(wv, (float)two.x, acc[2 * k]);
            acc[2 * k + 1] = fmaf(wv, (float)two.y, acc[2 * k + 1]);
          }
        }
      }
    }
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) l += __shfl_xor(l, o, 64);
    if (min(least.x, least.y) == kNanPart && l != 0.f) {  // (seldom: once more; a NaN that a row sees is one whatever its weight, in this form as in the other)
      for (int s = 0; s < n; ++s) {
        const Pack8 again = ld_global16(part + (int64_t)s * D + e);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] = (int16_t)(again.w[k >> 1] >> (16 * (k & 1))) == kNanPart ? NAN : acc[k];
      }
    }
    const bool empty = l == 0.f;
    const float inv = empty ? 0.f : 1.f / l;
    if (e < D) {
      Pack8 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) o.w[j] = pack2<T>(acc[2 * j] * inv, acc[2 * j + 1] * inv);
      *reinterpret_cast<Pack8 *>(reinterpret_cast<uint16_t *>(a.out) + (int64_t)t * a.o_row_stride + (int64_t)h * a.o_head_stride + e) = o;
    }
    if (li == 0) a.softmax_lse[(int64_t)h * a.total_q + t] = empty ? INFINITY : (ref + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
    if constexpr (WEIGHT) {
  #pragma unroll 1
    for (int s0 = 0; s0 < p.slots; s0 += LPR) {
        int c = c_first;
        float2 x = x_first;
        if (s0 > 0) visit(s0 + li, c, x);
        const float part_of = __builtin_amdgcn_exp2f(x.x - ref) * inv;
        if (!(part_of > 0.f) || c < 0) continue;
        const unsigned long long whole = (unsigned long long)rintf(part_of * 4294967296.f);
        if (at.b == b0 && c < cols)
          atomicAdd(&sWeight[c], whole);
        else
          receive(at.b, c, whole);
      }
    }
  }
  if constexpr (WEIGHT) {
    __syncthreads();
    for (int i = tid; i < cols; i += 256)
      if (sWeight[i] != 0ull) receive(b0, i, sWeight[i]);
  }
}

// ------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------
static size_t up(size_t x) { return (x + 255) & ~(size_t)255; }
struct ColumnSizes {
  size_t sel, bits, scores, head, part, total;
};
static ColumnSizes column_sizes(const fmoba_cache_attn_args &a, int cols, ColumnPlan &p) {
  const size_t rowheads = (size_t)a.total_q * a.heads;
  p.topk4 = (a.topk + 3) / 4 * 4;
  p.blocks = a.total_q / kTileRows + a.batch;
  p.row_blocks = ceil_div(std::min(a.max_seqlen_q, a.total_q), kTileRows);
  p.tiles = p.row_blocks * (a.heads / a.cache.heads_k);
  p.gates = (int)std::min<int64_t>((int64_t)p.row_blocks * a.heads * a.batch, std::max<int64_t>(kGateScores / gate_score_bytes(cols) / 256, 1) * 256);
  // Pages of one step (64 keys, or 128 of heads up to 128, whose scores of a row fit the registers): nothing before it has to be scaled for, and its next rows can be on their way.  Larger pages are
  // several columns of one step each, as far as the combine has places for a row's visits; else one column of many steps, whose keys come into LDS 64 at a time, again for every turn,
  // where two workgroups do not find room for all.  (Whole calls, with one product a weight: 8191 tokens, 16 over 4 heads of 128, pages of 256 keys, four a row: 260 us in two steps, 526 in one column; of 512, two a row: 245 and 670;
  // heads of 256, pages of 128, eight a row: 785 and 1013.)
  const int pages = std::min(a.topk, cols);
  p.step_keys = a.cache.head_dim <= 128 && a.cache.page_size % 128 == 0 ? 128 : 64;
  p.steps = a.cache.page_size / p.step_keys;
  if (pages * p.steps > kCombineSlots) p.steps = 1, p.step_keys = a.cache.page_size;
  p.slots = pages * p.steps;
  // Workgroups of a page: four turns of rows each, if rows choose evenly, and an odd number: the last ones of a late page, which few rows see, have nothing to
  // do, and would otherwise come to the same shader engines for every page (whole calls, with one product a weight: 8191 tokens, 16 heads: 223 us even, 201 odd; 8192, 16 over 2 heads: 380 and 254;
  // 4 x 4096, 32 over 8 heads: two turns 778, three 751, four 745, six 740, twelve 779; 16384, 28 over 4 heads: 870, 902, 949, 1037, 1126).
  const int64_t visits = (int64_t)p.tiles * kTileRows * std::min(a.topk, cols) / cols;
  p.parts = (int)std::min<int64_t>(std::max<int64_t>(std::max<int64_t>(visits / (4 * kColumnRows), ceil_div(p.tiles, kColumnPart - 32)), 1), ceil_div(p.tiles, 32)) | 1;
  ColumnSizes z;
  z.sel = up(rowheads * p.topk4 * 4);
  z.bits = up((size_t)a.heads * p.blocks * cols * 4);
  z.scores = cols > kGateCols ? up(p.gates * gate_score_bytes(cols)) : 0;
  z.head = up(rowheads * p.slots * 8);
  z.part = up(rowheads * p.slots * a.cache.head_dim * 2);
  z.total = z.sel + z.bits + z.scores + z.head + z.part;
  return z;
}
size_t column_workspace_bytes(const fmoba_cache_attn_args &a, int cols) {
  ColumnPlan p{};
  return column_sizes(a, cols, p).total;
}

bool column_grid_fits(const fmoba_cache_attn_args &a, int cols) {
  ColumnPlan p{};
  column_sizes(a, cols, p);
  // (gate: a block of rows; columns: a page; combine: 64 rows or more)
  return (int64_t)a.batch * a.cache.heads_k * cols * p.steps * p.parts * 256 <= UINT32_MAX && (int64_t)p.row_blocks * 256 <= UINT32_MAX && ceil_div64(a.total_q, 64) * 256 <= UINT32_MAX;
}

template <typename K>
static int with_lds(K kern, size_t bytes, const char *what) {
  if (bytes > 48 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess) {
    set_error("%s: cannot reserve %zu bytes of LDS", what, bytes);
    return 2;
  }
  return 0;
}

template <typename T, int HD>
static int launch_gate(const ColumnPlan &p, hipStream_t s) {
  const fmoba_cache_attn_args &a = p.c.a;
  const bool lds = p.c.cols <= kGateCols;
  const dim3 grid = lds ? dim3(p.row_blocks, a.heads, a.batch) : dim3(p.gates);
  const size_t bytes = ((size_t)p.c.cols + (lds ? (size_t)kTileRows * 2 * gate_stride(p.c.cols) : 0)) * 4;
  int page_bits = 1;
  while ((1 << page_bits) < p.c.cols) ++page_bits;
  auto kern = lds ? cache_gate_kernel<T, HD, true> : cache_gate_kernel<T, HD, false>;
  if (int rc = with_lds(kern, bytes, "cache_gate")) return rc;
  // whole calls (with one product a weight in the columns), us with one wave, two, four: 64 pages 270, 274, 293; 256 pages 124, 121, 127; 512 188, 169, 164; 1024 395, 320, 286
  const int waves = p.c.cols <= 64 ? 1 : p.c.cols <= 320 ? 2 : 4;
  hipLaunchKernelGGL(kern, grid, dim3(64 * waves), bytes, s, p, page_bits);
  FMOBA_LAUNCH_CHECK("cache_gate_kernel");
  return 0;
}
template <typename T, typename H, int HD, int KT, bool ONE>
static int launch_columns_as(const ColumnPlan &p, int held, hipStream_t s) {
  auto kern = cache_columns_kernel<T, H, HD, KT, ONE>;
  const size_t bytes = (size_t)held * HD * 4;
  if (int rc = with_lds(kern, bytes, "cache_columns")) return rc;
  const int64_t grid = (int64_t)p.c.a.batch * p.c.a.cache.heads_k * p.c.cols * p.steps * p.parts;
  hipLaunchKernelGGL(kern, dim3((uint32_t)grid), dim3(256), bytes, s, p, held);
  FMOBA_LAUNCH_CHECK("cache_columns_kernel");
  return 0;
}
template <typename T, typename H, int HD>
static int launch_columns(const ColumnPlan &p, hipStream_t s) {
  const int P = p.c.a.cache.page_size;
  if constexpr (HD <= 128) {
    if (p.step_keys == 128) return launch_columns_as<T, H, HD, 128, true>(p, 128, s);
  }
  if (p.step_keys == 64) return launch_columns_as<T, H, HD, 64, true>(p, 64, s);
  return launch_columns_as<T, H, HD, 64, false>(p, P * HD * 4 <= 64 * 1024 ? P : 64, s);
}
template <typename T, int LPR>
static void launch_combine(const ColumnPlan &p, hipStream_t s) {
  const int64_t pairs = (int64_t)p.c.a.total_q * p.c.a.heads;
  // Rows of a workgroup: fewer where there are few, more spare the weights' atomics.  Whole calls (with one product a weight in the columns), us with 16, 32, 64, 128 rows, heads of 128 without weights and with: 2048 pairs 35, 38, 44, 56
  // and 40, 42, 50, 64; 8192 49, 51, 56, 68 and 62, 59, 61, 75; 32768 78, 76, 80, 87 and 117, 99, 91, 96; 131056 219, 213, 212, 213 and 277, 243, 229, 225.
  const int rows = std::max(pairs <= 4096 ? 16 : pairs <= 16384 ? 32 : 64, 256 / LPR);
  const dim3 grid(ceil_div(p.c.a.total_q, rows), p.c.a.heads);
  if (p.c.a.add_weight)
    hipLaunchKernelGGL((cache_combine_kernel<T, LPR, true>), grid, dim3(256), 0, s, p, rows);
  else
    hipLaunchKernelGGL((cache_combine_kernel<T, LPR, false>), grid, dim3(256), 0, s, p, rows);
}
template <typename T, int HD>
static int run_columns_hd(const ColumnPlan &p, hipStream_t s) {
  if (int rc = launch_gate<T, HD>(p, s)) return rc;
  if (int rc = p.c.a.cache.format == FMOBA_CACHE_E4M3 ? launch_columns<T, HeldE4M3, HD>(p, s) : launch_columns<T, HeldInt8, HD>(p, s)) return rc;
  launch_combine<T, HD / 8>(p, s);
  FMOBA_LAUNCH_CHECK("cache_combine_kernel");
  return 0;
}
template <typename T>
static int run_columns_as(const ColumnPlan &p, hipStream_t s) {
  const int D = p.c.a.cache.head_dim;
  return D <= 64 ? run_columns_hd<T, 64>(p, s) : D <= 128 ? run_columns_hd<T, 128>(p, s) : run_columns_hd<T, 256>(p, s);
}

int run_cache_columns(const CacheAttn &c, hipStream_t s) {
  const fmoba_cache_attn_args &a = c.a;
  ColumnPlan p{};
  p.c = c;
  const ColumnSizes z = column_sizes(a, c.cols, p);
  uint8_t *at = reinterpret_cast<uint8_t *>(a.workspace);
  p.sel = reinterpret_cast<int32_t *>(at), at += z.sel;
  p.bits = reinterpret_cast<uint32_t *>(at), at += z.bits;
  p.scores = reinterpret_cast<float *>(at), at += z.scores;
  p.head = reinterpret_cast<float2 *>(at), at += z.head;
  p.part = reinterpret_cast<uint16_t *>(at);
  return a.cache.dtype == FMOBA_DTYPE_BF16 ? run_columns_as<bf16_t>(p, s) : run_columns_as<f16_t>(p, s);
}

}  // namespace fmoba
