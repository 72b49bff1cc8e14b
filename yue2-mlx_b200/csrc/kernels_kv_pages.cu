// kernels_kv_pages.cu — copies of cache pages, and compaction: the used pages of a pool
// moved to its front with the page tables rewritten.
//
// Both move bytes and nothing else, so both are bound by HBM (each byte read once and
// written once): a block moves a contiguous run with eight 16-byte loads a thread in flight.
// Measured: 63 pages of 28 layers (1.85 GB) 579 us = 6.39 TB/s, 98% of the measured copy
// rate; a compaction that moves 1.15 GB 371 us = 94% captured, 370 to 400 called (one more launch,
// for the plan, and the host's four tensors); one part of a page (15 MB) 7.2 us, two of them the launch.
#include <algorithm>

#include "common.cuh"
#include "kv_launch.cuh"
#include "kv_ops.h"

namespace yar {

namespace {
constexpr int kCopyThreads = 256, kCopyPairs = 256;

struct CopyPagesParams {
  const bf16 *src;
  bf16 *dst;
  long long src_layer, dst_layer;  // elements of one layer
  int page_tokens, head_dim, runs;  // runs: 2 * kv_heads (K and V of each head) per page
  int from[kCopyPairs], to[kCopyPairs], tokens[kCopyPairs];
};
static_assert(sizeof(CopyPagesParams) <= 4096, "kernel parameters must fit the 4 KB launch limit");

// 16-byte words [0, n) of src to dst with the block's threads, eight loads in flight each.
__device__ __forceinline__ void copy_words(const uint4 *src, uint4 *dst, int n) {
  int i = threadIdx.x;
  for (; i + 7 * kCopyThreads < n; i += 8 * kCopyThreads) {
    uint4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = ldg_stream(src + i + k * kCopyThreads);
#pragma unroll
    for (int k = 0; k < 8; ++k) dst[i + k * kCopyThreads] = v[k];
  }
  for (; i < n; i += kCopyThreads) dst[i] = ldg_stream(src + i);
}

// Grid (run, layer, pair): a run is one head's K or V positions of a page, contiguous.
__global__ void __launch_bounds__(kCopyThreads) k_kv_copy_pages(const __grid_constant__ CopyPagesParams p) {
  kv_overlap();
  const int pair = blockIdx.z;
  const size_t run = size_t(p.page_tokens) * p.head_dim, page = run * p.runs;
  const bf16 *s = p.src + blockIdx.y * p.src_layer + p.from[pair] * page + blockIdx.x * run;
  bf16 *d = p.dst + blockIdx.y * p.dst_layer + p.to[pair] * page + blockIdx.x * run;
  copy_words(reinterpret_cast<const uint4 *>(s), reinterpret_cast<uint4 *>(d), p.tokens[pair] * p.head_dim / 8);
}

// ---- compaction ------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

struct CompactParams {
  bf16 *pool;
  int layers, pages, page_words;  // 16-byte words of one (layer, page)
  const int *table;
  long long table_stride;
  int rows, pages_per_row;
  const int *counts;
  int *new_table;
  long long new_stride;
  int *remap, *used, *work;  // work: [0] moves, then (source, destination) per move
  int *error;
};

__device__ __forceinline__ bool listed_entry(const CompactParams &p, int row, int i) {
  return i < min(p.counts[row], p.pages_per_row);
}

// One CTA: a bitmap of the used pages in shared memory, its prefix sums, and the plan. With
// U used pages, the k-th used page at or behind U goes to the k-th unused page before U, so
// no destination is a source and every move can run at once.
__global__ void __launch_bounds__(kPlanThreads) k_kv_compact_plan(CompactParams p) {
  extern __shared__ unsigned bits[];
  __shared__ int warp_total[kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, words = (p.pages + 31) / 32;
  for (int i = tid; i < words; i += kPlanThreads) bits[i] = 0;
  kv_overlap();
  __syncthreads();
  // All entries of all rows in one pass (a row at a time would wait for each row's count).
  const long long entries = (long long)p.rows * p.pages_per_row;
  for (long long k = tid; k < entries; k += kPlanThreads) {
    const int r = int(k / p.pages_per_row), i = int(k % p.pages_per_row);
    const int n = p.counts[r], e = p.table[r * p.table_stride + i];
    if (i == 0 && p.error && (n < 0 || n > p.pages_per_row)) atomicOr(p.error, kKvBadLength);
    if (i >= n) continue;
    if (e >= 0 && e < p.pages)
      atomicOr(&bits[e >> 5], 1u << (e & 31));
    else if (e != -1 && p.error)
      atomicOr(p.error, kKvBadPage);
  }
  __syncthreads();
  // Thread t owns words [w0, w1): the used pages before its first word.
  const int per = (words + kPlanThreads - 1) / kPlanThreads, w0 = min(words, tid * per), w1 = min(words, w0 + per);
  int mine = 0;
  for (int w = w0; w < w1; ++w) mine += __popc(bits[w]);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_total[warp] = incl;
  __syncthreads();
  int before = incl - mine, total = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) before += warp_total[w];
    total += warp_total[w];
  }
  // Unused pages before U are the destinations, in order: work[2 + 2 k].
  const int base = before;
  __shared__ int s_low;  // used pages before U
  if (tid == 0) s_low = 0;
  __syncthreads();
  int low = 0;
  for (int w = w0; w < w1; ++w) {
    const int first = w * 32;
    if (first + 32 <= total)
      low += __popc(bits[w]);
    else if (first < total)
      low += __popc(bits[w] & ((1u << (total - first)) - 1u));
  }
  if (low) atomicAdd(&s_low, low);
  __syncthreads();
  const int used_low = s_low, moves = total - used_low;
  int rank = base;
  for (int w = w0; w < w1; ++w) {
    const unsigned b = bits[w];
    for (int k = 0; k < 32; ++k) {
      const int page = w * 32 + k;
      if (page >= p.pages) break;
      const bool on = (b >> k) & 1u;
      if (on) {
        p.remap[page] = page;
        if (page >= total) p.work[1 + 2 * (rank - used_low)] = page;
        ++rank;
      } else {
        p.remap[page] = -1;
        if (page < total) p.work[2 + 2 * (page - rank)] = page;
      }
    }
  }
  __syncthreads();
  for (int k = tid; k < moves; k += kPlanThreads) p.remap[p.work[1 + 2 * k]] = p.work[2 + 2 * k];
  if (tid == 0) {
    p.used[0] = total;
    p.work[0] = moves;
  }
}

// The moves (a grid-stride loop over (move, layer)) and the rewritten tables.
__global__ void __launch_bounds__(kCopyThreads) k_kv_compact_move(CompactParams p) {
  kv_overlap();  // the plan is complete
  const long long entries = (long long)p.rows * p.pages_per_row;
  for (long long i = (long long)blockIdx.x * kCopyThreads + threadIdx.x; i < entries;
       i += (long long)gridDim.x * kCopyThreads) {
    const int r = int(i / p.pages_per_row), c = int(i % p.pages_per_row);
    const int e = p.table[r * p.table_stride + c];
    p.new_table[r * p.new_stride + c] = listed_entry(p, r, c) && e >= 0 && e < p.pages ? p.remap[e] : e;
  }
  const int moves = p.work[0];
  constexpr int kPiece = 8 * kCopyThreads;  // words of one work item (16 and 32 of them: 2% slower)
  const int pieces = (p.page_words + kPiece - 1) / kPiece;
  const long long items = (long long)moves * p.layers * pieces;
  for (long long i = blockIdx.x; i < items; i += gridDim.x) {
    const int piece = int(i % pieces);
    const long long ml = i / pieces;
    const int k = int(ml % moves);
    const size_t layer = size_t(ml / moves) * p.pages * size_t(p.page_words);
    uint4 *pool = reinterpret_cast<uint4 *>(p.pool) + layer + size_t(piece) * kPiece;
    copy_words(pool + size_t(p.work[1 + 2 * k]) * p.page_words, pool + size_t(p.work[2 + 2 * k]) * p.page_words,
               min(kPiece, p.page_words - piece * kPiece));
  }
}
}  // namespace

void launch_kv_copy_pages(const KvPool &from, const KvPool &to, const int32_t *src, const int32_t *dst,
                          const int32_t *tokens, int n, cudaStream_t st) {
  CopyPagesParams p;
  p.src = from.data;
  p.dst = to.data;
  p.page_tokens = from.page_tokens;
  p.head_dim = from.head_dim;
  p.runs = 2 * from.kv_heads;
  p.src_layer = (long long)(from.pages * from.page_elems());
  p.dst_layer = (long long)(to.pages * to.page_elems());
  for (int i0 = 0; i0 < n; i0 += kCopyPairs) {
    const int k = std::min(kCopyPairs, n - i0);
    for (int i = 0; i < k; ++i) {
      p.from[i] = src[i0 + i];
      p.to[i] = dst[i0 + i];
      p.tokens[i] = tokens ? tokens[i0 + i] : from.page_tokens;
    }
    kv_launch(k_kv_copy_pages, dim3(p.runs, from.layers, k), kCopyThreads, 0, 1, st, p);
  }
}

void launch_kv_compact(const KvPool &pool, const int *table, long long table_stride, int rows, int pages_per_row,
                       const int *counts, int *new_table, long long new_stride, int *remap, int *used, int *work,
                       int *error, cudaStream_t st) {
  CompactParams p;
  p.pool = pool.data;
  p.layers = pool.layers;
  p.pages = pool.pages;
  p.page_words = int(pool.page_elems() / 8);
  p.table = table;
  p.table_stride = table_stride;
  p.rows = rows;
  p.pages_per_row = pages_per_row;
  p.counts = counts;
  p.new_table = new_table;
  p.new_stride = new_stride;
  p.remap = remap;
  p.used = used;
  p.work = work;
  p.error = error;
  kv_launch(k_kv_compact_plan, 1, kPlanThreads, size_t((pool.pages + 31) / 32) * 4, 1, st, p);
  kv_launch(k_kv_compact_move, 148 * 8, kCopyThreads, 0, 1, st, p);  // eight blocks fill an SM's threads
}

void configure_kv_kernels() {
  configure_kv_attn_kernels();
  configure_kv_prefill_kernels();
  YAR_CUDA(cudaFuncSetAttribute(k_kv_compact_plan, cudaFuncAttributeMaxDynamicSharedMemorySize, kKvMaxPages / 8));
}

}  // namespace yar
