// kv_ops.h — operators on a paged key/value pool in device memory: the session's own pool
// or the caller's (the yar_kv_* entry points). Launchers run on `st` of the current device.
#pragma once
#include "engine.h"

namespace yar {

// Bits of the device error word that these operators set (include/yue2ar.h).
constexpr int kKvBadPage = 1, kKvBadLength = 2, kKvBadOffsets = 4, kKvExpired = 64;
// A session's word has bits of its own (1 to 64): there these stand this many places higher, so
// that "device error flags 256" is a bad page, 512 a bad length and 16384 a wait that ran out.
constexpr int kKvSessionShift = 8;
constexpr int kKvMaxGroup = 16;          // query heads of one KV head
constexpr int kKvMaxPages = 1 << 20;     // pages of a pool that can be compacted
constexpr int kKvMaxPositions = 1 << 30;  // positions of one page table

// A pool [layer][page][k | v][kv_head][page_tokens][head_dim].
struct KvPool {
  bf16 *data = nullptr;
  int layers = 0, pages = 0, kv_heads = 0, page_tokens = 0, page_shift = 0, head_dim = 0;
  size_t page_elems() const { return size_t(2) * kv_heads * page_tokens * head_dim; }  // K and V of one page
};

// One attention call. A query sees the cached positions j <= p (p: its own position) with
// window == 0, or j < sinks, or j > p - window.
struct KvAttnParams {
  const bf16 *kv = nullptr;  // the layer's first page
  int pages = 0, heads = 0, kv_heads = 0, page_shift = 0;
  size_t page_elems = 0;
  const int *table = nullptr;  // [rows][table_stride], pages_per_row entries of each row
  long long table_stride = 0;
  int rows = 0, pages_per_row = 0;
  const int *lengths = nullptr;  // [rows] cached positions (null: `length` for the one row)
  int length = 0;
  const int *offsets = nullptr;  // prefill: [rows + 1] query offsets (null: one row holds them all)
  int n_queries = 0;
  const bf16 *q = nullptr;
  long long q_stride = 0;
  bf16 *out = nullptr;
  long long out_stride = 0;
  int window = 0, sinks = 0;
  float scale = 1.f;
  int max_length = 0;  // decode: a bound of the lengths, for the choice of splits only (0: the table's)
  float *partials = nullptr;  // decode: workspace of kv_attn_decode_workspace bytes (may be null)
  int *error = nullptr;
  int error_shift = 0;  // places by which the bits stand higher there
};

size_t kv_attn_decode_workspace(int heads, int kv_heads, int head_dim);
void launch_kv_attn_decode(const KvAttnParams &p, int head_dim, cudaStream_t st);
// `pool`: the whole pool (the tensor map covers it); p.kv lies in it.
void launch_kv_attn_prefill(const KvPool &pool, int layer, const KvAttnParams &p, cudaStream_t st);

// Pages src[i] of `from` to dst[i] of `to` (host arrays), the first tokens[i] positions
// (null: all) of every layer, K and V. The pools differ in their number of pages at most.
void launch_kv_copy_pages(const KvPool &from, const KvPool &to, const int32_t *src, const int32_t *dst,
                          const int32_t *tokens, int n, cudaStream_t st);
// Compaction (include/yue2ar.h yar_kv_compact).
void launch_kv_compact(const KvPool &pool, const int *table, long long table_stride, int rows, int pages_per_row,
                       const int *counts, int *new_table, long long new_stride, int *remap, int *used, int *work,
                       int *error, cudaStream_t st);
void configure_kv_attn_kernels();
void configure_kv_prefill_kernels();
void configure_kv_kernels();

}  // namespace yar
