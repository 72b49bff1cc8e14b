// kv_ops.cpp — the operators on a paged key/value pool in the caller's device memory: the
// argument checks of the yar_kv_* entry points, and their launches on the caller's stream.
// Nothing here allocates or waits.
#include "kv_ops.h"

#include <algorithm>
#include <cmath>
#include <mutex>
#include <string>
#include <vector>

#include "yue2ar.h"

namespace yar {

namespace {
void need(bool ok, const std::string &msg) {
  if (!ok) throw Error("ValueError", msg);
}

struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int device) {
    YAR_CUDA(cudaGetDevice(&prev));
    if (prev != device) YAR_CUDA(cudaSetDevice(device));
  }
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
  DeviceGuard(const DeviceGuard &) = delete;
  DeviceGuard &operator=(const DeviceGuard &) = delete;
};

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

KvPool checked_pool(const ::yar_kv_pool *c) {
  need(c && c->data, "the pool and its data are required");
  need(aligned(c->data, 16), "the pool must start on a 16-byte boundary");
  need(c->layers >= 1 && c->layers <= 4096 && c->pages >= 1 && c->kv_heads >= 1 && c->kv_heads <= 1024,
       "pool layers must be in [1, 4096], pages positive, kv_heads in [1, 1024]");
  need(c->page_tokens >= 16 && c->page_tokens <= 4096 && (c->page_tokens & (c->page_tokens - 1)) == 0,
       "page_tokens must be a power of two in [16, 4096]");
  need(c->head_dim == 64 || c->head_dim == 128, "head_dim must be 64 or 128");
  // Cached rows (one head's K or V of one position) are counted in 31 bits: 128 bytes each
  // at least, so 256 GiB.
  const double rows = 2.0 * c->layers * double(c->pages) * c->kv_heads * c->page_tokens;
  need(rows < 2147483648.0, "the pool holds more than 2**31 cached rows");
  KvPool p;
  p.data = static_cast<bf16 *>(c->data);
  p.layers = c->layers;
  p.pages = c->pages;
  p.kv_heads = c->kv_heads;
  p.page_tokens = c->page_tokens;
  while ((1 << p.page_shift) < p.page_tokens) ++p.page_shift;
  p.head_dim = c->head_dim;
  return p;
}

void check_table(const KvPool &p, const int32_t *table, int64_t stride, int rows, int pages_per_row) {
  need(rows >= 0 && rows <= 65535, "rows must be in [0, 65535]");
  need(pages_per_row >= 1 && (long long)pages_per_row * p.page_tokens <= kKvMaxPositions,
       "pages_per_row must be positive and a row's table at most 2**30 positions");
  need(stride >= pages_per_row, "the page table's stride must be at least pages_per_row");
  need(rows == 0 || (table && aligned(table, 4)), "the page table is required");
}

// Whether the entries of two tables of one shape share memory (rows of one stride may lie in each
// other's gaps; of two strides that cross, true).
bool tables_overlap(const int32_t *a, int64_t a_stride, const int32_t *b, int64_t b_stride, int rows, int per) {
  if (rows == 0) return false;
  const int64_t d = (reinterpret_cast<intptr_t>(b) - reinterpret_cast<intptr_t>(a)) / int64_t(sizeof(int32_t));
  if (d >= (rows - 1) * a_stride + per || -d >= (rows - 1) * b_stride + per) return false;
  if (a_stride != b_stride) return true;
  const int64_t off = (d % a_stride + a_stride) % a_stride;  // of b's rows in a's
  return off < per || off > a_stride - per;
}

// The one device that holds every listed pointer (null ones are skipped).
int device_of(std::initializer_list<std::pair<const char *, const void *>> ptrs) {
  int device = -1;
  for (const auto &[name, p] : ptrs) {
    if (!p) continue;
    cudaPointerAttributes a;
    YAR_CUDA(cudaPointerGetAttributes(&a, p));
    need(a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged,
         std::string(name) + " must be device memory");
    if (device < 0) device = a.device;
    need(a.device == device, std::string(name) + " is on another device than the pool");
  }
  return device;
}

// Kernel attributes are set once per device.
void configure_device(int device) {
  static std::mutex lock;
  static std::vector<char> done;
  std::lock_guard<std::mutex> hold(lock);
  if (device >= int(done.size())) done.resize(size_t(device) + 1, 0);
  if (done[size_t(device)]) return;
  configure_kv_kernels();
  done[size_t(device)] = 1;
}

KvAttnParams attn_params(const KvPool &pool, const ::yar_kv_attn &c) {
  const ::yar_kv_rows *rows = &c.rows;
  const int layer = c.layer, heads = c.heads, window = c.window, sinks = c.sinks;
  const int64_t q_stride = c.q_stride, out_stride = c.out_stride;
  const void *q = c.q;
  void *out = c.out;
  const double scale = c.scale;
  int32_t *error = c.error;
  need(layer >= 0 && layer < pool.layers, "layer outside the pool");
  check_table(pool, rows->page_table, rows->table_stride, rows->rows, rows->pages_per_row);
  need(rows->rows == 0 || (rows->lengths && aligned(rows->lengths, 4)), "lengths is required");
  need(heads >= 1 && heads % pool.kv_heads == 0 && heads / pool.kv_heads <= kKvMaxGroup,
       "heads must be a multiple of kv_heads, at most 16 for each");
  need(aligned(q, 16) && aligned(out, 16) && q_stride % 8 == 0 && out_stride % 8 == 0,
       "q and out must start on 16-byte boundaries, their strides be multiples of 8");
  const int64_t width = int64_t(heads) * pool.head_dim;
  need(q_stride >= width && out_stride >= width, "q and out strides must hold heads x head_dim values");
  need(window >= 0 && sinks >= 0, "window and sinks must not be negative");
  need(std::isfinite(scale) && scale > 0 && float(scale) > 0 && std::isfinite(float(scale)),
       "scale must be positive and finite");
  need(aligned(error, 4), "error must be a 4-byte aligned word");
  KvAttnParams p;
  p.kv = pool.data + size_t(layer) * pool.pages * pool.page_elems();
  p.pages = pool.pages;
  p.heads = heads;
  p.kv_heads = pool.kv_heads;
  p.page_shift = pool.page_shift;
  p.page_elems = pool.page_elems();
  p.table = rows->page_table;
  p.table_stride = rows->table_stride;
  p.rows = rows->rows;
  p.pages_per_row = rows->pages_per_row;
  p.lengths = rows->lengths;
  p.q = static_cast<const bf16 *>(q);
  p.q_stride = q_stride;
  p.out = static_cast<bf16 *>(out);
  p.out_stride = out_stride;
  p.window = std::min(window, kKvMaxPositions - 1);  // (no row holds more: position arithmetic stays in 32 bits)
  p.sinks = std::min(sinks, kKvMaxPositions - 1);
  p.scale = float(scale);
  p.error = error;
  return p;
}
}  // namespace

void kv_attn_decode(const ::yar_kv_attn *call, int max_length, void *workspace, int64_t workspace_bytes,
                    cudaStream_t st) {
  need(call, "the call's record is required");
  const KvPool pool = checked_pool(&call->pool);
  KvAttnParams p = attn_params(pool, *call);
  need(max_length >= 0, "max_length must not be negative");
  need(workspace_bytes >= 0 && (workspace || workspace_bytes == 0) && aligned(workspace, 4),
       "workspace must be a 4-byte aligned buffer of workspace_bytes (or NULL and 0)");
  p.max_length = max_length;
  if (workspace && size_t(workspace_bytes) >= kv_attn_decode_workspace(p.heads, pool.kv_heads, pool.head_dim))
    p.partials = static_cast<float *>(workspace);
  if (p.rows == 0) return;
  need(p.q && p.out, "q and out are required");
  const int device = device_of({{"the pool", pool.data}, {"the page table", p.table}, {"lengths", p.lengths}, {"q", p.q},
                                {"out", p.out}, {"workspace", workspace}, {"error", p.error}});
  DeviceGuard guard(device);
  configure_device(device);
  launch_kv_attn_decode(p, pool.head_dim, st);
}

void kv_attn_prefill(const ::yar_kv_attn *call, const int32_t *offsets, int64_t n_queries, cudaStream_t st) {
  need(call, "the call's record is required");
  const KvPool pool = checked_pool(&call->pool);
  KvAttnParams p = attn_params(pool, *call);
  need(n_queries >= 0 && n_queries <= kKvMaxPositions, "n_queries must be in [0, 2**30]");
  if (p.rows == 0 || n_queries == 0) return;
  need(p.q && p.out && offsets && aligned(offsets, 4), "q, out and offsets are required");
  p.offsets = offsets;
  p.n_queries = int(n_queries);
  const int device = device_of({{"the pool", pool.data}, {"the page table", p.table}, {"lengths", p.lengths},
                                {"offsets", offsets}, {"q", p.q}, {"out", p.out}, {"error", p.error}});
  DeviceGuard guard(device);
  configure_device(device);
  launch_kv_attn_prefill(pool, call->layer, p, st);
}

void kv_copy_pages(const ::yar_kv_pool *c_from, const ::yar_kv_pool *c_to, const int32_t *src, const int32_t *dst,
                   const int32_t *tokens, int n, cudaStream_t st) {
  const KvPool from = checked_pool(c_from), to = checked_pool(c_to);
  need(from.layers == to.layers && from.kv_heads == to.kv_heads && from.page_tokens == to.page_tokens &&
           from.head_dim == to.head_dim,
       "the pools must have the same layers, kv_heads, page_tokens and head_dim");
  need(n >= 0 && (n == 0 || (src && dst)), "the source and destination pages are required");
  const bool same = from.data == to.data;
  if (same) need(from.pages == to.pages, "one pool cannot have two page counts");
  // A destination is written once and is no source of the same call, so the copies may run
  // in any order.
  std::vector<char> written(size_t(to.pages), 0);
  for (int i = 0; i < n; ++i) {
    need(src[i] >= 0 && src[i] < from.pages && dst[i] >= 0 && dst[i] < to.pages, "page outside the pool");
    need(!tokens || (tokens[i] >= 0 && tokens[i] <= from.page_tokens), "tokens must be in [0, page_tokens]");
    need(!written[size_t(dst[i])], "a page is the destination of two copies");
    written[size_t(dst[i])] = 1;
  }
  if (same)
    for (int i = 0; i < n; ++i) need(!written[size_t(src[i])], "a destination page is also a source");
  if (n == 0) return;
  if (!same) {
    const char *a = reinterpret_cast<const char *>(from.data), *b = reinterpret_cast<const char *>(to.data);
    const size_t na = size_t(from.layers) * from.pages * from.page_elems() * sizeof(bf16);
    const size_t nb = size_t(to.layers) * to.pages * to.page_elems() * sizeof(bf16);
    need(a + na <= b || b + nb <= a, "the pools overlap");
  }
  const int device = device_of({{"the source pool", from.data}, {"the destination pool", to.data}});
  DeviceGuard guard(device);
  configure_device(device);
  launch_kv_copy_pages(from, to, src, dst, tokens, n, st);
}

void kv_compact(const ::yar_kv_pool *c_pool, const int32_t *table, int64_t table_stride, int rows, int pages_per_row,
                const int32_t *counts, int32_t *new_table, int64_t new_stride, int32_t *remap, int32_t *used,
                int32_t *work, int32_t *error, cudaStream_t st) {
  const KvPool pool = checked_pool(c_pool);
  check_table(pool, table, table_stride, rows, pages_per_row);
  check_table(pool, new_table, new_stride, rows, pages_per_row);
  need(pool.pages <= kKvMaxPages, "a pool of more than 2**20 pages cannot be compacted");
  need(rows == 0 || (counts && aligned(counts, 4)), "counts is required");
  need(remap && used && work && aligned(remap, 4) && aligned(used, 4) && aligned(work, 4) && aligned(error, 4),
       "remap, used and work are required, 4-byte aligned");
  if (table != new_table || table_stride != new_stride)
    need(!tables_overlap(table, table_stride, new_table, new_stride, rows, pages_per_row),
         "the new table overlaps the old one: pass the same one, or another");
  const int device = device_of({{"the pool", pool.data}, {"the page table", table}, {"counts", counts},
                                {"the new table", new_table}, {"remap", remap}, {"used", used}, {"work", work},
                                {"error", error}});
  DeviceGuard guard(device);
  configure_device(device);
  launch_kv_compact(pool, table, table_stride, rows, pages_per_row, counts, new_table, new_stride, remap, used, work,
                    error, st);
}

}  // namespace yar
