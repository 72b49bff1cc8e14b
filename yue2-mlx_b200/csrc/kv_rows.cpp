// kv_rows.cpp — a session's rows as lists of cache pages: forks that share the parent's full
// pages, rows cut back, pages behind a sliding window given back, the pool compacted. The page
// lists and their reference counts live on the host (every change happens between steps); the
// kernels see the tables that upload_row writes.
#include <algorithm>
#include <string>

#include "engine.h"
#include "kv_ops.h"

namespace yar {

const char *const kPagesExhausted = "KV page pool exhausted; generation was not shortened";

namespace {
void drop_page(Session &s, int page) {
  if (page >= 0 && --s.page_refs[page] == 0) s.free_pages.push_back(page);
}

KvPool session_pool(const Session &s) {
  KvPool p;
  p.data = s.kv;
  p.layers = s.m->d.layers;
  p.pages = s.num_pages;
  p.kv_heads = s.m->d.kv_heads;
  p.page_tokens = s.page_tokens;
  while ((1 << p.page_shift) < p.page_tokens) ++p.page_shift;
  p.head_dim = s.m->d.head_dim;
  return p;
}

void begin(Session &s) {
  YAR_CUDA(cudaSetDevice(s.m->device));
  YAR_CUDA(cudaStreamSynchronize(s.stream));
}
}  // namespace

int take_page(Session &s) {
  const int page = s.free_pages.back();
  s.free_pages.pop_back();
  s.page_refs[page] = 1;
  return page;
}

void drop_pages(Session &s, int row) {
  for (int p : s.row_pages[row]) drop_page(s, p);
  s.row_pages[row].clear();
}

int pages_for(const Session &s, int capacity) { return (capacity + s.page_tokens - 1) / s.page_tokens; }

int pages_after_drop(const Session &s, int row, int rows) {
  std::vector<int> theirs(s.num_pages, 0);  // of a page's references
  int n = int(s.free_pages.size());
  for (int r = row; r < row + rows; ++r)
    for (int p : s.row_pages[r]) n += p >= 0 && ++theirs[p] == s.page_refs[p];
  return n;
}

void upload_row(Session &s, int row) {
  // Entries without a page are never read; 0 keeps every entry inside the pool.
  std::vector<int> table(s.pages_per_row, 0);
  for (size_t i = 0; i < s.row_pages[row].size(); ++i) table[i] = std::max(0, s.row_pages[row][i]);
  YAR_CUDA(cudaMemcpyAsync(s.d_page_table + size_t(row) * s.pages_per_row, table.data(), table.size() * sizeof(int),
                           cudaMemcpyHostToDevice, s.stream));
  const int zero = 0;
  YAR_CUDA(cudaMemcpyAsync(s.d_pos + row, &s.pos[row], sizeof(int), cudaMemcpyHostToDevice, s.stream));
  YAR_CUDA(cudaMemcpyAsync(s.d_capacity + row, &s.capacity[row], sizeof(int), cudaMemcpyHostToDevice, s.stream));
  YAR_CUDA(cudaMemcpyAsync(s.d_active + row, &zero, sizeof(int), cudaMemcpyHostToDevice, s.stream));
  YAR_CUDA(cudaStreamSynchronize(s.stream));
}

void row_fork(Session &s, int src, int dst, int capacity) {
  check_row(s, src);
  check_row(s, dst);
  if (src == dst) throw Error("ValueError", "a row cannot be forked onto itself");
  const int P = s.page_tokens, n = s.pos[src];
  if (s.row_pages[src].empty()) throw Error("ValueError", "the source row holds no cache");
  if (capacity < 1 || capacity > s.max_ctx || capacity < n)
    throw Error("ValueError", "KV cache capacity must be in [" + std::to_string(std::max(1, n)) + ", " +
                                  std::to_string(s.max_ctx) + "]");
  begin(s);
  const int full = n / P, need = pages_for(s, capacity);
  if (pages_after_drop(s, dst) < need - full) throw Error("ValueError", kPagesExhausted);
  drop_pages(s, dst);
  std::vector<int> pages(s.row_pages[src].begin(), s.row_pages[src].begin() + full);
  for (int p : pages)
    if (p >= 0) ++s.page_refs[p];
  while (int(pages.size()) < need) pages.push_back(take_page(s));
  s.row_pages[dst] = pages;
  s.pos[dst] = n;
  s.capacity[dst] = capacity;
  if (n % P) {  // the page that is part full: both rows go on writing into it
    const int32_t from = s.row_pages[src][full], to = pages[full], tokens = n % P;
    launch_kv_copy_pages(session_pool(s), session_pool(s), &from, &to, &tokens, 1, s.stream);
  }
  YAR_CUDA(cudaMemcpyAsync(s.logits + size_t(dst) * s.logit_stride, s.logits + size_t(src) * s.logit_stride,
                           size_t(s.logit_stride) * sizeof(bf16), cudaMemcpyDeviceToDevice, s.stream));
  upload_row(s, dst);
}

void row_truncate(Session &s, int row, int n) {
  check_row(s, row);
  if (n < 0 || n > s.pos[row]) throw Error("ValueError", "a row can be cut back to [0, its position] only");
  if (s.row_pages[row].empty()) throw Error("ValueError", "the row holds no cache");
  begin(s);
  const int P = s.page_tokens;
  std::vector<int> &pages = s.row_pages[row];
  // What the next query, at position n, sees has to be there still.
  for (size_t i = 0; i < pages.size() && int(i) * P < n; ++i) {
    const int a = int(i) * P, b = std::min(n, a + P);
    if (pages[i] < 0 && (s.attn_window == 0 || a < s.attn_sinks || b - 1 > n - s.attn_window))
      throw Error("ValueError", "positions that the row would see again have been released");
  }
  // (A window of one position sees none of them; the page would count as whole from then on.)
  if (n % P && pages[size_t(n / P)] < 0)
    throw Error("ValueError", "the page that the row would go on in has been released");
  // Pages to be written from now on must be the row's own: shared ones are replaced (the one
  // that n falls into keeps its first n % P positions).
  int fresh = 0;
  for (size_t i = size_t(n / P); i < pages.size(); ++i) fresh += pages[i] < 0 || s.page_refs[pages[i]] > 1;
  if (int(s.free_pages.size()) < fresh) throw Error("ValueError", kPagesExhausted);
  for (size_t i = size_t(n / P); i < pages.size(); ++i) {
    const int old = pages[i];
    if (old >= 0 && s.page_refs[old] == 1) continue;
    pages[i] = take_page(s);
    if (old >= 0) {
      if (int(i) == n / P && n % P) {
        const int32_t from = old, to = pages[i], tokens = n % P;
        launch_kv_copy_pages(session_pool(s), session_pool(s), &from, &to, &tokens, 1, s.stream);
      }
      drop_page(s, old);
    }
  }
  s.pos[row] = n;
  upload_row(s, row);
}

void row_free(Session &s, int row) {
  check_row(s, row);
  begin(s);
  drop_pages(s, row);
  s.pos[row] = 0;
  s.capacity[row] = 0;
  upload_row(s, row);
}

int row_release(Session &s, int row) {
  check_row(s, row);
  if (s.attn_window == 0) throw Error("ValueError", "the session has no sliding window");
  begin(s);
  int released = 0;
  std::vector<int> &pages = s.row_pages[row];
  // The query at the row's position sees j < sinks and j > position - window; later ones less.
  for (size_t i = 0; i < pages.size(); ++i) {
    const long long a = (long long)(i) * s.page_tokens, last = a + s.page_tokens - 1;
    if (pages[i] < 0 || a < s.attn_sinks || last > (long long)s.pos[row] - s.attn_window) continue;
    drop_page(s, pages[i]);
    pages[i] = -1;
    ++released;
  }
  if (released) upload_row(s, row);
  return released;
}

int session_compact(Session &s) {
  begin(s);
  const int rows = s.max_rows, per = s.pages_per_row;
  std::vector<int> table(size_t(rows) * per, -1), counts(rows);
  for (int r = 0; r < rows; ++r) {
    counts[r] = int(s.row_pages[r].size());
    std::copy(s.row_pages[r].begin(), s.row_pages[r].end(), table.begin() + size_t(r) * per);
  }
  // table, counts, remap, used, work
  const size_t ints = table.size() + rows + size_t(s.num_pages) + 1 + 1 + 2 * size_t(s.num_pages);
  int *d = nullptr;
  YAR_CUDA(cudaMalloc(&d, ints * sizeof(int)));
  std::vector<int> remap(s.num_pages);
  int used = 0;
  try {
    int *d_counts = d + table.size(), *d_remap = d_counts + rows, *d_used = d_remap + s.num_pages, *d_work = d_used + 1;
    YAR_CUDA(cudaMemcpyAsync(d, table.data(), table.size() * sizeof(int), cudaMemcpyHostToDevice, s.stream));
    YAR_CUDA(cudaMemcpyAsync(d_counts, counts.data(), rows * sizeof(int), cudaMemcpyHostToDevice, s.stream));
    launch_kv_compact(session_pool(s), d, per, rows, per, d_counts, d, per, d_remap, d_used, d_work, nullptr, s.stream);
    YAR_CUDA(cudaMemcpyAsync(remap.data(), d_remap, remap.size() * sizeof(int), cudaMemcpyDeviceToHost, s.stream));
    YAR_CUDA(cudaMemcpyAsync(&used, d_used, sizeof(int), cudaMemcpyDeviceToHost, s.stream));
    YAR_CUDA(cudaStreamSynchronize(s.stream));
  } catch (...) {
    cudaFree(d);
    throw;
  }
  cudaFree(d);
  std::vector<int> refs(s.num_pages, 0);
  for (int p = 0; p < s.num_pages; ++p)
    if (remap[p] >= 0) refs[remap[p]] = s.page_refs[p];
  s.page_refs = refs;
  s.free_pages.clear();
  for (int p = s.num_pages - 1; p >= used; --p) s.free_pages.push_back(p);
  for (int r = 0; r < rows; ++r) {
    for (int &p : s.row_pages[r])
      if (p >= 0) p = remap[p];
    upload_row(s, r);
  }
  return used;
}

void session_set_window(Session &s, int window, int sinks) {
  if (window < 0 || sinks < 0 || window > s.max_ctx || sinks > s.max_ctx)
    throw Error("ValueError", "window and sinks must be in [0, " + std::to_string(s.max_ctx) + "]");
  if (s.m->tp_world > 1) throw Error("ValueError", "a sliding window needs a model on one GPU");
  if (window == 0) sinks = 0;
  // Rows whose pages were released behind the window cannot see more than they did. (Whether this row at
  // this position would is not asked: the answer would change from step to step.)
  const bool wider = window == 0 || window > s.attn_window || sinks > s.attn_sinks;
  if (s.attn_window > 0 && wider)
    for (const auto &pages : s.row_pages)
      if (std::find(pages.begin(), pages.end(), -1) != pages.end())
        throw Error("ValueError", "a row has released pages that a wider window would need: reset or free it first");
  begin(s);
  for (auto &g : s.graphs) cudaGraphExecDestroy(g.exec);  // graphs captured the old window
  s.graphs.clear();
  s.attn_window = window;
  s.attn_sinks = sinks;
}

}  // namespace yar
