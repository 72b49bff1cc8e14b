// kernels_kv_attn.cu — attention over a paged cache: softmax(scale q K^T) V of the visible
// positions, zeros for a query that sees nothing.
#include "common.cuh"
#include "kv_ops.h"

namespace yar {

namespace {
// One warp per (query, query head), 32 keys a pass: a lane's key for the scores, a lane's
// dims for the sum over V.
template <int D>
__global__ void __launch_bounds__(256) k_kv_attn_simple(KvAttnParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * 8 + warp;
  if (unit >= (long long)p.n_queries * p.heads) return;
  const int token = int(unit / p.heads), head = int(unit % p.heads), kvh = head / (p.heads / p.kv_heads);
  int row = 0, first = 0, n = 1;
  if (p.offsets) {
    for (row = 0; row < p.rows; ++row) {
      first = p.offsets[row], n = p.offsets[row + 1] - first;
      if (first < 0 || n < 0 || p.offsets[row + 1] > p.n_queries) {
        if (lane == 0 && p.error) atomicOr(p.error, kKvBadOffsets);
        continue;
      }
      if (token >= first && token < first + n) break;
    }
    if (row == p.rows) return;  // behind the last row's queries: left as it was
  } else if (p.lengths) {
    row = token, first = token;
  } else {
    n = p.n_queries;
  }
  const int cap = p.pages_per_row << p.page_shift, P = 1 << p.page_shift;
  int len = p.lengths ? p.lengths[row] : p.length;
  if (len > cap) {
    if (lane == 0 && p.error) atomicOr(p.error, kKvBadLength);
    len = cap;
  }
  const int pos = len - n + (token - first);
  const int lo = p.window ? max(0, pos - p.window + 1) : 0, sinks = p.window ? min(p.sinks, lo) : 0;
  const int seen = pos < 0 ? 0 : sinks + pos - lo + 1;
  const bf16 *q = p.q + size_t(token) * p.q_stride + size_t(head) * D;
  const int *tab = p.table + size_t(row) * p.table_stride;
  float m = -INFINITY, l = 0.f, o[D / 32] = {};
  for (int c = 0; c < seen; c += 32) {
    const int v = c + lane, j = v < sinks ? v : lo + v - sinks;
    const bf16 *kr = nullptr;
    if (v < seen) {
      const int page = tab[j >> p.page_shift];
      if (page >= 0 && page < p.pages)
        kr = p.kv + size_t(page) * p.page_elems + (size_t(kvh) * P + (j & (P - 1))) * D;
      else if (p.error)
        atomicOr(p.error, kKvBadPage);
    }
    float s = -INFINITY;
    if (kr) {
      s = 0.f;
      for (int d = 0; d < D; ++d) s += bf2f(q[d]) * bf2f(kr[d]);
      s *= p.scale;
    }
    const float mn = fmaxf(m, warp_max(s));
    if (mn == -INFINITY) continue;
    const float a = expf(m - mn), e = kr ? expf(s - mn) : 0.f;
    l = l * a + warp_sum(e);
    m = mn;
    for (int i = 0; i < D / 32; ++i) o[i] *= a;
    for (int k = 0; k < 32; ++k) {
      const float w = __shfl_sync(0xFFFFFFFFu, e, k);
      const unsigned long long at = __shfl_sync(0xFFFFFFFFu, (unsigned long long)kr, k);
      if (!at) continue;
      const bf16 *vr = reinterpret_cast<const bf16 *>(at) + p.page_elems / 2;
      for (int i = 0; i < D / 32; ++i) o[i] += w * bf2f(vr[lane + 32 * i]);
    }
  }
  bf16 *dst = p.out + size_t(token) * p.out_stride + size_t(head) * D;
  for (int i = 0; i < D / 32; ++i) dst[lane + 32 * i] = f2bf(l > 0.f ? o[i] / l : 0.f);
}

void simple(const KvAttnParams &p, int head_dim, cudaStream_t st) {
  const unsigned grid = unsigned(((long long)p.n_queries * p.heads + 7) / 8);
  if (grid == 0) return;
  if (head_dim == 128)
    k_kv_attn_simple<128><<<grid, 256, 0, st>>>(p);
  else
    k_kv_attn_simple<64><<<grid, 256, 0, st>>>(p);
  YAR_CUDA(cudaGetLastError());
}
}  // namespace

void launch_kv_attn_decode(const KvAttnParams &p, int head_dim, cudaStream_t st) {
  KvAttnParams d = p;
  d.n_queries = p.rows;
  simple(d, head_dim, st);
}

void launch_kv_attn_prefill(const KvPool &pool, int layer, const KvAttnParams &p, cudaStream_t st) {
  (void)layer;
  simple(p, pool.head_dim, st);
}

}  // namespace yar
