// kernels_kv_attn.cu — attention of single tokens over a paged cache: softmax(scale q K^T) V of
// the visible positions, zeros for a row that sees nothing.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "kv_launch.cuh"
#include "kv_ops.h"

namespace yar {

// q [rows][heads][D], one query per row and head.
//
// A query row of a KV head's group reads each cached K and V value once for the whole
// group, so the kernel is bound by HBM: 2 x 2 x D bytes per position and KV head. The work
// of one (row, kv head) is split over a thread-block cluster of C blocks (a power of two up
// to 16), the parts joined through distributed shared memory: no partials in global memory,
// no counters, nothing to clear between calls. Large clusters leave SMs unused (of 16 blocks
// with an SM each, 7 run at once), so a few long rows are split into as many parts as there
// are SMs instead, given a workspace, and joined by a second kernel.
//
// Each of a block's warps takes 8 KB at a time (a slice: 16 positions of 128 dims, or 32 of 64, whose
// two tiles of 16 take their steps side by side: 25 rows of up to 7,192 positions 77 -> 59 us, 33
// of up to 1,505 12.0 -> 10.5) through its own ring of cp.async copies (16 bytes a lane, any page
// size; rows that are not visible or whose page is bad arrive as zeros), so no barrier separates
// the warps until their states are joined. Per slice, on mma.m16n8k16 (BF16 in, FP32 out), with
// the group's queries as the eight columns (two column tiles for groups of more than eight):
//   S [keys x 8] = K q^T, D / 16 products for each 16;
//   m = max(m, S), P = 2^(S scale log2(e) - m), l += P in FP32;
//   O^T [D x 8] += V^T P, with P as two BF16 parts (P keeps 16 bits, so the result's error
//   is its own rounding): P's fragment is transposed in registers (movmatrix).
// The tensor and issue work per slice is well below the time in which HBM delivers its 8 KB to
// an SM (issue slots 40 % busy at 6.2 TB/s), which is why the plain mma.sync form suffices.
// Measured (calls in a graph on inputs in turn, which overlap as far as their launches let them): 64
// rows with 2,052 visible positions 81 us (524 MB, 6.5 TB/s); one row of 24,000 positions 23 us with
// a workspace, 29 without (98 MB, 15 us at a plain copy's rate: the start of the launch, the table's
// round trip and the join are the rest; a launch of its own for the join, 2 us, because a last part
// that joins would need a counter that is zero before a call, and a workspace may hold anything); one
// row of 513 positions 5.9 us, of 16 4.4; 33 rows of 14 heads of 64 on pages of 16, 9.3 us.
namespace {
constexpr int kDecMaxCluster = 16;
constexpr int dec_slice(int head_dim) { return 2048 / head_dim; }  // positions of a slice: its K and V are 8 KB

// W warps of a block: 8, one block per SM (192 KB of rings), or 4, two blocks per SM.
template <int D, int W>
struct DecCfg {
  static constexpr int kThreads = 32 * W;
  static constexpr int kSlice = dec_slice(D);
  static constexpr int kStage = 2 * kSlice * D * 2;  // bytes of one slice: K, then V
  static constexpr int kStages = 3;                  // ring depth of a warp
  static constexpr int kRing = W * kStages * kStage;
};

__device__ __forceinline__ uint32_t kv_smem(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// 16 bytes to shared memory; `ok` false: zeros, nothing read.
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 2^x by the PTX approximate base-2 exponential (relative error below 2^-22; 2^-inf = 0).
__device__ __forceinline__ float kv_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
// This block's shared memory address `a` as seen in block `rank` of the cluster.
__device__ __forceinline__ float ld_cluster(uint32_t a, uint32_t rank) {
  uint32_t r;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}

// Grid (C, kv_heads, rows), clusters of C blocks along x. NT: column tiles (groups of up to
// 8 NT heads).
template <int D, int NT, int W>
__global__ void __launch_bounds__(32 * W, 8 / W) k_kv_attn_decode(const __grid_constant__ KvAttnParams p) {
  using Cfg = DecCfg<D, W>;
  // mma steps, 16-byte chunks of a row, columns; positions of a slice, and mma tiles of them.
  constexpr int KS = D / 16, CPR = D / 8, Q = 8 * NT, SL = Cfg::kSlice, KT = SL / 16;
  extern __shared__ __align__(128) unsigned char ring[];
  // After the loop the ring's space holds the warps' outputs, [warp][Q][D] FP32.
  static_assert(W * Q * D * 4 <= Cfg::kRing, "the warps' outputs fit the ring");
  __shared__ float wml[W][Q][2];  // a warp's (m, l)
  __shared__ float part_ml[Q][2];         // the block's
  __shared__ float part_o[Q * D];         // the block's output, scaled to its m
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = gridDim.x, rank = blockIdx.x, kvh = blockIdx.y, row = blockIdx.z, G = p.heads / p.kv_heads;
  kv_overlap();

  const int P = 1 << p.page_shift, cap = p.pages_per_row << p.page_shift;
  const int *tab = p.table + size_t(row) * p.table_stride;
  // The table comes into the L2 while the length, which says where to look in it, is on its way (8.2
  // -> 7.9 us for 18 rows that see 185 positions): its first 2,048 entries, since a table may be far
  // wider than what its rows hold (one row of 100 positions in a table of 2^24 pages: 9 us, 271 with all).
  if (warp == 0)
    for (int i = lane * 32; i < min(p.pages_per_row, 2048); i += 1024)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(tab + i));
  int len = p.lengths[row];
  if (len > cap) {
    if (rank == 0 && kvh == 0 && tid == 0 && p.error) atomicOr(p.error, kKvBadLength << p.error_shift);
    len = cap;
  }
  // The visible positions in order: [0, sinks), then [lo, len).
  const int lo = p.window ? max(0, len - p.window) : 0, sinks = p.window ? min(p.sinks, lo) : 0;
  const int seen = len > 0 ? sinks + len - lo : 0;
  // Slices of this block: a contiguous share; warp w takes every W-th.
  const int slices = (seen + SL - 1) / SL, per = (slices + C - 1) / C;
  const int s0 = min(slices, rank * per), s1 = min(slices, s0 + per);
  const int n = max(0, (s1 - s0 - warp + W - 1) / W);  // this warp's slices

  // Lane l looks after key l % SL of a slice: its page-table entry (-1: no key),
  // loaded two slices before the copies that need it.
  auto entry_of = [&](int i) {
    const int v = (s0 + warp + i * W) * SL + lane % SL;
    if (i >= n || v >= seen) return -1;
    const int e = tab[(v < sinks ? v : lo + v - sinks) >> p.page_shift];
    return e < 0 || e >= p.pages ? -2 : e;
  };
  bool bad = false;  // an entry outside the pool (reported at the end)
  const uint32_t my_ring = kv_smem(ring) + warp * Cfg::kStages * Cfg::kStage;
  constexpr int RPI = 32 / CPR;  // rows that one warp-wide copy covers
  const int cr = lane / CPR, cc = lane % CPR;
  const char *head_base = reinterpret_cast<const char *>(p.kv) + size_t(kvh) * P * D * 2 + cc * 16;
  const size_t v_off = p.page_elems;  // bytes from a K row to its V row: page_elems / 2 values
  // Copy slice i into ring stage i % kStages; `page` as entry_of(i) gave it. Returns the keys
  // that are there, a bit each.
  auto issue = [&](int i, int page) -> uint32_t {
    bad |= page == -2;
    if (i < n) {
      const uint32_t st = my_ring + (i % Cfg::kStages) * Cfg::kStage;
      const int v0 = (s0 + warp + i * W) * SL;
#pragma unroll
      for (int r0 = 0; r0 < SL; r0 += RPI) {
        const int r = r0 + cr, pg = __shfl_sync(0xFFFFFFFFu, page, r), v = v0 + r;
        const int j = v < sinks ? v : lo + v - sinks;
        const bool ok = pg >= 0;
        const char *src = head_base + (ok ? size_t(pg) * p.page_elems * 2 + size_t(j & (P - 1)) * (D * 2) : 0);
        const uint32_t dst = st + r * (D * 2) + ((cc ^ (r & 7)) << 4);
        cp16(dst, src, ok);
        cp16(dst + SL * D * 2, src + v_off, ok);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    return __ballot_sync(0xFFFFFFFFu, page >= 0);
  };
  constexpr int S = Cfg::kStages;
  int pages[S + 1];
#pragma unroll
  for (int i = 0; i < S + 1; ++i) pages[i] = entry_of(i);
  int page_a = pages[S - 1], page_b = pages[S];
  uint32_t valid[S - 1];  // the keys of the slices in flight
#pragma unroll
  for (int i = 0; i < S - 1; ++i) valid[i] = issue(i, pages[i]);

  // The group's queries as B fragments: column lane / 4, dims 2 (lane % 4) and + 8 of each 16.
  uint32_t bq[NT][KS][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int h = 8 * t + (lane >> 2);
    const bf16 *qr = p.q + size_t(row) * p.q_stride + size_t(kvh * G + min(h, G - 1)) * D + 2 * (lane & 3);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      bq[t][k][0] = h < G ? *reinterpret_cast<const uint32_t *>(qr + 16 * k) : 0u;
      bq[t][k][1] = h < G ? *reinterpret_cast<const uint32_t *>(qr + 16 * k + 8) : 0u;
    }
  }
  const float sl2 = p.scale * 1.4426950408889634f;
  float m[NT][2], l[NT][2], o[NT][KS][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) o[t][k][0] = o[t][k][1] = o[t][k][2] = o[t][k][3] = 0.f;
  }
  const int kr = lane & 15, kc = lane >> 4;                               // K: row, chunk of the pair
  const int vr = (lane & 7) + ((lane >> 4) << 3), vc = (lane >> 3) & 1;   // V, transposed

  for (int i = 0; i < n; ++i) {
    // Refill the stage that slice i - 1 left.
    const uint32_t ahead = issue(i + S - 1, page_a);
    page_a = page_b;
    page_b = entry_of(i + S + 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
    __syncwarp();
    const uint32_t st = my_ring + (i % S) * Cfg::kStage, ok = valid[0];
#pragma unroll
    for (int k = 0; k + 2 < S; ++k) valid[k] = valid[k + 1];
    valid[S - 2] = ahead;

    float s[NT][KT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < KT; ++x) s[t][x][0] = s[t][x][1] = s[t][x][2] = s[t][x][3] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int x = 0; x < KT; ++x) {
        uint32_t a[4];
        ldsm4(a, st + (16 * x + kr) * (D * 2) + (((2 * k + kc) ^ (kr & 7)) << 4));
#pragma unroll
        for (int t = 0; t < NT; ++t) mma16816(s[t][x], a, bq[t][k][0], bq[t][k][1]);
      }
    uint32_t ph[NT][KT][2], pl[NT][KT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (ok != 0xFFFFFFFFu) {
#pragma unroll
        for (int x = 0; x < KT; ++x) {
          const bool in0 = (ok >> (16 * x + (lane >> 2))) & 1u, in1 = (ok >> (16 * x + (lane >> 2) + 8)) & 1u;
          s[t][x][0] = in0 ? s[t][x][0] : -INFINITY, s[t][x][1] = in0 ? s[t][x][1] : -INFINITY;
          s[t][x][2] = in1 ? s[t][x][2] : -INFINITY, s[t][x][3] = in1 ? s[t][x][3] : -INFINITY;
        }
      }
      float mn[2] = {fmaxf(s[t][0][0], s[t][0][2]), fmaxf(s[t][0][1], s[t][0][3])};
#pragma unroll
      for (int x = 1; x < KT; ++x) {
        mn[0] = fmaxf(mn[0], fmaxf(s[t][x][0], s[t][x][2]));
        mn[1] = fmaxf(mn[1], fmaxf(s[t][x][1], s[t][x][3]));
      }
      mn[0] *= sl2, mn[1] *= sl2;
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        mn[0] = fmaxf(mn[0], __shfl_xor_sync(0xFFFFFFFFu, mn[0], x));
        mn[1] = fmaxf(mn[1], __shfl_xor_sync(0xFFFFFFFFu, mn[1], x));
      }
      mn[0] = fmaxf(mn[0], m[t][0]), mn[1] = fmaxf(mn[1], m[t][1]);
      if (__any_sync(0xFFFFFFFFu, mn[0] > m[t][0] || mn[1] > m[t][1])) {
        // 0 when m was -inf, and 1 while it still is (no position seen).
        const float a0 = mn[0] == m[t][0] ? 1.f : kv_ex2(m[t][0] - mn[0]);
        const float a1 = mn[1] == m[t][1] ? 1.f : kv_ex2(m[t][1] - mn[1]);
        l[t][0] *= a0, l[t][1] *= a1;
#pragma unroll
        for (int k = 0; k < KS; ++k) o[t][k][0] *= a0, o[t][k][1] *= a1, o[t][k][2] *= a0, o[t][k][3] *= a1;
        m[t][0] = mn[0], m[t][1] = mn[1];
      }
      const float n0 = m[t][0] == -INFINITY ? 0.f : -m[t][0], n1 = m[t][1] == -INFINITY ? 0.f : -m[t][1];
#pragma unroll
      for (int x = 0; x < KT; ++x) {
        const float e0 = kv_ex2(fmaf(s[t][x][0], sl2, n0)), e1 = kv_ex2(fmaf(s[t][x][1], sl2, n1));
        const float e2 = kv_ex2(fmaf(s[t][x][2], sl2, n0)), e3 = kv_ex2(fmaf(s[t][x][3], sl2, n1));
        l[t][0] += e0 + e2, l[t][1] += e1 + e3;
        const uint32_t h0 = pack2(e0, e1), h1 = pack2(e2, e3);
        ph[t][x][0] = transpose8(h0), ph[t][x][1] = transpose8(h1);
        pl[t][x][0] = transpose8(pack2(e0 - bf_lo(h0), e1 - bf_hi(h0)));
        pl[t][x][1] = transpose8(pack2(e2 - bf_lo(h1), e3 - bf_hi(h1)));
      }
    }
#pragma unroll
    for (int x = 0; x < KT; ++x)
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t a[4];
        ldsm4t(a, st + SL * D * 2 + (16 * x + vr) * (D * 2) + (((2 * k + vc) ^ (vr & 7)) << 4));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          mma16816(o[t][k], a, ph[t][x][0], ph[t][x][1]);
          mma16816(o[t][k], a, pl[t][x][0], pl[t][x][1]);
        }
      }
    __syncwarp();
  }

  if (bad && p.error) atomicOr(p.error, kKvBadPage << p.error_shift);
  // Join the warps, then the cluster's blocks: each state weighted by 2^(m - M).
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // every warp is done with its ring
  float *wo = reinterpret_cast<float *>(ring);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float v = l[t][c];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, x);
      const int col = 8 * t + 2 * (lane & 3) + c;
      if (lane < 4) wml[warp][col][0] = m[t][c], wml[warp][col][1] = v;
      if (col < G) {
        float *dst = wo + (warp * Q + col) * D + (lane >> 2);
#pragma unroll
        for (int k = 0; k < KS; ++k) dst[16 * k] = o[t][k][c], dst[16 * k + 8] = o[t][k][c + 2];
      }
    }
  }
  __syncthreads();
  bf16 *out = p.out + size_t(row) * p.out_stride + size_t(kvh) * G * D;
  for (int e = tid; e < G * D; e += Cfg::kThreads) {
    const int h = e / D;
    float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, wml[w][h][0]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (wml[w][h][1] == 0.f) continue;  // saw nothing (a sum that is NaN goes on)
      const float a = wml[w][h][0] == M ? 1.f : kv_ex2(wml[w][h][0] - M);
      L += a * wml[w][h][1];
      O += a * wo[(w * Q + h) * D + e % D];
    }
    if (C == 1) {
      out[e] = f2bf(L == 0.f ? 0.f : O / L);
    } else if (p.partials) {
      float *dst = p.partials + ((size_t(row) * p.heads + kvh * G + h) * C + rank) * (D + 2);
      dst[2 + e % D] = O;
      if (e % D == 0) dst[0] = M, dst[1] = L;
    } else {
      part_o[e] = O;
      if (e % D == 0) part_ml[h][0] = M, part_ml[h][1] = L;
    }
  }
  if (C == 1 || p.partials) return;
  cluster_sync();
  const uint32_t ml = kv_smem(part_ml), po = kv_smem(part_o);
  for (int e = rank * Cfg::kThreads + tid; e < G * D; e += C * Cfg::kThreads) {
    const int h = e / D;
    // Every load is issued before any is used: one round trip.
    float mv[kDecMaxCluster], lv[kDecMaxCluster], ov[kDecMaxCluster], M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int c = 0; c < kDecMaxCluster; ++c) {
      mv[c] = -INFINITY, lv[c] = ov[c] = 0.f;
      if (c < C) {
        mv[c] = ld_cluster(ml + h * 8, c);
        lv[c] = ld_cluster(ml + h * 8 + 4, c);
        ov[c] = ld_cluster(po + e * 4, c);
      }
    }
#pragma unroll
    for (int c = 0; c < kDecMaxCluster; ++c) M = fmaxf(M, mv[c]);
#pragma unroll
    for (int c = 0; c < kDecMaxCluster; ++c) {
      if (lv[c] == 0.f) continue;
      const float a = mv[c] == M ? 1.f : kv_ex2(mv[c] - M);
      L += a * lv[c];
      O += a * ov[c];
    }
    out[e] = f2bf(L == 0.f ? 0.f : O / L);
  }
  cluster_sync();  // no block leaves while another reads its part
}

// Grid (heads, rows), one thread per dim: the parts' states [row][head][parts][D + 2] (m, l,
// o) joined as the cluster's blocks are.
template <int D>
__global__ void __launch_bounds__(D) k_kv_attn_join(const __grid_constant__ KvAttnParams p, int parts) {
  const int h = blockIdx.x, row = blockIdx.y, d = threadIdx.x;
  kv_overlap();
  const float *src = p.partials + (size_t(row) * p.heads + h) * parts * (D + 2);
  constexpr int B = 8;  // parts read in one round trip
  float M = -INFINITY, L = 0.f, O = 0.f;
  for (int c0 = 0; c0 < parts; c0 += B) {
    float mv[B], lv[B], ov[B], Mn = M;
#pragma unroll
    for (int c = 0; c < B; ++c) {
      mv[c] = -INFINITY, lv[c] = ov[c] = 0.f;
      if (c0 + c < parts) {
        const float *s = src + (c0 + c) * (D + 2);
        mv[c] = s[0], lv[c] = s[1], ov[c] = s[2 + d];
      }
    }
#pragma unroll
    for (int c = 0; c < B; ++c) Mn = fmaxf(Mn, mv[c]);
    const float r = M == Mn ? 1.f : kv_ex2(M - Mn);
    L *= r, O *= r, M = Mn;
#pragma unroll
    for (int c = 0; c < B; ++c) {
      if (lv[c] == 0.f) continue;
      const float a = mv[c] == M ? 1.f : kv_ex2(mv[c] - M);
      L += a * lv[c], O += a * ov[c];
    }
  }
  p.out[size_t(row) * p.out_stride + size_t(h) * D + d] = f2bf(L == 0.f ? 0.f : O / L);
}

// `split` blocks per (row, kv head): a cluster, or (p.partials) parts for k_kv_attn_join.
template <int D, int NT, int W>
void decode_launch(const KvAttnParams &p, int split, cudaStream_t st) {
  kv_launch(k_kv_attn_decode<D, NT, W>, dim3(split, p.kv_heads, p.rows), 32 * W, DecCfg<D, W>::kRing,
            p.partials ? 1 : split, st, p);
  if (p.partials) kv_launch(k_kv_attn_join<D>, dim3(p.heads, p.rows), D, 0, 1, st, p, split);
}

template <int D, int NT, int W>
void decode_configure() {
  const auto k = k_kv_attn_decode<D, NT, W>;
  YAR_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, DecCfg<D, W>::kRing));
  YAR_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
}

template <int D, int NT>
void decode_pick(const KvAttnParams &p, int split, int warps, cudaStream_t st) {
  warps == 4 ? decode_launch<D, NT, 4>(p, split, st) : decode_launch<D, NT, 8>(p, split, st);
}

// Blocks of clusters of 2^i that run at once (the occupancy query's answers on this part:
// large clusters leave SMs of a GPC unused).
constexpr int kSlots4[5] = {296, 296, 284, 264, 224}, kSlots8[5] = {148, 148, 132, 120, 112};
}  // namespace

size_t kv_attn_decode_workspace(int heads, int kv_heads, int head_dim) {
  return size_t(kSlots8[0]) * (heads / kv_heads) * (head_dim + 2) * sizeof(float);
}

void launch_kv_attn_decode(const KvAttnParams &p, int head_dim, cudaStream_t st) {
  const long long cap = (long long)p.pages_per_row << p.page_shift;
  long long most = p.max_length > 0 ? std::min<long long>(p.max_length, cap) : cap;
  if (p.window) most = std::min<long long>(most, (long long)p.window + p.sinks);
  const long long units = (long long)p.rows * p.kv_heads, slices = (most + dec_slice(head_dim) - 1) / dec_slice(head_dim);
  // The form with the smallest estimated time in us: `split` blocks per unit, a block streaming
  // at most at the rate that was measured (four warps 45 GB/s, 33 where two share an SM; eight 66),
  // all of them at HBM's; ~3.5 us to start and end a launch (3.7 with eight warps), 1.3 more to
  // join a cluster (1.8 of 16 blocks), 2 for the join kernel, 2.5 for each further wave of clusters
  // (their blocks start together). The host does not know the lengths: the estimate is the mean of
  // two, for rows of one length (a last wave that is not full counts half) and for ragged ones (0.55 of
  // the longest at the mean: the longest unit's blocks, or all bytes). Measured, 128 dims, both
  // kinds: 152 units of 4,000 positions 66 and 55 us with four warps, 80 and 42 with eight, 72 and
  // 42 split in four; 400 units of 3,000: 115 and 74 with four warps, 100 and 68 with eight.
  const double bytes = 2.0 * dec_slice(head_dim) * head_dim * 2;
  int split = 1, warps = 4;
  bool parts = false;
  double best = 1e30;
  auto consider = [&](int w, int c, int slots, double fixed) {
    const double blocks = double(units) * c, at_once = std::min(blocks, double(slots));
    const bool shared = w == 4 && blocks > kSlots8[0];
    const double mine = double((slices + c - 1) / c) * bytes, more = blocks / slots;
    const double waves = std::max(1.0, 0.5 * (more + std::ceil(more)));
    const double even = waves * mine / std::min(w == 8 ? 66e3 : shared ? 33e3 : 45e3, 6500e3 / at_once);
    const double ragged = std::max(mine / (w == 8 ? 66e3 : shared ? 39e3 : 45e3), 0.55 * units * slices * bytes / 6500e3);
    const double t = fixed + 0.5 * (even + ragged) + (c > 1 && more > 1 ? 1.25 * (waves + more) : 0.0);
    if (t >= best) return false;
    best = t, split = c, warps = w;
    return true;
  };
  for (int i = 0; i < 5; ++i) {
    const double fixed = i == 0 ? 3.5 : i < 4 ? 4.8 : 5.3;
    consider(4, 1 << i, kSlots4[i], fixed);
    if (i < 4) consider(8, 1 << i, kSlots8[i], fixed + 0.2);  // (16 blocks of eight warps: half as many run)
  }
  if (p.partials && 2 * units <= kSlots8[0])
    parts = consider(8, int(kSlots8[0] / units), kSlots8[0], 5.5);
  KvAttnParams d = p;
  if (!parts) d.partials = nullptr;
  const int group = p.heads / p.kv_heads;
  if (head_dim == 128)
    group <= 8 ? decode_pick<128, 1>(d, split, warps, st) : decode_pick<128, 2>(d, split, warps, st);
  else
    group <= 8 ? decode_pick<64, 1>(d, split, warps, st) : decode_pick<64, 2>(d, split, warps, st);
}

void configure_kv_attn_kernels() {
  decode_configure<128, 1, 4>();
  decode_configure<128, 2, 4>();
  decode_configure<64, 1, 4>();
  decode_configure<64, 2, 4>();
  decode_configure<128, 1, 8>();
  decode_configure<128, 2, 8>();
  decode_configure<64, 1, 8>();
  decode_configure<64, 2, 8>();
}

}  // namespace yar
