// kernels_kv_prefill.cu — causal attention of prompt chunks over a paged cache (any group of
// query heads, full or a sliding window with sinks), on the 5th-generation tensor cores.
//
// softmax(scale q K^T) V per query over the visible positions. The queries of one row and KV
// head are flattened to M rows (query-major: row m is query m / G, head m % G), so a group
// shares every K and V tile and short chunks fill their tiles. An item is 256 M rows as two
// tiles A and B of 128, which walk the 64-key tiles that any of the queries sees (the sinks'
// tiles, then the window's). A block takes the item of its own index, then those of blocks that
// have not started (a claim cancels their launch), so that one item's start hides behind another's
// end. Its warps:
//   * warp 10 finds the items and brings K and V tiles by TMA through a ring (one box per page
//     piece; pieces that nothing sees, or whose page is bad, are fetched out of bounds: zeros);
//     it claims the next item when the last copies of one are on their way;
//   * warp 11 brings Q as soon as a tile's last S is there, and looks for bad pages (groups that do
//     not divide 128 have no boxes of whole queries: the softmax warps bring their rows);
//   * one lane of warp 8 (A) and of warp 9 (B) issues the products: S = Q K^T into one of two
//     TMEM buffers of 64 columns, two key tiles ahead, and O += P V with P read from TMEM,
//     where the softmax warps left it in S's own columns;
//   * warps 0..3 (A) and 4..7 (B): a thread owns one M row (= TMEM lane). It reads its 64
//     scores, masks them (tiles on an edge only), raises its running maximum m when the tile
//     exceeds it by more than 8 (in log2 units; O in TMEM is rescaled only then: O / l is
//     the same quotient whichever m the terms share), writes P = 2^(s - m) as BF16 and adds
//     P to l in FP32; at the item's end it writes its row of O / l (32 bytes a store: rows through
//     shared memory, line by line, would keep Q's place from the next item).
// P in BF16 is off by up to 2^-8 of each weight, l is summed from the FP32 weights: at random, over
// many keys, that averages out to less than the rounding of the BF16 result; where one key carries
// the weight it is as much again (m lags by up to 8, so that weight is not a power of two). Two BF16
// parts would cost half as much tensor work again; l from the rounded weights, in which a key that
// dominates cancels, costs 3.5 % (16,384 tokens with a window: 303 -> 313 us, by mixed additions;
// 317 with the halves unpacked). Scores, m, l and O are FP32.
// Masked positions cannot leak: hidden keys' scores are replaced, V rows that nothing in the
// item sees are zeroed in shared memory, and when a tile that only some queries see holds
// a V value that is not finite (0 x inf), the tile's sums are recomputed key by key.
//
// Few blocks (a chunk of one prompt) are split along the keys over a cluster of 2 or 4, whose
// states are joined through distributed shared memory, each block finishing D / C columns.
//
// What bounds it: per 64-key step of A and B (~1,720 cycles) the tensor pipe has ~1,150 cycles
// of work (S at N = 64 reads Q again for every 64 keys: 53 cycles a product instead of 32), and
// a softmax group ~1,250, most of them exponentials; the rest is the hand-over between them. From
// one item's last P to the next one's first S ~4,500 cycles (O's division and stores 2,700).
// Measured (16 query / 8 KV heads of 128): 16,384 tokens with a window of 2,048: 270 us, 955
// TFLOP/s; 8,000 tokens without one: 234 us, 1,120; 1,024 queries over 8,192 positions: 73 us, 880
// (140 us without the split); 24 ragged rows: 121 us; 77 queries of 4 heads of 64: 8 us. With one
// item a block 302, -, 77, 147 and 10 us; items in turn with Q through registers 313 and 151 for
// the first and the ragged rows (the loads' latency stood between two items: ~10,000 cycles), by
// cp.async of the softmax warps 280 and 127. Tried and slower:
// 128-key tiles with one S buffer each (1.9 times the time, but of an early form whose products took
// their operands from a thread's registers, which alone cost more than the products; with uniform
// operands only 64 keys were measured), S and P V issued by warps
// of their own (84 us on the second case), A's and B's exponentials taking turns (151), the
// exponentials of a tile run beside the next one's maximum (182: S would have to be three
// tiles ahead), no maximum but for tiles that leave the range (146 against 139); of the form with
// items, two threads a row (294 against 270), P in columns of its own and S one tile ahead (283).
#include <cuda.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "kv_launch.cuh"
#include "kv_ops.h"
#include "tcgen05.cuh"

namespace yar {

namespace {
constexpr int kPreM = 128, kPreN = 64;  // M rows of a tile, keys of a tile
// Three warpgroups, launched with 168 registers a thread: the third (copies, products) gives
// up 96 of them and the two softmax ones take 48 each: 2 x 216 + 72 = 3 x 168.
constexpr int kPreThreads = 384, kPreRegs = 168, kPreRegsSoftmax = 216, kPreRegsIssue = 72;
static_assert(2 * kPreRegsSoftmax + kPreRegsIssue == 3 * kPreRegs, "no more registers than the launch holds");

template <int D>
struct PreCfg {
  static constexpr int kQSlice = kPreM * 128, kQ = (D / 64) * kQSlice;    // 128 rows of 64 values; a Q tile
  static constexpr int kSlice = kPreN * 128, kTile = (D / 64) * kSlice;  // the same of a K or V tile
  // A ring stage: V of tile i, then K of tile i + 2 (the products that follow P of tile i);
  // stage 0 of the walk: K of tiles 0 and 1. 160 KB in flight.
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr int kSmem = 2 * kQ + 2 * kStages * kTile + 1024;
  // kind::f16, FP32 accumulator, BF16 A and B, A K-major, N >> 3 at bit 17, M >> 4 at bit 24;
  // P V reads B (V) MN-major (bit 16).
  static constexpr uint32_t kIdescS =
      (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(kPreN >> 3) << 17) | (uint32_t(kPreM >> 4) << 24);
  static constexpr uint32_t kIdescO =
      (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (uint32_t(D >> 3) << 17) | (uint32_t(kPreM >> 4) << 24);
};
// Tensor memory: two S (and P) buffers of A at columns 0 and 64, of B at 128 and 192, O at 256, 384.
constexpr uint32_t kPreColO = 256, kPreCols = 512;
constexpr float kPreRescale = 8.f;
// Of 8 pairs of exponentials, those on the FMA units (1,024 at 7,168 unsplit: 145 us with 0, 143
// with 1, 139 with 2, 3 and 4).
constexpr int kPrePoly = 3;

struct PrefillExtra {
  int row0;        // the layer's first cached row in the pool seen as [rows][D]
  int total_rows;  // rows of the pool: the out-of-bounds coordinate
  int box_rows;    // keys of one box
  int pairs;       // upper bound of the blocks' M-row pairs
  int q_boxes;     // Q comes by TMA (its M rows are boxes of whole queries: the group divides a tile)
};

// A bounded wait (2^16 polls of up to 20 us each, not counted while a tile's rows are recomputed
// key by key) that also ends when another role gave up. state: [0] given up, [1], [2] tile A, B
// recomputes.
__device__ __forceinline__ bool pre_poll(uint64_t *bar, unsigned parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(at_smem(bar)), "r"(parity), "r"(20000u)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ bool pre_wait_slow(uint64_t *bar, unsigned parity, const volatile int *state) {
  for (int i = 0; i < 1 << 16; i += !(state[1] | state[2])) {
    if (pre_poll(bar, parity)) return true;
    if (state[0]) return false;
  }
  return false;
}
// True on every lane of the (converged) warp when the phase is over.
__device__ __forceinline__ bool pre_wait(uint64_t *bar, unsigned parity, const volatile int *state) {
  if (__all_sync(0xFFFFFFFFu, pre_poll(bar, parity))) return true;
  return __all_sync(0xFFFFFFFFu, pre_wait_slow(bar, parity, state));
}
// 2^x by the approximate base-2 exponential, results below 2^-126 as 0 (relative error below
// 2^-22): without that flush each exponential costs three more instructions.
__device__ __forceinline__ float pre_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two FP32 values in one operation (each rounded as the single one is).
__device__ __forceinline__ uint64_t pair64(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split64(uint64_t v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The largest of three; NaN when one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 2^t of two finite values t <= 100 on the FMA units (t below -125 gives 2^-125): t = n + f with f in
// [-1/2, 1/2], 2^f by the degree-4 polynomial of least maximal relative error on that interval
// (2.6e-6, Remez exchange), n added to its exponent.
__device__ __forceinline__ void exp2_poly2(uint64_t t, float &e0, float &e1) {
  float t0, t1, r0, r1, p0, p1;
  split64(t, t0, t1);
  t = pair64(fmaxf(t0, -125.f), fmaxf(t1, -125.f));
  const uint64_t big = pair64(12582912.f, 12582912.f);  // 1.5 x 2^23: the sum's last bit is one
  const uint64_t r = add2(t, big);
  const uint64_t f = fma2(add2(r, pair64(-12582912.f, -12582912.f)), pair64(-1.f, -1.f), t);
  uint64_t p = fma2(f, pair64(0.009570102207362652f, 0.009570102207362652f),
                    pair64(0.05591785907745361f, 0.05591785907745361f));
  p = fma2(f, p, pair64(0.240247443318367f, 0.240247443318367f));
  p = fma2(f, p, pair64(0.6931217908859253f, 0.6931217908859253f));
  p = fma2(f, p, pair64(0.9999992847442627f, 0.9999992847442627f));
  split64(r, r0, r1);
  split64(p, p0, p1);
  e0 = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(r0) << 23));
  e1 = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(r1) << 23));
}
// 16 columns of this warp's lanes (waited for).
__device__ __forceinline__ void ld16(uint32_t addr, float *v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];\n tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// Store 32 columns of this warp's lanes (not waited for).
__device__ __forceinline__ void st32_async(uint32_t addr, const uint32_t *v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
// Whether `mine` holds on any thread of the named barrier's group (and their barrier).
__device__ __forceinline__ bool pre_any(int barrier, bool mine) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n bar.red.or.pred p, %2, %3, q;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(r)
      : "r"(uint32_t(mine)), "r"(barrier), "n"(kPreM)
      : "memory");
  return r != 0;
}
// 16 values as BF16 to `to`: one 32-byte store, or two where only 16 bytes are aligned.
__device__ __forceinline__ void pre_store16(bf16 *to, const float *v, float scale, bool wide) {
  uint32_t w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * e] * scale, v[2 * e + 1] * scale);
    w[e] = *reinterpret_cast<const uint32_t *>(&h);
  }
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4 *>(to)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4 *>(to)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
__device__ __forceinline__ void pre_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t pre_mapa(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}

// Asks for a block of the grid that has not started, to do its work here: the answer lands in `to`
// (16 bytes) and completes `bar`.
__device__ __forceinline__ void pre_claim(void *to, uint64_t *bar) {
  asm volatile(
      "fence.proxy.async.shared::cta;\n"
      " mbarrier.arrive.expect_tx.shared::cta.b64 _, [%1], 16;\n"
      " clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(at_smem(to)),
      "r"(at_smem(bar))
      : "memory");
}
// The claimed block's index; false when none was left.
__device__ __forceinline__ bool pre_claimed(const void *from, int &bx) {
  uint32_t got, cx;
  asm volatile(
      "{\n .reg .b128 r;\n .reg .pred p;\n ld.shared.b128 r, [%2];\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n selp.u32 %0, 1, 0, p;\n mov.u32 %1, 0;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n}"
      : "=r"(got), "=r"(cx)
      : "r"(at_smem(from))
      : "memory");
  bx = int(cx);
  return got != 0;
}

// Where an item's work lies.
struct PreBlock {
  int row, first, n, len;  // the row (-1: no more items), its first query, its queries, its cached positions
  int kvh;                 // the KV head
  int q0, r0, rows;  // its first M row is head r0 (of the group) of query q0; its M rows
  int p0, p1;        // positions of its first and last query
  int kend, lo, sinks;       // keys seen by any query: [0, sinks) and [lo, kend)
  int sink_tiles, wfirst;    // key tile j: j < sink_tiles ? j : wfirst + j - sink_tiles
  int j0, j1;                // this block's share of the key tiles
};
struct PreTile {  // one of A, B
  int pmin, pmax;  // positions of its first and last row (pmax -1: it has no rows)
  int s1, w0, w1;  // the item's key tiles that it sees: [0, s1) (sinks) and [w0, w1)
  int sunk, whole0, whole1;  // of them, those that every row sees whole: [0, sunk) and [whole0, whole1)
};

template <int D>
__global__ void __launch_bounds__(kPreThreads, 1)
    k_kv_attn_prefill(const __grid_constant__ CUtensorMap map, const __grid_constant__ CUtensorMap q_map,
                      const __grid_constant__ KvAttnParams p,
                      const __grid_constant__ PrefillExtra x) {
  using Cfg = PreCfg<D>;
  constexpr int NST = Cfg::kStages;
  extern __shared__ unsigned char pre_raw[];
  unsigned char *sm = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(pre_raw) + 1023) & ~uintptr_t(1023));
  unsigned char *ring = sm + 2 * Cfg::kQ;
  __shared__ __align__(16) unsigned char claim[16];
  __shared__ __align__(8) uint64_t kv_full[NST], kv_empty[NST], s_full[2][2], p_ready[2][2], o_done[2][2], drain[2];
  __shared__ __align__(8) uint64_t item_full[2], item_empty[2], scanned[2], q_ready[2], q_free[2], claim_done;
  __shared__ PreBlock items[2];
  __shared__ PreTile tiles[2][2];
  __shared__ volatile int bad_keys[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int s_state[3];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = p.heads / p.kv_heads;
  uint32_t C, rank;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  // The copying warp sets the barriers up and goes on at once; the others also wait for the tensor memory.
  if (tid == 320) {
    for (int i = 0; i < 3; ++i) s_state[i] = 0;
    auto init = [](uint64_t *bar, int count) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(at_smem(bar)), "r"(count));
    };
    for (int s = 0; s < NST; ++s) init(&kv_full[s], 1), init(&kv_empty[s], 2);
    for (int i = 0; i < 4; ++i) {
      init(&s_full[i >> 1][i & 1], 1);
      init(&p_ready[i >> 1][i & 1], kPreM / 32);
      init(&o_done[i >> 1][i & 1], 1);
    }
    for (int i = 0; i < 2; ++i) {
      init(&drain[i], 1), init(&item_full[i], 1), init(&item_empty[i], 11), init(&scanned[i], 1);
      init(&q_ready[i], x.q_boxes ? 1 : kPreM / 32), init(&q_free[i], 1);
    }
    init(&claim_done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at_smem(&tmem_slot)),
                 "r"(kPreCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  kv_overlap();  // (nothing so far touches what the kernel before this one writes)
  if (warp == 10) {
    __syncwarp();
    asm volatile("bar.arrive 3, %0;" ::"n"(kPreThreads) : "memory");
  } else {
    asm volatile("bar.sync 3, %0;" ::"n"(kPreThreads) : "memory");
  }
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  // m / G for m < 512 and G <= 16 (the reciprocal's error, below 1, adds less than 512 / 2^16 < 1 / G).
  const int inv_g = (65536 + G - 1) / G;
  // Where M row m of an item is in q or out (by their row stride).
  auto row_at = [&](const PreBlock &b, int m, long long stride) {
    const int q = ((b.r0 + m) * inv_g) >> 16;
    return (long long)(b.first + b.q0 + q) * stride + (long long)(b.kvh * G + b.r0 + m - q * G) * D;
  };
  auto stage = [&](int it) { return ring + (it % NST) * 2 * Cfg::kTile; };  // (V of an item's tile i: it = its first + i + 1)
  const int pieces = kPreN / x.box_rows;
  auto key_tile = [](const PreBlock &b, int j) { return (j < b.sink_tiles ? j : b.wfirst + j - b.sink_tiles) * kPreN; };
  // Whether some query of the item sees a key in [k0, k1).
  auto needed = [](const PreBlock &b, int k0, int k1) { return k0 < b.kend && !(k0 >= b.sinks && k1 <= b.lo); };
  auto tile_of = [&](const PreBlock &b, int t) {
    PreTile r;
    const int nt = b.j1 - b.j0;
    const int m0 = t * kPreM, m1 = min(b.rows, m0 + kPreM) - 1, base = b.len - b.n + b.q0;
    r.pmin = base + (((b.r0 + m0) * inv_g) >> 16);
    r.pmax = m0 < b.rows ? base + (((b.r0 + m1) * inv_g) >> 16) : -1;
    // As key tiles of the row: the sinks' before `sunk`, the window's [first, last].
    const int last = r.pmax >> 6, first = p.window ? max(r.pmin - p.window + 1, 0) >> 6 : 0;
    const int sunk = p.window ? min((p.sinks + kPreN - 1) / kPreN, last + 1) : 0;
    r.s1 = max(0, min(nt, (sunk <= b.wfirst ? min(sunk, b.sink_tiles) : b.sink_tiles + sunk - b.wfirst) - b.j0));
    r.w0 = max(0, max(first, b.wfirst) - b.wfirst + b.sink_tiles - b.j0);
    r.w1 = min(nt, last + 1 - b.wfirst + b.sink_tiles - b.j0);
    const int shift = b.sink_tiles - b.wfirst - b.j0;  // a window tile's index i = its key tile + shift
    r.sunk = !p.window || r.pmin < 0 ? 0 : min(min(p.sinks, r.pmin + 1) / kPreN, b.sink_tiles) - b.j0;
    r.whole0 = !p.window || r.pmax < p.window ? b.sink_tiles - b.j0
                                              : max((r.pmax - p.window) / kPreN + 1, b.wfirst) + shift;
    r.whole1 = r.pmin < 0 ? 0 : (r.pmin + 1) / kPreN + shift;
    return r;
  };
  // Key tiles (by the item's index i) that some row of the tile sees: i < t.s1, and t.w0 <= i < t.w1.
  auto live = [](const PreTile &t, int i) { return i < t.s1 || (i >= t.w0 && i < t.w1); };
  // The block's k-th item, once it is known (false: a wait ran out); `taken` gives its place back.
  // The place of item k is refilled for k + 2 when all eleven warps have taken k.
  auto take = [&](int k) { return pre_wait(&item_full[k & 1], unsigned(k >> 1) & 1u, s_state); };
  auto taken = [&](int k) {
    __syncwarp();
    if (lane == 0) at_arrive(&item_empty[k & 1]);
  };

  // Whether there is a bad page among every step-th piece of the item's keys (its pieces are then
  // masked one by one).
  auto bad_page = [&](const PreBlock &b, int first, int step) {
    const int *tab = p.table + size_t(b.row) * p.table_stride;
    bool bad = false;
#pragma unroll 4
    for (int i = first; i < (b.j1 - b.j0) * pieces; i += step) {
      const int k0 = key_tile(b, b.j0 + i / pieces) + (i % pieces) * x.box_rows;
      if (needed(b, k0, k0 + x.box_rows)) {
        const int page = tab[k0 >> p.page_shift];
        bad = bad || page < 0 || page >= p.pages;
      }
    }
    if (bad && p.error) atomicOr(p.error, kKvBadPage << p.error_shift);
    return bad;
  };

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPreRegsIssue));
  if (warp == 10) {
    // ---- items and copies -----------------------------------------------------------------
    // The KV head, row and 256 M rows of block bx: the last pairs (the longest) of every head first, so
    // that the last blocks to start are short (4,096 tokens from nothing: 106 us head after head, 76
    // so; 8,000 282 and 234). That is longest first for one row; over a long cache, where all pairs
    // are about as long, it costs a little (5,000 queries over 8,000 cached 427 us head after head,
    // 449 so, 2,560 229 and 234), and so it does for batches of one pair a row (20 of 100 to 128
    // tokens 19.1, 19.8). False: none.
    auto find = [&](int bx, PreBlock &b) {
      const int unit = bx / int(C), slot = x.pairs - 1 - unit / p.kv_heads;
      b.kvh = unit % p.kv_heads;
      int row = -1, first = 0, n = 0, pair = 0, len = p.length;
      if (!p.offsets) {
        row = 0, n = p.n_queries, pair = slot;
        if ((long long)pair * 256 >= (long long)n * G) row = -1;
      } else {
        int before = 0, most = 0;
        bool wrong = false;
        for (int r0 = 0; r0 < p.rows && row < 0; r0 += 128) {  // four rows a lane: one latency for 128
          int f[5], k[4], l[4], mine = 0;
#pragma unroll
          for (int i = 0; i < 5; ++i) f[i] = r0 + lane * 4 + i <= p.rows ? p.offsets[r0 + lane * 4 + i] : 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) l[i] = r0 + lane * 4 + i < p.rows ? p.lengths[r0 + lane * 4 + i] : 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            k[i] = 0;
            if (r0 + lane * 4 + i < p.rows) {
              if (f[i] >= 0 && f[i + 1] >= f[i] && f[i + 1] <= p.n_queries)
                k[i] = f[i + 1] - f[i];
              else
                k[i] = -1;
            }
          }
          const bool bad = (k[0] | k[1] | k[2] | k[3]) < 0;
          if (bad && p.error) atomicOr(p.error, kKvBadOffsets << p.error_shift);
          // Behind a wrong offset rows could overlap (two blocks would write the same queries, and
          // the bound on the blocks not hold): those that start before an earlier offset are skipped.
          if (wrong || __any_sync(0xFFFFFFFFu, bad)) {
            if (!wrong) most = __shfl_sync(0xFFFFFFFFu, f[0], 0);  // (up to here they ascended)
            wrong = true;
            int top = max(max(f[0], f[1]), max(f[2], f[3]));
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const int v = __shfl_up_sync(0xFFFFFFFFu, top, o);
              if (lane >= o) top = max(top, v);
            }
            int over = __shfl_up_sync(0xFFFFFFFFu, top, 1);
            over = lane == 0 ? most : max(over, most);
            most = max(most, __shfl_sync(0xFFFFFFFFu, top, 31));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              k[i] = f[i] < over ? 0 : max(k[i], 0);
              over = max(over, f[i]);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) mine += int(((long long)k[i] * G + 255) / 256);
          int incl = mine;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
            if (lane >= o) incl += v;
          }
          const unsigned hit = __ballot_sync(0xFFFFFFFFu, slot - before < incl);
          if (hit) {
            const int src = __ffs(hit) - 1;
            int at = slot - before - (incl - mine), i = 0;  // (right on lane src)
#pragma unroll
            for (int j = 0; j < 3; ++j) {
              const int pairs = int(((long long)k[j] * G + 255) / 256);
              if (i == j && at >= pairs) at -= pairs, i = j + 1;
            }
            row = __shfl_sync(0xFFFFFFFFu, r0 + lane * 4 + i, src);
            first = __shfl_sync(0xFFFFFFFFu, i == 0 ? f[0] : i == 1 ? f[1] : i == 2 ? f[2] : f[3], src);
            n = __shfl_sync(0xFFFFFFFFu, i == 0 ? k[0] : i == 1 ? k[1] : i == 2 ? k[2] : k[3], src);
            pair = __shfl_sync(0xFFFFFFFFu, at, src);
            len = __shfl_sync(0xFFFFFFFFu, i == 0 ? l[0] : i == 1 ? l[1] : i == 2 ? l[2] : l[3], src);
          }
          before += __shfl_sync(0xFFFFFFFFu, incl, 31);
        }
      }
      if (row < 0) return false;
      b.row = row, b.first = first, b.n = n;
      const int cap = p.pages_per_row << p.page_shift;
      if (len > cap) {
        if (p.error && lane == 0) atomicOr(p.error, kKvBadLength << p.error_shift);
        len = cap;
      }
      b.len = max(len, 0);
      const long long m0 = (long long)pair * 256;
      b.rows = int(min((long long)n * G - m0, 256ll));
      b.q0 = int(m0 / G);
      b.r0 = int(m0 % G);
      b.p0 = b.len - n + b.q0;
      b.p1 = b.len - n + b.q0 + (b.r0 + b.rows - 1) / G;
      b.kend = b.p1 + 1;
      b.lo = p.window ? max(0, b.p0 - p.window + 1) : 0;
      b.sinks = p.window ? min(p.sinks, b.lo) : 0;
      b.sink_tiles = (b.sinks + kPreN - 1) / kPreN;
      b.wfirst = max(b.sink_tiles, b.lo / kPreN);
      const int total = b.kend <= 0 ? 0 : b.sink_tiles + max(0, (b.kend + kPreN - 1) / kPreN - b.wfirst);
      const int per = (total + int(C) - 1) / int(C);
      b.j0 = min(total, int(rank) * per), b.j1 = min(total, b.j0 + per);
      return true;
    };
    int bx = int(blockIdx.x), claims = 0, base = 0, issued = 0;
    bool ok = true, more = true;
    for (int k = 0; ok; ++k) {
      PreBlock b;
      while (more) {
        if (find(bx, b)) break;
        if (C > 1) {  // (a cluster's blocks share their pair)
          more = false;
          break;
        }
        if (lane == 0) pre_claim(claim, &claim_done);
        __syncwarp();
        ok = pre_wait(&claim_done, unsigned(claims++) & 1u, s_state);
        more = ok && pre_claimed(claim, bx);
      }
      if (!more) b.row = -1;
      if (!ok) break;
      if (k >= 2) ok = pre_wait(&item_empty[k & 1], unsigned((k >> 1) - 1) & 1u, s_state);
      if (!ok) break;
      if (lane == 0) {
        items[k & 1] = b;
        at_arrive(&item_full[k & 1]);
      }
      __syncwarp();
      if (!more) break;
      const int *tab = p.table + size_t(b.row) * p.table_stride;
      const int nt = b.j1 - b.j0;
      // The pool rows of the pieces' keys, a batch of 32 pieces at a time (lane l: piece l % pieces
      // of the batch's tile l / pieces), read a batch ahead: no copy waits for the page table.
      const int tpb = 32 / pieces;
      auto load_rows = [&](int batch) {
        int y = x.total_rows;  // out of bounds: zeros
        const int i = batch * tpb + lane / pieces;
        if (i < nt) {
          const int k0 = key_tile(b, b.j0 + i) + (lane % pieces) * x.box_rows;
          if (needed(b, k0, k0 + x.box_rows)) {
            const int page = tab[k0 >> p.page_shift];
            if (page >= 0 && page < p.pages)
              y = x.row0 + ((page * 2 * p.kv_heads + b.kvh) << p.page_shift) + (k0 & ((1 << p.page_shift) - 1));
          }
        }
        return y;
      };
      int rows_prev = 0, rows_cur = load_rows(0), rows_next = load_rows(1), batch = 0;
      // Tile i's K (kv = 0) or V into `dst`, this lane's piece of it.
      auto put = [&](int i, int kv, unsigned char *dst, uint64_t *bar) {
        int y = __shfl_sync(0xFFFFFFFFu, i / tpb == batch ? rows_cur : rows_prev, (i % tpb) * pieces + lane % pieces);
        if (kv && y != x.total_rows) y += p.kv_heads << p.page_shift;
        if (lane < pieces) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            asm volatile(
                "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
                "%4}], [%2];" ::"r"(at_smem(dst + c * Cfg::kSlice + lane * x.box_rows * 128)),
                "l"(&map), "r"(at_smem(bar)), "r"(c * 64), "r"(y)
                : "memory");
        }
      };
      for (int j = 0; j <= nt && nt > 0; ++j) {
        const int it = base + j, s = it % NST, i = j + 1;  // the stage's K tile (j = 0: tiles 0 and 1)
        if (it >= NST) ok = pre_wait(&kv_empty[s], unsigned(it / NST - 1) & 1u, s_state);
        if (!ok) break;
        const int tiles = j == 0 ? min(nt, 2) : 1 + (i < nt);
        if (lane == 0)
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(at_smem(&kv_full[s])),
                       "r"(tiles * Cfg::kTile)
                       : "memory");
        __syncwarp();
        issued = it + 1;
        put(j == 0 ? 0 : j - 1, j > 0, stage(it), &kv_full[s]);
        if (i < nt) {
          if (i / tpb > batch) {
            rows_prev = rows_cur, rows_cur = rows_next;
            rows_next = load_rows(++batch + 1);
          }
          put(i, 0, stage(it) + Cfg::kTile, &kv_full[s]);
        }
      }
      base = issued;
      // The next item, while the last tiles of this one wait in the ring.
      more = ok && C == 1;
      if (more) {
        if (lane == 0) pre_claim(claim, &claim_done);
        __syncwarp();
        ok = pre_wait(&claim_done, unsigned(claims++) & 1u, s_state);
        more = ok && pre_claimed(claim, bx);
      }
    }
    if (!ok) {  // leave no copy in flight
      s_state[0] = 1;
      for (int i = issued > NST ? issued - NST : 0; i < issued; ++i)
        at_wait(&kv_full[i % NST], unsigned(i / NST) & 1u);
      if (claims > 0) at_wait(&claim_done, unsigned(claims - 1) & 1u);
      if (lane == 0 && p.error) atomicOr(p.error, kKvExpired << p.error_shift);
    }
  } else if (warp < 10) {
    // ---- products of tile X = A (warp 8) or B (warp 9) ---------------------------------------
    // The loop's control values are the same on every lane; the shuffles tell the compiler so,
    // and it keeps them, and the operands made from them, in uniform registers (each tcgen05
    // operand copied from a thread's register would cost more than the product).
    auto uniform = [](int v) { return __shfl_sync(0xFFFFFFFFu, v, 0); };
    const int X = uniform(warp - 8);
    const uint32_t tm = uniform(tmem_slot + X * 128), q_lo = uniform(at_desc_lo(at_smem(sm + X * Cfg::kQ)));
    const uint32_t k_lo = uniform(at_desc_lo(at_smem(ring))), v_lo = uniform(at_desc_mn_lo(at_smem(ring), Cfg::kSlice));
    bool ok = true;
    int n_s = 0, n_p = 0;    // the tile's key tiles whose S, whose P V was issued (of all items)
    int slot = 0, ph = 0;    // the place in the ring and the parity of its use
    auto wait = [&](uint64_t *bar, int parity) {
      ok = pre_wait(bar, unsigned(parity), s_state);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    };
    auto next = [&] {
      if (++slot == NST) slot = 0, ph ^= 1;
    };
    // S of the tile's next key tile, whose K starts at descriptor k (by the elected lane).
    auto put_s = [&](uint32_t k, int n) {
      const int buf = n & 1;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
        at_mma_ss(tm + buf * 64, q_lo + (((ks >> 2) * Cfg::kQSlice) >> 4) + 2 * (ks & 3),
                  k + (((ks >> 2) * Cfg::kSlice) >> 4) + 2 * (ks & 3), Cfg::kIdescS, uint32_t(ks != 0));
      at_commit(&s_full[X][buf]);
    };
    for (int item = 0;; ++item) {
      ok = take(item);
      if (!ok) break;
      const PreBlock b = items[item & 1];
      if (uniform(b.row) < 0) break;
      wait(&scanned[item & 1], (item >> 1) & 1);
      if (!ok) break;
      const PreTile mine_t = tiles[item & 1][X];
      const PreTile tl = {0, 0, uniform(mine_t.s1), uniform(mine_t.w0), uniform(mine_t.w1), 0, 0, 0};
      const int n_tiles = uniform(b.j1 - b.j0), n_p0 = n_p;
      // Key tiles [e0, e1) and from e2 on hold V rows that nothing in the item sees.
      const int hide0 = uniform(max(0, b.sinks / kPreN - b.j0));
      const int hide1 = uniform(b.sinks < b.lo ? b.sink_tiles + (b.lo % kPreN && b.lo / kPreN >= b.sink_tiles) - b.j0 : 0);
      const int hide2 = uniform(b.kend % kPreN ? b.sink_tiles + b.kend / kPreN - b.wfirst - b.j0 : 1 << 30);
      taken(item);
      wait(&q_ready[X], item & 1);
      if (!ok) break;
      // When the tile's last S is there its Q makes room for the next item's.
      const int last_s = n_s + tl.s1 + max(0, tl.w1 - max(tl.w0, tl.s1));
      if (last_s == n_s) {
        if (at_elect()) at_arrive(&q_free[X]);
        __syncwarp();
      }
      if (n_tiles > 0) {
        wait(&kv_full[slot], ph);
        const bool on0 = live(tl, 0), on1 = n_tiles > 1 && live(tl, 1);
        if (ok && at_elect()) {
          const uint32_t k0 = k_lo + slot * (2 * Cfg::kTile >> 4);
          if (on0) put_s(k0, n_s);
          if (on1) put_s(k0 + (Cfg::kTile >> 4), n_s + on0);
          if (n_s + on0 + on1 == last_s && on0 + on1) at_commit(&q_free[X]);
          at_commit(&kv_empty[slot]);
        }
        __syncwarp();
        n_s += on0 + on1;
        next();
      }
      for (int i = 0; i < n_tiles && ok; ++i) {
        const bool on = live(tl, i), on_s = i + 2 < n_tiles && live(tl, i + 2);
        const int buf = n_p & 1;
        // The stage has landed long before P is written: both products follow P at once.
        wait(&kv_full[slot], ph);
        if (!ok) break;
        if ((i >= hide0 && i < hide1) || i >= hide2) {
          // V rows that nothing in the block sees: zeros (their P is 0, the rows may hold any
          // bits). Both tiles' warps do so, each before its own product.
          const int k0 = key_tile(b, b.j0 + i);
          unsigned char *v = ring + slot * 2 * Cfg::kTile;
          auto zero = [&](int r0, int r1) {
            for (int c = max(r0, 0) * (D / 8) + lane; c < min(r1, kPreN) * (D / 8); c += 32)
              *reinterpret_cast<uint4 *>(v + (c % (D / 8) >> 3) * Cfg::kSlice + c / (D / 8) * 128 + (c & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
          };
          zero(b.sinks - k0, b.lo - k0);
          zero(b.kend - k0, kPreN);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        const uint32_t at = slot * (2 * Cfg::kTile >> 4), acc = n_p > n_p0;
        if (on) {
          wait(&p_ready[X][buf], (n_p >> 1) & 1);
          if (!ok) break;
        }
        if (at_elect()) {
          if (on) {
#pragma unroll
            for (int ks = 0; ks < kPreN / 16; ++ks)
              at_mma_ts(tm + kPreColO, tm + buf * 64 + 8 * ks, v_lo + at + ks * (2048 >> 4), Cfg::kIdescO,
                        ks > 0 ? 1u : acc);
            at_commit(&o_done[X][buf]);
          }
          if (on_s) put_s(k_lo + at + (Cfg::kTile >> 4), n_s);
          if (on_s && n_s + 1 == last_s) at_commit(&q_free[X]);
          at_commit(&kv_empty[slot]);
        }
        __syncwarp();
        n_p += on;
        n_s += on_s;
        next();
      }
      if (!ok) break;
    }
    // Every product issued has completed before the block's tensor memory goes.
    if (at_elect()) at_commit(&drain[X]);
    __syncwarp();
    if (!at_wait(&drain[X], 0u) || !ok) {
      s_state[0] = 1;
      if (lane == 0 && p.error) atomicOr(p.error, kKvExpired << p.error_shift);
    }
  }
  if (warp == 11) {
    // ---- Q by TMA, and the next items' tables -----------------------------------------------------
    bool ok = true;
    int boxes[2] = {0, 0};  // loads of each tile's Q
    auto put_q = [&](const PreBlock &b, int k) {
#pragma unroll
      for (int X = 0; X < 2; ++X) {
        if (!ok || !x.q_boxes) break;
        if (k > 0) ok = pre_wait(&q_free[X], unsigned(k - 1) & 1u, s_state);
        if (ok && lane == 0) {
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(at_smem(&q_ready[X])), "r"(Cfg::kQ)
                       : "memory");
          // (Boxes may reach into the next row's queries, or past the last one: rows of no result.)
          for (int c = 0; c < D / 64; ++c)
            asm volatile(
                "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
                "%4, %5}], [%2];" ::"r"(at_smem(sm + X * Cfg::kQ + c * Cfg::kQSlice)),
                "l"(&q_map), "r"(at_smem(&q_ready[X])), "r"(c * 64), "r"(b.kvh * G), "r"(b.first + b.q0 + X * (kPreM / G))
                : "memory");
        }
        __syncwarp();
        boxes[X] += ok;
      }
    };
    for (int k = 0;; ++k) {
      ok = take(k);
      if (!ok || items[k & 1].row < 0) break;
      const PreBlock &b = items[k & 1];
      bool bad = false;
      if (k == 0) put_q(b, k);
      if (k > 0) bad = __any_sync(0xFFFFFFFFu, bad_page(b, lane, 32));  // (the first item's: by the softmax warps)
      if (lane < 2) tiles[k & 1][lane] = tile_of(b, lane);
      __syncwarp();
      if (lane == 0) {
        bad_keys[k & 1] = bad;
        at_arrive(&scanned[k & 1]);
      }
      __syncwarp();
      if (k > 0) put_q(b, k);
      if (!ok) break;
      taken(k);
    }
    for (int X = 0; X < 2; ++X)  // (leave no load in flight)
      if (boxes[X]) at_wait(&q_ready[X], unsigned(boxes[X] - 1) & 1u);
    if (!ok) {
      s_state[0] = 1;
      if (lane == 0 && p.error) atomicOr(p.error, kKvExpired << p.error_shift);
    }
  }
  if (C > 1) {  // (the softmax warps' two exchanges)
    pre_cluster_sync();
    pre_cluster_sync();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPreRegsSoftmax));
    // ---- softmax: the thread's M row ------------------------------------------------------
    const int wg = warp >> 2, t = tid & 127;
    const float sl2 = p.scale * 1.4426950408889634f;
    const uint32_t lanes = tmem_slot + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t col_s = lanes + wg * 128, col_o = lanes + kPreColO + wg * 128;
    // Without boxes a warp brings its 32 rows of Q itself, row by row (D / 8 lanes each: whole lines
    // of global memory), into the swizzled slices.
    auto load_q = [&](const PreBlock &b) {
      constexpr int CPR = D / 8;
#pragma unroll 4
      for (int i = 0; i < CPR; ++i) {
        const int r = (warp & 3) * 32 + (i * 32 + lane) / CPR, c = lane % CPR, m = wg * kPreM + r;
        const bf16 *src = p.q + row_at(b, min(m, b.rows - 1), p.q_stride) + c * 8;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         at_smem(sm + wg * Cfg::kQ + (c >> 3) * Cfg::kQSlice + at_sw(r, c & 7))),
                     "l"(src), "r"(m < b.rows ? 16 : 0)
                     : "memory");
      }
    };
    const bool wide = (reinterpret_cast<uintptr_t>(p.out) | uintptr_t(p.out_stride * 2)) % 32 == 0;
    bool bad = false;
    int n_s = 0, base = 0;  // the tile's key tiles so far, the item's first stage (of all items)
    // (The group's warps go on together or not at all: they share barriers.)
    bool ok = !pre_any(1 + wg, !take(0));
    bool more = ok && items[0].row >= 0;
    if (more) {
      if (!x.q_boxes) load_q(items[0]);
      bad = pre_any(1 + wg, bad_page(items[0], t, kPreM));
    }
    int syncs = 0;  // of the cluster
    for (int item = 0; more; ++item) {
      const PreBlock &b = items[item & 1];  // (stays in shared memory: the loop over the keys needs the registers)
      const int *tab = p.table + size_t(b.row) * p.table_stride;
      const int nt = b.j1 - b.j0, n_s0 = n_s;
      if (!x.q_boxes) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) at_arrive(&q_ready[wg]);
      }
      bool poison = false;
      ok = pre_wait(&scanned[item & 1], unsigned(item >> 1) & 1u, s_state);
      if (item > 0) bad = bad_keys[item & 1] != 0;
      const PreTile tl = tiles[item & 1][wg];
      // (With a bad page every tile is looked at piece by piece.)
      const int sunk = bad ? 0 : tl.sunk, whole0 = tl.whole0, whole1 = bad ? 0 : tl.whole1;
      const int pos = tid < b.rows ? max(b.len - b.n + b.q0 + (((b.r0 + tid) * inv_g) >> 16), -1) : -1;
      float row_m = -INFINITY, row_l = 0.f;  // running maximum and sum
      for (int i = 0; i < nt && ok; ++i) {
        const int j = b.j0 + i;
        if (!live(tl, i)) continue;
        const int buf = n_s & 1;
        ok = pre_wait(&s_full[wg][buf], unsigned(n_s >> 1) & 1u, s_state);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        float s[kPreN];
        at_ld64(col_s + buf * 64, s);
        const bool edge = i >= sunk && (i < whole0 || i >= whole1);
        if (edge) {
          const int k0 = key_tile(b, j);
          // Bit k: key k0 + k is visible (k <= hi, and k < sink or k > old).
          auto below = [](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; };
          unsigned long long seen = below(pos - k0 + 1);
          if (p.window) seen &= below(p.sinks - k0) | ~below(pos - p.window - k0 + 1);
          if (bad)
            for (int c = 0; c < kPreN; c += 16) {
              const int page = needed(b, k0 + c, k0 + c + 16) ? tab[(k0 + c) >> p.page_shift] : 0;
              if (page < 0 || page >= p.pages) seen &= ~(0xFFFFull << c);
            }
          const uint32_t seen_lo = uint32_t(seen), seen_hi = uint32_t(seen >> 32);
#pragma unroll
          for (int k = 0; k < kPreN; ++k)
            s[k] = ((k < 32 ? seen_lo : seen_hi) >> (k & 31)) & 1u ? s[k] : -INFINITY;
          // A V value that is not finite in a row that only some of the queries see: the product
          // with P = 0 would carry it into the others (a thread looks at half a V row).
          const int it = base + i + 1, r = t & (kPreN - 1);
          ok = pre_wait(&kv_full[it % NST], unsigned(it / NST) & 1u, s_state);
          if (!ok) break;
          if (k0 + r < b.kend && !(k0 + r >= b.sinks && k0 + r < b.lo)) {
            __nv_bfloat162 acc = __floats2bfloat162_rn(0.f, 0.f);
            const __nv_bfloat162 zero = acc;
            const unsigned char *v = stage(it) + r * 128;
#pragma unroll 2
            for (int c0 = 0; c0 < D / 16; ++c0) {
              const int c = c0 + (t >> 6) * (D / 16);
              const uint4 w = *reinterpret_cast<const uint4 *>(v + (c >> 3) * Cfg::kSlice + (c & 7) * 16);
              const uint32_t e[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int n = 0; n < 4; ++n) acc = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&e[n]), zero, acc);
            }
            const float2 f = __bfloat1622float2(acc);
            if (f.x != 0.f || f.y != 0.f) poison = true;
          }
        }
        float mx4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int k = 4; k + 8 <= kPreN; k += 8)
#pragma unroll
          for (int c = 0; c < 4; ++c) mx4[c] = max3(mx4[c], s[k + c], s[k + 4 + c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) mx4[c] = max3(mx4[c], mx4[c], s[kPreN - 4 + c]);
        const float mx = max3(max3(mx4[0], mx4[1], mx4[2]), mx4[2], mx4[3]) * sl2;
        const bool raise = mx > row_m + kPreRescale;  // false while both are -inf, and for NaN
        if (__any_sync(0xFFFFFFFFu, raise)) {
          const float c = raise ? pre_ex2(row_m - mx) : 1.f;  // 0 when m was -inf
          row_l *= c;
          row_m = raise ? mx : row_m;
          if (n_s > n_s0) {  // O, once the last P V has landed (the next one waits for this tile's P)
            ok = pre_wait(&o_done[wg][buf ^ 1], unsigned((n_s - 1) >> 1) & 1u, s_state);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int cb = 0; cb < D; cb += 32) {
              float v[32];
              at_ld32(col_o + cb, v);
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] *= c;
              at_st32(col_o + cb, v);
            }
          }
        }
        ++n_s;
        // P = 2^(s scale log2(e) - m): pairs of values in one FMA and one addition.
        const float nm = row_m == -INFINITY ? 0.f : -row_m;
        const uint64_t sl2x2 = pair64(sl2, sl2), nmx2 = pair64(nm, nm);
        uint64_t sum[2] = {0, 0};
        uint32_t w[kPreN / 2];
        auto weights = [&](auto some_poly) {
#pragma unroll
          for (int k = 0; k < kPreN / 2; ++k) {
            float e0, e1;
            const uint64_t t2 = fma2(pair64(s[2 * k], s[2 * k + 1]), sl2x2, nmx2);
            if (some_poly && k % 8 < kPrePoly) {
              exp2_poly2(t2, e0, e1);
            } else {
              split64(t2, e0, e1);
              e0 = pre_ex2(e0), e1 = pre_ex2(e1);
            }
            sum[k & 1] = add2(sum[k & 1], pair64(e0, e1));
            const __nv_bfloat162 h = __floats2bfloat162_rn(e0, e1);
            w[k] = *reinterpret_cast<const uint32_t *>(&h);
          }
        };
        // Tiles with masked scores (2^-inf has to be 0), or with infinite ones or NaN (they have to
        // stay NaN), take the exponential unit only.
        if (edge || __any_sync(0xFFFFFFFFu, !(fabsf(mx) < INFINITY)))
          weights(std::false_type{});
        else
          weights(std::true_type{});
        st32_async(col_s + buf * 64, w);
        float l0, l1;
        split64(add2(sum[0], sum[1]), l0, l1);
        row_l += l0 + l1;
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        // One arrival a warp: 32 lanes' arrivals on one barrier would take turns.
        __syncwarp();
        if (lane == 0) at_arrive(&p_ready[wg][buf]);
      }
      if (ok) ok = take(item + 1);
      more = ok && items[(item + 1) & 1].row >= 0;
      if (more && !x.q_boxes) {  // (once the item's S products are complete, which are so when it had any)
        ok = pre_wait(&q_free[wg], unsigned(item) & 1u, s_state);
        if (ok) load_q(items[(item + 1) & 1]);
      }
      if (ok && n_s > n_s0) ok = pre_wait(&o_done[wg][(n_s - 1) & 1], unsigned((n_s - 1) >> 1) & 1u, s_state);
      if (!ok) s_state[0] = 1;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // ---- the result ---------------------------------------------------------------------------
      bool failed = false;
      poison = pre_any(1 + wg, poison || !ok);
      if (poison) failed = pre_any(1 + wg, !ok);
      const bool my_row = tid < b.rows;
      bf16 *out_row = p.out + row_at(b, my_row ? tid : 0, p.out_stride);
      if (poison && !failed) {
        const bf16 *my_q = p.q + row_at(b, my_row ? tid : 0, p.q_stride);
        // Key by key with the statistics from above (V does not enter them), 32 columns at a time.
        if (t == 0) s_state[1 + wg] = 1;
        const float nm = row_m == -INFINITY ? 0.f : -row_m;
        for (int cb = 0; cb < D; cb += 32) {
          float o[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
          for (int j = b.j0; j < b.j1; ++j)
            for (int k = key_tile(b, j); k < key_tile(b, j) + kPreN; ++k) {
              if (!my_row || row_l == 0.f || k > pos || (p.window && k >= p.sinks && k <= pos - p.window)) continue;
              const int page = tab[k >> p.page_shift];
              if (page < 0 || page >= p.pages) continue;
              const bf16 *kr = p.kv + size_t(page) * p.page_elems +
                               ((size_t(b.kvh) << p.page_shift) + (k & ((1 << p.page_shift) - 1))) * D;
              float s = 0.f;
#pragma unroll 4
              for (int d = 0; d < D; ++d) s = fmaf(bf2f(my_q[d]), bf2f(kr[d]), s);
              const float e = pre_ex2(fmaf(s, sl2, nm));
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = fmaf(e, bf2f(kr[p.page_elems / 2 + cb + i]), o[i]);
            }
          __syncwarp();
          at_st32(col_o + cb, o);
        }
        pre_any(1 + wg, false);
        if (t == 0) s_state[1 + wg] = 0;
      }
      if (C == 1) {
        if (!failed) {
          const float inv = row_l == 0.f ? 0.f : 1.0f / row_l;
#pragma unroll 1
          for (int cb = 0; cb < D; cb += 32) {
            float v[32];
            at_ld32(col_o + cb, v);
            if (row_l == 0.f)  // (a row that saw nothing: O was never written)
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = 0.f;
            if (my_row)
#pragma unroll
              for (int e = 0; e < 32; e += 16) pre_store16(out_row + cb + e, v + e, inv, wide);
            __syncwarp();
          }
        }
      } else {
        // The cluster's states of a row weighted by 2^(m - M); block r finishes columns
        // [r D / C, (r + 1) D / C): the others send it theirs ([sender][4 columns][M row], 16 bytes
        // each) into its ring, which no copy or product uses any more.
        // m and l go where the tile's Q was: there is no next item, and its products are complete. A
        // tile that no key of this block's share concerns had none: its Q, which a copy brings whatever
        // the share holds, has to be there before it is written over.
        if (x.q_boxes && n_s == n_s0 && !pre_wait(&q_ready[wg], unsigned(item) & 1u, s_state)) failed = true;
        float2 *ml = reinterpret_cast<float2 *>(sm + wg * Cfg::kQ) + t;
        *ml = make_float2(row_m, row_l);
        pre_cluster_sync();
        float M = -INFINITY, L = 0.f, w = 0.f;
        {
          float mv[4], lv[4];
#pragma unroll
          for (uint32_t c = 0; c < 4; ++c) {
            mv[c] = -INFINITY, lv[c] = 0.f;
            if (c < C) {
              const uint32_t a = pre_mapa(at_smem(ml), c);
              asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(mv[c]), "=f"(lv[c]) : "r"(a) : "memory");
            }
            M = fmaxf(M, mv[c]);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (lv[c] != 0.f) L += lv[c] * (mv[c] == M ? 1.f : pre_ex2(mv[c] - M));
          w = row_l == 0.f ? 0.f : row_m == M ? 1.f : pre_ex2(row_m - M);
        }
        // (Loops of 16 columns, not unrolled: a block runs this once, and fetching the code of an
        // unrolled exchange took longer than the exchange.)
        const int cols = D / int(C), own = int(rank) * cols;
#pragma unroll 1
        for (int c16 = 0; c16 < D; c16 += 16) {
          const int r = c16 / cols;
          if (r == int(rank)) continue;
          float v[16];
          ld16(col_o + c16, v);
          const int sender = int(rank) < r ? int(rank) : int(rank) - 1;
          const uint32_t a = pre_mapa(
              at_smem(ring + ((size_t(sender) * (cols / 4) + (c16 % cols) / 4) * 256 + wg * kPreM + t) * 16), r);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a + c * 4096),
                         "f"(row_l == 0.f ? 0.f : v[4 * c] * w), "f"(row_l == 0.f ? 0.f : v[4 * c + 1] * w),
                         "f"(row_l == 0.f ? 0.f : v[4 * c + 2] * w), "f"(row_l == 0.f ? 0.f : v[4 * c + 3] * w)
                         : "memory");
        }
        pre_cluster_sync();
        syncs = 2;
        if (!failed) {
          const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll 1
          for (int c16 = 0; c16 < cols; c16 += 16) {
            float v[16];
            ld16(col_o + own + c16, v);
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = row_l == 0.f ? 0.f : v[e] * w;
            for (int s = 0; s + 1 < int(C); ++s)
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const float4 f = *reinterpret_cast<const float4 *>(
                    ring + ((size_t(s) * (cols / 4) + c16 / 4 + c) * 256 + wg * kPreM + t) * 16);
                v[4 * c] += f.x, v[4 * c + 1] += f.y, v[4 * c + 2] += f.z, v[4 * c + 3] += f.w;
              }
            if (my_row) pre_store16(out_row + own + c16, v, inv, wide);
            __syncwarp();
          }
        }
      }
      base += nt > 0 ? nt + 1 : 0;
      taken(item);
      ok = !failed;
      more = more && ok;
    }
    if (!ok) {
      s_state[0] = 1;
      if (lane == 0 && p.error) atomicOr(p.error, kKvExpired << p.error_shift);
    }
    if (C > 1 && !syncs) {  // every thread of a cluster takes its two exchanges
      pre_cluster_sync();
      pre_cluster_sync();
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_slot), "r"(kPreCols));
}

template <int D>
void prefill_launch(const CUtensorMap &map, const CUtensorMap &q_map, const KvAttnParams &p, const PrefillExtra &x, int cluster, cudaStream_t st) {
  kv_launch(k_kv_attn_prefill<D>, unsigned(x.pairs) * p.kv_heads * cluster, kPreThreads, PreCfg<D>::kSmem, cluster,
            st, map, q_map, p, x);
}
}  // namespace

void launch_kv_attn_prefill(const KvPool &pool, int layer, const KvAttnParams &p, cudaStream_t st) {
  if (p.n_queries <= 0 || p.rows <= 0) return;
  PrefillExtra x;
  const long long layer_rows = 2ll * pool.pages * pool.kv_heads * pool.page_tokens;
  x.row0 = int(layer * layer_rows);
  x.total_rows = int(pool.layers * layer_rows);
  x.box_rows = std::min(pool.page_tokens, kPreN);
  const long long G = p.heads / p.kv_heads;
  // Pairs of 256 M rows: exactly, or rounded up for each row of queries.
  const long long pairs = (p.n_queries * G + 255) / 256 + (p.offsets ? p.rows - 1 : 0);
  if (pairs * p.kv_heads > (1 << 28)) throw Error("ValueError", "too many queries for one call");
  x.pairs = int(pairs);
  CUtensorMap map;
  if (!encode_rows_map(&map, pool.data, uint64_t(x.total_rows), pool.head_dim, x.box_rows))
    throw Error("RuntimeError", "cuTensorMapEncodeTiled failed for the cache pool");
  CUtensorMap q_map = {};
  x.q_boxes = kPreM % G == 0 && encode_heads_map(&q_map, p.q, uint64_t(p.n_queries), p.heads, pool.head_dim,
                                                 uint64_t(p.q_stride), int(G), int(kPreM / G));
  // Blocks of one prompt's chunk that leave SMs idle are split along the keys (over 2, then 4
  // blocks), as long as each keeps five key tiles (24 blocks of
  // at most 512 positions: 13.6 us whole, 15.0 halved; 40 of 768: 19.8, 18.4).
  const long long blocks = pairs * p.kv_heads;
  const long long positions = p.offsets ? (long long)p.pages_per_row << p.page_shift : p.length;
  const long long keys = p.window ? std::min<long long>(positions, (long long)p.window + p.sinks) : positions;
  int cluster = 1;
  while (cluster < 4 && blocks * cluster * 2 <= 148 && keys >= cluster * 2 * 5 * kPreN) cluster *= 2;
  // One row with up to half a wave more blocks than SMs: halves end after 1.5 waves instead of 2, each
  // wave of them ~10 us more (2,560 queries over 10,560 positions 255 -> 230 us, over 6,560 of 64
  // dims 134 -> 136, over 4,560 87 -> 108). Ragged rows fill the gaps by themselves.
  if (cluster == 1 && p.rows == 1 && blocks > 148 && blocks <= 222 && keys - p.n_queries / 2 >= 6144) cluster = 2;
  if (pool.head_dim == 128)
    prefill_launch<128>(map, q_map, p, x, cluster, st);
  else
    prefill_launch<64>(map, q_map, p, x, cluster, st);
}

template <int D>
static void prefill_configure() {
  YAR_CUDA(cudaFuncSetAttribute(k_kv_attn_prefill<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, PreCfg<D>::kSmem));
  // The register split waits for ever when the launch holds fewer registers than it hands out.
  cudaFuncAttributes a;
  YAR_CUDA(cudaFuncGetAttributes(&a, k_kv_attn_prefill<D>));
  if (a.numRegs != kPreRegs)
    throw Error("RuntimeError", "prefill attention built with " + std::to_string(a.numRegs) + " registers, not 168");
}
void configure_kv_prefill_kernels() {
  prefill_configure<128>();
  prefill_configure<64>();
}

}  // namespace yar
