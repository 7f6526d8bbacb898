// Packed causal attention backward on the 5th-generation tensor cores (bf16, head size 64 or 128).  With
//   P = exp(q k^T / sqrt(hs) - lse),  dP = dO v^T,  delta = rowsum(P * dP),  dS = P * (dP - delta)
// the gradients are dV = P^T dO, dK = dS^T Q / sqrt(hs), dQ = dS K / sqrt(hs).  Two passes of one kernel, both free of atomics:
//   MODE_DQ   a CTA owns 128 queries of a query head and streams the keys and values they see
//   MODE_DKV  a CTA owns 128 keys of a key head and streams, for every query head of the group, the queries and their
//             cotangents that see them (so the gradient of a shared head is one sum in a fixed order).  The first keys of a
//             long sequence make the longest CTA by far; two CTAs of a cluster then take half of the group's heads each and
//             add up through distributed shared memory, one of them dV, the other dK
// Both have the same shape: two fixed tiles F0, F1 and streamed tiles X0, X1,
//   S = F0 X0^T,  dP = F1 X1^T  (TMEM, rows = the CTA's own rows)  ->  P, dS as bf16 over S, dP in TMEM
//   DQ  (F0 = Q, F1 = dO, X0 = K, X1 = V):  acc0 += P X0 (see below),  acc1 += dS X0 -> dQ
//   DKV (F0 = K, F1 = V, X0 = Q, X1 = dO):  acc0 += P X1 = dV,         acc1 += dS X0 -> dK
// so P and dS are TMEM operands of the accumulating products and never pass through shared memory.  The softmax threads'
// two phases run beside the products of the other phase: exponentials (S -> P) beside acc1(n-1) and dP(n), the score
// gradient (dP -> dS) beside acc0(n) and S(n+1).  S(n+1) may overwrite P(n), and dP(n+1) dS(n), because the tensor pipe
// runs the products of one thread in order.
//
// Head size 64 streams blocks of 64 rows: S, dP and the accumulators are then 256 TMEM columns and 75 KB of shared memory,
// two CTAs share an SM and one's set-up, waits and epilogue hide behind the other's products (8 x 1024 tokens, 12 heads:
// 167 us with one CTA and blocks of 128 rows, 129 us now).  Head size 128 takes all 512 columns with blocks of 128 rows.
//
// delta.  Taken from the output as rowsum(dO * o) it carries the rounding of o to bf16, which is not small beside
// dP - delta where a row sees few keys.  The query pass therefore also sums eps = rowsum(P * (dP - delta0)) in fp32 and
// acc0 = P K; dQ = (acc1 - eps * acc0) / sqrt(hs) is then the gradient for the exact delta = delta0 + eps, which it leaves
// behind for the key pass.  A tile whose keys fit one block settles eps before it forms dS.  delta0 itself is summed in the
// query pass from a TMA copy of o's rows (a kernel of its own for it read dO once more: 12 ragged documents 334 -> 329 us,
// 8 x 1024 tokens at 12 heads 131 -> 129 us; loads by the threads in its place took 334 to 365 us, as their latency
// stands before the first dS; L2 prefetches of the next CTA's tiles changed nothing).
//
// Bound: 8 products of 128 x 128 x hs per (query block, key block), of which 5 are the formula's; 512 cycles each at head
// size 128, 1024 cycles of exponentials.  A block's chain is 3550 cycles there (wait for S 640 to 1170, exponentials 1450, wait
// for dP 190 to 320, dS 670 to 860), and 2600 to 2900 for two CTAs' blocks of 64 rows at head size 64; set-up to the first S
// takes 3.3 to 4 us of a CTA and its epilogue 2 to 3, which short sequences pay per 128 rows.  12 ragged documents of 32/8 heads
// (4789 rows): 314 us, 350 TFLOP/s over the formula's 5 products; 8 x 1024 tokens of 12 heads of 64: 129 us, 250.  Tried and
// not kept: results through shared memory (129 -> 133 us), eight arrivals per meeting instead of 256 (no change).
// Rounding to bf16 happens to P, dS and the results; sums are fp32.  All waits are bounded.
#include <cuda.h>

#include "attention_packed.cuh"
#include "ptx_sm100.cuh"
#include "tensor_map.cuh"

namespace b200 {

namespace {

constexpr int BR = 128;
constexpr int PB_THREADS = 320;  // TMA warp, MMA warp, 8 softmax warps
constexpr int BSUB = 128 * 128;  // bytes of one [128 rows x 64 columns] bf16 sub-tile
constexpr int NX = 5;            // stages of streamed tiles (X0(0), X1(0), X0(1), ...)
enum { MODE_DKV = 0, MODE_DQ = 1 };
enum : uint32_t { ST_PACKEDB_TIMEOUT = 1u << 19, ST_PACKEDB_ALIGN = 1u << 20 };

template <int HS> struct BCfg {
  static constexpr int kBlock = HS;                    // streamed rows per block
  static constexpr int kSubs = HS / 64;
  static constexpr int kTile = kSubs * BSUB;           // fixed tile
  static constexpr int kXSub = kBlock * 128;           // one [kBlock rows x 64 columns] sub-tile
  static constexpr int kXTile = kSubs * kXSub;         // streamed tile
  static constexpr int kX = 2 * kTile;
  static constexpr int kOTiles = kTile / kXTile;       // stages, the last ones, that hold o's rows at first (DQ)
  static constexpr int kO = kX + (NX - kOTiles) * kXTile;
  static constexpr int kStat = kX + NX * kXTile;  // 2 stages x {-lse2[kBlock], -delta[kBlock]} of the streamed queries (DKV)
  static constexpr int kBars = kStat + 2 * 1024;
  static constexpr int kSmem = kBars + 256;
  static constexpr int cS = 0, cDP = kBlock, cAcc0 = 2 * kBlock, cAcc1 = 2 * kBlock + HS, kCols = 2 * kBlock + 2 * HS;
  static constexpr int kCtas = HS == 64 ? 2 : 1;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// D[tmem] (+)= A[tmem] * B[smem desc]
__device__ __forceinline__ void mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// N 32-bit columns of this thread's lane
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::
          "r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[32]) { ptx::tmem_ld32(taddr, v); }
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[64]) {
  ptx::tmem_ld32_at<0>(taddr, v);
  ptx::tmem_ld32_at<32>(taddr + 32u, v);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 16 bytes into the shared memory of CTA `rank` of the cluster, at the place `addr` has in this one
__device__ __forceinline__ void st_remote(uint32_t addr, uint32_t rank, const float* v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
}

// 16 numbers of one row: a thread writes a row by itself, so whole 32-byte sectors at a time where the rows allow it
__device__ __forceinline__ void store16(bf16* p, const float (&w)[16], bool wide) {
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(w[2 * i], w[2 * i + 1]);
    r[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  if (wide) {
    store32B(p, r);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]);
    *reinterpret_cast<uint4*>(p + 8) = make_uint4(r[4], r[5], r[6], r[7]);
  }
}

struct OwnGeo {
  int r0;       // first own row
  int x0;       // first streamed row
  int per_head; // streamed blocks per query head
  int n_it;     // blocks in all
};

template <int HS, int MODE, int SPLIT>
__global__ void __launch_bounds__(PB_THREADS, BCfg<HS>::kCtas)
    packed_bwd_tc_kernel(const __grid_constant__ CUtensorMap tmF0, const __grid_constant__ CUtensorMap tmF1,
                         const __grid_constant__ CUtensorMap tmX0, const __grid_constant__ CUtensorMap tmX1,
                         const __grid_constant__ CUtensorMap tmO, const __grid_constant__ PackedBwdArgs a, float scale, uint32_t* status) {
  using C = BCfg<HS>;
  constexpr int BN = C::kBlock, NC = BN / 2;  // streamed rows per block; of them per softmax thread
  const PackedArgs& f = a.f;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint64_t* fix_full = bars;            // fixed tiles landed
  uint64_t* x_full = bars + 1;          // [NX] streamed tile landed
  uint64_t* x_empty = x_full + NX;      // [NX] every product that reads the tile is complete
  uint64_t* stat_full = x_empty + NX;   // [2] lse and delta of the streamed queries are in shared memory (DKV)
  uint64_t* s_full = stat_full + 2;     // S complete in TMEM
  uint64_t* dp_full = s_full + 1;       // dP complete in TMEM
  uint64_t* p_full = dp_full + 1;       // P stands in TMEM
  uint64_t* ds_full = p_full + 1;       // dS stands in TMEM
  uint64_t* acc_done = ds_full + 1;     // the accumulators are complete
  uint64_t* met = acc_done + 1;         // the 256 softmax threads meet (a barrier whose wait is bounded too)
  uint64_t* o_full = bars + 24;         // the rows of o landed (DQ)
  uint64_t* o_done = bars + 25;         // they have been read
  OwnGeo* geo = reinterpret_cast<OwnGeo*>(bars + 20);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = f.n_heads / f.n_kv_heads;
  const int rank = MODE == MODE_DKV ? (int)blockIdx.x % SPLIT : 0;     // DKV: of the CTAs that share a key tile
  const int head = MODE == MODE_DKV ? (int)blockIdx.x / SPLIT : blockIdx.x;  // DKV: key head, DQ: query head
  auto meet_peer = [&]() {  // every thread of both CTAs, three times, whatever happened before
    if (SPLIT == 2) cluster_sync();
  };
  const int hk = MODE == MODE_DKV ? head : head / group;
  // the longest loops first: early keys are seen by the most queries, late queries see the most keys
  const int own = MODE == MODE_DKV ? (int)blockIdx.y : (int)gridDim.y - 1 - (int)blockIdx.y;
  pdl_launch_dependents();

  if (threadIdx.x == 0) {
    uint32_t bad = 0u;
    if (ptx::smem_u32(smem) & 1023u) {
      atomicOr(status, ST_PACKEDB_ALIGN);
      bad = 1u;
    }
    *abort_flag = bad;
    ptx::mbar_init(fix_full, 1);
    for (int i = 0; i < NX; ++i) {
      ptx::mbar_init(&x_full[i], 1);
      ptx::mbar_init(&x_empty[i], 1);
    }
    ptx::mbar_init(&stat_full[0], 32);
    ptx::mbar_init(&stat_full[1], 32);
    ptx::mbar_init(s_full, 1);
    ptx::mbar_init(dp_full, 1);
    ptx::mbar_init(p_full, 8);
    ptx::mbar_init(ds_full, 8);
    ptx::mbar_init(acc_done, 1);
    ptx::mbar_init(met, 256);
    ptx::mbar_init(o_full, 1);
    ptx::mbar_init(o_done, 8);
    ptx::fence_barrier_init();
    ptx::tma_prefetch_desc(&tmF0);
    ptx::tma_prefetch_desc(&tmF1);
    ptx::tma_prefetch_desc(&tmX0);
    ptx::tma_prefetch_desc(&tmX1);
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, C::kCols);
    ptx::tmem_relinquish();
  }
  pdl_wait();  // the operands come from the kernels before
  if (threadIdx.x == 0 && !*abort_flag) {  // the fixed tiles do not wait for the look-up of the sequences
    ptx::mbar_arrive_expect_tx(fix_full, 2 * C::kTile);
#pragma unroll
    for (int s = 0; s < C::kSubs; ++s) {
#pragma unroll
      for (int y = 0; y < BR; y += BN) {  // 128 bytes of a row each
        ptx::tma_load_2d(smem + s * BSUB + y * 128, &tmF0, head * HS + 64 * s, own * BR + y, fix_full);
        ptx::tma_load_2d(smem + C::kTile + s * BSUB + y * 128, &tmF1, head * HS + 64 * s, own * BR + y, fix_full);
      }
    }
    if (MODE == MODE_DQ) {
      ptx::mbar_arrive_expect_tx(o_full, C::kTile);
#pragma unroll
      for (int s = 0; s < C::kSubs; ++s)
#pragma unroll
        for (int y = 0; y < BR; y += BN)
          ptx::tma_load_2d(smem + C::kO + s * BSUB + y * 128, &tmO, head * HS + 64 * s, own * BR + y, o_full);
    }
  }
  if (warp == 2) {
    const int cu_first = max(0, *(f.cu)), end = min(f.rows, *(f.cu + f.n_seqs));
    OwnGeo g;
    g.r0 = own * BR;
    const int last_row = min(g.r0 + BR, end) - 1;  // last own row that belongs to a sequence
    const int probe = MODE == MODE_DKV ? max(0, last_row) : g.r0;
    const int s = seq_of_row_warp(f.cu, f.n_seqs, probe);
    const RowSpan sp = row_span(f.cu, f.n_seqs, s, probe, f.rows);
    int to;
    if (MODE == MODE_DKV) {  // queries from the first own row to the end of the last own row's sequence
      g.x0 = g.r0;
      to = sp.first <= probe ? sp.last : 0;
    } else {
      g.x0 = sp.first <= probe ? sp.first : cu_first;
      to = last_row + 1;
    }
    g.per_head = last_row >= g.r0 && to > g.x0 ? (to - g.x0 + BN - 1) / BN : 0;
    g.n_it = g.per_head * (MODE == MODE_DKV ? group / SPLIT : 1);
    if (lane == 0) *geo = g;
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const bool aborted = *abort_flag != 0u;
  const OwnGeo g = *geo;
  const int n_it = g.n_it;

  if (aborted || n_it == 0) {
    if (!aborted && threadIdx.x == 0) {  // no copy outlives the CTA
      ptx::mbar_wait(fix_full, 0, abort_flag, status, ST_PACKEDB_TIMEOUT);
      if (MODE == MODE_DQ) ptx::mbar_wait(o_full, 0, abort_flag, status, ST_PACKEDB_TIMEOUT);
    }
    __syncwarp();
    for (int i = 0; i < 3; ++i) meet_peer();
  } else if (warp == 0) {
    bool ok = true;
    for (int x = 0; x < 2 * n_it && ok; ++x) {
      const int st = x % NX, it = x >> 1;
      const int qh = MODE == MODE_DKV ? hk * group + rank * (group / SPLIT) + it / g.per_head : head;
      const int row = g.x0 + (it % g.per_head) * BN;
      ok = ptx::mbar_wait_warp(&x_empty[st], ((uint32_t)(x / NX) & 1u) ^ 1u, abort_flag, status, ST_PACKEDB_TIMEOUT);
      if (MODE == MODE_DQ && x < NX && st >= NX - C::kOTiles)
        ok = ok && ptx::mbar_wait_warp(o_done, 0, abort_flag, status, ST_PACKEDB_TIMEOUT);
      if (!ok) break;
      if (lane == 0) {
        const int col = (MODE == MODE_DKV ? qh : hk) * HS;
        ptx::mbar_arrive_expect_tx(&x_full[st], C::kXTile);
#pragma unroll
        for (int s = 0; s < C::kSubs; ++s)
          ptx::tma_load_2d(smem + C::kX + st * C::kXTile + s * C::kXSub, (x & 1) ? &tmX1 : &tmX0, col + 64 * s, row, &x_full[st]);
      }
      if (MODE == MODE_DKV && (x & 1)) {
        // X1(it) takes the stage X0(it - 2) or an older tile had, so the statistics of it - 2 have been used
        float* stat = reinterpret_cast<float*>(smem + C::kStat + (it & 1) * 1024);
#pragma unroll
        for (int c = lane; c < BN; c += 32) {
          const int t = row + c;
          const size_t at = (size_t)qh * f.rows + t;
          stat[c] = t < f.rows ? -f.lse[at] * 1.4426950408889634f : 0.f;
          stat[BN + c] = t < f.rows ? -a.delta[at] : 0.f;
        }
        ptx::mbar_arrive(&stat_full[it & 1]);
      }
      __syncwarp();
    }
    for (int i = 0; i < 3; ++i) meet_peer();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t id_kk = ptx::idesc_bf16_f32(BR, BN);               // both operands K-major
      constexpr uint32_t id_tm = ptx::idesc_bf16_f32(BR, HS) | (1u << 16);  // A in TMEM, B MN-major
      const uint64_t fix_k = ptx::smem_desc_sw128(ptx::smem_u32(smem));
      const uint64_t x_k = ptx::smem_desc_sw128(ptx::smem_u32(smem + C::kX));
      const uint64_t x_m = ptx::smem_desc_sw128_mn(ptx::smem_u32(smem + C::kX), C::kXSub);
      constexpr uint64_t kT = C::kTile >> 4, kXT = C::kXTile >> 4;
      bool ok = ptx::mbar_wait(fix_full, 0, abort_flag, status, ST_PACKEDB_TIMEOUT);
      auto wait_x = [&](int x) {
        ok = ok && ptx::mbar_wait(&x_full[x % NX], (uint32_t)(x / NX) & 1u, abort_flag, status, ST_PACKEDB_TIMEOUT);
        if (ok) ptx::tc_fence_after_sync();
      };
      auto scores = [&](int which, int it) {  // 0: S = F0 X0^T, 1: dP = F1 X1^T
        const uint64_t fa = fix_k + (uint64_t)which * kT, xa = x_k + (uint64_t)((2 * it + which) % NX) * kXT;
#pragma unroll
        for (int k = 0; k < HS / 16; ++k) {
          const uint64_t foff = (uint64_t)(((k >> 2) * BSUB + (k & 3) * 32) >> 4);
          const uint64_t xoff = (uint64_t)(((k >> 2) * C::kXSub + (k & 3) * 32) >> 4);
          ptx::mma_bf16_ss(tmem_base + (uint32_t)(which ? C::cDP : C::cS), fa + foff, xa + xoff, id_kk, k > 0 ? 1u : 0u);
        }
        ptx::mma_commit(which ? dp_full : s_full);
      };
      auto accumulate = [&](int which, int it) {  // 0: acc0 += P X, 1: acc1 += dS X0
        const int tile = 2 * it + (which == 0 && MODE == MODE_DKV ? 1 : 0);
        const uint64_t xa = x_m + (uint64_t)(tile % NX) * kXT;
        const uint32_t src = tmem_base + (uint32_t)(which ? C::cDP : C::cS);
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)  // P / dS of a half's NC columns stands in the first NC / 2 of them
          mma_bf16_ts(tmem_base + (uint32_t)(which ? C::cAcc1 : C::cAcc0), src + (uint32_t)(k / (NC / 16) * NC + k % (NC / 16) * 8),
                      xa + (uint64_t)(k * (2048 >> 4)), id_tm, (it > 0 || k > 0) ? 1u : 0u);
      };
      wait_x(0);
      if (ok) scores(0, 0);
      wait_x(1);
      if (ok) scores(1, 0);
      if (ok && MODE == MODE_DQ) ptx::mma_commit(&x_empty[1]);  // V has no second reader
      for (int it = 0; it < n_it && ok; ++it) {
        const uint32_t ph = (uint32_t)it & 1u;
        ok = ptx::mbar_wait(p_full, ph, abort_flag, status, ST_PACKEDB_TIMEOUT);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        accumulate(0, it);
        if (MODE == MODE_DKV) ptx::mma_commit(&x_empty[(2 * it + 1) % NX]);
        if (it + 1 < n_it) {
          wait_x(2 * it + 2);
          if (!ok) break;
          scores(0, it + 1);
        }
        ok = ptx::mbar_wait(ds_full, ph, abort_flag, status, ST_PACKEDB_TIMEOUT);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        accumulate(1, it);
        ptx::mma_commit(&x_empty[(2 * it) % NX]);
        if (it + 1 < n_it) {
          wait_x(2 * it + 3);
          if (!ok) break;
          scores(1, it + 1);
          if (MODE == MODE_DQ) ptx::mma_commit(&x_empty[(2 * it + 3) % NX]);
        }
      }
      if (ok) ptx::mma_commit(acc_done);
    }
    __syncwarp();
    for (int i = 0; i < 3; ++i) meet_peer();
  } else {
    const int qd = warp & 3;
    const int hf = (warp - 2) >> 2;   // columns NC hf .. NC hf + NC - 1 of a block
    const int row = qd * 32 + lane;   // TMEM lane: the CTA's own row
    const int r = g.r0 + row;
    const uint32_t lane_base = tmem_base + ((uint32_t)(qd * 32) << 16);
    const uint32_t t_s = lane_base + (uint32_t)(C::cS + hf * NC), t_dp = lane_base + (uint32_t)(C::cDP + hf * NC);
    const float sl2 = scale * 1.4426950408889634f;
    const int s = r < f.rows ? seq_of_row(f.cu, 0, f.n_seqs, r) : -1;
    const RowSpan span = row_span(f.cu, f.n_seqs, s, r, f.rows);
    const bool live = span.first <= r;
    float lse2 = 0.f, delta = 0.f, eps = 0.f;
    float* share = reinterpret_cast<float*>(smem + C::kStat);  // DQ: [2][128] halves of eps, behind them of delta0
    bool ok = true;
    uint32_t met_phase = 0u;
    auto meet = [&]() {
      ptx::mbar_arrive(met);
      ok = ptx::mbar_wait_warp(met, met_phase, abort_flag, status, ST_PACKEDB_TIMEOUT);
      met_phase ^= 1u;
      return ok;
    };
    if (MODE == MODE_DQ) {  // delta0 = dO.o, half a row per thread, beside the first products
      if (live) lse2 = f.lse[(size_t)head * f.rows + r] * 1.4426950408889634f;
      ok = ptx::mbar_wait_warp(fix_full, 0, abort_flag, status, ST_PACKEDB_TIMEOUT) &&
           ptx::mbar_wait_warp(o_full, 0, abort_flag, status, ST_PACKEDB_TIMEOUT);
      const uint8_t* po = smem + (C::kSubs == 2 ? hf * BSUB : 0) + row * 128;
#pragma unroll
      for (int c = 0; c < HS / 16; ++c) {
        const int at = ((C::kSubs == 2 ? c : hf * 4 + c) ^ (row & 7)) << 4;  // the 128-byte swizzle of a tile's row
        float x[8], y[8];
        load8(reinterpret_cast<const bf16*>(po + C::kO + at), x);
        load8(reinterpret_cast<const bf16*>(po + C::kTile + at), y);
#pragma unroll
        for (int i = 0; i < 8; ++i) delta = fmaf(x[i], y[i], delta);
      }
      share[2 * BR + hf * BR + row] = delta;
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(o_done);
      ok = ok && meet();
      delta = live ? delta + share[2 * BR + (hf ^ 1) * BR + row] : 0.f;
    }
    for (int it = 0; it < n_it && ok; ++it) {
      const uint32_t ph = (uint32_t)it & 1u;
      const int c0 = g.x0 + (it % g.per_head) * BN + hf * NC;  // streamed row of this thread's first column
      // columns lo..hi of the NC form a pair with the own row
      const int lo = live ? (MODE == MODE_DQ ? span.first : r) - c0 : NC;
      const int hi = live ? (MODE == MODE_DQ ? r : span.last - 1) - c0 : -1;
      // (one comparison per score and border: most blocks have none, most others one of the two)
      const bool cut_lo = __any_sync(0xffffffffu, lo > 0), cut_hi = __any_sync(0xffffffffu, hi < NC - 1);
      const float* stat = reinterpret_cast<const float*>(smem + C::kStat + (it & 1) * 1024) + hf * NC;
      if (MODE == MODE_DKV) {
        ok = ptx::mbar_wait_warp(&stat_full[it & 1], (uint32_t)(it >> 1) & 1u, abort_flag, status, ST_PACKEDB_TIMEOUT);
        if (!ok) break;
      }
      ok = ptx::mbar_wait_warp(s_full, ph, abort_flag, status, ST_PACKEDB_TIMEOUT);
      if (!ok) break;
      ptx::tc_fence_after_sync();
      float p[NC];
      tmem_ld(t_s, p);
      ptx::tmem_ld_wait();
      uint32_t pk[NC / 2];
      const float2 sl2v = make_float2(sl2, sl2);
#pragma unroll
      for (int e = 0; e < NC; e += 4) {
        float4 l4 = make_float4(-lse2, -lse2, -lse2, -lse2);
        if (MODE == MODE_DKV) l4 = *reinterpret_cast<const float4*>(stat + e);
        const float2 x0 = __ffma2_rn(make_float2(p[e], p[e + 1]), sl2v, make_float2(l4.x, l4.y));
        const float2 x1 = __ffma2_rn(make_float2(p[e + 2], p[e + 3]), sl2v, make_float2(l4.z, l4.w));
        p[e] = ex2(x0.x);
        p[e + 1] = ex2(x0.y);
        p[e + 2] = ex2(x1.x);
        p[e + 3] = ex2(x1.y);
      }
      if (cut_hi) {
#pragma unroll
        for (int e = 0; e < NC; ++e)
          if (e > hi) p[e] = 0.f;
      }
      if (cut_lo) {
#pragma unroll
        for (int e = 0; e < NC; ++e)
          if (e < lo) p[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < NC / 2; ++e) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(p[2 * e], p[2 * e + 1]);
        pk[e] = *reinterpret_cast<const uint32_t*>(&h);
      }
      // the two halves read and write disjoint columns of S
      tmem_st(t_s, pk);
      ptx::tmem_st_wait();
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(p_full);

      ok = ptx::mbar_wait_warp(dp_full, ph, abort_flag, status, ST_PACKEDB_TIMEOUT);
      if (!ok) break;
      ptx::tc_fence_after_sync();
      float dp[NC];
      tmem_ld(t_dp, dp);
      ptx::tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < NC; e += 4) {
        float4 d4 = make_float4(-delta, -delta, -delta, -delta);
        if (MODE == MODE_DKV) d4 = *reinterpret_cast<const float4*>(stat + BN + e);
        const float2 y0 = __fmul2_rn(__fadd2_rn(make_float2(dp[e], dp[e + 1]), make_float2(d4.x, d4.y)), make_float2(p[e], p[e + 1]));
        const float2 y1 = __fmul2_rn(__fadd2_rn(make_float2(dp[e + 2], dp[e + 3]), make_float2(d4.z, d4.w)), make_float2(p[e + 2], p[e + 3]));
        dp[e] = y0.x;
        dp[e + 1] = y0.y;
        dp[e + 2] = y1.x;
        dp[e + 3] = y1.y;
      }
      if (cut_hi) {
#pragma unroll
        for (int e = 0; e < NC; ++e)
          if (e > hi) dp[e] = 0.f;
      }
      if (cut_lo) {  // (holds where an `alone` row meets itself: there lo >= 0, and lo = 0 in lane 0 only, as blocks begin at
                     // multiples of 32 rows from the warp's first)
        const int from = lo + (MODE == MODE_DKV && alone(span.first, r) ? 1 : 0);
#pragma unroll
        for (int e = 0; e < NC; ++e)
          if (e < from) dp[e] = 0.f;
      }
      if (MODE == MODE_DQ) {
        float2 s0 = make_float2(0.f, 0.f), s1 = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < NC; e += 4) {
          s0 = __fadd2_rn(s0, make_float2(dp[e], dp[e + 1]));
          s1 = __fadd2_rn(s1, make_float2(dp[e + 2], dp[e + 3]));
        }
        float sum = (s0.x + s0.y) + (s1.x + s1.y);
        if (n_it == 1) {  // all keys of the row are here: settle delta before dS is rounded
          share[hf * BR + row] = sum;
          if (!meet()) break;
          sum += share[(hf ^ 1) * BR + row];
          delta += sum;
#pragma unroll
          for (int e = 0; e < NC; ++e) dp[e] = fmaf(-p[e], sum, dp[e]);
        } else {
          eps += sum;
        }
      }
#pragma unroll
      for (int e = 0; e < NC / 2; ++e) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(dp[2 * e], dp[2 * e + 1]);
        pk[e] = *reinterpret_cast<const uint32_t*>(&h);
      }
      tmem_st(t_dp, pk);
      ptx::tmem_st_wait();
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ds_full);
    }
    if (ok) ok = ptx::mbar_wait_warp(acc_done, 0, abort_flag, status, ST_PACKEDB_TIMEOUT);
    // Two CTAs: the first one adds up and writes dV, the second dK.  The streamed tiles' memory is free by now.
    const uint32_t swap = ptx::smem_u32(smem + C::kX) + (uint32_t)row * 16;
    constexpr bool shared = SPLIT == 2;
    meet_peer();
    if (shared && ok && hf != rank) {
      ptx::tc_fence_after_sync();
#pragma unroll 1
      for (int c = 0; c < HS; c += 32) {
        float v[32];
        ptx::tmem_ld32(lane_base + (uint32_t)((hf == 0 ? C::cAcc0 : C::cAcc1) + c), v);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; e += 4) st_remote(swap + (uint32_t)((c + e) / 4 * BR * 16), (uint32_t)(rank ^ 1), v + e);
      }
    }
    meet_peer();
    bool finite = true;
    if (ok && !(shared && hf != rank)) {
      ptx::tc_fence_after_sync();
      if (MODE == MODE_DKV) {
        // half 0 writes dV, half 1 dK
        bf16* dst = hf == 0 ? (bf16*)a.dv + (size_t)r * a.lddv : (bf16*)a.dk + (size_t)r * a.lddk;
        const uint32_t src = lane_base + (uint32_t)(hf == 0 ? C::cAcc0 : C::cAcc1);
        const float out_scale = hf == 0 ? 1.f : scale;
        const bool wide_rows = ((hf == 0 ? a.lddv : a.lddk) & 15) == 0 && aligned32(hf == 0 ? a.dv : a.dk);
#pragma unroll 1
        for (int c = 0; c < HS; c += 32) {
          float v[32];
          ptx::tmem_ld32(src + (uint32_t)c, v);
          ptx::tmem_ld_wait();
          if (shared) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 w = *reinterpret_cast<const float4*>(smem + C::kX + (c + e) / 4 * BR * 16 + row * 16);
              v[e] += w.x; v[e + 1] += w.y; v[e + 2] += w.z; v[e + 3] += w.w;
            }
          }
          if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 16) {
              float w[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                w[j] = v[e + j] * out_scale;
                finite = finite && fabsf(w[j]) < INFINITY;
              }
              store16(dst + head * HS + c + e, w, wide_rows);
            }
          }
        }
      } else {
        if (n_it > 1) {
          share[hf * BR + row] = eps;
          meet();
          eps += share[(hf ^ 1) * BR + row];
          delta += eps;
        }
        if (live && hf == 0) a.delta[(size_t)head * f.rows + r] = delta;
        bf16* dst = (bf16*)a.dq + (size_t)r * a.lddq + head * HS;
        const bool wide_rows = (a.lddq & 15) == 0 && aligned32(a.dq);
        const float out_scale = alone(span.first, r) ? 0.f : scale;
#pragma unroll 1
        for (int c = hf * (HS / 2); c < (hf + 1) * (HS / 2); c += 32) {
          float v[32], u[32];
          ptx::tmem_ld32(lane_base + (uint32_t)(C::cAcc1 + c), v);
          ptx::tmem_ld32(lane_base + (uint32_t)(C::cAcc0 + c), u);
          ptx::tmem_ld_wait();
          if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 16) {
              float w[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                w[j] = fmaf(-eps, u[e + j], v[e + j]) * out_scale;
                finite = finite && fabsf(w[j]) < INFINITY;
              }
              store16(dst + c + e, w, wide_rows);
            }
          }
        }
      }
    }
    meet_peer();
    if (ok) {
      // Both halves meet before either redoes a row, which the other may still write for the first time (dQ).
      meet();
      const unsigned bad = __ballot_sync(0xffffffffu, ok && live && !finite);
      if (bad) {
        const int r0 = g.r0 + qd * 32, x_end = min(f.rows, g.x0 + g.per_head * BN);
        if (MODE == MODE_DQ) redo_dq<HS>(a, bad, r0, head, g.x0, x_end, scale);
        else if (hf == 0) redo_dkv<HS, false>(a, bad, r0, hk, g.x0, x_end, scale);
        else redo_dkv<HS, true>(a, bad, r0, hk, g.x0, x_end, scale);
      }
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // copies in flight land before the shared memory is given back
  }
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, C::kCols);
  }
}

template <int HS>
int32_t launch_hs(const PackedBwdArgs& a, cudaStream_t stream) {
  using C = BCfg<HS>;
  const PackedArgs& f = a.f;
  // in boxes of a streamed block; a fixed tile is one or two of them
  CUtensorMap mq, mk, mv, mdo, mo;
  B200_TRY(make_map_2d(&mq, f.q, f.rows, f.n_heads * HS, f.ldq, C::kBlock));
  B200_TRY(make_map_2d(&mk, f.k, f.rows, f.n_kv_heads * HS, f.ldk, C::kBlock));
  B200_TRY(make_map_2d(&mv, f.v, f.rows, f.n_kv_heads * HS, f.ldv, C::kBlock));
  B200_TRY(make_map_2d(&mdo, a.d_o, f.rows, f.n_heads * HS, a.lddo, C::kBlock));
  B200_TRY(make_map_2d(&mo, f.o, f.rows, f.n_heads * HS, f.ldo, C::kBlock));
  auto dq = packed_bwd_tc_kernel<HS, MODE_DQ, 1>;
  auto dkv = packed_bwd_tc_kernel<HS, MODE_DKV, 1>;
  auto dkv2 = packed_bwd_tc_kernel<HS, MODE_DKV, 2>;
  static PerDeviceOnce attr_once;
  B200_TRY(attr_once.run([&](int&) -> int32_t {
    B200_CUDA_OK(cudaFuncSetAttribute(dq, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    B200_CUDA_OK(cudaFuncSetAttribute(dkv, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    B200_CUDA_OK(cudaFuncSetAttribute(dkv2, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    return B200_OK;
  }));
  uint32_t* status = device_status_word();
  if (!status) return fail(B200_ERR_CUDA, "no device status word");
  const float scale = 1.f / sqrtf((float)HS);
  const unsigned blocks = (unsigned)cdiv(f.rows, BR);
  B200_CUDA_OK(launch_pdl(dq, dim3(f.n_heads, blocks), dim3(PB_THREADS), C::kSmem, stream, mq, mdo, mk, mv, mo, a,
                          scale, status));
  B200_LAUNCH_OK("packed_bwd_tc_kernel<dq>");
  // Two CTAs per key tile where there are few tiles, or not many and the sequences are long on average (256 rows), so that the
  // first keys of one make a CTA that outlasts the others.  The lengths themselves are on the device: one long sequence among
  // many short ones is taken for a short batch, and its first tiles then end the pass alone.
  // Backward with one / two (us, heads of 128): 12 ragged documents of 32/8 heads (304 tiles) 333 / 317, 2048 tokens of 8/2
  // heads (32) 196 / 136; 8 x 1024 of 32/8 (512) 407 / 421, 64 x 128 of 32/8 (512) 216 / 246.  Heads of 64: 365 / 245 and
  // 214 / 141, 8 x 1024 of 12/6 (384) 159 / 151; 64 x 128 of 32/8 (512) 122 / 139.
  const long long key_tiles = (long long)f.n_kv_heads * blocks;
  const bool few = 2 * key_tiles <= sm_count();
  const bool uneven = key_tiles <= 3LL * sm_count() && f.rows >= 256LL * f.n_seqs;
  const bool two = (f.n_heads / f.n_kv_heads) % 2 == 0 && (few || uneven);
  if (two)
    B200_CUDA_OK(launch_pdl_cluster(dkv2, dim3(f.n_kv_heads * 2, blocks), dim3(PB_THREADS), 2, C::kSmem, stream, mk, mv, mq, mdo, mo,
                                    a, scale, status));
  else
    B200_CUDA_OK(launch_pdl(dkv, dim3(f.n_kv_heads, blocks), dim3(PB_THREADS), C::kSmem, stream, mk, mv, mq, mdo, mo, a, scale,
                            status));
  B200_LAUNCH_OK("packed_bwd_tc_kernel<dkv>");
  return B200_OK;
}

}  // namespace

bool packed_bwd_tc_supports(const PackedBwdArgs& a) {
  const PackedArgs& f = a.f;
  return f.dtype == B200_BF16 && (f.head_size == 64 || f.head_size == 128) && f.ldq % 8 == 0 && f.ldk % 8 == 0 &&
         f.ldv % 8 == 0 && f.ldo % 8 == 0 && a.lddo % 8 == 0 && a.lddq % 8 == 0 && a.lddk % 8 == 0 && a.lddv % 8 == 0 &&
         aligned16(f.q) && aligned16(f.k) && aligned16(f.v) && aligned16(f.o) && aligned16(a.d_o) && aligned16(a.dq) &&
         aligned16(a.dk) && aligned16(a.dv) && cdiv(f.rows, BR) <= 65535;
}

int32_t launch_packed_bwd_tc(const PackedBwdArgs& a, cudaStream_t stream) {
  if (!packed_bwd_tc_supports(a))
    return fail(B200_ERR_UNSUPPORTED, "packed attention backward on tensor cores needs bf16, head size 64 or 128 and 16-byte aligned rows");
  if (a.f.head_size == 64) return launch_hs<64>(a, stream);
  return launch_hs<128>(a, stream);
}

}  // namespace b200
