// Packed causal attention forward on the 5th-generation tensor cores (bf16, head size 64 or 128), in one pass over the keys
// with a running maximum and sum.
//
// A CTA owns TWO tiles of 128 query rows that read the same key head: the tiles of one key head are listed row block by
// row block with the heads of its group inside, and a CTA takes two neighbours of that list -- two heads of the group over
// the same rows, or, without grouping, two consecutive row blocks.  Every key / value block that comes into shared memory
// serves both tiles, and the two alternate: while the softmax threads of one work, the tensor pipe runs the products of
// the other.  Rows are rows of the packed axis; a tile may hold the ends and beginnings of several sequences, which costs
// a comparison per score on the blocks that need it and no tile is ever half empty.  Key blocks of 128 rows are counted
// from the first row the tile may see, so a short sequence costs one block, not two.
//   warp 0      TMA: Q of both tiles, then K_0, V_0, K_1, V_1, ... through one ring of stages
//   warp 1      one lane issues tcgen05.mma in the order  S0(n+1) after P0 V(n),  S1(n+1) after P1 V(n), ...
//   warps 2..5  softmax of tile 0, warps 6..9 of tile 1: a thread owns a row.  It takes the whole row of S from TMEM
//               (no shuffles), writes the probabilities as bf16 over the first half of the same columns, and the second
//               product reads them from there as its TMEM operand: they never touch shared memory, whose bandwidth the
//               two K-major operands of S already need in full (64 KB per 512 cycles).
// S(n+1) may overwrite P(n) because the tensor pipe runs the products of one thread in order.  A row's reference maximum
// is raised, and O in TMEM rescaled, only when a block exceeds it by more than 2^8; sums and maxima are fp32, the
// probabilities are rounded to bf16 (half a step, 2^-9 of the value) for the second product only.
// Bound: at head size 128 a tile and block are 2 x 512 cycles of tensor pipe and 1024 cycles of exponentials (16 per
// cycle and SM); at 64 the exponentials alone.  All waits are bounded.
// Measured at 32/8 heads of 128: 2 x 8192 tokens 1040 to 1160 us (950 to 1057 TFLOP/s over the pairs seen, 0.56 to 0.62 of a
// large library product; the power limit moves it), 24 ragged prompts (15,398 rows) 284 to 309 us (551 to 600 TFLOP/s: 77 % of
// the pairs computed are seen, and a CTA's first loads and last stores stand alone).  A tile's block takes 3640 cycles: 1800
// softmax, 250 until the product thread wakes, 1213 for P V and the next S, 380 until the softmax threads see it.  Tried and
// slower or the same: part of the exponentials as a polynomial on the FMA lanes, sixteen softmax warps with shared rows, P
// handed over in halves, TMEM loads in chunks with polled products, a running reference without the maximum pass, a
// persistent grid with cluster launch control, results through shared memory (281 -> 291 us), steps of 64 keys with two score
// buffers per tile (1080 -> 1490 us and 285 -> 350: products 64 columns wide run at half the rate).
#include <cuda.h>

#include "attention_packed.cuh"
#include "ptx_sm100.cuh"
#include "tensor_map.cuh"

namespace b200 {

namespace {

constexpr int TR = 128;          // query rows per tile, keys per block
constexpr int PK_THREADS = 320;  // TMA warp, MMA warp, 2 x 4 softmax warps
constexpr int SUBB = 128 * 128;  // bytes of one [128 rows x 64 columns] bf16 sub-tile

enum : uint32_t { ST_PACKED_TIMEOUT = 1u << 17, ST_PACKED_ALIGN = 1u << 18 };

template <int HS> struct PCfg {
  static constexpr int kSubs = HS / 64;
  static constexpr int kTile = kSubs * SUBB;           // Q tile, K or V block
  static constexpr int kStages = HS == 128 ? 5 : 6;    // 5 x 32 KB beside 64 KB of Q
  static constexpr int kKV = 2 * kTile;
  static constexpr int kBars = kKV + kStages * kTile;
  static constexpr int kSmem = kBars + 256;
  static constexpr int kO = 256;                       // TMEM columns: S0 0.., S1 128.., O0 256.., O1 384..
};

struct TileGeo { int head, t0, first, last; };  // blocks first..last of the CTA's list; last < first: nothing to do

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
__device__ __forceinline__ void tmem_st32u(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

template <int HS>
__global__ void __launch_bounds__(PK_THREADS, 1)
    packed_fwd_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                         const __grid_constant__ CUtensorMap tmV, PackedArgs a, float scale, uint32_t* status) {
  using C = PCfg<HS>;
  constexpr int NS = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint64_t* q_full = bars;            // [2]
  uint64_t* kv_full = bars + 2;       // [NS]
  uint64_t* kv_empty = kv_full + NS;  // [NS]
  uint64_t* s_full = kv_empty + NS;   // [2] S of the tile is complete
  uint64_t* p_full = s_full + 2;      // [2] the tile's probabilities stand in TMEM
  uint64_t* o_done = p_full + 2;      // [2] the tile's O += P V is complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  __shared__ TileGeo geo[2];
  __shared__ int k_base;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.n_heads / a.n_kv_heads;
  const int hk = blockIdx.x;
  const int n_tiles = (a.rows + TR - 1) / TR * group;
  const int pair = (int)gridDim.y - 1 - (int)blockIdx.y;  // late row blocks, which see the most keys, start first
  pdl_launch_dependents();

  if (threadIdx.x == 0) {
    uint32_t bad = 0u;
    if (ptx::smem_u32(smem) & 1023u) {
      atomicOr(status, ST_PACKED_ALIGN);
      bad = 1u;
    }
    *abort_flag = bad;
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&q_full[i], 1);
      ptx::mbar_init(&s_full[i], 1);
      ptx::mbar_init(&p_full[i], 128);
      ptx::mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < NS; ++i) {
      ptx::mbar_init(&kv_full[i], 1);
      ptx::mbar_init(&kv_empty[i], 1);
    }
    ptx::fence_barrier_init();
    ptx::tma_prefetch_desc(&tmQ);
    ptx::tma_prefetch_desc(&tmK);
    ptx::tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish();
  }
  pdl_wait();  // q, k, v and cu_seqlens come from the kernels before
  if (threadIdx.x == 0 && !*abort_flag) {  // the query tiles do not wait for the look-up of the sequences
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int idx = 2 * pair + i;
      if (idx >= n_tiles) break;
      ptx::mbar_arrive_expect_tx(&q_full[i], C::kTile);
#pragma unroll
      for (int s = 0; s < C::kSubs; ++s)
        ptx::tma_load_2d(smem + i * C::kTile + s * SUBB, &tmQ, (hk * group + idx % group) * HS + 64 * s, idx / group * TR, &q_full[i]);
    }
  }
  if (warp == 2) {
    // rows and keys of the two tiles
    const int cu_first = max(0, *(a.cu)), end = min(a.rows, *(a.cu + a.n_seqs));
    int from[2], to[2], base = 0x7fffffff;
    TileGeo g[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int idx = 2 * pair + i;
      const int rb = idx / group;
      g[i].head = hk * group + idx % group;
      g[i].t0 = rb * TR;
      to[i] = min(g[i].t0 + TR, end) - 1;
      from[i] = cu_first;
      if (idx >= n_tiles) {
        to[i] = -1;
      } else if (i && g[1].t0 == g[0].t0) {  // two heads of one row block
        from[1] = from[0];
      } else {
        const int s = seq_of_row_warp(a.cu, a.n_seqs, g[i].t0);
        if (s >= 0 && s < a.n_seqs) from[i] = max(0, min(g[i].t0, *(a.cu + s)));
      }
      if (to[i] < g[i].t0) to[i] = -1;
      if (to[i] >= from[i]) base = min(base, from[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool any = to[i] >= from[i];
      g[i].first = any ? (from[i] - base) / TR : 0;
      g[i].last = any ? (to[i] - base) / TR : -1;
      if (lane == 0) geo[i] = g[i];
    }
    if (lane == 0) k_base = base;
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const bool aborted = *abort_flag != 0u;
  const int n_blocks = max(geo[0].last, geo[1].last) + 1;

  if (aborted) {
    // fall through to the common exit
  } else if (warp == 0) {
    if (lane == 0) {
      const int kb = k_base;
      bool ok = true;
      for (int x = 0; x < 2 * n_blocks && ok; ++x) {  // K_0, V_0, K_1, V_1, ...
        const int st = x % NS;
        ok = ptx::mbar_wait(&kv_empty[st], ((uint32_t)(x / NS) & 1u) ^ 1u, abort_flag, status, ST_PACKED_TIMEOUT);
        if (!ok) break;
        ptx::mbar_arrive_expect_tx(&kv_full[st], C::kTile);
#pragma unroll
        for (int s = 0; s < C::kSubs; ++s)
          ptx::tma_load_2d(smem + C::kKV + st * C::kTile + s * SUBB, (x & 1) ? &tmV : &tmK, hk * HS + 64 * s,
                           kb + (x >> 1) * TR, &kv_full[st]);
      }
      for (int i = 0; i < 2 && ok; ++i)  // no copy outlives the CTA, a query tile without live rows neither
        if (2 * pair + i < n_tiles) ok = ptx::mbar_wait(&q_full[i], 0, abort_flag, status, ST_PACKED_TIMEOUT);
    }
    __syncwarp();
  } else if (n_blocks == 0) {
    // nothing to compute
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = ptx::idesc_bf16_f32(TR, TR);
      constexpr uint32_t idesc_o = ptx::idesc_bf16_f32(TR, HS) | (1u << 16);  // V is MN-major
      const uint64_t q_desc = ptx::smem_desc_sw128(ptx::smem_u32(smem));
      const uint64_t k_desc = ptx::smem_desc_sw128(ptx::smem_u32(smem + C::kKV));
      const uint64_t v_desc = ptx::smem_desc_sw128_mn(ptx::smem_u32(smem + C::kKV), SUBB);
      const int f[2] = {geo[0].first, geo[1].first}, l[2] = {geo[0].last, geo[1].last};
      bool ok = true;
      auto wait_kv = [&](int x) {
        ok = ok && ptx::mbar_wait(&kv_full[x % NS], (uint32_t)(x / NS) & 1u, abort_flag, status, ST_PACKED_TIMEOUT);
        if (ok) ptx::tc_fence_after_sync();
      };
      auto issue_s = [&](int i, int n) {  // S_i = Q_i K_n^T
        if (n < f[i] || n > l[i] || !ok) return;
        if (n == f[i]) ok = ptx::mbar_wait(&q_full[i], 0, abort_flag, status, ST_PACKED_TIMEOUT);
        if (!ok) return;
        const uint64_t qa = q_desc + (uint64_t)(i * (C::kTile >> 4));
        const uint64_t ka = k_desc + (uint64_t)((2 * n) % NS) * (C::kTile >> 4);
#pragma unroll
        for (int k = 0; k < HS / 16; ++k) {
          const uint64_t off = (uint64_t)(((k >> 2) * SUBB + (k & 3) * 32) >> 4);
          ptx::mma_bf16_ss(tmem_base + (uint32_t)(i * TR), qa + off, ka + off, idesc_s, k > 0 ? 1u : 0u);
        }
        ptx::mma_commit(&s_full[i]);
      };
      wait_kv(0);
      issue_s(0, 0);
      issue_s(1, 0);
      if (ok) ptx::mma_commit(&kv_empty[0]);
      for (int n = 0; n < n_blocks && ok; ++n) {
        wait_kv(2 * n + 1);
        const uint64_t va = v_desc + (uint64_t)((2 * n + 1) % NS) * (C::kTile >> 4);
        bool have_k = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (n >= f[i] && n <= l[i] && ok) {
            ok = ptx::mbar_wait(&p_full[i], (uint32_t)(n - f[i]) & 1u, abort_flag, status, ST_PACKED_TIMEOUT);
            if (!ok) break;
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int k = 0; k < TR / 16; ++k)  // O_i += P_i V_n: 16 keys are 8 TMEM columns of P and 2048 bytes of V
              mma_bf16_ts(tmem_base + (uint32_t)(C::kO + i * TR), tmem_base + (uint32_t)(i * TR + 8 * k),
                          va + (uint64_t)(k * (2048 >> 4)), idesc_o, (n > f[i] || k > 0) ? 1u : 0u);
            ptx::mma_commit(&o_done[i]);
          }
          if (i == 1) ptx::mma_commit(&kv_empty[(2 * n + 1) % NS]);
          if (n + 1 < n_blocks) {
            if (!have_k) wait_kv(2 * n + 2);
            have_k = true;
            issue_s(i, n + 1);
          }
        }
        if (n + 1 < n_blocks && ok) ptx::mma_commit(&kv_empty[(2 * n + 2) % NS]);
      }
    }
    __syncwarp();
  } else {
    const int i = (warp - 2) >> 2;
    const int qd = warp & 3;
    const TileGeo g = geo[i];
    const int t = g.t0 + qd * 32 + lane;  // this thread's row == TMEM lane of the tile
    const uint32_t t_s = tmem_base + ((uint32_t)(qd * 32) << 16) + (uint32_t)(i * TR);
    const uint32_t t_o = t_s + (uint32_t)C::kO;
    const float sl2 = scale * 1.4426950408889634f;  // scores are scaled inside the exp2
    RowSpan span{t + 1, t + 1};
    if (g.last >= g.first && t < a.rows) {
      const int s = seq_of_row(a.cu, 0, a.n_seqs, t);
      span = row_span(a.cu, a.n_seqs, s, t, a.rows);
    }
    const bool live = span.first <= t;
    float ms = -INFINITY, l = 0.f;
    bool ok = true;
    for (int n = g.first; n <= g.last; ++n) {
      const int m = n - g.first;
      ok = ptx::mbar_wait_warp(&s_full[i], (uint32_t)m & 1u, abort_flag, status, ST_PACKED_TIMEOUT);
      if (!ok) break;
      ptx::tc_fence_after_sync();
      float sv[128];
      ptx::tmem_ld32_at<0>(t_s, sv);
      ptx::tmem_ld32_at<32>(t_s + 32u, sv);
      ptx::tmem_ld32_at<64>(t_s + 64u, sv);
      ptx::tmem_ld32_at<96>(t_s + 96u, sv);
      ptx::tmem_ld_wait();
      const int k0 = k_base + n * TR;
      const int lo = live ? span.first - k0 : TR, hi = live ? t - k0 : -1;  // keys lo..hi of the block are seen
      if (__any_sync(0xffffffffu, hi < TR - 1)) {  // the diagonal (one comparison per score: hence the two branches)
#pragma unroll
        for (int e = 0; e < TR; ++e)
          if (e > hi) sv[e] = -INFINITY;
      }
      if (__any_sync(0xffffffffu, lo > 0)) {  // a sequence begins inside the block
#pragma unroll
        for (int e = 0; e < TR; ++e)
          if (e < lo) sv[e] = -INFINITY;
      }
      float b0 = -INFINITY, b1 = -INFINITY, b2 = -INFINITY, b3 = -INFINITY;
#pragma unroll
      for (int e = 0; e < TR; e += 8) {
        b0 = ptx::max3(b0, sv[e], sv[e + 1]);
        b1 = ptx::max3(b1, sv[e + 2], sv[e + 3]);
        b2 = ptx::max3(b2, sv[e + 4], sv[e + 5]);
        b3 = ptx::max3(b3, sv[e + 6], sv[e + 7]);
      }
      const float bm = fmaxf(fmaxf(b0, b1), fmaxf(b2, b3)) * sl2;
      if (m == 0) {
        ms = bm;
      } else if (__any_sync(0xffffffffu, bm > ms + 8.f)) {
        // raise the references (tcgen05.ld/st are warp-wide; rows that need no raise get the factor 1).  O must be at
        // rest: every O += P V issued so far has completed.
        const float nm = bm > ms + 8.f ? bm : ms;
        const float corr = nm == ms ? 1.f : ex2(ms - nm);
        ms = nm;
        l *= corr;
        ok = ptx::mbar_wait_warp(&o_done[i], (uint32_t)(m - 1) & 1u, abort_flag, status, ST_PACKED_TIMEOUT);
        if (!ok) break;
        ptx::tc_fence_after_sync();
#pragma unroll 1
        for (int c = 0; c < HS; c += 16) {
          float v[16];
          ptx::tmem_ld16(t_o + (uint32_t)c, v);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] *= corr;
          asm volatile(
              "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
              "%15, %16};" ::"r"(t_o + (uint32_t)c),
              "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
              "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
              "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
              "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])), "r"(__float_as_uint(v[15]))
              : "memory");
        }
        ptx::tmem_st_wait();
      }
      const float neg = ms == -INFINITY ? 0.f : -ms;  // a row that has seen no key yet keeps weights of zero
      const float2 sl2v = make_float2(sl2, sl2), negv = make_float2(neg, neg);
      float2 r0 = make_float2(0.f, 0.f), r1 = make_float2(0.f, 0.f);
      uint32_t pk[64];
#pragma unroll
      for (int e = 0; e < 64; ++e) {
        const float2 x = __ffma2_rn(make_float2(sv[2 * e], sv[2 * e + 1]), sl2v, negv);
        const float2 p = make_float2(ex2(x.x), ex2(x.y));
        if (e & 1) r1 = __fadd2_rn(r1, p);
        else r0 = __fadd2_rn(r0, p);
        const __nv_bfloat162 h = __floats2bfloat162_rn(p.x, p.y);
        pk[e] = *reinterpret_cast<const uint32_t*>(&h);
      }
      tmem_st32u(t_s, pk);
      tmem_st32u(t_s + 32u, pk + 32);
      l += (r0.x + r0.y) + (r1.x + r1.y);
      ptx::tmem_st_wait();
      ptx::tc_fence_before_sync();
      ptx::mbar_arrive(&p_full[i]);
    }
    if (ok && g.last >= g.first)
      ok = ptx::mbar_wait_warp(&o_done[i], (uint32_t)(g.last - g.first) & 1u, abort_flag, status, ST_PACKED_TIMEOUT);
    if (ok && g.last >= g.first) {
      ptx::tc_fence_after_sync();
      const float inv = 1.f / l;
      const bool wide_rows = (a.ldo & 15) == 0 && aligned32(a.o);
      bf16* dst = (bf16*)a.o + (size_t)t * a.ldo + g.head * HS;
      bool finite = true;
#pragma unroll 1
      for (int c = 0; c < HS; c += 32) {
        float v[32];
        ptx::tmem_ld32(t_o + (uint32_t)c, v);
        ptx::tmem_ld_wait();
        if (live) {
#pragma unroll
          for (int e = 0; e < 32; e += 16) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float x = v[e + 2 * j] * inv, y = v[e + 2 * j + 1] * inv;
              finite = finite && fabsf(x) < INFINITY && fabsf(y) < INFINITY;
              const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
              w[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
            if (wide_rows) {  // a thread writes a row: whole 32-byte sectors at a time where the rows allow it
              store32B(dst + c + e, w);
            } else {
              *reinterpret_cast<uint4*>(dst + c + e) = make_uint4(w[0], w[1], w[2], w[3]);
              *reinterpret_cast<uint4*>(dst + c + e + 8) = make_uint4(w[4], w[5], w[6], w[7]);
            }
          }
        }
      }
      if (live && a.lse) a.lse[(size_t)g.head * a.rows + t] = ms * 0.6931471805599453f + logf(l);
      // Zero weight times an infinity or NaN in a value row that is masked here is not zero: where there is one, rows that
      // did not come out finite are computed again over the rows they see alone.
      unsigned redo = __ballot_sync(0xffffffffu, live && !finite);
      while (redo) {
        const int r = __ffs(redo) - 1;
        redo &= redo - 1;
        const int tr = g.t0 + qd * 32 + r;
        const int first = __shfl_sync(0xffffffffu, span.first, r);
        __syncwarp();
        redo_fwd<HS>((const bf16*)a.q + (size_t)tr * a.ldq + g.head * HS, (const bf16*)a.k + hk * HS, (const bf16*)a.v + hk * HS,
                     (bf16*)a.o + (size_t)tr * a.ldo + g.head * HS, a.lse ? a.lse + (size_t)g.head * a.rows + tr : nullptr, a.ldk,
                     a.ldv, first, tr, scale, k_base + g.first * TR, min(a.rows, k_base + (g.last + 1) * TR));
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
    ptx::tmem_dealloc(tmem_base, 512);
  }
}

template <int HS>
int32_t launch_hs(const PackedArgs& a, cudaStream_t stream) {
  using C = PCfg<HS>;
  CUtensorMap tq, tk, tv;
  B200_TRY(make_map_2d(&tq, a.q, a.rows, a.n_heads * HS, a.ldq, TR));
  B200_TRY(make_map_2d(&tk, a.k, a.rows, a.n_kv_heads * HS, a.ldk, TR));
  B200_TRY(make_map_2d(&tv, a.v, a.rows, a.n_kv_heads * HS, a.ldv, TR));
  auto kern = packed_fwd_tc_kernel<HS>;
  static PerDeviceOnce attr_once;
  B200_TRY(attr_once.run([&](int&) -> int32_t {
    B200_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    return B200_OK;
  }));
  uint32_t* status = device_status_word();
  if (!status) return fail(B200_ERR_CUDA, "no device status word");
  const long long pairs = ((long long)cdiv(a.rows, TR) * (a.n_heads / a.n_kv_heads) + 1) / 2;
  B200_CUDA_OK(launch_pdl(kern, dim3(a.n_kv_heads, (unsigned)pairs), dim3(PK_THREADS), C::kSmem, stream, tq, tk, tv, a,
                          1.f / sqrtf((float)HS), status));
  B200_LAUNCH_OK("packed_fwd_tc_kernel");
  return B200_OK;
}

}  // namespace

bool packed_fwd_tc_supports(const PackedArgs& a) {
  return a.dtype == B200_BF16 && (a.head_size == 64 || a.head_size == 128) && a.ldq % 8 == 0 && a.ldk % 8 == 0 &&
         a.ldv % 8 == 0 && a.ldo % 8 == 0 && aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.o) &&
         ((long long)cdiv(a.rows, TR) * (a.n_heads / a.n_kv_heads) + 1) / 2 <= 65535;
}

int32_t launch_packed_fwd_tc(const PackedArgs& a, cudaStream_t stream) {
  if (!packed_fwd_tc_supports(a))
    return fail(B200_ERR_UNSUPPORTED, "packed attention on tensor cores needs bf16, head size 64 or 128 and 16-byte aligned rows");
  if (a.head_size == 64) return launch_hs<64>(a, stream);
  return launch_hs<128>(a, stream);
}

}  // namespace b200
