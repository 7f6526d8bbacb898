// Decode attention over the 4-bit cache with the codes as matrix operands (bf16 queries, head size 64 or 128, pages of a
// multiple of 16 rows, grouped heads).
//
// A byte of codes holds two elements, so at HBM speed an SM receives 23 bytes and would have to expand and multiply 46
// elements per cycle for q.k and for p.v -- more than its FP32 lanes do.  The codes therefore go into the integer
// mma.sync (m16n8k32, 8 x 8 bits, 32-bit sums) as they are: eight codes of a word become bytes with one shift and two
// masks.  (The same product on e4m3 numbers, which hold the codes too, is made of conversions here and took 1.3 times as
// long as bf16 operands; the integer one runs at twice their rate.)  The row's scale s and minimum m enter afterwards:
//   q.k = s sum q n + m sum q              o = sum_j (s_j p_j) n_j + sum_j p_j m_j
// The 16 rows of an A operand are 16 keys (q.k) or 16 head dimensions (p.v); its 8 columns are four query heads twice,
// because the other operand is a 16-bit integer in two bytes: query elements in steps of 1/32512 of their head's largest
// (two products), weights s p -- kept in fp32 until then -- in steps of 1/65535 of a power of two that is at most twice the
// largest of a tile of 32 keys and a head (columns 0..3 take the high bytes, 4..7 the low bytes of the same heads).  So a
// weight is rounded against its own tile, by 2^-16 of the largest there: a key that carries most of a head's weight, or a
// value row of a far larger scale, costs the long tail of the others nothing.  (One step for all tiles, from the largest
// weight so far, read every row far below it as its minimum.)  Sums of a tile's products are exact integers below 2^23; the
// product starts them at the bits of the float 2^23, so that one packed subtraction makes numbers of them, which are
// added up in fp32.  Five to eight heads are two such sets over the same codes, larger groups are cut into subsets of eight.
// The order of the elements inside a contraction is free: a lane takes 16 contiguous bytes of a key row with the query
// laid out to match; the values come through ldmatrix's byte transpose, which hands a lane two elements of four keys, and
// the rows of the key operand are ordered so that one 8x8 transpose gives the lane the weights of those four.  The odd
// elements of a value byte stay in its high half (16 n) and the factor is taken out of their sums.
// One warp brings units of 128 keys (codes and parameters of both halves, four TMA copies per page piece) into a ring of
// shared-memory stages and runs ahead over segment borders; four warps take 32 keys of a unit each.
// HBM-bound: hs + 8 bytes per (key, key head), each read once.  64 sequences of 4096 rows, 32 heads of 128: 201 us back to
// back (5.7 TB/s, 0.88 of a copy; 194 with one step for all tiles), 231 us behind a kernel that left L2 full of written lines
// (0.76).  16 sequences of up to 32,768 rows, 32/8 heads: 59 us (3.0 TB/s): at one segment per CTA the time is set-up, the
// first loads and the joining kernel.  Tried: codes loaded into registers with four CTAs per SM (290 us where this form took
// 265 then), four CTAs on two stages (275 against 249), scores without integer conversions (their sums begun at 1.5 2^23: no
// change).
#include <algorithm>

#include "kv4.cuh"
#include "ptx_sm100.cuh"
#include "tensor_map.cuh"

namespace b200 {

namespace {

constexpr int MW = 4;                       // consumer warps per CTA
constexpr int M_THREADS = 32 * (MW + 1);
constexpr int kStages = 3;
constexpr float kLow = -3e38f;  // reference of a column that has seen no key: finite, so that -inf - kLow is -inf
enum : uint32_t { ST_KV4_TIMEOUT = 1u << 21, ST_KV4_ALIGN = 1u << 22 };
constexpr int kCtas(int hs, int sets) { return hs == 128 ? (sets == 1 ? 3 : 2) : (sets == 1 ? 4 : 2); }  // resident CTAs per SM

// shared memory of a CTA
template <int HS> struct MCfg {
  static constexpr int kCode = kUnit * HS / 2;       // bytes of one half's codes of a unit
  static constexpr int kPrm = kUnit * 4;
  static constexpr int kStage = 2 * kCode + 2 * kPrm;  // key codes, value codes, key parameters, value parameters
  static constexpr int kBars = kStages * kStage;
  static constexpr int kPre = kBars + 128;           // unit prefix and lengths of the batch
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the first product of a sum
__device__ __forceinline__ void mma_u8s8_new(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
// a whole sum on top of the bits of the float 2^23: below 2^23 the result, read as a float, is 2^23 + sum
__device__ __forceinline__ void mma_u8u8_on_2p23(uint32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                 uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0x4b000000u));
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// four 8x8-byte blocks of 16 keys x 16 bytes, transposed: lane 4g + t gets bytes g (r[0], r[2]) and g + 8 (r[1], r[3]) of
// keys 4t .. 4t + 3 of the first and the second 16 keys; lane l gives the address of key l
__device__ __forceinline__ void ldmatrix_bytes(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// even and odd codes of a word, a byte each
__device__ __forceinline__ uint32_t even(uint32_t x) { return x & 0x0f0f0f0fu; }
__device__ __forceinline__ uint32_t odd(uint32_t x) { return (x >> 4) & 0x0f0f0f0fu; }

template <int W> struct Words;
template <> struct Words<2> { using V = uint2; };
template <> struct Words<4> { using V = uint4; };
template <int W> __device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&r)[W]) {
  const typename Words<W>::V x = *reinterpret_cast<const typename Words<W>::V*>(p);
  const uint32_t* s = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
  for (int i = 0; i < W; ++i) r[i] = s[i];
}
// untiled copy: 16-byte aligned on both sides, a multiple of 16 bytes
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(ptx::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(ptx::smem_u32(bar))
               : "memory");
}

// NS: sets of four heads.
template <int HS, int NS>
__global__ void __launch_bounds__(M_THREADS, kCtas(HS, NS))
    kv4_decode_mma_kernel(const __grid_constant__ CUtensorMap tm_codes, Kv4DecodeArgs a, int page_shift, int piece) {
  using C = MCfg<HS>;
  constexpr int KW = HS / 32, MT = HS / 16, RB = HS / 2;  // words of a key row per lane, 16-row products, bytes of a row
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int32_t warp_sums[MW + 1];
  __shared__ uint32_t s_valid[kStages], s_abort;
  __shared__ float s_o[MW][8 * NS][HS + 4], s_m[MW][4 * NS], s_l[MW][4 * NS], s_c[MW][4 * NS];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint64_t* empty = full + kStages;
  int32_t* pre = reinterpret_cast<int32_t*>(smem + C::kPre);
  int32_t* lens = pre + a.batch + 1;
  volatile uint32_t* abort_flag = &s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    s_abort = 0u;
    if (ptx::smem_u32(smem) & 1023u) {
      atomicOr(a.status, ST_KV4_ALIGN);
      s_abort = 1u;
    }
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(&full[i], 1);
      ptx::mbar_init(&empty[i], MW);
    }
    ptx::fence_barrier_init();
    ptx::tma_prefetch_desc(&tm_codes);
  }
  pdl_wait();  // everything below comes from the kernels before
  const UnitRange range = unit_range<M_THREADS>(a, pre, lens, warp_sums);
  const Kv4Pool& p = a.pool;
  const int nseg = p.n_kv_heads * a.subs;
  const long long r0 = range.first, r1 = range.last;
  if (r0 == r1 || s_abort) {
    if (a.whole) zero_segment<bf16>(a);
    return;
  }
  const size_t half = kv4_half(p);
  int b = range.seq;
  int st = 0;  // stage and phase of the next unit
  uint32_t phase = 0u;
  auto next_stage = [&]() {
    if (++st == kStages) {
      st = 0;
      phase ^= 1u;
    }
  };

  if (warp == MW) {
    const int at = (lane >> 2) * piece, kind = lane & 3;  // this lane's piece of a unit; key codes, value codes, and so on
    const int n_pieces = kUnit / piece;
    const uint32_t copy_bytes = (uint32_t)(piece * (kind < 2 ? RB : 4));
    const uint32_t* prm = p.params + (kind & 1) * half;
    const int dst = (kind < 2 ? kind * C::kCode : 2 * C::kCode + (kind - 2) * C::kPrm) + at * (kind < 2 ? RB : 4);
    bool ok = true;
    for (long long x = r0; x < r1 && ok;) {
      while ((long long)pre[b + 1] * nseg <= x) ++b;
      const int nb = pre[b + 1] - pre[b];
      const int off = (int)(x - (long long)pre[b] * nseg);
      const int hk = off / nb / a.subs, len = lens[b];
      int n = nb - off % nb;  // units of this range that lie in the segment
      if (n > r1 - x) n = (int)(r1 - x);
      x += n;
      int u = off % nb * kUnit + at;
      const int32_t* table = p.table + (size_t)b * p.max_pages;
      for (; n > 0 && ok; --n, u += kUnit) {
        // A piece is copied whole: rows of the page behind the end of the sequence come along and are not used.
        uint32_t bytes = 0u;
        size_t row = 0;
        if (u < len && (lane >> 2) < n_pieces) {
          const int slot = page_shift >= 0 ? u >> page_shift : u / p.page_size;
          const int page = table[slot];
          if ((unsigned)page < (unsigned)p.n_pages) {
            row = ((size_t)page * p.n_kv_heads + hk) * p.page_size + (u - slot * p.page_size);
            bytes = copy_bytes;
          } else if (kind == 0) {
            atomicOr(a.status, ST_BAD_PAGE);
          }
        }
        const uint32_t total = __reduce_add_sync(0xffffffffu, bytes);
        const uint32_t valid = __ballot_sync(0xffffffffu, bytes != 0u);
        ok = ptx::mbar_wait_warp(&empty[st], phase ^ 1u, abort_flag, a.status, ST_KV4_TIMEOUT);
        if (!ok) break;
        if (lane == 0) {
          s_valid[st] = valid;
          ptx::mbar_arrive_expect_tx(&full[st], total);
        }
        __syncwarp();
        if (bytes) {
          uint8_t* to = smem + st * C::kStage + dst;
          if (kind < 2) ptx::tma_load_3d(to, &tm_codes, 0, (int)row, kind, &full[st]);
          else bulk_load(to, prm + row, bytes, &full[st]);
        }
        next_stage();
      }
    }
  } else {
    const int group = a.n_heads / p.n_kv_heads;
    const float sl2 = a.scale * 1.4426950408889634f;
    const bool q_vec = (a.ldq & 7) == 0 && (reinterpret_cast<uintptr_t>(a.q) & 15u) == 0;
    const uint32_t part_sel = g < 4 ? 0x7531u : 0x6420u;  // high bytes, low bytes
    // Row g of the key operand's first eight is key 4 (g / 2) + g % 2 of the sixteen, row g of its second eight the key two
    // further.  TMA swizzles the 16-byte chunks of a row: by row / 2 % 4 (rows of 64 bytes) or row / 4 % 2 (of 32).
    const int kr = 4 * (g >> 1) + (g & 1);
    const uint8_t* k_lane[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = kr + 2 * r;
      const int chunk = HS == 128 ? t ^ ((row >> 1) & 3) : (t >> 1) ^ ((row >> 2) & 1);
      k_lane[r] = smem + (32 * warp + row) * RB + chunk * 16 + (HS == 128 ? 0 : (t & 1) * 8);
    }
    const uint32_t v_row = ptx::smem_u32(smem) + C::kCode + (32 * warp + lane) * RB;
    const uint32_t v_swz = HS == 128 ? (lane >> 1) & 3 : (lane >> 2) & 1;
    const uint8_t* p_lane = smem + 2 * C::kCode + (32 * warp + kr) * 4;
    const int bit0 = 32 * warp / piece * 4, bit1 = (32 * warp + 16) / piece * 4;  // of the tile's halves in `valid`
    bool ok = true;
    for (long long x = r0; x < r1;) {
      while ((long long)pre[b + 1] * nseg <= x) ++b;
      const int nb = pre[b + 1] - pre[b];
      const long long base = (long long)pre[b] * nseg;
      const int seg = (int)((x - base) / nb);
      const long long s0 = base + (long long)seg * nb, s1 = s0 + nb;
      const long long x1 = r1 < s1 ? r1 : s1;
      const int hk = seg / a.subs, first_head = (seg % a.subs) * a.cols;
      const int n_cols = min(a.cols, group - first_head);
      const int head0 = hk * group + first_head;
      const int c1 = lens[b];

      // query fragments: column g; the elements of a lane's words, even codes and odd codes, high bytes and low bytes
      uint32_t qh[NS][KW][2], ql[NS][KW][2];
      float q0[NS], q1[NS], f0[NS], f1[NS];  // of columns 2t, 2t + 1: sum of q, and the step of its elements
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const int col = 4 * n + (g & 3);
        const bool on = col < n_cols;
        const bf16* q = (const bf16*)a.q + (size_t)b * a.ldq + (head0 + (on ? col : 0)) * HS + t * (HS / 4);
        float e[8 * KW], top = 0.f, qs = 0.f;
        if (q_vec) {
#pragma unroll
          for (int i = 0; i < KW; ++i) {
            float x[8];
            load8(q + 8 * i, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) e[8 * i + j] = on ? x[j] : 0.f;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8 * KW; ++i) e[i] = on ? to_f32(q[i]) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8 * KW; ++i) {
          qs += e[i];
          top = fmaxf(top, fabsf(e[i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        qs += __shfl_xor_sync(0xffffffffu, qs, 1);
        qs += __shfl_xor_sync(0xffffffffu, qs, 2);
        const float up = top > 0.f ? fminf(32512.f / top, 1e30f) : 1.f;
#pragma unroll
        for (int i = 0; i < KW; ++i) {
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            uint32_t h = 0u, l = 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int v = __float2int_rn(e[8 * i + 2 * j + o] * up);
              const int vh = (v + 128) >> 8;
              h |= ((uint32_t)vh & 0xffu) << (8 * j);
              l |= ((uint32_t)(v - 256 * vh) & 0xffu) << (8 * j);
            }
            qh[n][i][o] = h;
            ql[n][i][o] = l;
          }
        }
        qs *= sl2;
        const float fs = sl2 / up;
        q0[n] = __shfl_sync(0xffffffffu, qs, 8 * (t & 1));
        q1[n] = __shfl_sync(0xffffffffu, qs, 8 * (t & 1) + 4);
        f0[n] = __shfl_sync(0xffffffffu, fs, 8 * (t & 1));
        f1[n] = __shfl_sync(0xffffffffu, fs, 8 * (t & 1) + 4);
      }

      float2 acc[NS][MT][2];                   // elements 2 (8i + g) and the next one (held as 16 n), columns 2t, 2t + 1
      float m0[NS], m1[NS];                    // references of columns 2t, 2t + 1 (uniform over g): p = e^(s - m) <= 1
      float l0[NS], l1[NS], c0s[NS], c1s[NS];  // this lane's share of sum p and of sum p m
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        m0[n] = m1[n] = kLow;
        l0[n] = l1[n] = c0s[n] = c1s[n] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[n][i][0] = acc[n][i][1] = make_float2(0.f, 0.f);
      }

      int u = (int)(x - s0) * kUnit + 32 * warp;  // first key of this warp's tile
      for (int left = (int)(x1 - x); left > 0; --left, u += kUnit, next_stage()) {
        ok = ok && ptx::mbar_wait_warp(&full[st], phase, abort_flag, a.status, ST_KV4_TIMEOUT);
        if (!ok) continue;  // the barriers below are still met
        if (u < c1) {
          const int so = st * C::kStage;
          const uint32_t valid = s_valid[st];
          const bool on[2] = {((valid >> bit0) & 1u) != 0u, ((valid >> bit1) & 1u) != 0u};
          const bool whole = u + 32 <= c1 && on[0] && on[1];
          float xs[NS][2][4], b0[NS], b1[NS];
          uint32_t vp[2][2];
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            int dh[NS][4], dl[NS][4];
            uint32_t kp[2], kw[2][KW];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              load_words<KW>(k_lane[r] + so + 16 * s * RB, kw[r]);
              kp[r] = *reinterpret_cast<const uint32_t*>(p_lane + so + (16 * s + 2 * r) * 4);
              vp[s][r] = *reinterpret_cast<const uint32_t*>(p_lane + so + C::kPrm + (16 * s + 2 * r) * 4);
              if (!whole && !(on[s] && u + 16 * s + 2 * r + kr < c1)) kp[r] = vp[s][r] = 0u;  // may be anything
            }
#pragma unroll
            for (int i = 0; i < KW; ++i) {
              const uint32_t ea = even(kw[0][i]), eb = even(kw[1][i]), oa = odd(kw[0][i]), ob = odd(kw[1][i]);
#pragma unroll
              for (int n = 0; n < NS; ++n) {
                if (i == 0) {
                  mma_u8s8_new(dh[n], ea, eb, oa, ob, qh[n][i][0], qh[n][i][1]);
                  mma_u8s8_new(dl[n], ea, eb, oa, ob, ql[n][i][0], ql[n][i][1]);
                } else {
                  mma_u8s8(dh[n], ea, eb, oa, ob, qh[n][i][0], qh[n][i][1]);
                  mma_u8s8(dl[n], ea, eb, oa, ob, ql[n][i][0], ql[n][i][1]);
                }
              }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float ks = __uint_as_float(kp[r] << 16), km = __uint_as_float(kp[r] & 0xffff0000u);
#pragma unroll
              for (int n = 0; n < NS; ++n) {
                const float2 d = make_float2((float)(256 * dh[n][2 * r] + dl[n][2 * r]), (float)(256 * dh[n][2 * r + 1] + dl[n][2 * r + 1]));
                const float2 x = __ffma2_rn(make_float2(ks, ks), __fmul2_rn(d, make_float2(f0[n], f1[n])),
                                            __fmul2_rn(make_float2(km, km), make_float2(q0[n], q1[n])));
                xs[n][s][2 * r] = x.x;
                xs[n][s][2 * r + 1] = x.y;
              }
            }
          }
          if (!whole) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int r = 0; r < 2; ++r)
                if (!(on[s] && u + 16 * s + 2 * r + kr < c1)) {
#pragma unroll
                  for (int n = 0; n < NS; ++n) xs[n][s][2 * r] = xs[n][s][2 * r + 1] = -INFINITY;
                }
          }
          bool raise = false;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            b0[n] = fmaxf(fmaxf(xs[n][0][0], xs[n][0][2]), fmaxf(xs[n][1][0], xs[n][1][2]));
            b1[n] = fmaxf(fmaxf(xs[n][0][1], xs[n][0][3]), fmaxf(xs[n][1][1], xs[n][1][3]));
            raise = raise || b0[n] > m0[n] || b1[n] > m1[n];
          }
          if (__any_sync(0xffffffffu, raise)) {
            // The new reference is 2^8 above the largest, which fp32 does not mind and which few later keys exceed.
#pragma unroll
            for (int n = 0; n < NS; ++n) {
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) {
                b0[n] = fmaxf(b0[n], __shfl_xor_sync(0xffffffffu, b0[n], o));
                b1[n] = fmaxf(b1[n], __shfl_xor_sync(0xffffffffu, b1[n], o));
              }
              const float n0 = b0[n] > m0[n] ? b0[n] + 8.f : m0[n], n1 = b1[n] > m1[n] ? b1[n] + 8.f : m1[n];
              const float e0 = n0 == m0[n] ? 1.f : ex2(m0[n] - n0), e1 = n1 == m1[n] ? 1.f : ex2(m1[n] - n1);
              m0[n] = n0; m1[n] = n1;
              l0[n] *= e0; l1[n] *= e1; c0s[n] *= e0; c1s[n] *= e1;
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                acc[n][i][0] = __fmul2_rn(acc[n][i][0], make_float2(e0, e1));
                acc[n][i][1] = __fmul2_rn(acc[n][i][1], make_float2(e0, e1));
              }
            }
          }
          float2 w[NS][2][2], step[NS];  // weights s p of columns 2t, 2t + 1
          uint32_t wb[NS][2];
#pragma unroll
          for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const float vs = __uint_as_float(vp[s][r] << 16), vm = __uint_as_float(vp[s][r] & 0xffff0000u);
                const float2 x = __fadd2_rn(make_float2(xs[n][s][2 * r], xs[n][s][2 * r + 1]), make_float2(-m0[n], -m1[n]));
                const float2 p = make_float2(ex2(x.x), ex2(x.y));
                const float2 l = __fadd2_rn(make_float2(l0[n], l1[n]), p);
                const float2 c = __ffma2_rn(p, make_float2(vm, vm), make_float2(c0s[n], c1s[n]));
                l0[n] = l.x; l1[n] = l.y;
                c0s[n] = c.x; c1s[n] = c.y;
                w[n][s][r] = __fmul2_rn(p, make_float2(vs, vs));
              }
            // exponents of the tile's largest weights: the upper halves of the two numbers in one word
            const float t0 = fmaxf(fmaxf(w[n][0][0].x, w[n][0][1].x), fmaxf(w[n][1][0].x, w[n][1][1].x));
            const float t1 = fmaxf(fmaxf(w[n][0][0].y, w[n][0][1].y), fmaxf(w[n][1][0].y, w[n][1][1].y));
            uint32_t top = __byte_perm(__float_as_uint(t0), __float_as_uint(t1), 0x7632u);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top = max2(top, __shfl_xor_sync(0xffffffffu, top, o));
            // weights below 2^(e + 1) count 65535 2^-(e + 1) each; the exponent field is kept where both factors are
            // normal numbers (a tile whose weights are all below 2^-111 loses bits)
            const uint32_t f0 = max(top << 16 & 0x7f800000u, 16u << 23), f1 = max(top & 0x7f800000u, 16u << 23);
            const uint32_t up_at = 0x477fff00u + (126u << 23), step_at = 0x37800080u - (126u << 23);  // 65535, 1/65535
            const float2 up = make_float2(__uint_as_float(up_at - f0), __uint_as_float(up_at - f1));
            step[n] = make_float2(__uint_as_float(step_at + f0), __uint_as_float(step_at + f1));
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              uint32_t tr[2];
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                // rounded to integers in the low 16 bits of 2^23 + w, column 2t in the low half, column 2t + 1 in the high one
                const float2 z = __ffma2_rn(w[n][s][r], up, make_float2(8388608.f, 8388608.f));
                tr[r] = transpose8x8(__byte_perm(__float_as_uint(z.x), __float_as_uint(z.y), 0x5410u));
              }
              // now the weights of column g for keys 4t .. 4t + 3: the byte this column takes
              wb[n][s] = __byte_perm(tr[0], tr[1], part_sel);
            }
          }
#pragma unroll
          for (int i = 0; i < HS / 32; ++i) {  // 16 bytes of every row
            uint32_t y[4];
            ldmatrix_bytes(y, v_row + so + ((i ^ v_swz) << 4));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t a0 = even(y[j]), a1 = y[j] & 0xf0f0f0f0u, a2 = even(y[j + 2]), a3 = y[j + 2] & 0xf0f0f0f0u;
#pragma unroll
              for (int n = 0; n < NS; ++n) {
                uint32_t d[4];
                mma_u8u8_on_2p23(d, a0, a1, a2, a3, wb[n][0], wb[n][1]);
                const float2 base = make_float2(-8388608.f, -8388608.f);
#pragma unroll
                for (int c = 0; c < 2; ++c)
                  acc[n][2 * i + j][c] = __ffma2_rn(
                      __fadd2_rn(make_float2(__uint_as_float(d[2 * c]), __uint_as_float(d[2 * c + 1])), base), step[n], acc[n][2 * i + j][c]);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&empty[st]);
      }

#pragma unroll
      for (int n = 0; n < NS; ++n) {
        // the lanes of a column
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          l0[n] += __shfl_xor_sync(0xffffffffu, l0[n], o);
          l1[n] += __shfl_xor_sync(0xffffffffu, l1[n], o);
          c0s[n] += __shfl_xor_sync(0xffffffffu, c0s[n], o);
          c1s[n] += __shfl_xor_sync(0xffffffffu, c1s[n], o);
        }
        // high bytes count 256 times; the odd elements were held as 16 n
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float f = (t < 2 ? 256.f : 1.f) * (c ? 0.0625f : 1.f);
            s_o[warp][8 * n + 2 * t][2 * (8 * i + g) + c] = acc[n][i][c].x * f;
            s_o[warp][8 * n + 2 * t + 1][2 * (8 * i + g) + c] = acc[n][i][c].y * f;
          }
        if (t < 2 && g == 0) {
          s_m[warp][4 * n + 2 * t] = m0[n]; s_m[warp][4 * n + 2 * t + 1] = m1[n];
          s_l[warp][4 * n + 2 * t] = l0[n]; s_l[warp][4 * n + 2 * t + 1] = l1[n];
          s_c[warp][4 * n + 2 * t] = c0s[n]; s_c[warp][4 * n + 2 * t + 1] = c1s[n];
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");  // the consumer warps; none of them leaves the loop early
      const bool finished = x == s0 && x1 == s1;
      float* part = a.partials + (size_t)(2 * blockIdx.x + (x == r0 ? 0 : 1)) * a.cols * (HS + 2);
      for (int e = threadIdx.x; e < n_cols * HS; e += MW * 32) {
        const int c = e / HS, d = e % HS;
        float gm = s_m[0][c];
#pragma unroll
        for (int w = 1; w < MW; ++w) gm = fmaxf(gm, s_m[w][c]);
        float v = 0.f, gl = 0.f;
#pragma unroll
        for (int w = 0; w < MW; ++w) {
          const float f = s_m[w][c] == gm ? 1.f : ex2(s_m[w][c] - gm);
          const int at = 8 * (c >> 2) + (c & 3);  // high bytes; low bytes four columns further
          v = fmaf(s_o[w][at][d] + s_o[w][at + 4][d] + s_c[w][c], f, v);
          gl = fmaf(s_l[w][c], f, gl);
        }
        if (finished) {
          ((bf16*)a.o)[(size_t)b * a.ldo + head0 * HS + e] = __float2bfloat16_rn(gl == 0.f ? 0.f : v / gl);
        } else {
          part[c * (HS + 2) + d] = v;
          if (d == 0) {
            part[c * (HS + 2) + HS] = gm * 0.6931471805599453f;  // the joining kernel counts in powers of e
            part[c * (HS + 2) + HS + 1] = gl;
          }
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");  // s_o is reused by the next segment
      x = x1;
    }
  }
  if (*abort_flag) {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // copies in flight land before the shared memory is given back
  }
}

// codes as [2][rows][hs/2] bytes; box: `piece` whole rows, 16-byte chunks swizzled by the row's width
int32_t make_map_codes(CUtensorMap* map, const Kv4Pool& p, int piece) {
  EncodeTiledFn fn = tensor_map_encoder();
  if (!fn) return fail(B200_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t rb = (cuuint64_t)p.head_size / 2, rows = (cuuint64_t)kv4_half(p);
  cuuint64_t dims[3] = {rb, rows, 2};
  cuuint64_t strides[2] = {rb, rb * rows};
  cuuint32_t box[3] = {(cuuint32_t)rb, (cuuint32_t)piece, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, p.codes, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  rb == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(B200_ERR_CUDA, "cuTensorMapEncodeTiled (codes) failed with %d", (int)r);
  return B200_OK;
}

template <int HS, int NS> int32_t launch_hs(const Kv4DecodeArgs& a, int grid, cudaStream_t stream) {
  using C = MCfg<HS>;
  const int ps = a.pool.page_size;
  const int shift = (ps & (ps - 1)) == 0 ? __builtin_ctz((unsigned)ps) : -1;
  const int piece = std::min(kUnit, ps & -ps);  // rows of a unit that never cross a page: 16, 32, 64 or 128
  const size_t smem = C::kPre + (size_t)(2 * a.batch + 1) * sizeof(int32_t);
  auto kern = kv4_decode_mma_kernel<HS, NS>;
  CUtensorMap codes;
  B200_TRY(make_map_codes(&codes, a.pool, piece));
  static PerDeviceOnce attr_once;
  B200_TRY(attr_once.run([&](int&) -> int32_t {
    B200_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(C::kPre + (2 * kMaxSlice + 1) * sizeof(int32_t))));
    return B200_OK;
  }));
  B200_CUDA_OK(launch_pdl(kern, dim3(grid), dim3(M_THREADS), smem, stream, codes, a, shift, piece));
  B200_LAUNCH_OK("kv4_decode_mma_kernel");
  return B200_OK;
}

}  // namespace

bool kv4_decode_mma_supports(const Kv4DecodeArgs& a) {
  return a.dtype == B200_BF16 && (a.pool.head_size == 64 || a.pool.head_size == 128) && a.pool.page_size % 16 == 0 &&
         aligned16(a.pool.codes) && aligned16(a.pool.params) &&
         kv4_half(a.pool) > 0 && kv4_half(a.pool) <= 0x7fffffffu;  // rows are TMA coordinates
}

int kv4_decode_mma_grid(int head_size, int cols) { return kCtas(head_size, cols > 4 ? 2 : 1) * sm_count(); }

int32_t launch_kv4_decode_mma(const Kv4DecodeArgs& a, int grid, cudaStream_t stream) {
  if (a.pool.head_size == 64) return a.cols > 4 ? launch_hs<64, 2>(a, grid, stream) : launch_hs<64, 1>(a, grid, stream);
  return a.cols > 4 ? launch_hs<128, 2>(a, grid, stream) : launch_hs<128, 1>(a, grid, stream);
}

}  // namespace b200
