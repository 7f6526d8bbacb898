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
// (two products), weights s p -- kept in fp32 until then -- in steps of 2^-16 of a reference that is at most 8 times the
// largest (columns 0..3 take the high bytes, 4..7 the low bytes of the same heads).  Sums of products are exact; they are
// brought into fp32 when a reference changes and at the end.  Five to eight heads are two such sets over the same codes,
// larger groups are cut into subsets of eight.
// The order of the elements inside a contraction is free: a lane takes 16 contiguous bytes of a key row with the query
// laid out to match, and the keys of a value operand are the ones whose weights the lane gets out of one 8x8 transpose.
// Warps walk their keys 32 at a time with the next 32 keys in flight in registers (4.3 KB per warp).
// HBM-bound: hs + 8 bytes per (key, key head), each read once.
#include <algorithm>

#include "kv4.cuh"

namespace b200 {

namespace {

constexpr int MW = 4;  // warps per CTA
constexpr int kTileKeys = 32;

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
__device__ __forceinline__ void mma_u8u8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// even and odd codes of a word, a byte each
__device__ __forceinline__ uint32_t even(uint32_t x) { return x & 0x0f0f0f0fu; }
__device__ __forceinline__ uint32_t odd(uint32_t x) { return (x >> 4) & 0x0f0f0f0fu; }

template <int W> struct Words;
template <> struct Words<1> { using V = uint32_t; };
template <> struct Words<2> { using V = uint2; };
template <> struct Words<4> { using V = uint4; };
template <int W> __device__ __forceinline__ void load_words(const uint32_t* p, uint32_t (&r)[W]) {
  const typename Words<W>::V x = *(reinterpret_cast<const typename Words<W>::V*>(p));
  const uint32_t* s = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
  for (int i = 0; i < W; ++i) r[i] = s[i];
}

// 32 keys of one key head: what a lane holds of them.
template <int HS> struct Tile {
  static constexpr int KW = HS / 32;  // words of a key row per lane (4 lanes to a row)
  static constexpr int VW = HS / 64;  // words of a value row per lane (8 lanes to a row)
  uint32_t k[2][2][KW];               // [16-key half][row lane/4, lane/4 + 8]
  uint32_t v[2][4][VW];               // [half][keys 2t, 2t+1, 2t+8, 2t+9],  t = lane % 4
  uint32_t kp[2][2], vp[2][2];        // parameters of rows lane/4 and lane/4 + 8
  bool on[2];                         // the half exists (its page is in the pool and it begins before the end)
};

// NS: sets of four heads.  P32: pages of a multiple of 32 rows, so that a tile lies in one page.
template <int HS, int NS, bool P32>
__global__ void __launch_bounds__(MW * 32, NS == 1 ? 3 : 2) kv4_decode_mma_kernel(Kv4DecodeArgs a, int page_shift) {
  using T = Tile<HS>;
  constexpr int KW = T::KW, VW = T::VW, MT = HS / 16, RW = HS / 8;  // RW: words of a row
  extern __shared__ int32_t pre[];
  __shared__ int32_t warp_sums[MW];
  __shared__ float s_o[MW][8 * NS][HS + 4], s_m[MW][4 * NS], s_l[MW][4 * NS], s_c[MW][4 * NS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  pdl_wait();  // everything below comes from the kernels before
  unit_prefix<MW * 32>(a, pre, warp_sums);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= a.batch; i += blockDim.x) a.prefix[i] = pre[i];
  const Kv4Pool& p = a.pool;
  const int nseg = p.n_kv_heads * a.subs;
  const long long units = (long long)pre[a.batch] * nseg;
  const int ctas = (int)(units < (long long)gridDim.x ? units : (long long)gridDim.x);
  if ((int)blockIdx.x >= ctas) return;
  const long long r0 = range_start(units, ctas, blockIdx.x), r1 = range_start(units, ctas, blockIdx.x + 1);
  const size_t half = kv4_half(p);
  // this lane's part of a row block: 16 bytes of key row g, the value rows 2t.., the parameters of row g
  const uint32_t* kbase = reinterpret_cast<const uint32_t*>(p.codes) + g * RW + t * KW;
  const uint32_t* vbase = reinterpret_cast<const uint32_t*>(p.codes) + half * RW + 2 * t * RW + g * VW;
  const uint32_t* kprm = p.params + g;
  const uint32_t* vprm = p.params + half + g;
  const int group = a.n_heads / p.n_kv_heads;
  const float sl2 = a.scale * 1.4426950408889634f;
  const uint32_t part_sel = g < 4 ? 0x7531u : 0x6420u;  // high bytes, low bytes
  int b = 0;
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
    const int len = kv4_len(a, b);
    const int c0 = (int)(x - s0) * kUnit, c1 = min(len, (int)(x1 - s0) * kUnit);
    const int32_t* table = p.table + (size_t)b * p.max_pages;

    struct Place { int page[2], row[2]; };
    auto place = [&](int u, int* page, int* row) {  // u: first key of a 16-key half
      const int slot = page_shift >= 0 ? u >> page_shift : u / p.page_size;
      *row = u - slot * p.page_size;
      *page = u < c1 ? table[slot] : -1;
    };
    auto places = [&](int u) {
      Place q;
      place(u, &q.page[0], &q.row[0]);
      if (P32) {
        q.page[1] = q.page[0];
        q.row[1] = q.row[0] + 16;
      } else {
        place(u + 16, &q.page[1], &q.row[1]);
      }
      return q;
    };
    auto load = [&](T& w, const Place& q, int u) {
      size_t at = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        w.on[s] = u + 16 * s < c1;
        if (w.on[s] && (unsigned)q.page[s] >= (unsigned)p.n_pages) {
          w.on[s] = false;
          if (lane == 0) atomicOr(a.status, ST_BAD_PAGE);
        }
        if (s == 0 || !P32) at = ((size_t)q.page[s] * p.n_kv_heads + hk) * p.page_size + q.row[s];
        const int more = P32 ? 16 * s : 0;  // rows behind `at`
        if (w.on[s]) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            load_words<KW>(kbase + at * RW + (more + 8 * r) * RW, w.k[s][r]);
            w.kp[s][r] = kprm[at + more + 8 * r];
            w.vp[s][r] = vprm[at + more + 8 * r];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) load_words<VW>(vbase + at * RW + (more + (j & 1) + 8 * (j >> 1)) * RW, w.v[s][j]);
        } else {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            w.kp[s][r] = w.vp[s][r] = 0u;
#pragma unroll
            for (int i = 0; i < KW; ++i) w.k[s][r][i] = 0u;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < VW; ++i) w.v[s][j][i] = 0u;
        }
      }
    };

    // query fragments: column g; the elements of a lane's words, even codes and odd codes, high bytes and low bytes
    uint32_t qh[NS][KW][2], ql[NS][KW][2];
    float q0[NS], q1[NS], f0[NS], f1[NS];  // of columns 2t, 2t + 1: sum of q, and the step of its elements
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int col = 4 * n + (g & 3);
      const bool on = col < n_cols;
      const bf16* q = (const bf16*)a.q + (size_t)b * a.ldq + (head0 + (on ? col : 0)) * HS + t * (HS / 4);
      float e[8 * KW], top = 0.f, qs = 0.f;
#pragma unroll
      for (int i = 0; i < 8 * KW; ++i) {
        e[i] = on ? to_f32(q[i]) : 0.f;
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

    int acc[NS][MT][4];
    float m0[NS], m1[NS];                          // references of columns 2t, 2t + 1 (uniform over g): weights are <= 1
    float l0[NS], l1[NS], c0s[NS], c1s[NS];        // this lane's share of sum p and of sum p m
    float sc = __uint_as_float(254u << 23);        // power of two that keeps the value scales at most 1 (uniform)
    bool kept = false;                             // s_o holds sums (uniform)
    int tiles = 0;                                 // a sum of 255 * 15 a key stays below 2^31 for 2^18 keys and more
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      m0[n] = m1[n] = -INFINITY;
      l0[n] = l1[n] = c0s[n] = c1s[n] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[n][i][j] = 0;
    }
    // Adds the integer sums of one set to its fp32 sums in shared memory (columns 8n .. 8n + 7), which are then scaled by
    // e0, e1, and clears them.
    auto keep = [&](int n, float e0, float e1) {
      const float step = (t < 2 ? 256.f : 1.f) / 65535.f / sc;
#pragma unroll
      for (int i = 0; i < VW; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {  // elements 2j, 2j + 1 of the word, columns 2t, 2t + 1
            float& at = s_o[warp][8 * n + 2 * t + (c & 1)][g * (HS / 8) + 8 * i + 2 * j + (c >> 1)];
            const float was = kept ? at : 0.f;
            at = fmaf((float)acc[n][4 * i + j][c], step, was) * ((c & 1) ? e1 : e0);
            acc[n][4 * i + j][c] = 0;
          }
        }
      }
    };

    auto compute = [&](const T& w, int u) {
      float xs[NS][2][4], b0[NS], b1[NS], smax = 0.f;
      bool raise = (++tiles & 8191) == 0;
#pragma unroll
      for (int n = 0; n < NS; ++n) b0[n] = b1[n] = -INFINITY;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        int dh[NS][4], dl[NS][4];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) dh[n][j] = dl[n][j] = 0;
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const uint32_t ka = w.k[s][0][i], kb = w.k[s][1][i];
          const uint32_t ea = even(ka), eb = even(kb), oa = odd(ka), ob = odd(kb);
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            mma_u8s8(dh[n], ea, eb, oa, ob, qh[n][i][0], qh[n][i][1]);
            mma_u8s8(dl[n], ea, eb, oa, ob, ql[n][i][0], ql[n][i][1]);
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const bool in = w.on[s] && u + 16 * s + 8 * r + g < c1;
          const float ks = __uint_as_float(w.kp[s][r] << 16), km = __uint_as_float(w.kp[s][r] & 0xffff0000u);
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            const float d0 = (float)(256 * dh[n][2 * r] + dl[n][2 * r]), d1 = (float)(256 * dh[n][2 * r + 1] + dl[n][2 * r + 1]);
            xs[n][s][2 * r] = in ? fmaf(ks, d0 * f0[n], km * q0[n]) : -INFINITY;
            xs[n][s][2 * r + 1] = in ? fmaf(ks, d1 * f1[n], km * q1[n]) : -INFINITY;
            b0[n] = fmaxf(b0[n], xs[n][s][2 * r]);
            b1[n] = fmaxf(b1[n], xs[n][s][2 * r + 1]);
          }
          smax = fmaxf(smax, in ? fabsf(__uint_as_float(w.vp[s][r] << 16)) : 0.f);
        }
      }
#pragma unroll
      for (int n = 0; n < NS; ++n) raise = raise || b0[n] > m0[n] || b1[n] > m1[n];
      if (__any_sync(0xffffffffu, raise || smax * sc > 1.f)) {
        // Set the references 2 above the largest score, so that weights begin at 1/4 and may grow to 1, and the scales'
        // factor so that they lie between 1/2 and 1.
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, o));
        const bool rescale = smax * sc > 1.f;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            b0[n] = fmaxf(b0[n], __shfl_xor_sync(0xffffffffu, b0[n], o));
            b1[n] = fmaxf(b1[n], __shfl_xor_sync(0xffffffffu, b1[n], o));
          }
          const float n0 = b0[n] > m0[n] ? b0[n] + 2.f : m0[n], n1 = b1[n] > m1[n] ? b1[n] + 2.f : m1[n];
          const float e0 = n0 == m0[n] ? 1.f : ex2(m0[n] - n0), e1 = n1 == m1[n] ? 1.f : ex2(m1[n] - n1);
          m0[n] = n0; m1[n] = n1;
          l0[n] *= e0; l1[n] *= e1; c0s[n] *= e0; c1s[n] *= e1;
          keep(n, e0, e1);
        }
        kept = true;
        if (rescale) sc = __uint_as_float((uint32_t)max(1, 253 - (int)(__float_as_uint(smax) >> 23)) << 23);
      }
      uint32_t wb[NS][2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        uint32_t tr[NS][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const bool in = w.on[s] && u + 16 * s + 8 * r + g < c1;
          const float vs = in ? __uint_as_float(w.vp[s][r] << 16) * sc * 65535.f : 0.f;
          const float vm = in ? __uint_as_float(w.vp[s][r] & 0xffff0000u) : 0.f;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            const float p0 = in ? ex2(xs[n][s][2 * r] - m0[n]) : 0.f, p1 = in ? ex2(xs[n][s][2 * r + 1] - m1[n]) : 0.f;
            l0[n] += p0; l1[n] += p1;
            c0s[n] = fmaf(p0, vm, c0s[n]); c1s[n] = fmaf(p1, vm, c1s[n]);
            // rounded to integers in the low 16 bits of 2^23 + w, column 2t in the low half, column 2t + 1 in the high one
            const uint32_t i0 = __float_as_uint(fmaf(p0, vs, 8388608.f)), i1 = __float_as_uint(fmaf(p1, vs, 8388608.f));
            tr[n][r] = transpose8x8(__byte_perm(i0, i1, 0x5410u));
          }
        }
        // now the weights of column g for keys 2t, 2t + 1 of each eight: the byte this column takes
#pragma unroll
        for (int n = 0; n < NS; ++n) wb[n][s] = __byte_perm(tr[n][0], tr[n][1], part_sel);
      }
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        uint32_t y[2][4];  // [half][j]: codes 2j (low nibbles) and 2j + 1 of the lane's four keys, a byte per key
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint32_t z0 = __byte_perm(w.v[s][0][i], w.v[s][1][i], 0x5140u), z1 = __byte_perm(w.v[s][2][i], w.v[s][3][i], 0x5140u);
          const uint32_t z2 = __byte_perm(w.v[s][0][i], w.v[s][1][i], 0x7362u), z3 = __byte_perm(w.v[s][2][i], w.v[s][3][i], 0x7362u);
          y[s][0] = __byte_perm(z0, z1, 0x5410u);
          y[s][1] = __byte_perm(z0, z1, 0x7632u);
          y[s][2] = __byte_perm(z2, z3, 0x5410u);
          y[s][3] = __byte_perm(z2, z3, 0x7632u);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a0 = even(y[0][j]), a1 = odd(y[0][j]), a2 = even(y[1][j]), a3 = odd(y[1][j]);
#pragma unroll
          for (int n = 0; n < NS; ++n) mma_u8u8(acc[n][4 * i + j], a0, a1, a2, a3, wb[n][0], wb[n][1]);
        }
      }
    };

    constexpr int STEP = MW * kTileKeys;
    int u = c0 + warp * kTileKeys;
    T ta, tb;
    if (u < c1) {
      load(ta, places(u), u);
      Place nx = places(u + STEP);
      for (;;) {
        load(tb, nx, u + STEP);
        nx = places(u + 2 * STEP);
        compute(ta, u);
        u += STEP;
        if (u >= c1) break;
        load(ta, nx, u + STEP);
        nx = places(u + 2 * STEP);
        compute(tb, u);
        u += STEP;
        if (u >= c1) break;
      }
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
      keep(n, 1.f, 1.f);
      if (t < 2 && g == 0) {
        s_m[warp][4 * n + 2 * t] = m0[n]; s_m[warp][4 * n + 2 * t + 1] = m1[n];
        s_l[warp][4 * n + 2 * t] = l0[n]; s_l[warp][4 * n + 2 * t + 1] = l1[n];
        s_c[warp][4 * n + 2 * t] = c0s[n]; s_c[warp][4 * n + 2 * t + 1] = c1s[n];
      }
    }
    __syncthreads();
    const bool whole = x == s0 && x1 == s1;
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
      if (whole) {
        ((bf16*)a.o)[(size_t)b * a.ldo + head0 * HS + e] = __float2bfloat16_rn(gl == 0.f ? 0.f : v / gl);
      } else {
        part[c * (HS + 2) + d] = v;
        if (d == 0) {
          part[c * (HS + 2) + HS] = gm * 0.6931471805599453f;  // the joining kernel counts in powers of e
          part[c * (HS + 2) + HS + 1] = gl;
        }
      }
    }
    __syncthreads();  // s_o is reused by the next segment
    x = x1;
  }
}

template <int HS> int32_t launch_hs(const Kv4DecodeArgs& a, int grid, cudaStream_t stream) {
  const int ps = a.pool.page_size;
  const int shift = (ps & (ps - 1)) == 0 ? __builtin_ctz((unsigned)ps) : -1;
  const size_t smem = (size_t)(a.batch + 1) * sizeof(int32_t);
  auto go = [&](auto kern) { return launch_pdl(kern, dim3(grid), dim3(MW * 32), smem, stream, a, shift); };
  const bool p32 = ps % 32 == 0;
  if (a.cols > 4) {
    B200_CUDA_OK(p32 ? go(kv4_decode_mma_kernel<HS, 2, true>) : go(kv4_decode_mma_kernel<HS, 2, false>));
  } else {
    B200_CUDA_OK(p32 ? go(kv4_decode_mma_kernel<HS, 1, true>) : go(kv4_decode_mma_kernel<HS, 1, false>));
  }
  B200_LAUNCH_OK("kv4_decode_mma_kernel");
  return B200_OK;
}

}  // namespace

bool kv4_decode_mma_supports(const Kv4DecodeArgs& a) {
  return a.dtype == B200_BF16 && (a.pool.head_size == 64 || a.pool.head_size == 128) && a.pool.page_size % 16 == 0;
}

int kv4_decode_mma_grid(int cols) { return (cols > 4 ? 2 : 3) * sm_count(); }

int32_t launch_kv4_decode_mma(const Kv4DecodeArgs& a, int grid, cudaStream_t stream) {
  if (a.pool.head_size == 64) return launch_hs<64>(a, grid, stream);
  return launch_hs<128>(a, grid, stream);
}

}  // namespace b200
