// Decode attention over the 4-bit cache with the codes as matrix operands (bf16 queries, head size 64 or 128, pages of a
// multiple of 16 rows, grouped heads).
//
// A byte of codes holds two elements, so at HBM speed an SM receives 23 bytes and would have to expand and multiply 46
// elements per cycle for q.k and for p.v -- more than its FP32 lanes do.  The codes therefore go into mma.sync
// (m16n8k16, bf16, fp32 sums) as they are: a 4-bit code n shifted into bits 3..6 of a bf16 whose exponent is that of 1.0
// IS the number 1 + n/16, exactly, so two elements cost one shift and one logic operation.  The row's scale s and
// minimum m enter afterwards, once per row:
//   q.k = 16 s sum q (1 + n/16) + (m - 16 s) sum q
//   o   = sum_j (16 s_j p_j) (1 + n_j/16) + sum_j p_j (m_j - 16 s_j)
// The 16 rows of an A operand are 16 keys (q.k) or 16 head dimensions (p.v); its 8 columns are the query heads of the
// group.  The order of the elements inside a contraction is free, so a lane takes 16 contiguous bytes of a key row and
// the query fragments are laid out to match; nothing is shuffled.  The weights 16 s p are kept to 16 bits as the sum of
// two bf16 numbers: with up to four heads both parts share one product (columns 0..3 and 4..7 carry the same heads, the
// first the leading part, the last the rest), with five to eight heads a second product adds the rest.  Groups beyond
// eight are cut into subsets of eight.
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
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// codes J and J + 4 of a word as the bf16 pair (1 + n/16)
template <int J> __device__ __forceinline__ uint32_t expand(uint32_t x) {
  const uint32_t y = J == 0 ? x << 3 : x >> (J == 0 ? 0 : 4 * J - 3);
  return (y & 0x00780078u) | 0x3f803f80u;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

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

// WIDE: five to eight heads per subset.
template <int HS, bool WIDE>
__global__ void __launch_bounds__(MW * 32, 3) kv4_decode_mma_kernel(Kv4DecodeArgs a, int page_shift) {
  using T = Tile<HS>;
  constexpr int KW = T::KW, VW = T::VW, MT = HS / 16;
  extern __shared__ int32_t pre[];
  __shared__ int32_t warp_sums[MW];
  __shared__ float s_o[MW][8][HS + 4], s_m[MW][8], s_l[MW][8];
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
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(p.codes);
  const size_t half = kv4_half(p);
  const int group = a.n_heads / p.n_kv_heads;
  const float sl2 = a.scale * 1.4426950408889634f;
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

    auto place = [&](int u, int* page, int* row) {  // u: first key of a 16-key half
      const int slot = page_shift >= 0 ? u >> page_shift : u / p.page_size;
      *row = u - slot * p.page_size;
      *page = u < c1 ? *(table + slot) : -1;
    };
    struct Place { int page[2], row[2]; };
    auto places = [&](int u) {
      Place q;
      place(u, &q.page[0], &q.row[0]);
      place(u + 16, &q.page[1], &q.row[1]);
      return q;
    };
    auto load = [&](T& w, const Place& q, int u) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        w.on[s] = u + 16 * s < c1;
        if (w.on[s] && (unsigned)q.page[s] >= (unsigned)p.n_pages) {
          w.on[s] = false;
          if (lane == 0) atomicOr(a.status, ST_BAD_PAGE);
        }
        if (w.on[s]) {
          const size_t row = ((size_t)q.page[s] * p.n_kv_heads + hk) * p.page_size + q.row[s];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            load_words<KW>(codes + (row + g + 8 * r) * (HS / 8) + t * KW, w.k[s][r]);
            w.kp[s][r] = *(p.params + row + g + 8 * r);
            w.vp[s][r] = *(p.params + half + row + g + 8 * r);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            load_words<VW>(codes + (half + row + 2 * t + (j & 1) + 8 * (j >> 1)) * (HS / 8) + g * VW, w.v[s][j]);
        }
      }
    };

    // query fragments: column g; the elements a lane's words hold, in their order
    uint32_t qf[2 * KW][2];
    float qs = 0.f;
    {
      const int col = WIDE ? g : (g & 3);
      const bool on = col < n_cols;
      const bf16* q = (const bf16*)a.q + (size_t)b * a.ldq + (head0 + (on ? col : 0)) * HS + t * (HS / 4);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          e[i] = on ? to_f32(q[8 * w + i]) : 0.f;
          qs += e[i];
        }
        qf[2 * w][0] = pack2(e[0], e[4]);
        qf[2 * w][1] = pack2(e[1], e[5]);
        qf[2 * w + 1][0] = pack2(e[2], e[6]);
        qf[2 * w + 1][1] = pack2(e[3], e[7]);
      }
    }
    qs += __shfl_xor_sync(0xffffffffu, qs, 1);
    qs += __shfl_xor_sync(0xffffffffu, qs, 2);
    const float q0 = __shfl_sync(0xffffffffu, qs, 8 * t), q1 = __shfl_sync(0xffffffffu, qs, 8 * t + 4);  // columns 2t, 2t + 1

    float acc[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY;            // reference maxima of columns 2t, 2t + 1 (uniform over g)
    float l0 = 0.f, l1 = 0.f, k0s = 0.f, k1s = 0.f;  // this lane's share of sum p and of sum p (m - 16 s)

    auto compute = [&](const T& w, int u) {
      float sc[2][4];
      float bm0 = -INFINITY, bm1 = -INFINITY;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        if (w.on[s]) {
#pragma unroll
          for (int i = 0; i < KW; ++i) {
            const uint32_t ka = w.k[s][0][i], kb = w.k[s][1][i];
            mma16816(d, expand<0>(ka), expand<0>(kb), expand<1>(ka), expand<1>(kb), qf[2 * i][0], qf[2 * i][1]);
            mma16816(d, expand<2>(ka), expand<2>(kb), expand<3>(ka), expand<3>(kb), qf[2 * i + 1][0], qf[2 * i + 1][1]);
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const bool in = w.on[s] && u + 16 * s + 8 * r + g < c1;
          const float s16 = 16.f * __uint_as_float(w.kp[s][r] << 16);
          const float ka = s16 * sl2, kc = (__uint_as_float(w.kp[s][r] & 0xffff0000u) - s16) * sl2;
          sc[s][2 * r] = in ? fmaf(ka, d[2 * r], kc * q0) : -INFINITY;
          sc[s][2 * r + 1] = in ? fmaf(ka, d[2 * r + 1], kc * q1) : -INFINITY;
          bm0 = fmaxf(bm0, sc[s][2 * r]);
          bm1 = fmaxf(bm1, sc[s][2 * r + 1]);
        }
      }
      if (__any_sync(0xffffffffu, bm0 > m0 + 8.f || bm1 > m1 + 8.f)) {
        // raise the references of the columns to the tile's maxima; until then weights stay below 2^8
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          bm0 = fmaxf(bm0, __shfl_xor_sync(0xffffffffu, bm0, o));
          bm1 = fmaxf(bm1, __shfl_xor_sync(0xffffffffu, bm1, o));
        }
        const float n0 = fmaxf(m0, bm0), n1 = fmaxf(m1, bm1);
        const float f0 = n0 == m0 ? 1.f : ex2(m0 - n0), f1 = n1 == m1 ? 1.f : ex2(m1 - n1);
        m0 = n0; m1 = n1;
        l0 *= f0; l1 *= f1; k0s *= f0; k1s *= f1;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          acc[i][0] *= f0; acc[i][1] *= f1; acc[i][2] *= f0; acc[i][3] *= f1;
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (!w.on[s]) continue;
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const bool in = u + 16 * s + 8 * r + g < c1;
          const float p0 = in ? ex2(sc[s][2 * r] - m0) : 0.f, p1 = in ? ex2(sc[s][2 * r + 1] - m1) : 0.f;
          const float s16 = in ? 16.f * __uint_as_float(w.vp[s][r] << 16) : 0.f;
          const float mc = in ? __uint_as_float(w.vp[s][r] & 0xffff0000u) - s16 : 0.f;
          l0 += p0; l1 += p1;
          k0s = fmaf(p0, mc, k0s); k1s = fmaf(p1, mc, k1s);
          const float w0 = p0 * s16, w1 = p1 * s16;
          const uint32_t h = pack2(w0, w1);
          const uint32_t rest = pack2(w0 - __uint_as_float(h << 16), w1 - __uint_as_float(h & 0xffff0000u));
          if (WIDE) {
            hi[r] = transpose8x8(h);
            lo[r] = transpose8x8(rest);
          } else {
            hi[r] = transpose8x8(t < 2 ? h : rest);
          }
        }
#pragma unroll
        for (int i = 0; i < VW; ++i) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {  // codes 0..3, then 4..7 of the words
            const uint32_t sel = y ? 0x7632u : 0x5410u;
            const uint32_t a01 = __byte_perm(w.v[s][0][i], w.v[s][1][i], sel), a23 = __byte_perm(w.v[s][2][i], w.v[s][3][i], sel);
            const uint32_t e0 = expand<0>(a01), e1 = expand<1>(a01), e2 = expand<2>(a01), e3 = expand<3>(a01);
            const uint32_t f0 = expand<0>(a23), f1 = expand<1>(a23), f2 = expand<2>(a23), f3 = expand<3>(a23);
            mma16816(acc[4 * i + 2 * y], e0, e1, f0, f1, hi[0], hi[1]);
            mma16816(acc[4 * i + 2 * y + 1], e2, e3, f2, f3, hi[0], hi[1]);
            if (WIDE) {
              mma16816(acc[4 * i + 2 * y], e0, e1, f0, f1, lo[0], lo[1]);
              mma16816(acc[4 * i + 2 * y + 1], e2, e3, f2, f3, lo[0], lo[1]);
            }
          }
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
    // the lanes of a column
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
      k0s += __shfl_xor_sync(0xffffffffu, k0s, o);
      k1s += __shfl_xor_sync(0xffffffffu, k1s, o);
    }
    if (!WIDE) {  // the rest of the weights stands four columns to the right
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += __shfl_xor_sync(0xffffffffu, acc[i][j], 2);
    }
    if (WIDE || t < 2) {
#pragma unroll
      for (int i = 0; i < VW; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // elements 2j, 2j + 1 of the word
          const int d = g * (HS / 8) + 8 * i + 2 * j;
          s_o[warp][2 * t][d] = acc[4 * i + j][0] + k0s;
          s_o[warp][2 * t + 1][d] = acc[4 * i + j][1] + k1s;
          s_o[warp][2 * t][d + 1] = acc[4 * i + j][2] + k0s;
          s_o[warp][2 * t + 1][d + 1] = acc[4 * i + j][3] + k1s;
        }
      }
      if (g == 0) {
        s_m[warp][2 * t] = m0; s_m[warp][2 * t + 1] = m1;
        s_l[warp][2 * t] = l0; s_l[warp][2 * t + 1] = l1;
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
        v = fmaf(s_o[w][c][d], f, v);
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
  if (a.cols > 4) {
    B200_CUDA_OK(launch_pdl(kv4_decode_mma_kernel<HS, true>, dim3(grid), dim3(MW * 32), smem, stream, a, shift));
  } else {
    B200_CUDA_OK(launch_pdl(kv4_decode_mma_kernel<HS, false>, dim3(grid), dim3(MW * 32), smem, stream, a, shift));
  }
  B200_LAUNCH_OK("kv4_decode_mma_kernel");
  return B200_OK;
}

}  // namespace

bool kv4_decode_mma_supports(const Kv4DecodeArgs& a) {
  return a.dtype == B200_BF16 && (a.pool.head_size == 64 || a.pool.head_size == 128) && a.pool.page_size % 16 == 0;
}

int kv4_decode_mma_grid() { return 3 * sm_count(); }

int32_t launch_kv4_decode_mma(const Kv4DecodeArgs& a, int grid, cudaStream_t stream) {
  if (a.pool.head_size == 64) return launch_hs<64>(a, grid, stream);
  return launch_hs<128>(a, grid, stream);
}

}  // namespace b200
