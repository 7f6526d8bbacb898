// The 4-bit key/value cache: append (quantise into pages), read back, and decode attention.
//
// Append.  A row x of one head becomes
//   minimum = bf16 rounded down of min x,   scale = bf16 rounded up of (max x - minimum) / 15,
//   code    = round-half-even((x - minimum) / scale) in 0..15.
// With those directions of rounding every x lies between the values of code 0 and code 15, so the error is at most half
// a scale.  A row that holds an infinity or NaN (or whose spread overflows) gets NaN parameters and reads back as NaN:
// one bad value must not come back as a plausible one.
// A warp takes a packed row (or, when rows are few, a part of its heads): it finds the row's sequence and page once, then
// hs/8 lanes share a (head, half), 8 elements and one 32-bit word of codes each.  A quotient is a product with the
// reciprocal, rounded, and then checked against its exact remainder, which costs half of a division; elements go two at a
// time through the packed fp32 instructions, minimum and maximum through one packed 16-bit reduction.
// Bound: bytes of the inputs plus hs/2 + 4 per row and half at HBM speed.  What bounds it now is instruction issue (2.7 of 4
// per cycle before the packed forms) and the look-ups in front of the first store: 15,398 ragged prompt rows of 8 heads of 128,
// appended and read back, take 54 us, 119 us with plain divisions and a look-up per row and head.  More items in flight per
// warp, or fewer with more warps, changed nothing.
#include "kv4.cuh"
#include "attention_packed.cuh"

#include <algorithm>
#include <type_traits>

namespace b200 {

namespace {

__host__ __device__ constexpr int lanes_of(int hs) { return hs <= 16 ? 2 : hs <= 32 ? 4 : hs <= 64 ? 8 : 16; }

__device__ __forceinline__ float bf16_down(float x) {
  const uint32_t b = __float_as_uint(x), cut = b & 0xffff0000u;
  return __uint_as_float((b >> 31) && cut != b ? cut + 0x10000u : cut);
}
__device__ __forceinline__ float bf16_up_nonneg(float x) { return __uint_as_float((__float_as_uint(x) + 0xffffu) & 0xffff0000u); }

struct Kv4RowsArgs {
  Kv4Pool pool;
  const int32_t* cu = nullptr;      // [n_seqs + 1]
  const int32_t* before = nullptr;  // [n_seqs] rows each sequence held already, or null
  int n_seqs = 0, rows = 0;
  uint32_t* status = nullptr;
};

// Page and row inside the page of packed row t, the same for all lanes of the warp; false when the row belongs to no
// sequence or the page table has no valid page for it.
__device__ __forceinline__ bool place_of(const Kv4RowsArgs& a, int t, int* page, int* in_page) {
  const int s = seq_of_row_warp(a.cu, a.n_seqs, t);
  if (s < 0 || s >= a.n_seqs) return false;
  const long long pos = (long long)(t - a.cu[s]) + (a.before ? a.before[s] : 0);
  if (pos < 0 || pos >= (long long)a.pool.max_pages * a.pool.page_size || pos > 0x7fffffffLL) {
    if ((threadIdx.x & 31) == 0) atomicOr(a.status, ST_BAD_PAGE);
    return false;
  }
  const int slot = (int)pos / a.pool.page_size;
  *in_page = (int)pos - slot * a.pool.page_size;
  *page = a.pool.table[(size_t)s * a.pool.max_pages + slot];
  if ((unsigned)*page >= (unsigned)a.pool.n_pages) {
    if ((threadIdx.x & 31) == 0) atomicOr(a.status, ST_BAD_PAGE);
    return false;
  }
  return true;
}

constexpr int AT = 256;  // threads of the append and read kernels

__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Minimum and maximum over the L lanes of a group, NaN if there is one.
template <int L> __device__ __forceinline__ float group_min(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = min_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int L> __device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// a / b from the correctly rounded reciprocal of b: the product corrected once by its exact remainder is the rounded
// quotient (Markstein), so halves come out as halves.  For numbers away from the ends of the range.
__device__ __forceinline__ float divide(float a, float b, float inv_b) {
  const float q = a * inv_b;
  return fmaf(fmaf(-q, b, a), inv_b, q);
}

// Rows of equal elements, of a spread at the ends of the fp32 range, and rows that are not finite.
__device__ __noinline__ uint2 quantise_rare(float4 x, float4 y, float mn, float spread) {
  if (!(spread < INFINITY) || !(mn > -INFINITY)) return make_uint2(0u, 0x7fc07fc0u);
  const float scale = bf16_up_nonneg(__fdiv_rn(spread, 15.f));
  uint32_t w = 0u;
  if (scale > 0.f) {
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= (uint32_t)fminf(rintf(__fdiv_rn(v[e] - mn, scale)), 15.f) << (4 * e);
  }
  return make_uint2(w, __byte_perm(__float_as_uint(scale), __float_as_uint(mn), 0x7632));
}

__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Eight elements as they stand in memory.  range<L>: their smallest and largest number over the L lanes of a group (lanes
// that are not `on` count for nothing), NaN if there is one.
template <typename T> struct Raw8;
template <> struct Raw8<bf16> {
  uint4 r;
  // both in one word, the largest negated: one shuffle and one minimum per step
  template <int L> __device__ __forceinline__ float2 range(bool on) const {
    const uint32_t lo = min2_nan(min2_nan(r.x, r.y), min2_nan(r.z, r.w)), hi = max2_nan(max2_nan(r.x, r.y), max2_nan(r.z, r.w));
    uint32_t m = min2_nan(__byte_perm(lo, hi, 0x5410) ^ 0x80000000u, __byte_perm(lo, hi, 0x7632) ^ 0x80000000u);
    if (!on) m = 0x7f807f80u;
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) m = min2_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    return make_float2(__uint_as_float(m << 16), __uint_as_float((m & 0xffff0000u) ^ 0x80000000u));
  }
  __device__ __forceinline__ void load(const bf16* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void set(int e, bf16 v) {
    uint32_t& w = (&r.x)[e >> 1];
    const uint32_t b = *reinterpret_cast<const uint16_t*>(&v);
    w = (e & 1) ? (w & 0xffffu) | (b << 16) : (w & 0xffff0000u) | b;
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <> struct Raw8<float> {
  float4 a, b;
  template <int L> __device__ __forceinline__ float2 range(bool on) const {
    float lo = min3_nan(min3_nan(a.x, a.y, a.z), min3_nan(a.w, b.x, b.y), min_nan(b.z, b.w));
    float hi = max3_nan(max3_nan(a.x, a.y, a.z), max3_nan(a.w, b.x, b.y), max_nan(b.z, b.w));
    return make_float2(group_min<L>(on ? lo : INFINITY), group_max<L>(on ? hi : -INFINITY));
  }
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void set(int e, float v) { (e < 4 ? (&a.x)[e] : (&b.x)[e - 4]) = v; }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
};

// `part` of `parts` equal shares of the 2 n_kv_heads (half, head) items of a row; U items per lane group in flight, the
// first of them requested before the row's place is looked up.
template <typename T, int HS>
__global__ void __launch_bounds__(AT, 4) kv4_append_kernel(Kv4RowsArgs a, const T* __restrict__ k, const T* __restrict__ v,
                                                           int ldk, int ldv, bool vec, int parts, int per_part) {
  constexpr int LPR = lanes_of(HS), GPW = 32 / LPR, U = sizeof(T) == 2 ? 4 : 2;
  const int lane = threadIdx.x & 31, li = lane % LPR, sub = lane / LPR;
  const long long w = (long long)blockIdx.x * (AT / 32) + (threadIdx.x >> 5);
  const int t = (int)(w / parts), part = (int)(w - (long long)t * parts);
  if (t >= a.rows) return;
  const int nk = a.pool.n_kv_heads;
  const int first = part * per_part, last = min(2 * nk, first + per_part);
  const bool lane_on = li * 8 < HS;
  const T* kt = k + (size_t)t * ldk + li * 8;
  const T* vt = v + (size_t)t * ldv + li * 8;
  Raw8<T> raw[U];
  auto load = [&](int i0) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int item = i0 + j * GPW + sub;
      if (item < last && lane_on) {
        const T* src = item >= nk ? vt + (item - nk) * HS : kt + item * HS;
        if (vec) {
          raw[j].load(src);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) raw[j].set(e, src[e]);
        }
      }
    }
  };
  load(first);
  int page, in_page;
  if (!place_of(a, t, &page, &in_page)) return;
  const size_t row0 = (size_t)page * nk * a.pool.page_size + in_page, half = kv4_half(a.pool);
  uint32_t* codes_k = reinterpret_cast<uint32_t*>(a.pool.codes) + row0 * (HS / 8) + li;
  uint32_t* codes_v = codes_k + half * (HS / 8);
  uint32_t* prm_k = a.pool.params + row0;
  for (int i0 = first; i0 < last; i0 += U * GPW) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int item = i0 + j * GPW + sub;
      if (i0 + j * GPW >= last) break;  // the same for the warp
      float x[8];
      raw[j].get(x);
      const float2 range = raw[j].template range<LPR>(item < last && lane_on);
      const float mn = sizeof(T) == 2 ? range.x : bf16_down(range.x);  // a 16-bit minimum is one already
      const float spread = range.y - mn;
      uint32_t word, prm;
      if (spread > 0x1p-90f && spread < 0x1p90f) {
        const float scale = bf16_up_nonneg(divide(spread, 15.f, 1.f / 15.f));
        float inv;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
        inv = fmaf(fmaf(-scale, inv, 1.f), inv, inv);  // correctly rounded: no 8-bit number has a reciprocal near a midpoint
        // `divide` for elements e and e + 4 at a time; adding 1.5 * 2^23 rounds to integers, ties to even
        const float2 mn2 = make_float2(-mn, -mn), inv2 = make_float2(inv, inv), ns2 = make_float2(-scale, -scale);
        const float2 up = make_float2(12582912.f, 12582912.f), down = make_float2(-12582912.f, -12582912.f);
        float2 c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 d = __fadd2_rn(make_float2(x[e], x[e + 4]), mn2);
          const float2 q = __fmul2_rn(d, inv2);
          c[e] = __fadd2_rn(__fadd2_rn(__ffma2_rn(__ffma2_rn(q, ns2, d), inv2, q), up), down);
        }
        // four codes are a number below 2^16: packed by the multiply-add pipe, the integer pipe being the busier one
        const float2 f16 = make_float2(16.f, 16.f), f256 = make_float2(256.f, 256.f), base = make_float2(8388608.f, 8388608.f);
        const float2 w4 = __fadd2_rn(__ffma2_rn(__ffma2_rn(c[3], f16, c[2]), f256, __ffma2_rn(c[1], f16, c[0])), base);
        word = __byte_perm(__float_as_uint(w4.x), __float_as_uint(w4.y), 0x5410);
        prm = __byte_perm(__float_as_uint(scale), __float_as_uint(mn), 0x7632);
      } else {
        const uint2 r = quantise_rare(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), mn, spread);
        word = r.x;
        prm = r.y;
      }
      if (item < last) {
        const bool is_v = item >= nk;
        const size_t at = (size_t)((unsigned)(is_v ? item - nk : item) * (unsigned)a.pool.page_size);  // inside a page: 32 bits
        if (lane_on) (is_v ? codes_v : codes_k)[at * (HS / 8)] = word;
        if (li == 0) (is_v ? prm_k + half : prm_k)[at] = prm;
      }
    }
    load(i0 + U * GPW);
  }
}

// Reads packed rows back: minimum + scale * code (the product is exact in fp32), rounded to T.
template <typename T, int HS>
__global__ void __launch_bounds__(AT) kv4_read_kernel(Kv4RowsArgs a, T* __restrict__ k, T* __restrict__ v, int ldk, int ldv,
                                                      bool vec, int parts, int per_part) {
  constexpr int LPR = lanes_of(HS), GPW = 32 / LPR, U = 4;
  const int lane = threadIdx.x & 31, li = lane % LPR, sub = lane / LPR;
  const long long w = (long long)blockIdx.x * (AT / 32) + (threadIdx.x >> 5);
  const int t = (int)(w / parts), part = (int)(w - (long long)t * parts);
  if (t >= a.rows) return;
  int page, in_page;
  if (!place_of(a, t, &page, &in_page)) return;
  const int nk = a.pool.n_kv_heads;
  const int first = part * per_part, last = min(2 * nk, first + per_part);
  const size_t row0 = (size_t)page * nk * a.pool.page_size + in_page, half = kv4_half(a.pool);
  if (li * 8 >= HS) return;
  const uint32_t* codes_k = reinterpret_cast<const uint32_t*>(a.pool.codes) + row0 * (HS / 8) + li;
  const uint32_t* codes_v = codes_k + half * (HS / 8);
  const uint32_t* prm_k = a.pool.params + row0;
  T* kt = k + (size_t)t * ldk + li * 8;
  T* vt = v + (size_t)t * ldv + li * 8;
  for (int i0 = first; i0 < last; i0 += U * GPW) {
    uint32_t word[U], prm[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int item = i0 + j * GPW + sub;
      const bool is_v = item >= nk;
      if (item < last) {
        const size_t at = (size_t)((unsigned)(is_v ? item - nk : item) * (unsigned)a.pool.page_size);
        word[j] = (is_v ? codes_v : codes_k)[at * (HS / 8)];
        prm[j] = (is_v ? prm_k + half : prm_k)[at];
      }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int item = i0 + j * GPW + sub;
      if (item >= last) break;
      const bool is_v = item >= nk;
      const float scale = __uint_as_float(prm[j] << 16), mn = __uint_as_float(prm[j] & 0xffff0000u);
      const uint32_t even = word[j] & 0x0f0f0f0fu, odd = (word[j] >> 4) & 0x0f0f0f0fu;
      const float2 base = make_float2(-8388608.f, -8388608.f), scale2 = make_float2(scale, scale), mn2 = make_float2(mn, mn);
      float x[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // 2^23 + code, less 2^23: exact
        const float2 n = make_float2(__uint_as_float(__byte_perm(even, 0x4b000000u, 0x7440 + e)),
                                     __uint_as_float(__byte_perm(odd, 0x4b000000u, 0x7440 + e)));
        const float2 y = __ffma2_rn(__fadd2_rn(n, base), scale2, mn2);
        x[2 * e] = y.x;
        x[2 * e + 1] = y.y;
      }
      T* dst = is_v ? vt + (item - nk) * HS : kt + item * HS;
      if (vec) {
        store8(dst, x);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) dst[e] = from_f32<T>(x[e]);
      }
    }
  }
}

// How many warps share a packed row: enough to fill the GPU when rows are few, never less than one item per lane group.
void split_rows(int rows, int n_kv_heads, int head_size, int* parts, int* per_part) {
  const int groups = 32 / lanes_of(head_size), items = 2 * n_kv_heads;
  const int want = std::max(1, 32 * sm_count() / std::max(1, rows));
  const int most = (items + groups - 1) / groups;
  *parts = std::min(want, most);
  *per_part = ((items + *parts - 1) / *parts + groups - 1) / groups * groups;
  *parts = (items + *per_part - 1) / *per_part;
}

// ---- decode attention on the CUDA cores ----------------------------------------------------------------------------
// One query head per segment; LPK lanes hold one key (8 dims each), so a warp-wide load brings in 32/LPK rows.  q.k is
// taken over the codes, scale and minimum enter once per row: s = scale * (q.code) + minimum * sum(q).  fp32 throughout.
// Bound by the FP32 lanes and the conversions of the codes: 8 x 4096 rows of 12 fp32 heads of 64 take 43 us, 0.66 TB/s.
constexpr int SW = 4, SG = 4;  // warps per CTA, keys in flight per lane

template <typename T, int HS>
__global__ void __launch_bounds__(SW * 32) kv4_decode_simt_kernel(Kv4DecodeArgs a) {
  constexpr int LPK = lanes_of(HS), KPW = 32 / LPK;
  extern __shared__ int32_t pre[];
  int32_t* lens = pre + a.batch + 1;
  __shared__ int32_t warp_sums[SW];
  __shared__ float s_acc[SW][HS], s_m[SW], s_l[SW];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LPK, li = lane % LPK;
  const bool lane_on = li * 8 < HS;
  pdl_launch_dependents();
  pdl_wait();  // everything below comes from the kernels before
  const UnitRange range = unit_range<SW * 32>(a, pre, lens, warp_sums);
  const Kv4Pool& p = a.pool;
  const int nseg = p.n_kv_heads * a.subs;
  const long long r0 = range.first, r1 = range.last;
  if (r0 == r1) {
    if (a.whole) zero_segment<T>(a);
    return;
  }
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(p.codes);
  const size_t half = kv4_half(p);
  int b = range.seq;
  for (long long x = r0; x < r1;) {
    while ((long long)pre[b + 1] * nseg <= x) ++b;
    const int nb = pre[b + 1] - pre[b];
    const long long base = (long long)pre[b] * nseg;
    const int seg = (int)((x - base) / nb);
    const long long s0 = base + (long long)seg * nb, s1 = s0 + nb;
    const long long x1 = r1 < s1 ? r1 : s1;
    const int hk = seg / a.subs, head = hk * a.subs + seg % a.subs;
    const int len = lens[b];
    const int c0 = (int)(x - s0) * kUnit, c1 = min(len, (int)(x1 - s0) * kUnit);
    const int32_t* table = p.table + (size_t)b * p.max_pages;

    float qf[8], acc[8], qsum = 0.f, m = -INFINITY, l = 0.f, cmin = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      qf[i] = lane_on ? to_f32(((const T*)a.q)[(size_t)b * a.ldq + head * HS + li * 8 + i]) * a.scale : 0.f;
      qsum += qf[i];
      acc[i] = 0.f;
    }
#pragma unroll
    for (int o = LPK / 2; o > 0; o >>= 1) qsum += __shfl_xor_sync(0xffffffffu, qsum, o);
    for (int u0 = c0 + warp * (SG * KPW); u0 < c1; u0 += SW * SG * KPW) {
      uint32_t kw[SG], vw[SG], kp[SG], vp[SG];
      bool live[SG];
#pragma unroll
      for (int g = 0; g < SG; ++g) {
        const int u = u0 + g * KPW + sub;
        live[g] = u < c1;
        kw[g] = vw[g] = kp[g] = vp[g] = 0u;
        if (live[g]) {
          const int page = *(table + u / p.page_size);
          live[g] = (unsigned)page < (unsigned)p.n_pages;
          if (live[g]) {
            const size_t row = ((size_t)page * p.n_kv_heads + hk) * p.page_size + u % p.page_size;
            kp[g] = p.params[row];
            vp[g] = p.params[row + half];
            if (lane_on) {
              kw[g] = codes[row * (HS / 8) + li];
              vw[g] = codes[(row + half) * (HS / 8) + li];
            }
          } else {
            atomicOr(a.status, ST_BAD_PAGE);
          }
        }
      }
      float s[SG], bm = -INFINITY;
#pragma unroll
      for (int g = 0; g < SG; ++g) {
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) d = fmaf(qf[i], (float)((kw[g] >> (4 * i)) & 15u), d);
#pragma unroll
        for (int o = LPK / 2; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        d = fmaf(__uint_as_float(kp[g] << 16), d, __uint_as_float(kp[g] & 0xffff0000u) * qsum);
        s[g] = live[g] ? d : -INFINITY;
        bm = fmaxf(bm, s[g]);
      }
      const float nm = fmaxf(m, bm);
      const float corr = m == nm ? 1.f : exp_by_build(m - nm);
      const float ref = nm == -INFINITY ? 0.f : nm;  // scores of minus infinity alone: no weight yet (a NaN keeps its own)
      l *= corr;
      cmin *= corr;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= corr;
#pragma unroll
      for (int g = 0; g < SG; ++g) {
        if (live[g]) {  // a row behind the end may hold anything
          const float pr = exp_by_build(s[g] - ref);
          l += pr;
          const float w = pr * __uint_as_float(vp[g] << 16);
          cmin = fmaf(pr, __uint_as_float(vp[g] & 0xffff0000u), cmin);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, (float)((vw[g] >> (4 * i)) & 15u), acc[i]);
        }
      }
      m = nm;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] += cmin;
    // key groups of the warp, then the warps of the CTA
#pragma unroll
    for (int o = LPK; o < 32; o <<= 1) {
      const float mo = __shfl_xor_sync(0xffffffffu, m, o), lo = __shfl_xor_sync(0xffffffffu, l, o);
      const float nm = fmaxf(m, mo);
      const float f0 = m == nm ? 1.f : exp_by_build(m - nm), f1 = mo == nm ? 1.f : exp_by_build(mo - nm);
      l = l * f0 + lo * f1;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = acc[i] * f0 + __shfl_xor_sync(0xffffffffu, acc[i], o) * f1;
      m = nm;
    }
    if (sub == 0 && lane_on) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s_acc[warp][li * 8 + i] = acc[i];
    }
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
    __syncthreads();
    float gm = -INFINITY;
#pragma unroll
    for (int w = 0; w < SW; ++w) gm = fmaxf(gm, s_m[w]);
    float f[SW], gl = 0.f;
#pragma unroll
    for (int w = 0; w < SW; ++w) {
      f[w] = s_m[w] == gm ? 1.f : exp_by_build(s_m[w] - gm);
      gl += s_l[w] * f[w];
    }
    const bool whole = x == s0 && x1 == s1;
    float* part = a.partials + (size_t)(2 * blockIdx.x + (x == r0 ? 0 : 1)) * (HS + 2);
    for (int e = threadIdx.x; e < HS; e += blockDim.x) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < SW; ++w) v = fmaf(s_acc[w][e], f[w], v);
      if (whole) ((T*)a.o)[(size_t)b * a.ldo + head * HS + e] = from_f32<T>(gl == 0.f ? 0.f : v / gl);
      else part[e] = v;
    }
    if (!whole && threadIdx.x == 0) { part[HS] = gm; part[HS + 1] = gl; }
    __syncthreads();  // s_acc is reused by the next segment
    x = x1;
  }
}

// Joins the partial blocks of the segments that several CTAs shared, and writes zeros for sequences without cached rows.
// One CTA per (segment, query head): its warps share the partials out (a single long sequence has one per SM and more).
constexpr int JW = 8;

template <typename T, int HS>
__global__ void __launch_bounds__(JW * 32) kv4_join_kernel(Kv4DecodeArgs a, int grid) {
  constexpr int N = (HS + 31) / 32;
  __shared__ float s_acc[JW][HS], s_l[JW];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nseg = a.pool.n_kv_heads * a.subs;
  const int c = blockIdx.x % a.cols, seg = blockIdx.x / a.cols % nseg, b = blockIdx.x / a.cols / nseg;
  const int group = a.n_heads / a.pool.n_kv_heads;
  const int first = (seg % a.subs) * a.cols;
  if (c >= group - first) return;  // the last subset of a head may be smaller
  pdl_launch_dependents();
  pdl_wait();
  const int p0 = a.prefix[b], nb = a.prefix[b + 1] - p0;
  const long long units = (long long)a.prefix[a.batch] * nseg;
  T* o = (T*)a.o + (size_t)b * a.ldo + ((seg / a.subs) * group + first + c) * HS;
  if (nb == 0) {
    for (int e = threadIdx.x; e < HS; e += blockDim.x) o[e] = from_f32<T>(0.f);
    return;
  }
  const int ctas = (int)(units < (long long)grid ? units : (long long)grid);
  const long long s0 = (long long)p0 * nseg + (long long)seg * nb, s1 = s0 + nb;
  const int ca = range_owner(units, ctas, s0), cb = range_owner(units, ctas, s1 - 1);
  if (ca == cb) return;  // finished by its CTA
  const size_t slot = (size_t)a.cols * (HS + 2);
  // only the first of the CTAs can have had another segment before this one
  const size_t first_slot = range_start(units, ctas, ca) == s0 ? 0 : 1;
  auto part = [&](int i) { return a.partials + (2 * (size_t)i + (i == ca ? first_slot : 0)) * slot + (size_t)c * (HS + 2); };
  float m = -INFINITY;
  for (int i = ca + lane; i <= cb; i += 32) m = fmaxf(m, part(i)[HS]);
  m = warp_max(m);
  float l = 0.f, acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
#pragma unroll 4
  for (int i = ca + warp; i <= cb; i += JW) {
    const float* q = part(i);
    const float f = q[HS] == m ? 1.f : exp_by_build(q[HS] - m);
    l = fmaf(q[HS + 1], f, l);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (HS % 32 == 0 || lane + 32 * j < HS) acc[j] = fmaf(q[lane + 32 * j], f, acc[j]);
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (HS % 32 == 0 || lane + 32 * j < HS) s_acc[warp][lane + 32 * j] = acc[j];
  if (lane == 0) s_l[warp] = l;
  __syncthreads();
  for (int e = threadIdx.x; e < HS; e += blockDim.x) {
    float v = 0.f, gl = 0.f;
#pragma unroll
    for (int w = 0; w < JW; ++w) {
      v += s_acc[w][e];
      gl += s_l[w];
    }
    o[e] = from_f32<T>(gl == 0.f ? 0.f : v / gl);
  }
}

template <typename F> int32_t by_type(const char* what, int dtype, int hs, F&& f) {
  auto go = [&](auto t) -> int32_t {
    switch (hs) {
      case 16: return f(t, std::integral_constant<int, 16>());
      case 32: return f(t, std::integral_constant<int, 32>());
      case 48: return f(t, std::integral_constant<int, 48>());
      case 64: return f(t, std::integral_constant<int, 64>());
      case 128: return f(t, std::integral_constant<int, 128>());
    }
    return fail(B200_ERR_BAD_SHAPE, "%s: head size %d is not one of 16/32/48/64/128", what, hs);
  };
  if (dtype == B200_F32) return go(float());
  if (dtype == B200_BF16) return go(bf16());
  return fail(B200_ERR_BAD_DTYPE, "%s: unsupported dtype %d", what, dtype);
}

int32_t check_pool(const char* what, const Kv4Pool& p) {
  if (p.n_pages < 0 || p.n_kv_heads <= 0 || p.page_size <= 0 || p.max_pages < 0 || p.head_size <= 0)
    return fail(B200_ERR_BAD_SHAPE, "%s: sizes must be positive", what);
  if ((long long)p.n_kv_heads * p.page_size > 0x7fffffffLL)
    return fail(B200_ERR_BAD_SHAPE, "%s: %d rows of %d heads are too many for one page", what, p.page_size, p.n_kv_heads);
  switch (p.head_size) {
    case 16: case 32: case 48: case 64: case 128: return B200_OK;
  }
  return fail(B200_ERR_BAD_SHAPE, "%s: head size %d is not one of 16/32/48/64/128", what, p.head_size);
}
int32_t check_pool_ptrs(const char* what, const Kv4Pool& p) {
  // (memory of no bytes may have no address: a pool without pages, page tables without columns)
  if ((p.n_pages > 0 && (!p.codes || !p.params)) || (p.max_pages > 0 && !p.table))
    return fail(B200_ERR_INVALID_ARG, "%s: null operand", what);
  if ((reinterpret_cast<uintptr_t>(p.codes) | reinterpret_cast<uintptr_t>(p.params)) & 3u)
    return fail(B200_ERR_MISALIGNED, "%s: codes and params must be 4-byte aligned", what);
  return B200_OK;
}

// Grid of the CUDA-core decode kernel: the CTAs an SM can hold (a range may hold less than a whole segment, so a single
// long sequence fills the GPU too).
int decode_simt_grid() { return 7 * sm_count(); }

long long table_units(int page_size, int max_pages) { return ((long long)max_pages * page_size + kUnit - 1) / kUnit; }

// (by what the kernels are made for: a tensor-core shape that another alignment sends to the CUDA cores counts as one)
int whole_units(int dtype, int head_size, int page_size) {
  return dtype == B200_BF16 && (head_size == 64 || head_size == 128) && page_size % 16 == 0 ? kWholeUnitsMma : kWholeUnitsSimt;
}

// How a step is shared out: CTAs of either kernel, segments whole or not, scratch.
struct DecodePlan {
  int mma_cols, mma_subs, mma_grid, simt_grid;
  bool whole;
  size_t prefix_bytes, bytes;
};
DecodePlan decode_plan(int batch, int n_heads, int n_kv_heads, int head_size, long long cap_units, int whole_units) {
  DecodePlan p;
  const int group = n_heads / n_kv_heads;
  const long long slice = std::min(batch, kMaxSlice);
  p.mma_cols = std::min(8, group);
  p.mma_subs = (group + p.mma_cols - 1) / p.mma_cols;
  const long long mma_segs = slice * n_kv_heads * p.mma_subs, simt_segs = slice * n_heads;
  const long long mma_max = kv4_decode_mma_grid(head_size, p.mma_cols), simt_max = decode_simt_grid();
  p.whole = cap_units <= whole_units && mma_segs <= mma_max && simt_segs <= simt_max;
  p.mma_grid = (int)std::max(1LL, std::min(mma_max, mma_segs * cap_units));
  p.simt_grid = (int)std::max(1LL, std::min(simt_max, simt_segs * cap_units));
  const size_t slots = std::max((size_t)p.simt_grid, (size_t)p.mma_grid * p.mma_cols);
  p.prefix_bytes = align_up((size_t)(slice + 1) * 4, 256);
  p.bytes = p.prefix_bytes + 2 * slots * (head_size + 2) * sizeof(float);
  if (p.whole) {
    p.mma_grid = (int)mma_segs;
    p.simt_grid = (int)simt_segs;
  }
  return p;
}

}  // namespace

}  // namespace b200

using namespace b200;

extern "C" {

int32_t b200_kv4_append(const void* k, const void* v, void* codes, void* params, const int32_t* page_table,
                        const int32_t* cu_seqlens, const int32_t* ctx_before, int32_t n_seqs, int32_t rows,
                        int32_t n_kv_heads, int32_t head_size, int32_t ldk, int32_t ldv, int32_t n_pages,
                        int32_t page_size, int32_t max_pages, int32_t dtype, b200_stream_t stream) {
  Kv4RowsArgs a;
  a.pool.codes = (uint8_t*)codes; a.pool.params = (uint32_t*)params; a.pool.table = page_table;
  a.pool.n_pages = n_pages; a.pool.n_kv_heads = n_kv_heads; a.pool.page_size = page_size;
  a.pool.head_size = head_size; a.pool.max_pages = max_pages;
  a.cu = cu_seqlens; a.before = ctx_before; a.n_seqs = n_seqs; a.rows = rows;
  B200_TRY(check_pool("kv4 append", a.pool));
  if (n_seqs < 0 || rows < 0) return fail(B200_ERR_BAD_SHAPE, "kv4 append: n_seqs=%d rows=%d", n_seqs, rows);
  if (ldk < (long long)n_kv_heads * head_size || ldv < (long long)n_kv_heads * head_size)
    return fail(B200_ERR_BAD_SHAPE, "kv4 append: a row pitch is smaller than the row");
  if (dtype != B200_F32 && dtype != B200_BF16) return fail(B200_ERR_BAD_DTYPE, "kv4 append: unsupported dtype %d", dtype);
  if (rows == 0 || n_seqs == 0) return B200_OK;
  if (!k || !v || !cu_seqlens) return fail(B200_ERR_INVALID_ARG, "kv4 append: null operand");
  B200_TRY(check_pool_ptrs("kv4 append", a.pool));
  a.status = device_status_word();
  if (!a.status) return fail(B200_ERR_CUDA, "no device status word");
  const bool vec = aligned16(k) && aligned16(v) && ldk % 8 == 0 && ldv % 8 == 0;
  int parts, per_part;
  split_rows(rows, n_kv_heads, head_size, &parts, &per_part);
  const long long blocks = ((long long)rows * parts + AT / 32 - 1) / (AT / 32);
  if (blocks > 0x7fffffffLL) return fail(B200_ERR_BAD_SHAPE, "kv4 append: too many rows");
  return by_type("kv4 append", dtype, head_size, [&](auto t, auto hs) -> int32_t {
    using T = decltype(t);
    constexpr int HS = decltype(hs)::value;
    kv4_append_kernel<T, HS><<<(unsigned)blocks, AT, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a, (const T*)k, (const T*)v, ldk, ldv, vec, parts, per_part);
    B200_LAUNCH_OK("kv4_append_kernel");
    return B200_OK;
  });
}

int32_t b200_kv4_read(void* k, void* v, const void* codes, const void* params, const int32_t* page_table,
                      const int32_t* cu_seqlens, const int32_t* ctx_before, int32_t n_seqs, int32_t rows,
                      int32_t n_kv_heads, int32_t head_size, int32_t ldk, int32_t ldv, int32_t n_pages,
                      int32_t page_size, int32_t max_pages, int32_t dtype, b200_stream_t stream) {
  Kv4RowsArgs a;
  a.pool.codes = (uint8_t*)const_cast<void*>(codes); a.pool.params = (uint32_t*)const_cast<void*>(params);
  a.pool.table = page_table;
  a.pool.n_pages = n_pages; a.pool.n_kv_heads = n_kv_heads; a.pool.page_size = page_size;
  a.pool.head_size = head_size; a.pool.max_pages = max_pages;
  a.cu = cu_seqlens; a.before = ctx_before; a.n_seqs = n_seqs; a.rows = rows;
  B200_TRY(check_pool("kv4 read", a.pool));
  if (n_seqs < 0 || rows < 0) return fail(B200_ERR_BAD_SHAPE, "kv4 read: n_seqs=%d rows=%d", n_seqs, rows);
  if (ldk < (long long)n_kv_heads * head_size || ldv < (long long)n_kv_heads * head_size)
    return fail(B200_ERR_BAD_SHAPE, "kv4 read: a row pitch is smaller than the row");
  if (dtype != B200_F32 && dtype != B200_BF16) return fail(B200_ERR_BAD_DTYPE, "kv4 read: unsupported dtype %d", dtype);
  if (rows == 0 || n_seqs == 0) return B200_OK;
  if (!k || !v || !cu_seqlens) return fail(B200_ERR_INVALID_ARG, "kv4 read: null operand");
  B200_TRY(check_pool_ptrs("kv4 read", a.pool));
  a.status = device_status_word();
  if (!a.status) return fail(B200_ERR_CUDA, "no device status word");
  const bool vec = aligned16(k) && aligned16(v) && ldk % 8 == 0 && ldv % 8 == 0;
  int parts, per_part;
  split_rows(rows, n_kv_heads, head_size, &parts, &per_part);
  const long long blocks = ((long long)rows * parts + AT / 32 - 1) / (AT / 32);
  if (blocks > 0x7fffffffLL) return fail(B200_ERR_BAD_SHAPE, "kv4 read: too many rows");
  return by_type("kv4 read", dtype, head_size, [&](auto t, auto hs) -> int32_t {
    using T = decltype(t);
    constexpr int HS = decltype(hs)::value;
    kv4_read_kernel<T, HS><<<(unsigned)blocks, AT, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a, (T*)k, (T*)v, ldk, ldv, vec, parts, per_part);
    B200_LAUNCH_OK("kv4_read_kernel");
    return B200_OK;
  });
}

int32_t b200_attention_decode_kv4_scratch_bytes(int32_t batch, int32_t n_heads, int32_t n_kv_heads, int32_t head_size,
                                                size_t* bytes) {
  if (!bytes) return fail(B200_ERR_INVALID_ARG, "bytes is null");
  if (batch < 0 || n_heads <= 0 || n_kv_heads <= 0 || head_size <= 0 || n_heads % n_kv_heads)
    return fail(B200_ERR_BAD_SHAPE, "kv4 decode: batch=%d heads=%d kv_heads=%d head_size=%d", batch, n_heads, n_kv_heads, head_size);
  *bytes = decode_plan(batch, n_heads, n_kv_heads, head_size, 0x7fffffffLL, 0).bytes;
  return B200_OK;
}

int32_t b200_attention_decode_kv4_scratch_bytes_for(int32_t batch, int32_t n_heads, int32_t n_kv_heads, int32_t head_size,
                                                    int32_t page_size, int32_t max_pages, int32_t dtype, size_t* bytes) {
  if (!bytes) return fail(B200_ERR_INVALID_ARG, "bytes is null");
  if (batch < 0 || n_heads <= 0 || n_kv_heads <= 0 || head_size <= 0 || n_heads % n_kv_heads || page_size <= 0 || max_pages < 0)
    return fail(B200_ERR_BAD_SHAPE, "kv4 decode: batch=%d heads=%d kv_heads=%d head_size=%d, %d pages of %d rows", batch, n_heads,
                n_kv_heads, head_size, max_pages, page_size);
  const DecodePlan plan = decode_plan(batch, n_heads, n_kv_heads, head_size, table_units(page_size, max_pages), whole_units(dtype, head_size, page_size));
  *bytes = plan.whole ? 0 : plan.bytes;
  return B200_OK;
}

int32_t b200_attention_decode_kv4(const void* q, const void* codes, const void* params, const int32_t* page_table,
                                  const int32_t* ctx_lens, void* o, void* scratch, size_t scratch_bytes, int32_t batch,
                                  int32_t n_heads, int32_t n_kv_heads, int32_t head_size, int32_t ldq, int32_t ldo,
                                  int32_t n_pages, int32_t page_size, int32_t max_pages, int32_t dtype, int32_t impl,
                                  b200_stream_t stream) {
  Kv4DecodeArgs a;
  a.pool.codes = (uint8_t*)const_cast<void*>(codes); a.pool.params = (uint32_t*)const_cast<void*>(params);
  a.pool.table = page_table;
  a.pool.n_pages = n_pages; a.pool.n_kv_heads = n_kv_heads; a.pool.page_size = page_size;
  a.pool.head_size = head_size; a.pool.max_pages = max_pages;
  B200_TRY(check_pool("kv4 decode", a.pool));
  if (batch < 0 || n_heads <= 0 || n_heads % n_kv_heads)
    return fail(B200_ERR_BAD_SHAPE, "kv4 decode: batch=%d, %d query heads over %d key heads", batch, n_heads, n_kv_heads);
  if (ldq < (long long)n_heads * head_size || ldo < (long long)n_heads * head_size)
    return fail(B200_ERR_BAD_SHAPE, "kv4 decode: a row pitch is smaller than the row");
  if (dtype != B200_F32 && dtype != B200_BF16) return fail(B200_ERR_BAD_DTYPE, "kv4 decode: unsupported dtype %d", dtype);
  if (impl < 0 || impl > 2) return fail(B200_ERR_INVALID_ARG, "impl %d is not 0, 1 or 2", impl);
  if (batch == 0) return B200_OK;
  const long long cap_units = table_units(page_size, max_pages);
  if (cap_units * std::min(batch, kMaxSlice) > 0x7fffffffLL)
    return fail(B200_ERR_BAD_SHAPE, "kv4 decode: %d page tables of %d pages of %d rows are too long together", batch, max_pages, page_size);
  const DecodePlan plan = decode_plan(batch, n_heads, n_kv_heads, head_size, cap_units, whole_units(dtype, head_size, page_size));
  if (!q || !o || !ctx_lens || (!scratch && !plan.whole)) return fail(B200_ERR_INVALID_ARG, "kv4 decode: null operand");
  B200_TRY(check_pool_ptrs("kv4 decode", a.pool));
  if (!aligned16(scratch)) return fail(B200_ERR_MISALIGNED, "kv4 decode: scratch must be 16-byte aligned");
  if (scratch && scratch_bytes < plan.bytes)
    return fail(B200_ERR_WORKSPACE, "kv4 decode: scratch needs %zu bytes, %zu given", plan.bytes, scratch_bytes);
  a.status = device_status_word();
  if (!a.status) return fail(B200_ERR_CUDA, "no device status word");
  a.n_heads = n_heads; a.ldq = ldq; a.ldo = ldo; a.dtype = dtype;
  a.scale = 1.f / sqrtf((float)head_size);
  a.prefix = (int32_t*)scratch;
  a.partials = (float*)((char*)scratch + plan.prefix_bytes);
  a.whole = plan.whole;
  const bool mma = impl != 2 && kv4_decode_mma_supports(a);
  if (impl == 1 && !mma)
    return fail(B200_ERR_UNSUPPORTED, "kv4 decode on tensor cores needs bf16, head size 64 or 128 and pages of a multiple of 16 rows");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  a.cols = mma ? plan.mma_cols : 1;
  a.subs = mma ? plan.mma_subs : n_heads / n_kv_heads;
  const int grid = mma ? plan.mma_grid : plan.simt_grid;  // (of a full slice: CTAs without work return)
  const size_t es = dtype == B200_BF16 ? 2 : 4;
  for (int b0 = 0; b0 < batch; b0 += kMaxSlice) {
    a.batch = std::min(kMaxSlice, batch - b0);
    a.q = (const char*)q + (size_t)b0 * ldq * es;
    a.o = (char*)o + (size_t)b0 * ldo * es;
    a.ctx = ctx_lens + b0;
    a.pool.table = page_table + (size_t)b0 * max_pages;
    B200_TRY(by_type("kv4 decode", dtype, head_size, [&](auto t, auto hs) -> int32_t {
      using T = decltype(t);
      constexpr int HS = decltype(hs)::value;
      if (mma) {
        B200_TRY(launch_kv4_decode_mma(a, grid, s));
      } else {
        B200_CUDA_OK(launch_pdl(kv4_decode_simt_kernel<T, HS>, dim3(grid), dim3(SW * 32), (2 * a.batch + 1) * sizeof(int32_t), s, a));
        B200_LAUNCH_OK("kv4_decode_simt_kernel");
      }
      if (plan.whole) return B200_OK;
      B200_CUDA_OK(launch_pdl(kv4_join_kernel<T, HS>, dim3(a.batch * n_kv_heads * a.subs * a.cols), dim3(JW * 32), 0, s, a, grid));
      B200_LAUNCH_OK("kv4_join_kernel");
      return B200_OK;
    }));
  }
  return B200_OK;
}

}  // extern "C"
