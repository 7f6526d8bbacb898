// Causal attention over packed sequences with grouped heads: argument blocks, the search of a row's sequence, and the
// row-by-row forms that every tile kernel falls back to.
//
// The sequences of a batch lie one behind the other in the rows of q, k, v and o; sequence s owns rows
// cu_seqlens[s] .. cu_seqlens[s+1] - 1.  Query row t attends to the rows of its own sequence up to itself:
//   s_tu = q_t.k_u / sqrt(hs),  start(t) <= u <= t        lse_t = log sum_u exp s_tu        o_t = sum_u exp(s_tu - lse_t) v_u
// Query head h reads key head h / (n_heads / n_kv_heads).
#pragma once

#include "common.cuh"

namespace b200 {

struct PackedArgs {
  const void* q = nullptr;   // [rows, ldq]
  const void* k = nullptr;   // [rows, ldk]
  const void* v = nullptr;   // [rows, ldv]
  void* o = nullptr;         // [rows, ldo]
  float* lse = nullptr;      // [n_heads, rows] or null
  const int32_t* cu = nullptr;  // [n_seqs + 1] on the device
  int n_seqs = 0, rows = 0, n_heads = 0, n_kv_heads = 0, head_size = 0;
  int ldq = 0, ldk = 0, ldv = 0, ldo = 0;
  int dtype = B200_BF16;
};

struct PackedBwdArgs {
  PackedArgs f;
  const void* d_o = nullptr;
  void* dq = nullptr;
  void* dk = nullptr;
  void* dv = nullptr;
  int lddo = 0, lddq = 0, lddk = 0, lddv = 0;
  float* delta = nullptr;  // scratch [n_heads, rows]: rowsum(P * dP)
};

bool packed_fwd_tc_supports(const PackedArgs& a);
int32_t launch_packed_fwd_tc(const PackedArgs& a, cudaStream_t stream);
int32_t launch_packed_fwd_simt(const PackedArgs& a, cudaStream_t stream);
bool packed_bwd_tc_supports(const PackedBwdArgs& a);
int32_t launch_packed_bwd_tc(const PackedBwdArgs& a, cudaStream_t stream);
int32_t launch_packed_bwd_simt(const PackedBwdArgs& a, cudaStream_t stream);

// ---- rows and sequences --------------------------------------------------------------------------------------------

// Largest s in [lo, hi] with cu[s] <= t, or lo - 1 when there is none: the sequence of row t (an empty sequence shares
// its first row with the next one and is never the largest), -1 before the first sequence, n_seqs behind the last one.
__device__ __forceinline__ int seq_of_row(const int32_t* __restrict__ cu, int lo, int hi, int t) {
  --lo;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (*(cu + mid) <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// The same for the whole array by one warp, 32 probes at a time: two or three dependent loads instead of ten.
__device__ __forceinline__ int seq_of_row_warp(const int32_t* __restrict__ cu, int n_seqs, int t) {
  const int lane = threadIdx.x & 31;
  int lo = -1, hi = n_seqs;  // the answer is in [lo, hi]
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;
    const int probe = lo + 1 + lane * step;  // ascending; the answer is behind every probe that holds
    const bool holds = probe <= hi && *(cu + probe) <= t;
    const unsigned m = __ballot_sync(0xffffffffu, holds);
    // with cu ascending the lanes that hold are the lowest ones; their number alone bounds the answer in any case
    const int n = __popc(m);
    const int nlo = n ? lo + 1 + (n - 1) * step : lo;
    const int nhi = min(hi, lo + n * step);
    lo = nlo;
    hi = max(nlo, nhi);
  }
  return lo;
}

// First and one-past-last row of the sequence of row t; first > t when the row belongs to no sequence.  Whatever the
// array holds, 0 <= first and last <= rows.
struct RowSpan { int first, last; };
__device__ __forceinline__ RowSpan row_span(const int32_t* __restrict__ cu, int n_seqs, int s, int t, int rows) {
  RowSpan r{t + 1, t + 1};
  if (s >= 0 && s < n_seqs && t < rows) {
    const int end = cu[s + 1];
    if (t < end) {  // (a search among some of the sequences only may stop at one before the row)
      r.first = max(0, min(t, cu[s]));
      r.last = min(rows, end);
    }
  }
  return r;
}

// ---- one row by one warp -------------------------------------------------------------------------------------------
// Masked pairs are skipped, not multiplied by zero: what stands in rows a query may not see (another sequence, a later
// position, rows of no sequence) never reaches it, infinities and NaN included.  The tensor-core kernels, whose products
// run over whole tiles, redo through these functions every row that did not come out finite.

template <typename T, int HS> __device__ __forceinline__ float row_dot(const T* a, const T* b) {
  const int lane = threadIdx.x & 31;
  float d = 0.f;
#pragma unroll
  for (int e = 0; e < HS; e += 32)
    if (HS % 32 == 0 || e + lane < HS) d = fmaf(to_f32(a[e + lane]), to_f32(b[e + lane]), d);
  return warp_sum(d);
}

template <typename T, int HS>
__device__ __noinline__ void packed_fwd_row(const T* q, const T* k, const T* v, T* o, float* lse, int ldk, int ldv,
                                            int first, int t, float scale) {
  constexpr int N = (HS + 31) / 32;
  const int lane = threadIdx.x & 31;
  float acc[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  for (int u = first; u <= t; ++u) {
    const float s = row_dot<T, HS>(q, k + (size_t)u * ldk) * scale;
    const float nm = fmaxf(m, s);
    const float corr = m == nm ? 1.f : exp_by_build(m - nm);
    const float p = nm == -INFINITY && s == s ? 0.f : exp_by_build(s - nm);  // (a score of minus infinity has no weight, a NaN is one)
    l = l * corr + p;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (HS % 32 == 0 || lane + 32 * i < HS) acc[i] = fmaf(p, to_f32(v[(size_t)u * ldv + lane + 32 * i]), acc[i] * corr);
    m = nm;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (HS % 32 == 0 || lane + 32 * i < HS) o[lane + 32 * i] = from_f32<T>(acc[i] / l);
  if (lse && lane == 0) *lse = m + logf(l);
}

// The first row of a sequence sees one key: its softmax is the constant 1 and dS = P (dP - delta) is zero.  The backward
// kernels say so themselves (`alone`), since dP and delta are sums in different orders and differ in their last bits.
__device__ __forceinline__ bool alone(int first, int t) { return first == t; }

template <typename T, int HS>
__device__ __noinline__ void packed_dq_row(const T* q, const T* k, const T* v, const T* d_o, float lse, float delta, T* dq,
                                           int ldk, int ldv, int first, int t, float scale) {
  constexpr int N = (HS + 31) / 32;
  const int lane = threadIdx.x & 31;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  const float out_scale = alone(first, t) ? 0.f : scale;
  for (int u = first; u <= t; ++u) {
    const float p = exp_by_build(row_dot<T, HS>(q, k + (size_t)u * ldk) * scale - lse);
    const float ds = p * (row_dot<T, HS>(d_o, v + (size_t)u * ldv) - delta) * out_scale;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (HS % 32 == 0 || lane + 32 * i < HS) acc[i] = fmaf(ds, to_f32(k[(size_t)u * ldk + lane + 32 * i]), acc[i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (HS % 32 == 0 || lane + 32 * i < HS) dq[lane + 32 * i] = from_f32<T>(acc[i]);
}

// Key row u of one key head: sums over the `group` query heads (head-major statistics with pitch `rows`) and the query
// rows u .. last-1 of its sequence, which begins at row `first`.
template <typename T, int HS>
__device__ __noinline__ void packed_dkv_row(const T* q, const T* k, const T* v, const T* d_o, const float* lse,
                                            const float* delta, T* dk, T* dv, int ldq, int lddo, int rows, int group,
                                            int u, int first, int last, float scale) {
  constexpr int N = (HS + 31) / 32;
  const int lane = threadIdx.x & 31;
  float ak[N], av[N];
#pragma unroll
  for (int i = 0; i < N; ++i) ak[i] = av[i] = 0.f;
  for (int g = 0; g < group; ++g) {
    for (int t = u; t < last; ++t) {
      const T* qr = q + (size_t)t * ldq + g * HS;
      const T* gr = d_o + (size_t)t * lddo + g * HS;
      const size_t st = (size_t)g * rows + t;
      const float p = exp_by_build(row_dot<T, HS>(qr, k) * scale - lse[st]);
      const float ds = p * (row_dot<T, HS>(gr, v) - delta[st]) * (alone(first, t) ? 0.f : scale);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (HS % 32 == 0 || lane + 32 * i < HS) {
          av[i] = fmaf(p, to_f32(gr[lane + 32 * i]), av[i]);
          ak[i] = fmaf(ds, to_f32(qr[lane + 32 * i]), ak[i]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (HS % 32 == 0 || lane + 32 * i < HS) {
      dk[lane + 32 * i] = from_f32<T>(ak[i]);
      dv[lane + 32 * i] = from_f32<T>(av[i]);
    }
  }
}

}  // namespace b200
