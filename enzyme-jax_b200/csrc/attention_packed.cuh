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

// The first row of a sequence sees one key: its softmax is the constant 1 and dS = P (dP - delta) is zero.  The backward
// kernels say so themselves (`alone`), since dP and delta are sums in different orders and differ in their last bits.
__device__ __forceinline__ bool alone(int first, int t) { return first == t; }

// ---- rows that are not finite --------------------------------------------------------------------------------------
// What stands in rows a query may not see (another sequence, a later position, rows of no sequence) never reaches it,
// infinities and NaN included.  The tensor-core kernels multiply whole tiles, and zero weight times an infinity or NaN is
// not zero.  They therefore redo every row that did not come out finite while a row it may not see, among those its tile
// was multiplied with, is not finite either (spoiled_rows): one warp, pair by pair, masked pairs skipped.  A row whose own
// pairs made it infinite or NaN stands as it is -- one bad number in a key would otherwise send every later row of its
// sequence down this path (4096 tokens of 8/2 heads of 128 with one NaN among the keys, forward and backward: 64 and 318 ms
// when every such row was redone one pair at a time, 0.33 and 0.27 ms now; 0.10 and 0.23 ms without the NaN).  Eight pairs are
// in flight, and a row that is NaN throughout is left at once.  What is left slow is a masked place and a visible one that are
// both infinite in the same column, row after row (all of d_o infinite, the same tokens: 50 ms; 315 before).  These functions
// are out of line, so that the kernels' loops keep their registers; the forward's takes one row at a time and its operands one
// by one, which costs the ragged prompts 1 % (286 -> 289 us) where other forms of the call cost 2 to 4.

// HS bf16 numbers of a row over the lanes of a warp, as they stand in memory (16-byte aligned rows)
template <int HS> struct RowBits {
  static constexpr int N = HS / 32;  // elements per lane
  uint32_t w[HS / 64];
  __device__ __forceinline__ void load(const bf16* row) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(row) + (threadIdx.x & 31) * (HS / 64);
    if constexpr (HS == 128) {
      const uint2 x = *reinterpret_cast<const uint2*>(p);
      w[0] = x.x;
      w[1] = x.y;
    } else {
      w[0] = *p;
    }
  }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
  __device__ __forceinline__ bool finite() const {
    bool f = true;
#pragma unroll
    for (int i = 0; i < HS / 64; ++i) f = f && (w[i] & 0x7f80u) != 0x7f80u && (w[i] & 0x7f800000u) != 0x7f800000u;
    return f;
  }
  __device__ __forceinline__ float dot(const RowBits& o) const {
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) d = fmaf(at(i), o.at(i), d);
    return warp_sum(d);
  }
  __device__ __forceinline__ void add_to(float (&acc)[N], float f) const {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = fmaf(f, at(i), acc[i]);
  }
  static __device__ __forceinline__ void store(bf16* row, const float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) row[(threadIdx.x & 31) * N + i] = from_f32<bf16>(x[i]);
  }
};
constexpr int kRowPairs = 8;  // pairs, or rows looked at, in flight

// Of the rows the warp's lanes stand for (those that are `mine`; the lane's row sees rows lo .. hi-1 of x), the ones for
// which x holds an infinity or NaN in a row of from .. to-1 that they do not see: a mask of lanes, the same in every lane.
// Rows that all of them see are not looked at.
template <int HS>
__device__ __forceinline__ unsigned spoiled_rows(const bf16* x, int ld, int from, int to, int lo, int hi, bool mine) {
  const int all_lo = __reduce_max_sync(0xffffffffu, mine ? lo : 0), all_hi = __reduce_min_sync(0xffffffffu, mine ? hi : 0x7fffffff);
  bool spoiled = false;
  for (int u0 = from; u0 < to;) {
    if (u0 >= all_lo && u0 < all_hi) {
      u0 = all_hi;
      continue;
    }
    const int end = min(u0 < all_lo && all_lo < all_hi ? all_lo : to, min(u0 + kRowPairs, to));
    RowBits<HS> row[kRowPairs];
#pragma unroll
    for (int j = 0; j < kRowPairs; ++j) row[j].load(x + (size_t)min(u0 + j, end - 1) * ld);
#pragma unroll
    for (int j = 0; j < kRowPairs; ++j)
      if (__any_sync(0xffffffffu, !row[j].finite()) && u0 + j < end) spoiled = spoiled || u0 + j < lo || u0 + j >= hi;
    u0 = end;
  }
  return __ballot_sync(0xffffffffu, mine && spoiled);
}

// Row t of a query head that did not come out finite; its tile was multiplied with value rows from .. to-1.  By a whole warp.
template <int HS>
__device__ __noinline__ void redo_fwd(const bf16* qp, const bf16* k, const bf16* v, bf16* o, float* lse, int ldk, int ldv, int first, int t,
                                      float scale, int from, int to) {
  using Row = RowBits<HS>;
  if (!spoiled_rows<HS>(v, ldv, from, to, first, t + 1, true)) return;
  Row q;
  q.load(qp);
  float acc[Row::N] = {}, m = -INFINITY, l = 0.f;
  for (int u0 = first; u0 <= t && l == l; u0 += kRowPairs) {  // (a sum that is NaN stays so, and the whole row with it)
    Row kr[kRowPairs], vr[kRowPairs];
    float s[kRowPairs], nm = m;
#pragma unroll
    for (int j = 0; j < kRowPairs; ++j) {  // (behind the end the last pair again, which then has no weight)
      kr[j].load(k + (size_t)min(u0 + j, t) * ldk);
      vr[j].load(v + (size_t)min(u0 + j, t) * ldv);
    }
#pragma unroll
    for (int j = 0; j < kRowPairs; ++j) {
      s[j] = q.dot(kr[j]) * scale;
      nm = fmaxf(nm, s[j]);
    }
    const float corr = m == nm ? 1.f : exp_by_build(m - nm);
    const float ref = nm == -INFINITY ? 0.f : nm;  // a score of minus infinity has no weight, a NaN is one
    l *= corr;
#pragma unroll
    for (int i = 0; i < Row::N; ++i) acc[i] *= corr;
#pragma unroll
    for (int j = 0; j < kRowPairs; ++j) {
      if (u0 + j <= t) {
        const float p = exp_by_build(s[j] - ref);
        l += p;
        vr[j].add_to(acc, p);
      }
    }
    m = nm;
  }
#pragma unroll
  for (int i = 0; i < Row::N; ++i) acc[i] /= l;
  Row::store(o, acc);
  if (lse && (threadIdx.x & 31) == 0) *lse = m + logf(l);
}

// The same for rows of dQ, whose tile was multiplied with key rows from .. to-1; delta is the corrected one.
template <int HS>
__device__ __noinline__ void redo_dq(const PackedBwdArgs& a, unsigned rows, int r0, int head, int from, int to, float scale) {
  using Row = RowBits<HS>;
  const PackedArgs& f = a.f;
  const int t = r0 + (threadIdx.x & 31), first = row_span(f.cu, f.n_seqs, seq_of_row(f.cu, 0, f.n_seqs, t), t, f.rows).first;
  const int hk = head / (f.n_heads / f.n_kv_heads);
  const bf16* k = (const bf16*)f.k + hk * HS;
  const bf16* v = (const bf16*)f.v + hk * HS;
  unsigned redo = spoiled_rows<HS>(k, f.ldk, from, to, first, t + 1, (rows >> (threadIdx.x & 31)) & 1u);
  for (; redo; redo &= redo - 1) {
    const int b = __ffs(redo) - 1;
    const int r = __shfl_sync(0xffffffffu, t, b), begin = __shfl_sync(0xffffffffu, first, b);
    const float dl = a.delta[(size_t)head * f.rows + r], lse = f.lse[(size_t)head * f.rows + r];
    const float out_scale = alone(begin, r) ? 0.f : scale;
    Row q, g;
    q.load((const bf16*)f.q + (size_t)r * f.ldq + head * HS);
    g.load((const bf16*)a.d_o + (size_t)r * a.lddo + head * HS);
    float acc[Row::N] = {};
    bool lost = false;  // a NaN score gradient makes the whole row NaN
    for (int u0 = begin; u0 <= r && !lost; u0 += kRowPairs) {
      Row kr[kRowPairs], vr[kRowPairs];
#pragma unroll
      for (int j = 0; j < kRowPairs; ++j) {
        kr[j].load(k + (size_t)min(u0 + j, r) * f.ldk);
        vr[j].load(v + (size_t)min(u0 + j, r) * f.ldv);
      }
      float ds[kRowPairs];
#pragma unroll
      for (int j = 0; j < kRowPairs; ++j)
        ds[j] = exp_by_build(q.dot(kr[j]) * scale - lse) * (g.dot(vr[j]) - dl) * out_scale;
#pragma unroll
      for (int j = 0; j < kRowPairs; ++j) {
        if (u0 + j <= r) {
          lost = lost || ds[j] != ds[j];
          kr[j].add_to(acc, ds[j]);
        }
      }
    }
    Row::store((bf16*)a.dq + (size_t)r * a.lddq + head * HS, acc);
  }
}

// The same for rows of dK or dV of a key head, whose tile was multiplied with rows from .. to-1 of Q or dO of every query
// head of the group.
template <int HS, bool DK>
__device__ __noinline__ void redo_dkv(const PackedBwdArgs& a, unsigned rows, int r0, int hk, int from, int to, float scale) {
  using Row = RowBits<HS>;
  const PackedArgs& f = a.f;
  const int u = r0 + (threadIdx.x & 31);
  const RowSpan span = row_span(f.cu, f.n_seqs, seq_of_row(f.cu, 0, f.n_seqs, u), u, f.rows);
  const int group = f.n_heads / f.n_kv_heads;
  unsigned redo = 0u;
  for (int h = hk * group; h < (hk + 1) * group; ++h)
    redo |= spoiled_rows<HS>((DK ? (const bf16*)f.q : (const bf16*)a.d_o) + h * HS, DK ? f.ldq : a.lddo, from, to, u, span.last,
                             (rows >> (threadIdx.x & 31)) & 1u);
  for (; redo; redo &= redo - 1) {
    const int b = __ffs(redo) - 1;
    const int r = __shfl_sync(0xffffffffu, u, b), begin = __shfl_sync(0xffffffffu, span.first, b), end = __shfl_sync(0xffffffffu, span.last, b);
    Row k, v;
    k.load((const bf16*)f.k + (size_t)r * f.ldk + hk * HS);
    if (DK) v.load((const bf16*)f.v + (size_t)r * f.ldv + hk * HS);
    float acc[Row::N] = {};
    bool lost = false;  // the row is NaN throughout
    for (int h = hk * group; h < (hk + 1) * group; ++h) {
      for (int t0 = r; t0 < end && !lost; t0 += kRowPairs) {
        Row qr[kRowPairs], gr[kRowPairs];
        float w[kRowPairs], dl[kRowPairs];
#pragma unroll
        for (int j = 0; j < kRowPairs; ++j) {
          const int t = min(t0 + j, end - 1);
          qr[j].load((const bf16*)f.q + (size_t)t * f.ldq + h * HS);
          gr[j].load((const bf16*)a.d_o + (size_t)t * a.lddo + h * HS);
          w[j] = f.lse[(size_t)h * f.rows + t];
          if (DK) dl[j] = a.delta[(size_t)h * f.rows + t];
        }
#pragma unroll
        for (int j = 0; j < kRowPairs; ++j) {
          w[j] = exp_by_build(qr[j].dot(k) * scale - w[j]);
          if (DK) w[j] *= (gr[j].dot(v) - dl[j]) * (alone(begin, t0 + j) ? 0.f : scale);
        }
#pragma unroll
        for (int j = 0; j < kRowPairs; ++j) {
          if (t0 + j < end) {
            (DK ? qr[j] : gr[j]).add_to(acc, w[j]);
          }
        }
        bool nan = true;
#pragma unroll
        for (int i = 0; i < Row::N; ++i) nan = nan && acc[i] != acc[i];
        lost = __all_sync(0xffffffffu, nan);
      }
    }
    if (DK) Row::store((bf16*)a.dk + (size_t)r * a.lddk + hk * HS, acc);
    else Row::store((bf16*)a.dv + (size_t)r * a.lddv + hk * HS, acc);
  }
}

}  // namespace b200
