// Packed causal attention with grouped heads on the CUDA cores: fp32 or bf16 storage, fp32 arithmetic, head sizes 16 to
// 128, any alignment.  This is the exact-fp32 path and serves the head sizes and layouts the tensor-core kernels refuse.
//
// A CTA of 128 threads owns 32 consecutive rows of the packed axis (they may belong to several sequences); four threads
// share a row and own a quarter of the head dimension each.  Rows of the other operand stream through shared memory 32
// at a time, as fp32, the quarters of a row 16 bytes apart in the banks (DPT + 4 words) so that the four threads of a
// row read without conflicts.  Bound by the FFMA pipe and the shared-memory reads that feed it: every value read (16
// bytes per 4 FFMA) serves one row per thread.  8 x 1024 tokens of 12 fp32 heads of 64: forward 1041 us, backward 2701 us (12
// TFLOP/s of 64 in FFMA).  Built without fast math.
#include <type_traits>

#include "attention_packed.cuh"

namespace b200 {

namespace {

constexpr int RB = 32;  // rows per CTA and per streamed block

template <int HS> struct Quarter {
  static constexpr int kDims = HS / 4;       // dims per thread
  static constexpr int kPitch = kDims + 4;   // words between quarters in shared memory
  static constexpr int kRow = 4 * kPitch;
  static_assert(kDims % 4 == 0, "head size must be a multiple of 16");
};

// Rows r0 .. r0+31 (those below `end`; zeros elsewhere) of one head into shared memory as fp32.
template <typename T, int HS>
__device__ __forceinline__ void stage_rows(float* __restrict__ dst, const T* __restrict__ src, int ld, int r0, int end,
                                           bool vec) {
  using Q = Quarter<HS>;
  constexpr int PIECES = RB * HS / 4;  // 4 dims each: a piece never crosses a quarter
  for (int idx = threadIdx.x; idx < PIECES; idx += 128) {
    const int r = idx / (HS / 4), d = (idx % (HS / 4)) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r0 + r < end) {
      const T* p = src + (size_t)(r0 + r) * ld + d;
      if (vec) {
        if constexpr (sizeof(T) == 4) {
          x = *reinterpret_cast<const float4*>(p);
        } else {
          const uint2 raw = *reinterpret_cast<const uint2*>(p);
          const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
          const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
          x = make_float4(a.x, a.y, b.x, b.y);
        }
      } else {
        x = make_float4(to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3]));
      }
    }
    *reinterpret_cast<float4*>(dst + r * Q::kRow + (d / Q::kDims) * Q::kPitch + d % Q::kDims) = x;
  }
}

template <int N> __device__ __forceinline__ float dot_quarter(const float (&a)[N], const float* b) {
  float d = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 x = *reinterpret_cast<const float4*>(b + i);
    d = fmaf(a[i], x.x, fmaf(a[i + 1], x.y, fmaf(a[i + 2], x.z, fmaf(a[i + 3], x.w, d))));
  }
  d += __shfl_xor_sync(0xffffffffu, d, 1);
  return d + __shfl_xor_sync(0xffffffffu, d, 2);
}
template <int N> __device__ __forceinline__ void axpy_quarter(float (&acc)[N], float p, const float* b) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 x = *reinterpret_cast<const float4*>(b + i);
    acc[i] = fmaf(p, x.x, acc[i]); acc[i + 1] = fmaf(p, x.y, acc[i + 1]);
    acc[i + 2] = fmaf(p, x.z, acc[i + 2]); acc[i + 3] = fmaf(p, x.w, acc[i + 3]);
  }
}

// Row `row0 + tid/4` of the CTA with its sequence; lo / hi (shared) become the first and one-past-last row any of the
// CTA's live rows may see.
struct CtaRows { RowSpan span; bool live; };
__device__ __forceinline__ CtaRows cta_rows(const int32_t* cu, int n_seqs, int row0, int rows, int* lo, int* hi) {
  const int t = row0 + (threadIdx.x >> 2);
  if (threadIdx.x == 0) { *lo = rows; *hi = 0; }
  __syncthreads();
  const int s = t < rows ? seq_of_row(cu, 0, n_seqs, t) : -1;
  CtaRows r;
  r.span = row_span(cu, n_seqs, s, t, rows);
  r.live = r.span.first <= t;
  if (r.live && (threadIdx.x & 3) == 0) {
    atomicMin(lo, r.span.first);
    atomicMax(hi, r.span.last);
  }
  __syncthreads();
  return r;
}

template <typename T, int HS>
__global__ void __launch_bounds__(128) packed_fwd_simt_kernel(PackedArgs a, float scale, bool vec) {
  using Q = Quarter<HS>;
  constexpr int DPT = Q::kDims;
  __shared__ __align__(16) float Ks[RB * Q::kRow];
  __shared__ __align__(16) float Vs[RB * Q::kRow];
  __shared__ int lo, hi;
  const int part = threadIdx.x & 3;
  const int row0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * RB, t = row0 + (threadIdx.x >> 2);
  const int h = blockIdx.y, hk = h / (a.n_heads / a.n_kv_heads);
  const T* k = (const T*)a.k + hk * HS;
  const T* v = (const T*)a.v + hk * HS;
  const CtaRows me = cta_rows(a.cu, a.n_seqs, row0, a.rows, &lo, &hi);

  float qr[DPT], acc[DPT];
#pragma unroll
  for (int i = 0; i < DPT; ++i) {
    qr[i] = me.live ? to_f32(((const T*)a.q)[(size_t)t * a.ldq + h * HS + part * DPT + i]) * scale : 0.f;
    acc[i] = 0.f;
  }
  float mx = -INFINITY, l = 0.f;
  const int last = min(row0 + RB, hi);
  for (int u0 = lo; u0 < last; u0 += RB) {
    __syncthreads();
    stage_rows<T, HS>(Ks, k, a.ldk, u0, last, vec);
    stage_rows<T, HS>(Vs, v, a.ldv, u0, last, vec);
    __syncthreads();
    const float* kq = Ks + part * Q::kPitch;
    const float* vq = Vs + part * Q::kPitch;
    float s[RB], bm = -INFINITY;
    const int from = me.live ? me.span.first - u0 : RB, to = me.live ? t - u0 : -1;  // keys from..to of the block are seen
#pragma unroll
    for (int uu = 0; uu < RB; ++uu) {
      const float d = dot_quarter(qr, kq + uu * Q::kRow);
      s[uu] = (uu >= from && uu <= to) ? d : -INFINITY;
      bm = fmaxf(bm, s[uu]);
    }
    if (from <= to && from < RB && to >= 0) {
      const float nm = fmaxf(mx, bm);
      const float corr = mx == nm ? 1.f : exp_by_build(mx - nm);
      const float ref = nm == -INFINITY ? 0.f : nm;  // scores of minus infinity alone: no weight yet
      l *= corr;
#pragma unroll
      for (int i = 0; i < DPT; ++i) acc[i] *= corr;
      if (from <= 0 && to >= RB - 1) {
#pragma unroll
        for (int uu = 0; uu < RB; ++uu) {
          const float p = exp_by_build(s[uu] - ref);
          l += p;
          axpy_quarter(acc, p, vq + uu * Q::kRow);
        }
      } else {  // keys outside are skipped: zero times what stands there need not be zero
#pragma unroll
        for (int uu = 0; uu < RB; ++uu) {
          if (uu >= from && uu <= to) {
            const float p = exp_by_build(s[uu] - ref);
            l += p;
            axpy_quarter(acc, p, vq + uu * Q::kRow);
          }
        }
      }
      mx = nm;
    }
  }
  if (me.live) {
    const float inv = 1.f / l;
    T* o = (T*)a.o + (size_t)t * a.ldo + h * HS + part * DPT;
#pragma unroll
    for (int i = 0; i < DPT; ++i) o[i] = from_f32<T>(acc[i] * inv);
    if (a.lse && part == 0) a.lse[(size_t)h * a.rows + t] = mx + logf(l);
  }
}

// delta[h, t] = sum_e dO[t, e] * O[t, e]: 32 rows per CTA, four threads to a row.
template <typename T, int HS>
__global__ void __launch_bounds__(128) packed_delta_kernel(PackedBwdArgs a) {
  constexpr int DPT = HS / 4;
  const int part = threadIdx.x & 3, t = blockIdx.x * RB + (threadIdx.x >> 2), h = blockIdx.y;
  const int tr = t < a.f.rows ? t : 0;
  const T* o = (const T*)a.f.o + (size_t)tr * a.f.ldo + h * HS;
  const T* g = (const T*)a.d_o + (size_t)tr * a.lddo + h * HS;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < DPT; ++i) s = fmaf(to_f32(o[part + 4 * i]), to_f32(g[part + 4 * i]), s);
  s += __shfl_xor_sync(0xffffffffu, s, 1);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  if (t < a.f.rows && part == 0) a.delta[(size_t)h * a.f.rows + t] = s;
}

// dQ: a CTA owns 32 query rows and streams the keys and values they see.  With bf16 outputs rowsum(dO * o) carries the
// rounding of o, which is not small beside dP - delta where a row sees few keys: the pass then also sums
// eps = rowsum(P * (dP - delta0)) and P K, subtracts eps P K / sqrt(hs) and leaves delta0 + eps for the key pass.
template <typename T, int HS>
__global__ void __launch_bounds__(128) packed_dq_simt_kernel(PackedBwdArgs a, float scale, bool vec) {
  using Q = Quarter<HS>;
  constexpr int DPT = Q::kDims;
  __shared__ __align__(16) float Ks[RB * Q::kRow];
  __shared__ __align__(16) float Vs[RB * Q::kRow];
  __shared__ int lo, hi;
  const PackedArgs& f = a.f;
  const int part = threadIdx.x & 3;
  const int row0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * RB, t = row0 + (threadIdx.x >> 2);
  const int h = blockIdx.y, hk = h / (f.n_heads / f.n_kv_heads);
  const CtaRows me = cta_rows(f.cu, f.n_seqs, row0, f.rows, &lo, &hi);
  constexpr bool kExact = sizeof(T) == 2;
  float qr[DPT], gr[DPT], acc[DPT], pk[kExact ? DPT : 4], eps = 0.f;
#pragma unroll
  for (int i = 0; i < DPT; ++i) {
    qr[i] = me.live ? to_f32(((const T*)f.q)[(size_t)t * f.ldq + h * HS + part * DPT + i]) : 0.f;
    gr[i] = me.live ? to_f32(((const T*)a.d_o)[(size_t)t * a.lddo + h * HS + part * DPT + i]) : 0.f;
    acc[i] = 0.f;
    if (kExact) pk[i] = 0.f;
  }
  const float lse = me.live ? f.lse[(size_t)h * f.rows + t] : 0.f;
  const float delta = me.live ? a.delta[(size_t)h * f.rows + t] : 0.f;
  const float out_scale = alone(me.span.first, t) ? 0.f : scale;
  const int last = min(row0 + RB, hi);
  for (int u0 = lo; u0 < last; u0 += RB) {
    __syncthreads();
    stage_rows<T, HS>(Ks, (const T*)f.k + hk * HS, f.ldk, u0, last, vec);
    stage_rows<T, HS>(Vs, (const T*)f.v + hk * HS, f.ldv, u0, last, vec);
    __syncthreads();
    const float* kq = Ks + part * Q::kPitch;
    const float* vq = Vs + part * Q::kPitch;
    const int from = me.live ? me.span.first - u0 : RB, to = me.live ? t - u0 : -1;
#pragma unroll 4
    for (int uu = 0; uu < RB; ++uu) {
      const float s = dot_quarter(qr, kq + uu * Q::kRow);
      const float dp = dot_quarter(gr, vq + uu * Q::kRow);
      if (uu >= from && uu <= to) {
        const float p = exp_by_build(s * scale - lse);
        const float w = p * (dp - delta);
        axpy_quarter(acc, w * out_scale, kq + uu * Q::kRow);
        if constexpr (kExact) {
          eps += w;
          axpy_quarter(pk, p, kq + uu * Q::kRow);
        }
      }
    }
  }
  if (me.live) {
    T* dq = (T*)a.dq + (size_t)t * a.lddq + h * HS + part * DPT;
#pragma unroll
    for (int i = 0; i < DPT; ++i) dq[i] = from_f32<T>(kExact ? fmaf(-eps * out_scale, pk[i], acc[i]) : acc[i]);
    if (kExact && part == 0) a.delta[(size_t)h * f.rows + t] = delta + eps;
  }
}

// dK, dV: a CTA owns 32 key rows of one key head and streams, for every query head of the group, the queries that see
// them.  One CTA adds up the whole group, so the shared heads need no atomics and the order of the sums is fixed.
template <typename T, int HS>
__global__ void __launch_bounds__(128) packed_dkv_simt_kernel(PackedBwdArgs a, float scale, bool vec) {
  using Q = Quarter<HS>;
  constexpr int DPT = Q::kDims;
  __shared__ __align__(16) float Qs[RB * Q::kRow];
  __shared__ __align__(16) float Gs[RB * Q::kRow];
  __shared__ float Ls[RB], Ds[RB];
  __shared__ int lo, hi;
  const PackedArgs& f = a.f;
  const int part = threadIdx.x & 3;
  const int row0 = blockIdx.x * RB, u = row0 + (threadIdx.x >> 2);
  const int hk = blockIdx.y, group = f.n_heads / f.n_kv_heads;
  const CtaRows me = cta_rows(f.cu, f.n_seqs, row0, f.rows, &lo, &hi);
  float kr[DPT], vr[DPT], ak[DPT], av[DPT];
#pragma unroll
  for (int i = 0; i < DPT; ++i) {
    kr[i] = me.live ? to_f32(((const T*)f.k)[(size_t)u * f.ldk + hk * HS + part * DPT + i]) : 0.f;
    vr[i] = me.live ? to_f32(((const T*)f.v)[(size_t)u * f.ldv + hk * HS + part * DPT + i]) : 0.f;
    ak[i] = av[i] = 0.f;
  }
  for (int g = 0; g < group; ++g) {
    const int h = hk * group + g;
    for (int t0 = row0; t0 < hi; t0 += RB) {
      __syncthreads();
      stage_rows<T, HS>(Qs, (const T*)f.q + h * HS, f.ldq, t0, hi, vec);
      stage_rows<T, HS>(Gs, (const T*)a.d_o + h * HS, a.lddo, t0, hi, vec);
      if (threadIdx.x < RB) {
        const int t = t0 + threadIdx.x;
        Ls[threadIdx.x] = t < hi ? f.lse[(size_t)h * f.rows + t] : 0.f;
        Ds[threadIdx.x] = t < hi ? a.delta[(size_t)h * f.rows + t] : 0.f;
      }
      __syncthreads();
      const float* qq = Qs + part * Q::kPitch;
      const float* gq = Gs + part * Q::kPitch;
      const int from = me.live ? u - t0 : RB, to = me.live ? me.span.last - t0 : 0;  // queries from..to-1 see this key
      const int zero = alone(me.span.first, u) ? from : -1;
#pragma unroll 4
      for (int tt = 0; tt < RB; ++tt) {
        const float s = dot_quarter(kr, qq + tt * Q::kRow);
        const float dp = dot_quarter(vr, gq + tt * Q::kRow);
        if (tt >= from && tt < to) {
          const float p = exp_by_build(s * scale - Ls[tt]);
          axpy_quarter(av, p, gq + tt * Q::kRow);
          axpy_quarter(ak, p * (dp - Ds[tt]) * (tt == zero ? 0.f : scale), qq + tt * Q::kRow);
        }
      }
    }
  }
  if (me.live) {
    T* dk = (T*)a.dk + (size_t)u * a.lddk + hk * HS + part * DPT;
    T* dv = (T*)a.dv + (size_t)u * a.lddv + hk * HS + part * DPT;
#pragma unroll
    for (int i = 0; i < DPT; ++i) {
      dk[i] = from_f32<T>(ak[i]);
      dv[i] = from_f32<T>(av[i]);
    }
  }
}

inline bool rows_vec(const void* p, int ld) { return aligned16(p) && ld % 8 == 0; }

template <typename T, int HS> int32_t fwd_hs(const PackedArgs& a, cudaStream_t stream) {
  const dim3 grid(cdiv(a.rows, RB), a.n_heads);
  packed_fwd_simt_kernel<T, HS><<<grid, 128, 0, stream>>>(a, 1.f / sqrtf((float)HS), rows_vec(a.k, a.ldk) && rows_vec(a.v, a.ldv));
  B200_LAUNCH_OK("packed_fwd_simt_kernel");
  return B200_OK;
}

template <typename T, int HS> int32_t bwd_hs(const PackedBwdArgs& a, cudaStream_t stream) {
  const PackedArgs& f = a.f;
  const float scale = 1.f / sqrtf((float)HS);
  const int blocks = cdiv(f.rows, RB);
  packed_delta_kernel<T, HS><<<dim3(blocks, f.n_heads), 128, 0, stream>>>(a);
  B200_LAUNCH_OK("packed_delta_kernel");
  packed_dq_simt_kernel<T, HS><<<dim3(blocks, f.n_heads), 128, 0, stream>>>(a, scale, rows_vec(f.k, f.ldk) && rows_vec(f.v, f.ldv));
  B200_LAUNCH_OK("packed_dq_simt_kernel");
  packed_dkv_simt_kernel<T, HS><<<dim3(blocks, f.n_kv_heads), 128, 0, stream>>>(a, scale, rows_vec(f.q, f.ldq) && rows_vec(a.d_o, a.lddo));
  B200_LAUNCH_OK("packed_dkv_simt_kernel");
  return B200_OK;
}

template <typename F> int32_t by_type(int dtype, int hs, F&& f) {
  auto go = [&](auto t) -> int32_t {
    using T = decltype(t);
    switch (hs) {
      case 16: return f(t, std::integral_constant<int, 16>());
      case 32: return f(t, std::integral_constant<int, 32>());
      case 48: return f(t, std::integral_constant<int, 48>());
      case 64: return f(t, std::integral_constant<int, 64>());
      case 128: return f(t, std::integral_constant<int, 128>());
    }
    return fail(B200_ERR_BAD_SHAPE, "packed attention: head size %d is not one of 16/32/48/64/128", hs);
  };
  if (dtype == B200_F32) return go(float());
  if (dtype == B200_BF16) return go(bf16());
  return fail(B200_ERR_BAD_DTYPE, "packed attention: unsupported dtype %d", dtype);
}

}  // namespace

int32_t launch_packed_fwd_simt(const PackedArgs& a, cudaStream_t stream) {
  return by_type(a.dtype, a.head_size, [&](auto t, auto hs) { return fwd_hs<decltype(t), decltype(hs)::value>(a, stream); });
}
int32_t launch_packed_bwd_simt(const PackedBwdArgs& a, cudaStream_t stream) {
  return by_type(a.f.dtype, a.f.head_size, [&](auto t, auto hs) { return bwd_hs<decltype(t), decltype(hs)::value>(a, stream); });
}

}  // namespace b200

using namespace b200;

namespace {

int32_t check_packed(const PackedArgs& a) {
  if (a.n_seqs < 0 || a.rows < 0) return fail(B200_ERR_BAD_SHAPE, "packed attention: n_seqs=%d rows=%d", a.n_seqs, a.rows);
  if (a.n_heads <= 0 || a.n_kv_heads <= 0 || a.head_size <= 0) return fail(B200_ERR_BAD_SHAPE, "packed attention: head counts and head size must be positive");
  if (a.n_heads % a.n_kv_heads)
    return fail(B200_ERR_BAD_SHAPE, "packed attention: %d query heads are not a multiple of %d key heads", a.n_heads, a.n_kv_heads);
  if (a.n_heads > 65535) return fail(B200_ERR_BAD_SHAPE, "packed attention: more than 65535 heads");
  const long long wq = (long long)a.n_heads * a.head_size, wk = (long long)a.n_kv_heads * a.head_size;
  if (a.ldq < wq || a.ldo < wq || a.ldk < wk || a.ldv < wk)
    return fail(B200_ERR_BAD_SHAPE, "packed attention: a row pitch is smaller than the row");
  if (a.dtype != B200_F32 && a.dtype != B200_BF16) return fail(B200_ERR_BAD_DTYPE, "packed attention: unsupported dtype %d", a.dtype);
  switch (a.head_size) {
    case 16: case 32: case 48: case 64: case 128: return B200_OK;
  }
  return fail(B200_ERR_BAD_SHAPE, "packed attention: head size %d is not one of 16/32/48/64/128", a.head_size);
}

}  // namespace

extern "C" {

int32_t b200_attention_packed(const void* q, const void* k, const void* v, void* o, float* lse, const int32_t* cu_seqlens,
                              int32_t n_seqs, int32_t rows, int32_t n_heads, int32_t n_kv_heads, int32_t head_size,
                              int32_t ldq, int32_t ldk, int32_t ldv, int32_t ldo, int32_t dtype, int32_t impl,
                              b200_stream_t stream) {
  PackedArgs a;
  a.q = q; a.k = k; a.v = v; a.o = o; a.lse = lse; a.cu = cu_seqlens;
  a.n_seqs = n_seqs; a.rows = rows; a.n_heads = n_heads; a.n_kv_heads = n_kv_heads; a.head_size = head_size;
  a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo; a.dtype = dtype;
  B200_TRY(check_packed(a));
  if (impl < 0 || impl > 2) return fail(B200_ERR_INVALID_ARG, "impl %d is not 0, 1 or 2", impl);
  if (rows == 0 || n_seqs == 0) return B200_OK;
  if (!q || !k || !v || !o || !cu_seqlens) return fail(B200_ERR_INVALID_ARG, "null operand");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (impl == 1 || (impl == 0 && packed_fwd_tc_supports(a))) return launch_packed_fwd_tc(a, s);
  return launch_packed_fwd_simt(a, s);
}

int32_t b200_attention_packed_backward(const void* q, const void* k, const void* v, const void* o, const float* lse,
                                       const void* d_o, void* dq, void* dk, void* dv, float* delta_scratch,
                                       const int32_t* cu_seqlens, int32_t n_seqs, int32_t rows, int32_t n_heads,
                                       int32_t n_kv_heads, int32_t head_size, int32_t ldq, int32_t ldk, int32_t ldv,
                                       int32_t ldo, int32_t lddo, int32_t lddq, int32_t lddk, int32_t lddv, int32_t dtype,
                                       int32_t impl, b200_stream_t stream) {
  PackedBwdArgs a;
  a.f.q = q; a.f.k = k; a.f.v = v; a.f.o = const_cast<void*>(o); a.f.lse = const_cast<float*>(lse); a.f.cu = cu_seqlens;
  a.f.n_seqs = n_seqs; a.f.rows = rows; a.f.n_heads = n_heads; a.f.n_kv_heads = n_kv_heads; a.f.head_size = head_size;
  a.f.ldq = ldq; a.f.ldk = ldk; a.f.ldv = ldv; a.f.ldo = ldo; a.f.dtype = dtype;
  a.d_o = d_o; a.dq = dq; a.dk = dk; a.dv = dv;
  a.lddo = lddo; a.lddq = lddq; a.lddk = lddk; a.lddv = lddv; a.delta = delta_scratch;
  B200_TRY(check_packed(a.f));
  const long long wq = (long long)n_heads * head_size, wk = (long long)n_kv_heads * head_size;
  if (lddo < wq || lddq < wq || lddk < wk || lddv < wk)
    return fail(B200_ERR_BAD_SHAPE, "packed attention: a row pitch is smaller than the row");
  if (impl < 0 || impl > 2) return fail(B200_ERR_INVALID_ARG, "impl %d is not 0, 1 or 2", impl);
  if (rows == 0 || n_seqs == 0) return B200_OK;
  if (!q || !k || !v || !o || !lse || !d_o || !dq || !dk || !dv || !delta_scratch || !cu_seqlens)
    return fail(B200_ERR_INVALID_ARG, "null operand");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (impl == 1 || (impl == 0 && packed_bwd_tc_supports(a))) return launch_packed_bwd_tc(a, s);
  return launch_packed_bwd_simt(a, s);
}

}  // extern "C"
