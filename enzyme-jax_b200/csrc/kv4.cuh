// A key/value cache in 4 bits.  One layer is
//   codes   uint8 [2, n_pages, n_kv_heads, page_size, hs/2]   element 2i in the low half of byte i; keys, then values
//   params  bf16  [2, n_pages, n_kv_heads, page_size, 2]      (scale, minimum) of the row
// and a row stands for minimum + scale * code.  The scale is one number per cached row of a head: it leaves the dot
// product q.k and enters the weight p of a value row, so neither row is ever expanded in memory.
#pragma once

#include "common.cuh"

namespace b200 {

// What kernels of the cache OR into the device status word when a page table names a page outside the pool.
enum : uint32_t { ST_BAD_PAGE = 1u << 16 };

struct Kv4Pool {
  uint8_t* codes = nullptr;
  uint32_t* params = nullptr;  // low half: scale, high half: minimum
  const int32_t* table = nullptr;  // [batch, max_pages]
  int n_pages = 0, n_kv_heads = 0, page_size = 0, head_size = 0, max_pages = 0;
};

// Row index of (page, head, row) inside the key half; the value half begins kv4_half() rows later.
__host__ __device__ __forceinline__ size_t kv4_half(const Kv4Pool& p) {
  return (size_t)p.n_pages * p.n_kv_heads * p.page_size;
}

struct Kv4DecodeArgs {
  Kv4Pool pool;
  const void* q = nullptr;         // [batch, ldq]
  void* o = nullptr;               // [batch, ldo]
  const int32_t* ctx = nullptr;    // [batch] cached rows of each sequence
  float* partials = nullptr;       // 2 * grid slots of [columns][head_size + 2]
  int32_t* prefix = nullptr;       // [batch + 1]
  uint32_t* status = nullptr;
  int batch = 0, n_heads = 0, ldq = 0, ldo = 0, dtype = B200_BF16;
  bool whole = false;              // one CTA per segment, no partials
  int subs = 1;                    // head subsets per key head: segments of a sequence are (key head, subset)
  int cols = 1;                    // query heads per subset (the last one may hold fewer)
  float scale = 1.f;
};

// ---- sharing the cached rows out ------------------------------------------------------------------------------------
// The work of a step is the units of kUnit cached rows of every (sequence, key head, subset), in that order.  Each CTA
// takes one contiguous range of the whole list, so lengths that differ by any factor balance by themselves.  A segment
// that lies inside one CTA is finished there; the others leave partial (sum, maximum, accumulator) blocks that a second
// kernel joins.  Partials are addressed by CTA: 2 slots each (the range's first segment, its last one).
constexpr int kUnit = 128;
constexpr int kMaxSlice = 4096;  // sequences per launch: their unit prefix is held in shared memory

__device__ __forceinline__ int kv4_len(const Kv4DecodeArgs& a, int b) {
  const long long cap = (long long)a.pool.max_pages * a.pool.page_size;
  const int n = *(a.ctx + b);
  return n <= 0 ? 0 : (n < cap ? n : (int)cap);
}
__device__ __forceinline__ int units_of(int len) { return (int)(((unsigned)len + kUnit - 1) / kUnit); }
__device__ __forceinline__ long long range_start(long long units, int ctas, int c) { return units * c / ctas; }
__device__ __forceinline__ int range_owner(long long units, int ctas, long long u) { return (int)(((u + 1) * ctas - 1) / units); }

// Short tables, few segments: CTA i takes the whole of segment i (`whole`), which needs neither scratch nor a second kernel.
// Up to this many units per segment, as long as every segment has a resident CTA.  The border is where a step of few segments,
// most of whose SMs stay idle, stops gaining; it goes by the table's length alone, so steps of many segments, which gain at
// longer tables too, are split there.  Device time at 32/8 heads of 128, whole against split and joined: 500 rows 6.8 / 7.7 us
// (1 sequence), 8.8 / 13.8 (16); 1000 rows 9.9 / 8.1 (1), 13.1 / 16.0 (16); on the CUDA cores (6 fp32 heads of 48): 250 rows
// 8.3 / 8.4, 500 rows 13.9 / 8.4.  The call on the host takes 12 / 15 us.
constexpr int kWholeUnitsMma = 4, kWholeUnitsSimt = 2;

// Exclusive prefix of the sequences' unit counts into `pre` [batch + 1] and their lengths into `lens` [batch] (shared
// memory), by all threads of the block.
template <int THREADS>
__device__ __forceinline__ void unit_prefix(const Kv4DecodeArgs& a, int32_t* pre, int32_t* lens, int32_t* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    const int len = b < a.batch ? kv4_len(a, b) : 0;
    const int mine = units_of(len);
    if (b < a.batch) lens[b] = len;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    int before = base, total = base;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += warp_sums[w];
      total += warp_sums[w];
    }
    if (b < a.batch) pre[b] = before + inc - mine;
    base = total;
    __syncthreads();
  }
  if (threadIdx.x == 0) pre[a.batch] = base;
  __syncthreads();
}

// The CTA's range of units and the sequence it begins in; `ctas`: CTAs with work.
struct UnitRange { long long first, last; int seq; };
template <int THREADS>
__device__ __forceinline__ UnitRange unit_range(const Kv4DecodeArgs& a, int32_t* pre, int32_t* lens, int32_t* warp_sums) {
  const int nseg = a.pool.n_kv_heads * a.subs;
  if (a.whole) {
    const int b = (int)blockIdx.x / nseg, seg = (int)blockIdx.x % nseg, len = kv4_len(a, b), nb = units_of(len);
    if (threadIdx.x == 0) {
      pre[b] = 0;
      pre[b + 1] = nb;
      lens[b] = len;
    }
    __syncthreads();
    return {(long long)seg * nb, (long long)(seg + 1) * nb, b};
  }
  unit_prefix<THREADS>(a, pre, lens, warp_sums);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= a.batch; i += blockDim.x) a.prefix[i] = pre[i];
  const long long units = (long long)pre[a.batch] * nseg;
  const int ctas = (int)(units < (long long)gridDim.x ? units : (long long)gridDim.x);
  if ((int)blockIdx.x >= ctas) return {0, 0, 0};
  return {range_start(units, ctas, blockIdx.x), range_start(units, ctas, blockIdx.x + 1), 0};
}

// `whole` and a sequence without rows: zeros.
template <typename T> __device__ __forceinline__ void zero_segment(const Kv4DecodeArgs& a) {
  const int nseg = a.pool.n_kv_heads * a.subs, hs = a.pool.head_size;
  const int b = (int)blockIdx.x / nseg, seg = (int)blockIdx.x % nseg;
  const int group = a.n_heads / a.pool.n_kv_heads, first = (seg % a.subs) * a.cols;
  const int n = min(a.cols, group - first) * hs;
  T* o = (T*)a.o + (size_t)b * a.ldo + (size_t)((seg / a.subs) * group + first) * hs;
  for (int e = threadIdx.x; e < n; e += blockDim.x) o[e] = from_f32<T>(0.f);
}

bool kv4_decode_mma_supports(const Kv4DecodeArgs& a);
int kv4_decode_mma_grid(int head_size, int cols);  // resident CTAs
int32_t launch_kv4_decode_mma(const Kv4DecodeArgs& a, int grid, cudaStream_t stream);

}  // namespace b200
