// Copies of whole or partly filled pages inside one pool of a paged cache, over all layers and both halves at once, with
// the rewrite of the page table that goes with a compaction.
//
// The pool is [planes, n_pages, heads, page_size, row_bytes] (planes = layers x {key, value}; any element type).  Copy i
// brings page src[i] to page dst[i] in every plane, the first rows[i] rows of every head when rows are given.  Pure HBM
// traffic: 2 bytes moved per byte copied.  A CTA takes one slice of one (page, plane), every thread several 16-byte
// pieces that are all requested before the first is stored.  16 partly filled pages of 32 layers, 32 heads of 128 (546 MB
// moved): 95 us, 5.8 TB/s = 0.89 of a copy; 12 whole pages of 12 layers, 12 heads of 64, with the table (57 MB): 13 us = 0.67.
#include "kv4.cuh"

namespace b200 {

namespace {

constexpr int CT = 256;  // threads per CTA
constexpr int CU = 8;    // pieces in flight per thread

struct CopyArgs {
  char* pool;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* rows;       // or null: whole pages
  int32_t* table;            // or null
  const int32_t* page_map;   // [n_pages]
  long long plane_bytes, page_bytes, head_bytes;  // head_bytes: one head of a page
  int n, n_planes, n_pages, page_size, row_bytes;
  int slices;                // CTAs per (copy, plane)
  int table_blocks;
  long long table_entries;
  uint32_t* status;
};

template <typename V>
__global__ void __launch_bounds__(CT) copy_pages_kernel(CopyArgs a) {
  if ((int)blockIdx.x < a.table_blocks) {
    // page-table entries: moved pages get their new place, entries that name no page stay
    const long long i = (long long)blockIdx.x * CT + threadIdx.x;
    if (i < a.table_entries) {
      const int p = a.table[i];
      if ((unsigned)p < (unsigned)a.n_pages) {
        const int to = __ldg(a.page_map + p);
        if ((unsigned)to < (unsigned)a.n_pages) a.table[i] = to;
        else atomicOr(a.status, ST_BAD_PAGE);
      }
    }
    return;
  }
  const long long item = (long long)blockIdx.x - a.table_blocks;
  const int slice = (int)(item % a.slices);
  const long long cp = item / a.slices;
  const int plane = (int)(cp % a.n_planes), i = (int)(cp / a.n_planes);
  const int s = __ldg(a.src + i), d = __ldg(a.dst + i);
  if ((unsigned)s >= (unsigned)a.n_pages || (unsigned)d >= (unsigned)a.n_pages) {
    if (threadIdx.x == 0) atomicOr(a.status, ST_BAD_PAGE);
    return;
  }
  if (s == d) return;
  const char* from = a.pool + plane * a.plane_bytes + s * a.page_bytes;
  char* to = a.pool + plane * a.plane_bytes + d * a.page_bytes;
  int rows = a.page_size;
  if (a.rows) rows = max(0, min(a.page_size, __ldg(a.rows + i)));
  const bool whole = rows == a.page_size;
  // pieces of the copy: one run of the whole page, or `rows` rows of every head
  const long long run = whole ? a.page_bytes / (long long)sizeof(V) : (long long)rows * a.row_bytes / (long long)sizeof(V);
  const long long pieces = whole ? run : run * (a.page_bytes / a.head_bytes);
  for (long long p0 = (long long)slice * CT * CU; p0 < pieces; p0 += (long long)a.slices * CT * CU) {
    V x[CU];
    long long off[CU];
#pragma unroll
    for (int j = 0; j < CU; ++j) {
      const long long p = p0 + j * CT + threadIdx.x;
      off[j] = -1;
      if (p < pieces) {
        off[j] = whole ? p * (long long)sizeof(V)
                       : (long long)((uint32_t)p / (uint32_t)run) * a.head_bytes + (long long)((uint32_t)p % (uint32_t)run) * (long long)sizeof(V);
        x[j] = *reinterpret_cast<const V*>(from + off[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < CU; ++j)
      if (off[j] >= 0) *reinterpret_cast<V*>(to + off[j]) = x[j];
  }
}

template <typename V> int32_t launch_copy(const CopyArgs& a, cudaStream_t stream) {
  const long long blocks = a.table_blocks + (long long)a.n * a.n_planes * a.slices;
  if (blocks > 0x7fffffffLL) return fail(B200_ERR_BAD_SHAPE, "copy pages: too many copies for one call");
  if (blocks == 0) return B200_OK;
  copy_pages_kernel<V><<<(unsigned)blocks, CT, 0, stream>>>(a);
  B200_LAUNCH_OK("copy_pages_kernel");
  return B200_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int32_t b200_copy_pages(void* pool, int32_t n_planes, int32_t n_pages, int32_t n_heads, int32_t page_size,
                                   int32_t row_bytes, const int32_t* src, const int32_t* dst, const int32_t* rows,
                                   int32_t n, int32_t* page_table, int64_t table_entries, const int32_t* page_map,
                                   b200_stream_t stream) {
  if (n_planes <= 0 || n_pages < 0 || n_heads <= 0 || page_size <= 0 || row_bytes <= 0 || n < 0 || table_entries < 0)
    return fail(B200_ERR_BAD_SHAPE, "copy pages: sizes must be positive");
  if (page_table && !page_map) return fail(B200_ERR_INVALID_ARG, "copy pages: a page table needs a page map");
  CopyArgs a;
  a.head_bytes = (long long)page_size * row_bytes;
  a.page_bytes = a.head_bytes * n_heads;
  if (a.head_bytes > 0x7fffffffLL || a.page_bytes > 0x7fffffffLL) return fail(B200_ERR_BAD_SHAPE, "copy pages: a page exceeds 2 GiB");
  a.plane_bytes = a.page_bytes * n_pages;
  a.pool = (char*)pool; a.src = src; a.dst = dst; a.rows = rows; a.n = n;
  a.n_planes = n_planes; a.n_pages = n_pages; a.page_size = page_size; a.row_bytes = row_bytes;
  a.table = page_table; a.page_map = page_map; a.table_entries = page_table ? table_entries : 0;
  if (n == 0 && a.table_entries == 0) return B200_OK;
  if (n > 0 && (!pool || !src || !dst)) return fail(B200_ERR_INVALID_ARG, "copy pages: null operand");
  a.status = device_status_word();
  if (!a.status) return fail(B200_ERR_CUDA, "no device status word");
  a.table_blocks = (int)((a.table_entries + CT - 1) / CT);
  // the widest piece that divides a row (a whole page when no row counts are given) and the pool's alignment
  const unsigned long long grain = (unsigned long long)(rows ? (long long)row_bytes : a.page_bytes) | reinterpret_cast<uintptr_t>(pool) | (1ULL << 4) |
                                   (unsigned long long)a.page_bytes;
  const int width = (int)(grain & (~grain + 1));
  a.slices = (int)((a.page_bytes / width + CT * CU - 1) / (CT * CU));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (width) {
    case 16: return launch_copy<uint4>(a, s);
    case 8: return launch_copy<uint2>(a, s);
    case 4: return launch_copy<uint32_t>(a, s);
    case 2: return launch_copy<uint16_t>(a, s);
    default: return launch_copy<uint8_t>(a, s);
  }
}
