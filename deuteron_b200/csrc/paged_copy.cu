// Copies whole pages of a cache inside its pool: forks (the shared last page of a beam) and compaction (live pages moved to
// low numbers). Bytes read once and written once; bound by memory: 600 pages of 32 KB in 32 planes (1.26 GB) 191 us, the copy
// rate (205 us with one vector per thread in flight); 8 pages in 64 planes (34 MB) 5.9 us, 0.87 of it.
#include "paged.cuh"

namespace dtn {

struct CopyParams {
  char* pool;
  int64_t plane_stride, page_stride, page_bytes;   // bytes
  int64_t planes, pages, pairs;
  const int *sources, *destinations;
  int* status;
};

// GROUP threads copy one page of one plane, COPY_AHEAD vectors each at a time, all requested before the first is stored; V is
// the widest vector that divides every address and extent.
constexpr int COPY_THREADS = 256;
constexpr int COPY_AHEAD = 8;

template <typename V, int GROUP>
__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(const CopyParams p) {
  const int64_t page = (int64_t)blockIdx.x * (COPY_THREADS / GROUP) + threadIdx.x / GROUP;
  if (page >= p.pairs * p.planes) return;
  const int64_t plane = page / p.pairs, pair = page - plane * p.pairs;
  const int lane = threadIdx.x % GROUP;
  const int from = p.sources[pair], to = p.destinations[pair];
  if (from < 0 || from >= p.pages || to < 0 || to >= p.pages) {
    if (lane == 0) paged_report(p.status, PAGED_STATUS_COPY);
    return;
  }
  const V* src = reinterpret_cast<const V*>(p.pool + plane * p.plane_stride + from * p.page_stride);
  V* dst = reinterpret_cast<V*>(p.pool + plane * p.plane_stride + to * p.page_stride);
  const int64_t vectors = p.page_bytes / (int64_t)sizeof(V);
  for (int64_t i = lane; i < vectors; i += COPY_AHEAD * GROUP) {
    V x[COPY_AHEAD];
#pragma unroll
    for (int j = 0; j < COPY_AHEAD; ++j)
      if (i + j * GROUP < vectors) x[j] = src[i + j * GROUP];
#pragma unroll
    for (int j = 0; j < COPY_AHEAD; ++j)
      if (i + j * GROUP < vectors) dst[i + j * GROUP] = x[j];
  }
}

template <typename V>
static int copy_pages_launch(const CopyParams& p, cudaStream_t s) {
  const int64_t pages = p.pairs * p.planes;
  // a block per page, or a warp where a block's threads would have less than two vectors each
  if (p.page_bytes / (int64_t)sizeof(V) >= 2 * COPY_THREADS)
    copy_pages_kernel<V, COPY_THREADS><<<(unsigned)pages, COPY_THREADS, 0, s>>>(p);
  else
    copy_pages_kernel<V, 32><<<(unsigned)((pages + COPY_THREADS / 32 - 1) / (COPY_THREADS / 32)), COPY_THREADS, 0, s>>>(p);
  DTN_LAUNCH_CHECK("copy_pages_kernel");
  return DTN_OK;
}

}  // namespace dtn

extern "C" int dtn_copy_pages(void* pool, int64_t planes, int64_t plane_stride_bytes, int64_t pages, int64_t page_stride_bytes, int64_t page_bytes,
                              const int* sources, const int* destinations, int64_t pairs, void* stream) {
  using namespace dtn;
  DTN_REQUIRE(planes >= 0 && pages >= 0 && page_bytes >= 0 && pairs >= 0, DTN_ERR_INVALID, "copy pages: negative extent");
  if (planes == 0 || pages == 0 || page_bytes == 0 || pairs == 0) return DTN_OK;
  DTN_REQUIRE(pool && sources && destinations, DTN_ERR_INVALID, "copy pages: null pointer");
  DTN_REQUIRE(pages < (1LL << 31) && pairs < (1LL << 31) && planes <= ((1LL << 31) - 1) / pairs, DTN_ERR_UNSUPPORTED, "copy pages: too many pages for one launch");
  cudaStream_t s = as_stream(stream);
  CopyParams p = {static_cast<char*>(pool), plane_stride_bytes, page_stride_bytes, page_bytes, planes, pages, pairs, sources, destinations,
                  device_status_word_unless_capturing(s)};
  const uint64_t all = reinterpret_cast<uintptr_t>(pool) | (uint64_t)plane_stride_bytes | (uint64_t)page_stride_bytes | (uint64_t)page_bytes;
  if (all % 16 == 0) return copy_pages_launch<uint4>(p, s);
  if (all % 4 == 0) return copy_pages_launch<uint32_t>(p, s);
  return copy_pages_launch<uint8_t>(p, s);
}
