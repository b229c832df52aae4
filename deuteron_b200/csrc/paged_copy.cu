// Copies whole pages of a cache inside its pool: forks (the shared last page of a beam) and compaction (live pages moved to
// low numbers). Bytes read once and written once; bound by memory.
#include "paged.cuh"

namespace dtn {

struct CopyParams {
  char* pool;
  int64_t plane_stride, page_stride, page_bytes;   // bytes
  int64_t planes, pages, pairs;
  const int *sources, *destinations;
  int* status;
};

// One block per (pair, plane); V is the widest vector that divides every address and extent.
template <typename V>
__global__ void __launch_bounds__(256) copy_pages_kernel(const CopyParams p) {
  const int64_t pair = blockIdx.x % p.pairs, plane = blockIdx.x / p.pairs;
  const int from = p.sources[pair], to = p.destinations[pair];
  if (from < 0 || from >= p.pages || to < 0 || to >= p.pages) {
    if (threadIdx.x == 0) paged_report(p.status, PAGED_STATUS_COPY);
    return;
  }
  const V* src = reinterpret_cast<const V*>(p.pool + plane * p.plane_stride + from * p.page_stride);
  V* dst = reinterpret_cast<V*>(p.pool + plane * p.plane_stride + to * p.page_stride);
  for (int64_t i = threadIdx.x; i < p.page_bytes / (int64_t)sizeof(V); i += blockDim.x) dst[i] = src[i];
}

}  // namespace dtn

extern "C" int dtn_copy_pages(void* pool, int64_t planes, int64_t plane_stride_bytes, int64_t pages, int64_t page_stride_bytes, int64_t page_bytes,
                              const int* sources, const int* destinations, int64_t pairs, void* stream) {
  using namespace dtn;
  DTN_REQUIRE(planes >= 0 && pages >= 0 && page_bytes >= 0 && pairs >= 0, DTN_ERR_INVALID, "copy pages: negative extent");
  if (planes == 0 || pages == 0 || page_bytes == 0 || pairs == 0) return DTN_OK;
  DTN_REQUIRE(pool && sources && destinations, DTN_ERR_INVALID, "copy pages: null pointer");
  DTN_REQUIRE(pages < (1LL << 31) && pairs < (1LL << 31) && planes * pairs < (1LL << 31), DTN_ERR_UNSUPPORTED, "copy pages: too many pages for one launch");
  cudaStream_t s = as_stream(stream);
  CopyParams p = {static_cast<char*>(pool), plane_stride_bytes, page_stride_bytes, page_bytes, planes, pages, pairs, sources, destinations,
                  device_status_word_unless_capturing(s)};
  const uint64_t all = reinterpret_cast<uintptr_t>(pool) | (uint64_t)plane_stride_bytes | (uint64_t)page_stride_bytes | (uint64_t)page_bytes;
  const unsigned blocks = (unsigned)(planes * pairs);
  if (all % 16 == 0)
    copy_pages_kernel<uint4><<<blocks, 256, 0, s>>>(p);
  else if (all % 4 == 0)
    copy_pages_kernel<uint32_t><<<blocks, 256, 0, s>>>(p);
  else
    copy_pages_kernel<uint8_t><<<blocks, 256, 0, s>>>(p);
  DTN_LAUNCH_CHECK("copy_pages_kernel");
  return DTN_OK;
}
