// What the operators of a paged key-value cache share: element conversion, the report of a bad page number.
#pragma once

#include "dtn_common.cuh"

namespace dtn {

// The status word when it can be had without an allocation that a stream capture forbids: nullptr (no reports) for the
// first call on a device when that call is being captured.
int* device_status_word_unless_capturing(cudaStream_t s);

// Status codes, role in the upper bits as for the bounded waits: a page number, position or length that the tables do not cover.
constexpr int PAGED_STATUS_ATTENTION = 0x6100;
constexpr int PAGED_STATUS_APPEND = 0x6200;
constexpr int PAGED_STATUS_COPY = 0x6300;

static inline bool paged_storage_known(int64_t storage) {
  return storage == DTN_STORAGE_F32 || storage == DTN_STORAGE_F16 || storage == DTN_STORAGE_BF16;
}
static inline int paged_storage_bytes(int64_t storage) { return storage == DTN_STORAGE_F32 ? 4 : 2; }

#ifdef __CUDACC__

// The first report stands until it is read: a wait that ran out before is not covered by a bad page that may follow from it.
__device__ __forceinline__ void paged_report(int* status, int code) {
  if (status != nullptr) atomicCAS(status, 0, code | (int)(blockIdx.x & 0xff));
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

#endif  // __CUDACC__

}  // namespace dtn
