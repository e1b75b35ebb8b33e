// The device status word of a library image and its host-side readers.
#include <mutex>

#include "device_common.cuh"
#include "../../include/mllmb200.h"

namespace mllmb200 {

__device__ unsigned int g_device_status = 0;
__device__ unsigned int g_taken_status = 0;

namespace {
// The first bit of a group that is set, taken out of the word; all else stays in it for the next reader.
__global__ void take_status_kernel(unsigned int group) {
  const unsigned int word = atomicOr(&g_device_status, 0u) >> group;
  const unsigned int bit = word & kDevStatusTimeout ? kDevStatusTimeout : word & kDevStatusBadHeader ? kDevStatusBadHeader : word & kDevStatusBadPage;
  if (bit) atomicAnd(&g_device_status, ~(bit << group));
  g_taken_status = bit;
}
cudaError_t take_status(cudaStream_t st, int* status, unsigned int group) {
  static std::mutex one;  // (g_taken_status is everybody's)
  const std::lock_guard<std::mutex> lock(one);
  unsigned int bit = 0;
  take_status_kernel<<<1, 1, 0, st>>>(group);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(&bit, g_taken_status, sizeof(bit), 0, cudaMemcpyDeviceToHost, st);
  const cudaError_t waited = cudaStreamSynchronize(st);
  if (e == cudaSuccess) e = waited;
  *status = bit == kDevStatusTimeout ? MLLMB200_TIMEOUT : bit == kDevStatusBadHeader ? MLLMB200_BAD_BLOB : bit == kDevStatusBadPage ? MLLMB200_BAD_PAGE : MLLMB200_OK;
  return e;
}
}  // namespace

// Both wait for the stream, and read what the kernels of this image reported on the current device, on any stream: one kind a call.
cudaError_t read_device_status(cudaStream_t st, int* status) { return take_status(st, status, 0); }
cudaError_t read_operator_status(cudaStream_t st, int* status) { return take_status(st, status, kDevStatusOfOperators); }

}  // namespace mllmb200
