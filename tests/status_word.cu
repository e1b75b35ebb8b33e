// What the readers of the device status word tell and leave, for bits that a kernel sets; built by test_device_status.py.
#include <cstdio>

#include "../mllm-advanced_b200/csrc/device_common.cuh"

namespace mllmb200 {
cudaError_t read_device_status(cudaStream_t, int*);
cudaError_t read_operator_status(cudaStream_t, int*);
}  // namespace mllmb200
using namespace mllmb200;

__global__ void raise_bits(unsigned bits) { atomicOr(&g_device_status, bits); }

int main() {
  const unsigned far = kDevStatusOfOperators;
  const unsigned raised[] = {kDevStatusBadPage << far, kDevStatusTimeout, kDevStatusTimeout | kDevStatusBadHeader, (kDevStatusTimeout | kDevStatusBadPage) << far | kDevStatusTimeout, 0};
  for (unsigned bits : raised) {
    raise_bits<<<1, 1>>>(bits);
    for (int i = 0; i < 6; ++i) {  // operators', engines', operators', ...
      int status = -1;
      if ((i & 1 ? read_device_status : read_operator_status)(nullptr, &status) != cudaSuccess) return 1;
      std::printf("%d ", status);
    }
    std::printf("\n");
  }
  return 0;
}
