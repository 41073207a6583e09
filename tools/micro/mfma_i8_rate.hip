// Rate of v_mfma_i32_32x32x32_i8 on this card: W waves per SIMD, each a loop over 6 accumulators with operands in registers, once all zeros and once
// mixed bits (the clock under the power limit depends on them).  Median of 7 launches.
//   hipcc --offload-arch=gfx950 -O3 tools/micro/mfma_i8_rate.hip -o tools/micro/mfma_i8_rate
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cstdio>
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
enum { ACC = 6, ITERS = 2000 };
__global__ void __launch_bounds__(256) k_mfma_i8(int* out, int mix) {
  const int lane = threadIdx.x;
  const v4i a = {mix * lane, mix * lane * 3, mix * 7, mix * lane * 11}, b = {mix * 5, mix * lane, mix * 13, mix * 3};
  v16i c[ACC] = {};
  for (int r = 0; r < ITERS; ++r)
#pragma unroll
    for (int i = 0; i < ACC; ++i) c[i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c[i], 0, 0, 0);
  int s = 0;
#pragma unroll
  for (int i = 0; i < ACC; ++i) s += c[i][0] + c[i][15];
  out[blockIdx.x * 256 + threadIdx.x] = s;
}
int main() {
  int* out;
  hipEvent_t e0, e1;
  if (hipMalloc(&out, 512 * 256 * sizeof(int)) != hipSuccess || hipEventCreate(&e0) != hipSuccess || hipEventCreate(&e1) != hipSuccess) return 1;
  for (int waves = 1; waves <= 2; ++waves)
    for (int mix : {0, 12345677}) {
      float ms[8];
      for (int i = 0; i < 8; ++i) {
        (void)hipEventRecord(e0);
        hipLaunchKernelGGL(k_mfma_i8, dim3(256 * waves), dim3(256), 0, 0, out, mix);
        (void)hipEventRecord(e1);
        if (hipEventSynchronize(e1) != hipSuccess) return 1;
        (void)hipEventElapsedTime(&ms[i], e0, e1);
      }
      std::sort(ms + 1, ms + 8);
      printf("v_mfma_i32_32x32x32_i8, %s operands, %d wave(s) a SIMD: %.0f TOP/s\n", mix ? "mixed" : "zero", waves,
             2.0 * 32768 * ACC * ITERS * 1024.0 * waves / (ms[4] * 1e-3) / 1e12);
    }
  return 0;
}
