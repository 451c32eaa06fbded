// NVFP4 weight times 16-bit activations for a few rows (vfb_nvfp4_weight_only):
// one warp per output feature, each lane decoding 32 consecutive weights at a
// time, fp32 sums.
#include "common.cuh"
#include "nvfp4_quant.cuh"

namespace vfb {
namespace {

// Decodes two e2m1 codes (low nibble first); every value is exact in fp16.
__device__ __forceinline__ float2 e2m1_pair(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 b0, b1;\n\t"
      "mov.b16 {b0, b1}, %1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t}"
      : "=r"(h)
      : "h"(static_cast<uint16_t>(byte)));
  return __half22float2(*reinterpret_cast<__half2 *>(&h));
}

template <typename T>
__global__ void __launch_bounds__(256) weight_only_kernel(const T *__restrict__ x, int64_t M, int64_t ldx,
                                                          const uint8_t *__restrict__ codes,
                                                          const uint8_t *__restrict__ sf,
                                                          const float *__restrict__ alpha,
                                                          const __nv_bfloat16 *__restrict__ bias, int64_t N,
                                                          int64_t K, __nv_bfloat16 *__restrict__ out,
                                                          int64_t ldo) {
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= N) return;
  for (int64_t m = 0; m < M; ++m) {
    float acc = 0.0f;
    for (int64_t g = lane; g < K / 16; g += 32) {
      const uint2 w = *reinterpret_cast<const uint2 *>(codes + n * (K / 2) + g * 8);
      const uint32_t word[2] = {w.x, w.y};
      float sum = 0.0f;
      for (int i = 0; i < 8; ++i) {
        const float2 f = e2m1_pair((word[i / 4] >> (8 * (i % 4))) & 0xff);
        const T *xp = x + m * ldx + g * 16 + 2 * i;
        sum = fmaf(f.x, static_cast<float>(xp[0]), sum);
        sum = fmaf(f.y, static_cast<float>(xp[1]), sum);
      }
      acc = fmaf(sum, e4m3_value(sf[sf_offset(n, g, K / 64)]), acc);
    }
    for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(~0u, acc, o);
    if (lane == 0)
      out[m * ldo + n] = __float2bfloat16_rn(*alpha * acc + (bias ? __bfloat162float(bias[n]) : 0.0f));
  }
}

}  // namespace
}  // namespace vfb

extern "C" int64_t vfb_nvfp4_weight_only_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N <= 0 || K <= 0 || N % 128 || K % 64) return -1;
  return 0;
}

extern "C" int vfb_nvfp4_weight_only(const void *x, int32_t dtype, int64_t M, int64_t ldx, const void *w_codes,
                                     const void *w_sf, const float *alpha, const void *bias, int64_t N,
                                     int64_t K, void *out, int64_t ldo, void *workspace,
                                     int64_t workspace_bytes, void *stream) {
  using namespace vfb;
  const int64_t need = vfb_nvfp4_weight_only_workspace_bytes(M, N, K);
  if (need < 0 || ldx < K || ldo < N || (dtype != 0 && dtype != 1))
    return set_error(VFB_EINVAL,
                     "vfb_nvfp4_weight_only: need K %% 64 == 0, N %% 128 == 0, ldx >= K, ldo >= N, dtype 0 "
                     "(bf16) or 1 (fp16)");
  if (M == 0) return VFB_OK;
  if (!x || !w_codes || !w_sf || !alpha || !out)
    return set_error(VFB_EINVAL, "vfb_nvfp4_weight_only: NULL pointer");
  if (!aligned16(w_codes) || reinterpret_cast<uintptr_t>(w_sf) % 4)
    return set_error(VFB_EINVAL, "vfb_nvfp4_weight_only: codes must be 16-byte aligned, scales 4-byte aligned");
  if (workspace_bytes < need || (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256)))
    return set_error(VFB_EINVAL, "vfb_nvfp4_weight_only: needs %lld bytes of 256-byte aligned workspace",
                     (long long)need);
  int rc = check_device(nullptr);
  if (rc != VFB_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned blocks = static_cast<unsigned>((N + 7) / 8);
  auto *w = static_cast<const uint8_t *>(w_codes);
  auto *f = static_cast<const uint8_t *>(w_sf);
  auto *b = static_cast<const __nv_bfloat16 *>(bias);
  auto *o = static_cast<__nv_bfloat16 *>(out);
  if (dtype == 0)
    weight_only_kernel<<<blocks, 256, 0, s>>>(static_cast<const __nv_bfloat16 *>(x), M, ldx, w, f, alpha, b, N, K, o, ldo);
  else
    weight_only_kernel<<<blocks, 256, 0, s>>>(static_cast<const __half *>(x), M, ldx, w, f, alpha, b, N, K, o, ldo);
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return set_error(VFB_ECUDA, "vfb_nvfp4_weight_only launch: %s", cudaGetErrorString(err));
  return VFB_OK;
}
