// NVFP4 weight times 16-bit activations for a few rows (vfb_nvfp4_weight_only).
//
//   y[m,n] = bf16( alpha * sum_k x[m,k] e2m1(W[n,k]) e4m3(sf[n,k/16]) + bias[n] )
//
// The work is reading the weight once (K/2 + K/16 bytes a row), so the kernel
// is built around many wide loads in flight and few instructions for a weight:
//   * mma.m16n8k16 with the weights as the 16-row operand and up to 8 rows of x
//     as the 8 columns: one instruction multiplies 256 weights, whatever M <= 8.
//     (tcgen05 wants its operands in shared memory, 128 rows at a time: the
//     decoded weights would make a round trip that the product is too small to
//     pay for.)
//   * a decoded weight e2m1 * e4m3 has at most six significant bits and lies in
//     2^-10 .. 2688, so it is exact in fp16: cvt.f16x2.e2m1x2 and one HMUL2.
//     x is brought to fp16 too, each row multiplied by a power of two that puts
//     its largest magnitude (of the block's K range) into [2^14, 2^15): exact
//     for elements down to 2^-30 of it, 2^-39 of it absolute below.  Products
//     are exact, sums fp32.
//   * the order of k inside a product is free as long as both operands agree.
//     A lane takes 32 consecutive weights of a row (one 16-byte load), a quad 128
//     of them (a "step": 64 bytes of every row), and x is laid out in shared
//     memory so that the matching fragments are conflict-free 16-byte loads.
//   * the 16 rows of a unit are four neighbours in each of the four 32-row
//     quarters of a 128-row scale tile, whose scales for four groups are then
//     64 consecutive bytes.
//
// A block has eight warps: WR row groups of RU units each, the steps of the
// block's K range dealt out to the 8 / WR warps of a row group.  The warps'
// sums are added in shared memory, those of the blocks of a cluster (one K
// range each) through distributed shared memory, always in the same order.
#include <type_traits>

#include "common.cuh"

namespace vfb {
namespace {

constexpr int kWarps = 8;
constexpr int kStep = 128;  // k of a step

struct Args {
  const void *x;
  const uint8_t *codes, *sf;
  const float *alpha;
  const __nv_bfloat16 *bias;
  __nv_bfloat16 *out;
  int64_t ldx, ldo;
  int32_t M, N, K;
  int32_t steps;      // steps of a block's K range
  uint32_t chunk_inverse;  // 2^32 / (16 * steps), rounded up: exact for the i / (16 * steps) that occur
  int32_t vector_x;   // rows of x are 16-byte aligned
};

// Loads that are skipped (the registers keep what they held) unless `in`.  The
// results are only touched when they are multiplied, two steps later.
__device__ __forceinline__ void load_stream(uint4 &v, const void *p, bool in) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %5, 0;\n\t"
      "@p ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}"
      : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
      : "l"(p), "r"(static_cast<uint32_t>(in)));
}

__device__ __forceinline__ void load_word(uint32_t &v, const void *p, bool in) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "@p ld.global.nc.u32 %0, [%1];\n\t}"
      : "+r"(v)
      : "l"(p), "r"(static_cast<uint32_t>(in)));
}

// Four bytes of e2m1 pairs -> four f16x2 (low nibble in the low half).
__device__ __forceinline__ void decode_e2m1x8(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

__device__ __forceinline__ uint32_t decode_e4m3x2(uint16_t s) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(s));
  return h;
}

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ void mma_m16n8k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight elements of a row of x, zeros behind `left`.
template <typename T>
__device__ __forceinline__ uint4 load_x8(const T *p, bool vector, int left) {
  if (vector && left >= 8) return __ldg(reinterpret_cast<const uint4 *>(p));
  uint32_t w[4] = {};
  const uint16_t *u = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) w[j / 2] |= static_cast<uint32_t>(__ldg(u + j)) << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// Exponent of the power of two that a row with this largest magnitude (as bits
// of a non-negative f32) is multiplied by.
__device__ __forceinline__ int row_shift(uint32_t max_bits) {
  const int e = static_cast<int>(max_bits >> 23);  // biased; 0 for subnormals and zero
  if (max_bits == 0) return 0;
  return min(14 - (min(e, 254) - 127), 126);
}

template <int NT, int RU, int WR>
struct Shape {
  static constexpr int tokens = 8 * NT;
  static constexpr int rows = 16 * RU * WR;       // of the weight, in a block
  static constexpr int k_warps = kWarps / WR;
  static constexpr int row_bytes(int steps) { return steps * kStep * 2 + 64; }  // of x, padded against bank conflicts
  static constexpr int sum_bytes = k_warps * rows * tokens * 4;
};

// Blocks that share an SM (by registers).
template <int NT, int RU>
constexpr int blocks_per_sm() { return NT == 1 && RU == 2 ? 3 : 2; }

template <int RU>
struct Batch {  // the weights of one step
  uint4 w[RU][2];
  uint32_t s[RU][2];  // four groups' scales, of which a lane uses two
};

template <typename T, int NT, int RU, int WR>
__global__ void __launch_bounds__(32 * kWarps, blocks_per_sm<NT, RU>()) weight_only_kernel(const Args p) {
  using S = Shape<NT, RU, WR>;
  constexpr bool kScaled = std::is_same<T, __nv_bfloat16>::value;  // rows of x carry a power of two
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t row_max[S::tokens];
  __shared__ float bias[S::rows];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int split = gridDim.x;  // cluster: blocks along K
  const int part = blockIdx.x;
  const int m0 = blockIdx.z * S::tokens;
  const int tokens = min(S::tokens, p.M - m0);
  const int unit0 = (blockIdx.y * WR + warp % WR) * RU;  // of 16 rows; eight units in 128 rows
  const int64_t row_block = unit0 / 8;
  const int k_warp = warp / WR;
  const int k_begin = part * p.steps * kStep;
  const int steps = max(0, min(p.steps, (p.K - k_begin + kStep - 1) / kStep));

  // weight row of row r of the block: a quarter's rows of all its units
  const auto feature = [&](int r) {
    const int first = blockIdx.y * WR * RU, quarter_rows = 4 * RU * WR;
    return static_cast<int64_t>(first / 8) * 128 + r / quarter_rows * 32 + 4 * (first % 8) + r % quarter_rows;
  };

  grid_dependency_wait();

  // rows g and g + 8 of unit u: see the header; 32-bit offsets inside the scale tile's 128 rows
  const uint32_t half_k = p.K / 2;
  const uint8_t *codes = p.codes + row_block * 128 * half_k;
  const uint8_t *sf = p.sf + row_block * (p.K / 64) * 512;
  const uint32_t in_quarter = 4 * (unit0 % 8) + g / 4;
  const uint32_t code_at = ((g % 4) * 32 + in_quarter) * half_k + k_begin / 2 + 16 * t;
  const uint32_t sf_at = (k_begin / 64 + t / 2) * 512 + in_quarter * 16 + (g % 4) * 4;
  const int in_steps = max(0, (p.K - k_begin - 32 * t + kStep - 1) / kStep);
  const auto load = [&](Batch<RU> &b, int step) {
    const bool in = step < min(steps, in_steps);
#pragma unroll
    for (int u = 0; u < RU; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        load_stream(b.w[u][r], codes + (code_at + (4 * u + 2 * r) * half_k + step * (kStep / 2)), in);
        load_word(b.s[u][r], sf + (sf_at + (4 * u + 2 * r) * 16 + step * 1024), in);
      }
  };
  Batch<RU> batch[2] = {};
  load(batch[0], k_warp);
  load(batch[1], k_warp + S::k_warps);

  const float alpha = __ldg(p.alpha);
  if (tid < S::rows) bias[tid] = p.bias != nullptr ? __bfloat162float(p.bias[feature(tid)]) : 0.0f;

  // ---- x to fp16 in shared memory ----
  const int row_bytes = S::row_bytes(p.steps);
  const T *x = static_cast<const T *>(p.x) + m0 * p.ldx;
  const int chunks = p.steps * (kStep / 8);  // of eight elements, in a row; a multiple of 16
  const int items = tokens * chunks;
  const auto row_of = [&](int i) { return static_cast<int>(__umulhi(i, p.chunk_inverse)); };  // i / chunks
  // chunk 4 * t + i of a step is read by lane t in its i-th pair of products
  const auto place = [&](int m, int c) {
    return reinterpret_cast<uint4 *>(smem + m * row_bytes + (c / 16) * 256 + (c % 4) * 64 + (c % 16) / 4 * 16);
  };
  if (kScaled) {
    if (tid < S::tokens) row_max[tid] = 0;
    __syncthreads();
  }
  for (int i0 = tid; i0 < items; i0 += 4 * 32 * kWarps) {
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * 32 * kWarps, m = row_of(i), c = i - m * chunks;
      if (i < items) v[j] = load_x8(x + m * p.ldx + k_begin + 8 * c, p.vector_x, p.K - k_begin - 8 * c);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * 32 * kWarps, m = row_of(i), c = i - m * chunks;
      if (i >= items) break;  // for all 16 lanes of a row's piece at once
      *place(m, c) = v[j];
      if (!kScaled) continue;
      const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // magnitudes compare as integers; NaN is left out
        const uint32_t lo = (w[e] << 16) & 0x7FFFFFFFu, hi = w[e] & 0x7FFF0000u;
        top = max(top, lo > 0x7F800000u ? 0u : lo);
        top = max(top, hi > 0x7F800000u ? 0u : hi);
      }
      top = __reduce_max_sync(0xFFFFu << (lane & 16), top);
      if (lane % 16 == 0 && top) atomicMax(&row_max[m], top);
    }
  }
  __syncthreads();
  if (kScaled) {
    for (int i = tid; i < items; i += 32 * kWarps) {
      const int m = row_of(i), c = i - m * chunks;
      const float factor = power_of_two(row_shift(row_max[m]));
      uint4 v = *place(m, c);
      uint32_t *w = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __half2 h = __floats2half2_rn(__uint_as_float(w[e] << 16) * factor,
                                            __uint_as_float(w[e] & 0xFFFF0000u) * factor);
        w[e] = *reinterpret_cast<const uint32_t *>(&h);
      }
      *place(m, c) = v;
    }
    __syncthreads();
  }

  // ---- products ----
  float acc[RU][NT][4] = {};
  const auto multiply = [&](const Batch<RU> &b, int step) {
    const bool in = step < in_steps;  // K may end on half a step: a zero scale makes any code 0
    uint32_t scale[RU][2][2];         // unit, row, group: the scale in both halves
#pragma unroll
    for (int u = 0; u < RU; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t h = decode_e4m3x2(in ? static_cast<uint16_t>(b.s[u][r] >> (16 * (t % 2))) : 0);
        scale[u][r][0] = __byte_perm(h, 0, 0x1010);
        scale[u][r][1] = __byte_perm(h, 0, 0x3232);
      }
    const uint8_t *xs = smem + g * row_bytes + step * 256 + t * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 f[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        f[n] = make_uint4(0, 0, 0, 0);
        if (8 * n + g < tokens) f[n] = *reinterpret_cast<const uint4 *>(xs + 8 * n * row_bytes + i * 64);
      }
#pragma unroll
      for (int u = 0; u < RU; ++u) {
        uint32_t a[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          decode_e2m1x8(reinterpret_cast<const uint32_t *>(&b.w[u][r])[i], a[r]);
#pragma unroll
          for (int j = 0; j < 4; ++j) a[r][j] = mul_f16x2(a[r][j], scale[u][r][i / 2]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_m16n8k16(acc[u][n], a[0][0], a[1][0], a[0][1], a[1][1], f[n].x, f[n].y);
          mma_m16n8k16(acc[u][n], a[0][2], a[1][2], a[0][3], a[1][3], f[n].z, f[n].w);
        }
      }
    }
  };
  for (int step = k_warp; step < steps; step += 2 * S::k_warps) {
    multiply(batch[0], step);
    load(batch[0], step + 2 * S::k_warps);
    if (step + S::k_warps < steps) multiply(batch[1], step + S::k_warps);
    load(batch[1], step + 3 * S::k_warps);
  }

  // ---- sums over the warps, then over the blocks of the cluster ----
  __syncthreads();  // x is read
  float *sums = reinterpret_cast<float *>(smem);  // [k warp][token][row]
#pragma unroll
  for (int u = 0; u < RU; ++u)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = (g % 4) * (4 * RU * WR) + 4 * ((warp % WR) * RU + u) + g / 4 + 2 * (j / 2);
        const int token = 8 * n + 2 * t + j % 2;
        sums[(k_warp * S::tokens + token) * S::rows + row] = acc[u][n][j];
      }
  __syncthreads();
  for (int i = tid; i < tokens * S::rows; i += 32 * kWarps) {
    float v = sums[i];
#pragma unroll
    for (int w = 1; w < S::k_warps; ++w) v += sums[w * S::tokens * S::rows + i];
    v *= alpha;
    if (kScaled) v *= power_of_two(-row_shift(row_max[i / S::rows]));
    sums[i] = v;
  }
  cluster_sync();
  for (int i = tid * split + part; i < tokens * S::rows; i += 32 * kWarps * split) {
    float v = 0.0f;
    for (int c = 0; c < split; ++c) {
      float other;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other) : "r"(map_to_rank(smem_u32(sums + i), c)));
      v += other;
    }
    const int token = i / S::rows, row = i % S::rows;
    p.out[(m0 + token) * p.ldo + feature(row)] = __float2bfloat16_rn(v + bias[row]);
  }
  cluster_sync();  // the others have read this block's sums
}

template <typename T, int NT, int RU, int WR>
int launch(Args p, int split, cudaStream_t stream) {
  using S = Shape<NT, RU, WR>;
  auto kernel = weight_only_kernel<T, NT, RU, WR>;
  const int steps = (p.K + kStep - 1) / kStep;
  p.steps = (steps + split - 1) / split;
  p.chunk_inverse = static_cast<uint32_t>((1ull << 32) / (p.steps * 16)) + 1;
  const int x_bytes = (p.M < S::tokens ? p.M : S::tokens) * S::row_bytes(p.steps);
  const int smem = x_bytes > S::sum_bytes ? x_bytes : S::sum_bytes;
  constexpr int kMost = 200 * 1024;
  if (smem > kMost) return set_error(VFB_EINVAL, "vfb_nvfp4_weight_only: K is too large");
  static std::atomic<uint64_t> smem_set[kMaxAttrDevices];
  int rc = ensure_smem_optin(reinterpret_cast<const void *>(kernel), kMost, smem_set);
  if (rc != VFB_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(split, p.N / S::rows, (p.M + S::tokens - 1) / S::tokens);
  cfg.blockDim = dim3(32 * kWarps, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p);
  if (err != cudaSuccess) return set_error(VFB_ECUDA, "vfb_nvfp4_weight_only launch: %s", cudaGetErrorString(err));
  return VFB_OK;
}

// Blocks along K: as many as still run at once, but every warp keeps two steps;
// more where x of a K range would not let that many blocks share an SM.
template <typename T, int NT, int RU, int WR>
int launch_split(const Args &p, int sms, cudaStream_t stream) {
  using S = Shape<NT, RU, WR>;
  const int steps = (p.K + kStep - 1) / kStep;
  const int tokens = p.M < S::tokens ? p.M : S::tokens;
  const int64_t blocks = static_cast<int64_t>(p.N / S::rows) * ((p.M + S::tokens - 1) / S::tokens);
  const int resident = blocks_per_sm<NT, RU>();
  const int x_most = 216 * 1024 / resident;
  int split = 1;
  while (split < 8 && ((2 * blocks * split <= resident * sms && steps >= 4 * split * S::k_warps) ||
                       tokens * S::row_bytes((steps + split - 1) / split) > x_most))
    split *= 2;
  return launch<T, NT, RU, WR>(p, split, stream);
}

template <typename T>
int run(const Args &p, int sms, cudaStream_t s) {
  if (p.M <= 2) return launch_split<T, 1, 2, 1>(p, sms, s);
  if (p.M <= 8) return launch_split<T, 1, 4, 2>(p, sms, s);
  if (p.M <= 16 || p.K > 16384) return launch_split<T, 2, 2, 4>(p, sms, s);
  return launch_split<T, 4, 2, 4>(p, sms, s);
}

constexpr int64_t kMaxK = 32768;

}  // namespace
}  // namespace vfb

extern "C" int vfb_nvfp4_weight_only(const void *x, int32_t dtype, int64_t M, int64_t ldx, const void *w_codes,
                                     const void *w_sf, const float *alpha, const void *bias, int64_t N,
                                     int64_t K, void *out, int64_t ldo, void *stream) {
  using namespace vfb;
  if (M < 0 || N <= 0 || K <= 0 || N % 128 || K % 64 || K > kMaxK || N > (1 << 20) || M > (1 << 19) || ldx < K ||
      ldo < N || (dtype != 0 && dtype != 1))
    return set_error(VFB_EINVAL,
                     "vfb_nvfp4_weight_only: need K %% 64 == 0, K <= %lld, N %% 128 == 0, N <= 1048576, M <= 524288, "
                     "ldx >= K, ldo >= N, dtype 0 (bf16) or 1 (fp16)",
                     (long long)kMaxK);
  if (M == 0) return VFB_OK;
  if (!x || !w_codes || !w_sf || !alpha || !out)
    return set_error(VFB_EINVAL, "vfb_nvfp4_weight_only: NULL pointer");
  if (!aligned16(w_codes) || reinterpret_cast<uintptr_t>(w_sf) % 4)
    return set_error(VFB_EINVAL, "vfb_nvfp4_weight_only: codes must be 16-byte aligned, scales 4-byte aligned");
  int sms = 0;
  int rc = check_device(&sms);
  if (rc != VFB_OK) return rc;
  Args p = {};
  p.x = x;
  p.codes = static_cast<const uint8_t *>(w_codes);
  p.sf = static_cast<const uint8_t *>(w_sf);
  p.alpha = alpha;
  p.bias = static_cast<const __nv_bfloat16 *>(bias);
  p.out = static_cast<__nv_bfloat16 *>(out);
  p.ldx = ldx;
  p.ldo = ldo;
  p.M = static_cast<int32_t>(M);
  p.N = static_cast<int32_t>(N);
  p.K = static_cast<int32_t>(K);
  p.vector_x = aligned16(x) && ldx % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == 0 ? run<__nv_bfloat16>(p, sms, s) : run<__half>(p, sms, s);
}
