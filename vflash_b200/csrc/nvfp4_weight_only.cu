// NVFP4 weight times 16-bit activations for a few rows (vfb_nvfp4_weight_only).
//
//   y[m,n] = bf16( alpha * sum_k x[m,k] e2m1(W[n,k]) e4m3(sf[n,k/16]) + bias[n] )
//
// The work is reading the weight once (K/2 + K/16 bytes a row), so the kernel
// is built around many wide loads in flight and few instructions for a weight:
//   * mma.m16n8k16 with the weights as the 16-row operand and up to 8 rows of x
//     as the 8 columns: one instruction multiplies 256 weights, whatever M <= 8.
//     (tcgen05 reads its operands from shared memory, the first also from TMEM, 128
//     rows at a time: the decoded weights would make a round trip through either, which a
//     few columns do not pay for.)
//   * a decoded weight e2m1 * e4m3 has at most six significant bits and lies in
//     2^-10 .. 2688, so it is exact in fp16: cvt.f16x2.e2m1x2 and one HMUL2.
//     x is brought to fp16 too, each row multiplied by a power of two that puts
//     its largest magnitude (of the block's K range) into [2^14, 2^15), which is
//     exact for elements down to 2^-31 of it and leaves 2^-39 of it of those below.
//     That is nothing beside the rest where at least one element in four lies
//     within 2^-12 of the largest: for weights of like size 2^-25 of their products,
//     below fp32's own roundings.  A row that is a few large elements and many small ones
//     would lose the small ones, and all of the result where the large ones meet
//     weights of 0.  A block with such a row takes bf16 for both operands: a decoded
//     weight is exact there too, but takes three more instructions for a pair (1 row,
//     12288 x 4096 14.9 us instead of 10.3, 32 rows, 16384 x 4096 35.2 instead of 24.7).
//     Sums are fp32 either way.
//   * the order of k inside a product is free as long as both operands agree.
//     A lane takes 32 consecutive weights of a row (one 16-byte load), a quad 128
//     of them (a "step": 64 bytes of every row), and x is laid out in shared
//     memory so that the matching fragments are conflict-free 16-byte loads.
//   * the 16 rows of a unit are four neighbours in each of the four 32-row
//     quarters of a 128-row scale tile, whose scales for four groups are then
//     64 consecutive bytes.
//
// A block's warps are WR row groups of RU units each, the steps of the block's K
// range dealt out to the warps of a row group.  Every warp copies its steps into
// a ring of its own in shared memory with cp.async, two steps ahead, so that
// the loads in flight hold no registers and wait for nothing but themselves; the
// loop over the steps stays rolled and small.  The warps' sums are added in shared
// memory, those of the blocks of a cluster (one K range each) through distributed
// shared memory, always in the same order.
//
// Measured (replayed graphs, weights that left L2): 1 row, N = 12288, K = 4096 10.2 us
// (2.8 TB/s with 4 us of it start and end), N = 28672, K = 5376 22.3 us (3.9 TB/s); 7
// rows of that 26.5 us, in fp16, which needs no power of two, 22.9; 32 rows, N = 12288,
// K = 4096 24.1 us: bringing x to fp16 a quarter of a block's time, products and
// decoding, with 96 of 148 SMs, most of the rest.
#include <type_traits>

#include "common.cuh"

namespace vfb {
namespace {

constexpr int kStep = 128;                   // k of a step
constexpr int kUnitBytes = 16 * kStep / 2;  // codes of a unit's step
constexpr int kUnitStage = kUnitBytes + 16 * 8;  // and their scales
constexpr int kMostSmem = 222 * 1024;       // of a block alone on its SM; its static part takes less than 2 KB

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

// Asynchronous copies to shared memory; nothing is read and zeros are written
// unless `in`.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// ---- decoded weights in bf16, times 2^-kWideShift: 2^-22 .. 0.66 ------------------
// An e2m1 number as fp16 has its sign, five bits of exponent and one of mantissa; the
// same bits three places further down are its bf16 form times 2^-112 (15 and 127 are the
// exponents' biases).
constexpr int kWideShift = 12;
__device__ __forceinline__ uint32_t low_bf16x2(uint32_t h) { return (h >> 3 & 0x0FFF0FFFu) | (h & 0x80008000u); }

// The two scales of an e4m3 pair as f16x2, each twice as bf16 and times 2^(112 - kWideShift).
__device__ __forceinline__ void wide_scales(uint32_t h, uint32_t (&s)[2]) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
  const float up = __int_as_float((112 - kWideShift + 127) << 23);
  const __nv_bfloat162 a = __float2bfloat162_rn(f.x * up), b = __float2bfloat162_rn(f.y * up);
  s[0] = *reinterpret_cast<const uint32_t *>(&a);
  s[1] = *reinterpret_cast<const uint32_t *>(&b);
}

template <bool BF16>
__device__ __forceinline__ void mma_m16n8k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight elements of a row of x that lie anywhere.
template <typename T>
__device__ __forceinline__ uint4 gather_x8(const T *p) {
  uint32_t w[4] = {};
  const uint16_t *u = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j / 2] |= static_cast<uint32_t>(__ldg(u + j)) << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Largest magnitudes of the even and the odd ones of eight bf16 numbers and of those
// behind `two`; NaN is left out.
__device__ __forceinline__ __nv_bfloat162 largest_x8(const uint4 &v, __nv_bfloat162 two) {
  const auto magnitudes = [](uint32_t w) {
    w &= 0x7FFF7FFFu;
    return *reinterpret_cast<const __nv_bfloat162 *>(&w);
  };
  return __hmax2(__hmax2(__hmax2(magnitudes(v.x), magnitudes(v.y)), __hmax2(magnitudes(v.z), magnitudes(v.w))), two);
}
// The larger one, as the bits of an f32.
__device__ __forceinline__ uint32_t upper_half(__nv_bfloat162 two) {
  const uint32_t w = *reinterpret_cast<const uint32_t *>(&two);
  return max(w << 16, w & 0xFFFF0000u);
}

// Smallest magnitude other than 0 of eight bf16 numbers and of those behind `low`,
// whose halves are magnitudes' bits less 1: 0 becomes 2^16 - 1 there, the largest.
constexpr uint32_t kNoneLow = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t smallest_x8(const uint4 &v, uint32_t low) {
  const auto with = [&](uint32_t w) { low = __viaddmin_u16x2(w & 0x7FFF7FFFu, 0xFFFFFFFFu, low); };
  with(v.x), with(v.y), with(v.z), with(v.w);
  return low;
}
__device__ __forceinline__ uint32_t lower_half(uint32_t low) { return min(low & 0xFFFFu, low >> 16); }

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// Exponent of the power of two that a row with this largest magnitude (as bits
// of a non-negative f32) is multiplied by.
__device__ __forceinline__ int row_shift(uint32_t max_bits) {
  const int e = static_cast<int>(max_bits >> 23);  // biased; 0 for subnormals and zero
  if (max_bits == 0) return 0;
  return min(14 - (min(e, 254) - 127), 126);
}

// True when a row so multiplied has numbers of which fp16 loses bits: below 2^-17, its
// last place being 2^-24 and bf16's significand eight bits long.
__device__ __forceinline__ bool loses_bits(uint32_t max_bits, uint32_t low) {
  const int smallest = max(static_cast<int>(low + 1) >> 7, 1);  // its exponent, biased; subnormals share that of the smallest normal one
  return low != 0xFFFFu && smallest - 127 + row_shift(max_bits) < -17;
}

// How many of eight fp16 numbers are at least 4, 2^-12 of the largest that a row may hold.
__device__ __forceinline__ int large_x8(const uint4 &h) {
  const auto signs = [](uint32_t w) { return ((w & 0x7FFF7FFFu) + 0x3C003C00u) & 0x80008000u; };  // 4 is 0x4400
  return __popc(signs(h.x) | signs(h.y) >> 1 | signs(h.z) >> 2 | signs(h.w) >> 3);
}

// The power of two of a row whose block takes bf16: it puts the largest magnitude at
// 2^60, so that sums of 2^15 products stay far from overflow and products with the
// smallest weight keep all their bits down to 2^-160 of the largest.
__device__ __forceinline__ int wide_row_shift(uint32_t max_bits) {
  const int e = static_cast<int>(max_bits >> 23);
  if (max_bits == 0) return 0;
  return min(60 - (min(e, 254) - 127), 126);
}

template <int NT, int RU, int WR, int WARPS>
struct Shape {
  static constexpr int tokens = 8 * NT;
  static constexpr int rows = 16 * RU * WR;       // of the weight, in a block
  static constexpr int k_warps = WARPS / WR;
  static constexpr int depth = 2;                 // steps in flight, for a warp
  static constexpr int stage = RU * kUnitStage;
  static constexpr int ring_bytes = WARPS * depth * stage;
  static constexpr int row_bytes(int steps) { return steps * kStep * 2 + 64; }  // of x, padded against bank conflicts
  static constexpr int sum_row = rows + 4;        // likewise
  static constexpr int sum_bytes = k_warps * sum_row * tokens * 4;
};

template <typename T, int NT, int RU, int WR, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, WARPS == 8 ? 3 : 1)
    weight_only_kernel(const Args p) {
  using S = Shape<NT, RU, WR, WARPS>;
  static_assert(NT == 1 || S::tokens <= 2 * WARPS, "a warp prepares at most two rows");
  constexpr bool kScaled = std::is_same<T, __nv_bfloat16>::value;  // rows of x carry a power of two
  constexpr int kThreads = 32 * WARPS;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *xs = smem + S::ring_bytes;
  __shared__ uint32_t row_max[S::tokens];
  __shared__ float bias[S::rows];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int split = gridDim.x;  // cluster: blocks along K
  const int part = blockIdx.x;
  const int m0 = blockIdx.z * S::tokens;
  const int tokens = min(S::tokens, p.M - m0);
  const int first_unit = blockIdx.y * WR * RU;  // of 16 rows; eight units in 128 rows
  const int k_warp = warp / WR;
  const int k_begin = part * p.steps * kStep;
  const int steps = max(0, min(p.steps, (p.K - k_begin + kStep - 1) / kStep));
  const int own_steps = max(0, (steps - k_warp + S::k_warps - 1) / S::k_warps);
  // weight row of row r of the block's output: a quarter's rows of all its units
  const auto feature = [&](int r) {
    constexpr int quarter_rows = 4 * RU * WR;
    const int unit = r % quarter_rows / 4;
    return static_cast<int64_t>((first_unit + unit) / 8) * 128 + r / quarter_rows * 32 + 4 * ((first_unit + unit) % 8) +
           r % 4;
  };

  grid_dependency_wait();

  // ---- copies: lane (g, t) brings 16 bytes of rows g and g + 8 and one word of scales ----
  const uint32_t half_k = p.K / 2;
  const uint32_t ring = smem_u32(smem) + warp * S::depth * S::stage;
  const int unit0 = first_unit + warp % WR * RU;
  // rows g and g + 8 of unit u: see the header; 32-bit offsets inside the scale tile's 128 rows
  const uint8_t *codes = p.codes + static_cast<int64_t>(unit0 / 8) * 128 * half_k;
  const uint8_t *sf = p.sf + static_cast<int64_t>(unit0 / 8) * (p.K / 64) * 512;
  const uint32_t code_at = ((g % 4) * 32 + 4 * (unit0 % 8) + g / 4) * half_k + k_begin / 2 + 16 * t;
  // scales: 64 consecutive bytes for the 16 rows and four groups, in the order of (row / 4, row % 4)
  const uint32_t sf_at = (k_begin / 64 + lane / 16) * 512 + 4 * (unit0 % 8) * 16 + lane % 16 * 4;
  const int k_left = p.K - k_begin;
  const auto copy = [&](int i) {  // the i-th of this warp's steps
    if (i < own_steps) {
      const int step = k_warp + i * S::k_warps;
      const uint32_t stage = ring + i % S::depth * S::stage;
      const bool in = step * kStep + 32 * t < k_left;  // K may end on half a step
      const bool sf_in = step * kStep + lane / 16 * 64 < k_left;
#pragma unroll
      for (int u = 0; u < RU; ++u) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
          copy16(stage + u * kUnitStage + r * 512 + lane * 16,
                 codes + (in ? code_at + (4 * u + 2 * r) * half_k + step * (kStep / 2) : 0u), in);
        copy4(stage + u * kUnitStage + kUnitBytes + lane * 4, sf + (sf_in ? sf_at + u * 64 + step * 1024 : 0u), sf_in);
      }
    }
    copies_commit();
  };

  // ---- x to fp16 in shared memory; its first loads go out before the copies, which would delay them ----
  const int row_bytes = S::row_bytes(p.steps);
  const T *x = static_cast<const T *>(p.x) + m0 * p.ldx;
  const int chunks = p.steps * (kStep / 8);  // of eight elements, in a row; a multiple of 16
  // Up to eight rows: all threads share them.  More: a warp has one or two rows to
  // itself and needs no other's maximum (32 rows, N = 12288, K = 4096: 24.7 us, before that 27.0).
  constexpr bool kOwnRows = NT > 1;
  constexpr int kStride = kOwnRows ? 32 : kThreads;
  const int first = kOwnRows ? lane : tid;
  const int items = (kOwnRows ? (tokens - warp + WARPS - 1) / WARPS : tokens) * chunks;
  const auto nth_row = [&](int i) { return static_cast<int>(__umulhi(i, p.chunk_inverse)); };  // i / chunks
  const auto row_of = [&](int i) { return kOwnRows ? warp + WARPS * nth_row(i) : nth_row(i); };
  const auto chunk_of = [&](int i) { return i - nth_row(i) * chunks; };
  // chunk 4 * t + i of a step is read by lane t in its i-th pair of products
  const auto place = [&](int i) {
    const int c = chunk_of(i);
    return reinterpret_cast<uint4 *>(xs + row_of(i) * row_bytes + (c / 16) * 256 + (c % 4) * 64 + (c % 16) / 4 * 16);
  };
  const auto from = [&](int i) { return x + row_of(i) * p.ldx + k_begin + 8 * chunk_of(i); };
  const auto inside = [&](int i) { return 8 * chunk_of(i) < k_left; };  // K is a multiple of eight
  // of a warp's own rows; the smallest without own rows of all of them
  __nv_bfloat162 best[2] = {__nv_bfloat162(0.0f, 0.0f), __nv_bfloat162(0.0f, 0.0f)};
  uint32_t low[2] = {kNoneLow, kNoneLow};
  const auto note = [&](int i, const uint4 &v) {
    const int r = kOwnRows ? nth_row(i) : 0;
    if (r == 0) low[0] = smallest_x8(v, low[0]);
    else low[1] = smallest_x8(v, low[1]);
    if (kOwnRows) {
      if (r == 0) best[0] = largest_x8(v, best[0]);
      else best[1] = largest_x8(v, best[1]);
    } else {  // 16 lanes with one row's chunks
      const uint32_t top = __reduce_max_sync(0xFFFFu << (lane & 16), upper_half(largest_x8(v, best[0])));
      if (lane % 16 == 0 && top) atomicMax(&row_max[row_of(i)], top);
    }
  };
  constexpr int kFlight = NT == 1 ? 8 : 12;  // chunks of a thread in flight
  constexpr int kFlightItems = kFlight * kStride;
  uint4 v[kFlight];
  const auto load = [&](int base) {
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
      const int i = base + j * kStride + first;
      if (i >= items) break;
      v[j] = make_uint4(0, 0, 0, 0);
      if (inside(i)) v[j] = __ldg(reinterpret_cast<const uint4 *>(from(i)));
    }
  };
  if (p.vector_x) load(0);
#pragma unroll
  for (int i = 0; i < S::depth; ++i) copy(i);
  const float alpha = __ldg(p.alpha);
  for (int r = tid; r < S::rows; r += kThreads) bias[r] = p.bias != nullptr ? __bfloat162float(p.bias[feature(r)]) : 0.0f;
  if (kScaled && !kOwnRows) {
    if (tid < S::tokens) row_max[tid] = 0;
    __syncthreads();
  }
  int base = 0;  // of the last flight, which stays in registers until the rows' maxima are known
  if (p.vector_x) {
#pragma unroll 1
    for (;; base += kFlightItems, load(base)) {
      if (kScaled) {
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
          const int i = base + j * kStride + first;
          if (i >= items) break;
          note(i, v[j]);
        }
      }
      if (base + kFlightItems >= items) break;
#pragma unroll
      for (int j = 0; j < kFlight; ++j) *place(base + j * kStride + first) = v[j];
    }
  } else {
    base = items;
#pragma unroll 1
    for (int i = first; i < items; i += kStride) {
      const uint4 c = inside(i) ? gather_x8(from(i)) : make_uint4(0, 0, 0, 0);
      if (kScaled) note(i, c);
      *place(i) = c;
    }
  }
  bool lossy = false;  // this thread has numbers that lose bits in fp16
  const auto scaled = [&](uint4 c, float factor) {
    uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __half2 h =
          __floats2half2_rn(__uint_as_float(w[e] << 16) * factor, __uint_as_float(w[e] & 0xFFFF0000u) * factor);
      w[e] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  if (kScaled) {
    if (kOwnRows) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, upper_half(best[r]));
        lossy |= loses_bits(top, lower_half(low[r]));
        if (lane == 0 && warp + r * WARPS < S::tokens) row_max[warp + r * WARPS] = top;
      }
      __syncwarp();
    } else {  // its smallest number beside the largest of all rows: never too few are found
      __syncthreads();
      lossy = loses_bits(__reduce_max_sync(0xFFFFFFFFu, lane < tokens ? row_max[lane] : 0u), lower_half(low[0]));
    }
#pragma unroll 4
    for (int i = first; i < base; i += kStride)
      *place(i) = scaled(*place(i), power_of_two(row_shift(row_max[row_of(i)])));
  }
#pragma unroll
  for (int j = 0; j < kFlight; ++j) {
    const int i = base + j * kStride + first;
    if (i >= items) break;
    *place(i) = kScaled ? scaled(v[j], power_of_two(row_shift(row_max[row_of(i)]))) : v[j];
  }

  // ---- rows whose numbers lie too far apart for fp16: all of x again, in bf16 ----
  bool wide = __syncthreads_or(lossy) && kScaled;
  if (wide) {  // unless enough of every row are large: a few lanes count them, one warp a row
    bool few = false;
    for (int r = warp; r < tokens; r += WARPS) {
      int large = 0;
      for (int at = 16 * lane; at < 256 * p.steps; at += 512) {
        const uint4 h = *reinterpret_cast<const uint4 *>(xs + r * row_bytes + at);
        large += large_x8(h);
      }
      few |= row_max[r] != 0 && 4 * __reduce_add_sync(0xFFFFFFFFu, large) < min(p.steps * kStep, k_left);
    }
    wide = __syncthreads_or(few);
  }
  if (wide) {
#pragma unroll 1
    for (int i = first; i < items; i += kStride) {
      uint4 c = make_uint4(0, 0, 0, 0);
      if (inside(i)) c = p.vector_x ? __ldg(reinterpret_cast<const uint4 *>(from(i))) : gather_x8(from(i));
      const float factor = power_of_two(wide_row_shift(row_max[row_of(i)]));
      uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = pack_bf16x2(__uint_as_float(w[e] << 16) * factor, __uint_as_float(w[e] & 0xFFFF0000u) * factor);
      *place(i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncthreads();
  }

  // ---- products ----
  float acc[RU][NT][4] = {};
  const uint8_t *own_ring = smem + warp * S::depth * S::stage;
  const auto products = [&](auto as_bf16) {
    constexpr bool kWide = decltype(as_bf16)::value;
#pragma unroll 1
    for (int i = 0; i < own_steps; ++i) {
      copies_wait<S::depth - 1>();
      __syncwarp();
      const uint8_t *stage = own_ring + i % S::depth * S::stage;
      const uint8_t *x_step = xs + g * row_bytes + (k_warp + i * S::k_warps) * 256 + t * 16;
      uint4 w[RU][2];
      uint32_t scale[RU][2][2];  // unit, row, group: the scale in both halves
#pragma unroll
      for (int u = 0; u < RU; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          w[u][r] = *reinterpret_cast<const uint4 *>(stage + u * kUnitStage + r * 512 + lane * 16);
          // lane's groups 2t and 2t + 1 of row g + 8r, which is row (g / 4 + 2r) of quarter g % 4
          const uint16_t s = *reinterpret_cast<const uint16_t *>(stage + u * kUnitStage + kUnitBytes + t / 2 * 64 +
                                                                 (g / 4 + 2 * r) * 16 + g % 4 * 4 + t % 2 * 2);
          const uint32_t h = decode_e4m3x2(s);
          if (kWide) {
            wide_scales(h, scale[u][r]);
          } else {
            scale[u][r][0] = __byte_perm(h, 0, 0x1010);
            scale[u][r][1] = __byte_perm(h, 0, 0x3232);
          }
        }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint4 f[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          f[n] = make_uint4(0, 0, 0, 0);
          if (8 * n + g < tokens) f[n] = *reinterpret_cast<const uint4 *>(x_step + 8 * n * row_bytes + q * 64);
        }
#pragma unroll
        for (int u = 0; u < RU; ++u) {
          uint32_t a[2][4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            decode_e2m1x8(reinterpret_cast<const uint32_t *>(&w[u][r])[q], a[r]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              a[r][j] = kWide ? mul_bf16x2(low_bf16x2(a[r][j]), scale[u][r][q / 2]) : mul_f16x2(a[r][j], scale[u][r][q / 2]);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_m16n8k16<kWide>(acc[u][n], a[0][0], a[1][0], a[0][1], a[1][1], f[n].x, f[n].y);
            mma_m16n8k16<kWide>(acc[u][n], a[0][2], a[1][2], a[0][3], a[1][3], f[n].z, f[n].w);
          }
        }
      }
      __syncwarp();  // the stage is read by all lanes
      copy(i + S::depth);
    }
  };
  if (wide) products(std::true_type());
  else products(std::false_type());
  copies_wait<0>();

  // ---- sums over the warps, then over the blocks of the cluster ----
  __syncthreads();  // ring and x are read
  float *sums = reinterpret_cast<float *>(smem);  // [k warp][token][row of the products]
#pragma unroll
  for (int u = 0; u < RU; ++u)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sums[(k_warp * S::tokens + 8 * n + 2 * t + j % 2) * S::sum_row + ((warp % WR) * RU + u) * 16 + g + 8 * (j / 2)] =
            acc[u][n][j];
  __syncthreads();
  // four neighbours of the products' rows are the four quarters' rows of one place in them
  const auto store = [&](int m, int l, const float4 &sum) {
    const float v[4] = {sum.x, sum.y, sum.z, sum.w};
    const int64_t at = (m0 + m) * p.ldo + feature(l);
#pragma unroll
    for (int j = 0; j < 4; ++j) p.out[at + 32 * j] = __float2bfloat16_rn(v[j] + bias[j * (S::rows / 4) + l]);
  };
  const int fours = tokens * (S::rows / 4);
#pragma unroll 2
  for (int i = tid; i < fours; i += kThreads) {
    const int m = i / (S::rows / 4), l = i % (S::rows / 4);
    float4 *at = reinterpret_cast<float4 *>(sums + m * S::sum_row + 4 * l);
    float4 sum = *at;
#pragma unroll
    for (int w = 1; w < S::k_warps; ++w) {
      const float4 other = at[w * S::tokens * S::sum_row / 4];
      sum.x += other.x, sum.y += other.y, sum.z += other.z, sum.w += other.w;
    }
    const float back =
        !kScaled ? 1.0f : power_of_two(wide ? kWideShift - wide_row_shift(row_max[m]) : -row_shift(row_max[m]));
    sum = make_float4(sum.x * alpha * back, sum.y * alpha * back, sum.z * alpha * back, sum.w * alpha * back);
    if (split == 1)
      store(m, l, sum);
    else
      *at = sum;
  }
  if (split == 1) return;
  cluster_sync();
#pragma unroll 1
  for (int i = part * kThreads + tid; i < fours; i += kThreads * split) {
    const int m = i / (S::rows / 4), l = i % (S::rows / 4);
    const uint32_t at = smem_u32(sums + m * S::sum_row + 4 * l);
    float4 other[8] = {};  // all in flight before the first is added
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < split)
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(other[c].x), "=f"(other[c].y), "=f"(other[c].z), "=f"(other[c].w)
                     : "r"(map_to_rank(at, c)));
    float4 sum = other[0];
#pragma unroll
    for (int c = 1; c < 8; ++c)
      sum.x += other[c].x, sum.y += other[c].y, sum.z += other[c].z, sum.w += other[c].w;
    store(m, l, sum);
  }
  cluster_sync();  // the others have read this block's sums
}

template <typename T, int NT, int RU, int WR, int WARPS>
int launch(Args p, int split, cudaStream_t stream) {
  using S = Shape<NT, RU, WR, WARPS>;
  auto kernel = weight_only_kernel<T, NT, RU, WR, WARPS>;
  const int steps = (p.K + kStep - 1) / kStep;
  p.steps = (steps + split - 1) / split;
  p.chunk_inverse = static_cast<uint32_t>((1ull << 32) / (p.steps * 16)) + 1;
  const int used = S::ring_bytes + (p.M < S::tokens ? p.M : S::tokens) * S::row_bytes(p.steps);
  const int smem = used > S::sum_bytes ? used : S::sum_bytes;
  if (smem > kMostSmem) return set_error(VFB_EINVAL, "vfb_nvfp4_weight_only: K is too large");
  static std::atomic<uint64_t> smem_set[kMaxAttrDevices];
  int rc = ensure_smem_optin(reinterpret_cast<const void *>(kernel), kMostSmem, smem_set);
  if (rc != VFB_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(split, p.N / S::rows, (p.M + S::tokens - 1) / S::tokens);
  cfg.blockDim = dim3(32 * WARPS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 2 : 1;
  cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p);
  if (err != cudaSuccess) return set_error(VFB_ECUDA, "vfb_nvfp4_weight_only launch: %s", cudaGetErrorString(err));
  return VFB_OK;
}

// Blocks along K: as many as still run at once while every warp keeps two steps;
// more where x of a K range would not leave room for `resident` blocks on an SM.
// Powers of two only: three blocks of 16 warps in a cluster leave SMs unused (8
// rows, N = 12288, K = 4096: 144 blocks in threes 22.8 us, 96 in pairs 15.1).
template <typename T, int NT, int RU, int WR, int WARPS>
int launch_split(const Args &p, int sms, int resident, cudaStream_t stream) {
  using S = Shape<NT, RU, WR, WARPS>;
  const int steps = (p.K + kStep - 1) / kStep;
  const int tokens = p.M < S::tokens ? p.M : S::tokens;
  const int64_t blocks = static_cast<int64_t>(p.N / S::rows) * ((p.M + S::tokens - 1) / S::tokens);
  const int most = (kMostSmem + 2048) / resident - 2048 - S::ring_bytes;
  int split = 1;
  while (split < 8 && ((2 * blocks * split <= resident * sms && steps >= 4 * split * S::k_warps) ||
                       tokens * S::row_bytes((steps + split - 1) / split) > most))
    split *= 2;
  return launch<T, NT, RU, WR, WARPS>(p, split, stream);
}

// Rows of the weight in a block.  Every block prepares x for itself, so tall
// blocks share that work, the more the more rows x has; low blocks spread a low
// weight over the SMs, and three of them share an SM, so that a last round of
// few blocks costs less.  Measured (us, N x K):
//   8 rows of x, 64 / 128 rows a block: 1152 x 1024 4.3 / 5.2, 128 x 16384 7.9 / 10.1,
//   4096 x 4096 7.3 / 7.0, 12288 x 4096 14.6 / 12.8, 4096 x 16384 22.7 / 16.3;
//   one row 1152 x 1024 3.2 / 4.3, 128 x 16384 5.5 / 7.8, 1152 x 16384 8.0 / 8.7,
//   2048 x 16384 8.6 / 11.2, 4096 x 4096 6.3 / 6.1, 4096 x 16384 12.9 / 12.4 (two rows
//   12% more on either side);
//   128 / 256 rows, with tall blocks that fill the rounds on 148 SMs: 14336 x 5376
//   21.3 / 16.8, 16384 x 4096 15.8 / 14.2, 28672 x 5376 33.8 / 26.6, 36864 x 4096
//   29.1 / 22.8, and for one row of x 14.7 / 14.0, 12.2 / 12.0, 23.9 / 22.7, 19.8 / 19.5;
//   where they do not: 12288 x 4096 12.8 / 13.5, 40960 x 4096 31.7 / 39.0 (one row
//   of x 25.3 / 32.6).
//   32 rows of x, 128 / 256 rows a block (16 warps): 4096 x 4096 11.8 / 20.8,
//   12288 x 4096 38.9 / 27.1, 28672 x 5376 99 / 76, 40960 x 4096 94.8 / 77.8 (before
//   warps had rows of x to themselves, which took 10 % off all of these).
// 32 rows of x (sixteen at a time otherwise) do not fit for K > 16384, and where they
// only fit with K dealt out to eight blocks, these take more than one round unless
// the weight is low: 4096 x 16384, 20 rows 45.7 / 35.3, 17 rows (four blocks along K) 27.3 /
// 34.9; 4096 x 12288, 24 rows 22.0 / 27.7, 32 rows 41.4 / 29.4; 1024 x 16384, 32 rows
// 17.4 / 22.2.
template <typename T>
int run(const Args &p, int sms, cudaStream_t s) {
  const int64_t blocks = p.N % 256 ? 0 : (2 * p.N / 256 <= sms ? 2 : 1) * (p.N / 256);  // tall ones, with two along K
  const int64_t rounds = (blocks + sms - 1) / sms;
  if (p.M <= 8) {
    if (p.N <= 2048) return launch_split<T, 1, 2, 2, 8>(p, sms, 3, s);
    const bool tall = blocks > 0 && p.N >= 14336 && 10 * blocks >= 7 * rounds * sms;
    return tall ? launch_split<T, 1, 2, 8, 16>(p, sms, 1, s) : launch_split<T, 1, 2, 4, 8>(p, sms, 3, s);
  }
  const bool tall = blocks > 0 && p.N >= 8192;
  const int64_t x_block = static_cast<int64_t>(p.M < 32 ? p.M : 32) * p.K;
  const bool deep = p.K > 16384 || (x_block > 300000 && 8 * (p.N / 128) > sms);
  if (p.M <= 16 || deep)
    return tall ? launch_split<T, 2, 2, 8, 16>(p, sms, 1, s) : launch_split<T, 2, 2, 4, 16>(p, sms, 1, s);
  return tall ? launch_split<T, 4, 2, 8, 16>(p, sms, 1, s) : launch_split<T, 4, 2, 4, 16>(p, sms, 1, s);
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
  // Blocks write their part of out while others still read.
  const Extent written{out, 2 * N, {M, 1}, {2 * ldo, 0}};
  const Extent read[] = {{x, 2 * K, {M, 1}, {2 * ldx, 0}},
                         {w_codes, N * K / 2, {1, 1}, {}},
                         {w_sf, N * K / 16, {1, 1}, {}},
                         {alpha, 4, {1, 1}, {}},
                         {bias, 2 * N, {bias != nullptr, 1}, {}}};
  for (const Extent &t : read)
    if (may_overlap(written, t))
      return set_error(VFB_EINVAL, "vfb_nvfp4_weight_only: out may not overlap x, the weight, alpha or bias");
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
