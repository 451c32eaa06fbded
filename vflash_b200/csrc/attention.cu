// Attention over packed sequences (vfb_attention): one warp per query row and
// head, scores of 32 keys at a time (one key per lane), running maximum and
// sum in fp32, only the keys the row may see.
#include "common.cuh"

namespace vfb {
namespace {

struct Params {
  vfb_attention_args a;
  float scale_log2;
};

template <typename T>
__device__ __forceinline__ float widen(T x);
template <>
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ void narrow(float f, __nv_bfloat16 *p) { *p = __float2bfloat16_rn(f); }
__device__ __forceinline__ void narrow(float f, __half *p) { *p = __float2half_rn(f); }

// Offsets are clamped to the buffers, so no input makes the kernel leave them.
__device__ __forceinline__ int64_t clamp64(int64_t x, int64_t lo, int64_t hi) {
  return x < lo ? lo : (x > hi ? hi : x);
}

template <typename T>
__global__ void __launch_bounds__(128) attention_rows_kernel(Params p) {
  const vfb_attention_args &a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= a.total_q * a.heads) return;
  const int64_t row = item / a.heads;
  const int head = static_cast<int>(item - row * a.heads);
  const int kv = head / (a.heads / a.kv_heads);
  int64_t q0 = 0, q1 = a.total_q, k0 = 0, nk = a.total_k;
  bool behind = false;
  if (a.cu_seqlens_q != nullptr) {
    int lo = 0, hi = a.batch;  // the last sequence that starts at or before the row
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.cu_seqlens_q[mid] <= row) lo = mid; else hi = mid;
    }
    while (lo + 1 < a.batch && a.cu_seqlens_q[lo + 1] <= row) ++lo;
    q0 = clamp64(a.cu_seqlens_q[lo], 0, a.total_q);
    q1 = clamp64(a.cu_seqlens_q[lo + 1], q0, a.total_q);
    behind = row >= q1;
    const int32_t *cu_k = a.cu_seqlens_k != nullptr ? a.cu_seqlens_k : a.cu_seqlens_q;
    k0 = clamp64(cu_k[lo], 0, a.total_k);
    nk = clamp64(cu_k[lo + 1], k0, a.total_k) - k0;
    if (a.lengths_k != nullptr) nk = clamp64(a.lengths_k[lo], 0, nk);
  } else if (a.lengths_k != nullptr) {
    nk = clamp64(a.lengths_k[0], 0, nk);
  }
  int64_t limit = nk;
  if (a.causal) limit = clamp64(row - q0 + 1 + nk - (q1 - q0), 0, nk);
  if (behind) limit = 0;

  const T *q = static_cast<const T *>(a.q) + row * a.q_token_stride + head * a.q_head_stride;
  const T *k = static_cast<const T *>(a.k) + k0 * a.k_token_stride + kv * a.k_head_stride;
  const T *v = static_cast<const T *>(a.v) + k0 * a.v_token_stride + kv * a.v_head_stride;
  float m = -INFINITY, l = 0.0f, acc[4] = {};
  for (int64_t j0 = 0; j0 < limit; j0 += 32) {
    const int64_t j = j0 + lane;
    float s = -INFINITY;
    if (j < limit) {
      s = 0.0f;
      for (int d = 0; d < a.dim; ++d) s = fmaf(widen(q[d]), widen(k[j * a.k_token_stride + d]), s);
    }
    float top = s;
    bool nan = s != s;
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    if (__any_sync(~0u, nan)) top = NAN;
    const float m_new = top != top || m != m ? NAN : fmaxf(m, top);
    const float base = m_new == -INFINITY ? 0.0f : m_new;
    const float e = j < limit ? exp2f((s - base) * p.scale_log2) : 0.0f;
    const float alpha = m == -INFINITY ? 0.0f : exp2f((m - base) * p.scale_log2);
    l = l * alpha + e;
    for (int i = 0; i < 4; ++i) acc[i] *= alpha;
    const int n = static_cast<int>(limit - j0 < 32 ? limit - j0 : 32);
    for (int t = 0; t < n; ++t) {
      const float w = __shfl_sync(~0u, e, t);
      for (int i = 0; i < 4; ++i) {
        const int d = lane + 32 * i;
        if (d < a.dim) acc[i] = fmaf(w, widen(v[(j0 + t) * a.v_token_stride + d]), acc[i]);
      }
    }
    m = m_new;
  }
  for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
  if (!behind || a.fill_tail) {
    T *out = static_cast<T *>(a.out) + row * a.out_token_stride + head * a.out_head_stride;
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 32 * i;
      if (d < a.dim) narrow(limit > 0 ? acc[i] / l : 0.0f, out + d);
    }
  }
  if (a.lse != nullptr && lane == 0)
    a.lse[head * a.total_q + row] =
        limit > 0 ? (m * p.scale_log2 + log2f(l)) * 0.693147180559945309f : -INFINITY;
}

int check_args(const vfb_attention_args *a) {
  if (a == nullptr) return set_error(VFB_EINVAL, "vfb_attention: args is NULL");
  if (a->total_q < 0 || a->total_k < 0 || a->total_q >= (1ll << 31) || a->total_k >= (1ll << 31))
    return set_error(VFB_EINVAL, "vfb_attention: rows must be >= 0 and below 2^31");
  if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads || a->heads > 65535)
    return set_error(VFB_EINVAL, "vfb_attention: heads must be a multiple of kv_heads, 1 to 65535");
  if (a->dim < 8 || a->dim > 128 || a->dim % 8)
    return set_error(VFB_EINVAL, "vfb_attention: dim must be a multiple of 8 from 8 to 128");
  if (a->dtype != 0 && a->dtype != 1) return set_error(VFB_EINVAL, "vfb_attention: dtype must be 0 (bf16) or 1 (fp16)");
  if (a->batch < 1 || (a->cu_seqlens_q == nullptr && (a->batch != 1 || a->cu_seqlens_k != nullptr)))
    return set_error(VFB_EINVAL, "vfb_attention: batch must be >= 1, and 1 without cu_seqlens_q");
  if (a->cu_seqlens_q != nullptr && a->cu_seqlens_k == nullptr && a->total_k != a->total_q)
    return set_error(VFB_EINVAL, "vfb_attention: keys of another length need cu_seqlens_k");
  if (!(a->scale > 0.0f) || a->scale > 3.0e38f)
    return set_error(VFB_EINVAL, "vfb_attention: scale must be positive and finite");
  const int64_t strides[] = {a->q_token_stride, a->q_head_stride, a->k_token_stride,   a->k_head_stride,
                             a->v_token_stride, a->v_head_stride, a->out_token_stride, a->out_head_stride};
  for (int64_t s : strides)
    if (s < a->dim || s % 8 || s >= (1ll << 38))
      return set_error(VFB_EINVAL, "vfb_attention: strides must be multiples of 8, at least dim");
  return VFB_OK;
}

}  // namespace
}  // namespace vfb

extern "C" int64_t vfb_attention_workspace_bytes(const vfb_attention_args *args) {
  if (vfb::check_args(args) != VFB_OK) return -1;
  return 0;
}

extern "C" int vfb_attention(const vfb_attention_args *args, void *stream) {
  using namespace vfb;
  int rc = check_args(args);
  if (rc != VFB_OK) return rc;
  const vfb_attention_args &a = *args;
  if (a.total_q == 0) return VFB_OK;
  if (!a.q || !a.out || (a.total_k > 0 && (!a.k || !a.v)))
    return set_error(VFB_EINVAL, "vfb_attention: NULL pointer");
  if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.out))
    return set_error(VFB_EINVAL, "vfb_attention: q, k, v and out must be 16-byte aligned");
  rc = check_device(nullptr);
  if (rc != VFB_OK) return rc;
  Params p{a, a.scale * 1.44269504088896341f};
  const int64_t blocks = (a.total_q * a.heads + 3) / 4;
  if (blocks > 0x7fffffff) return set_error(VFB_EINVAL, "vfb_attention: too many rows");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.dtype == 0) attention_rows_kernel<__nv_bfloat16><<<(unsigned)blocks, 128, 0, s>>>(p);
  else attention_rows_kernel<__half><<<(unsigned)blocks, 128, 0, s>>>(p);
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return set_error(VFB_ECUDA, "vfb_attention launch: %s", cudaGetErrorString(err));
  return VFB_OK;
}
