// Causal attention over packed sequences with grouped heads.
#include <cuda_fp16.h>

#include "common.cuh"

namespace {

constexpr int kThreads = 128;

template <typename E>
__device__ __forceinline__ float val(E v);
template <>
__device__ __forceinline__ float val(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float val(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename E>
__device__ __forceinline__ E rounded(float v);
template <>
__device__ __forceinline__ __half rounded(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 rounded(float v) { return __float2bfloat16_rn(v); }

// A warp per (query, head): 32 keys at a time, a lane each for the scores,
// then the lanes share out the value columns. The running maximum and sum of
// the softmax make one pass over the keys.
template <typename E, int kDim, int kVDim>
__global__ void __launch_bounds__(kThreads) attention_simple_kernel(sl_attention_args a,
                                                                    int32_t* status) {
  __shared__ float q_sm[kThreads / 32][kDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  sl::pdl_wait();
  sl::pdl_trigger();
  if (blockIdx.x == 0 && threadIdx.x == 0) *status = SL_OK;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + warp;
  if (item >= a.Tq * a.heads) return;
  const int64_t row = item / a.heads;
  const int h = static_cast<int>(item % a.heads), hk = h / (a.heads / a.kv_heads);
  // the sequence: the last one that begins at or before the row
  int lo = 0, hi = a.B;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu_q[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  if (lo >= a.B || row < a.cu_q[0]) return;
  const int64_t q0 = a.cu_q[lo], q1 = a.cu_q[lo + 1];
  const int64_t k0 = max(a.cu_k[lo], 0), k1 = min(static_cast<int64_t>(a.cu_k[lo + 1]), a.Tk);
  const int64_t seen = min(max(k1 - k0, static_cast<int64_t>(0)), row - q0 + 1 + (k1 - k0) - (q1 - q0));
  const E* q = static_cast<const E*>(a.q) + row * a.q_token + h * a.q_head;
  for (int d = lane; d < kDim; d += 32) q_sm[warp][d] = val(q[d]);
  __syncwarp();
  const int own = kDim - a.shared_dim;
  float m = -INFINITY, l = 0.f, o[kVDim / 32] = {};
  for (int64_t j0 = 0; j0 < seen; j0 += 32) {
    const int64_t j = j0 + lane;
    float s = -INFINITY;
    if (j < seen) {
      const E* k = static_cast<const E*>(a.k) + (k0 + j) * a.k_token + hk * a.k_head;
      s = 0.f;
      for (int d = 0; d < own; ++d) s = fmaf(q_sm[warp][d], val(k[d]), s);
      if (a.shared_dim) {
        const E* ks = static_cast<const E*>(a.k_shared) + (k0 + j) * a.k_shared_token;
        for (int d = own; d < kDim; ++d) s = fmaf(q_sm[warp][d], val(ks[d - own]), s);
      }
      s *= a.scale;
    }
    float top = s;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float m1 = fmaxf(m, top);
    // (a row whose scores are all -inf so far keeps zero weights)
    const float base = m1 == -INFINITY ? 0.f : m1;
    const float corr = __expf(m - base), p = __expf(s - base);
    float sum = p;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * corr + sum;
    m = m1;
#pragma unroll
    for (int c = 0; c < kVDim / 32; ++c) o[c] *= corr;
    const int n = static_cast<int>(min(static_cast<int64_t>(32), seen - j0));
    for (int u = 0; u < n; ++u) {
      const float pu = __shfl_sync(0xffffffffu, p, u);
      const E* v = static_cast<const E*>(a.v) + (k0 + j0 + u) * a.v_token + hk * a.v_head;
#pragma unroll
      for (int c = 0; c < kVDim / 32; ++c) o[c] = fmaf(pu, val(v[lane + 32 * c]), o[c]);
    }
  }
  E* out = static_cast<E*>(a.out) + row * a.out_token + h * a.out_head;
#pragma unroll
  for (int c = 0; c < kVDim / 32; ++c)
    out[lane + 32 * c] = rounded<E>(seen > 0 ? o[c] / l : 0.f);
}

template <typename E>
int run(const sl_attention_args& a, int32_t* status, cudaStream_t st) {
  const int64_t ctas = (a.Tq * a.heads + kThreads / 32 - 1) / (kThreads / 32);
  if (ctas > 0x7fffffff) return SL_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(ctas));
  cudaError_t e;
  if (a.dim == 64)
    e = sl::launch(attention_simple_kernel<E, 64, 64>, grid, dim3(kThreads), 0, st, a, status);
  else if (a.dim == 128)
    e = sl::launch(attention_simple_kernel<E, 128, 128>, grid, dim3(kThreads), 0, st, a, status);
  else
    e = sl::launch(attention_simple_kernel<E, 192, 128>, grid, dim3(kThreads), 0, st, a, status);
  SL_CUDA_TRY(e);
  return SL_OK;
}

}  // namespace

extern "C" size_t sl_prompt_attention_workspace_bytes(int B, int64_t Tq, int64_t Tk, int heads,
                                                      int kv_heads, int v_dim) {
  if (B <= 0 || Tq < 0 || Tk < 0 || heads <= 0 || kv_heads <= 0 || v_dim <= 0) return 0;
  return 256;
}

extern "C" int sl_prompt_attention(const sl_attention_args* args, void* workspace,
                                   size_t workspace_bytes, sl_stream_t stream) {
  if (!args) return SL_ERR_INVALID;
  const sl_attention_args& a = *args;
  if (a.B <= 0 || a.Tq < 0 || a.Tk < 0 || a.heads <= 0 || a.kv_heads <= 0 ||
      a.heads % a.kv_heads || !(a.scale > 0.f) || !(a.scale < INFINITY) || a.shared_dim < 0)
    return SL_ERR_INVALID;
  const bool dims = (a.dim == 64 && a.v_dim == 64) || (a.dim == 128 && a.v_dim == 128) ||
                    (a.dim == 192 && a.v_dim == 128);
  if (!dims || (a.shared_dim != 0 && !(a.shared_dim == 64 && a.dim == 192)) ||
      (a.dtype != SL_DTYPE_BF16 && a.dtype != SL_DTYPE_FP16) || a.heads / a.kv_heads > 128 ||
      a.Tq > 0x7fffffff || a.Tk > 0x7fffffff)
    return SL_ERR_UNSUPPORTED;
  if (a.Tq == 0) return SL_OK;
  const bool keys = a.Tk > 0;
  if (!a.q || !a.out || !a.cu_q || !a.cu_k || !workspace || (keys && (!a.k || !a.v)) ||
      (keys && a.shared_dim && !a.k_shared))
    return SL_ERR_INVALID;
  if (workspace_bytes < sl_prompt_attention_workspace_bytes(a.B, a.Tq, a.Tk, a.heads, a.kv_heads,
                                                            a.v_dim))
    return SL_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
       reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.k_shared) |
       reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return SL_ERR_INVALID;
  if ((a.q_token | a.q_head | a.k_token | a.k_head | a.v_token | a.v_head | a.k_shared_token |
       a.out_token | a.out_head) & 7)
    return SL_ERR_INVALID;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int32_t* status = static_cast<int32_t*>(workspace);
  return a.dtype == SL_DTYPE_BF16 ? run<__nv_bfloat16>(a, status, st) : run<__half>(a, status, st);
}
