// logprobs.cu -- log probabilities of given tokens, the entropy and the top alternatives of rows of logits,
// with the sampler's rules for the probabilities (gsd_lq_cpu_runtime.py:422-434; the reference returns only
// the pick).
//
// With z the cleaned logits over the temperature, c the index of the row's first maximum and u_i = z_i - z_c:
//   S = sum_{i != c} e^{u_i},  T = sum_{i != c} e^{u_i} u_i   (every term of T is <= 0)
//   log p_i = u_i - log1p(S),  entropy = log1p(S) - T / (1 + S)
// Leaving the maximum's own 1 out of S keeps peaked rows exact: where S is far below 1, log(1 + S) in fp32
// would lose S to the rounding of 1 + S.
#include <cfloat>
#include <cmath>

#include "common.cuh"

namespace gsdlq {

constexpr int LP_THREADS = 256;

__device__ __forceinline__ float lp_clean(float x, float temp) {
  // -0 becomes 0, which ties with it; a quotient past fp32 stays finite, so that differences are defined
  return fminf(fmaxf(__fdiv_rn(sanitize_logit(x), temp), -FLT_MAX), FLT_MAX) + 0.0f;
}
__device__ __forceinline__ unsigned long long lp_key(float z, int i) {
  return ((unsigned long long)ordered_key(z) << 32) | (0xffffffffu - (uint32_t)i);
}

__device__ unsigned long long lp_block_max(unsigned long long* red, unsigned long long k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = k;
  __syncthreads();
  k = red[threadIdx.x & (LP_THREADS / 32 - 1)];
#pragma unroll
  for (int o = LP_THREADS / 64; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  return k;
}
__device__ float lp_block_sum(float* red, float v) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & (LP_THREADS / 32 - 1)];
#pragma unroll
  for (int o = LP_THREADS / 64; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__global__ void __launch_bounds__(LP_THREADS) logprobs_rows_kernel(const __grid_constant__ gsdlq_logprobs_job_t J) {
  __shared__ unsigned long long kred[LP_THREADS / 32];
  __shared__ float fred[LP_THREADS / 32];
  const int r = blockIdx.x, tid = threadIdx.x;
  const float* x = J.logits + r * (J.row_stride ? J.row_stride : (size_t)J.n);
  const float temp = fmaxf(J.temperature, 1e-4f);
  unsigned long long best = 0ull;
  for (int i = tid; i < J.n; i += LP_THREADS) best = max(best, lp_key(lp_clean(x[i], temp), i));
  best = lp_block_max(kred, best);
  const float m = key_to_float((uint32_t)(best >> 32));
  const int c = (int)(0xffffffffu - (uint32_t)best);
  float s = 0.f, t = 0.f;
  for (int i = tid; i < J.n; i += LP_THREADS) {
    const float u = lp_clean(x[i], temp) - m, e = expf(u);
    if (i != c) {
      s += e;
      if (e > 0.f) t = fmaf(e, u, t);  // (u may be -inf where e is 0)
    }
  }
  s = lp_block_sum(fred, s);
  t = lp_block_sum(fred, t);
  const float ls = log1pf(s);
  if (tid == 0) {
    if (J.ids) {
      const int id = J.ids[r];
      float lp = 0.f;
      if (id >= 0 && id < J.n)
        lp = (lp_clean(x[id], temp) - m) - ls;
      else if (id != -1)
        raise_flag(GSDLQ_FLAG_BAD_TOKEN);
      J.logprob[r] = lp;
    }
    if (J.entropy) J.entropy[r] = ls - t / (1.0f + s);
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < J.top; ++j) {
    unsigned long long b = 0ull;
    for (int i = tid; i < J.n; i += LP_THREADS) {
      const unsigned long long k = lp_key(lp_clean(x[i], temp), i);
      if (k < last) b = max(b, k);
    }
    last = lp_block_max(kred, b);
    if (tid == 0) {
      J.top_ids[(size_t)r * J.top + j] = (int)(0xffffffffu - (uint32_t)last);
      J.top_logprobs[(size_t)r * J.top + j] = (key_to_float((uint32_t)(last >> 32)) - m) - ls;
    }
  }
}

}  // namespace gsdlq

using namespace gsdlq;

extern "C" int gsdlq_logprobs_rows(const gsdlq_logprobs_job_t* job, gsdlq_stream_t stream) {
  if (!job || !job->logits || job->rows <= 0 || job->n <= 0) return GSDLQ_ERR_INVALID;
  const gsdlq_logprobs_job_t& J = *job;
  if ((reinterpret_cast<uintptr_t>(J.logits) & 3u) || (J.row_stride && J.row_stride < (size_t)J.n)) return GSDLQ_ERR_INVALID;
  if (!(J.temperature > 0.f) || !std::isfinite(J.temperature)) return GSDLQ_ERR_INVALID;
  if ((J.ids != nullptr) != (J.logprob != nullptr)) return GSDLQ_ERR_INVALID;
  if (J.top < 0 || J.top > GSDLQ_MAX_TOP || J.top > J.n || (J.top > 0 && (!J.top_ids || !J.top_logprobs)))
    return GSDLQ_ERR_INVALID;
  if (!J.ids && !J.entropy && J.top == 0) return GSDLQ_ERR_INVALID;
  logprobs_rows_kernel<<<J.rows, LP_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(J);
  GSDLQ_CUDA_CHECK_LAUNCH();
  return GSDLQ_OK;
}
