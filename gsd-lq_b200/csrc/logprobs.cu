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

// A row is read once, by a cluster of 1 to 8 CTAs that each take a contiguous part of it.  A thread keeps the
// maximum m of its logits, and of the others the sums s of e^u and t of u e^u with u = (x - m) / temperature (in
// units of ln 2): a logit above m costs a rescaling and pushes the old maximum into the sums, every other one an
// ex2 and two additions.  Partial results (m1 >= m2) join as
//   d = (m2 - m1) / temperature,  f = e^d,  s = s1 + f (s2 + 1),  t = t1 + f (t2 + d (s2 + 1)).
//
// Alternatives without a second pass over the row: the threads' own maxima come with their indices, the maxima of
// the 64 groups of eight threads are ranked, and every token of the row's top k has a key of at least the k-th
// largest group maximum, K, since k tokens have; and it lies in one of the k groups whose maximum is at least K.
// Only those groups' tokens are looked at again (they are in the L2 cache), those at or above K -- mostly a few
// more than k -- are collected and ranked by counting.  Keys are (z, lowest index first) with z as the sampler
// rounds it, so equal z (different logits can share one) go by index.
constexpr int LP_THREADS = 512, LP_WARPS = LP_THREADS / 32;
constexpr int LP_GROUPS = LP_THREADS / 8;      // >= GSDLQ_MAX_TOP
constexpr int LP_CAP = 1280;                   // tokens collected before the slow path takes over
constexpr int LP_MAX_CLUSTER = 8;
typedef unsigned long long lp_key_t;

struct LpSums {
  float m, s, t;  // maximum (-inf: nothing yet), sums of the others
};
struct LpShared {
  LpSums sums[LP_WARPS];
  LpSums part;                  // this CTA's
  int n_top;                    // entries of top: k, or fewer where the CTA's part is shorter
  lp_key_t top[GSDLQ_MAX_TOP];  // this CTA's best, in order
  lp_key_t group[LP_GROUPS];
  lp_key_t K, red[LP_WARPS];
  lp_key_t all[LP_MAX_CLUSTER][GSDLQ_MAX_TOP];
  LpSums parts[LP_MAX_CLUSTER];
  int counts[LP_MAX_CLUSTER];
  int found;
  lp_key_t cand[LP_CAP];
};

__device__ __forceinline__ float lp_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float lp_clean(float x) {
  const uint32_t b = __float_as_uint(x);
  if ((b & 0x7fffffffu) >= 0x7f800000u) x = b == 0x7f800000u ? 100.f : -1e4f;
  return x;
}
// z of a cleaned logit; -0 becomes 0, which ties with it; a quotient past fp32 stays finite
__device__ __forceinline__ float lp_z(float x, float temp) {
  if (temp != 1.0f) x = fminf(fmaxf(__fdiv_rn(x, temp), -FLT_MAX), FLT_MAX);
  return x + 0.0f;
}
__device__ __forceinline__ lp_key_t lp_key(float z, int i) {
  return ((lp_key_t)ordered_key(z) << 32) | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ int lp_index(lp_key_t k) { return (int)(0xffffffffu - (uint32_t)k); }
// a little below x: logits that may round to the same z as x lie above it
__device__ __forceinline__ float lp_below(float x) { return x - fmaf(fabsf(x), 9.5367431640625e-07f, FLT_MIN); }

__device__ __forceinline__ LpSums lp_join(LpSums a, LpSums b, float c) {
  const LpSums hi = a.m >= b.m ? a : b, lo = a.m >= b.m ? b : a;
  if (lo.m == -INFINITY) return hi;
  const float d = fmaxf((lo.m - hi.m) * c, -200.f), f = lp_ex2(d);
  return {hi.m, fmaf(f, lo.s + 1.f, hi.s), fmaf(f, fmaf(d, lo.s + 1.f, lo.t), hi.t)};
}

struct LpThread {
  LpSums a;
  float near;  // logits at or above it are looked at closely
  float z;     // the best z, and its first index
  int i;
};
__device__ __forceinline__ void lp_add(LpThread& T, float x, int i, float temp, float c) {
  x = lp_clean(x);
  if (x >= T.near) {
    const float z = lp_z(x, temp);
    if (z > T.z) {
      T.z = z;
      T.i = i;
    }
    if (x > T.a.m) {
      if (T.a.m != -INFINITY) {
        const float d = fmaxf((T.a.m - x) * c, -200.f), f = lp_ex2(d), s1 = T.a.s + 1.f;
        T.a.t = f * fmaf(d, s1, T.a.t);
        T.a.s = f * s1;
      }
      T.a.m = x;
      T.near = lp_below(x);
      return;
    }
  }
  const float d = fmaxf((x - T.a.m) * c, -200.f), e = lp_ex2(d);
  T.a.s += e;
  T.a.t = fmaf(e, d, T.a.t);
}

__device__ lp_key_t lp_block_max(LpShared& S, lp_key_t k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) S.red[threadIdx.x >> 5] = k;
  __syncthreads();
  k = S.red[threadIdx.x & (LP_WARPS - 1)];
#pragma unroll
  for (int o = LP_WARPS / 2; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  return k;
}

__global__ void __launch_bounds__(LP_THREADS, 2)
    logprobs_rows_kernel(const __grid_constant__ gsdlq_logprobs_job_t J, int cluster) {
  __shared__ LpShared S;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x / cluster, rank = blockIdx.x - r * cluster;
  const float* const x = J.logits + (size_t)r * (J.row_stride ? J.row_stride : (size_t)J.n);
  const float temp = fmaxf(J.temperature, 1e-4f), c = 1.4426950408889634f / temp;
  const int per = (J.n + cluster - 1) / cluster;
  const int lo = min(rank * per, J.n), hi = (int)min((long long)lo + per, (long long)J.n);
  // 16-byte loads from v0 on: `head` single logits before it, `tail` behind the last whole four
  const int head = min((int)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(x + lo) & 15u)) & 15u) / 4, hi - lo);
  const int v0 = lo + head, nv = (hi - v0) / 4, tail = hi - v0 - 4 * nv;
  const float4* const xv = reinterpret_cast<const float4*>(x + v0);

  LpThread T = {{-INFINITY, 0.f, 0.f}, -INFINITY, -INFINITY, 0};
  if (tid < head) lp_add(T, x[lo + tid], lo + tid, temp, c);
  constexpr int UN = 4;
  for (int v = tid; v < nv; v += UN * LP_THREADS) {
    float4 w[UN];
#pragma unroll
    for (int k = 0; k < UN; ++k)
      if (v + k * LP_THREADS < nv) w[k] = __ldg(xv + v + k * LP_THREADS);
#pragma unroll
    for (int k = 0; k < UN; ++k)
      if (v + k * LP_THREADS < nv) {
        const int i = v0 + 4 * (v + k * LP_THREADS);
        lp_add(T, w[k].x, i, temp, c);
        lp_add(T, w[k].y, i + 1, temp, c);
        lp_add(T, w[k].z, i + 2, temp, c);
        lp_add(T, w[k].w, i + 3, temp, c);
      }
  }
  if (tid < tail) lp_add(T, x[v0 + 4 * nv + tid], v0 + 4 * nv + tid, temp, c);

  // ---- sums of the CTA's part
  LpSums a = T.a;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = lp_join(a, {__shfl_down_sync(0xffffffffu, a.m, o), __shfl_down_sync(0xffffffffu, a.s, o),
                    __shfl_down_sync(0xffffffffu, a.t, o)}, c);
  if (lane == 0) S.sums[warp] = a;
  if (J.top > 0) {
    lp_key_t g = T.z == -INFINITY ? 0ull : lp_key(T.z, T.i);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if ((lane & 7) == 0) S.group[tid >> 3] = g;
  }
  if (tid == 0) {
    S.K = 0ull;
    S.found = 0;
  }
  __syncthreads();
  if (warp == 0) {
    a = lane < LP_WARPS ? S.sums[lane] : LpSums{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = LP_WARPS / 2; o > 0; o >>= 1)
      a = lp_join(a, {__shfl_down_sync(0xffffffffu, a.m, o), __shfl_down_sync(0xffffffffu, a.s, o),
                      __shfl_down_sync(0xffffffffu, a.t, o)}, c);
    if (lane == 0) S.part = a;
  }

  // ---- the CTA's best J.top tokens
  if (J.top > 0) {
    const int k = min(J.top, hi - lo);
    if (tid < LP_GROUPS) {
      const lp_key_t g = S.group[tid];
      int above = 0;
#pragma unroll 8
      for (int j = 0; j < LP_GROUPS; ++j) above += S.group[j] > g;
      if (above == k - 1 && g != 0ull) S.K = g;  // the keys of groups with tokens differ: one thread
    }
    __syncthreads();
    const lp_key_t K = S.K;  // 0: fewer groups than k have tokens, and all tokens are collected
    const float zk = K ? key_to_float((uint32_t)(K >> 32)) : -INFINITY;
    const float close = K ? lp_below(zk * temp) : -INFINITY;
    auto look = [&](float v, int i) {
      v = lp_clean(v);
      if (v >= close) {
        const lp_key_t key = lp_key(lp_z(v, temp), i);
        if (key >= K) {
          const int at = atomicAdd(&S.found, 1);
          if (at < LP_CAP) S.cand[at] = key;
        }
      }
    };
    for (int g = warp; g < LP_GROUPS; g += LP_WARPS) {
      const lp_key_t key = S.group[g];
      if (key == 0ull || key < K) continue;
      for (int v = g * 8 + (lane & 7) + (lane >> 3) * LP_THREADS; v < nv; v += 4 * LP_THREADS) {
        const float4 w = __ldg(xv + v);
        const int i = v0 + 4 * v;
        look(w.x, i);
        look(w.y, i + 1);
        look(w.z, i + 2);
        look(w.w, i + 3);
      }
      if (g == 0) {  // the single logits belong to the first threads
        if (lane < head) look(x[lo + lane], lo + lane);
        if (lane < tail) look(x[v0 + 4 * nv + lane], v0 + 4 * nv + lane);
      }
    }
    __syncthreads();
    const int found = S.found;
    if (found <= LP_CAP) {
      for (int i = tid; i < found; i += LP_THREADS) {
        const lp_key_t key = S.cand[i];
        int above = 0;
        for (int j = 0; j < found; ++j) above += S.cand[j] > key;
        if (above < k) S.top[above] = key;
      }
    } else {
      // more tokens at or above K than the list holds (they crowd in a few groups): the largest, one by one
      lp_key_t last = ~0ull;
      for (int j = 0; j < k; ++j) {
        lp_key_t b = 0ull;
        for (int i = lo + tid; i < hi; i += LP_THREADS) {
          const lp_key_t key = lp_key(lp_z(lp_clean(x[i]), temp), i);
          if (key < last) b = max(b, key);
        }
        last = lp_block_max(S, b);
        if (tid == 0) S.top[j] = last;
      }
    }
    if (tid == 0) S.n_top = k;
  }

  // ---- the row
  if (cluster > 1) {
    cluster_sync_all();  // every CTA's part and top are written
    if (rank == 0) {
      const uint32_t at_part = smem_u32(&S.part), at_n = smem_u32(&S.n_top), at_top = smem_u32(S.top);
      if (tid < cluster) {
        const uint32_t p = mapa_shared(at_part, tid);
        S.parts[tid] = {ld_cluster_f32(p), ld_cluster_f32(p + 4), ld_cluster_f32(p + 8)};
        if (J.top > 0) S.counts[tid] = __float_as_int(ld_cluster_f32(mapa_shared(at_n, tid)));
      }
      if (J.top > 0 && tid < cluster * GSDLQ_MAX_TOP) {
        const int q = tid / GSDLQ_MAX_TOP, j = tid % GSDLQ_MAX_TOP;
        const uint32_t p = mapa_shared(at_top, q) + j * 8;
        const uint32_t l = __float_as_uint(ld_cluster_f32(p)), h = __float_as_uint(ld_cluster_f32(p + 4));
        S.all[q][j] = ((lp_key_t)h << 32) | l;
      }
    }
    cluster_sync_all();  // ... and read
    if (rank != 0) return;
  } else {
    __syncthreads();
  }
  LpSums row = cluster > 1 ? S.parts[0] : S.part;
  for (int q = 1; q < cluster; ++q) row = lp_join(row, S.parts[q], c);
  const float ls = log1pf(row.s), inv = 1.0f / temp;
  auto logp = [&](float v) { return (v - row.m) * inv - ls; };
  if (tid == 0) {
    if (J.ids) {
      const int id = J.ids[r];
      float lp = 0.f;
      if (id >= 0 && id < J.n)
        lp = logp(lp_clean(x[id]));
      else if (id != -1)
        raise_flag(GSDLQ_FLAG_BAD_TOKEN);
      J.logprob[r] = lp;
    }
    if (J.entropy) J.entropy[r] = ls - 0.6931471805599453f * row.t / (1.0f + row.s);
  }
  auto put = [&](int j, lp_key_t key) {
    const int i = lp_index(key);
    J.top_ids[(size_t)r * J.top + j] = i;
    J.top_logprobs[(size_t)r * J.top + j] = logp(lp_clean(x[i]));
  };
  if (cluster == 1) {
    if (tid < J.top) put(tid, S.top[tid]);
  } else if (J.top > 0 && tid < cluster * GSDLQ_MAX_TOP) {
    // the place of entry j of CTA q's list: j, and what the other lists have above it
    const int q = tid / GSDLQ_MAX_TOP, j = tid % GSDLQ_MAX_TOP;
    if (j < S.counts[q]) {
      const lp_key_t key = S.all[q][j];
      int at = j;
      for (int o = 0; o < cluster; ++o) {
        if (o == q) continue;
        int a = 0, b = S.counts[o];
        while (a < b) {
          const int mid = (a + b) / 2;
          if (S.all[o][mid] > key)
            a = mid + 1;
          else
            b = mid;
        }
        at += a;
      }
      if (at < J.top) put(at, key);
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
  // CTAs a row: enough for about four an SM, none with less than 2048 logits
  int cluster = 1;
  while (cluster < LP_MAX_CLUSTER && (long long)J.rows * cluster * 2 <= 4 * num_sms() && J.n / (cluster * 2) >= 2048)
    cluster *= 2;
  if ((long long)J.rows * cluster > INT32_MAX) return GSDLQ_ERR_INVALID;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(J.rows * cluster));
  cfg.blockDim = dim3(LP_THREADS);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, logprobs_rows_kernel, J, cluster);
  return e == cudaSuccess ? GSDLQ_OK : record_cuda_error(e);
}
