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
#include <climits>
#include <cmath>

#include "common.cuh"

namespace gsdlq {

// A row is read once, by a cluster of 1 to 8 CTAs that each take a contiguous part of it.  A warp keeps the
// maximum m of its logits, and of the others the sums s of e^u and t of u e^u with u = (x - m) / temperature (in
// units of ln 2): a logit costs an ex2 and two additions, a batch with a new maximum a rescaling besides, which puts
// the old maximum into the sums.  (With a maximum per thread nearly every batch had a new one in some lane.)
// Partial results (m1 >= m2) join as
//   d = (m2 - m1) / temperature,  f = e^d,  s = s1 + f (s2 + 1),  t = t1 + f (t2 + d (s2 + 1)).
//
// Alternatives without a second pass over the row: the maxima of the 128 groups of four threads are ranked.  Every
// token of the best k has a key of at least the k-th largest group maximum, K, since k tokens have; and it lies in
// one of the k groups whose maximum is at least K.  Only those groups' tokens are looked at again (they are in the
// L2 cache); those at or above K -- mostly a few more than k -- are collected and ranked by counting.  Keys are
// (z, lowest index first) with z as the sampler rounds it, so equal z (different logits can share one) go by index;
// the tokens' indices are looked up only where the k-th maximum is shared by more groups than are wanted, as in
// rows with fewer unmasked tokens than k.
//
// 128 rows of 151936 (78 MB): 18.4 us without alternatives, 25.6 with 20; 592 rows: 61 us (5.9 TB/s) and 81.  Large
// batches are bound by HBM, 128 rows by the start and the end of 256 CTAs that all run at once; the alternatives
// cost a tail of barriers, a second look at 2 % of the tokens and the joining of the cluster's lists.
constexpr int LP_THREADS = 512, LP_WARPS = LP_THREADS / 32;
constexpr int LP_LANES = 4, LP_GROUPS = LP_THREADS / LP_LANES;  // groups of neighbouring lanes; >= GSDLQ_MAX_TOP
constexpr int LP_CAP = 1280;                   // tokens collected before the slow path takes over
constexpr int LP_MAX_CLUSTER = 8;
typedef unsigned long long lp_key_t;

struct LpSums {
  float m, s, t;  // maximum (-inf: nothing yet), sums of the others
};
struct LpShared {
  LpSums sums[LP_WARPS];
  LpSums part;                  // this CTA's
  lp_key_t top[GSDLQ_MAX_TOP];  // this CTA's best, in order, then zeros
  alignas(16) uint32_t gz[LP_GROUPS];  // the groups' maxima
  uint32_t kz;                 // the k-th largest of them
  int over;                    // how many of the groups that share it are wanted, where not all are
  lp_key_t group[LP_GROUPS];   // their keys then
  lp_key_t K, red[LP_WARPS];
  lp_key_t all[LP_MAX_CLUSTER][GSDLQ_MAX_TOP];
  LpSums parts[LP_MAX_CLUSTER];
  int n_list, list[GSDLQ_MAX_TOP];  // the groups that hold the CTA's best
  int found;
  lp_key_t cand[LP_CAP];
};

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
// A logit below which no quotient reaches z.  A quotient is z if it lies less than z's own rounding step away (a share
// of 2^-23, or 2^-149 where z is subnormal), and the product with the temperature rounds too; the quotients at -FLT_MAX
// include all that lie below it.
__device__ __forceinline__ float lp_below(float z, float temp) {
  constexpr float REL = 9.5367431640625e-07f, TINY = 2.8025969e-45f;  // 2^-20; two subnormal steps
  const float x = (z - fmaf(fabsf(z), REL, TINY)) * temp;             // -inf for z = -FLT_MAX
  return x - fmaf(fabsf(x), REL, FLT_MIN);
}

__device__ __forceinline__ LpSums lp_join(LpSums a, LpSums b, float c) {
  const LpSums hi = a.m >= b.m ? a : b, lo = a.m >= b.m ? b : a;
  if (lo.m == -INFINITY) return hi;
  const float d = fmaxf((lo.m - hi.m) * c, -200.f), f = ex2_ftz(d);
  return {hi.m, fmaf(f, lo.s + 1.f, hi.s), fmaf(f, fmaf(d, lo.s + 1.f, lo.t), hi.t)};
}

// What a warp has read of its part: the lanes share the maximum m as reference; `holds` says in which lane it lies.
struct LpWarp {
  float m, s, t;  // s and t: this lane's, without the maximum
  bool holds;
  float top;      // this lane's largest logit (-inf: nothing yet)
};
// clean N logits; -inf for those that are not there
template <int N>
__device__ __forceinline__ void lp_clean(float (&x)[N]) {
  float wild = 0.f;  // not finite if a logit is not
#pragma unroll
  for (int k = 0; k < N; ++k) wild = fmaf(x[k], 0.f, wild);
  if (wild != 0.f) {
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = lp_clean(x[k]);
  }
}
// N logits of each lane (-inf: none).  Only a new maximum of the whole warp costs more than the sums.
template <int N>
__device__ __forceinline__ void lp_add(LpWarp& T, float (&x)[N], float c) {
  float top = x[0];
#pragma unroll
  for (int k = 1; k < N; ++k) top = fmaxf(top, x[k]);
  T.top = fmaxf(T.top, top);
  const float wtop = key_to_float(__reduce_max_sync(0xffffffffu, ordered_key(top + 0.0f)));
  if (wtop > T.m) {
    const float d = fmaxf((T.m - wtop) * c, -200.f), f = ex2_ftz(d), s1 = T.s + (T.holds ? 1.f : 0.f);
    T.t = f * fmaf(d, s1, T.t);
    T.s = f * s1;
    T.m = wtop;
    T.holds = __ffs(__ballot_sync(0xffffffffu, top == wtop)) - 1 == (int)(threadIdx.x & 31);
    if (T.holds) {
      bool out = false;  // the first one that equals it is the maximum, which the sums leave out
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const bool it = !out && x[k] == wtop;
        out |= it;
        x[k] = it ? -INFINITY : x[k];
      }
    }
  }
  // (four of each sum, so that a chain of additions is short)
  float s4[4] = {0.f, 0.f, 0.f, 0.f}, t4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float d = fmaxf((x[k] - T.m) * c, -200.f), e = ex2_ftz(d);
    s4[k & 3] += e;
    t4[k & 3] = fmaf(e, d, t4[k & 3]);
  }
  T.s += (s4[0] + s4[1]) + (s4[2] + s4[3]);
  T.t += (t4[0] + t4[1]) + (t4[2] + t4[3]);
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
  pdl_wait();
  pdl_launch_dependents();
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

  // the given token's logit, early
  const int id = rank == 0 && tid == 0 && J.ids ? J.ids[r] : -1;
  const float x_id = id >= 0 && id < J.n ? x[id] : 0.f;

  LpWarp T = {-INFINITY, 0.f, 0.f, false, -INFINITY};
  if (warp == 0 && head > 0) {
    float w[1] = {-INFINITY};
    if (tid < head) w[0] = lp_clean(x[lo + tid]);
    lp_add<1>(T, w, c);
  }
  constexpr int UN = 4;  // vectors of a batch, one every LP_THREADS
  int v = tid;           // (the loops' ends are the warp's, not the lane's)
  for (; v - lane + 31 + (UN - 1) * LP_THREADS < nv; v += UN * LP_THREADS) {
    float w[UN][4];
#pragma unroll
    for (int k = 0; k < UN; ++k) *reinterpret_cast<float4*>(w[k]) = __ldg(xv + v + k * LP_THREADS);
#pragma unroll
    for (int k = 0; k < UN; ++k) lp_clean<4>(w[k]);
    lp_add<4 * UN>(T, reinterpret_cast<float(&)[4 * UN]>(w), c);
  }
  for (; v - lane < nv; v += LP_THREADS) {
    float w[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (v < nv) {
      *reinterpret_cast<float4*>(w) = __ldg(xv + v);
      lp_clean<4>(w);
    }
    lp_add<4>(T, w, c);
  }
  if (warp == 0 && tail > 0) {
    float w[1] = {-INFINITY};
    if (tid < tail) w[0] = lp_clean(x[v0 + 4 * nv + tid]);
    lp_add<1>(T, w, c);
  }

  // ---- sums of the CTA's part
  {
    const float ws = warp_sum(T.s), wt = warp_sum(T.t);
    if (lane == 0) S.sums[warp] = {T.m, ws, wt};
  }
  const float my_top = lp_z(T.top, temp);
  const uint32_t my_z = T.top == -INFINITY ? 0u : ordered_key(my_top);  // 0: no token
  if (J.top > 0) {
    uint32_t g = my_z;
#pragma unroll
    for (int o = LP_LANES / 2; o > 0; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (lane % LP_LANES == 0) S.gz[tid / LP_LANES] = g;
  }
  if (tid == 0) {
    S.kz = 0u;
    S.over = S.found = S.n_list = 0;
  }
  __syncthreads();
  if (warp == 0) {
    LpSums a = lane < LP_WARPS ? S.sums[lane] : LpSums{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = LP_WARPS / 2; o > 0; o >>= 1)
      a = lp_join(a, {__shfl_down_sync(0xffffffffu, a.m, o), __shfl_down_sync(0xffffffffu, a.s, o),
                      __shfl_down_sync(0xffffffffu, a.t, o)}, c);
    if (lane == 0) S.part = a;
  }

  // ---- the CTA's best J.top tokens
  if (J.top > 0) {
    const int k = min(J.top, hi - lo);
    {
      // a group's lanes count a quarter of the others each
      const int grp = tid / LP_LANES;
      const uint32_t g = S.gz[grp];
      int above = 0, same = 0;
#pragma unroll
      for (int j = 0; j < LP_GROUPS / (4 * LP_LANES); ++j) {
        const uint4 z = *reinterpret_cast<const uint4*>(S.gz + 4 * (j * LP_LANES + lane % LP_LANES));
        above += (z.x > g) + (z.y > g) + (z.z > g) + (z.w > g);
        same += (z.x == g) + (z.y == g) + (z.z == g) + (z.w == g);
      }
#pragma unroll
      for (int o = LP_LANES / 2; o > 0; o >>= 1) {
        above += __shfl_xor_sync(0xffffffffu, above, o);
        same += __shfl_xor_sync(0xffffffffu, same, o);
      }
      if (lane % LP_LANES == 0 && above < k && g != 0u) {
        if (above + same > k)  // more groups share this maximum than belong to the best k
          S.over = k - above;  // (the same from all of them)
        else
          S.list[atomicAdd(&S.n_list, 1)] = grp;
        if (above + same >= k) S.kz = g;  // (the same value from all that write it)
      }
    }
    __syncthreads();
    // the k-th largest group maximum; 0: fewer groups than k have tokens, and all tokens are collected
    lp_key_t K = (lp_key_t)S.kz << 32;
    if (S.over > 0) {  // (uniform) of the groups that share it, those with the lowest indices
      lp_key_t g = 0ull;
      if (my_z == S.kz && S.gz[tid / LP_LANES] == S.kz) {
        // the thread's first token with its best z
        int i = tid < head && lp_z(lp_clean(x[lo + tid]), temp) == my_top ? lo + tid : INT_MAX;
        for (int q = tid; q < nv && i == INT_MAX; q += LP_THREADS) {
          const float4 w = __ldg(xv + q);
          const float e[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 3; j >= 0; --j)
            if (lp_z(lp_clean(e[j]), temp) == my_top) i = v0 + 4 * q + j;
        }
        if (i == INT_MAX) i = v0 + 4 * nv + tid;
        g = lp_key(my_top, i);
      }
#pragma unroll
      for (int o = LP_LANES / 2; o > 0; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
      if (lane % LP_LANES == 0) S.group[tid / LP_LANES] = g;
      __syncthreads();
      if (tid < LP_GROUPS && S.group[tid] != 0ull) {
        int above = 0;
        for (int j = 0; j < LP_GROUPS; ++j) above += S.group[j] > S.group[tid];
        if (above < S.over) S.list[atomicAdd(&S.n_list, 1)] = tid;
        if (above == S.over - 1) S.K = S.group[tid];
      }
      __syncthreads();
      K = S.K;
    }
    const float zk = K ? key_to_float((uint32_t)(K >> 32)) : -INFINITY;
    const float close = K ? lp_below(zk, temp) : -INFINITY;
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
    // the listed groups' vectors, dealt to all threads, LOOKS loads at a time
    constexpr int LOOKS = 4;
    const int per_group = LP_LANES * ((nv + LP_THREADS - 1) / LP_THREADS), looks = S.n_list * per_group;
    for (int e0 = tid; e0 < looks; e0 += LOOKS * LP_THREADS) {
      float4 w[LOOKS];
      int at[LOOKS];
#pragma unroll
      for (int u = 0; u < LOOKS; ++u) {
        const int e = e0 + u * LP_THREADS, g = e / per_group, j = e - g * per_group;
        at[u] = e < looks ? S.list[g] * LP_LANES + j % LP_LANES + j / LP_LANES * LP_THREADS : nv;
        if (at[u] < nv) w[u] = __ldg(xv + at[u]);
      }
#pragma unroll
      for (int u = 0; u < LOOKS; ++u)
        if (at[u] < nv) {
          const int i = v0 + 4 * at[u];
          look(w[u].x, i);
          look(w[u].y, i + 1);
          look(w[u].z, i + 2);
          look(w[u].w, i + 3);
        }
    }
    if (tid < max(head, tail)) {  // the single logits belong to the first threads
      if (tid < head) look(x[lo + tid], lo + tid);
      if (tid < tail) look(x[v0 + 4 * nv + tid], v0 + 4 * nv + tid);
    }
    __syncthreads();
    const int found = S.found;
    if (found <= LP_CAP) {
      for (int i = tid; i < found; i += LP_THREADS) {
        const lp_key_t key = S.cand[i];
        int above = 0;
#pragma unroll 8
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
    if (tid >= k && tid < GSDLQ_MAX_TOP) S.top[tid] = 0ull;  // below every key
  }

  // ---- the row
  if (cluster > 1) {
    cluster_sync_all();  // every CTA's part and top are written
    if (rank == 0) {
      const uint32_t at_part = smem_u32(&S.part), at_top = smem_u32(S.top);
      if (tid < cluster) {
        const uint32_t p = mapa_shared(at_part, tid);
        S.parts[tid] = {ld_cluster_f32(p), ld_cluster_f32(p + 4), ld_cluster_f32(p + 8)};
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
  const float zm = lp_z(row.m, temp);
  if (tid == 0) {
    if (J.ids) {
      float lp = 0.f;
      if (id >= 0 && id < J.n)
        lp = (lp_clean(x_id) - row.m) * inv - ls;
      else if (id != -1)
        raise_flag(GSDLQ_FLAG_BAD_TOKEN);
      J.logprob[r] = lp;
    }
    if (J.entropy) J.entropy[r] = ls - 0.6931471805599453f * row.t / (1.0f + row.s);
  }
  auto put = [&](int j, lp_key_t key) {
    J.top_ids[(size_t)r * J.top + j] = lp_index(key);
    J.top_logprobs[(size_t)r * J.top + j] = (key_to_float((uint32_t)(key >> 32)) - zm) - ls;
  };
  if (cluster == 1) {
    if (tid < J.top) put(tid, S.top[tid]);
  } else if (J.top > 0 && tid < cluster * GSDLQ_MAX_TOP) {
    // the place of entry j of CTA q's list: j, and what the other lists have above it
    // (all searches side by side: list o has at[o] keys above it)
    const int q = tid / GSDLQ_MAX_TOP, j = tid % GSDLQ_MAX_TOP;
    const lp_key_t key = S.all[q][j];
    int at[LP_MAX_CLUSTER];
#pragma unroll
    for (int o = 0; o < LP_MAX_CLUSTER; ++o) at[o] = 0;
#pragma unroll
    for (int step = GSDLQ_MAX_TOP / 2; step > 0; step >>= 1)
#pragma unroll
      for (int o = 0; o < LP_MAX_CLUSTER; ++o)
        if (o < cluster && S.all[o][at[o] + step - 1] > key) at[o] += step;
    int place = 0;
#pragma unroll
    for (int o = 0; o < LP_MAX_CLUSTER; ++o)
      if (o < cluster) place += at[o] + (at[o] == GSDLQ_MAX_TOP - 1 && S.all[o][GSDLQ_MAX_TOP - 1] > key);
    if (key != 0ull && place < J.top) put(place, key);
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
  // CTAs a row: as many as run at once, two an SM, none with less than 8192 logits (a row of 32768 with 5
  // alternatives: 7.6 us with 8 CTAs, 6.6 with 4, 7.1 with 2, 7.6 with 1; of 151936 with 20: 10.2 with 8, 11.8 with 4)
  int cluster = 1;
  while (cluster < LP_MAX_CLUSTER && (long long)J.rows * cluster * 2 <= 2 * num_sms() && J.n / (cluster * 2) >= 8192)
    cluster *= 2;
  if ((long long)J.rows * cluster > INT32_MAX) return GSDLQ_ERR_INVALID;
  return launch_pdl(logprobs_rows_kernel, (unsigned)(J.rows * cluster), LP_THREADS, 0, static_cast<cudaStream_t>(stream),
                    (unsigned)cluster, J, cluster);
}
