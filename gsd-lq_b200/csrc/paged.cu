// paged.cu -- a batch of sequences over one pool of K/V pages: RoPE + append, decode attention, and the
// pages' own operations (fork, reserve, compact, copy).  No reference counterpart: the reference keeps
// one contiguous cache (gsd_lq_cpu_engine.c:186-330); the per-row arithmetic is that of its functions.
#include <algorithm>
#include <cmath>

#include "common.cuh"

namespace gsdlq {

// ---------------------------------------------------------------------------------------
// rows

// Sequence of row r, and how many positions it has with its own (0: idle).  `flag`: report what is wrong
// with it (once per launch is enough).
struct PagedRow {
  int seq, len;
};
__device__ __forceinline__ PagedRow paged_row(const gsdlq_paged_kv_t& kv, const int* row_seq, const int* pos, int r,
                                              bool flag) {
  const int p = pos[r], s = row_seq ? row_seq[r] : r;
  if (p == -1) return {s, 0};
  if (s < 0 || s >= kv.n_seqs) {
    if (flag) raise_flag(GSDLQ_FLAG_BAD_PAGE);
    return {s, 0};
  }
  if (p < 0 || (long long)p >= (long long)kv.max_blocks * kv.page_size) {
    if (flag) raise_flag(GSDLQ_FLAG_BAD_POS);
    return {s, 0};
  }
  return {s, p + 1};
}

__device__ __forceinline__ bool paged_valid(const gsdlq_paged_kv_t& kv, int page) {
  return page >= 0 && page < kv.n_pages;
}

template <bool BF16>
__device__ __forceinline__ uint16_t kv_round(float v) {
  return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : f2h(v);
}
template <bool BF16>
__device__ __forceinline__ float kv_value(uint16_t b) {
  return BF16 ? __uint_as_float((uint32_t)b << 16) : h2f(b);
}

// ---------------------------------------------------------------------------------------
// RoPE + append.  One CTA per row.
template <bool BF16>
__global__ void __launch_bounds__(256) rope_kv_paged_kernel(const __grid_constant__ gsdlq_paged_append_job_t J) {
  const gsdlq_paged_kv_t& kv = J.kv;
  const int r = blockIdx.x, tid = threadIdx.x, hd = kv.head_dim, half = hd / 2;
  PagedRow row = paged_row(kv, J.row_seq, J.pos, r, tid == 0);
  if (row.len > J.max_pos) {
    if (tid == 0) raise_flag(GSDLQ_FLAG_BAD_POS);
    row.len = 0;
  }
  const int pos = row.len - 1;
  const size_t qw = (size_t)J.n_heads * hd, kw = (size_t)kv.n_kv_heads * hd;
  const float* q = J.q + r * (J.q_stride ? (size_t)J.q_stride : qw);
  float* qo = J.q_out + r * (J.q_out_stride ? (size_t)J.q_out_stride : qw);
  if (row.len == 0) {
    if (q != qo)
      for (size_t i = tid; i < qw; i += blockDim.x) qo[i] = q[i];
    return;
  }
  const float2* cs = reinterpret_cast<const float2*>(J.rope_cs) + (size_t)pos * half;
  for (int e = tid; e < J.n_heads * half; e += blockDim.x) {
    const int h = e / half, i = e - h * half;
    const int i0 = h * hd + (J.interleaved ? 2 * i : i), i1 = h * hd + (J.interleaved ? 2 * i + 1 : i + half);
    const float a = q[i0], b = q[i1];
    const float2 c = cs[i];
    qo[i0] = __fsub_rn(__fmul_rn(a, c.x), __fmul_rn(b, c.y));
    qo[i1] = __fadd_rn(__fmul_rn(a, c.y), __fmul_rn(b, c.x));
  }
  const int page = kv.table[(size_t)row.seq * kv.max_blocks + pos / kv.page_size];
  if (!paged_valid(kv, page) || kv.refs[page] != 1) {
    if (tid == 0) raise_flag(GSDLQ_FLAG_BAD_PAGE);
    return;
  }
  const size_t at = (((size_t)J.layer * kv.n_pages + page) * kv.page_size + pos % kv.page_size) * kw;
  uint16_t* kd = static_cast<uint16_t*>(kv.k) + at;
  uint16_t* vd = static_cast<uint16_t*>(kv.v) + at;
  const float* k = J.k + r * (J.kv_stride ? (size_t)J.kv_stride : kw);
  const float* v = J.v + r * (J.kv_stride ? (size_t)J.kv_stride : kw);
  for (int e = tid; e < kv.n_kv_heads * half; e += blockDim.x) {
    const int h = e / half, i = e - h * half;
    const int i0 = h * hd + (J.interleaved ? 2 * i : i), i1 = h * hd + (J.interleaved ? 2 * i + 1 : i + half);
    const float a = k[i0], b = k[i1];
    const float2 c = cs[i];
    kd[i0] = kv_round<BF16>(__fsub_rn(__fmul_rn(a, c.x), __fmul_rn(b, c.y)));
    kd[i1] = kv_round<BF16>(__fadd_rn(__fmul_rn(a, c.y), __fmul_rn(b, c.x)));
    vd[i0] = kv_round<BF16>(v[i0]);
    vd[i1] = kv_round<BF16>(v[i1]);
  }
}

// ---------------------------------------------------------------------------------------
// Attention: a warp per (row, query head), lanes over the head's dimensions, position by position with a
// running maximum and sum.
template <int HD, bool BF16>
__global__ void __launch_bounds__(128) attention_paged_kernel(const __grid_constant__ gsdlq_paged_attn_job_t J) {
  constexpr int DL = HD / 32;
  const gsdlq_paged_kv_t& kv = J.kv;
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= (long long)J.rows * J.n_heads) return;
  const int r = (int)(item / J.n_heads), h = (int)(item % J.n_heads), g = h / (J.n_heads / kv.n_kv_heads);
  const PagedRow row = paged_row(kv, J.row_seq, J.pos, r, lane == 0);
  const float* q = J.q + r * (J.q_stride ? (size_t)J.q_stride : (size_t)J.n_heads * HD) + h * HD + lane * DL;
  float qv[DL], acc[DL], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < DL; ++d) {
    qv[d] = q[d] * J.sm_scale;
    acc[d] = 0.f;
  }
  const size_t kw = (size_t)kv.n_kv_heads * HD;
  for (int t = 0; t < row.len; ++t) {
    const int page = kv.table[(size_t)row.seq * kv.max_blocks + t / kv.page_size];
    if (!paged_valid(kv, page)) {
      if (lane == 0) raise_flag(GSDLQ_FLAG_BAD_PAGE);
      continue;
    }
    const size_t at =
        (((size_t)J.layer * kv.n_pages + page) * kv.page_size + t % kv.page_size) * kw + (size_t)g * HD + lane * DL;
    const uint16_t* k = static_cast<const uint16_t*>(kv.k) + at;
    const uint16_t* v = static_cast<const uint16_t*>(kv.v) + at;
    float s = 0.f;
#pragma unroll
    for (int d = 0; d < DL; ++d) s = fmaf(qv[d], kv_value<BF16>(k[d]), s);
    s = warp_sum(s);
    const float mn = fmaxf(m, s), f = expf(m - mn), p = expf(s - mn);
    l = l * f + p;
    m = mn;
#pragma unroll
    for (int d = 0; d < DL; ++d) acc[d] = fmaf(p, kv_value<BF16>(v[d]), acc[d] * f);
  }
  float* o = J.out + ((size_t)r * J.n_heads + h) * HD + lane * DL;
#pragma unroll
  for (int d = 0; d < DL; ++d) o[d] = l > 0.f ? acc[d] / l : 0.f;
}

constexpr int PA_MAX_CTAS = 320;  // largest grid of an attention launch
constexpr int PA_GROUP = 8;       // query heads of one kv head taken together
inline size_t attention_paged_counters(int rows, int n_heads, int n_kv) {
  const size_t items = (size_t)rows * n_kv * ((n_heads / n_kv + PA_GROUP - 1) / PA_GROUP);
  return (items * sizeof(unsigned) + 15) / 16 * 16;
}
inline size_t attention_paged_work(int rows, int n_heads, int n_kv, int hd) {
  return attention_paged_counters(rows, n_heads, n_kv) + sizeof(float) * (size_t)PA_MAX_CTAS * 2 * PA_GROUP * (hd + 2);
}

// ---------------------------------------------------------------------------------------
// Pages: fork.  A CTA owns `cols` columns of the table: it reads them whole, then writes the entries that
// change and moves their counts.  The counts are integers, so the order of the atomics does not show.
__global__ void __launch_bounds__(256) pages_fork_kernel(const __grid_constant__ gsdlq_paged_kv_t kv,
                                                         const int* __restrict__ parent, int cols) {
  extern __shared__ int fork_tile[];  // [n_seqs][cols]
  const int c0 = blockIdx.x * cols, nc = min(cols, kv.max_blocks - c0);
  for (int e = threadIdx.x; e < kv.n_seqs * cols; e += blockDim.x) {
    const int b = e / cols, c = e - b * cols;
    if (c < nc) fork_tile[e] = kv.table[(size_t)b * kv.max_blocks + c0 + c];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kv.n_seqs * cols; e += blockDim.x) {
    const int b = e / cols, c = e - b * cols;
    if (c >= nc) continue;
    const int p = parent[b];
    if (p < -1 || p >= kv.n_seqs) {
      if (c == 0) raise_flag(GSDLQ_FLAG_BAD_PAGE);
      continue;
    }
    const int was = fork_tile[e], now = p < 0 ? -1 : fork_tile[p * cols + c];
    if (was == now) continue;
    kv.table[(size_t)b * kv.max_blocks + c0 + c] = now;
    if (paged_valid(kv, was)) atomicAdd(&kv.refs[was], -1);
    if (paged_valid(kv, now)) atomicAdd(&kv.refs[now], 1);
  }
}

// ---------------------------------------------------------------------------------------
// Block-wide scans over the pages' counts, 1024 threads: PG_PER pages a thread and step, a warp's 32
// consecutive pages as one ballot, and one warp's scan over the step's 32 * PG_PER ballots.
constexpr int PG_THREADS = 1024, PG_PER = 4, PG_STEP = PG_THREADS * PG_PER;
struct PageScan {
  unsigned cnt[32 * PG_PER];
  unsigned total;
};
// f[i]: whether page base + i * 1024 + tid is wanted; rank[i]: how many wanted pages of this step come before
// it.  Returns the number of wanted pages of the step.
__device__ __forceinline__ unsigned page_scan(PageScan& S, const bool (&f)[PG_PER], unsigned (&rank)[PG_PER]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned m[PG_PER];
  __syncthreads();  // the previous step's counts are read
#pragma unroll
  for (int i = 0; i < PG_PER; ++i) {
    m[i] = __ballot_sync(0xffffffffu, f[i]);
    if (lane == 0) S.cnt[i * 32 + warp] = __popc(m[i]);
  }
  __syncthreads();
  if (warp == 0) {
    unsigned v[PG_PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PG_PER; ++i) {
      v[i] = sum;
      sum += S.cnt[lane * PG_PER + i];
    }
    unsigned inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
#pragma unroll
    for (int i = 0; i < PG_PER; ++i) S.cnt[lane * PG_PER + i] = inc - sum + v[i];
    if (lane == 31) S.total = inc;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PG_PER; ++i) rank[i] = S.cnt[i * 32 + warp] + __popc(m[i] & ((1u << lane) - 1u));
  return S.total;
}

// Pages: reserve.  One CTA, thread r = row r.  The rows act in order, so a row that shares its page with
// `before` earlier rows of the call finds refs - before entries on it when its turn comes: it takes a copy
// while that is more than one, and the last holder keeps the page.  Two rows at one table entry: the first
// one acts.
__global__ void __launch_bounds__(PG_THREADS) pages_reserve_kernel(const __grid_constant__ gsdlq_paged_kv_t kv,
                                                                   const int* __restrict__ row_seq,
                                                                   const int* __restrict__ pos, int rows, int* src,
                                                                   int* dst, int max_pairs, int* counts) {
  __shared__ long long slot[GSDLQ_PAGED_MAX_SEQS];
  __shared__ int page[GSDLQ_PAGED_MAX_SEQS], fresh[GSDLQ_PAGED_MAX_SEQS];
  __shared__ unsigned char dup[GSDLQ_PAGED_MAX_SEQS], failed[GSDLQ_PAGED_MAX_SEQS];
  __shared__ PageScan S;
  const int r = threadIdx.x;
  long long my_slot = -1;
  int my_page = -1;
  if (r < rows) {
    const PagedRow row = paged_row(kv, row_seq, pos, r, true);
    if (row.len > 0) {
      my_slot = (long long)row.seq * kv.max_blocks + (row.len - 1) / kv.page_size;
      my_page = kv.table[my_slot];
      if (!paged_valid(kv, my_page)) {
        if (my_page != -1) raise_flag(GSDLQ_FLAG_BAD_PAGE);
        my_page = -1;
      }
    }
    slot[r] = my_slot;
    page[r] = my_page;
    failed[r] = 0;
  }
  __syncthreads();
  bool again = false;
  if (my_slot >= 0)
    for (int i = 0; i < r; ++i) again |= slot[i] == my_slot;
  if (r < rows) dup[r] = again;
  __syncthreads();
  const bool acts = my_slot >= 0 && !again;
  int before = 0;
  if (acts && my_page >= 0)
    for (int i = 0; i < r; ++i) before += page[i] == my_page && slot[i] >= 0 && !dup[i];
  const int held = acts && my_page >= 0 ? kv.refs[my_page] : 0;
  const bool shared = held - before > 1;
  const bool need = acts && (my_page < 0 || shared);
  bool f[PG_PER] = {need, false, false, false};
  unsigned rank[PG_PER];
  const unsigned wanted = page_scan(S, f, rank);
  const unsigned my_rank = rank[0];
  // the lowest free pages
  unsigned have = 0;
  for (int base = 0; base < kv.n_pages && have < wanted; base += PG_STEP) {
#pragma unroll
    for (int i = 0; i < PG_PER; ++i) {
      const int p = base + i * PG_THREADS + r;
      f[i] = p < kv.n_pages && kv.refs[p] <= 0;
    }
    const unsigned n = page_scan(S, f, rank);
#pragma unroll
    for (int i = 0; i < PG_PER; ++i)
      if (f[i] && have + rank[i] < wanted) fresh[have + rank[i]] = base + i * PG_THREADS + r;
    have += n;
  }
  __syncthreads();  // fresh[] is complete, and every count has been read
  const bool got = need && my_rank < have;
  f[0] = got && my_page >= 0;
  f[1] = f[2] = f[3] = false;
  const unsigned pairs = page_scan(S, f, rank);
  if (got) {
    const int p = fresh[my_rank];
    kv.table[my_slot] = p;
    kv.refs[p] = 1;
    if (my_page >= 0) {
      atomicAdd(&kv.refs[my_page], -1);
      src[rank[0]] = my_page;
      dst[rank[0]] = p;
    }
  }
  for (int i = pairs + r; i < max_pairs; i += PG_THREADS) src[i] = dst[i] = -1;
  int short_of = 0;
  if (have < wanted) {  // exhausted (uniform): the last holder of a page that an earlier row could not leave fails too
    bool fails = need && !got;
    if (r < rows) failed[r] = fails;
    __syncthreads();
    if (acts && !need && my_page >= 0 && before > 0)
      for (int i = 0; i < r; ++i) fails |= page[i] == my_page && failed[i];
    if (fails) raise_flag(GSDLQ_FLAG_NO_PAGE);
    short_of = __syncthreads_count(fails);
  }
  if (r == 0) {
    counts[0] = (int)pairs;
    counts[1] = short_of;
    counts[2] = (int)min(wanted, have);
  }
}

// Pages: compact.  One CTA plans: the number of pages in use, then the free pages below it in ascending
// order against the pages in use at and above it in descending order; `to` maps old to new pages.
__global__ void __launch_bounds__(PG_THREADS) pages_compact_kernel(const __grid_constant__ gsdlq_paged_kv_t kv, int* src,
                                                                   int* dst, int max_pairs, int* counts, int* to) {
  __shared__ PageScan S;
  __shared__ int high;
  const int tid = threadIdx.x;
  bool f[PG_PER];
  unsigned rank[PG_PER], live = 0, holes = 0;
  if (tid == 0) high = 0;
  auto scan = [&](auto wanted, auto take) {
    unsigned seen = 0;
    for (int base = 0; base < kv.n_pages; base += PG_STEP) {
#pragma unroll
      for (int i = 0; i < PG_PER; ++i) {
        const int p = base + i * PG_THREADS + tid;
        f[i] = p < kv.n_pages && wanted(p);
      }
      const unsigned n = page_scan(S, f, rank);
#pragma unroll
      for (int i = 0; i < PG_PER; ++i)
        if (f[i]) take(base + i * PG_THREADS + tid, seen + rank[i]);
      seen += n;
    }
    return seen;
  };
  live = scan([&](int p) { return to[p] = p, kv.refs[p] > 0; }, [](int, unsigned) {});
  holes = scan([&](int p) { return p < (int)live && kv.refs[p] <= 0; },
               [&](int p, unsigned i) {
                 if (i < (unsigned)max_pairs) dst[i] = p;
               });
  const unsigned moves = min(holes, (unsigned)max_pairs);
  scan([&](int p) { return p >= (int)live && kv.refs[p] > 0; },
       [&](int p, unsigned t) {
         const unsigned i = holes - 1u - t;  // as many pages are in use above as are free below
         if (i < moves) src[i] = p;
         if (i == moves) high = p + 1;
       });
  __syncthreads();
  for (unsigned i = tid; i < moves; i += PG_THREADS) {
    const int a = src[i], b = dst[i];
    to[a] = b;
    kv.refs[b] = kv.refs[a];
    kv.refs[a] = 0;
  }
  for (unsigned i = moves + tid; i < (unsigned)max_pairs; i += PG_THREADS) src[i] = dst[i] = -1;
  if (tid == 0) {
    counts[0] = (int)moves;
    counts[1] = (int)live;
    counts[2] = moves == holes ? (int)live : high;
  }
}
__global__ void __launch_bounds__(256) pages_renumber_kernel(const __grid_constant__ gsdlq_paged_kv_t kv,
                                                             const int* __restrict__ to) {
  const size_t n = (size_t)kv.n_seqs * kv.max_blocks;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
    const int p = kv.table[i];
    if (paged_valid(kv, p) && to[p] != p) kv.table[i] = to[p];
  }
}

// Pages: copy.  The pairs' pages of all layers are cut into pieces of COPY_PIECE 16-byte words, dealt to the
// CTAs in turn.
constexpr int COPY_THREADS = 256, COPY_PER = 4, COPY_PIECE = COPY_THREADS * COPY_PER;
__global__ void __launch_bounds__(COPY_THREADS) pages_copy_kernel(const __grid_constant__ gsdlq_paged_kv_t kv,
                                                                  const int* __restrict__ src,
                                                                  const int* __restrict__ dst,
                                                                  const int* __restrict__ counts, int max_pairs) {
  const int n = min(max(*counts, 0), max_pairs);
  const size_t words = (size_t)kv.page_size * kv.n_kv_heads * kv.head_dim / 8;  // of a page, one layer
  const size_t pieces = (words + COPY_PIECE - 1) / COPY_PIECE, per_pair = pieces * 2 * kv.layers;
  for (size_t c = blockIdx.x; c < (size_t)n * per_pair; c += gridDim.x) {
    const int i = (int)(c / per_pair);
    const size_t u = c - (size_t)i * per_pair, plane = u / pieces, piece = u - plane * pieces;
    const int a = src[i], b = dst[i];
    if (!paged_valid(kv, a) || !paged_valid(kv, b)) {
      if (threadIdx.x == 0) raise_flag(GSDLQ_FLAG_BAD_PAGE);
      continue;
    }
    uint4* pool = reinterpret_cast<uint4*>(plane & 1 ? kv.v : kv.k) + (plane >> 1) * kv.n_pages * words;
    const uint4* from = pool + a * words;
    uint4* into = pool + b * words;
    uint4 w[COPY_PER];
#pragma unroll
    for (int k = 0; k < COPY_PER; ++k) {
      const size_t e = piece * COPY_PIECE + k * COPY_THREADS + threadIdx.x;
      if (e < words) w[k] = from[e];
    }
#pragma unroll
    for (int k = 0; k < COPY_PER; ++k) {
      const size_t e = piece * COPY_PIECE + k * COPY_THREADS + threadIdx.x;
      if (e < words) into[e] = w[k];
    }
  }
}

// ---------------------------------------------------------------------------------------
// host checks
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
static bool pages_ok(const gsdlq_paged_kv_t& kv) {  // table and counts
  return kv.table && kv.refs && kv.n_pages > 0 && kv.n_pages <= (1 << 28) && kv.page_size > 0 && kv.max_blocks > 0 && kv.n_seqs > 0 &&
         kv.n_seqs <= GSDLQ_PAGED_MAX_SEQS;
}
static bool pool_ok(const gsdlq_paged_kv_t& kv) {  // and the pool itself
  return pages_ok(kv) && kv.k && kv.v && aligned16(kv.k) && aligned16(kv.v) && kv.layers > 0 && kv.n_kv_heads > 0 &&
         (kv.kv_type == GSDLQ_KV_F16 || kv.kv_type == GSDLQ_KV_BF16) &&
         (kv.head_dim == 32 || kv.head_dim == 64 || kv.head_dim == 128);
}
static bool rows_ok(const gsdlq_paged_kv_t& kv, const int* row_seq, const int* pos, int rows) {
  return pos && rows > 0 && (row_seq || rows <= kv.n_seqs);
}

}  // namespace gsdlq

using namespace gsdlq;

extern "C" {

int gsdlq_rope_kv_paged(const gsdlq_paged_append_job_t* job, gsdlq_stream_t stream) {
  if (!job || !pool_ok(job->kv) || !rows_ok(job->kv, job->row_seq, job->pos, job->rows)) return GSDLQ_ERR_INVALID;
  const gsdlq_paged_append_job_t& J = *job;
  if (!J.q || !J.k || !J.v || !J.q_out || !J.rope_cs || J.max_pos <= 0 || J.n_heads <= 0) return GSDLQ_ERR_INVALID;
  if (J.layer < 0 || J.layer >= J.kv.layers) return GSDLQ_ERR_INVALID;
  const long long qw = (long long)J.n_heads * J.kv.head_dim, kw = (long long)J.kv.n_kv_heads * J.kv.head_dim;
  if (qw > INT32_MAX || kw > INT32_MAX) return GSDLQ_ERR_INVALID;
  if ((J.q_stride && J.q_stride < qw) || (J.q_out_stride && J.q_out_stride < qw) || (J.kv_stride && J.kv_stride < kw))
    return GSDLQ_ERR_INVALID;
  if (J.q == J.q_out && J.q_stride != J.q_out_stride) return GSDLQ_ERR_INVALID;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (J.kv.kv_type == GSDLQ_KV_BF16)
    rope_kv_paged_kernel<true><<<J.rows, 256, 0, st>>>(J);
  else
    rope_kv_paged_kernel<false><<<J.rows, 256, 0, st>>>(J);
  GSDLQ_CUDA_CHECK_LAUNCH();
  return GSDLQ_OK;
}

int gsdlq_attention_paged_work_size(int rows, int n_heads, int n_kv_heads, int head_dim, size_t* bytes) {
  if (!bytes || rows <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads) return GSDLQ_ERR_INVALID;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) return GSDLQ_ERR_INVALID;
  *bytes = attention_paged_work(rows, n_heads, n_kv_heads, head_dim);
  return GSDLQ_OK;
}

int gsdlq_attention_paged(const gsdlq_paged_attn_job_t* job, gsdlq_stream_t stream) {
  if (!job || !pool_ok(job->kv) || !rows_ok(job->kv, job->row_seq, job->pos, job->rows)) return GSDLQ_ERR_INVALID;
  const gsdlq_paged_attn_job_t& J = *job;
  if (!J.q || !J.out || !J.work || J.layer < 0 || J.layer >= J.kv.layers) return GSDLQ_ERR_INVALID;
  if (J.n_heads <= 0 || J.n_heads % J.kv.n_kv_heads || (long long)J.n_heads * J.kv.head_dim > INT32_MAX)
    return GSDLQ_ERR_INVALID;
  if (!aligned16(J.q) || !aligned16(J.out) || !aligned16(J.work) || J.q_stride % 4) return GSDLQ_ERR_INVALID;
  if (J.q_stride && J.q_stride < J.n_heads * J.kv.head_dim) return GSDLQ_ERR_INVALID;
  if (J.work_bytes < attention_paged_work(J.rows, J.n_heads, J.kv.n_kv_heads, J.kv.head_dim)) return GSDLQ_ERR_INVALID;
  const long long items = (long long)J.rows * J.n_heads;
  if ((items + 3) / 4 > INT32_MAX) return GSDLQ_ERR_INVALID;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)((items + 3) / 4);
#define GSDLQ_PA(hd)                                                    \
  if (J.kv.kv_type == GSDLQ_KV_BF16)                                    \
    attention_paged_kernel<hd, true><<<grid, 128, 0, st>>>(J);          \
  else                                                                  \
    attention_paged_kernel<hd, false><<<grid, 128, 0, st>>>(J)
  switch (J.kv.head_dim) {
    case 32: GSDLQ_PA(32); break;
    case 64: GSDLQ_PA(64); break;
    default: GSDLQ_PA(128); break;
  }
#undef GSDLQ_PA
  GSDLQ_CUDA_CHECK_LAUNCH();
  return GSDLQ_OK;
}

int gsdlq_pages_fork(const gsdlq_paged_kv_t* kv, const int* parent, gsdlq_stream_t stream) {
  if (!kv || !pages_ok(*kv) || !parent) return GSDLQ_ERR_INVALID;
  // columns of a CTA: 32 (whole 128-byte lines) while the tile of all sequences fits 48 KB, else 8
  const int cols = kv->n_seqs <= 384 ? 32 : 8;
  const unsigned grid = ((unsigned)kv->max_blocks + cols - 1) / cols;
  pages_fork_kernel<<<grid, 256, sizeof(int) * (size_t)kv->n_seqs * cols, static_cast<cudaStream_t>(stream)>>>(*kv, parent,
                                                                                                          cols);
  GSDLQ_CUDA_CHECK_LAUNCH();
  return GSDLQ_OK;
}

int gsdlq_pages_reserve(const gsdlq_paged_kv_t* kv, const int* row_seq, const int* pos, int rows, int* src, int* dst,
                        int max_pairs, int* counts, gsdlq_stream_t stream) {
  if (!kv || !pages_ok(*kv) || !rows_ok(*kv, row_seq, pos, rows) || rows > GSDLQ_PAGED_MAX_SEQS) return GSDLQ_ERR_INVALID;
  if (!src || !dst || !counts || max_pairs < rows) return GSDLQ_ERR_INVALID;
  pages_reserve_kernel<<<1, PG_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(*kv, row_seq, pos, rows, src, dst,
                                                                               max_pairs, counts);
  GSDLQ_CUDA_CHECK_LAUNCH();
  return GSDLQ_OK;
}

int gsdlq_pages_compact(const gsdlq_paged_kv_t* kv, int* src, int* dst, int max_pairs, int* counts, void* work,
                        size_t work_bytes, gsdlq_stream_t stream) {
  if (!kv || !pages_ok(*kv) || !src || !dst || !counts || max_pairs <= 0 || !work) return GSDLQ_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(work) & 3u) || work_bytes < sizeof(int) * (size_t)kv->n_pages) return GSDLQ_ERR_INVALID;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  pages_compact_kernel<<<1, PG_THREADS, 0, st>>>(*kv, src, dst, max_pairs, counts, static_cast<int*>(work));
  GSDLQ_CUDA_CHECK_LAUNCH();
  const size_t n = (size_t)kv->n_seqs * kv->max_blocks;
  pages_renumber_kernel<<<(unsigned)std::min<size_t>((n + 255) / 256, 1184), 256, 0, st>>>(*kv, static_cast<int*>(work));
  GSDLQ_CUDA_CHECK_LAUNCH();
  return GSDLQ_OK;
}

int gsdlq_pages_copy(const gsdlq_paged_kv_t* kv, const int* src, const int* dst, const int* counts, int max_pairs,
                     gsdlq_stream_t stream) {
  if (!kv || !pool_ok(*kv) || !src || !dst || !counts || max_pairs <= 0) return GSDLQ_ERR_INVALID;
  pages_copy_kernel<<<num_sms() * 8, COPY_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(*kv, src, dst, counts,
                                                                                          max_pairs);
  GSDLQ_CUDA_CHECK_LAUNCH();
  return GSDLQ_OK;
}

}  // extern "C"
