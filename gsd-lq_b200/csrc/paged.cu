// paged.cu -- a batch of sequences over one pool of K/V pages: RoPE + append, and the pages' own operations
// (fork, reserve, compact, copy); their attention is in paged_attn.cu.  No reference counterpart: the reference
// keeps one contiguous cache (gsd_lq_cpu_engine.c:186-330); the per-row arithmetic is that of its functions.
#include <algorithm>
#include <cstdint>

#include "paged.cuh"

namespace gsdlq {

template <bool BF16>
__device__ __forceinline__ uint16_t kv_round(float v) {
  return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : f2h(v);
}

// ---------------------------------------------------------------------------------------
// RoPE + append.  A thread per pair of one of the row's heads: query heads, then key heads, then value heads.  Few rows
// are bound by the chain of look-ups (position, then angle and page, then the page's count), so no thread does more than
// one pair, and q does not wait for the page: 1.6 us for one row of 32 + 8 + 8 heads of 128 (4.4 with a CTA per row).
// Many rows are bound by the number of threads, each with look-ups of its own: 1.6 us and 1.5 us for each thousand CTAs,
// 3.8 us for 128 rows of 32 + 32 + 32 heads of 64 (1536 CTAs; 4.6 with a CTA per row).
constexpr int RK_THREADS = 256;
template <bool BF16>
__global__ void __launch_bounds__(RK_THREADS)
    rope_kv_paged_kernel(const __grid_constant__ gsdlq_paged_append_job_t J, int parts, int half_shift) {
  pdl_wait();
  const gsdlq_paged_kv_t& kv = J.kv;
  const int r = blockIdx.x / parts, e = (blockIdx.x - r * parts) * RK_THREADS + threadIdx.x;
  const int half = 1 << half_shift, hd = 2 * half, h = e >> half_shift, i = e & (half - 1);
  if (h >= J.n_heads + 2 * kv.n_kv_heads) return;
  PagedRow row = paged_row(kv, J.row_seq, J.pos, r, e == 0);
  if (row.len > J.max_pos) {
    if (e == 0) raise_flag(GSDLQ_FLAG_BAD_POS);
    row.len = 0;
  }
  const int pos = row.len - 1;
  const int i0 = J.interleaved ? 2 * i : i, i1 = J.interleaved ? 2 * i + 1 : i + half;
  const float2* const cs = reinterpret_cast<const float2*>(J.rope_cs) + (size_t)pos * half + i;
  if (h < J.n_heads) {
    const size_t qw = (size_t)J.n_heads * hd;
    const float* const q = J.q + r * (J.q_stride ? (size_t)J.q_stride : qw) + (size_t)h * hd;
    float* const out = J.q_out + r * (J.q_out_stride ? (size_t)J.q_out_stride : qw) + (size_t)h * hd;
    float x = q[i0], y = q[i1];
    if (row.len > 0) {
      const float2 c = *cs;
      const float a = x, b = y;
      x = __fsub_rn(__fmul_rn(a, c.x), __fmul_rn(b, c.y));
      y = __fadd_rn(__fmul_rn(a, c.y), __fmul_rn(b, c.x));
    }
    out[i0] = x;
    out[i1] = y;
    return;
  }
  if (row.len == 0) return;
  const bool is_v = h >= J.n_heads + kv.n_kv_heads;
  const int g = h - J.n_heads - (is_v ? kv.n_kv_heads : 0);
  const size_t kw = (size_t)kv.n_kv_heads * hd;
  const float* const in = (is_v ? J.v : J.k) + r * (J.kv_stride ? (size_t)J.kv_stride : kw) + (size_t)g * hd;
  float x = in[i0], y = in[i1];
  if (!is_v) {
    const float2 c = *cs;
    const float a = x, b = y;
    x = __fsub_rn(__fmul_rn(a, c.x), __fmul_rn(b, c.y));
    y = __fadd_rn(__fmul_rn(a, c.y), __fmul_rn(b, c.x));
  }
  const int block = pos / kv.page_size, page = kv.table[(size_t)row.seq * kv.max_blocks + block];
  if (!paged_valid(kv, page) || kv.refs[page] != 1) {
    if (i == 0 && g == 0) raise_flag(GSDLQ_FLAG_BAD_PAGE);
    return;
  }
  const size_t at = (((size_t)J.layer * kv.n_pages + page) * kv.page_size + (pos - block * kv.page_size)) * kw + (size_t)g * hd;
  uint16_t* const to = static_cast<uint16_t*>(is_v ? kv.v : kv.k) + at;
  to[i0] = kv_round<BF16>(x);
  to[i1] = kv_round<BF16>(y);
}

// ---------------------------------------------------------------------------------------
// Pages: fork.  A CTA owns FORK_COLS columns of the table (whole 32-byte sectors): it reads them whole, then writes
// the entries that change and moves their counts.  The counts are integers, so the order of the atomics does not
// show.  1.5 us for 64 sequences of 33 blocks, bound by its two dependent reads (5.3 us with 32 columns a CTA).
constexpr int FORK_COLS = 8, FORK_THREADS = 512, FORK_ROWS = FORK_THREADS / FORK_COLS;
__global__ void __launch_bounds__(FORK_THREADS) pages_fork_kernel(const __grid_constant__ gsdlq_paged_kv_t kv,
                                                                  const int* __restrict__ parent) {
  __shared__ int tile[GSDLQ_PAGED_MAX_SEQS][FORK_COLS];
  pdl_wait();
  const int c = threadIdx.x % FORK_COLS, b0 = threadIdx.x / FORK_COLS, col = blockIdx.x * FORK_COLS + c;
  constexpr int UN = 4;  // rows in flight
  for (int b = b0; b < kv.n_seqs; b += UN * FORK_ROWS) {
    int e[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i)
      if (b + i * FORK_ROWS < kv.n_seqs && col < kv.max_blocks)
        e[i] = kv.table[(size_t)(b + i * FORK_ROWS) * kv.max_blocks + col];
#pragma unroll
    for (int i = 0; i < UN; ++i)
      if (b + i * FORK_ROWS < kv.n_seqs && col < kv.max_blocks) tile[b + i * FORK_ROWS][c] = e[i];
  }
  int p[UN];  // the first rows' parents, before the barrier
#pragma unroll
  for (int i = 0; i < UN; ++i) p[i] = b0 + i * FORK_ROWS < kv.n_seqs ? parent[b0 + i * FORK_ROWS] : 0;
  __syncthreads();
  if (col >= kv.max_blocks) return;
  for (int b = b0; b < kv.n_seqs; b += UN * FORK_ROWS) {
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int r = b + i * FORK_ROWS;
      if (r >= kv.n_seqs) break;
      const int from = b == b0 ? p[i] : parent[r];
      if (from < -1 || from >= kv.n_seqs) {
        if (col == 0) raise_flag(GSDLQ_FLAG_BAD_PAGE);
        continue;
      }
      const int was = tile[r][c], now = from < 0 ? -1 : tile[from][c];
      if (was == now) continue;
      kv.table[(size_t)r * kv.max_blocks + col] = now;
      if (paged_valid(kv, was)) atomicAdd(&kv.refs[was], -1);
      if (paged_valid(kv, now)) atomicAdd(&kv.refs[now], 1);
    }
  }
}

// ---------------------------------------------------------------------------------------
// Block-wide scans over the pages' counts, 1024 threads: PG_PER consecutive pages a thread and step.
constexpr int PG_THREADS = 1024, PG_WARPS = PG_THREADS / 32, PG_PER = 16, PG_STEP = PG_THREADS * PG_PER;
// Exclusive sum of n over the block's threads, and the total.  `turn` alternates between calls, so that one
// barrier a call is enough.
__device__ __forceinline__ unsigned page_sum(unsigned (&sums)[2][PG_WARPS], int& turn, unsigned n, unsigned& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned inc = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  if (lane == 31) sums[turn][warp] = inc;
  __syncthreads();
  unsigned w = sums[turn][lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned x = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += x;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const unsigned before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  turn ^= 1;
  return (warp > 0 ? before : 0u) + inc - n;
}
// the counts of pages base .. base + PG_PER - 1 (0 past the end: neither in use nor, by `in`, free)
__device__ __forceinline__ void page_counts(const gsdlq_paged_kv_t& kv, int base, int (&r)[PG_PER], unsigned& in) {
  if (base + PG_PER <= kv.n_pages && (reinterpret_cast<uintptr_t>(kv.refs) & 15u) == 0u) {
#pragma unroll
    for (int i = 0; i < PG_PER; i += 4) *reinterpret_cast<int4*>(r + i) = *reinterpret_cast<const int4*>(kv.refs + base + i);
    in = (1u << PG_PER) - 1u;
  } else {
    in = 0u;
#pragma unroll
    for (int i = 0; i < PG_PER; ++i) {
      const bool ok = base + i < kv.n_pages;
      r[i] = ok ? kv.refs[base + i] : 0;
      in |= (unsigned)ok << i;
    }
  }
}

// Pages: reserve.  One CTA, thread r = row r.  The rows act in order, so a row that shares its page with
// `before` earlier rows of the call finds refs - before entries on it when its turn comes: it takes a copy
// while that is more than one, and the last holder keeps the page.  Two rows at one table entry: the first
// one acts.  Latency bound: about 2 us where every row has a page of its own (the usual step), 5-6 us where 64 rows
// take pages, of which the chain position -> table -> counts is 2.
__global__ void __launch_bounds__(PG_THREADS) pages_reserve_kernel(const __grid_constant__ gsdlq_paged_kv_t kv,
                                                                   const int* __restrict__ row_seq,
                                                                   const int* __restrict__ pos, int rows, int* src,
                                                                   int* dst, int max_pairs, int* counts) {
  __shared__ long long slot[GSDLQ_PAGED_MAX_SEQS];
  __shared__ int page[GSDLQ_PAGED_MAX_SEQS], fresh[GSDLQ_PAGED_MAX_SEQS];
  __shared__ bool failed[GSDLQ_PAGED_MAX_SEQS];
  __shared__ unsigned sums[2][PG_WARPS];
  pdl_wait();
  const int r = threadIdx.x;
  int turn = 0;
  int c[PG_PER];  // the first pages' counts, on their way while the rows are looked up
  unsigned in;
  page_counts(kv, r * PG_PER, c, in);
  long long my_slot = -1;
  int my_page = -1, held = 0;
  if (r < rows) {
    const PagedRow row = paged_row(kv, row_seq, pos, r, true);
    if (row.len > 0) {
      my_slot = (long long)row.seq * kv.max_blocks + (row.len - 1) / kv.page_size;
      my_page = kv.table[my_slot];
      if (!paged_valid(kv, my_page)) {
        if (my_page != -1) raise_flag(GSDLQ_FLAG_BAD_PAGE);
        my_page = -1;
      } else {
        held = kv.refs[my_page];
      }
    }
  }
  // rows that may need a page: those of rows with one of their own need nothing, whatever the others do
  const bool open = my_slot >= 0 && (my_page < 0 || held > 1);
  unsigned wanted = 0, have = 0, pairs = 0, mine = 0;
  int short_of = 0;
  if (__syncthreads_or(open)) {
    if (r < rows) {
      slot[r] = my_slot;
      page[r] = -1;
      failed[r] = false;
    }
    __syncthreads();
    bool acts = open;
    if (row_seq != nullptr && open)  // (without it every row has a sequence of its own)
#pragma unroll 8
      for (int i = 0; i < r; ++i) acts = acts && slot[i] != my_slot;
    if (acts) page[r] = my_page;  // shared pages only, and of rows that act
    __syncthreads();
    int before = 0;
    if (acts && my_page >= 0)
#pragma unroll 8
      for (int i = 0; i < r; ++i) before += page[i] == my_page;
    const bool need = acts && (my_page < 0 || held - before > 1);
    mine = page_sum(sums, turn, need, wanted);
    // the lowest free pages
    for (int base = 0; base < kv.n_pages && have < wanted; base += PG_STEP) {
      unsigned n;
      if (base > 0) page_counts(kv, base + r * PG_PER, c, in);
#pragma unroll
      for (int i = 0; i < PG_PER; ++i)
        if (c[i] > 0) in &= ~(1u << i);
      unsigned at = have + page_sum(sums, turn, __popc(in), n);
      for (; in != 0u && at < wanted; in &= in - 1u) fresh[at++] = base + r * PG_PER + __ffs(in) - 1;
      have += n;
    }
    __syncthreads();  // fresh[] is complete, and every count has been read
    const bool got = need && mine < have, copies = got && my_page >= 0;
    const unsigned at = page_sum(sums, turn, copies, pairs);
    if (got) {
      const int p = fresh[mine];
      kv.table[my_slot] = p;
      kv.refs[p] = 1;
      if (copies) {
        atomicAdd(&kv.refs[my_page], -1);
        src[at] = my_page;
        dst[at] = p;
      }
    }
    if (have < wanted) {  // exhausted (uniform): the last holder of a page that an earlier row could not leave fails too
      bool fails = need && !got;
      if (r < rows) failed[r] = fails;
      __syncthreads();
      if (acts && !need && before > 0)
        for (int i = 0; i < r; ++i) fails |= page[i] == my_page && failed[i];
      if (fails) raise_flag(GSDLQ_FLAG_NO_PAGE);
      short_of = __syncthreads_count(fails);
    }
  }
  for (int i = pairs + r; i < max_pairs; i += PG_THREADS) src[i] = dst[i] = -1;
  if (r == 0) {
    counts[0] = (int)pairs;
    counts[1] = short_of;
    counts[2] = (int)min(wanted, have);
  }
}

// Pages: compact.  One CTA plans: the number of pages in use, then the free pages below it in ascending
// order against the pages in use at and above it in descending order; `to` maps old to new pages.  Which pages are
// in use is kept as bits in shared memory (of pools up to PG_KEPT * PG_STEP pages).  A table of up to PG_TABLE
// entries is rewritten by the same CTA, a larger one by pages_renumber_kernel.  One CTA: 4 us for 2,300 pages, 22 us
// for 100,000, beside copies of some 60 us and more.
constexpr int PG_KEPT = 16, PG_TABLE = 8192;
__device__ __forceinline__ void pages_renumber(const gsdlq_paged_kv_t& kv, const int* to, size_t i, size_t step) {
  const size_t n = (size_t)kv.n_seqs * kv.max_blocks;
  for (; i < n; i += step) {
    const int p = kv.table[i];
    if (paged_valid(kv, p)) {
      const int q = to[p];
      if (q != p) kv.table[i] = q;
    }
  }
}
__global__ void __launch_bounds__(PG_THREADS) pages_compact_kernel(const __grid_constant__ gsdlq_paged_kv_t kv, int* src,
                                                                   int* dst, int max_pairs, int* counts, int* to) {
  __shared__ unsigned sums[2][PG_WARPS];
  __shared__ unsigned short kept[PG_KEPT][PG_THREADS];
  __shared__ int high;
  pdl_wait();
  const int tid = threadIdx.x, steps = (kv.n_pages + PG_STEP - 1) / PG_STEP;
  int turn = 0;
  if (tid == 0) high = 0;
  // pages base .. base + PG_PER - 1 of step k: in use, and in the pool
  auto used = [&](int k, bool again, unsigned& in) -> unsigned {
    const int base = (k * PG_THREADS + tid) * PG_PER, left = kv.n_pages - base;
    in = left >= PG_PER ? (1u << PG_PER) - 1u : left > 0 ? (1u << left) - 1u : 0u;
    if (again && k < PG_KEPT) return kept[k][tid];
    int c[PG_PER];
    unsigned ok, m = 0u;
    page_counts(kv, base, c, ok);
#pragma unroll
    for (int i = 0; i < PG_PER; ++i) m |= (unsigned)(c[i] > 0) << i;
    if (k < PG_KEPT) kept[k][tid] = (unsigned short)m;
    return m;
  };
  unsigned live = 0, in, n;
  for (int k = 0; k < steps; ++k) live += __popc(used(k, false, in));
  for (int p = tid; p < kv.n_pages; p += PG_THREADS) to[p] = p;
  page_sum(sums, turn, live, n);
  live = n;
  // free pages below `live`, and pages in use at and above it: as many of the one as of the other
  unsigned holes = 0, tails = 0;
  auto below = [&](int base) -> unsigned {  // those of base .. that lie below `live`
    const int left = (int)live - base;
    return left >= PG_PER ? (1u << PG_PER) - 1u : left > 0 ? (1u << left) - 1u : 0u;
  };
  for (int k = 0; k * PG_STEP < (int)live; ++k) {
    const int base = (k * PG_THREADS + tid) * PG_PER;
    unsigned m = ~used(k, true, in);
    m &= in & below(base);
    unsigned at = holes + page_sum(sums, turn, __popc(m), n);
    for (; m != 0u && at < (unsigned)max_pairs; m &= m - 1u) dst[at++] = base + __ffs(m) - 1;
    holes += n;
  }
  const unsigned moves = min(holes, (unsigned)max_pairs);
  for (int k = (int)(live / PG_STEP); k < steps && holes > 0; ++k) {
    const int base = (k * PG_THREADS + tid) * PG_PER;
    unsigned m = used(k, true, in) & ~below(base);
    unsigned t = tails + page_sum(sums, turn, __popc(m), n);
    for (; m != 0u; m &= m - 1u, ++t) {
      const unsigned i = holes - 1u - t;
      const int p = base + __ffs(m) - 1;
      if (i < moves) src[i] = p;
      if (i == moves) high = p + 1;
    }
    tails += n;
  }
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
  if ((long long)kv.n_seqs * kv.max_blocks <= PG_TABLE) {
    __syncthreads();  // `to` is complete
    pages_renumber(kv, to, tid, PG_THREADS);
  }
}
__global__ void __launch_bounds__(256) pages_renumber_kernel(const __grid_constant__ gsdlq_paged_kv_t kv, const int* to) {
  pdl_wait();
  pages_renumber(kv, to, (size_t)blockIdx.x * 256 + threadIdx.x, (size_t)gridDim.x * 256);
}

// Pages: copy.  The planes (layer, K or V) of the pairs' pages are cut into pieces of at most COPY_PIECE 16-byte
// words, dealt to the CTAs in turn; the next piece's pair is looked up while a piece is copied.  Bound by HBM: 5.8 TB/s
// read and written for 448 pages of 28 layers x 2 x 8 KB, 6.9 TB/s for 32 pages of 32 layers x 2 x 32 KB (some of it
// from L2); other shapes of the pieces and 16 CTAs an SM are within 3 %.
constexpr int COPY_THREADS = 128, COPY_PER = 4, COPY_PIECE = COPY_THREADS * COPY_PER;
constexpr int COPY_PER_SM = 8;
struct CopyPlan {
  unsigned words;                   // of a plane of a page
  unsigned pieces, per_pair;        // of a plane; of a page
  unsigned step_pair, step_piece;   // from a CTA's piece to its next one: pairs, and pieces of them
};
__global__ void __launch_bounds__(COPY_THREADS, COPY_PER_SM)
    pages_copy_kernel(const __grid_constant__ gsdlq_paged_kv_t kv, const __grid_constant__ CopyPlan P,
                      const int* __restrict__ src, const int* __restrict__ dst, const int* __restrict__ counts,
                      int max_pairs) {
  pdl_wait();
  const int n = min(max(*counts, 0), max_pairs);
  unsigned i = blockIdx.x / P.per_pair, u = blockIdx.x % P.per_pair;
  int a = -1, b = -1;
  if (i < (unsigned)n) {
    a = src[i];
    b = dst[i];
  }
  while (i < (unsigned)n) {
    const unsigned plane = u / P.pieces, e0 = (u - plane * P.pieces) * COPY_PIECE + threadIdx.x;
    const bool ok = paged_valid(kv, a) && paged_valid(kv, b);
    uint4 w[COPY_PER];
    uint4* const pool = reinterpret_cast<uint4*>(plane & 1 ? kv.v : kv.k) + (size_t)(plane >> 1) * kv.n_pages * P.words;
    if (ok) {
      const uint4* const from = pool + (size_t)a * P.words;
#pragma unroll
      for (int k = 0; k < COPY_PER; ++k)
        if (e0 + k * COPY_THREADS < P.words) w[k] = __ldcs(from + e0 + k * COPY_THREADS);
    } else if (threadIdx.x == 0) {
      raise_flag(GSDLQ_FLAG_BAD_PAGE);
    }
    uint4* const into = pool + (size_t)b * P.words;
    i += P.step_pair;
    u += P.step_piece;
    if (u >= P.per_pair) {
      u -= P.per_pair;
      ++i;
    }
    if (i < (unsigned)n) {
      a = src[i];
      b = dst[i];
    }
    if (ok) {
#pragma unroll
      for (int k = 0; k < COPY_PER; ++k)
        if (e0 + k * COPY_THREADS < P.words) __stcs(into + e0 + k * COPY_THREADS, w[k]);
    }
  }
}

}  // namespace gsdlq

using namespace gsdlq;

extern "C" {

int gsdlq_rope_kv_paged(const gsdlq_paged_append_job_t* job, gsdlq_stream_t stream) {
  if (!job || !pool_ok(job->kv) || !rows_ok(job->kv, job->row_seq, job->pos, job->rows)) return GSDLQ_ERR_INVALID;
  const gsdlq_paged_append_job_t& J = *job;
  if (!J.q || !J.k || !J.v || !J.q_out || !J.rope_cs || J.max_pos <= 0 || J.n_heads <= 0) return GSDLQ_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(J.rope_cs) & 7u) return GSDLQ_ERR_INVALID;  // read in pairs
  if (J.layer < 0 || J.layer >= J.kv.layers) return GSDLQ_ERR_INVALID;
  const long long qw = (long long)J.n_heads * J.kv.head_dim, kw = (long long)J.kv.n_kv_heads * J.kv.head_dim;
  if (qw > INT32_MAX / 4 || kw > INT32_MAX / 4) return GSDLQ_ERR_INVALID;
  if ((J.q_stride && J.q_stride < qw) || (J.q_out_stride && J.q_out_stride < qw) || (J.kv_stride && J.kv_stride < kw))
    return GSDLQ_ERR_INVALID;
  if (J.q == J.q_out && (J.q_stride ? J.q_stride : qw) != (J.q_out_stride ? J.q_out_stride : qw)) return GSDLQ_ERR_INVALID;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int half_shift = J.kv.head_dim == 128 ? 6 : J.kv.head_dim == 64 ? 5 : 4;
  const long long parts = ((qw + 2 * kw) / 2 + RK_THREADS - 1) / RK_THREADS;
  if (J.rows * parts > INT32_MAX) return GSDLQ_ERR_UNSUPPORTED;
  return launch_pdl(J.kv.kv_type == GSDLQ_KV_BF16 ? rope_kv_paged_kernel<true> : rope_kv_paged_kernel<false>,
                    (unsigned)(J.rows * parts), RK_THREADS, 0, st, 1, J, (int)parts, half_shift);
}

int gsdlq_pages_fork(const gsdlq_paged_kv_t* kv, const int* parent, gsdlq_stream_t stream) {
  if (!kv || !pages_ok(*kv) || !parent) return GSDLQ_ERR_INVALID;
  const unsigned grid = ((unsigned)kv->max_blocks + FORK_COLS - 1) / FORK_COLS;
  return launch_pdl(pages_fork_kernel, grid, FORK_THREADS, 0, static_cast<cudaStream_t>(stream), 1, *kv, parent);
}

int gsdlq_pages_reserve(const gsdlq_paged_kv_t* kv, const int* row_seq, const int* pos, int rows, int* src, int* dst,
                        int max_pairs, int* counts, gsdlq_stream_t stream) {
  if (!kv || !pages_ok(*kv) || !rows_ok(*kv, row_seq, pos, rows) || rows > GSDLQ_PAGED_MAX_SEQS) return GSDLQ_ERR_INVALID;
  if (!src || !dst || !counts || max_pairs < rows) return GSDLQ_ERR_INVALID;
  return launch_pdl(pages_reserve_kernel, 1, PG_THREADS, 0, static_cast<cudaStream_t>(stream), 1, *kv, row_seq, pos,
                    rows, src, dst, max_pairs, counts);
}

int gsdlq_pages_compact(const gsdlq_paged_kv_t* kv, int* src, int* dst, int max_pairs, int* counts, void* work,
                        size_t work_bytes, gsdlq_stream_t stream) {
  if (!kv || !pages_ok(*kv) || !src || !dst || !counts || max_pairs <= 0 || !work) return GSDLQ_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(work) & 3u) || work_bytes < sizeof(int) * (size_t)kv->n_pages) return GSDLQ_ERR_INVALID;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int status = launch_pdl(pages_compact_kernel, 1, PG_THREADS, 0, st, 1, *kv, src, dst, max_pairs, counts,
                                static_cast<int*>(work));
  if (status != GSDLQ_OK) return status;
  const size_t n = (size_t)kv->n_seqs * kv->max_blocks;
  if (n <= PG_TABLE) return GSDLQ_OK;
  return launch_pdl(pages_renumber_kernel, (unsigned)std::min<size_t>((n + 255) / 256, 1184), 256, 0, st, 1, *kv,
                    static_cast<const int*>(work));
}

int gsdlq_pages_copy(const gsdlq_paged_kv_t* kv, const int* src, const int* dst, const int* counts, int max_pairs,
                     gsdlq_stream_t stream) {
  if (!kv || !pool_ok(*kv) || !src || !dst || !counts || max_pairs <= 0) return GSDLQ_ERR_INVALID;
  const unsigned long long words = (unsigned long long)kv->page_size * kv->n_kv_heads * kv->head_dim / 8;
  const unsigned long long per_pair = (words + COPY_PIECE - 1) / COPY_PIECE * 2 * kv->layers;
  if (words > UINT32_MAX / 2 || per_pair > INT32_MAX) return GSDLQ_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)num_sms() * COPY_PER_SM, pp = (unsigned)per_pair;
  const CopyPlan P = {(unsigned)words, (unsigned)((words + COPY_PIECE - 1) / COPY_PIECE), pp, grid / pp, grid % pp};
  return launch_pdl(pages_copy_kernel, grid, COPY_THREADS, 0, static_cast<cudaStream_t>(stream), 1, *kv, P, src, dst,
                    counts, max_pairs);
}

}  // extern "C"
