// paged.cu -- a batch of sequences over one pool of K/V pages: RoPE + append, decode attention, and the
// pages' own operations (fork, reserve, compact, copy).  No reference counterpart: the reference keeps
// one contiguous cache (gsd_lq_cpu_engine.c:186-330); the per-row arithmetic is that of its functions.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>

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

// ---------------------------------------------------------------------------------------
// RoPE + append.  A thread per pair of one of the row's heads: query heads, then key heads, then value heads.  The
// chain of look-ups (position, then angle and page, then the page's count) bounds it, so no thread does more than
// one pair, and q does not wait for the page.
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
// Attention.  An item is a row and up to eight query heads of one kv head; its positions are cut into units of
// PA_TOK.  All units of the launch, row by row, item by item, are dealt to the CTAs in equal contiguous runs,
// whatever the rows' lengths are (they are known on the device only); an item counts some units more, for what
// it costs besides its positions.  A short item that lies whole inside a run is taken by one warp, the next one by
// the next warp; of any other item the warps take the units in turn, and merge through shared memory where it
// ends.  An item that several CTAs share is joined by the CTA that arrives last, in the order of the CTAs, so
// that the result does not depend on who that is.
//
// Each warp has a K and a V tile of its own (cp.async, no CTA-wide barrier in the loop): the next unit's K is on its
// way while the weights and the second product are worked on, its V during the next first product.  Twelve such
// warps an SM keep more bytes in flight and more instructions to choose from than eight with three tiles each.
//
// Both products run on mma.m16n8k16 with the 16-bit cache values as they are, so K and V go from shared
// memory to the matrix unit without a conversion.  q and the weights p are fp32 and enter as parts of 16 bits:
//   fp16: q = 2^-e (hi + lo), p 2^11 = hi + lo, about 22 bits: rows 0-7 of A hold the heads' hi, rows 8-15 their lo
//   bf16: hi + mid + lo, 24 bits: hi and mid in the two halves of one A, lo in the lower half of another
// so that one product gives both parts and c[0] + c[2], c[1] + c[3] are the sums.  With A = q, B = K^T the score
// fragment is already p's A fragment for the second product, B = V.  The second product starts from zero each
// unit and is added to fp32 registers, which keeps the tensor core's truncating accumulation short.
constexpr int PA_MAX_CTAS = 480;  // largest grid of an attention launch
constexpr int PA_PER_SM = 2;
constexpr int PA_GROUP = 8;       // query heads of one kv head taken together
constexpr int PA_WARPS = 4, PA_THREADS = PA_WARPS * 32;
constexpr int PA_SHORT = 4;       // units of an item that one warp may take
// units that an item counts besides its own, for its queries, and for the merge of the warps where it has one
__host__ __device__ constexpr int pa_over(int tiles) { return tiles <= PA_SHORT ? 2 : 4; }

constexpr int pa_tok(int hd) { return hd == 128 ? 32 : 64; }  // positions of a unit

template <int HD>
struct PagedAttnSmem {
  uint8_t tile[PA_WARPS][2][pa_tok(HD) * HD * 2];  // K, V
  float acc[PA_WARPS][PA_GROUP][HD < 64 ? HD : 64];  // the warps' results of an item, 64 dimensions at a time
  float m[PA_WARPS][PA_GROUP], l[PA_WARPS][PA_GROUP];
  int warp_sum[PA_WARPS];
  int row, base, last;
};

inline size_t attention_paged_counters(int rows, int n_heads, int n_kv) {
  const size_t items = (size_t)rows * n_kv * ((n_heads / n_kv + PA_GROUP - 1) / PA_GROUP);
  return (items * sizeof(unsigned) + 15) / 16 * 16;
}
// counters of the items, then two partial results per CTA (its first and its last item)
inline size_t attention_paged_work(int rows, int n_heads, int n_kv, int hd) {
  return attention_paged_counters(rows, n_heads, n_kv) + sizeof(float) * (size_t)PA_MAX_CTAS * 2 * PA_GROUP * (hd + 2);
}

template <bool BF16>
__device__ __forceinline__ void pa_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                       const float (&c)[4]) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void pa_ldm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void pa_ldm_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void pa_cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void pa_cp16(uint32_t dst, const void* src, int bytes) {  // 16, or 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// (x, y) as parts of 16 bits: fp16 hi + lo, bf16 hi + mid + lo
template <bool BF16>
__device__ __forceinline__ void pa_split(float x, float y, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  if constexpr (BF16) {
    hi = pack_bf16x2(x, y);
    const float rx = x - bf16lo_to_f(hi), ry = y - bf16hi_to_f(hi);
    mid = pack_bf16x2(rx, ry);
    lo = pack_bf16x2(rx - bf16lo_to_f(mid), ry - bf16hi_to_f(mid));
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    mid = *reinterpret_cast<const uint32_t*>(&r);
    lo = 0u;
  }
}

// byte offset of 16-byte chunk c of position j in a tile: the chunk is moved by the position so that the eight
// rows of an ldmatrix fall in eight different bank groups
template <int HD>
__device__ __forceinline__ uint32_t pa_at(int j, int c) {
  constexpr int CH = HD / 8;
  const int x = CH >= 8 ? (j & 7) : ((j >> 1) & 3);
  return (uint32_t)(j * (HD * 2) + ((c ^ x) << 4));
}

// a walk over a CTA's run, segment by segment: the part of an item that lies in it
struct PagedWalk {
  int row, seq, len, tiles;  // tiles: units of each of the row's items
  int item, s;               // its first unit is the launch's unit s
  int a, b;                  // the segment is its units a .. b - 1
  int t, step;               // this warp's next unit of it, and how far apart they are
  unsigned long long load;   // what the warps have taken of short items, 16 bits each
  __device__ bool whole() const { return a == 0 && b == tiles; }
};

template <int HD, bool BF16>
__global__ void __launch_bounds__(PA_THREADS, PA_PER_SM)
    attention_paged_kernel(const __grid_constant__ gsdlq_paged_attn_job_t J, int subs, int page_shift) {
  constexpr int TOK = pa_tok(HD);
  constexpr int TILE = TOK * HD * 2;       // bytes of a tile
  constexpr int CH = HD / 8;               // 16-byte chunks of a position
  constexpr int KS = HD / 16;              // k steps of the first product
  constexpr int TPL = TOK / 32;            // positions a lane looks up
  constexpr float P_SHIFT = BF16 ? 0.f : 11.f;
  typedef typename std::conditional<TOK == 64, unsigned long long, unsigned>::type mask_t;  // a bit per position
  constexpr mask_t FULL = ~(mask_t)0;
  extern __shared__ __align__(1024) uint8_t pa_smem[];
  PagedAttnSmem<HD>& S = *reinterpret_cast<PagedAttnSmem<HD>*>(pa_smem);
  const gsdlq_paged_kv_t& kv = J.kv;
  const int tid = threadIdx.x, lane = tid & 31, cta = blockIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // (the same in all lanes, for the compiler to see)
  const int gq_all = J.n_heads / kv.n_kv_heads, items_row = kv.n_kv_heads * subs;
  const size_t kw = (size_t)kv.n_kv_heads * HD;
  auto row_tiles = [&](int len) { return (len + TOK - 1) / TOK; };
  auto row_units = [&](int len) { return len > 0 ? (row_tiles(len) + pa_over(row_tiles(len))) * items_row : 0; };

  pdl_wait();
  pdl_launch_dependents();

  // ---- the launch's units, this CTA's run of them, and the row where it begins
  int mine0 = 0, sum = 0;  // of this thread's first row; of all its rows
  for (int r = tid; r < J.rows; r += PA_THREADS) {
    const int n = row_units(paged_row(kv, J.row_seq, J.pos, r, cta == 0).len);
    if (r == tid) mine0 = n;
    sum += n;
  }
  auto scan = [&](int n, int& total) {  // exclusive, over the CTA
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (lane == 31) S.warp_sum[warp] = inc;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) {
      before += w < warp ? S.warp_sum[w] : 0;
      total += S.warp_sum[w];
    }
    return before + inc - n;
  };
  int units;
  const int base0 = scan(sum, units);  // with one row a thread, also where that row begins
  const int per = max((units + (int)gridDim.x - 1) / (int)gridDim.x, PA_WARPS);
  const long long v0l = (long long)per * cta;
  const int v0 = v0l < units ? (int)v0l : units, v1 = min(v0 + per, units);
  for (int r = cta; r < J.rows; r += gridDim.x)  // idle rows
    if (paged_row(kv, J.row_seq, J.pos, r, false).len == 0)
      for (int i = tid; i < J.n_heads * HD; i += PA_THREADS) J.out[(size_t)r * J.n_heads * HD + i] = 0.f;
  if (v0 >= v1) return;
  if (J.rows <= PA_THREADS) {
    if (base0 <= v0 && v0 < base0 + mine0) {
      S.row = tid;
      S.base = base0;
    }
  } else {
    int before = 0;
    for (int r0 = 0; before <= v0; r0 += PA_THREADS) {  // (ends: v0 < units)
      const int r = r0 + tid, n = r < J.rows ? row_units(paged_row(kv, J.row_seq, J.pos, r, false).len) : 0;
      int total;
      __syncthreads();  // the previous sums are read
      const int b = before + scan(n, total);
      if (b <= v0 && v0 < b + n) {
        S.row = r;
        S.base = b;
      }
      before += total;
    }
  }
  __syncthreads();

  auto enter = [&](PagedWalk& w, int row) {
    const PagedRow pr = paged_row(kv, J.row_seq, J.pos, row, false);
    w.row = row;
    w.seq = pr.seq;
    w.len = pr.len;
    w.tiles = row_tiles(pr.len);
  };
  auto begin = [&](PagedWalk& w) {
    enter(w, S.row);
    const int n = w.tiles + pa_over(w.tiles);
    w.item = (v0 - S.base) / n - 1;  // the one before the run's first
    w.s = S.base + (w.item + 1) * n - w.tiles;
    w.load = 0ull;
    w.t = w.b = 0;
  };
  auto advance = [&](PagedWalk& w) {  // to the next segment; false: the run is at its end
    do {
      const int end = w.s + w.tiles;
      if (++w.item >= items_row) {
        do {
          if (w.row + 1 >= J.rows) return false;
          enter(w, w.row + 1);
        } while (w.tiles == 0);
        w.item = 0;
      }
      w.s = end + pa_over(w.tiles);
      if (w.s >= v1) return false;
      w.a = max(v0 - w.s, 0);
      w.b = min(v1 - w.s, w.tiles);
    } while (w.a >= w.b);
    // one warp for a short item, the one with the least so far; only where there is work for the others
    const bool is_short = w.whole() && w.tiles <= PA_SHORT && w.tiles * 2 * PA_WARPS <= v1 - v0;
    w.step = is_short ? 1 : PA_WARPS;
    w.t = w.a + warp;
    if (is_short) {
      int who = 0;
      unsigned least = (unsigned)w.load & 0xffffu;
#pragma unroll
      for (int i = 1; i < PA_WARPS; ++i) {
        const unsigned x = (unsigned)(w.load >> (16 * i)) & 0xffffu;
        if (x < least) {
          least = x;
          who = i;
        }
      }
      // (every warp comes to the same answer; a share past 16 bits would cost balance, nothing else)
      w.load += (unsigned long long)(w.tiles + pa_over(w.tiles)) << (16 * who);
      w.t = who == warp ? 0 : w.b;
    }
    return true;
  };

  // ---- the tiles
  const uint16_t* const kp = static_cast<const uint16_t*>(kv.k) + (size_t)J.layer * kv.n_pages * kv.page_size * kw;
  const uint16_t* const vp = static_cast<const uint16_t*>(kv.v) + (size_t)J.layer * kv.n_pages * kv.page_size * kw;
  const uint32_t row_bytes = (uint32_t)kw * 2;
  const uint32_t kt = smem_u32(S.tile[warp][0]);
  struct Unit {            // where a unit's positions are
    int page[TPL], at[TPL];  // page (-1: none), position in it, of position lane + 32 i
    int head;                // kv head, -1: no unit
  };
  PagedWalk ahead;
  bool more = true;
  begin(ahead);
  PagedWalk cur = ahead;
  auto look = [&](Unit& U) {
    U.head = -1;
#pragma unroll
    for (int i = 0; i < TPL; ++i) U.page[i] = -1;
    while (more && ahead.t >= ahead.b) more = advance(ahead);
    if (!more) return;
    U.head = subs == 1 ? ahead.item : ahead.item / subs;
#pragma unroll
    for (int i = 0; i < TPL; ++i) {
      const int t = ahead.t * TOK + i * 32 + lane;
      if (t < ahead.len) {
        const int b = page_shift >= 0 ? t >> page_shift : t / kv.page_size;
        U.at[i] = t - b * kv.page_size;
        U.page[i] = kv.table[(size_t)ahead.seq * kv.max_blocks + b];
        if (U.page[i] < 0) U.page[i] = kv.n_pages;  // missing: reported below
      }
    }
    ahead.t += ahead.step;
  };
  // the unit's positions as places in the pool, -1: none
  auto resolve = [&](const Unit& U, int (&slot)[TPL]) -> mask_t {
    mask_t valid = 0;
#pragma unroll
    for (int i = 0; i < TPL; ++i) {
      const bool ok = paged_valid(kv, U.page[i]);
      if (!ok && U.page[i] != -1) raise_flag(GSDLQ_FLAG_BAD_PAGE);
      slot[i] = ok ? U.page[i] * kv.page_size + U.at[i] : -1;
      valid |= (mask_t)__ballot_sync(0xffffffffu, ok) << (32 * i);
    }
    return valid;
  };
  // chunk addresses differ by constants that are or-ed in below the tile's alignment: pa_at(j + 8 i, c) is
  // pa_at(j, c) + 16 HD i, and pa_at(j, c ^ d) is pa_at(j, c) ^ 16 d
  const uint32_t dst0 = kt + pa_at<HD>(lane / CH, lane % CH);
  auto copy = [&](const uint16_t* pool, int head, const int (&slot)[TPL], mask_t valid, int to) {
    if (head >= 0) {
      const char* const src = reinterpret_cast<const char*>(pool + (size_t)head * HD + (lane % CH) * 8);
      const uint32_t dst = dst0 + to * TILE;
#pragma unroll
      for (int it = 0; it < TOK * CH / 32; ++it) {
        constexpr int RI = 32 / CH;  // positions of a step; their bits of the position are below the lane's chunk's
        const int j = it * RI;
        const uint32_t x = CH >= 8 ? (uint32_t)((j & 7) << 4) : (uint32_t)(((j >> 1) & 3) << 4);
        const int p = __shfl_sync(0xffffffffu, slot[j / 32], (j & 31) + lane / CH);
        const uint32_t d = (dst ^ x) + j * (HD * 2);
        if (valid == FULL)
          pa_cp16(d, src + (size_t)(uint32_t)p * row_bytes);
        else
          pa_cp16(d, src + (size_t)(uint32_t)max(p, 0) * row_bytes, p < 0 ? 0 : 16);
      }
    }
    cp_async_commit();
  };

  // ---- queries of a segment, as loaded
  float2 x[KS][2];
  auto seg_heads = [&](const PagedWalk& w, int& head0) {  // first query head, and how many
    const int g = subs == 1 ? w.item : w.item / subs, sub = subs == 1 ? 0 : w.item - g * subs;
    head0 = g * gq_all + sub * PA_GROUP;
    return min(PA_GROUP, gq_all - sub * PA_GROUP);
  };
  auto next_seg = [&]() {  // to this warp's next segment, with its queries on their way
    do {
      if (!advance(cur)) return false;
    } while (cur.step == 1 && cur.t >= cur.b);
    int head0;
    const int gq = seg_heads(cur, head0);
    const float* q = J.q + cur.row * (J.q_stride ? (size_t)J.q_stride : (size_t)J.n_heads * HD) +
                     (size_t)(head0 + min(lane >> 2, gq - 1)) * HD + 2 * (lane & 3);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) x[k][i] = *reinterpret_cast<const float2*>(q + k * 16 + i * 8);
    return true;
  };

  // unit 0's K and V on their way, unit 1 looked up
  Unit U;
  int slot[TPL], head;  // of the next unit
  mask_t valid, valid_next;
  look(U);
  valid = resolve(U, slot);
  copy(kp, U.head, slot, valid, 0);
  copy(vp, U.head, slot, valid, 1);
  look(U);
  bool have = next_seg();

  float* const part = reinterpret_cast<float*>(static_cast<uint8_t*>(J.work) +
                                               ((size_t)J.rows * items_row * sizeof(unsigned) + 15) / 16 * 16);
  // this lane's rows of the first K and V matrices
  const uint32_t k0 = kt + pa_at<HD>(lane & 7, lane >> 3), vt0 = kt + TILE + pa_at<HD>(lane & 15, lane >> 4);
  while (have) {
    // q of this lane's head as A fragments
    uint32_t qa[KS][4], ql[KS][2];
    float s_scale = J.sm_scale * 1.4426950408889634f;
    {
      float up = copysignf(1.f, s_scale);  // scores with the sign of the scale: the largest has the largest weight
      if (!BF16) {
        // the largest entry to [2^14, 2^15), by a power of two (a row below 2^-112 not quite so far)
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) top = fmaxf(top, fmaxf(fabsf(x[k][i].x), fabsf(x[k][i].y)));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = top > 0.f && top < INFINITY ? min(14 - ilogbf(top), 126) : 0;  // -113 .. 126
        up *= __int_as_float((127 + e) << 23);
        s_scale *= __int_as_float((127 - e) << 23);
      }
      s_scale = fmaxf(fabsf(s_scale), FLT_MIN);  // (a masked position's -inf stays -inf)
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          pa_split<BF16>(x[k][i].x * up, x[k][i].y * up, qa[k][2 * i], qa[k][2 * i + 1], ql[k][i]);
    }
    float m = -INFINITY, l = 0.f, acc[CH][2];
#pragma unroll
    for (int n = 0; n < CH; ++n) acc[n][0] = acc[n][1] = 0.f;
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (; cur.t < cur.b; cur.t += cur.step) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
      // scores, 8 positions a step
      float s[TOK / 8][4];
#pragma unroll
      for (int k = 0; k < KS; k += 2) {
#pragma unroll
        for (int n = 0; n < TOK / 8; ++n) {
          uint32_t b[4];
          pa_ldm(b, (k0 ^ (k << 5)) + n * (HD * 16));
          if (k == 0)
            pa_mma<BF16>(s[n], qa[k], b[0], b[1], zero);
          else
            pa_mma<BF16>(s[n], qa[k], b[0], b[1], s[n]);
          pa_mma<BF16>(s[n], qa[k + 1], b[2], b[3], s[n]);
          if constexpr (BF16) {
            const uint32_t a0[4] = {ql[k][0], 0u, ql[k][1], 0u}, a1[4] = {ql[k + 1][0], 0u, ql[k + 1][1], 0u};
            pa_mma<BF16>(s[n], a0, b[0], b[1], s[n]);
            pa_mma<BF16>(s[n], a1, b[2], b[3], s[n]);
          }
        }
      }
      __syncwarp();  // the K tile is read
      valid_next = resolve(U, slot);
      head = U.head;
      copy(kp, head, slot, valid_next, 0);
      // the scores, their maximum, the weights as powers of 2
      float top = -INFINITY, p[TOK / 8][2];
#pragma unroll
      for (int n = 0; n < TOK / 8; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) p[n][j] = s[n][j] + s[n][j + 2];
      if (valid != FULL) {
        const mask_t mine = valid >> (2 * (lane & 3));
#pragma unroll
        for (int n = 0; n < TOK / 8; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (!((mine >> (n * 8 + j)) & 1)) p[n][j] = -INFINITY;
      }
#pragma unroll
      for (int n = 0; n < TOK / 8; ++n) top = fmaxf(top, fmaxf(p[n][0], p[n][1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // m: the largest score so far, before the scale
      const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn, f = ex2_ftz((m - ref) * s_scale);
      const float shift = fmaf(-ref, s_scale, P_SHIFT);
      m = mn;
      uint32_t pa[TOK / 16][4], pl[TOK / 16][2];
      float ps = 0.f;
#pragma unroll
      for (int n = 0; n < TOK / 8; ++n) {
        const float p0 = ex2_ftz(fmaf(p[n][0], s_scale, shift)), p1 = ex2_ftz(fmaf(p[n][1], s_scale, shift));
        ps += p0 + p1;
        pa_split<BF16>(p0, p1, pa[n / 2][(n & 1) * 2], pa[n / 2][(n & 1) * 2 + 1], pl[n / 2][n & 1]);
      }
      l = fmaf(l, f, ps);
      // weighted values, 16 positions a step
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
#pragma unroll
      for (int n = 0; n < CH; n += 2) {
        float o0[4], o1[4];
#pragma unroll
        for (int k = 0; k < TOK / 16; ++k) {
          uint32_t b[4];
          pa_ldm_trans(b, (vt0 ^ (n << 4)) + k * (HD * 32));
          if (k == 0) {
            pa_mma<BF16>(o0, pa[k], b[0], b[1], zero);
            pa_mma<BF16>(o1, pa[k], b[2], b[3], zero);
          } else {
            pa_mma<BF16>(o0, pa[k], b[0], b[1], o0);
            pa_mma<BF16>(o1, pa[k], b[2], b[3], o1);
          }
          if constexpr (BF16) {
            const uint32_t a[4] = {pl[k][0], 0u, pl[k][1], 0u};
            pa_mma<BF16>(o0, a, b[0], b[1], o0);
            pa_mma<BF16>(o1, a, b[2], b[3], o1);
          }
        }
        acc[n][0] = fmaf(acc[n][0], f, o0[0] + o0[2]);
        acc[n][1] = fmaf(acc[n][1], f, o0[1] + o0[3]);
        acc[n + 1][0] = fmaf(acc[n + 1][0], f, o1[0] + o1[2]);
        acc[n + 1][1] = fmaf(acc[n + 1][1], f, o1[1] + o1[3]);
      }
      __syncwarp();  // the V tile is read
      copy(vp, head, slot, valid_next, 1);
      valid = valid_next;
      look(U);
    }
    // ---- the segment's result
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    int head0;
    const int gq = seg_heads(cur, head0), h = lane >> 2;
    float* const out = J.out + ((size_t)cur.row * J.n_heads + head0) * HD;
    auto inverse = [](float x) { return x > 0.f ? 1.f / x : (x == 0.f ? 0.f : NAN); };  // 0: no position left
    if (cur.step == 1) {  // all of the item, in this warp
      if (h < gq) {
        const float inv = inverse(l);
#pragma unroll
        for (int n = 0; n < CH; ++n)
          *reinterpret_cast<float2*>(out + h * HD + n * 8 + 2 * (lane & 3)) = make_float2(acc[n][0] * inv, acc[n][1] * inv);
      }
      have = next_seg();
      continue;
    }
    const bool whole = cur.whole();
    const int first = cur.s / per, n_parts = (cur.s + cur.tiles - 1) / per - first + 1;  // CTAs that hold the item
    float* const mine = part + ((size_t)cta * 2 + (cur.s >= v0)) * PA_GROUP * (HD + 2);
    unsigned* const count = static_cast<unsigned*>(J.work) + (size_t)cur.row * items_row + cur.item;
    constexpr int DIMS = HD < 64 ? HD : 64;
#pragma unroll
    for (int d0 = 0; d0 < HD; d0 += DIMS) {
      if (d0 > 0) __syncthreads();  // the first dimensions are merged
      if (h < gq) {
#pragma unroll
        for (int n = 0; n < DIMS / 8; ++n)
          *reinterpret_cast<float2*>(&S.acc[warp][h][n * 8 + 2 * (lane & 3)]) =
              make_float2(acc[d0 / 8 + n][0], acc[d0 / 8 + n][1]);
        if (d0 == 0 && (lane & 3) == 0) {
          S.m[warp][h] = m * s_scale;
          S.l[warp][h] = l;
        }
      }
      if (d0 + DIMS == HD) have = next_seg();
      __syncthreads();
      for (int e = tid; e < gq * DIMS / 4; e += PA_THREADS) {
        const int hh = e / (DIMS / 4), d = e % (DIMS / 4) * 4;
        float M = S.m[0][hh];
#pragma unroll
        for (int w = 1; w < PA_WARPS; ++w) M = fmaxf(M, S.m[w][hh]);
        const float ref = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) {
          const float f = ex2_ftz(S.m[w][hh] - ref);
          const float4 o = *reinterpret_cast<const float4*>(&S.acc[w][hh][d]);
          L = fmaf(S.l[w][hh], f, L);
          A = make_float4(fmaf(o.x, f, A.x), fmaf(o.y, f, A.y), fmaf(o.z, f, A.z), fmaf(o.w, f, A.w));
        }
        if (whole) {
          const float inv = inverse(L);
          *reinterpret_cast<float4*>(out + hh * HD + d0 + d) = make_float4(A.x * inv, A.y * inv, A.z * inv, A.w * inv);
        } else {
          __stcg(reinterpret_cast<float4*>(mine + hh * HD + d0 + d), A);
          if (d0 + d == 0) __stcg(reinterpret_cast<float2*>(mine + PA_GROUP * HD) + hh, make_float2(M, L));
        }
      }
    }
    if (!whole) {
      // an item's part lies in its CTA's second place where it begins, else in the first
      __threadfence();
      __syncthreads();
      if (tid == 0) S.last = atomicAdd(count, 1u) == (unsigned)n_parts - 1u;
      __syncthreads();
      if (S.last) {
        __threadfence();
        constexpr int BATCH = 8;  // parts whose loads are in flight together
        for (int e = tid; e < gq * HD / 4; e += PA_THREADS) {
          const int hh = e / (HD / 4);
          float M = -INFINITY, L = 0.f;
          float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int i0 = 0; i0 < n_parts; i0 += BATCH) {
            float4 o[BATCH];
            float2 ml[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
              const int q = min(i0 + i, n_parts - 1);
              const float* const at = part + ((size_t)(first + q) * 2 + (q == 0)) * PA_GROUP * (HD + 2);
              o[i] = __ldcg(reinterpret_cast<const float4*>(at) + e);
              ml[i] = __ldcg(reinterpret_cast<const float2*>(at + PA_GROUP * HD) + hh);
              if (i0 + i >= n_parts) ml[i].x = -INFINITY;
            }
            float top = M;
#pragma unroll
            for (int i = 0; i < BATCH; ++i) top = fmaxf(top, ml[i].x);
            const float ref = top == -INFINITY ? 0.f : top, f0 = ex2_ftz(M - ref);
            M = top;
            L *= f0;
            A = make_float4(A.x * f0, A.y * f0, A.z * f0, A.w * f0);
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
              const float f = ex2_ftz(ml[i].x - ref);
              L = fmaf(ml[i].y, f, L);
              A = make_float4(fmaf(o[i].x, f, A.x), fmaf(o[i].y, f, A.y), fmaf(o[i].z, f, A.z), fmaf(o[i].w, f, A.w));
            }
          }
          const float inv = inverse(L);
          *(reinterpret_cast<float4*>(out) + e) = make_float4(A.x * inv, A.y * inv, A.z * inv, A.w * inv);
        }
        if (tid == 0) *count = 0u;
      }
    }
    __syncthreads();  // the merge area is free again
  }
  cp_async_wait_all();
}

// ---------------------------------------------------------------------------------------
// Pages: fork.  A CTA owns FORK_COLS columns of the table (whole 32-byte sectors): it reads them whole, then writes
// the entries that change and moves their counts.  The counts are integers, so the order of the atomics does not
// show.
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
// one acts.
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
// entries is rewritten by the same CTA, a larger one by pages_renumber_kernel.
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
// words, dealt to the CTAs in turn; the next piece's pair is looked up while a piece is copied.
constexpr int COPY_THREADS = 128, COPY_PER = 4, COPY_PIECE = COPY_THREADS * COPY_PER;
constexpr int COPY_PER_SM = 16;
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

// ---------------------------------------------------------------------------------------
// host side
template <int HD, bool BF16>
static int launch_attention_paged(const gsdlq_paged_attn_job_t& J, int subs, cudaStream_t st) {
  constexpr int smem = (int)sizeof(PagedAttnSmem<HD>);
  static_assert(PA_PER_SM * (smem + 1024) <= 228 * 1024, "shared memory of the CTAs of an SM");
  static std::atomic<bool> set[64];  // the opt-in shared memory size, once per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return record_cuda_error(e);
  if (dev >= 64 || !set[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(attention_paged_kernel<HD, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev < 64) set[dev].store(true, std::memory_order_release);
  }
  const int grid = std::min(PA_PER_SM * num_sms(), PA_MAX_CTAS);
  const int ps = J.kv.page_size, shift = ps & (ps - 1) ? -1 : __builtin_ctz((unsigned)ps);
  return launch_pdl(attention_paged_kernel<HD, BF16>, grid, PA_THREADS, smem, st, 1, J, subs, shift);
}

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
  if (qw > INT32_MAX / 4 || kw > INT32_MAX / 4) return GSDLQ_ERR_INVALID;
  if ((J.q_stride && J.q_stride < qw) || (J.q_out_stride && J.q_out_stride < qw) || (J.kv_stride && J.kv_stride < kw))
    return GSDLQ_ERR_INVALID;
  if (J.q == J.q_out && J.q_stride != J.q_out_stride) return GSDLQ_ERR_INVALID;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int half_shift = J.kv.head_dim == 128 ? 6 : J.kv.head_dim == 64 ? 5 : 4;
  const long long parts = ((qw + 2 * kw) / 2 + RK_THREADS - 1) / RK_THREADS;
  if (J.rows * parts > INT32_MAX) return GSDLQ_ERR_UNSUPPORTED;
  return launch_pdl(J.kv.kv_type == GSDLQ_KV_BF16 ? rope_kv_paged_kernel<true> : rope_kv_paged_kernel<false>,
                    (unsigned)(J.rows * parts), RK_THREADS, 0, st, 1, J, (int)parts, half_shift);
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
  const int gq = J.n_heads / J.kv.n_kv_heads, subs = (gq + PA_GROUP - 1) / PA_GROUP;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // units and places of a layer's pool are counted in 31 bits
  const long long row_units = ((long long)J.kv.max_blocks * J.kv.page_size / pa_tok(J.kv.head_dim) + 8) * J.kv.n_kv_heads * subs;
  if (row_units > INT32_MAX / 2 / J.rows || (long long)J.kv.n_pages * J.kv.page_size > INT32_MAX ||
      (long long)J.kv.n_kv_heads * J.kv.head_dim * 2 > INT32_MAX)
    return GSDLQ_ERR_UNSUPPORTED;
  switch (J.kv.head_dim * 2 + J.kv.kv_type) {
    case 32 * 2: return launch_attention_paged<32, false>(J, subs, st);
    case 32 * 2 + 1: return launch_attention_paged<32, true>(J, subs, st);
    case 64 * 2: return launch_attention_paged<64, false>(J, subs, st);
    case 64 * 2 + 1: return launch_attention_paged<64, true>(J, subs, st);
    case 128 * 2: return launch_attention_paged<128, false>(J, subs, st);
    default: return launch_attention_paged<128, true>(J, subs, st);
  }
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
