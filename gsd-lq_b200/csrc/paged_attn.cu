// paged_attn.cu -- attention of single rows over a paged K/V cache (gsd_cpu_gqa_attention, gsd_lq_cpu_engine.c:265-330,
// per row).
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "paged.cuh"

namespace gsdlq {

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

}  // namespace gsdlq

using namespace gsdlq;

extern "C" {

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

}  // extern "C"
