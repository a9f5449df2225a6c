// paged.cu -- a batch of sequences over one pool of K/V pages: RoPE + append, decode attention, and the
// pages' own operations (fork, reserve, compact, copy).  No reference counterpart: the reference keeps
// one contiguous cache (gsd_lq_cpu_engine.c:186-330); the per-row arithmetic is that of its functions.
#include <algorithm>
#include <atomic>
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
// Attention.  Work is cut into units of PA_TOK positions of one item -- a row and up to eight query heads of
// one kv head -- and all units of the launch, row by row, item by item, are dealt to the CTAs in equal
// contiguous runs, whatever the rows' lengths are (they are known on the device only).  Inside a CTA the
// warps take the units of its run in turn, each through a ring of its own of K and V tiles (cp.async, no
// CTA-wide barrier in the loop), with a running maximum and sum per head.  Where an item ends, the warps merge
// through shared memory; an item that several CTAs share is joined by the CTA that arrives last, in the
// order of the CTAs, so the result does not depend on who that is.
//
// Both products run on mma.m16n8k16 with the 16-bit cache values as they are, so K and V go from shared
// memory to the matrix unit without a conversion.  q and the weights p are fp32 and enter as parts of 16 bits:
//   fp16: q = 2^-e (hi + lo), p 2^11 = hi + lo, about 22 bits: rows 0-7 of A hold the heads' hi, rows 8-15 their lo
//   bf16: hi + mid + lo, 24 bits: hi and mid in the two halves of one A, lo in the lower half of another
// so that one product gives both parts and c[0] + c[2], c[1] + c[3] are the sums.  With A = q, B = K^T the score
// fragment is already p's A fragment for the second product, B = V.  The second product starts from zero each
// unit and is added to fp32 registers, which keeps the tensor core's truncating accumulation short.
constexpr int PA_MAX_CTAS = 320;  // largest grid of an attention launch
constexpr int PA_GROUP = 8;       // query heads of one kv head taken together
constexpr int PA_WARPS = 4, PA_THREADS = PA_WARPS * 32;
constexpr int PA_STAGES = 3;
constexpr int PA_TILE = 4096;     // bytes of a unit's K or V tile

template <int HD>
struct PagedAttnSmem {
  uint8_t ring[PA_WARPS][PA_STAGES][2 * PA_TILE];
  union {
    float acc[PA_WARPS][PA_GROUP][HD];  // the warps' results of an item
    float f[PA_GROUP][PA_MAX_CTAS];     // factors of the CTAs' parts, once those are written
  };
  float m[PA_WARPS][PA_GROUP], l[PA_WARPS][PA_GROUP];
  float fl[PA_GROUP];
  unsigned long long valid[PA_WARPS][PA_STAGES];
  long long warp_sum[PA_WARPS];
  long long base;
  int row, last;
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
__device__ __forceinline__ void pa_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
__device__ __forceinline__ void pa_cp16(uint32_t dst, const void* src, bool ok) {  // zeros where not ok
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
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

// a walk over the units of the launch: the row and the unit it begins with
struct PagedWalk {
  long long base;  // first unit of the row
  int row, tiles;  // units per item of the row
  PagedRow pr;
};

template <int HD, bool BF16>
__global__ void __launch_bounds__(PA_THREADS, 2)
    attention_paged_kernel(const __grid_constant__ gsdlq_paged_attn_job_t J, int subs) {
  constexpr int TOK = PA_TILE / (HD * 2);  // positions of a unit: 16, 32, 64
  constexpr int CH = HD / 8;               // 16-byte chunks of a row
  constexpr int KS = HD / 16;              // k steps of the first product
  constexpr int TPL = (TOK + 31) / 32;     // positions a lane looks up
  constexpr float P_SHIFT = BF16 ? 0.f : 11.f;
  extern __shared__ __align__(16) uint8_t pa_smem[];
  PagedAttnSmem<HD>& S = *reinterpret_cast<PagedAttnSmem<HD>*>(pa_smem);
  const gsdlq_paged_kv_t& kv = J.kv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
  const int gq_all = J.n_heads / kv.n_kv_heads, items_row = kv.n_kv_heads * subs;
  const size_t kw = (size_t)kv.n_kv_heads * HD;

  // the launch's units, this CTA's run of them, and the row where it begins
  long long sum = 0;
  for (int r = tid; r < J.rows; r += PA_THREADS)
    sum += (paged_row(kv, J.row_seq, J.pos, r, cta == 0).len + TOK - 1) / TOK;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) S.warp_sum[warp] = sum;
  if (tid == 0) S.row = -1;
  for (int r = cta; r < J.rows; r += gridDim.x)  // idle rows
    if (paged_row(kv, J.row_seq, J.pos, r, false).len == 0)
      for (int i = tid; i < J.n_heads * HD; i += PA_THREADS) J.out[(size_t)r * J.n_heads * HD + i] = 0.f;
  __syncthreads();
  long long units = 0;
#pragma unroll
  for (int w = 0; w < PA_WARPS; ++w) units += S.warp_sum[w];
  units *= items_row;
  const long long per = max((units + gridDim.x - 1) / (long long)gridDim.x, (long long)PA_WARPS);
  const long long u0 = per * cta, u1 = min(units, u0 + per);
  if (u0 >= u1) return;
  if (warp == 0) {  // find the row of u0
    long long before = 0;
    for (int r0 = 0; r0 < J.rows; r0 += 32) {
      const int r = r0 + lane;
      const long long n =
          r < J.rows ? (long long)((paged_row(kv, J.row_seq, J.pos, r, false).len + TOK - 1) / TOK) * items_row : 0;
      long long inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      if (before + inc - n <= u0 && u0 < before + inc) {
        S.row = r;
        S.base = before + inc - n;
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
      if (before > u0) break;
    }
  }
  __syncthreads();
  auto enter = [&](PagedWalk& w, int row, long long base) {
    w.row = row;
    w.base = base;
    w.pr = paged_row(kv, J.row_seq, J.pos, row, false);
    w.tiles = (w.pr.len + TOK - 1) / TOK;
  };
  auto advance = [&](PagedWalk& w, long long u) {  // to the row of unit u (u < units: it exists)
    while (u >= w.base + (long long)w.tiles * items_row) enter(w, w.row + 1, w.base + (long long)w.tiles * items_row);
  };

  // ---- the ring: where a unit's rows are, one step before they are copied
  const uint16_t* const kp = static_cast<const uint16_t*>(kv.k) + (size_t)J.layer * kv.n_pages * kv.page_size * kw;
  const uint16_t* const vp = static_cast<const uint16_t*>(kv.v) + (size_t)J.layer * kv.n_pages * kv.page_size * kw;
  const uint32_t ring = smem_u32(S.ring[warp][0]);
  PagedWalk ahead;
  enter(ahead, S.row, S.base);
  long long u_look = u0 + warp;  // next unit to look up
  int at_page[TPL], at_slot[TPL], at_head;
  auto look = [&]() {
    at_head = -1;
    if (u_look < u1) {
      advance(ahead, u_look);
      const int rel = (int)(u_look - ahead.base), item = rel / ahead.tiles, tile = rel - item * ahead.tiles;
      at_head = item / subs;
#pragma unroll
      for (int i = 0; i < TPL; ++i) {
        const int t = tile * TOK + i * 32 + lane;
        at_page[i] = -1;
        at_slot[i] = 0;
        if ((TOK >= 32 || lane < TOK) && t < ahead.pr.len) {
          const int b = t / kv.page_size;
          at_slot[i] = t - b * kv.page_size;
          at_page[i] = kv.table[(size_t)ahead.pr.seq * kv.max_blocks + b];
          if (!paged_valid(kv, at_page[i])) raise_flag(GSDLQ_FLAG_BAD_PAGE);
        }
      }
    }
    u_look += PA_WARPS;
  };
  auto copy = [&](int stage) {
    if (at_head >= 0) {
      long long off[TPL];
      unsigned long long valid = 0;
#pragma unroll
      for (int i = 0; i < TPL; ++i) {
        const bool ok = paged_valid(kv, at_page[i]);
        off[i] = ok ? (long long)(((size_t)at_page[i] * kv.page_size + at_slot[i]) * kw + (size_t)at_head * HD) : -1;
        valid |= (unsigned long long)__ballot_sync(0xffffffffu, ok) << (32 * i);
      }
      if (lane == 0) S.valid[warp][stage] = valid;
      const uint32_t dst = ring + stage * 2 * PA_TILE;
#pragma unroll
      for (int it = 0; it < TOK * CH / 32; ++it) {
        const int e = it * 32 + lane, j = e / CH, c = e % CH;
        const long long o = __shfl_sync(0xffffffffu, off[(it * 32 / CH) / 32], j & 31);
        const size_t src = o < 0 ? 0 : (size_t)o + c * 8;
        pa_cp16(dst + pa_at<HD>(j, c), kp + src, o >= 0);
        pa_cp16(dst + PA_TILE + pa_at<HD>(j, c), vp + src, o >= 0);
      }
    }
    cp_async_commit();
  };
  look();
#pragma unroll
  for (int s = 0; s < PA_STAGES - 1; ++s) {
    copy(s);
    look();
  }

  // ---- item by item
  float* const part = reinterpret_cast<float*>(static_cast<uint8_t*>(J.work) +
                                               ((size_t)J.rows * items_row * sizeof(unsigned) + 15) / 16 * 16);
  unsigned* const arrived = static_cast<unsigned*>(J.work);
  PagedWalk cur;
  enter(cur, S.row, S.base);
  long long u = u0 + warp;  // this warp's next unit
  int stage = 0;
  for (long long item_u = u0; item_u < u1;) {
    advance(cur, item_u);
    const int item = (int)((item_u - cur.base) / cur.tiles);
    const long long i0 = cur.base + (long long)item * cur.tiles, i1 = i0 + cur.tiles;  // the item's units
    const long long end = min(i1, u1);
    const int g = item / subs, sub = item - g * subs, gq = min(PA_GROUP, gq_all - sub * PA_GROUP);
    const int head0 = g * gq_all + sub * PA_GROUP;
    // q of this lane's head as A fragments
    uint32_t qa[KS][4], ql[KS][2];
    float s_scale;
    {
      const int h = lane >> 2;
      const float* q = J.q + cur.row * (J.q_stride ? (size_t)J.q_stride : (size_t)J.n_heads * HD) +
                       (size_t)(head0 + min(h, gq - 1)) * HD + 2 * (lane & 3);
      float2 x[KS][2];
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[k][i] = *reinterpret_cast<const float2*>(q + k * 16 + i * 8);
          top = fmaxf(top, fmaxf(fabsf(x[k][i].x), fabsf(x[k][i].y)));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // fp16: the largest entry to [2^14, 2^15), by a power of two; both factors stay normal numbers
      const int e = BF16 ? 0 : (top > 0.f && top < INFINITY) ? min(max(14 - ilogbf(top), -100), 140) : 0;
      const float up = exp2f((float)(e / 2)), up2 = exp2f((float)(e - e / 2));
      s_scale = J.sm_scale * 1.4426950408889634f;
      if (!BF16) s_scale = s_scale / up / up2;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t lo;
          pa_split<BF16>(BF16 ? x[k][i].x : x[k][i].x * up * up2, BF16 ? x[k][i].y : x[k][i].y * up * up2, qa[k][2 * i],
                         qa[k][2 * i + 1], lo);
          ql[k][i] = lo;
        }
    }
    float m = -INFINITY, l = 0.f, acc[CH][2];
#pragma unroll
    for (int n = 0; n < CH; ++n) acc[n][0] = acc[n][1] = 0.f;
    for (; u < end; u += PA_WARPS) {
      int next = stage + PA_STAGES - 1;
      next = next >= PA_STAGES ? next - PA_STAGES : next;
      copy(next);
      look();
      asm volatile("cp.async.wait_group %0;" ::"n"(PA_STAGES - 1) : "memory");
      __syncwarp();
      const uint32_t kt = ring + stage * 2 * PA_TILE, vt = kt + PA_TILE;
      const unsigned long long valid = S.valid[warp][stage];
      // scores of 8 positions a step
      float s[TOK / 8][4];
#pragma unroll
      for (int n = 0; n < TOK / 8; ++n) {
        s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          uint32_t b[4];
          pa_ldm(b, kt + pa_at<HD>(n * 8 + (lane & 7), k * 2 + (lane >> 3)));
          pa_mma<BF16>(s[n], qa[k], b[0], b[1]);
          pa_mma<BF16>(s[n], qa[k + 1], b[2], b[3]);
          if constexpr (BF16) {
            const uint32_t a0[4] = {ql[k][0], 0u, ql[k][1], 0u}, a1[4] = {ql[k + 1][0], 0u, ql[k + 1][1], 0u};
            pa_mma<BF16>(s[n], a0, b[0], b[1]);
            pa_mma<BF16>(s[n], a1, b[2], b[3]);
          }
        }
      }
      // log2 weights, the running maximum
      float top = -INFINITY;
      float p[TOK / 8][2];
#pragma unroll
      for (int n = 0; n < TOK / 8; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float x = (s[n][j] + s[n][j + 2]) * s_scale;
          p[n][j] = (valid >> (n * 8 + 2 * (lane & 3) + j)) & 1ull ? x : -INFINITY;
          top = fmaxf(top, p[n][j]);
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float mn = fmaxf(m, top);
      const float ref = mn == -INFINITY ? 0.f : mn - P_SHIFT;
      const float f = m == -INFINITY ? 0.f : exp2f(m - mn);
      m = mn;
      l *= f;
      uint32_t pa[TOK / 16][4], pl[TOK / 16][2];
#pragma unroll
      for (int n = 0; n < TOK / 8; ++n) {
        p[n][0] = exp2f(p[n][0] - ref);
        p[n][1] = exp2f(p[n][1] - ref);
        l += p[n][0] + p[n][1];
        uint32_t lo;
        pa_split<BF16>(p[n][0], p[n][1], pa[n / 2][(n & 1) * 2], pa[n / 2][(n & 1) * 2 + 1], lo);
        pl[n / 2][n & 1] = lo;
      }
      // weighted values, 16 positions a step
#pragma unroll
      for (int n = 0; n < CH; n += 2) {
        float o0[4] = {0.f, 0.f, 0.f, 0.f}, o1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < TOK / 16; ++k) {
          uint32_t b[4];
          pa_ldm_trans(b, vt + pa_at<HD>(k * 16 + (lane & 15), n + (lane >> 4)));
          pa_mma<BF16>(o0, pa[k], b[0], b[1]);
          pa_mma<BF16>(o1, pa[k], b[2], b[3]);
          if constexpr (BF16) {
            const uint32_t a[4] = {pl[k][0], 0u, pl[k][1], 0u};
            pa_mma<BF16>(o0, a, b[0], b[1]);
            pa_mma<BF16>(o1, a, b[2], b[3]);
          }
        }
        acc[n][0] = fmaf(acc[n][0], f, o0[0] + o0[2]);
        acc[n][1] = fmaf(acc[n][1], f, o0[1] + o0[3]);
        acc[n + 1][0] = fmaf(acc[n + 1][0], f, o1[0] + o1[2]);
        acc[n + 1][1] = fmaf(acc[n + 1][1], f, o1[1] + o1[3]);
      }
      __syncwarp();  // the tile is read
      stage = stage + 1 == PA_STAGES ? 0 : stage + 1;
    }
    // ---- the warps' results of the item
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    {
      const int h = lane >> 2;
      if (h < gq) {
#pragma unroll
        for (int n = 0; n < CH; ++n)
          *reinterpret_cast<float2*>(&S.acc[warp][h][n * 8 + 2 * (lane & 3)]) = make_float2(acc[n][0], acc[n][1]);
        if ((lane & 3) == 0) {
          S.m[warp][h] = m;
          S.l[warp][h] = l;
        }
      }
    }
    __syncthreads();
    const bool whole = i0 >= u0 && i1 <= u1;
    float* const mine = part + ((size_t)cta * 2 + (i0 >= u0)) * PA_GROUP * (HD + 2);
    float* const out = J.out + ((size_t)cur.row * J.n_heads + head0) * HD;
    for (int e = tid; e < gq * HD; e += PA_THREADS) {
      const int h = e / HD, d = e % HD;
      float M = S.m[0][h];
#pragma unroll
      for (int w = 1; w < PA_WARPS; ++w) M = fmaxf(M, S.m[w][h]);
      float L = 0.f, A = 0.f;
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) {
        const float f = S.m[w][h] == -INFINITY ? 0.f : exp2f(S.m[w][h] - M);
        L = fmaf(S.l[w][h], f, L);
        A = fmaf(S.acc[w][h][d], f, A);
      }
      if (whole) {
        out[e] = L > 0.f ? A / L : (L == 0.f ? 0.f : NAN);
      } else {
        __stcg(mine + e, A);
        if (d == 0) {
          __stcg(mine + PA_GROUP * HD + h, M);
          __stcg(mine + PA_GROUP * (HD + 1) + h, L);
        }
      }
    }
    if (!whole) {
      // CTAs first .. last hold the item; its part lies in their second slot where it begins, else in the first
      const int first = (int)(i0 / per), n_parts = (int)((i1 - 1) / per) - first + 1;
      unsigned* const count = arrived + (size_t)cur.row * items_row + item;
      __threadfence();
      __syncthreads();
      if (tid == 0) S.last = atomicAdd(count, 1u) == (unsigned)n_parts - 1u;
      __syncthreads();
      if (S.last) {
        __threadfence();
        auto slot = [&](int i) { return part + ((size_t)(first + i) * 2 + (i == 0)) * PA_GROUP * (HD + 2); };
        for (int h = warp; h < gq; h += PA_WARPS) {
          float M = -INFINITY, L = 0.f;
          for (int i = lane; i < n_parts; i += 32) {
            const float x = __ldcg(slot(i) + PA_GROUP * HD + h);
            S.f[h][i] = x;
            M = fmaxf(M, x);
          }
          M = warp_max(M);
          for (int i = lane; i < n_parts; i += 32) {
            const float f = S.f[h][i] == -INFINITY ? 0.f : exp2f(S.f[h][i] - M);
            S.f[h][i] = f;
            L = fmaf(__ldcg(slot(i) + PA_GROUP * (HD + 1) + h), f, L);
          }
          L = warp_sum(L);
          if (lane == 0) S.fl[h] = L;
        }
        __syncthreads();
        for (int e = tid; e < gq * HD; e += PA_THREADS) {
          const int h = e / HD;
          float A = 0.f;
#pragma unroll 8
          for (int i = 0; i < n_parts; ++i) A = fmaf(__ldcg(slot(i) + e), S.f[h][i], A);
          const float L = S.fl[h];
          out[e] = L > 0.f ? A / L : (L == 0.f ? 0.f : NAN);
        }
        if (tid == 0) *count = 0u;
      }
    }
    __syncthreads();  // the merge area is free again
    item_u = end;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
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
// host side
template <int HD, bool BF16>
static int launch_attention_paged(const gsdlq_paged_attn_job_t& J, int subs, cudaStream_t st) {
  constexpr int smem = (int)sizeof(PagedAttnSmem<HD>);
  static_assert(2 * (smem + 1024) <= 228 * 1024, "two CTAs an SM");
  static std::atomic<bool> set[64];  // the opt-in shared memory size, once per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return record_cuda_error(e);
  if (dev >= 64 || !set[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(attention_paged_kernel<HD, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev < 64) set[dev].store(true, std::memory_order_release);
  }
  const int grid = std::min(2 * num_sms(), PA_MAX_CTAS);
  attention_paged_kernel<HD, BF16><<<grid, PA_THREADS, smem, st>>>(J, subs);
  GSDLQ_CUDA_CHECK_LAUNCH();
  return GSDLQ_OK;
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
  const int gq = J.n_heads / J.kv.n_kv_heads, subs = (gq + PA_GROUP - 1) / PA_GROUP;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // a row's units are counted in 31 bits
  const int tok = PA_TILE / (J.kv.head_dim * 2);
  if (((long long)J.kv.max_blocks * J.kv.page_size / tok + 1) * J.kv.n_kv_heads * subs > INT32_MAX)
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
