// paged_attn.cu -- attention of single rows over a paged K/V cache (gsd_cpu_gqa_attention, gsd_lq_cpu_engine.c:265-330,
// per row).
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>
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
// way while the weights and the second product are worked on, its V during the next first product.  Two CTAs an SM
// keep up to 128 KB on their way; three (at 168 registers a thread, with spills) were slower: 74 us against 63 for 64
// rows of 1 to 8191 positions.
//
// Both products run on mma.m16n8k16 with the 16-bit cache values as they are, so K and V go from shared
// memory to the matrix unit without a conversion.  q and the weights p are fp32 and enter as parts of 16 bits:
//   fp16: q = 2^-e (hi + lo), p 2^11 = hi + lo, about 22 bits: rows 0-7 of A hold the heads' hi, rows 8-15 their lo
//   bf16: hi + mid + lo, 24 bits: hi and mid in the two halves of one A, lo in the lower half of another
// so that one product gives both parts and c[0] + c[2], c[1] + c[3] are the sums.  With A = q, B = K^T the score
// fragment is already p's A fragment for the second product, B = V.  The second product starts from zero each
// unit and is added to fp32 registers, which keeps the tensor core's truncating accumulation short.  (A tile of
// tcgen05.mma has 128 rows; eight columns in two parts would fill an eighth of it, and at 13-31 % of its cycles the
// tensor pipe bounds nothing here.)
//
// Bound by HBM.  Measured on one B200 (device time, L2 cold): 16 rows x 32 kv heads of 64 over 1025-2047 positions,
// fp16: 41 us for 195 MB (4.8 TB/s; 5.9 TB/s from the first tile to the last, then 3-4 us of joining); 64 rows x 8 kv
// heads of 128 over 1-8191 positions, bf16: 53 us for 250 MB; one row x 8 kv heads of 128 over 1537 positions: 9.7 us,
// of which 2.6 pass before the first tile (positions, table, tile: three dependent look-ups) and 3.5 in the join.
// Heads of 128 take all 255 registers; in bf16 14 words spill (52 bytes stored, 56 loaded), in fp16 one.
constexpr int PA_MAX_CTAS = 320;  // largest grid of an attention launch
constexpr int PA_PER_SM = 2;
constexpr int PA_GROUP = 8;       // query heads of one kv head taken together
constexpr int PA_WARPS = 4, PA_THREADS = PA_WARPS * 32;
constexpr int PA_SHORT = 4;       // units of an item that one warp may take
// units that an item counts besides its own, for its queries, and for the merge of the warps where it has one
// (64 rows of 1-8191 positions: 1 and 2 units 62 us, 1 and 4 58, 2 and 4 54, 3 and 5 53, 4 and 6 55)
__host__ __device__ constexpr int pa_over(int tiles) { return tiles <= PA_SHORT ? 2 : 4; }

constexpr int pa_tok(int hd) { return hd == 128 ? 32 : 64; }  // positions of a unit

template <int HD>
struct PagedAttnSmem {
  uint8_t tile[PA_WARPS][2][pa_tok(HD) * HD * 2];  // K, V
  float acc[PA_WARPS][PA_GROUP][HD];               // the warps' results of an item
  float m[PA_WARPS][PA_GROUP], l[PA_WARPS][PA_GROUP];
  int warp_sum[PA_WARPS];
  int row, base, last;
};

// The work area: two partial results per CTA (its first and its last item), in the form for rows that share sequences
// one per warp, then the items' counters, which are zero between launches.  The results' part has the same size for
// every launch, whatever its rows, heads and head size are, so none ever writes where another one counts, and one area
// serves launches of any shapes in turn.
constexpr size_t PA_PARTS = sizeof(float) * (size_t)PA_MAX_CTAS * 2 * PA_WARPS * PA_GROUP * (128 + 2);
static_assert(PA_PARTS % 16 == 0, "the counters follow");
inline size_t attention_paged_work(int rows, int n_heads, int n_kv) {
  const size_t items = (size_t)rows * n_kv * ((n_heads / n_kv + PA_GROUP - 1) / PA_GROUP);
  return PA_PARTS + (items * sizeof(unsigned) + 15) / 16 * 16;
}
__device__ __forceinline__ float* pa_parts(void* work) { return static_cast<float*>(work); }
__device__ __forceinline__ unsigned* pa_counter(void* work, size_t item) {
  return reinterpret_cast<unsigned*>(static_cast<uint8_t*>(work) + PA_PARTS) + item;
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

// Up to eight query columns -- heads, or heads of several rows -- in a warp; a lane's column is lane / 4.
template <int HD, bool BF16>
struct PaColumns {
  static constexpr int TOK = pa_tok(HD), CH = HD / 8, KS = HD / 16;
  static constexpr float P_SHIFT = BF16 ? 0.f : 11.f;
  uint32_t qa[KS][4], ql[KS][2];  // q as A fragments
  float scale, m, l;              // of the log2 scores; largest score so far, before the scale; this lane's sum of weights
  float acc[CH][2];
  typedef float2 Raw[KS][2];      // this lane's entries of its column's q, as loaded

  static __device__ __forceinline__ void load(Raw& x, const float* q) {  // q of the column
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) x[k][i] = *reinterpret_cast<const float2*>(q + 2 * (threadIdx.x & 3) + k * 16 + i * 8);
  }
  __device__ __forceinline__ void begin(const Raw& x, float sm_scale) {
    scale = sm_scale * 1.4426950408889634f;
    float up = copysignf(1.f, scale);  // scores with the sign of the scale: the largest has the largest weight
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
      scale *= __int_as_float((127 - e) << 23);
    }
    scale = fmaxf(fabsf(scale), FLT_MIN);  // (a masked position's -inf stays -inf)
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        pa_split<BF16>(x[k][i].x * up, x[k][i].y * up, qa[k][2 * i], qa[k][2 * i + 1], ql[k][i]);
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int n = 0; n < CH; ++n) acc[n][0] = acc[n][1] = 0.f;
  }
  // scores of a unit, 8 positions a step; k0: this lane's row of the tile's first matrices
  __device__ __forceinline__ void scores(float (&p)[TOK / 8][2], uint32_t k0) const {
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
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
#pragma unroll
    for (int n = 0; n < TOK / 8; ++n) {
      p[n][0] = s[n][0] + s[n][2];
      p[n][1] = s[n][1] + s[n][3];
    }
  }
  struct Weights {
    uint32_t a[TOK / 16][4], lo[TOK / 16][2];  // as A fragments
    float f;                                   // what the earlier results are worth now
  };
  // the weights of scores p (-inf: masked); the running maximum and sum move on
  __device__ __forceinline__ void weights(Weights& W, const float (&p)[TOK / 8][2]) {
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < TOK / 8; ++n) top = fmaxf(top, fmaxf(p[n][0], p[n][1]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn;
    W.f = ex2_ftz((m - ref) * scale);
    const float shift = fmaf(-ref, scale, P_SHIFT);
    m = mn;
    float ps = 0.f;
#pragma unroll
    for (int n = 0; n < TOK / 8; ++n) {
      const float p0 = ex2_ftz(fmaf(p[n][0], scale, shift)), p1 = ex2_ftz(fmaf(p[n][1], scale, shift));
      ps += p0 + p1;
      pa_split<BF16>(p0, p1, W.a[n / 2][(n & 1) * 2], W.a[n / 2][(n & 1) * 2 + 1], W.lo[n / 2][n & 1]);
    }
    l = fmaf(l, W.f, ps);
  }
  // weighted values, 16 positions a step; v0: this lane's row of the tile's first matrices
  __device__ __forceinline__ void values(const Weights& W, uint32_t v0) {
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < CH; n += 2) {
      float o0[4], o1[4];
#pragma unroll
      for (int k = 0; k < TOK / 16; ++k) {
        uint32_t b[4];
        pa_ldm_trans(b, (v0 ^ (n << 4)) + k * (HD * 32));
        if (k == 0) {
          pa_mma<BF16>(o0, W.a[k], b[0], b[1], zero);
          pa_mma<BF16>(o1, W.a[k], b[2], b[3], zero);
        } else {
          pa_mma<BF16>(o0, W.a[k], b[0], b[1], o0);
          pa_mma<BF16>(o1, W.a[k], b[2], b[3], o1);
        }
        if constexpr (BF16) {
          const uint32_t a[4] = {W.lo[k][0], 0u, W.lo[k][1], 0u};
          pa_mma<BF16>(o0, a, b[0], b[1], o0);
          pa_mma<BF16>(o1, a, b[2], b[3], o1);
        }
      }
      acc[n][0] = fmaf(acc[n][0], W.f, o0[0] + o0[2]);
      acc[n][1] = fmaf(acc[n][1], W.f, o0[1] + o0[3]);
      acc[n + 1][0] = fmaf(acc[n + 1][0], W.f, o1[0] + o1[2]);
      acc[n + 1][1] = fmaf(acc[n + 1][1], W.f, o1[1] + o1[3]);
    }
  }
  // What values() of a tile without its non-finite entries (pa_finite) leaves out: those of the positions `mine`, into
  // their own dimensions.
  template <typename M>
  __device__ __forceinline__ void add_not_finite(const uint8_t* tile, M mine) {
    for (int j = 0; j < TOK; ++j) {
      if (!((mine >> j) & 1)) continue;
#pragma unroll
      for (int n = 0; n < CH; ++n) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + pa_at<HD>(j, n) + 4 * (threadIdx.x & 3));
        float2 f;
        if constexpr (BF16) {
          f = make_float2(bf16lo_to_f(w), bf16hi_to_f(w));
        } else {
          f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        }
        if (!isfinite(f.x)) acc[n][0] += f.x;
        if (!isfinite(f.y)) acc[n][1] += f.y;
      }
    }
  }
  // this lane's sums over its column's four lanes
  __device__ __forceinline__ void finish() {
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
  }
};
// Those of the positions lo .. hi - 1 of a tile (and their neighbours) that hold entries that are not finite (exponent all
// ones); if there are any, `to` receives the tile with zeros for them.
template <int HD, bool BF16, typename M>
__device__ __forceinline__ M pa_finite(const uint8_t* tile, int lo, int hi, uint8_t* to) {
  constexpr int CH = HD / 8, POS = 32 / CH, STEPS = pa_tok(HD) / POS;  // CH lanes a position
  constexpr uint32_t E = BF16 ? 0x7f807f80u : 0x7c007c00u, ONE = BF16 ? 0x00800080u : 0x04000400u;
  const int lane = threadIdx.x & 31, s0 = lo / POS, s1 = (hi + POS - 1) / POS;
  const uint4* const at = reinterpret_cast<const uint4*>(tile) + lane;
  auto test = [](uint32_t w) { return ((w & E) + ONE) & 0x80008000u; };  // the upper bit of each such half
  uint32_t any = 0u;
#pragma unroll 2
  for (int it = s0; it < s1; ++it) {
    const uint4 w = at[it * 32];
    any |= test(w.x) | test(w.y) | test(w.z) | test(w.w);
  }
  if (!__any_sync(0xffffffffu, any)) return 0;
  M bad = 0;
  __syncwarp();  // what the lanes read of `to` before
#pragma unroll 1
  for (int it = 0; it < STEPS; ++it) {
    uint4 w = at[it * 32];
    if (it >= s0 && it < s1) {
      const uint32_t x = test(w.x), y = test(w.y), z = test(w.z), u = test(w.w);
      const unsigned b = __ballot_sync(0xffffffffu, x | y | z | u);
      for (int i = 0; i < POS; ++i)
        if ((b >> (i * CH)) & ((1u << CH) - 1u)) bad |= (M)1 << (it * POS + i);
      w = make_uint4(w.x & ~((x >> 15) * 0xffffu), w.y & ~((y >> 15) * 0xffffu), w.z & ~((z >> 15) * 0xffffu),
                     w.w & ~((u >> 15) * 0xffffu));
    }
    reinterpret_cast<uint4*>(to)[it * 32 + lane] = w;
  }
  __syncwarp();
  return bad;
}

__device__ __forceinline__ float pa_inverse(float x) { return x > 0.f ? 1.f / x : (x == 0.f ? 0.f : NAN); }  // 0: no position left

// One thread, after a barrier behind which the CTA's part is written: whether it is the last of n_parts CTAs, whose
// parts the CTA may then read, after another barrier.
__device__ __forceinline__ bool pa_arrive(unsigned* count, int n_parts) {
  __threadfence();
  const bool last = atomicAdd(count, 1u) == (unsigned)n_parts - 1u;
  if (last) __threadfence();
  return last;
}

// Joining the parts of an item that n_parts CTAs from `first` on hold.  A CTA's part lies in its second place where the
// item begins, else in the first; places are `slot` floats apart.  A place: [PA_GROUP][HD] weighted sums, then the
// columns' (maximum, sum of weights).  The joining warps are alone on their SM, so what counts is how many loads are in
// flight and how few instructions follow one another: one load after the other, joining 13 parts took 7 us; it takes 2.
__device__ __forceinline__ const float* pa_place(const float* part, size_t slot, int first, int i) {
  return part + ((size_t)(first + i) * 2 + (i == 0)) * slot;
}
// A thread's four values of column c (the e-th four), with its own sums of the weights.
template <int HD>
__device__ __forceinline__ float4 pa_join(const float* part, size_t slot, int first, int n_parts, int c, int e) {
  constexpr int BATCH = 8;  // parts whose loads are in flight together
  float M = -INFINITY, L = 0.f;
  float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n_parts; i0 += BATCH) {
    float4 o[BATCH];
    float2 ml[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float* const at = pa_place(part, slot, first, min(i0 + i, n_parts - 1));
      o[i] = __ldcg(reinterpret_cast<const float4*>(at + c * HD) + e);
      ml[i] = __ldcg(reinterpret_cast<const float2*>(at + PA_GROUP * HD) + c);
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
  const float inv = pa_inverse(L);
  return make_float4(A.x * inv, A.y * inv, A.z * inv, A.w * inv);
}
// For many values a thread: the parts' factors once per column, then the sums.
// factors f[i] of a column over the lanes `lane`, `lane + lanes`, ... of those that share it (xor distances from..16)
template <int HD>
__device__ __forceinline__ void pa_factors(float* f, const float* part, size_t slot, int first, int n_parts, int c, int i0,
                                           int lanes) {
  float M = -INFINITY, L = 0.f;
  for (int i = i0; i < n_parts; i += lanes) {
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(pa_place(part, slot, first, i) + PA_GROUP * HD) + c);
    f[i] = ml.x;
    const float top = fmaxf(M, ml.x), ref = top == -INFINITY ? 0.f : top;
    L = fmaf(L, ex2_ftz(M - ref), ml.y * ex2_ftz(ml.x - ref));
    M = top;
  }
  for (int o = 32 / lanes; o < 32; o <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, M, o), l2 = __shfl_xor_sync(0xffffffffu, L, o);
    const float top = fmaxf(M, m2), ref = top == -INFINITY ? 0.f : top;
    L = fmaf(L, ex2_ftz(M - ref), l2 * ex2_ftz(m2 - ref));
    M = top;
  }
  const float ref = M == -INFINITY ? 0.f : M, inv = pa_inverse(L);
  for (int i = i0; i < n_parts; i += lanes) f[i] = ex2_ftz(f[i] - ref) * inv;
}
// fours e0, e0 + step, .. of the item's columns: the parts' sums times their factors (f: a row of `f_row` per column)
template <int HD, int E, int BATCH>
__device__ __forceinline__ void pa_sums(float4 (&A)[E], const float* f, int f_row, const float* part, size_t slot,
                                        int first, int n_parts, int e0, int step) {
#pragma unroll
  for (int k = 0; k < E; ++k) A[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n_parts; i0 += BATCH) {
    float4 o[BATCH][E];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float4* const at = reinterpret_cast<const float4*>(pa_place(part, slot, first, min(i0 + i, n_parts - 1))) + e0;
#pragma unroll
      for (int k = 0; k < E; ++k) o[i][k] = __ldcg(at + k * step);
    }
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const float* const fk = f + (e0 + k * step) / (HD / 4) * f_row + i0;
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const float x = i0 + i < n_parts ? fk[i] : 0.f;
        A[k] = make_float4(fmaf(o[i][k].x, x, A[k].x), fmaf(o[i][k].y, x, A[k].y), fmaf(o[i][k].z, x, A[k].z),
                           fmaf(o[i][k].w, x, A[k].w));
      }
    }
  }
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
  constexpr int TPL = TOK / 32;            // positions a lane looks up
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
  // (the row is found unless the positions change meanwhile, which ends in no row and no wait)
  if (tid == 0) S.row = -1;
  __syncthreads();
  if (J.rows <= PA_THREADS) {
    if (base0 <= v0 && v0 < base0 + mine0) {
      S.row = tid;
      S.base = base0;
    }
  } else {
    int before = 0;
    for (int r0 = 0; r0 < J.rows && before <= v0; r0 += PA_THREADS) {
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
  if (S.row < 0) return;

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
  typedef PaColumns<HD, BF16> Cols;
  Cols C;
  typename Cols::Raw x;
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
    Cols::load(x, J.q + cur.row * (J.q_stride ? (size_t)J.q_stride : (size_t)J.n_heads * HD) +
                      (size_t)(head0 + min(lane >> 2, gq - 1)) * HD);
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

  float* const part = pa_parts(J.work);
  // this lane's rows of the first K and V matrices
  const uint32_t k0 = kt + pa_at<HD>(lane & 7, lane >> 3), vt0 = kt + TILE + pa_at<HD>(lane & 15, lane >> 4);
  while (have) {
    C.begin(x, J.sm_scale);
    for (; cur.t < cur.b; cur.t += cur.step) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
      float p[TOK / 8][2];
      C.scores(p, k0);
      __syncwarp();  // the K tile is read
      valid_next = resolve(U, slot);
      head = U.head;
      copy(kp, head, slot, valid_next, 0);
      if (valid != FULL) {
        const mask_t mine = valid >> (2 * (lane & 3));
#pragma unroll
        for (int n = 0; n < TOK / 8; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (!((mine >> (n * 8 + j)) & 1)) p[n][j] = -INFINITY;
      }
      typename Cols::Weights W;
      C.weights(W, p);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
      C.values(W, vt0);
      __syncwarp();  // the V tile is read
      copy(vp, head, slot, valid_next, 1);
      valid = valid_next;
      look(U);
    }
    // ---- the segment's result
    C.finish();
    int head0;
    const int gq = seg_heads(cur, head0), h = lane >> 2;
    float* const out = J.out + ((size_t)cur.row * J.n_heads + head0) * HD;
    if (cur.step == 1) {  // all of the item, in this warp
      if (h < gq) {
        const float inv = pa_inverse(C.l);
#pragma unroll
        for (int n = 0; n < CH; ++n)
          *reinterpret_cast<float2*>(out + h * HD + n * 8 + 2 * (lane & 3)) = make_float2(C.acc[n][0] * inv, C.acc[n][1] * inv);
      }
      have = next_seg();
      continue;
    }
    const bool whole = cur.whole();
    const int first = cur.s / per, n_parts = (cur.s + cur.tiles - 1) / per - first + 1;  // CTAs that hold the item
    float* const mine = part + ((size_t)cta * 2 + (cur.s >= v0)) * PA_GROUP * (HD + 2);
    unsigned* const count = pa_counter(J.work, (size_t)cur.row * items_row + cur.item);
    if (h < gq) {
#pragma unroll
      for (int n = 0; n < CH; ++n)
        *reinterpret_cast<float2*>(&S.acc[warp][h][n * 8 + 2 * (lane & 3)]) = make_float2(C.acc[n][0], C.acc[n][1]);
      if ((lane & 3) == 0) {
        S.m[warp][h] = C.m * C.scale;
        S.l[warp][h] = C.l;
      }
    }
    have = next_seg();
    __syncthreads();
    for (int e = tid; e < gq * HD / 4; e += PA_THREADS) {
      const int hh = e / (HD / 4), d = e % (HD / 4) * 4;
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
        const float inv = pa_inverse(L);
        *reinterpret_cast<float4*>(out + hh * HD + d) = make_float4(A.x * inv, A.y * inv, A.z * inv, A.w * inv);
      } else {
        __stcg(reinterpret_cast<float4*>(mine + hh * HD + d), A);
        if (d == 0) __stcg(reinterpret_cast<float2*>(mine + PA_GROUP * HD) + hh, make_float2(M, L));
      }
    }
    if (!whole) {
      __syncthreads();
      if (tid == 0) S.last = pa_arrive(count, n_parts);
      __syncthreads();
      if (S.last) {
        for (int e = tid; e < gq * HD / 4; e += PA_THREADS)
          *(reinterpret_cast<float4*>(out) + e) =
              pa_join<HD>(part, PA_GROUP * (HD + 2), first, n_parts, e / (HD / 4), e % (HD / 4));
        if (tid == 0) *count = 0u;
      }
    }
    __syncthreads();  // the merge area is free again
  }
  cp_async_wait_all();
}

// ---------------------------------------------------------------------------------------
// Rows that share sequences (chunks of prompts, drafted tokens of many sequences): an item is a pack of neighbouring rows of
// one sequence and a kv head.  The CTA's warps share the tiles of K and V, and each has rows of its own: as many as
// fill its eight columns.  So a tile is fetched once for up to 32 rows, where the kernel above fetches it for every
// row.  A pack is a run of rows with the same sequence inside PA_WARPS * rows_warp rows from a multiple of that
// on, so that every CTA finds the same packs from a row's neighbours alone.  The units are the tiles up to the
// longest row's end, dealt to the CTAs as above; a warp passes over those that lie behind all its rows.
// 128 rows at positions 1024-1151 of one sequence, 12 query and 2 kv heads of 128: 23.6 us (28 without sharing), of which
// 5 pass before the first tile, 9.5 in eight units a CTA and 5 in writing and joining the parts; the units are bound by
// the latency of a warp's dependent instructions (issue slots 28 % used, tensor pipe 22 % of active cycles).  Looking
// for entries of V that are not finite, in tiles where a row ends, is 0.2 us of it (up to 5 % with 32/8 heads, in bf16).
constexpr int PC_STAGES = 4;  // tiles of K and V on their way or in use
constexpr int PC_OVER = 2;    // units that an item counts besides its own (those 128 rows: 0 26.8 us, 1 25.7, 2 24.9, 4 26.2)

template <int HD>
struct PagedChunkSmem {
  uint8_t tile[PC_STAGES][2][pa_tok(HD) * HD * 2];  // K, V
  // the parts' factors, while they are joined; before that each warp's copy of a tile of V without what is not finite
  alignas(1024) float f[PA_WARPS][PA_GROUP][PA_MAX_CTAS];
  unsigned long long bad[PA_WARPS];     // positions whose entries of V are not all finite, of a warp's tile
  unsigned valid[PC_STAGES][PA_WARPS];  // of the positions that a warp has looked up
  int seq[PA_THREADS], len[PA_THREADS];             // of the rows, while the packs are counted
  int warp_sum[PA_WARPS];
  int row, base, last;
};

static_assert(sizeof(float) * PA_GROUP * PA_MAX_CTAS % 1024 == 0 && sizeof(float) * PA_GROUP * PA_MAX_CTAS >= 32 * 128 * 2,
              "a warp's copy of a tile: its size and alignment");

struct PagedPack {
  int row, n, seq, len, tiles;  // its rows, their sequence, the longest one's positions and units
  int own;                      // positions of this lane's row
  int item, s, a, b, t;         // as in PagedWalk; t: the next unit
};

template <int HD, bool BF16>
__global__ void __launch_bounds__(PA_THREADS, PA_PER_SM)
    attention_paged_chunk_kernel(const __grid_constant__ gsdlq_paged_attn_job_t J, int subs, int page_shift, int rows_warp) {
  constexpr int TOK = pa_tok(HD), CH = HD / 8;
  constexpr int TILE = TOK * HD * 2;
  constexpr int TOKW = TOK / PA_WARPS;  // positions of a tile that a warp looks up and copies
  typedef typename std::conditional<TOK == 64, unsigned long long, unsigned>::type mask_t;
  constexpr mask_t FULL = ~(mask_t)0;
  extern __shared__ __align__(1024) uint8_t pa_smem[];
  PagedChunkSmem<HD>& S = *reinterpret_cast<PagedChunkSmem<HD>*>(pa_smem);
  const gsdlq_paged_kv_t& kv = J.kv;
  const int tid = threadIdx.x, lane = tid & 31, cta = blockIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int gq_all = J.n_heads / kv.n_kv_heads, items_row = kv.n_kv_heads * subs;
  const int group = PA_WARPS * rows_warp;  // rows of a pack; divides 32
  const size_t kw = (size_t)kv.n_kv_heads * HD;
  // this lane's column: row rl of its warp's, query head hl of the item's
  const int gq_max = min(gq_all, PA_GROUP), rl = (lane >> 2) / gq_max, hl = (lane >> 2) - rl * gq_max;

  pdl_wait();
  pdl_launch_dependents();

  // ---- the launch's units, this CTA's run of them, and the pack where it begins
  auto pack_units = [&](int r0, bool flag) {  // of the pack that row r0 + tid leads, else 0
    const int r = r0 + tid;
    __syncthreads();
    if (r < J.rows) {
      const PagedRow pr = paged_row(kv, J.row_seq, J.pos, r, flag);
      S.seq[tid] = pr.seq;
      S.len[tid] = pr.len;
    }
    __syncthreads();
    if (r >= J.rows || (tid % group != 0 && S.seq[tid - 1] == S.seq[tid])) return 0;
    int len = S.len[tid];
    for (int i = tid + 1; i % group != 0 && r0 + i < J.rows && S.seq[i] == S.seq[tid]; ++i) len = max(len, S.len[i]);
    return len > 0 ? ((len + TOK - 1) / TOK + PC_OVER) * items_row : 0;
  };
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
  int units = 0, n0 = 0, base0 = 0;
  for (int r0 = 0; r0 < J.rows; r0 += PA_THREADS) {
    const int n = pack_units(r0, cta == 0);
    int total;
    const int b = scan(n, total);
    if (r0 == 0) {
      n0 = n;
      base0 = b;
    }
    units += total;
  }
  const int per = max((units + (int)gridDim.x - 1) / (int)gridDim.x, PC_OVER + 1);
  const long long v0l = (long long)per * cta;
  const int v0 = v0l < units ? (int)v0l : units, v1 = min(v0 + per, units);
  for (int r = cta; r < J.rows; r += gridDim.x)  // idle rows
    if (paged_row(kv, J.row_seq, J.pos, r, false).len == 0)
      for (int i = tid; i < J.n_heads * HD; i += PA_THREADS) J.out[(size_t)r * J.n_heads * HD + i] = 0.f;
  if (v0 >= v1) return;
  if (tid == 0) S.row = -1;  // as above
  __syncthreads();
  int before = 0;
  for (int r0 = 0; r0 < J.rows && before <= v0; r0 += PA_THREADS) {
    int n = n0, b = base0, total = 0;
    if (J.rows > PA_THREADS) {
      n = pack_units(r0, false);
      b = scan(n, total);
    } else {
      total = units;
    }
    if (before + b <= v0 && v0 < before + b + n) {
      S.row = r0 + tid;
      S.base = before + b;
    }
    before += total;
  }
  __syncthreads();
  if (S.row < 0) return;

  auto enter = [&](PagedPack& w, int row) {  // the pack that begins with `row`
    const int r = row + lane;
    PagedRow pr = {-1, 0};
    const bool in = lane < group - row % group && r < J.rows;
    if (in) pr = paged_row(kv, J.row_seq, J.pos, r, false);
    const int seq = __shfl_sync(0xffffffffu, pr.seq, 0);
    const unsigned same = __ballot_sync(0xffffffffu, in && pr.seq == seq);
    w.row = row;
    w.n = same == 0xffffffffu ? 32 : __ffs(~same) - 1;
    w.seq = seq;
    w.len = __reduce_max_sync(0xffffffffu, lane < w.n ? pr.len : 0);
    w.tiles = (w.len + TOK - 1) / TOK;
    const int mine = warp * rows_warp + rl, own = __shfl_sync(0xffffffffu, pr.len, mine & 31);
    w.own = rl < rows_warp && mine < w.n ? own : 0;
  };
  auto advance = [&](PagedPack& w) {  // to the next segment; false: the run is at its end
    do {
      const int end = w.s + w.tiles;
      if (++w.item >= items_row) {
        do {
          if (w.row + w.n >= J.rows) return false;
          enter(w, w.row + w.n);
        } while (w.tiles == 0);
        w.item = 0;
      }
      w.s = end + PC_OVER;
      if (w.s >= v1) return false;
      w.a = max(v0 - w.s, 0);
      w.b = min(v1 - w.s, w.tiles);
    } while (w.a >= w.b);
    w.t = w.a;
    return true;
  };
  PagedPack ahead;
  enter(ahead, S.row);
  ahead.item = (v0 - S.base) / (ahead.tiles + PC_OVER) - 1;
  ahead.s = S.base + (ahead.item + 1) * (ahead.tiles + PC_OVER) - ahead.tiles;
  ahead.t = ahead.b = 0;
  PagedPack cur = ahead;
  bool more = true;

  // ---- the tiles
  const uint16_t* const kp = static_cast<const uint16_t*>(kv.k) + (size_t)J.layer * kv.n_pages * kv.page_size * kw;
  const uint16_t* const vp = static_cast<const uint16_t*>(kv.v) + (size_t)J.layer * kv.n_pages * kv.page_size * kw;
  const uint32_t row_bytes = (uint32_t)kw * 2, tiles = smem_u32(S.tile[0][0]);
  struct Unit {
    int page, at, head;  // as above, of position warp * TOKW + lane
  };
  auto look = [&](Unit& U) {
    U.head = U.page = -1;
    while (more && ahead.t >= ahead.b) more = advance(ahead);
    if (!more) return;
    U.head = subs == 1 ? ahead.item : ahead.item / subs;
    const int t = ahead.t * TOK + warp * TOKW + lane;
    if (lane < TOKW && t < ahead.len) {
      const int b = page_shift >= 0 ? t >> page_shift : t / kv.page_size;
      U.at = t - b * kv.page_size;
      U.page = kv.table[(size_t)ahead.seq * kv.max_blocks + b];
      if (U.page < 0) U.page = kv.n_pages;  // missing: reported below
    }
    ++ahead.t;
  };
  const uint32_t dst0 = tiles + pa_at<HD>(warp * TOKW + lane / CH, lane % CH);
  auto copy = [&](const Unit& U, int stage) {
    const bool ok = paged_valid(kv, U.page);
    if (!ok && U.page != -1) raise_flag(GSDLQ_FLAG_BAD_PAGE);
    const unsigned valid = __ballot_sync(0xffffffffu, ok);
    if (U.head >= 0) {
      if (lane == 0) S.valid[stage][warp] = valid;
      const int slot = ok ? U.page * kv.page_size + U.at : -1;
      const size_t off = ((size_t)U.head * HD + (lane % CH) * 8) * 2;
      const char* const ks = reinterpret_cast<const char*>(kp) + off;
      const char* const vs = reinterpret_cast<const char*>(vp) + off;
      const uint32_t dst = dst0 + stage * 2 * TILE;
#pragma unroll
      for (int it = 0; it < TOKW * CH / 32; ++it) {
        const int j = it * (32 / CH);
        const uint32_t x = CH >= 8 ? (uint32_t)((j & 7) << 4) : (uint32_t)(((j >> 1) & 3) << 4);
        const int p = __shfl_sync(0xffffffffu, slot, j + lane / CH);
        const uint32_t d = (dst ^ x) + j * (HD * 2);
        const size_t from = (size_t)(uint32_t)max(p, 0) * row_bytes;
        pa_cp16(d, ks + from, p < 0 ? 0 : 16);
        pa_cp16(d + TILE, vs + from, p < 0 ? 0 : 16);
      }
    }
    cp_async_commit();
  };

  // ---- queries of a segment
  typedef PaColumns<HD, BF16> Cols;
  Cols C;
  typename Cols::Raw x;
  auto first_head = [&](const PagedPack& w, int& gq) {  // of the item's query heads, and how many
    const int g = subs == 1 ? w.item : w.item / subs, sub = subs == 1 ? 0 : w.item - g * subs;
    gq = min(PA_GROUP, gq_all - sub * PA_GROUP);
    return g * gq_all + sub * PA_GROUP;
  };
  int least = 0, most = 0;  // positions of the warp's shortest row (idle ones apart) and of its longest
  auto next_seg = [&]() {
    if (!advance(cur)) return false;
    least = __reduce_min_sync(0xffffffffu, cur.own > 0 ? cur.own : INT_MAX);
    most = __reduce_max_sync(0xffffffffu, cur.own);
    int gq;
    const int head0 = first_head(cur, gq);
    // (columns without a row or a head of their own repeat another's)
    const int r = cur.row + min(warp * rows_warp + min(rl, rows_warp - 1), cur.n - 1);
    Cols::load(x, J.q + r * (J.q_stride ? (size_t)J.q_stride : (size_t)J.n_heads * HD) + (size_t)(head0 + min(hl, gq - 1)) * HD);
    return true;
  };

  Unit U;
  {
    Unit first[PC_STAGES - 1];
#pragma unroll
    for (int i = 0; i < PC_STAGES - 1; ++i) look(first[i]);
#pragma unroll
    for (int i = 0; i < PC_STAGES - 1; ++i) copy(first[i], i);
  }
  look(U);
  bool have = next_seg();
  int stage = 0;
  constexpr size_t PLACE = (size_t)PA_WARPS * PA_GROUP * (HD + 2);  // floats of a CTA's part
  float* const part = pa_parts(J.work) + warp * PA_GROUP * (HD + 2);
  while (have) {
    C.begin(x, J.sm_scale);
    for (; cur.t < cur.b; ++cur.t) {
      asm volatile("cp.async.wait_group %0;" ::"n"(PC_STAGES - 2) : "memory");
      __syncthreads();  // the tile is there, and the one before it is read
      copy(U, stage == 0 ? PC_STAGES - 1 : stage - 1);
      look(U);
      const int limit = cur.own - cur.t * TOK;  // positions of the tile that this lane's row has
      if (cur.t * TOK < most) {
        // Positions of the tile behind a row's end that other rows of the pack use must not reach its sums, not even as 0
        // times what is not finite: the product is taken without such entries, and the rows that use them add them.
        uint8_t* const clean = reinterpret_cast<uint8_t*>(S.f[warp]);
        bool wild = false;
        if (least < min(cur.t * TOK + TOK, cur.len)) {
          const mask_t bad = pa_finite<HD, BF16, mask_t>(S.tile[stage][1], max(least - cur.t * TOK, 0),
                                                         min(cur.len - cur.t * TOK, TOK), clean);
          wild = bad != 0;
          if (wild) S.bad[warp] = bad;  // (not kept in registers through the products: they would spill)
        }
        const uint32_t k0 = tiles + stage * 2 * TILE + pa_at<HD>(lane & 7, lane >> 3);
        const uint32_t v0s = tiles + stage * 2 * TILE + TILE + pa_at<HD>(lane & 15, lane >> 4);
        float p[TOK / 8][2];
        C.scores(p, k0);
        mask_t valid = 0;
#pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) valid |= (mask_t)S.valid[stage][w] << (w * TOKW);
        if (limit < TOK) valid &= limit > 0 ? ((mask_t)1 << limit) - 1 : 0;
        if (valid != FULL) {
          const mask_t mine = valid >> (2 * (lane & 3));
#pragma unroll
          for (int n = 0; n < TOK / 8; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (!((mine >> (n * 8 + j)) & 1)) p[n][j] = -INFINITY;
        }
        typename Cols::Weights W;
        C.weights(W, p);
        C.values(W, !wild ? v0s : smem_u32(clean) + pa_at<HD>(lane & 15, lane >> 4));
        if (wild) C.add_not_finite(S.tile[stage][1], (mask_t)S.bad[warp] & valid);
      }
      stage = stage + 1 == PC_STAGES ? 0 : stage + 1;
    }
    // ---- the segment's result, each warp its rows'
    C.finish();
    if (C.l == 0.f) {  // no position: zeros, also for an idle row among others whose values are not finite
#pragma unroll
      for (int n = 0; n < CH; ++n) C.acc[n][0] = C.acc[n][1] = 0.f;
    }
    int gq;
    const int head0 = first_head(cur, gq), h = lane >> 2;
    const bool mine = rl < rows_warp && hl < gq && warp * rows_warp + rl < cur.n;
    if (cur.a == 0 && cur.b == cur.tiles) {
      if (mine) {
        const float inv = pa_inverse(C.l);
        float* const out = J.out + ((size_t)(cur.row + warp * rows_warp + rl) * J.n_heads + head0 + hl) * HD;
#pragma unroll
        for (int n = 0; n < CH; ++n)
          *reinterpret_cast<float2*>(out + n * 8 + 2 * (lane & 3)) = make_float2(C.acc[n][0] * inv, C.acc[n][1] * inv);
      }
      have = next_seg();
      continue;
    }
    const int first = cur.s / per, n_parts = (cur.s + cur.tiles - 1) / per - first + 1;  // CTAs that hold the item
    float* const place = part + ((size_t)cta * 2 + (cur.s >= v0)) * PLACE;
    if (mine) {
#pragma unroll
      for (int n = 0; n < CH; ++n)
        __stcg(reinterpret_cast<float2*>(place + h * HD + n * 8 + 2 * (lane & 3)), make_float2(C.acc[n][0], C.acc[n][1]));
      if ((lane & 3) == 0) __stcg(reinterpret_cast<float2*>(place + PA_GROUP * HD) + h, make_float2(C.m * C.scale, C.l));
    }
    unsigned* const count = pa_counter(J.work, (size_t)cur.row * items_row + cur.item);
    const int row = cur.row, n = cur.n;
    have = next_seg();
    __syncthreads();
    if (tid == 0) S.last = pa_arrive(count, n_parts);
    __syncthreads();
    if (S.last) {
      constexpr int E = HD == 32 ? 2 : 4;
      const int columns = min(PA_GROUP, rows_warp * gq_max);  // (what columns of no row hold is not looked at)
      pa_factors<HD>(S.f[warp][lane & 7], part, PLACE, first, n_parts, lane & 7, lane >> 3, 4);
      __syncwarp();
      for (int e0 = lane; e0 < columns * (HD / 4); e0 += 32 * E) {
        float4 A[E];
        pa_sums<HD, E, 6>(A, S.f[warp][0], PA_MAX_CTAS, part, PLACE, first, n_parts, e0, 32);
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const int e = e0 + 32 * k, c = e / (HD / 4), cr = c / gq_max, ch = c - cr * gq_max, r = warp * rows_warp + cr;
          if (c < columns && ch < gq && r < n)
            *(reinterpret_cast<float4*>(J.out + ((size_t)(row + r) * J.n_heads + head0 + ch) * HD) + e % (HD / 4)) = A[k];
        }
      }
      if (tid == 0) *count = 0u;
    }
  }
  cp_async_wait_all();
}

// ---------------------------------------------------------------------------------------
// host side
template <int HD, bool BF16>
static int launch_attention_paged(const gsdlq_paged_attn_job_t& J, int subs, cudaStream_t st) {
  constexpr int smem = (int)sizeof(PagedAttnSmem<HD>), smem_chunk = (int)sizeof(PagedChunkSmem<HD>);
  static_assert(PA_PER_SM * (smem + 1024) <= 228 * 1024 && PA_PER_SM * (smem_chunk + 1024) <= 228 * 1024,
                "shared memory of the CTAs of an SM");
  static std::atomic<bool> set[64];  // the opt-in shared memory size, once per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return record_cuda_error(e);
  if (dev >= 64 || !set[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(attention_paged_kernel<HD, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(attention_paged_chunk_kernel<HD, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               smem_chunk);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev < 64) set[dev].store(true, std::memory_order_release);
  }
  const int grid = std::min(PA_PER_SM * num_sms(), PA_MAX_CTAS);
  const int ps = J.kv.page_size, shift = ps & (ps - 1) ? -1 : __builtin_ctz((unsigned)ps);
  // Several rows a sequence of the table on average (which rows share one is known on the device only), and enough of
  // them: the tiles are worth sharing.  A CTA's warps without rows are idle then, and its start and end take 4-5 us
  // more.  One tile per row against shared tiles, us:
  //   16 sequences of 1500, 32/32 heads of 64: 2 rows each 62 / 73, 3 rows 83 / 76; 32/8 of 128: 3 rows 51 / 49, 8 rows
  //   99 / 45; 12/2 of 128: 3 rows 18.7 / 22.9, 4 rows 23.4 / 22.3; 16/2 of 64: 3 rows 13.5 / 15.9, 4 rows 15.6 / 15.3
  //   one sequence of 1500, 32/32 of 64: 4 rows 14.9 / 13.4; 32/8 of 128: 8 rows 15.3 / 18.9, 16 rows 20.9 / 20.2;
  //   12/2 of 128: 32 rows 16.6 / 19.6, 128 rows 28 / 23
  const int gq = J.n_heads / J.kv.n_kv_heads;
  if (J.row_seq != nullptr && J.rows >= (gq <= 4 ? 3 : 4) * J.kv.n_seqs && (long long)J.rows * J.kv.n_kv_heads >= 128) {
    const int rows_warp = gq == 1 ? 8 : gq == 2 ? 4 : gq <= 4 ? 2 : 1;  // rows whose heads fill a warp's columns
    return launch_pdl(attention_paged_chunk_kernel<HD, BF16>, grid, PA_THREADS, smem_chunk, st, 1, J, subs, shift, rows_warp);
  }
  return launch_pdl(attention_paged_kernel<HD, BF16>, grid, PA_THREADS, smem, st, 1, J, subs, shift);
}

}  // namespace gsdlq

using namespace gsdlq;

extern "C" {

int gsdlq_attention_paged_work_size(int rows, int n_heads, int n_kv_heads, int head_dim, size_t* bytes) {
  if (!bytes || rows <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads) return GSDLQ_ERR_INVALID;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) return GSDLQ_ERR_INVALID;
  *bytes = attention_paged_work(rows, n_heads, n_kv_heads);
  return GSDLQ_OK;
}

int gsdlq_attention_paged(const gsdlq_paged_attn_job_t* job, gsdlq_stream_t stream) {
  if (!job || !pool_ok(job->kv) || !rows_ok(job->kv, job->row_seq, job->pos, job->rows)) return GSDLQ_ERR_INVALID;
  const gsdlq_paged_attn_job_t& J = *job;
  if (!J.q || !J.out || !J.work || J.layer < 0 || J.layer >= J.kv.layers) return GSDLQ_ERR_INVALID;
  if (!std::isfinite(J.sm_scale)) return GSDLQ_ERR_INVALID;
  if (J.n_heads <= 0 || J.n_heads % J.kv.n_kv_heads || (long long)J.n_heads * J.kv.head_dim > INT32_MAX)
    return GSDLQ_ERR_INVALID;
  if (!aligned16(J.q) || !aligned16(J.out) || !aligned16(J.work) || J.q_stride % 4) return GSDLQ_ERR_INVALID;
  if (J.q_stride && J.q_stride < J.n_heads * J.kv.head_dim) return GSDLQ_ERR_INVALID;
  if (J.work_bytes < attention_paged_work(J.rows, J.n_heads, J.kv.n_kv_heads)) return GSDLQ_ERR_INVALID;
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
