// Attention of one query token per session over the quantised cache (layout: mc_kv.cuh).
//
// With keys and values held as center + scale * m, m an 8-bit integer, both products of the
// attention have integer operands on one side:
//   s_j = a (kscale_j * sum_d q_d m_jd + kcenter_j * sum_d q_d)
//   o_d = sum_j (p_j vscale_j) m_jd + sum_j p_j vcenter_j,   p_j = exp(s_j - max)
// and both run as 8-bit matrix products with exact 32-bit sums: the codes are the MMA's B operand
// as they lie in memory (an and-or per word for 4 bits, nothing for 8), and the other side is cut
// into 8-bit planes. A query row becomes PLANES signed digits of base 254 relative to its largest
// element, a row of weights p_j vscale_j becomes a fixed-point integer of 16 bits (PLANES 2) or 23
// bits (3) relative to the tile's largest, whose bytes are the planes: adding 2^23 to
// the scaled weight leaves them in the mantissa, so cutting costs one fused multiply-add a weight.
// PLANES is 3 for float32 queries (errors of 2^-23 and below, as float32 itself) and 2 for 16-bit
// ones (2^-16, far below their rounding).
//
// An m16n8k32 MMA has rows 0-7 = the first plane of up to eight query heads that share a key/value
// head, rows 8-15 = their second plane, so both planes of a score end up in the same thread. The
// score layout of four MMAs over slots 4g + i (i = MMA) is, in turn, exactly the A-operand
// layout of the weights for the value product if its k order is taken as the thread's own slots:
// the scores never leave their registers.
//
// What bounds it: reading the codes. Per 32 slots of a 128-wide head in 4 bits a warp reads 4.3 KB
// and issues about 450 instructions for any number of heads up to eight.
#pragma once
#include "mc_kv.cuh"

namespace mc {
namespace kv {

constexpr int kAttendWarps = 4;
constexpr int kAttendRows = 8;          // query heads of one item
constexpr int kMaxPartials = 2048;      // partial results (items x pieces) that fit the workspace
constexpr int kMaxPieces = 128;         // pieces of one item

struct AttendArgs {
  Cache c;
  Rows q, out;
  int n, q_heads, group, row_groups, window, dtype;
  int vec;               // rows of q and out take 16-byte (eight elements) and pair accesses
  int pieces;            // CTAs an item's slots are split over
  const int *sess, *lens;
  float scale;           // of the scores, times log2(e)
  float* partial;        // [item][piece][8][2 + dim]: maximum, sum, weighted values
  int* arrived;          // [item] pieces done (zero between calls)
};

// d += a x b, a and b 8-bit (A unsigned for the weights, signed for the queries), 32-bit sums
__device__ __forceinline__ void mma_s8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Eight consecutive elements.
template <class T>
__device__ __forceinline__ void load8(float (&x)[8], const T* p, bool vec) {
  if constexpr (sizeof(T) == 4) {
    if (vec) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(p)), v = __ldg(reinterpret_cast<const float4*>(p) + 1);
      x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
      return;
    }
  } else {
    if (vec) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = to_float<T>(e[i]);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_float<T>(p[i]);
}

__device__ __forceinline__ void load_query(float (&x)[8], const void* p, long long i, int dtype, bool vec) {
  if (dtype == kF32) load8<float>(x, static_cast<const float*>(p) + i, vec);
  else if (dtype == kF16) load8<__half>(x, static_cast<const __half*>(p) + i, vec);
  else load8<__nv_bfloat16>(x, static_cast<const __nv_bfloat16*>(p) + i, vec);
}
__device__ __forceinline__ uint32_t word_of(const uint4& w, int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
__device__ __forceinline__ void store_element(void* p, long long i, int dtype, float x) {
  if (dtype == kF32) static_cast<float*>(p)[i] = x;
  else if (dtype == kF16) static_cast<__half*>(p)[i] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

// Elements i and i + 1, i even.
__device__ __forceinline__ void store_pair(void* p, long long i, int dtype, bool vec, float x, float y) {
  if (!vec) {
    store_element(p, i, dtype, x);
    store_element(p, i + 1, dtype, y);
  } else if (dtype == kF32) {
    *reinterpret_cast<float2*>(static_cast<float*>(p) + i) = make_float2(x, y);
  } else if (dtype == kF16) {
    *reinterpret_cast<__half2*>(static_cast<__half*>(p) + i) = __floats2half2_rn(x, y);
  } else {
    *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p) + i) = __floats2bfloat162_rn(x, y);
  }
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint32_t* p) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 x = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 x = reinterpret_cast<const uint2*>(p)[i];
      w[2 * i] = x.x, w[2 * i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = p[i];
  }
}

// The slots a query sees, in slot order: [0, e0) and [s1, e1), as tiles of TS slots.
struct SlotSpan {
  int e0, s1, e1;
  int tiles0, first1, tiles;
};
template <int TS>
__device__ __forceinline__ SlotSpan slot_span(const Cache& c, int len, int window) {
  SlotSpan s{0, 0, 0, 0, 0, 0};
  if (len <= 0) return s;
  s.e0 = min(c.sinks, len);
  if (len > c.sinks) {
    int lo = max(c.sinks, len - c.ring);
    if (window > 0) lo = max(lo, len - window);
    const int a = (lo - c.sinks) % c.ring, count = len - lo;  // in [1, ring]
    s.s1 = c.sinks + a;
    if (a + count > c.ring) {
      s.e0 = c.sinks + a + count - c.ring;
      s.e1 = c.slots;
    } else {
      s.e1 = s.s1 + count;
    }
  }
  s.tiles0 = (s.e0 + TS - 1) / TS;
  s.first1 = max(s.s1 / TS, s.tiles0);
  s.tiles = s.tiles0 + max(0, (s.e1 + TS - 1) / TS - s.first1);
  return s;
}

constexpr int attend_slots(int bits, int planes) { return bits == 4 && planes == 2 ? 64 : 32; }
constexpr int attend_stage_bytes(int bits, int dim, int planes) {
  return attend_slots(bits, planes) * (2 * dim * bits / 8 + 8);
}
// Tiles in flight per warp: what fits three CTAs of four warps on an SM.
constexpr int attend_stages(int bits, int dim, int planes) {
  const int n = 71680 / (kAttendWarps * attend_stage_bytes(bits, dim, planes));
  return n > 4 ? 4 : n < 2 ? 2 : n;
}
constexpr int attend_smem(int bits, int dim, int planes) {
  const int ring = kAttendWarps * attend_stages(bits, dim, planes) * attend_stage_bytes(bits, dim, planes);
  const int join = kAttendWarps * kAttendRows * (dim + 2) * 4;  // the warps' results, in the same place
  return ring > join ? ring : join;
}

// Where a warp is in its work: an item (a session's up to eight query heads of one key/value head)
// and a tile of its visible slots.
struct AttendCursor {
  long long item;
  int t, end;
  int tiles0, first1;
  const uint8_t* region;
};

// WPI warps of a CTA share an item: 1 gives every warp items of its own, one after the other with
// the next one's tiles already in flight; kAttendWarps gives the CTA one piece of one item.
template <int BITS, int DIM, int PLANES, int WPI>
__global__ void __launch_bounds__(kAttendWarps * 32, 3) attend_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int TS = attend_slots(BITS, PLANES), HALVES = TS / 32;
  constexpr int CB = DIM * BITS / 8;             // code bytes per slot
  constexpr int KS = (DIM + 31) / 32;            // MMA steps along the dimensions
  constexpr int NI = BITS == 4 ? DIM / 16 : DIM / 8;  // value words of a group of slots per thread
  constexpr int NT = DIM / 8;                    // 8-column tiles of the output
  constexpr float kOne = BITS == 4 ? 0.125f : 1.0f;   // the MMA's codes are 8m (4 bits) or m
  constexpr int STAGES = attend_stages(BITS, DIM, PLANES), STAGE = attend_stage_bytes(BITS, DIM, PLANES);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kAttendWarps][STAGES];
  const Cache& c = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, cc = lane & 3;
  uint8_t* ring = smem + warp * STAGES * STAGE;
  uint64_t* bars = full[warp];
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(bars + i, 1);
    fence_barrier_init();
  }
  __syncwarp();

  const int per = c.heads * a.row_groups;
  const long long items = (long long)a.n * per, stride = WPI == 1 ? (long long)gridDim.x * kAttendWarps : items;
  const int piece = WPI == 1 ? 0 : blockIdx.y;
  const int part = WPI == 1 ? 0 : piece * WPI + warp, parts = WPI == 1 ? 1 : a.pieces * WPI;

  auto open = [&](AttendCursor& u, SlotSpan& span) {
    const int b = (int)(u.item / per), head = (int)(u.item % per) / a.row_groups;
    int session = a.sess ? a.sess[b] : b, len = 0;
    if ((unsigned)session < (unsigned)c.sessions) {
      len = a.lens[b];
    } else {
      if (lane == 0) atomicExch(c.error, 1);
      session = 0;
    }
    span = slot_span<TS>(c, len, a.window);
    u.t = (int)((long long)span.tiles * part / parts);
    u.end = (int)((long long)span.tiles * (part + 1) / parts);
    u.tiles0 = span.tiles0;
    u.first1 = span.first1;
    u.region = region_of(c, session, head);
  };
  auto slot_at = [](const AttendCursor& u, int t) { return (t < u.tiles0 ? t : u.first1 + t - u.tiles0) * TS; };

  // ---- the producer's side: lane 0 copies the tiles of this warp's items in their order
  AttendCursor next{WPI == 1 ? (long long)blockIdx.x * kAttendWarps + warp : (long long)blockIdx.x, 0, 0, 0, 0, nullptr};
  AttendCursor cur = next;
  int issued = 0;
  SlotSpan scratch;
  if (next.item < items) open(next, scratch);
  auto issue = [&]() {
    while (next.t >= next.end) {
      if (next.item >= items) return;
      next.item += stride;
      if (next.item >= items) return;
      open(next, scratch);
    }
    if (lane == 0) {
      const int slot0 = slot_at(next, next.t), stage = issued % STAGES;
      uint8_t* dst = ring + stage * STAGE;
      const uint8_t* codes = next.region + (long long)slot0 * CB;
      const uint8_t* params = next.region + params_offset(c) + (long long)slot0 * 4;
      mbar_arrive_expect_tx(bars + stage, STAGE);
      bulk_load(dst, codes, TS * CB, bars + stage);
      bulk_load(dst + TS * CB, codes + values_offset(c), TS * CB, bars + stage);
      bulk_load(dst + 2 * TS * CB, params, TS * 4, bars + stage);
      bulk_load(dst + 2 * TS * CB + TS * 4, params + (long long)c.cap * 4, TS * 4, bars + stage);
    }
    ++issued;
    ++next.t;
  };
  for (int i = 0; i < STAGES; ++i) issue();

  int done = 0;
  bool ok = true;  // false after a wait gave up
  float o[NT][2];
  float top, total, csum;
  int b, rows, h0;
  for (; cur.item < items; cur.item += stride) {
    SlotSpan span;
    open(cur, span);
    b = (int)(cur.item / per);
    const int hr = (int)(cur.item % per), head = hr / a.row_groups, rg = hr % a.row_groups;
    rows = min(kAttendRows, a.group - rg * kAttendRows);  // query heads of this item
    h0 = head * a.group + rg * kAttendRows;

    // ---- the queries as digit planes: thread (r, cc) holds row r's dimensions 8w..8w+7, w = cc + 4i
    uint32_t qa[KS][PLANES][2];
    float qstep, qsum = 0.f;
    {
      float x[KS][8], big = 0.f;
      const long long base = b * a.q.row + (h0 + r) * a.q.head;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int w = cc + 4 * i;
        const bool in = r < rows && 8 * w < DIM;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
        if (in) load_query(x[i], a.q.p, base + 8 * w, a.dtype, a.vec);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          qsum = __fadd_rn(qsum, x[i][e]);
          big = fmaxf(big, fabsf(x[i][e]));
        }
      }
#pragma unroll
      for (int x = 1; x <= 2; x <<= 1) {
        qsum = __fadd_rn(qsum, __shfl_xor_sync(~0u, qsum, x));
        big = fmaxf(big, __shfl_xor_sync(~0u, big, x));
      }
      const float inv = row_inv_step(big);
      // a non-finite query has no digits: its scores become NaN by qsum
      qstep = __fmul_rn(__fmul_rn(row_step(big), a.scale), kOne / 254.0f);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        uint32_t u[8][3];
#pragma unroll
        for (int e = 0; e < 8; ++e) slice3_bits(x[i][e], inv, u[e][0], u[e][1], u[e][2]);
#pragma unroll
        for (int p = 0; p < PLANES; ++p) {
          qa[i][p][0] = pack_low_bytes(u[0][p], u[1][p], u[2][p], u[3][p]);
          qa[i][p][1] = pack_low_bytes(u[4][p], u[5][p], u[6][p], u[7][p]);
        }
      }
      qsum = __fmul_rn(qsum, a.scale);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = 0.f;
    top = -INFINITY, total = 0.f, csum = 0.f;

    for (int t = cur.t; t < cur.end; ++t) {
      const int slot0 = slot_at(cur, t), stage = done % STAGES;
      ok = __all_sync(~0u, ok && mbar_wait_or_abort(bars + stage, (done / STAGES) & 1, kErrWaitFull));
      if (!ok) break;
      const uint8_t* kcodes = ring + stage * STAGE;
      const uint8_t* vcodes = kcodes + TS * CB;
      const uint32_t* kparam = reinterpret_cast<const uint32_t*>(vcodes + TS * CB);
      const uint32_t* vparam = kparam + TS;
      // ---- scores: s[h][i][u] of slot 32h + 8cc + 4u + i
      float s[HALVES][4][2];
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        const uint4* kp4 = reinterpret_cast<const uint4*>(kparam + 32 * h + 8 * cc);
        const uint4 kp[2] = {kp4[0], kp4[1]};
        const uint8_t* kc = kcodes + (8 * h + r) * 4 * CB;
        int acc[4][4] = {}, acc3[4][4] = {};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const int w = cc + 4 * i;
          uint32_t b0[4], b1[4];
          if (DIM % 32 == 0 || 8 * w < DIM) {
            if constexpr (BITS == 4) {
              uint32_t x[4];
              load_words<4>(x, reinterpret_cast<const uint32_t*>(kc + 16 * w));
#pragma unroll
              for (int j = 0; j < 4; ++j) b0[j] = low_codes(x[j]), b1[j] = high_codes(x[j]);
            } else {
              load_words<4>(b0, reinterpret_cast<const uint32_t*>(kc + 32 * w));
              load_words<4>(b1, reinterpret_cast<const uint32_t*>(kc + 32 * w + 16));
            }
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) b0[j] = b1[j] = 0;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma_s8s8(acc[j], qa[i][0][0], qa[i][1][0], qa[i][0][1], qa[i][1][1], b0[j], b1[j]);
            if constexpr (PLANES == 3) mma_s8s8(acc3[j], qa[i][2][0], 0u, qa[i][2][1], 0u, b0[j], b1[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            // |first| <= 128 * 127 * 127, so 254 * first + second fits 32 bits
            float f = (float)(acc[j][u] * 254 + acc[j][2 + u]);
            if constexpr (PLANES == 3) f = __fmaf_rn((float)acc3[j][u], 1.0f / 254.0f, f);
            const uint32_t w = word_of(kp[u], j);
            s[h][j][u] = __fmaf_rn(__fmul_rn(f, qstep), param_scale(w), __fmul_rn(param_center(w), qsum));
          }
        }
      }
      const bool whole = slot0 + TS <= span.e0 || (slot0 >= span.s1 && slot0 + TS <= span.e1);
      if (!whole) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int slot = slot0 + 32 * h + 8 * cc + 4 * u + j;
              if (!(slot < span.e0 || (slot >= span.s1 && slot < span.e1))) s[h][j][u] = -INFINITY;
            }
      }
      // ---- running maximum and sum (a row's slots are on the four threads of its quad)
      float m = top;
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) m = fmaxf(m, fmaxf(s[h][j][0], s[h][j][1]));
      m = fmaxf(m, __shfl_xor_sync(~0u, m, 1));
      m = fmaxf(m, __shfl_xor_sync(~0u, m, 2));
      if (__any_sync(~0u, m > top)) {
        const float keep = top == -INFINITY ? 0.f : exp2_fast(__fsub_rn(top, m));
        total = __fmul_rn(total, keep);
        csum = __fmul_rn(csum, keep);
#pragma unroll
        for (int i = 0; i < NT; ++i) o[i][0] = __fmul_rn(o[i][0], keep), o[i][1] = __fmul_rn(o[i][1], keep);
        top = m;
      }
      // ---- weights p, their sum, and p * vscale in place of the scores
      float pmax = 0.f;
      const float shift = top == -INFINITY ? 0.f : top;  // nothing but scores of minus infinity so far
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        const uint4* vp4 = reinterpret_cast<const uint4*>(vparam + 32 * h + 8 * cc);
        const uint4 vp[2] = {vp4[0], vp4[1]};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float p = exp2_fast(__fsub_rn(s[h][j][u], shift));
            uint32_t w = word_of(vp[u], j);
            if (!whole && s[h][j][u] == -INFINITY) w = 0;  // a hidden slot may hold a scale of NaN
            total = __fadd_rn(total, p);
            csum = __fmaf_rn(p, param_center(w), csum);
            s[h][j][u] = __fmul_rn(p, param_scale(w));
            pmax = fmaxf(pmax, s[h][j][u]);
          }
      }
      pmax = fmaxf(pmax, __shfl_xor_sync(~0u, pmax, 1));
      pmax = fmaxf(pmax, __shfl_xor_sync(~0u, pmax, 2));
      // below 1e-30 the inverse leaves float32's range: such weights count as nothing
      constexpr float kFull = PLANES == 3 ? 8388607.0f : 65535.0f;
      const float inv = pmax > 1e-30f ? __fdividef(kFull, pmax) : 0.f;
      const float unit = __fmul_rn(pmax > 1e-30f ? pmax : 0.f, kOne / kFull);
      // ---- the weights' bytes as A operands: plane 0 (highest) in rows 0-7, plane 1 in rows 8-15
      uint32_t pa[HALVES][PLANES][2];
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            x[j] = __float_as_uint(fminf(__fmaf_rn(s[h][j][u], inv, 8388608.0f), 8388608.0f + kFull));
          const uint32_t lo01 = __byte_perm(x[0], x[1], 0x5140), lo23 = __byte_perm(x[2], x[3], 0x5140);
          pa[h][PLANES - 1][u] = __byte_perm(lo01, lo23, 0x5410);  // bytes 0
          pa[h][PLANES - 2][u] = __byte_perm(lo01, lo23, 0x7632);  // bytes 1
          if constexpr (PLANES == 3) {
            const uint32_t hi01 = __byte_perm(x[0], x[1], 0x0062), hi23 = __byte_perm(x[2], x[3], 0x0062);
            pa[h][0][u] = __byte_perm(hi01, hi23, 0x5410);  // bits 16-22
          }
        }
      // ---- the weighted values
      constexpr int STEP = NI % 4 == 0 ? 4 : NI % 2 == 0 ? 2 : 1;
#pragma unroll
      for (int i0 = 0; i0 < NI; i0 += STEP) {
        uint32_t v[HALVES][2][STEP];
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            load_words<STEP>(v[h][u], reinterpret_cast<const uint32_t*>(vcodes + (8 * h + 2 * cc + u) * 4 * CB) + r * NI + i0);
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
#pragma unroll
          for (int nib = 0; nib < (BITS == 4 ? 2 : 1); ++nib) {
            int acc[4] = {}, acc3[4] = {};
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
              uint32_t b0 = v[h][0][i], b1 = v[h][1][i];
              if constexpr (BITS == 4) {
                b0 = nib ? high_codes(b0) : low_codes(b0);
                b1 = nib ? high_codes(b1) : low_codes(b1);
              }
              mma_u8s8(acc, pa[h][0][0], pa[h][1][0], pa[h][0][1], pa[h][1][1], b0, b1);
              if constexpr (PLANES == 3) mma_u8s8(acc3, pa[h][2][0], 0u, pa[h][2][1], 0u, b0, b1);
            }
            const int nt = BITS == 4 ? 2 * (i0 + i) + nib : i0 + i;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              // |first| <= 255 * 127 * 64, so 256 * first + second fits 32 bits
              float f = (float)(acc[u] * 256 + acc[2 + u]);
              if constexpr (PLANES == 3) f = __fmaf_rn(f, 256.0f, (float)acc3[u]);
              o[nt][u] = __fmaf_rn(f, unit, o[nt][u]);
            }
          }
        }
      }
      ++done;
      __syncwarp();  // every lane has read the stage: it takes the next tile
      issue();
    }
    if (!ok) break;
    // ---- the row's sums over its quad; the centers' share goes to every dimension
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      total = __fadd_rn(total, __shfl_xor_sync(~0u, total, x));
      csum = __fadd_rn(csum, __shfl_xor_sync(~0u, csum, x));
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = __fadd_rn(o[i][0], csum), o[i][1] = __fadd_rn(o[i][1], csum);
    // thread (r, cc) has dimensions 8i + 2cc and 8i + 2cc + 1 of row r
    if constexpr (WPI == 1) {
      if (r < rows) {
        const float inv = total == 0.f ? 0.f : __fdiv_rn(1.0f, total);
        const long long base = b * a.out.row + (h0 + r) * a.out.head;
#pragma unroll
        for (int i = 0; i < NT; ++i)
          store_pair(a.out.p, base + 8 * i + 2 * cc, a.dtype, a.vec, __fmul_rn(o[i][0], inv), __fmul_rn(o[i][1], inv));
      }
    }
  }
  // a wait that gave up: never leave with copies in flight into this warp's buffers
  if (!ok && lane == 0)
    for (; done < issued; ++done) mbar_wait(bars + done % STAGES, (done / STAGES) & 1, kErrWaitFull);

  if constexpr (WPI != 1) {
    constexpr int W = 2 + DIM;  // maximum, sum, weighted values of a row
    float* results = reinterpret_cast<float*>(smem);  // [warp][row][W], over the ring of tiles
    __shared__ float keeps[kMaxPieces * kAttendRows];
    __shared__ int last;
    const long long item = blockIdx.x;
    __syncthreads();
    {
      float* mine = results + (warp * kAttendRows + r) * W;
      if (cc == 0) mine[0] = top, mine[1] = total;
#pragma unroll
      for (int i = 0; i < NT; ++i) mine[2 + 8 * i + 2 * cc] = o[i][0], mine[3 + 8 * i + 2 * cc] = o[i][1];
    }
    __syncthreads();
    float* out = a.partial + (item * a.pieces + piece) * kAttendRows * W;
    for (int e = threadIdx.x; e < rows * DIM; e += kAttendWarps * 32) {
      const int row = e / DIM, d = e % DIM;
      float m = -INFINITY, l = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < WPI; ++w) m = fmaxf(m, results[(w * kAttendRows + row) * W]);
#pragma unroll
      for (int w = 0; w < WPI; ++w) {
        const float* q = results + (w * kAttendRows + row) * W;
        // a part without visible slots has maximum -inf and sums of zero
        const float keep = q[0] == -INFINITY ? 0.f : exp2_fast(__fsub_rn(q[0], m));
        l = __fmaf_rn(q[1], keep, l);
        x = __fmaf_rn(q[2 + d], keep, x);
      }
      if (a.pieces == 1) {
        store_element(a.out.p, b * a.out.row + (h0 + row) * a.out.head + d, a.dtype, l == 0.f ? 0.f : __fdiv_rn(x, l));
      } else {
        if (d == 0) out[row * W] = m, out[row * W + 1] = l;
        out[row * W + 2 + d] = x;
      }
    }
    if (a.pieces == 1) return;
    // ---- the item's last CTA to arrive joins the pieces, in their order
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(a.arrived + item, 1) == a.pieces - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    const float* all = a.partial + item * a.pieces * kAttendRows * W;
    // the pieces' factors: a quarter-warp's worth of threads per row
    {
      const int row = threadIdx.x / 16, l16 = threadIdx.x % 16;  // 128 threads: eight rows
      float m = -INFINITY, l = 0.f;
      if (row < rows) {
        for (int p = l16; p < a.pieces; p += 16) m = fmaxf(m, __ldcg(all + (p * kAttendRows + row) * W));
      }
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, x));
      if (row < rows) {
        for (int p = l16; p < a.pieces; p += 16) {
          const float pm = __ldcg(all + (p * kAttendRows + row) * W), keep = pm == -INFINITY ? 0.f : exp2_fast(__fsub_rn(pm, m));
          keeps[row * kMaxPieces + p] = keep;
          l = __fmaf_rn(__ldcg(all + (p * kAttendRows + row) * W + 1), keep, l);
        }
      }
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) l = __fadd_rn(l, __shfl_xor_sync(~0u, l, x));
      if (l16 == 0) results[row] = l;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * (DIM / 2); e += kAttendWarps * 32) {
      const int row = e / (DIM / 2), d = 2 * (e % (DIM / 2));
      float x0 = 0.f, x1 = 0.f;
#pragma unroll 16
      for (int p = 0; p < a.pieces; ++p) {
        const float2 q = __ldcg(reinterpret_cast<const float2*>(all + (p * kAttendRows + row) * W + 2 + d));
        const float keep = keeps[row * kMaxPieces + p];
        x0 = __fmaf_rn(q.x, keep, x0);
        x1 = __fmaf_rn(q.y, keep, x1);
      }
      const float l = results[row], inv = l == 0.f ? 0.f : __fdiv_rn(1.0f, l);
      store_pair(a.out.p, b * a.out.row + (h0 + row) * a.out.head + d, a.dtype, a.vec, __fmul_rn(x0, inv), __fmul_rn(x1, inv));
    }
    if (threadIdx.x == 0) a.arrived[item] = 0;
  }
}

struct AttendVariant {
  void (*f)(AttendArgs);
  int smem;
};

template <int BITS, int DIM>
inline AttendVariant attend_variant(int planes, bool split) {
  if (planes == 3)
    return {split ? attend_kernel<BITS, DIM, 3, kAttendWarps> : attend_kernel<BITS, DIM, 3, 1>, attend_smem(BITS, DIM, 3)};
  return {split ? attend_kernel<BITS, DIM, 2, kAttendWarps> : attend_kernel<BITS, DIM, 2, 1>, attend_smem(BITS, DIM, 2)};
}

template <int BITS>
inline AttendVariant attend_variant_of(int dim, int planes, bool split) {
  switch (dim) {
    case 16: return attend_variant<BITS, 16>(planes, split);
    case 32: return attend_variant<BITS, 32>(planes, split);
    case 48: return attend_variant<BITS, 48>(planes, split);
    case 64: return attend_variant<BITS, 64>(planes, split);
    case 80: return attend_variant<BITS, 80>(planes, split);
    case 96: return attend_variant<BITS, 96>(planes, split);
    case 112: return attend_variant<BITS, 112>(planes, split);
    default: return attend_variant<BITS, 128>(planes, split);
  }
}

}  // namespace kv
}  // namespace mc
