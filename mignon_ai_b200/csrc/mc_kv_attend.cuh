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
  int pieces;            // CTAs an item's slots are split over; 0: every warp has items of its own
  const int *sess, *lens;
  float scale;           // of the scores, times log2(e)
  float* partial;        // [item][piece][8][2 + dim]: maximum, sum, weighted values
  int* arrived;          // [item] pieces done (zero between calls)
};

// d (+)= a x b on 8-bit operands with 32-bit sums: B signed, A signed (the queries) or unsigned (the
// weights). FIRST: d starts from zero.
template <bool UNSIGNED, bool FIRST>
__device__ __forceinline__ void mma_8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
#define MC_MMA_8(TYPE)                                                                                                    \
  if constexpr (FIRST)                                                                                                    \
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32." TYPE ".s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};" \
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])                                                         \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));                                         \
  else                                                                                                                    \
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32." TYPE ".s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};" \
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])                                                         \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
  if constexpr (UNSIGNED) {
    MC_MMA_8("u8");
  } else {
    MC_MMA_8("s8");
  }
#undef MC_MMA_8
}

// Two float32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b));
  return d;
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

// CTAs that share an SM: four where 128 registers a thread hold the work.
constexpr int attend_ctas(int dim) { return dim <= 64 ? 4 : 3; }
// Slots of a tile: 64 (two blocks) where two tiles a warp then fit shared memory, and where the third
// plane leaves the registers for it.
constexpr int attend_slots(int bits, int dim, int planes) {
  return bits == 4 ? (planes == 3 && dim > 64 ? 32 : 64) : dim <= 32 ? 64 : 32;
}
constexpr int attend_stage_bytes(int bits, int dim, int planes) {
  return attend_slots(bits, dim, planes) / kBlockSlots * block_bytes(dim * bits / 8);
}
// Tiles in flight per warp.
constexpr int attend_stages(int bits, int dim, int planes) {
  const int n = (221184 / attend_ctas(dim) - 1024) / (kAttendWarps * attend_stage_bytes(bits, dim, planes));
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
  unsigned item;  // items fit 31 bits, and a stride beyond them 32
  int t, end;
  int tiles0, first1;
  const uint8_t* region;
};

// With few heads to an item the MMA's eight rows repeat them: HEADS rows of heads (8, 4 or 1), and the
// rows of one head take different slots of the tile (row r: HEADS 4, the groups 2cc + r / 4; HEADS 1,
// the slot r % 4 of those), so that no thread does another's exponentials. They share the
// running maximum, and their sums meet at the end of the item.
//
// With a.pieces a CTA has one piece of one item; without, every warp goes through items of its own,
// the next one's tiles already in flight.
template <int BITS, int DIM, int PLANES, int HEADS>
__global__ void __launch_bounds__(kAttendWarps * 32, attend_ctas(DIM)) attend_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int TS = attend_slots(BITS, DIM, PLANES), HALVES = TS / 32;
  constexpr int NJ = HEADS == 1 ? 1 : 4, NU = HEADS == 8 ? 2 : 1;  // slots of a half that a thread weighs: NJ x NU
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

  const unsigned per = c.heads * a.row_groups, items = a.n * per;
  const unsigned stride = a.pieces ? items : gridDim.x * kAttendWarps;
  const int piece = blockIdx.y;
  const unsigned part = piece * kAttendWarps + warp, parts = a.pieces * kAttendWarps;
  const int row_head = HEADS == 8 ? r : HEADS == 4 ? r & 3 : 0;  // the thread's query head in the item
  const int my_u = r >> 2, my_j = r & 3;                         // and its slots: see above

  auto open = [&](AttendCursor& u, SlotSpan& span) {
    const unsigned b = u.item / per, hr = u.item - b * per, head = a.row_groups == 1 ? hr : hr / a.row_groups;
    int session = a.sess ? a.sess[b] : b, len = 0;
    if ((unsigned)session < (unsigned)c.sessions) {
      len = a.lens[b];
    } else {
      if (lane == 0) atomicExch(c.error, 1);
      session = 0;
    }
    span = slot_span<TS>(c, len, a.window);
    u.t = 0;
    u.end = span.tiles;
    if (a.pieces) {  // an even share of the tiles, the first parts one more
      const unsigned share = (unsigned)span.tiles / parts, more = (unsigned)span.tiles - share * parts;
      u.t = part * share + min(part, more);
      u.end = u.t + share + (part < more ? 1 : 0);
    }
    u.tiles0 = span.tiles0;
    u.first1 = span.first1;
    u.region = region_of(c, session, head);
  };
  auto slot_at = [](const AttendCursor& u, int t) { return (t < u.tiles0 ? t : u.first1 + t - u.tiles0) * TS; };

  // ---- the producer's side: lane 0 copies the tiles of this warp's items in their order
  AttendCursor next{a.pieces ? blockIdx.x : blockIdx.x * kAttendWarps + warp, 0, 0, 0, 0, nullptr};
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
      mbar_arrive_expect_tx(bars + stage, STAGE);
      bulk_load(ring + stage * STAGE, next.region + (long long)(slot0 >> 5) * block_bytes(CB), STAGE, bars + stage);
    }
    ++issued;
    ++next.t;
  };
  for (int i = 0; i < STAGES; ++i) issue();

  int done = 0;
  bool ok = true;  // false after a wait gave up
  float2 o[NT];
  float top, total, csum;
  int b, rows, h0;
  for (; cur.item < items; cur.item += stride) {
    SlotSpan span;
    open(cur, span);
    b = cur.item / per;
    const unsigned hr = cur.item - b * per, head = a.row_groups == 1 ? hr : hr / a.row_groups, rg = hr - head * a.row_groups;
    rows = min(kAttendRows, a.group - (int)rg * kAttendRows);  // query heads of this item
    h0 = head * a.group + rg * kAttendRows;

    // ---- the queries as digit planes: thread (r, cc) holds row r's dimensions 8w..8w+7, w = cc + 4i
    uint32_t qa[KS][PLANES][2];
    float qstep, qsum = 0.f;
    {
      float x[KS][8], big = 0.f;
      const long long base = b * a.q.row + (h0 + row_head) * a.q.head;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int w = cc + 4 * i;
        const bool in = row_head < rows && 8 * w < DIM;
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
    for (int i = 0; i < NT; ++i) o[i] = make_float2(0.f, 0.f);
    top = -INFINITY, total = 0.f, csum = 0.f;

    for (int t = cur.t; t < cur.end; ++t) {
      const int slot0 = slot_at(cur, t), stage = done % STAGES;
      ok = __all_sync(~0u, ok && mbar_wait_or_abort(bars + stage, (done / STAGES) & 1, kErrWaitFull));
      if (!ok) break;
      const uint8_t* tile = ring + stage * STAGE;
      // ---- scores: s[h][j * NU + u] of slot 32h + slot_in(j, u), this thread's share of the tile
      auto slot_in = [&](int j, int u) { return 8 * cc + 4 * (HEADS == 8 ? u : my_u) + (HEADS == 1 ? my_j : j); };
      float s[HALVES][NJ * NU];
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        const uint8_t* kc = tile + h * block_bytes(CB) + r * 4 * CB;
        const uint32_t* kparam = reinterpret_cast<const uint32_t*>(tile + h * block_bytes(CB) + 2 * kBlockSlots * CB);
        int acc[4][4], acc3[4][4];
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
            if (i == 0) {
              mma_8<false, true>(acc[j], qa[i][0][0], qa[i][1][0], qa[i][0][1], qa[i][1][1], b0[j], b1[j]);
              if constexpr (PLANES == 3) mma_8<false, true>(acc3[j], qa[i][2][0], 0u, qa[i][2][1], 0u, b0[j], b1[j]);
            } else {
              mma_8<false, false>(acc[j], qa[i][0][0], qa[i][1][0], qa[i][0][1], qa[i][1][1], b0[j], b1[j]);
              if constexpr (PLANES == 3) mma_8<false, false>(acc3[j], qa[i][2][0], 0u, qa[i][2][1], 0u, b0[j], b1[j]);
            }
          }
        }
        auto score = [&](int first, int second, int third, uint32_t w) {
          // |first| <= 128 * 127 * 127, so 254 * first + second fits 32 bits
          float f = (float)(first * 254 + second);
          if constexpr (PLANES == 3) f = __fmaf_rn((float)third, 1.0f / 254.0f, f);
          return __fmaf_rn(__fmul_rn(f, qstep), param_scale(w), __fmul_rn(param_center(w), qsum));
        };
        if constexpr (HEADS == 8) {
          const uint4* kp4 = reinterpret_cast<const uint4*>(kparam + 8 * cc);
          const uint4 kp[2] = {kp4[0], kp4[1]};
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) s[h][2 * j + u] = score(acc[j][u], acc[j][2 + u], PLANES == 3 ? acc3[j][u] : 0, word_of(kp[u], j));
        } else {
          int x[4][3];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[j][0] = my_u ? acc[j][1] : acc[j][0];
            x[j][1] = my_u ? acc[j][3] : acc[j][2];
            x[j][2] = PLANES == 3 ? (my_u ? acc3[j][1] : acc3[j][0]) : 0;
          }
          if constexpr (HEADS == 4) {
            const uint4 kp = *reinterpret_cast<const uint4*>(kparam + 8 * cc + 4 * my_u);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[h][j] = score(x[j][0], x[j][1], x[j][2], word_of(kp, j));
          } else {
            int y[3];
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
              const int lo = my_j & 1 ? x[1][p] : x[0][p], hi = my_j & 1 ? x[3][p] : x[2][p];
              y[p] = my_j & 2 ? hi : lo;
            }
            s[h][0] = score(y[0], y[1], PLANES == 3 ? y[2] : 0, kparam[slot_in(0, 0)]);
          }
        }
      }
      const bool whole = slot0 + TS <= span.e0 || (slot0 >= span.s1 && slot0 + TS <= span.e1);
      if (!whole) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int u = 0; u < NU; ++u) {
              const int slot = slot0 + 32 * h + slot_in(j, u);
              if (!(slot < span.e0 || (slot >= span.s1 && slot < span.e1))) s[h][j * NU + u] = -INFINITY;
            }
      }
      // ---- running maximum of the head (its slots are on the row's quad and on the rows that repeat it)
      float m = top;
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int e = 0; e < NJ * NU; ++e) m = fmaxf(m, s[h][e]);
      m = fmaxf(m, __shfl_xor_sync(~0u, m, 1));
      m = fmaxf(m, __shfl_xor_sync(~0u, m, 2));
      if constexpr (HEADS <= 4) m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
      if constexpr (HEADS == 1) {
        m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
        m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
      }
      if (__any_sync(~0u, m > top)) {
        const float keep = top == -INFINITY ? 0.f : exp2_fast(__fsub_rn(top, m));
        total = __fmul_rn(total, keep);
        csum = __fmul_rn(csum, keep);
#pragma unroll
        for (int i = 0; i < NT; ++i) o[i] = mul2(o[i], keep);
        top = m;
      }
      // ---- weights p, their sum, and p * vscale in place of the scores
      float pmax = 0.f;
      const float shift = top == -INFINITY ? 0.f : top;  // nothing but scores of minus infinity so far
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        const uint32_t* vparam =
            reinterpret_cast<const uint32_t*>(tile + h * block_bytes(CB) + 2 * kBlockSlots * CB) + kBlockSlots;
        uint32_t vp[NJ * NU];
        if constexpr (HEADS == 1) {
          vp[0] = vparam[slot_in(0, 0)];
        } else {
#pragma unroll
          for (int u = 0; u < NU; ++u) {
            const uint4 w = *reinterpret_cast<const uint4*>(vparam + slot_in(0, u));
#pragma unroll
            for (int j = 0; j < 4; ++j) vp[j * NU + u] = word_of(w, j);
          }
        }
#pragma unroll
        for (int e = 0; e < NJ * NU; ++e) {
          const float p = exp2_fast(__fsub_rn(s[h][e], shift));
          uint32_t w = vp[e];
          if (!whole && s[h][e] == -INFINITY) w = 0;  // a hidden slot may hold a scale of NaN
          total = __fadd_rn(total, p);
          csum = __fmaf_rn(p, param_center(w), csum);
          s[h][e] = __fmul_rn(p, param_scale(w));
          pmax = fmaxf(pmax, s[h][e]);
        }
      }
      pmax = fmaxf(pmax, __shfl_xor_sync(~0u, pmax, 1));
      pmax = fmaxf(pmax, __shfl_xor_sync(~0u, pmax, 2));
      // below 1e-30 the inverse leaves float32's range: such weights count as nothing
      constexpr float kFull = PLANES == 3 ? 8388607.0f : 65535.0f;
      const float inv = pmax > 1e-30f ? __fdividef(kFull, pmax) : 0.f;
      const float unit = __fmul_rn(pmax > 1e-30f ? pmax : 0.f, kOne / kFull);
      // ---- the weights' bytes as A operands: plane 0 (highest) in rows 0-7, plane 1 in rows 8-15;
      // a word holds the four slots of group 2cc + u, of which a row's are its own
      uint32_t pa[HALVES][PLANES][2];
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        uint32_t x[NJ * NU];
#pragma unroll
        for (int e = 0; e < NJ * NU; ++e)
          x[e] = __float_as_uint(fminf(__fmaf_rn(s[h][e], inv, 8388608.0f), 8388608.0f + kFull));
        if constexpr (HEADS == 1) {
#pragma unroll
          for (int p = 0; p < PLANES; ++p) {
            const uint32_t word = ((x[0] >> (8 * (PLANES - 1 - p))) & (p == 0 && PLANES == 3 ? 0x7Fu : 0xFFu)) << (8 * my_j);
            pa[h][p][0] = my_u ? 0u : word;
            pa[h][p][1] = my_u ? word : 0u;
          }
        } else {
#pragma unroll
          for (int u = 0; u < NU; ++u) {
            const uint32_t lo01 = __byte_perm(x[u], x[NU + u], 0x5140), lo23 = __byte_perm(x[2 * NU + u], x[3 * NU + u], 0x5140);
            uint32_t word[3];
            word[PLANES - 1] = __byte_perm(lo01, lo23, 0x5410);  // bytes 0
            word[PLANES - 2] = __byte_perm(lo01, lo23, 0x7632);  // bytes 1
            if constexpr (PLANES == 3) {
              const uint32_t hi01 = __byte_perm(x[u], x[NU + u], 0x0062), hi23 = __byte_perm(x[2 * NU + u], x[3 * NU + u], 0x0062);
              word[0] = __byte_perm(hi01, hi23, 0x5410);  // bits 16-22
            }
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
              if constexpr (HEADS == 8) {
                pa[h][p][u] = word[p];
              } else {
                pa[h][p][0] = my_u ? 0u : word[p];
                pa[h][p][1] = my_u ? word[p] : 0u;
              }
            }
          }
        }
      }
      // ---- the weighted values
      const float2 unit2 = make_float2(unit, unit);
      constexpr int STEP = NI % 4 == 0 ? 4 : NI % 2 == 0 ? 2 : 1;
#pragma unroll
      for (int i0 = 0; i0 < NI; i0 += STEP) {
        uint32_t v[HALVES][2][STEP];
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            load_words<STEP>(v[h][u], reinterpret_cast<const uint32_t*>(tile + h * block_bytes(CB) + kBlockSlots * CB) +
                                          (2 * cc + u) * CB + r * NI + i0);
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
#pragma unroll
          for (int nib = 0; nib < (BITS == 4 ? 2 : 1); ++nib) {
            int acc[4], acc3[4];
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
              uint32_t b0 = v[h][0][i], b1 = v[h][1][i];
              if constexpr (BITS == 4) {
                b0 = nib ? high_codes(b0) : low_codes(b0);
                b1 = nib ? high_codes(b1) : low_codes(b1);
              }
              if (h == 0) {
                mma_8<true, true>(acc, pa[h][0][0], pa[h][1][0], pa[h][0][1], pa[h][1][1], b0, b1);
                if constexpr (PLANES == 3) mma_8<true, true>(acc3, pa[h][2][0], 0u, pa[h][2][1], 0u, b0, b1);
              } else {
                mma_8<true, false>(acc, pa[h][0][0], pa[h][1][0], pa[h][0][1], pa[h][1][1], b0, b1);
                if constexpr (PLANES == 3) mma_8<true, false>(acc3, pa[h][2][0], 0u, pa[h][2][1], 0u, b0, b1);
              }
            }
            const int nt = BITS == 4 ? 2 * (i0 + i) + nib : i0 + i;
            // |first| <= 255 * 127 * 64, so 256 * first + second fits 32 bits
            float2 f = make_float2((float)(acc[0] * 256 + acc[2]), (float)(acc[1] * 256 + acc[3]));
            if constexpr (PLANES == 3) f = fma2(f, make_float2(256.0f, 256.0f), make_float2((float)acc3[0], (float)acc3[1]));
            o[nt] = fma2(f, unit2, o[nt]);
          }
        }
      }
      ++done;
      __syncwarp();  // every lane has read the stage: it takes the next tile
      issue();
    }
    if (!ok) break;
    // ---- the sums over the row's quad and over the rows of its head; the centers' share goes to
    // every dimension
    auto join = [&](int x) {
      total = __fadd_rn(total, __shfl_xor_sync(~0u, total, x));
      csum = __fadd_rn(csum, __shfl_xor_sync(~0u, csum, x));
      if (x < 4) return;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        o[i].x = __fadd_rn(o[i].x, __shfl_xor_sync(~0u, o[i].x, x));
        o[i].y = __fadd_rn(o[i].y, __shfl_xor_sync(~0u, o[i].y, x));
      }
    };
    join(1);
    join(2);
    if constexpr (HEADS <= 4) join(16);
    if constexpr (HEADS == 1) {
      join(4);
      join(8);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] = make_float2(__fadd_rn(o[i].x, csum), __fadd_rn(o[i].y, csum));
    // thread (r, cc) has dimensions 8i + 2cc and 8i + 2cc + 1 of row r
    if (!a.pieces && r < min(rows, HEADS)) {
      const float inv = total == 0.f ? 0.f : __fdiv_rn(1.0f, total);
      const long long base = b * a.out.row + (h0 + r) * a.out.head;
#pragma unroll
      for (int i = 0; i < NT; ++i)
        store_pair(a.out.p, base + 8 * i + 2 * cc, a.dtype, a.vec, __fmul_rn(o[i].x, inv), __fmul_rn(o[i].y, inv));
    }
  }
  // a wait that gave up: never leave with copies in flight into this warp's buffers
  if (!ok && lane == 0)
    for (; done < issued; ++done) mbar_wait(bars + done % STAGES, (done / STAGES) & 1, kErrWaitFull);

  if (a.pieces) {
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
      for (int i = 0; i < NT; ++i) *reinterpret_cast<float2*>(mine + 2 + 8 * i + 2 * cc) = o[i];
    }
    __syncthreads();
    float* out = a.partial + (item * a.pieces + piece) * kAttendRows * W;
    for (int e = threadIdx.x; e < rows * DIM; e += kAttendWarps * 32) {
      const int row = e / DIM, d = e % DIM;
      float m = -INFINITY, l = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < kAttendWarps; ++w) m = fmaxf(m, results[(w * kAttendRows + row) * W]);
#pragma unroll
      for (int w = 0; w < kAttendWarps; ++w) {
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
  int smem, ctas;
};

template <int BITS, int DIM, int PLANES>
inline AttendVariant attend_variant_of(int heads) {
  return {heads > 4 ? attend_kernel<BITS, DIM, PLANES, 8> : heads > 1 ? attend_kernel<BITS, DIM, PLANES, 4> : attend_kernel<BITS, DIM, PLANES, 1>,
          attend_smem(BITS, DIM, PLANES), attend_ctas(DIM)};
}
template <int BITS, int DIM>
inline AttendVariant attend_variant_of(int planes, int heads) {
  return planes == 3 ? attend_variant_of<BITS, DIM, 3>(heads) : attend_variant_of<BITS, DIM, 2>(heads);
}
template <int BITS>
inline AttendVariant attend_variant_of(int dim, int planes, int heads) {
  switch (dim) {
    case 16: return attend_variant_of<BITS, 16>(planes, heads);
    case 32: return attend_variant_of<BITS, 32>(planes, heads);
    case 48: return attend_variant_of<BITS, 48>(planes, heads);
    case 64: return attend_variant_of<BITS, 64>(planes, heads);
    case 80: return attend_variant_of<BITS, 80>(planes, heads);
    case 96: return attend_variant_of<BITS, 96>(planes, heads);
    case 112: return attend_variant_of<BITS, 112>(planes, heads);
    default: return attend_variant_of<BITS, 128>(planes, heads);
  }
}
// heads: query heads that share a key/value head (more than 8: in several items)
inline AttendVariant attend_variant(int bits, int dim, int planes, int heads) {
  return bits == 4 ? attend_variant_of<4>(dim, planes, heads) : attend_variant_of<8>(dim, planes, heads);
}

}  // namespace kv
}  // namespace mc
