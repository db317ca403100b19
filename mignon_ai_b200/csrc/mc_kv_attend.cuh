// Attention of one query token per session over the quantised cache (layout: mc_kv.cuh).
//
// With keys and values held as center + scale * m, m an 8-bit integer, both products of the
// attention have integer operands on one side:
//   s_j = a (kscale_j * sum_d q_d m_jd + kcenter_j * sum_d q_d)
//   o_d = sum_j (p_j vscale_j) m_jd + sum_j p_j vcenter_j,   p_j = exp(s_j - max)
// and both run as 8-bit matrix products with exact 32-bit sums: the codes are the MMA's B operand
// as they lie in memory (an and-or per word for 4 bits, nothing for 8), and the other side is cut
// into 8-bit planes. A query row becomes integers of 16 (PLANES 2) or 23 bits (3) relative to its
// largest element, cut into signed bytes, a row of weights p_j vscale_j becomes a fixed-point integer of 16 bits (PLANES 2) or 23
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
// What bounds it: for long sessions reading the codes, once the loop runs (one session of 262,144
// positions, 32/8 heads of 128 in 4 bits: 66 us, of which the loop's 285 MB are 43; 9 us go by until the first
// tile is done and 6 for the last join). For short ones instruction issue: about 890 instructions a tile of
// 64 slots of a 128-wide head, for any number of heads up to four, and 1350 a (session, head) of 64 visible
// slots at width 32 in float32 (4096 sessions of 4 heads: 41 us, memory's share 7). 16 warps an SM
// (128 registers) with a tile's keys and values in flight; 64-slot tiles on 12 warps without separate
// buffers took 68 us for the long session, 32-slot tiles 78.
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

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
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

// Elements 8 (cc + 4i) .. + 7 of a row, all loads at once; zeros past dim and for a row that is not there.
template <class T, int KS>
__device__ __forceinline__ void load_row(float (&x)[KS][8], const T* p, int cc, int dim, bool in, bool vec) {
#pragma unroll
  for (int i = 0; i < KS; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
    if (in && 8 * (cc + 4 * i) < dim) load8<T>(x[i], p + 8 * (cc + 4 * i), vec);
  }
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

// CTAs that share an SM: 16 warps where 128 registers a thread hold the work.
constexpr int attend_ctas(int dim, int planes) { return (planes == 3 && dim > 64 ? 8 : 16) / kAttendWarps; }
// Slots of a tile: 64 (two blocks) where a tile's keys and values then fit, and where the third plane
// leaves the registers for it.
constexpr int attend_slots(int bits, int dim, int planes) {
  return bits == 4 ? (planes == 3 && dim > 64 ? 32 : 64) : dim <= 48 ? 64 : 32;
}
// A tile's keys (or values) with their scales and centers; each has buffers of its own, so that the next
// keys are on their way during a tile's weights and value product, and the next values during its scores.
constexpr int attend_part_bytes(int bits, int dim, int planes) {
  return attend_slots(bits, dim, planes) * (dim * bits / 8 + 4);
}
constexpr int attend_parts(int bits, int dim, int planes) {
  const int n = (221184 / attend_ctas(dim, planes) - 8192) / (kAttendWarps * attend_part_bytes(bits, dim, planes));
  return n > 8 ? 8 : n < 2 ? 2 : n;
}
constexpr int attend_smem(int bits, int dim, int planes) {
  const int ring = kAttendWarps * attend_parts(bits, dim, planes) * attend_part_bytes(bits, dim, planes);
  const int join = kAttendWarps * kAttendRows * (dim + 2) * 4;  // the warps' results, in the same place
  return ring > join ? ring : join;
}

// What a warp does of an item (a session's up to eight query heads of one key/value head): tiles
// [t, end) of its visible slots.
struct AttendItem {
  SlotSpan span;
  int t, end;
  const uint8_t* region;
};
// Items a warp may have opened (to copy their tiles) ahead of the one it works on, a power of two.
constexpr int kAttendAhead = 8;

// With few heads to an item the MMA's eight rows repeat them: HEADS rows of heads (8, 4 or 1), and the
// rows of one head take different slots of the tile (row r: HEADS 4, the groups 2cc + r / 4; HEADS 1,
// the slot r % 4 of those), so that no thread does another's exponentials. They share the
// running maximum, and their sums meet at the end of the item.
//
// With a.pieces a CTA has one piece of one item; without, every warp goes through items of its own,
// the next one's tiles already in flight.
template <int BITS, int DIM, int PLANES, int HEADS>
__global__ void __launch_bounds__(kAttendWarps * 32, attend_ctas(DIM, PLANES)) attend_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int TS = attend_slots(BITS, DIM, PLANES), HALVES = TS / 32;
  constexpr int NJ = HEADS == 1 ? 1 : 4, NU = HEADS == 8 ? 2 : 1;  // slots of a half that a thread weighs: NJ x NU
  constexpr int CB = DIM * BITS / 8;             // code bytes per slot
  constexpr int KS = (DIM + 31) / 32;            // MMA steps along the dimensions
  constexpr int NI = BITS == 4 ? DIM / 16 : DIM / 8;  // value words of a group of slots per thread
  constexpr int NT = DIM / 8;                    // 8-column tiles of the output
  constexpr float kOne = BITS == 4 ? 0.125f : 1.0f;   // the MMA's codes are 8m (4 bits) or m
  constexpr int PART = attend_part_bytes(BITS, DIM, PLANES), PARTS = attend_parts(BITS, DIM, PLANES);
  constexpr int NK = (PARTS + 1) / 2, NV = PARTS / 2;  // buffers of keys and of values
  constexpr int BLOCK_PART = kBlockSlots * (CB + 4);   // a block's keys or values
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kAttendWarps][NK + NV];
  __shared__ AttendItem queue[kAttendWarps][kAttendAhead];
  __shared__ const uint8_t* sources[kAttendWarps][4];  // of the tiles whose keys have been asked for
  const Cache& c = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, cc = lane & 3;
  uint8_t *kring = smem + warp * PARTS * PART, *vring = kring + NK * PART;
  uint64_t *kfull = full[warp], *vfull = kfull + NK;
  if (lane == 0) {
    for (int i = 0; i < NK + NV; ++i) mbar_init(kfull + i, 1);
    fence_barrier_init();
  }
  __syncwarp();

  const unsigned per = c.heads * a.row_groups, items = a.n * per;
  const unsigned stride = a.pieces ? items : gridDim.x * kAttendWarps;
  const int piece = blockIdx.y;
  const unsigned part = piece * kAttendWarps + warp, parts = a.pieces * kAttendWarps;
  const int row_head = HEADS == 8 ? r : HEADS == 4 ? r & 3 : 0;  // the thread's query head in the item
  const int my_u = r >> 2, my_j = r & 3;                         // and its slots: see above

  // ---- the producer's side: lane 0 copies the tiles of this warp's items in their order. `next` is the
  // item being copied, the opened-th of the warp's; the warp works on the taken-th.
  AttendItem next;
  const unsigned item0 = a.pieces ? blockIdx.x : blockIdx.x * kAttendWarps + warp;
  unsigned next_id = item0;
  int opened = 0, taken = 0, kissued = 0, vissued = 0, done = 0;
  auto open = [&]() {  // next_id's, into the queue
    const unsigned b = next_id / per, hr = next_id - b * per, head = a.row_groups == 1 ? hr : hr / a.row_groups;
    int session = a.sess ? a.sess[b] : b, len = 0;
    if ((unsigned)session < (unsigned)c.sessions) {
      len = a.lens[b];
    } else {
      if (lane == 0) atomicExch(c.error, 1);
      session = 0;
    }
    next.span = slot_span<TS>(c, len, a.window);
    next.t = 0;
    next.end = next.span.tiles;
    if (a.pieces) {  // an even share of the tiles, the first parts one more
      const unsigned share = (unsigned)next.span.tiles / parts, more = (unsigned)next.span.tiles - share * parts;
      next.t = part * share + min(part, more);
      next.end = next.t + share + (part < more ? 1 : 0);
    }
    next.region = region_of(c, session, head);
    if (lane == 0) queue[warp][opened & (kAttendAhead - 1)] = next;
    ++opened;
  };
  auto slot_at = [](const SlotSpan& s, int t) { return (t < s.tiles0 ? t : s.first1 + t - s.tiles0) * TS; };
  auto copy = [&](uint8_t* dst, const uint8_t* src, uint64_t* bar) {
    mbar_arrive_expect_tx(bar, PART);
#pragma unroll
    for (int h = 0; h < HALVES; ++h) bulk_load(dst + h * BLOCK_PART, src + h * 2 * BLOCK_PART, BLOCK_PART, bar);
  };
  auto issue_keys = [&]() {
    while (next.t >= next.end) {  // on to the next item, if there is one and room for it in the queue
      if (next_id + stride < next_id || next_id + stride >= items || opened - taken >= kAttendAhead) return false;
      next_id += stride;
      open();
    }
    if (lane == 0) {
      const uint8_t* src = next.region + (long long)(slot_at(next.span, next.t) >> 5) * block_bytes(CB);
      sources[warp][kissued & 3] = src;
      copy(kring + kissued % NK * PART, src, kfull + kissued % NK);
    }
    ++kissued;
    ++next.t;
    return true;
  };
  auto issue_values = [&]() {  // NV <= NK <= 4: the source is still there
    if (vissued >= kissued) return;
    if (lane == 0) copy(vring + vissued % NV * PART, sources[warp][vissued & 3] + BLOCK_PART, vfull + vissued % NV);
    ++vissued;
  };

  bool ok = true;  // false after a wait gave up
  float2 o[NT];
  float top, total, csum;
  int b = 0, rows = 0, h0 = 0;
  if (item0 < items) open();
  for (unsigned id = item0; id < items; id += stride, ++taken) {
    // the buffers that are free ask for tiles: at the start, and after items without any
    while (kissued - done < NK && issue_keys()) {
    }
    while (vissued - done < NV && vissued < kissued) issue_values();
    __syncwarp();
    const AttendItem cur = queue[warp][taken & (kAttendAhead - 1)];
    const SlotSpan& span = cur.span;
    b = id / per;
    const unsigned hr = id - b * per, head = a.row_groups == 1 ? hr : hr / a.row_groups, rg = hr - head * a.row_groups;
    rows = min(kAttendRows, a.group - (int)rg * kAttendRows);  // query heads of this item
    h0 = head * a.group + rg * kAttendRows;

    // ---- the queries as digit planes: thread (r, cc) holds row r's dimensions 8w..8w+7, w = cc + 4i
    uint32_t qa[KS][PLANES][2];
    float qstep, qsum = 0.f;
    {
      float x[KS][8], big = 0.f;
      const long long base = b * a.q.row + (h0 + row_head) * a.q.head;
      const bool in = row_head < rows;
      if (a.dtype == kF32) load_row<float, KS>(x, static_cast<const float*>(a.q.p) + base, cc, DIM, in, a.vec);
      else if (a.dtype == kF16) load_row<__half, KS>(x, static_cast<const __half*>(a.q.p) + base, cc, DIM, in, a.vec);
      else load_row<__nv_bfloat16, KS>(x, static_cast<const __nv_bfloat16*>(a.q.p) + base, cc, DIM, in, a.vec);
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[i][e]));
#pragma unroll
      for (int x = 1; x <= 2; x <<= 1) big = fmaxf(big, __shfl_xor_sync(~0u, big, x));
      // rows near the ends of float32's range, whose sum or inverse would leave it, move to its middle by a
      // power of two, and their scale back
      float scale = a.scale;
      if (__any_sync(~0u, big > 0x1p100f || (big < 0x1p-60f && big > 0.f))) {
        const bool up = big < 0x1p-60f, down = big > 0x1p100f;
        const float lift = up ? 0x1p64f : down ? 0x1p-64f : 1.f;
        scale = __fmul_rn(scale, up ? 0x1p-64f : down ? 0x1p64f : 1.f);
        big = __fmul_rn(big, lift);
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[i][e] = __fmul_rn(x[i][e], lift);
      }
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) qsum = __fadd_rn(qsum, x[i][e]);
#pragma unroll
      for (int x = 1; x <= 2; x <<= 1) qsum = __fadd_rn(qsum, __shfl_xor_sync(~0u, qsum, x));
      // n = q / step in 16 or 23 bits, cut into signed bytes: adding 0x80 to the lower ones carries into
      // the next what a byte above 127 stands for. 1.5 * 2^23 leaves n in the mantissa's low bits.
      constexpr float kMost = PLANES == 3 ? 4161000.0f : 32600.0f, kBias = PLANES == 3 ? 32896.0f : 128.0f;
      // a row of zeros has no inverse; a query that is not all finite has no digits: its scores are NaN, by the
      // sum that holds a NaN, or by the step where there are infinities (whose signs the digits do not know)
      const float inv = big > 0.f ? __fdividef(kMost, big) : 0.f;
      qstep = big < INFINITY ? __fmul_rn(__fmul_rn(big, 1.0f / kMost), __fmul_rn(scale, kOne)) : __int_as_float(0x7FFF0000);
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t u[4];
#pragma unroll
          for (int d = 0; d < 4; ++d) u[d] = __float_as_uint(__fadd_rn(__fmaf_rn(x[i][4 * e + d], inv, 12582912.0f), kBias));
          const uint32_t lo01 = __byte_perm(u[0], u[1], 0x5140), lo23 = __byte_perm(u[2], u[3], 0x5140);
          qa[i][PLANES - 1][e] = __byte_perm(lo01, lo23, 0x5410) ^ 0x80808080u;
          qa[i][PLANES - 2][e] = __byte_perm(lo01, lo23, 0x7632);
          if constexpr (PLANES == 3) {
            qa[i][1][e] ^= 0x80808080u;
            // bits 16-22 above the mantissa's 0x40: v - 64 as a signed byte
            const uint32_t hi = __byte_perm(__byte_perm(u[0], u[1], 0x0062), __byte_perm(u[2], u[3], 0x0062), 0x5410);
            qa[i][0][e] = ((hi | 0x80808080u) - 0x40404040u) ^ 0x80808080u;
          }
        }
      qsum = __fmul_rn(qsum, scale);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] = make_float2(0.f, 0.f);
    top = -INFINITY, total = 0.f, csum = 0.f;

    for (int t = cur.t; t < cur.end; ++t) {
      const int slot0 = slot_at(span, t);
      ok = __all_sync(~0u, mbar_wait_or_abort(kfull + done % NK, (done / NK) & 1, kErrWaitFull));
      if (!ok) break;
      const uint8_t* ktile = kring + done % NK * PART;
      // ---- scores: s[h][j * NU + u] of slot 32h + slot_in(j, u), this thread's share of the tile
      auto slot_in = [&](int j, int u) { return 8 * cc + 4 * (HEADS == 8 ? u : my_u) + (HEADS == 1 ? my_j : j); };
      float s[HALVES][NJ * NU];
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        const uint8_t* kc = ktile + h * BLOCK_PART + r * 4 * CB;
        const uint32_t* kparam = reinterpret_cast<const uint32_t*>(ktile + h * BLOCK_PART + kBlockSlots * CB);
        int acc[4][4], acc3[4][4];
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const int w = cc + 4 * i;
          uint32_t b0[4], b1[4];
          if (DIM % 32 == 0 || 8 * w < DIM) {
            if constexpr (BITS == 4) {
              uint32_t x[4];
              load_words<4>(x, reinterpret_cast<const uint32_t*>(kc + 16 * key_unit(w, r, CB, 4)));
#pragma unroll
              for (int j = 0; j < 4; ++j) b0[j] = low_codes(x[j]), b1[j] = high_codes(x[j]);
            } else {
              load_words<4>(b0, reinterpret_cast<const uint32_t*>(kc + 16 * key_unit(2 * w, r, CB, 8)));
              load_words<4>(b1, reinterpret_cast<const uint32_t*>(kc + 16 * key_unit(2 * w + 1, r, CB, 8)));
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
          // |first| <= 128 * 128 * 127, so 256 * first + second fits 32 bits
          float f = (float)(first * 256 + second);
          if constexpr (PLANES == 3) f = __fmaf_rn(f, 256.0f, (float)third);
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
      __syncwarp();  // every lane has read the keys: their buffer takes the next tile's
      issue_keys();
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
        for (int e = 0; e + 1 < NJ * NU; e += 2) m = max3(m, s[h][e], s[h][e + 1]);
      if constexpr (HEADS == 1) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) m = fmaxf(m, s[h][0]);
      }
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
      ok = __all_sync(~0u, mbar_wait_or_abort(vfull + done % NV, (done / NV) & 1, kErrWaitFull));
      if (!ok) break;
      const uint8_t* vtile = vring + done % NV * PART;
      float pmax = 0.f;
      const float shift = top == -INFINITY ? 0.f : top;  // nothing but scores of minus infinity so far
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        const uint32_t* vparam = reinterpret_cast<const uint32_t*>(vtile + h * BLOCK_PART + kBlockSlots * CB);
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
          if (e & 1) pmax = max3(pmax, s[h][e - 1], s[h][e]);
        }
        if constexpr (HEADS == 1) pmax = fmaxf(pmax, s[h][0]);
      }
      pmax = fmaxf(pmax, __shfl_xor_sync(~0u, pmax, 1));
      pmax = fmaxf(pmax, __shfl_xor_sync(~0u, pmax, 2));
      // below 1e-30 the inverse leaves float32's range: such weights count as nothing. kFull leaves room
      // below 2^23 and 2^16 for the quotient's and the product's rounding
      constexpr float kFull = PLANES == 3 ? 8388600.0f : 65534.9f;
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
          x[e] = __float_as_uint(__fmaf_rn(s[h][e], inv, 8388608.0f));
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
        for (int h = 0; h < HALVES; ++h) {
          const uint32_t* pair = reinterpret_cast<const uint32_t*>(vtile + h * BLOCK_PART) + cc * 2 * CB;
          if constexpr (NI == 2) {
            uint32_t both[4];
            load_words<4>(both, pair + value_word(r, 0, 2 * cc, NI));
            v[h][0][0] = both[0], v[h][0][1] = both[1], v[h][1][0] = both[2], v[h][1][1] = both[3];
          } else {
            load_words<STEP>(v[h][0], pair + value_word(r, i0, 2 * cc, NI));
            load_words<STEP>(v[h][1], pair + value_word(r, i0, 2 * cc + 1, NI));
          }
        }
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
      __syncwarp();  // and the values
      issue_values();
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
  if (!ok && lane == 0) {
    for (int i = max(0, kissued - NK); i < kissued; ++i) mbar_wait(kfull + i % NK, (i / NK) & 1, kErrWaitFull);
    for (int i = max(0, vissued - NV); i < vissued; ++i) mbar_wait(vfull + i % NV, (i / NV) & 1, kErrWaitFull);
  }

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
    {  // the pieces' factors: a share of the threads to a row, all their loads at once
      constexpr int SHARE = kAttendWarps * 32 / kAttendRows, PER = kMaxPieces / SHARE;
      static_assert(SHARE == 16 || SHARE == 32, "a row's threads are in one warp");
      const int row = threadIdx.x / SHARE, l16 = threadIdx.x % SHARE;
      float2 ml[PER];
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int p = l16 + SHARE * i;
        ml[i] = make_float2(-INFINITY, 0.f);
        if (row < rows && p < a.pieces) ml[i] = __ldcg(reinterpret_cast<const float2*>(all + (p * kAttendRows + row) * W));
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) m = fmaxf(m, ml[i].x);
#pragma unroll
      for (int x = 1; x < SHARE; x <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, x));
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const float keep = ml[i].x == -INFINITY ? 0.f : exp2_fast(__fsub_rn(ml[i].x, m));
        keeps[row * kMaxPieces + l16 + SHARE * i] = keep;
        l = __fmaf_rn(ml[i].y, keep, l);
      }
#pragma unroll
      for (int x = 1; x < SHARE; x <<= 1) l = __fadd_rn(l, __shfl_xor_sync(~0u, l, x));
      if (l16 == 0) results[row] = l;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * (DIM / 2); e += kAttendWarps * 32) {
      const int row = e / (DIM / 2), d = 2 * (e % (DIM / 2));
      float2 x = make_float2(0.f, 0.f);
      for (int p0 = 0; p0 < a.pieces; p0 += 32) {  // 32 loads in flight; past the last piece the factor is zero
        float2 q[32];
#pragma unroll
        for (int i = 0; i < 32; ++i)
          q[i] = __ldcg(reinterpret_cast<const float2*>(all + (min(p0 + i, a.pieces - 1) * kAttendRows + row) * W + 2 + d));
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float keep = p0 + i < a.pieces ? keeps[row * kMaxPieces + p0 + i] : 0.f;
          x = fma2(q[i], make_float2(keep, keep), x);
        }
      }
      const float l = results[row], inv = l == 0.f ? 0.f : __fdiv_rn(1.0f, l);
      store_pair(a.out.p, b * a.out.row + (h0 + row) * a.out.head + d, a.dtype, a.vec, __fmul_rn(x.x, inv), __fmul_rn(x.y, inv));
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
          attend_smem(BITS, DIM, PLANES), attend_ctas(DIM, PLANES)};
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
