// Window attention of float32 (and of 16-bit rows that TMA cannot fetch) on m16n8k8 tf32 MMAs.
//
// A float32 operand x is cut into hi = x with the low 13 bits cleared (tf32, 11 significant bits)
// and lo = x - hi (exact); a product is hi*hi + hi*lo + lo*hi, whose error, about 2^-22 of
// |a||b|, is float32's own size. The tensor unit does not round its sums to nearest: summed over a row of
// 8192 keys that alone came to 1.3e-5 of the result. So the two small products have a sum of their own,
// each tile's value sums start from zero, and what they are added up in is float32. 16-bit operands are exact in tf32 and their weights need no more
// than tf32's bits before a 16-bit output: one product.
//
// A CTA of four warps takes 64 rows (tokens x the query heads that share a key/value head), a warp
// 16 of them, for one or more key/value heads one after the other. Queries, and keys and values of 64
// positions at a time, are staged as float32 in shared memory: the next keys (and the next head's
// queries) in flight behind the softmax and the value product, the next values behind the score
// product (cp.async where rows are 16-byte aligned float32). Scores stay in
// registers: the layout in which an MMA leaves them is the one its A operand wants if the k order
// of the value product is taken as (2c, 2c + 1) for a thread's (c, c + 4). Row strides of dim + 8 and
// dim + 4 floats keep the operands' shared loads free of bank conflicts.
//
// What bounds it: for long rows the three products at the legacy tensor rate (275 TFLOP/s of tf32
// measured, so 92 of float32); for prompts of a tile or less the latency of each phase and the fetching of
// instructions (2000 prompts of 16-64 rows, 6 heads of 64: 319 us, memory's share of it 75; 128 registers,
// 16 warps an SM, tensor pipe 17 % busy). Warps skip the columns that none of their 16 rows sees.
#pragma once
#include "mc_window_row.cuh"

namespace mc {
namespace win {

constexpr int kTileThreads = 128;
constexpr int kTileRows = 64;
constexpr int kTileKeys = 64;
constexpr int kTileMaxDim = 128;

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cut(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xFFFFE000u;
  lo = __float_as_uint(__fsub_rn(x, __uint_as_float(hi)));
}
// The A operands, fewer than B's, are cut to nearest: their low parts then have either sign, and the
// low-by-low products that are left out no longer add up. The carry turns a NaN's high part into anything: its low
// part is NaN, and where that is not used something else has to be (a row's sum, for weights).
__device__ __forceinline__ void cut_nearest(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
  lo = __float_as_uint(__fsub_rn(x, __uint_as_float(hi)));
}

// d[j] + small[j] += a x b[j] for four independent sums, product by product, so that no MMA waits for the
// one before it; with a's and b's parts (PRODUCTS 1: the high parts alone)
template <int PRODUCTS>
__device__ __forceinline__ void mma_cut(float (*d)[4], float (*small)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], const float (&b)[4][2]) {
  uint32_t bh[4][2], bl[4][2];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) cut(b[j][e], bh[j][e], bl[j][e]);
  if constexpr (PRODUCTS == 3) {
#pragma unroll
    for (int j = 0; j < 4; ++j) mma_tf32(small[j], al, bh[j][0], bh[j][1]);
#pragma unroll
    for (int j = 0; j < 4; ++j) mma_tf32(small[j], ah, bl[j][0], bl[j][1]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) mma_tf32(d[j], ah, bh[j][0], bh[j][1]);
}

struct TileArgs {
  Args a;
  int vec;    // float32 rows of keys and values, 16-byte aligned, of a multiple of 4 dimensions
  int qvec;   // and of queries
  int pairs;  // rows of outputs take accesses of two elements
  int heads;  // key/value heads that a CTA takes one after the other
};

template <class T>
__device__ __forceinline__ void store_pair(T* p, float x, float y) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p) = make_float2(x, y);
  else *reinterpret_cast<uint32_t*>(p) = pack16<T>(x, y);
}

__device__ __forceinline__ void copy16_async(float* dst, const float* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Rows [0, count) of 64 staged with stride S, zeros past count and past the head's width. Row j is token
// j / group, head j % group of it.
template <class T, int DIMP, int S>
__device__ __forceinline__ void stage(float* dst, const T* src, long long row, long long head, unsigned group, int count, int dim,
                                      bool vec) {
  auto offset = [&](unsigned j) { return group == 1 ? j * row : (j / group) * row + (j % group) * head; };
  if constexpr (std::is_same<T, float>::value) {
    if (vec) {
#pragma unroll 4
      for (int e = threadIdx.x; e < kTileKeys * DIMP / 4; e += kTileThreads) {
        const int j = e / (DIMP / 4), d = 4 * (e % (DIMP / 4));
        const bool in = j < count && d < dim;
        copy16_async(dst + j * S + d, src + (in ? offset(j) + d : 0), in);
      }
      return;
    }
  }
#pragma unroll 4
  for (int e = threadIdx.x; e < kTileKeys * DIMP; e += kTileThreads) {
    const int j = e / DIMP, d = e % DIMP;
    dst[j * S + d] = j < count && d < dim ? to_float<T>(src[offset(j) + d]) : 0.f;
  }
}

// queries and keys (stride dimp + 8), values (dimp + 4)
inline size_t tile_smem(int dimp) { return (size_t)kTileKeys * (3 * dimp + 20) * sizeof(float); }

// DIMP: the head width rounded up to 16, 32, 64, 96 or 128 (dimensions past the width are zeros).
template <class T, int DIMP>
__global__ void __launch_bounds__(kTileThreads, DIMP <= 64 ? 4 : 2) tile_kernel(const __grid_constant__ TileArgs args) {
  const Args& a = args.a;
  constexpr int PRODUCTS = std::is_same<T, float>::value ? 3 : 1;
  constexpr int KD = DIMP / 8;                   // MMA steps along the dimensions
  constexpr int NK = kTileKeys / 8;              // 8-key columns of a tile
  constexpr int DV = (DIMP / 8 + 3) / 4 * 4;     // 8-dimension columns of the output, in fours
  constexpr int SK = DIMP + 8, SV = DIMP + 4;    // row strides of the staged keys and values
  extern __shared__ float sm[];
  __shared__ float redo[kTileThreads / 32][kTileMaxDim];
  float* sq = sm;
  float* sk = sq + kTileRows * SK;
  float* sv = sk + kTileKeys * SK;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;

  check_segments(a);
  const int tt = kTileRows / a.group, tile_id = gridDim.x - 1 - blockIdx.x;
  const int h0 = blockIdx.y * args.heads, n_heads = min(args.heads, a.heads - h0);
  const int b = a.q_start ? tile_segment(a.q_start, a.n_seg, tt, tile_id) : 0;
  const Segment seg = segment(a, b);
  const int first = (tile_id - (a.q_start ? a.q_start[b] / tt + b : 0)) * tt;  // first token in the segment
  if (first < 0 || first >= seg.nq) return;
  const int tokens = min(tt, seg.nq - first);
  const int base = seg.nk - seg.nq + first;  // position of the first token

  // the warp's rows 16w + r and 16w + r + 8: tokens and heads, positions, bounds of what they see
  int pos[2], lo[2], row[2], head[2];
  bool real[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 16 * warp + r + 8 * e, token = i / a.group;
    real[e] = token < tokens;
    pos[e] = real[e] ? base + token : -1;
    lo[e] = window_begin(a.window, pos[e]);
    row[e] = seg.q0 + first + token;
    head[e] = i - token * a.group;  // among those that share a key/value head
  }
  // positions of the CTA's and of the warp's first and last real rows
  const int last_token = min(tokens - 1, (16 * warp + 15) / a.group), first_token = 16 * warp / a.group;
  const int w_hi = first_token < tokens ? base + last_token : -1;
  const int w_lo = window_begin(a.window, base + first_token);  // the warp's first windowed key
  const int cta_hi = base + tokens - 1, cta_lo = window_begin(a.window, base);
  const int win_tile = cta_lo / kTileKeys;
  const int sink_tiles = cta_hi < 0 ? 0 : min(win_tile, (min(a.sinks, cta_lo) + kTileKeys - 1) / kTileKeys);
  const int n_tiles = cta_hi < 0 ? 0 : sink_tiles + cta_hi / kTileKeys - win_tile + 1;

  auto tile_key = [&](int i) { return (i < sink_tiles ? i : win_tile + i - sink_tiles) * kTileKeys; };
  // steps: the tiles of head h0, then those of the next. Keys past cta_hi are seen by no row and stay zero.
  const int steps = n_heads * n_tiles;
  auto load = [&](int step, bool values) {
    if (step < steps) {
      const int hk = h0 + (n_heads == 1 ? 0 : step / n_tiles), i = step - (hk - h0) * n_tiles;
      const int key = tile_key(i), count = min(kTileKeys, cta_hi + 1 - key);
      if (values) {
        stage<T, DIMP, SV>(sv, static_cast<const T*>(a.v.p) + (seg.k0 + key) * a.v.row + hk * a.v.head, a.v.row, 0, 1, count, a.dim,
                           args.vec);
      } else {
        if (i == 0)
          stage<T, DIMP, SK>(sq, static_cast<const T*>(a.q.p) + (seg.q0 + first) * a.q.row + (long long)hk * a.group * a.q.head,
                             a.q.row, a.q.head, a.group, tokens * a.group, a.dim, args.qvec);
        stage<T, DIMP, SK>(sk, static_cast<const T*>(a.k.p) + (seg.k0 + key) * a.k.row + hk * a.k.head, a.k.row, 0, 1, count, a.dim,
                           args.vec);
      }
    }
    copies_commit();
  };
  load(0, false);
  load(0, true);
  int step = 0;
  for (int hk = h0; hk < h0 + n_heads; ++hk) {
  float o[DV][4];
#pragma unroll
  for (int i = 0; i < DV; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float top[2] = {-INFINITY, -INFINITY}, total[2] = {0.f, 0.f};
  for (int i = 0; i < n_tiles; ++i, ++step) {
    const int key = tile_key(i);
    // 8-key columns that some row of the warp sees
    const int n_end = w_hi < key ? 0 : min(NK, (w_hi - key) / 8 + 1);
    const int n_begin = key < a.sinks ? 0 : max(0, (w_lo - key) / 8);
    copies_wait<1>();
    __syncthreads();
    float s[NK][4];
#pragma unroll
    for (int n = 0; n < NK; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int n = 0; n < NK; n += 4) {
      if (n + 4 <= n_begin || n >= n_end) continue;
      float small[4][4] = {};
      // not unrolled: short CTAs out of step with one another wait for instructions first (2000 prompts: 319 us,
      // 342 unrolled)
#pragma unroll 1
      for (int k = 0; k < KD; ++k) {
        // step k, thread (r, c): dimensions 8k + 2c (a0, a1) and 8k + 2c + 1 (a2, a3) of rows r and r + 8
        uint32_t ah[4], al[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 q = *reinterpret_cast<const float2*>(&sq[(16 * warp + r + 8 * e) * SK + 8 * k + 2 * c]);
          // 16-bit values stay exact in tf32: their scores are scaled instead
          if constexpr (PRODUCTS == 3) {
            cut_nearest(__fmul_rn(q.x, a.scale), ah[e], al[e]);
            cut_nearest(__fmul_rn(q.y, a.scale), ah[2 + e], al[2 + e]);
          } else {  // nothing to cut
            ah[e] = __float_as_uint(q.x), ah[2 + e] = __float_as_uint(q.y);
          }
        }
        float x[4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<float2*>(x[j]) = *reinterpret_cast<const float2*>(&sk[(8 * (n + j) + r) * SK + 8 * k + 2 * c]);
        mma_cut<PRODUCTS>(s + n, small, ah, al, x);
      }
      if (PRODUCTS == 3) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n + j][e] = __fadd_rn(s[n + j][e], small[j][e]);
      }
    }
    __syncthreads();
    load(step + 1, false);
    // ---- what each row sees, its maximum, its weights. s[n][2e + u]: row e, key 8n + 2c + u
    float keep[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j_lo = lo[e] - key - 2 * c, j_hi = pos[e] - key - 2 * c, j_sink = min(a.sinks, pos[e] + 1) - key - 2 * c;
      float m = -INFINITY;
#pragma unroll
      for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int j = 8 * n + u;
          if (n < n_begin || n >= n_end || !((j >= j_lo && j <= j_hi) || j < j_sink)) s[n][2 * e + u] = -INFINITY;
          else if (PRODUCTS == 1) s[n][2 * e + u] = __fmul_rn(s[n][2 * e + u], a.scale);
          m = fmaxf(m, s[n][2 * e + u]);
        }
      m = fmaxf(m, __shfl_xor_sync(~0u, m, 1));
      m = fmaxf(m, __shfl_xor_sync(~0u, m, 2));
      m = fmaxf(m, top[e]);
      keep[e] = top[e] == -INFINITY ? 0.f : kv::exp2_fast(__fsub_rn(top[e], m));
      top[e] = m;
      const float shift = m == -INFINITY ? 0.f : m;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float p = kv::exp2_fast(__fsub_rn(s[n][2 * e + u], shift));
          s[n][2 * e + u] = p;
          sum = __fadd_rn(sum, p);
        }
      total[e] = __fmaf_rn(total[e], keep[e], sum);
    }
    copies_wait<1>();
    __syncthreads();
    // a tile's sums start from zero and are added to the row's in float32: the tensor unit does not round
    // its sums to nearest, which would add up over a long row
#pragma unroll
    for (int d = 0; d < DV; d += 4) {
      float sum[4][4] = {}, small[4][4] = {};
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        if (n < n_begin || n >= n_end) continue;
        uint32_t ph[4], pl[4];
        cut_nearest(s[n][0], ph[0], pl[0]);
        cut_nearest(s[n][2], ph[1], pl[1]);
        cut_nearest(s[n][1], ph[2], pl[2]);
        cut_nearest(s[n][3], ph[3], pl[3]);
        float x[4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float* v = &sv[(8 * n + 2 * c) * SV + 8 * (d + j) + r];
          x[j][0] = d + j < DIMP / 8 ? v[0] : 0.f;
          x[j][1] = d + j < DIMP / 8 ? v[SV] : 0.f;
        }
        mma_cut<PRODUCTS>(sum, small, ph, pl, x);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d + j][e] = __fmaf_rn(o[d + j][e], keep[e >> 1], PRODUCTS == 3 ? __fadd_rn(sum[j][e], small[j][e]) : sum[j][e]);
    }
    __syncthreads();
    load(step + 1, true);
  }
  // ---- the output rows: o[d][2e + u] is row e, dimension 8d + 2c + u. A row that is not all finite is not
  // stored: outputs may be in place of the queries, which its second computation reads.
  uint32_t again[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float sum = total[e];
    sum = __fadd_rn(sum, __shfl_xor_sync(~0u, sum, 1));
    sum = __fadd_rn(sum, __shfl_xor_sync(~0u, sum, 2));
    const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.0f, sum);
    float bad = __fmul_rn(sum, 0.f);
#pragma unroll
    for (int d = 0; d < DIMP / 8; ++d) {  // NaN once a value is not finite
      o[d][2 * e] = __fmul_rn(o[d][2 * e], inv);
      o[d][2 * e + 1] = __fmul_rn(o[d][2 * e + 1], inv);
      bad = __fmaf_rn(o[d][2 * e], 0.f, __fmaf_rn(o[d][2 * e + 1], 0.f, bad));
    }
    again[e] = __ballot_sync(~0u, real[e] && !(bad == 0.f));
    const bool store = real[e] && !(again[e] & (0xFu << (lane & ~3)));
    T* out = static_cast<T*>(a.out.p) + row[e] * a.out.row + (long long)(hk * a.group + head[e]) * a.out.head;
#pragma unroll
    for (int d = 0; d < DIMP / 8; ++d) {
      const float x = o[d][2 * e], y = o[d][2 * e + 1];
      const int at = 8 * d + 2 * c;
      if (store && args.pairs) {
        if (at < a.dim) store_pair<T>(out + at, x, y);
      } else if (store) {
        if (at < a.dim) out[at] = from_float<T>(x);
        if (at + 1 < a.dim) out[at + 1] = from_float<T>(y);
      }
    }
  }
  // a non-finite row may have met a hidden key's infinity or NaN times its weight of zero: key by key
#pragma unroll
  for (int e = 0; e < 2; ++e)
    for (int i = 0; i < 8; ++i) {
      if (!(again[e] & (0xFu << (4 * i)))) continue;
      const int at = 16 * warp + 8 * e + i;
      __syncwarp();
      row_attention<T>(a, seg.q0 + first + at / a.group, hk * a.group + at % a.group, seg.k0, base + at / a.group, redo[warp]);
    }
  }
}

template <class T>
inline void (*tile_variant(int dim, int* dimp))(TileArgs) {
  *dimp = dim <= 16 ? 16 : dim <= 32 ? 32 : dim <= 48 ? 48 : dim <= 64 ? 64 : dim <= 96 ? 96 : 128;
  switch (*dimp) {
    case 16: return tile_kernel<T, 16>;
    case 32: return tile_kernel<T, 32>;
    case 48: return tile_kernel<T, 48>;
    case 64: return tile_kernel<T, 64>;
    case 96: return tile_kernel<T, 96>;
    default: return tile_kernel<T, 128>;
  }
}

}  // namespace win
}  // namespace mc
