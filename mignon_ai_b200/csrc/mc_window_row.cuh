// Window attention: its arguments, and one query row by one warp, key by key. The tiled kernels
// fall back to it for rows that need it.
#pragma once
#include "mc_kv.cuh"

namespace mc {
namespace win {

using kv::Rows;
using kv::from_float;
using kv::to_float;

constexpr int kMaxDim = 256;

struct Args {
  Rows q, k, v, out;
  int n_q, n_k, n_seg, q_heads, heads, group, dim, window, sinks;
  const int *q_start, *k_start;
  float scale;  // of the scores, times log2(e)
};

// The first key that the window shows a query at position pos. No subtraction leaves 32 bits, whatever the
// window and for the negative positions of queries before every key.
__device__ __forceinline__ int window_begin(int window, int pos) {
  return window > 0 && pos >= window ? pos - window + 1 : 0;
}

// One query row by one warp, key by key: lane j scores keys j, j + 32, ..; then the lanes own
// dimensions. Masked keys and values are not read, so whatever they hold reaches nothing. query(d): element
// d of the row's query, all read before anything is stored.
template <class T, class Q>
__device__ void row_attention(const Args& a, int row, int h, int k0, int pos, float* qs, Q query) {
  const int lane = threadIdx.x & 31, dim = a.dim, hk = h / a.group;
  T* out = static_cast<T*>(a.out.p) + row * a.out.row + h * a.out.head;
  const T* k = static_cast<const T*>(a.k.p) + k0 * a.k.row + hk * a.k.head;
  const T* v = static_cast<const T*>(a.v.p) + k0 * a.v.row + hk * a.v.head;
  for (int d = lane; d < dim; d += 32) qs[d] = to_float<T>(query(d));
  __syncwarp();
  const int lo = window_begin(a.window, pos);
  const int sink_end = min(a.sinks, lo);                        // visible keys before it
  float top = -INFINITY, total = 0.f, acc[kMaxDim / 32] = {};
  const int n = sink_end + (pos + 1 - lo);
  for (int t = 0; t < n; t += 32) {
    const int i = t + lane;
    const bool seen = i < n;
    const int j = i < sink_end ? i : i - sink_end + lo;
    float s = -INFINITY;
    if (seen) {
      float dot = 0.f;
      for (int d = 0; d < dim; ++d) dot = __fmaf_rn(qs[d], to_float<T>(k[j * a.k.row + d]), dot);
      s = __fmul_rn(dot, a.scale);
    }
    float m = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float other = __shfl_xor_sync(~0u, m, o);
      m = m >= other || isnan(m) ? m : other;  // a NaN score stays
    }
    m = m >= top || isnan(m) ? m : top;
    if (m == -INFINITY) continue;  // nothing but scores of minus infinity so far
    const float keep = exp2f(__fsub_rn(top, m));
    const float p = exp2f(__fsub_rn(s, m));
    top = m;
    total = __fmul_rn(total, keep) + p;  // per lane; summed over the lanes at the end
#pragma unroll
    for (int u = 0; u < kMaxDim / 32; ++u) acc[u] = __fmul_rn(acc[u], keep);
    const int count = min(32, n - t);
    for (int e = 0; e < count; ++e) {
      const float pe = __shfl_sync(~0u, p, e);
      const T* vr = v + __shfl_sync(~0u, j, e) * a.v.row;
#pragma unroll
      for (int u = 0; u < kMaxDim / 32; ++u) {
        const int d = lane + 32 * u;
        if (d < dim) acc[u] = __fmaf_rn(pe, to_float<T>(vr[d]), acc[u]);
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) total = __fadd_rn(total, __shfl_xor_sync(~0u, total, o));
#pragma unroll
  for (int u = 0; u < kMaxDim / 32; ++u) {
    const int d = lane + 32 * u;
    if (d < dim) out[d] = from_float<T>(total == 0.f ? 0.f : __fdiv_rn(acc[u], total));
  }
}

template <class T>
__device__ void row_attention(const Args& a, int row, int h, int k0, int pos, float* qs) {
  const T* q = static_cast<const T*>(a.q.p) + row * a.q.row + h * a.q.head;
  row_attention<T>(a, row, h, k0, pos, qs, [&](int d) { return q[d]; });
}

// The segment of row r: the last b with start[b] <= r (null starts: one row per segment), or -1.
__device__ __forceinline__ int segment_of(const int* start, int n, int r) {
  if (!start) return r < n ? r : -1;
  if (r < start[0] || r >= start[n]) return -1;
  int lo = 0, hi = n;  // start[lo] <= r < start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The segment's queries and keys, with its bounds checked against the rows there are.
struct Segment {
  int q0, nq, k0, nk;
  bool fits;
};
__device__ __forceinline__ Segment segment(const Args& a, int b) {
  Segment s{0, a.n_q, 0, a.n_k, true};
  if (a.q_start) {
    s.q0 = a.q_start[b];
    s.nq = a.q_start[b + 1] - s.q0;
  }
  if (a.k_start) {
    s.k0 = a.k_start[b];
    s.nk = a.k_start[b + 1] - s.k0;
  }
  if (s.q0 < 0 || s.nq < 0 || s.nq > a.n_q - s.q0 || s.k0 < 0 || s.nk < 0 || s.nk > a.n_k - s.k0) s = Segment{0, 0, 0, 0, false};
  return s;
}

// Set once a segment did not fit (read and cleared by mc_window_error).
static __device__ int g_window_bounds = 0;

// Reports the segments that do not fit, of which no row is computed; by the grid's first row of blocks together.
// A call: in line it made the tcgen05 kernel spill in its loop.
__device__ __noinline__ void check_segments(const Args& a) {
  if (!a.q_start || blockIdx.y) return;
  for (long long b = (long long)blockIdx.x * blockDim.x + threadIdx.x; b < a.n_seg; b += (long long)gridDim.x * blockDim.x)
    if (!segment(a, (int)b).fits) atomicExch(&g_window_bounds, 1);
}

// The tiled kernels hand out tiles of tt tokens so that segment b's begin at start[b] / tt + b: each
// segment has room for all of its own, and a tile finds its segment by a search (by whole warps).
__device__ __forceinline__ int tile_segment(const int* start, int n, int tt, int tile) {
  return kv::last_at_most(n, [&](int i) { return start[i] / tt + i <= tile; });
}

}  // namespace win
}  // namespace mc
