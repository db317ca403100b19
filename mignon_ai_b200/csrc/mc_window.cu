// Causal attention of whole segments with a sliding window and a few first positions that stay
// visible (sinks), over keys and values that are not quantised:
//   s_ij = scale q_i . k_j,  visible: j <= i and (j < sinks or j > i - window),
//   o_i = sum_j softmax(s_i)_j v_j,  zero for a row that sees nothing.
// A segment's queries are its last positions: query t of nq over nk keys is position nk - nq + t.
#include "mc_kv.cuh"

namespace mc {
namespace win {

using kv::Rows;
using kv::from_float;
using kv::to_float;

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;

struct Args {
  Rows q, k, v, out;
  int n_q, n_k, n_seg, q_heads, heads, group, dim, window, sinks;
  const int *q_start, *k_start;
  float scale;  // of the scores, times log2(e)
};

// One query row by one warp, key by key: lane j scores keys j, j + 32, ..; then the lanes own
// dimensions. Masked keys and values are not read, so whatever they hold reaches nothing.
template <class T>
__device__ void row_attention(const Args& a, int row, int h, int k0, int pos, float* qs) {
  const int lane = threadIdx.x & 31, dim = a.dim, hk = h / a.group;
  const T* q = static_cast<const T*>(a.q.p) + row * a.q.row + h * a.q.head;
  T* out = static_cast<T*>(a.out.p) + row * a.out.row + h * a.out.head;
  const T* k = static_cast<const T*>(a.k.p) + k0 * a.k.row + hk * a.k.head;
  const T* v = static_cast<const T*>(a.v.p) + k0 * a.v.row + hk * a.v.head;
  for (int d = lane; d < dim; d += 32) qs[d] = to_float<T>(q[d]);
  __syncwarp();
  const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;  // first key of the window
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

// The segment's queries and keys, with its bounds checked against the rows there are.
struct Segment {
  int q0, nq, k0, nk;
};
__device__ __forceinline__ Segment segment(const Args& a, int b) {
  Segment s{0, a.n_q, 0, a.n_k};
  if (a.q_start) {
    s.q0 = a.q_start[b];
    s.nq = a.q_start[b + 1] - s.q0;
  }
  if (a.k_start) {
    s.k0 = a.k_start[b];
    s.nk = a.k_start[b + 1] - s.k0;
  }
  if (s.q0 < 0 || s.nq < 0 || s.nq > a.n_q - s.q0 || s.k0 < 0 || s.nk < 0 || s.nk > a.n_k - s.k0) s = Segment{0, 0, 0, 0};
  return s;
}

template <class T>
__global__ void __launch_bounds__(kThreads) row_kernel(const __grid_constant__ Args a) {
  __shared__ float qs[kThreads / 32][kMaxDim];
  const int warp = threadIdx.x >> 5;
  const long long item = (long long)blockIdx.x * (kThreads / 32) + warp;
  const int row = (int)(item / a.q_heads), h = (int)(item % a.q_heads);
  if (row >= a.n_q) return;
  const int b = a.q_start ? kv::segment_of(a.q_start, a.n_seg, row) : 0;
  if (b < 0) return;
  const Segment s = segment(a, b);
  if (s.nq == 0) return;
  row_attention<T>(a, row, h, s.k0, s.nk - s.nq + row - s.q0, qs[warp]);
}

}  // namespace win
}  // namespace mc

extern "C" int mc_window_attn_dev(const mc_rows* q, const mc_rows* k, const mc_rows* v, const mc_rows* out, int dtype,
                                  int q_heads, int kv_heads, int head_dim, int n_q, int n_k, const int32_t* q_start,
                                  const int32_t* k_start, int n_segments, int window, int sinks, float scale,
                                  void* stream) {
  using namespace mc;
  using namespace mc::win;
  clear_error();
  if (!kv::rows_ok(q) || !kv::rows_ok(k) || !kv::rows_ok(v) || !kv::rows_ok(out))
    return set_error(kInvalidArgument, "mc_window_attn_dev: null argument");
  if (dtype < kv::kF32 || dtype > kv::kBF16) return set_error(kInvalidArgument, "mc_window_attn_dev: unknown dtype");
  if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads)
    return set_error(kInvalidArgument, "mc_window_attn_dev: q_heads must be a positive multiple of kv_heads");
  if (head_dim < 1 || head_dim > kMaxDim) return set_error(kInvalidArgument, "mc_window_attn_dev: head_dim must be 1 to 256");
  if (n_q < 0 || n_k < 0 || n_segments < 0 || window < 0 || sinks < 0)
    return set_error(kInvalidArgument, "mc_window_attn_dev: counts must not be negative");
  if ((!q_start || !k_start) && (q_start != k_start || n_segments != 1))
    return set_error(kInvalidArgument, "mc_window_attn_dev: q_start and k_start come together, or not at all for one segment");
  if (!(scale > 0.f) || !std::isfinite(scale)) return set_error(kInvalidArgument, "mc_window_attn_dev: scale must be positive");
  if (n_q == 0 || n_segments == 0) return kOk;
  const Args a{kv::rows_of(q), kv::rows_of(k), kv::rows_of(v), kv::rows_of(out), n_q, n_k, n_segments, q_heads, kv_heads,
               q_heads / kv_heads, head_dim, window, sinks, q_start, k_start, scale * 1.4426950408889634f};
  const long long blocks = ((long long)n_q * q_heads + kThreads / 32 - 1) / (kThreads / 32);
  if (blocks > INT_MAX) return set_error(kInvalidArgument, "mc_window_attn_dev: too many rows");
  void (*f)(Args) = dtype == kv::kF32 ? row_kernel<float> : dtype == kv::kF16 ? row_kernel<__half> : row_kernel<__nv_bfloat16>;
  f<<<(unsigned)blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  MC_CUDA(cudaGetLastError());
  return kOk;
}
