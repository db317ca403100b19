// Causal attention of whole segments with a sliding window and a few first positions that stay
// visible (sinks), over keys and values that are not quantised:
//   s_ij = scale q_i . k_j,  visible: j <= i and (j < sinks or j > i - window),
//   o_i = sum_j softmax(s_i)_j v_j,  zero for a row that sees nothing.
// A segment's queries are its last positions: query t of nq over nk keys is position nk - nq + t.
#include <type_traits>

#include "mc_kv_attend.cuh"
#include "mc_window_row.cuh"
#include "mc_window_tc.cuh"
#include "mc_window_tile.cuh"

namespace mc {
namespace win {

constexpr int kWindowRowThreads = 256;

template <class T>
__global__ void __launch_bounds__(kWindowRowThreads) row_kernel(const __grid_constant__ Args a) {
  __shared__ float qs[kWindowRowThreads / 32][kMaxDim];
  check_segments(a);
  const int warp = threadIdx.x >> 5;
  const long long item = (long long)blockIdx.x * (kWindowRowThreads / 32) + warp;
  const int row = (int)(item / a.q_heads), h = (int)(item % a.q_heads);
  if (row >= a.n_q) return;
  const int b = a.q_start ? segment_of(a.q_start, a.n_seg, row) : 0;
  if (b < 0) return;
  const Segment s = segment(a, b);
  if (s.nq == 0) return;
  row_attention<T>(a, row, h, s.k0, s.nk - s.nq + row - s.q0, qs[warp]);
}

// The tensor-core kernel takes head widths that are a multiple of its 16-wide products and rows that
// TMA can fetch: 16-byte aligned addresses and strides.
static bool tc_fits(const Args& a) {
  auto fits = [](const Rows& r) {
    return reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.row % 8 == 0 && r.head % 8 == 0 && r.row > 0 && r.head > 0 &&
           r.row < (1ll << 38) && r.head < (1ll << 38);
  };
  return a.dim % 16 == 0 && a.dim <= 128 && a.group <= 128 && a.n_k > 0 && fits(a.q) && fits(a.k) && fits(a.v);
}

template <class T>
static int tc_launch(const Args& a, cudaStream_t stream) {
  constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
  const int tokens = 128 / a.group;
  TcArgs args{a, tokens, reinterpret_cast<uintptr_t>(a.out.p) % 16 == 0 && a.out.row % 8 == 0 && a.out.head % 8 == 0};
  CUtensorMap mq, mk, mv;
  if (!make_tmap_16(&mq, a.q.p, bf, a.dim, a.q_heads, a.n_q, 2 * a.q.head, 2 * a.q.row, a.group, tokens)) return kCudaError;
  if (!make_tmap_16(&mk, a.k.p, bf, a.dim, a.heads, a.n_k, 2 * a.k.head, 2 * a.k.row, 1, kTcKeys)) return kCudaError;
  if (!make_tmap_16(&mv, a.v.p, bf, a.dim, a.heads, a.n_k, 2 * a.v.head, 2 * a.v.row, 1, kTcKeys)) return kCudaError;
  const size_t smem = tc_smem(a.dim);
  int device = 0;
  MC_CUDA(cudaGetDevice(&device));
  MC_CUDA(kv::allow_smem(reinterpret_cast<const void*>(tc_kernel<T>), device, (int)tc_smem(128)));
  const long long tiles = a.n_q / tokens + (long long)a.n_seg;
  if (tiles > INT_MAX || a.heads > 65535) return set_error(kInvalidArgument, "mc_window_attn_dev: too many rows or heads");
  tc_kernel<T><<<dim3((unsigned)tiles, a.heads), kTcThreads, smem, stream>>>(mq, mk, mv, args);
  MC_CUDA(cudaGetLastError());
  return kOk;
}

template <class T>
static int tile_launch(const Args& a, cudaStream_t stream) {
  int dimp = 0;
  auto f = tile_variant<T>(a.dim, &dimp);
  const size_t smem = tile_smem(dimp);
  const long long tiles = a.n_q / (kTileRows / a.group) + (long long)a.n_seg;
  if (tiles > INT_MAX || a.heads > 65535) return set_error(kInvalidArgument, "mc_window_attn_dev: too many rows or heads");
  auto aligned = [](const Rows& r) { return reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.row % 4 == 0 && r.head % 4 == 0; };
  auto paired = [](const Rows& r) { return reinterpret_cast<uintptr_t>(r.p) % (2 * sizeof(T)) == 0 && r.row % 2 == 0 && r.head % 2 == 0; };
  const bool quads = std::is_same<T, float>::value && a.dim % 4 == 0;
  // Heads one after the other in a CTA hide the start of all but the first (2000 prompts of 16-64 rows, 6
  // heads of 64: 319 us against 339), as long as the tiles, about half of the segments' last ones among
  // them, leave three waves of four CTAs an SM.
  int device = 0, n_sm = 0, heads = 1;
  MC_CUDA(cudaGetDevice(&device));
  MC_CUDA(kv::allow_smem(reinterpret_cast<const void*>(f), device, (int)smem));
  MC_CUDA(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, device));
  while (heads < a.heads && (a.n_q / (kTileRows / a.group) + a.n_seg / 2ll) * ((a.heads + heads) / (heads + 1)) >= 12ll * n_sm) ++heads;
  const TileArgs args{a, quads && aligned(a.k) && aligned(a.v), quads && aligned(a.q), a.dim % 2 == 0 && paired(a.out), heads};
  f<<<dim3((unsigned)tiles, (a.heads + args.heads - 1) / args.heads), kTileThreads, smem, stream>>>(args);
  MC_CUDA(cudaGetLastError());
  return kOk;
}

}  // namespace win
}  // namespace mc

extern "C" int mc_window_error(int device) {
  using namespace mc;
  clear_error();
  DeviceRestore restore_device;
  MC_CUDA(cudaSetDevice(device));
  MC_CUDA(cudaDeviceSynchronize());
  const int st = kv::take_timeout();
  if (st != kOk) return st;
  int code = 0;
  MC_CUDA(cudaMemcpyFromSymbol(&code, win::g_window_bounds, sizeof(int)));
  if (!code) return kOk;
  const int zero = 0;
  MC_CUDA(cudaMemcpyToSymbol(win::g_window_bounds, &zero, sizeof(int)));
  MC_CUDA(cudaDeviceSynchronize());
  return set_error(kInvalidArgument, "mc_window_attn_dev: a segment was out of range; its rows were skipped");
}

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
  if (dtype != kv::kF32 && tc_fits(a)) return dtype == kv::kF16 ? tc_launch<__half>(a, (cudaStream_t)stream) : tc_launch<__nv_bfloat16>(a, (cudaStream_t)stream);
  if (a.dim <= kTileMaxDim && a.group <= kTileRows)
    return dtype == kv::kF32   ? tile_launch<float>(a, (cudaStream_t)stream)
           : dtype == kv::kF16 ? tile_launch<__half>(a, (cudaStream_t)stream)
                               : tile_launch<__nv_bfloat16>(a, (cudaStream_t)stream);
  // wider heads and groups: a warp per row
  const long long blocks = ((long long)n_q * q_heads + kWindowRowThreads / 32 - 1) / (kWindowRowThreads / 32);
  if (blocks > INT_MAX) return set_error(kInvalidArgument, "mc_window_attn_dev: too many rows");
  void (*f)(Args) = dtype == kv::kF32 ? row_kernel<float> : dtype == kv::kF16 ? row_kernel<__half> : row_kernel<__nv_bfloat16>;
  f<<<(unsigned)blocks, kWindowRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  MC_CUDA(cudaGetLastError());
  return kOk;
}
