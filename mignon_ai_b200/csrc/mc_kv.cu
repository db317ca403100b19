// Kernels of the quantised key/value cache (mc_kv.cuh): quantising rows as they are written,
// reading them back, and one query token's attention over a session's cached positions.
#include <algorithm>
#include <climits>
#include <cmath>
#include <new>

#include "../../include/mignon_cuda.h"
#include "mc_host.h"
#include "mc_kv.cuh"
#include "mc_kv_attend.cuh"

namespace mc {
namespace kv {

constexpr int kCacheThreads = 256;

// ------------------------------------------------------------------------------------------------
// Write and read: one warp per (row, head), keys then values
// ------------------------------------------------------------------------------------------------
struct RowArgs {
  Cache c;
  Rows k, v;
  int n_rows, n_seg;
  const int *start, *sess, *pos0, *lens;
};

struct RowPlace {
  int session, slot;
};

// The warp's row: its session and slot; slot -1 where nothing is to be done.
__device__ __forceinline__ RowPlace write_place(const RowArgs& a, int row) {
  RowPlace w{0, -1};
  const int b = segment_of(a.start, a.n_seg, row);
  if (b < 0) return w;
  const int first = a.start ? a.start[b] : row, rows = a.start ? a.start[b + 1] - first : 1;
  w.session = a.sess ? a.sess[b] : b;
  const int pos0 = a.pos0[b];
  if ((unsigned)w.session >= (unsigned)a.c.sessions || pos0 < 0 || pos0 > INT_MAX - rows) {
    atomicExch(a.c.error, 1);
    return w;
  }
  const int pos = pos0 + (row - first);
  // a segment longer than the ring: only the positions that it leaves behind are written
  if (is_held(a.c, pos, pos0 + rows)) w.slot = slot_of(a.c, pos);
  return w;
}

template <class T>
__global__ void __launch_bounds__(kCacheThreads) write_kernel(const __grid_constant__ RowArgs a) {
  __shared__ int8_t codes[kCacheThreads / 32][kMaxDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * (kCacheThreads / 32) + warp;
  const int row = (int)(item / a.c.heads), head = (int)(item % a.c.heads);
  if (row >= a.n_rows) return;
  const RowPlace w = write_place(a, row);
  if (w.slot < 0) return;
  const int dim = a.c.dim, bits = a.c.bits, cb = a.c.cb;
  uint8_t* region = region_of(a.c, w.session, head);
  int8_t* cs = codes[warp];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const Rows& r = which ? a.v : a.k;
    const T* x = static_cast<const T*>(r.p) + row * r.row + head * r.head;
    float v[kMaxDim / 32];
    float hi = -INFINITY, lo = INFINITY, bad = 0.f;
#pragma unroll
    for (int u = 0; u < kMaxDim / 32; ++u) {
      const int d = lane + 32 * u;
      if (d >= dim) break;
      v[u] = to_float<T>(x[d]);
      hi = fmaxf(hi, v[u]);
      lo = fminf(lo, v[u]);
      bad = __fmaf_rn(v[u], 0.f, bad);  // NaN once an element is not finite
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, o));
      lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
      bad = __fadd_rn(bad, __shfl_xor_sync(~0u, bad, o));
    }
    const Quant q = quant_of(hi, lo, bad == 0.f, bits);
#pragma unroll
    for (int u = 0; u < kMaxDim / 32; ++u) {
      const int d = lane + 32 * u;
      if (d < dim) cs[d] = (int8_t)code_of(q, v[u], bits);
    }
    __syncwarp();
    const int g = w.slot >> 2, s = w.slot & 3;
    if (which == 0) {
      uint32_t* out = reinterpret_cast<uint32_t*>(region + (long long)g * 4 * cb);
      for (int i = lane; i < cb / 4; i += 32) {
        uint32_t word = 0;
        for (int b = 0; b < 4; ++b)
          word |= (uint32_t)(bits == 4 ? (cs[8 * i + b] & 15) | ((cs[8 * i + 4 + b] & 15) << 4) : (uint8_t)cs[4 * i + b])
                  << (8 * b);
        out[4 * i + s] = word;
      }
    } else {
      uint8_t* out = region + values_offset(a.c) + (long long)g * 4 * cb;
      const int ni = cb / 8;
      for (int j = lane; j < cb; j += 32) {
        const int n = j / ni, i = j % ni;
        out[4 * j + s] = (uint8_t)(bits == 4 ? (cs[16 * i + n] & 15) | ((cs[16 * i + 8 + n] & 15) << 4) : cs[8 * i + n]);
      }
    }
    if (lane == 0)
      reinterpret_cast<uint32_t*>(region + params_offset(a.c))[(which ? a.c.cap : 0) + w.slot] = param_word(q);
    __syncwarp();
  }
}

__device__ __forceinline__ int signed_nibble(uint32_t byte, int high) {
  return (int)(byte << (high ? 24 : 28)) >> 28;
}

template <class T>
__global__ void __launch_bounds__(kCacheThreads) read_kernel(const __grid_constant__ RowArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * (kCacheThreads / 32) + warp;
  const int row = (int)(item / a.c.heads), head = (int)(item % a.c.heads);
  if (row >= a.n_rows) return;
  const int b = segment_of(a.start, a.n_seg, row);
  int session = 0, pos = 0;
  bool held = b >= 0;  // rows of no segment, and positions that are not held, come back as zeros
  if (held) {
    session = a.sess ? a.sess[b] : b;
    const int ahead = a.start ? row - a.start[b] : 0;
    held = (unsigned)session < (unsigned)a.c.sessions && a.pos0[b] >= 0 && a.pos0[b] <= INT_MAX - ahead;
    if (!held) atomicExch(a.c.error, 1);
    pos = held ? a.pos0[b] + ahead : 0;
    held = held && is_held(a.c, pos, a.lens[b]);
  }
  const int dim = a.c.dim, bits = a.c.bits, cb = a.c.cb;
  const int slot = held ? slot_of(a.c, pos) : 0, g = slot >> 2, s = slot & 3;
  const uint8_t* region = region_of(a.c, held ? session : 0, head);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const Rows& r = which ? a.v : a.k;
    T* y = static_cast<T*>(r.p) + row * r.row + head * r.head;
    const uint8_t* codes = region + (which ? values_offset(a.c) : 0) + (long long)g * 4 * cb;
    uint32_t param = 0;
    if (held) param = reinterpret_cast<const uint32_t*>(region + params_offset(a.c))[(which ? a.c.cap : 0) + slot];
    const float scale = param_scale(param), center = param_center(param);
    for (int d = lane; d < dim; d += 32) {
      float m = 0.f;
      if (held) {
        if (which == 0) {
          const int word = bits == 4 ? d / 8 : d / 4;
          const uint32_t byte = codes[16 * word + 4 * s + d % 4];
          m = bits == 4 ? (float)(2 * signed_nibble(byte, (d >> 2) & 1) + 1) : (float)(int8_t)byte;
        } else {
          const int ni = cb / 8, n = d % 8, i = bits == 4 ? d / 16 : d / 8;
          const uint32_t byte = codes[4 * (n * ni + i) + s];
          m = bits == 4 ? (float)(2 * signed_nibble(byte, (d >> 3) & 1) + 1) : (float)(int8_t)byte;
        }
      }
      y[d] = from_float<T>(held ? __fmaf_rn(scale, m, center) : 0.f);
    }
  }
}

}  // namespace kv
}  // namespace mc

// ------------------------------------------------------------------------------------------------
// C-ABI
// ------------------------------------------------------------------------------------------------
struct mc_kv {
  int device = 0;
  mc::kv::Cache c{};
  void* mem = nullptr;       // error word, arrival counters, partial results, regions
  int* arrived = nullptr;
  float* partial = nullptr;
  int n_sm = 0;
};

namespace mc {
namespace kv {

static bool rows_ok(const mc_rows* r) { return r && r->data; }
static Rows rows_of(const mc_rows* r) { return Rows{r->data, (long long)r->row_stride, (long long)r->head_stride}; }

static int row_launch(const char* name, bool write, mc_kv* kv, const mc_rows* k, const mc_rows* v, int dtype, int n_rows,
                      const int32_t* start, const int32_t* sess, const int32_t* pos0, const int32_t* lens, int n_seg,
                      cudaStream_t stream) {
  clear_error();
  if (!kv || !rows_ok(k) || !rows_ok(v) || !pos0 || (!write && !lens))
    return set_error(kInvalidArgument, std::string(name) + ": null argument");
  if (dtype < kF32 || dtype > kBF16) return set_error(kInvalidArgument, std::string(name) + ": unknown dtype");
  if (n_rows < 0 || n_seg < 0 || (!start && n_rows != n_seg))
    return set_error(kInvalidArgument, std::string(name) + ": negative counts, or rows without row_start that are not one per segment");
  if (n_rows == 0 || n_seg == 0) return kOk;
  DeviceRestore restore_device;
  MC_CUDA(cudaSetDevice(kv->device));
  const RowArgs a{kv->c, rows_of(k), rows_of(v), n_rows, n_seg, start, sess, pos0, lens};
  const long long blocks = ((long long)n_rows * kv->c.heads + kCacheThreads / 32 - 1) / (kCacheThreads / 32);
  if (blocks > INT_MAX) return set_error(kInvalidArgument, std::string(name) + ": too many rows");
  void (*f)(RowArgs) = nullptr;
  if (write) f = dtype == kF32 ? write_kernel<float> : dtype == kF16 ? write_kernel<__half> : write_kernel<__nv_bfloat16>;
  else f = dtype == kF32 ? read_kernel<float> : dtype == kF16 ? read_kernel<__half> : read_kernel<__nv_bfloat16>;
  f<<<(unsigned)blocks, kCacheThreads, 0, stream>>>(a);
  MC_CUDA(cudaGetLastError());
  return kOk;
}

}  // namespace kv
}  // namespace mc

extern "C" int mc_kv_open(int device, const mc_kv_spec* spec, mc_kv** out) {
  using namespace mc;
  clear_error();
  if (!spec || !out) return set_error(kInvalidArgument, "mc_kv_open: null argument");
  *out = nullptr;
  const mc_kv_spec& s = *spec;
  if (s.sessions < 1 || s.heads < 1 || s.slots < 1)
    return set_error(kInvalidArgument, "mc_kv_open: sessions, heads and slots must be positive");
  if (s.head_dim < 16 || s.head_dim > kv::kMaxDim || s.head_dim % 16)
    return set_error(kInvalidArgument, "mc_kv_open: head_dim must be a multiple of 16 from 16 to 128");
  if (s.bits != 4 && s.bits != 8) return set_error(kInvalidArgument, "mc_kv_open: bits must be 4 or 8");
  if (s.sinks < 0 || s.sinks >= s.slots) return set_error(kInvalidArgument, "mc_kv_open: sinks must be in [0, slots)");
  if (s.slots > (1 << 30)) return set_error(kInvalidArgument, "mc_kv_open: slots above 2^30");
  DeviceRestore restore_device;
  MC_CUDA(cudaSetDevice(device));
  kv::Cache c{};
  c.sessions = s.sessions;
  c.heads = s.heads;
  c.dim = s.head_dim;
  c.bits = s.bits;
  c.slots = s.slots;
  c.sinks = s.sinks;
  c.ring = s.slots - s.sinks;
  c.cap = (s.slots + 63) / 64 * 64;
  c.cb = s.head_dim * s.bits / 8;
  c.region = 2ll * c.cap * (c.cb + 4);
  // the workspace of mc_kv_attend_dev is part of the cache, so that no call allocates
  const size_t head = 256 + kv::kMaxPartials * (sizeof(int) + kv::kAttendRows * (2 + s.head_dim) * sizeof(float));
  const double need = (double)c.region * s.sessions * s.heads + (double)head;
  size_t bytes = 0;
  void* mem = nullptr;
  int n_sm = 0;
  MC_CUDA(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, device));
  if (need < 9e18) bytes = (size_t)c.region * s.sessions * s.heads + head;
  if (!bytes || cudaMalloc(&mem, bytes) != cudaSuccess) {
    (void)cudaGetLastError();
    return set_error(kOutOfMemory, "mc_kv_open: no room for a cache of " + std::to_string(need) + " bytes");
  }
  const cudaError_t e = cudaMemset(mem, 0, bytes);
  if (e != cudaSuccess) {
    cudaFree(mem);
    return set_error(kCudaError, std::string("mc_kv_open: cudaMemset: ") + cudaGetErrorString(e));
  }
  c.error = static_cast<int*>(mem);
  c.base = static_cast<uint8_t*>(mem) + head;  // a multiple of 256
  mc_kv* kv = new (std::nothrow) mc_kv;
  if (!kv) {
    cudaFree(mem);
    return set_error(kOutOfMemory, "mc_kv_open: out of host memory");
  }
  kv->device = device;
  kv->c = c;
  kv->mem = mem;
  kv->arrived = reinterpret_cast<int*>(static_cast<uint8_t*>(mem) + 256);
  kv->partial = reinterpret_cast<float*>(kv->arrived + kv::kMaxPartials);
  kv->n_sm = n_sm;
  *out = kv;
  return kOk;
}

extern "C" int mc_kv_close(mc_kv* kv) {
  using namespace mc;
  clear_error();
  if (!kv) return kOk;
  DeviceRestore restore_device;
  cudaSetDevice(kv->device);
  const cudaError_t e = cudaFree(kv->mem);  // waits for the device's work
  delete kv;
  if (e != cudaSuccess) return set_error(kCudaError, std::string("mc_kv_close: ") + cudaGetErrorString(e));
  return kOk;
}

extern "C" int mc_kv_error(mc_kv* kv) {
  using namespace mc;
  clear_error();
  if (!kv) return set_error(kInvalidArgument, "mc_kv_error: null cache");
  DeviceRestore restore_device;
  MC_CUDA(cudaSetDevice(kv->device));
  MC_CUDA(cudaDeviceSynchronize());
  const int st = check_device_error(0);
  if (st != kOk) return st;
  int code = 0;
  MC_CUDA(cudaMemcpy(&code, kv->c.error, sizeof(int), cudaMemcpyDeviceToHost));
  if (!code) return kOk;
  MC_CUDA(cudaMemset(kv->c.error, 0, sizeof(int)));
  return set_error(kInvalidArgument, "mc_kv: a session or a position was out of range; its rows were skipped");
}

extern "C" int mc_kv_write_dev(mc_kv* kv, const mc_rows* k, const mc_rows* v, int dtype, int n_rows,
                               const int32_t* row_start, const int32_t* sessions, const int32_t* pos0, int n_segments,
                               void* stream) {
  return mc::kv::row_launch("mc_kv_write_dev", true, kv, k, v, dtype, n_rows, row_start, sessions, pos0, nullptr,
                            n_segments, static_cast<cudaStream_t>(stream));
}

extern "C" int mc_kv_read_dev(mc_kv* kv, const mc_rows* k, const mc_rows* v, int dtype, int n_rows,
                              const int32_t* row_start, const int32_t* sessions, const int32_t* pos0,
                              const int32_t* lens, int n_segments, void* stream) {
  return mc::kv::row_launch("mc_kv_read_dev", false, kv, k, v, dtype, n_rows, row_start, sessions, pos0, lens,
                            n_segments, static_cast<cudaStream_t>(stream));
}

extern "C" int mc_kv_attend_dev(mc_kv* kv, const mc_rows* q, const mc_rows* out, int dtype, int q_heads,
                                const int32_t* sessions, const int32_t* lens, int n, int window, float scale,
                                void* stream) {
  using namespace mc;
  using namespace mc::kv;
  clear_error();
  if (!kv || !rows_ok(q) || !rows_ok(out) || !lens) return set_error(kInvalidArgument, "mc_kv_attend_dev: null argument");
  if (dtype < kF32 || dtype > kBF16) return set_error(kInvalidArgument, "mc_kv_attend_dev: unknown dtype");
  if (n < 0 || window < 0) return set_error(kInvalidArgument, "mc_kv_attend_dev: n and window must not be negative");
  if (q_heads < 1 || q_heads % kv->c.heads)
    return set_error(kInvalidArgument, "mc_kv_attend_dev: q_heads must be a multiple of the cache's heads");
  if (!(scale > 0.f) || !std::isfinite(scale)) return set_error(kInvalidArgument, "mc_kv_attend_dev: scale must be positive");
  if (n == 0) return kOk;
  DeviceRestore restore_device;
  MC_CUDA(cudaSetDevice(kv->device));
  const Cache& c = kv->c;
  const int group = q_heads / c.heads, row_groups = (group + kAttendRows - 1) / kAttendRows;
  const long long items = (long long)n * c.heads * row_groups;
  // warps an item's slots are split over: enough for two waves of the 16 warps an SM holds, while
  // each keeps two tiles of 64 slots
  const int seen = window > 0 ? (int)std::min<long long>(c.slots, (long long)window + c.sinks) : c.slots;
  const long long wanted = std::min<long long>((2ll * 16 * kv->n_sm + items - 1) / items, (seen + 127) / 128);
  const bool split = wanted > 1;
  int pieces = 1;
  if (split) pieces = (int)std::max<long long>(1, std::min<long long>((wanted + kAttendWarps - 1) / kAttendWarps, kMaxPartials / items));
  const AttendArgs a{c, rows_of(q), rows_of(out), n, q_heads, group, row_groups, window, dtype, pieces, sessions, lens,
                     scale * 1.4426950408889634f, kv->partial, kv->arrived};
  const long long blocks = split ? items : (items + kAttendWarps - 1) / kAttendWarps;
  if (blocks > INT_MAX) return set_error(kInvalidArgument, "mc_kv_attend_dev: too many rows");
  const int planes = dtype == kF32 ? 3 : 2;
  auto f = c.bits == 4 ? attend_variant_of<4>(c.dim, planes, split) : attend_variant_of<8>(c.dim, planes, split);
  f<<<dim3((unsigned)blocks, pieces), kAttendWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(a);
  MC_CUDA(cudaGetLastError());
  return kOk;
}
