// Window attention of 16-bit types on the 5th-generation tensor cores.
//
// A CTA takes 128 rows: TT = floor(128 / group) tokens times the group's query heads, which share
// their keys and values, and walks the 128-key tiles that any of the rows sees. Per tile
//   S = Q K^T      tcgen05 128 x 128 x dim, operands by TMA in the 128-byte swizzle, S in TMEM
//   P = exp2(S - m) two threads own a row (a TMEM lane), 64 keys each; they exchange their maxima
//   O += P V       P from TMEM (over S's columns, 16-bit pairs), V as it lies in memory (MN-major)
// The running maximum m is only raised when a row's tile maximum exceeds it by more than 8 (in
// log2): until then the weights are at most 2^8 and nothing has to be rescaled; a raise rescales
// O in TMEM. Weights are rounded to the operands' type for the product (as the output is), their sum
// is not. Float16 weights, and their sum with them, are 2^7 times as large, up to 2^15: so those down to 2^-21
// of the maximum keep all their bits and those below 2^-32 of it are lost, not 2^-14 and 2^-25, which many
// small ones behind one large would show.
//
// Two CTAs share an SM (96 KB of operands and 256 TMEM columns each), so one's products run
// under the other's exponentials: per tile the tensor pipe needs about 1000 cycles at dim 128 and
// the exponentials as many. 8192 positions, 32/8 heads of 128, window 1024 with 4 sinks, bfloat16: 245 us,
// 527 TFLOP/s of the visible pairs (a third more is computed, in tiles that the window cuts); the
// tensor pipe is 32 % busy. What bounds it is the chain of a tile in one CTA, 6500 cycles: 1700 for
// the products, 1400 until the maximum is known, 2200 for the weights, 700 of meeting and handing over.
// Other forms, measured beside one of 243 us: one thread a row (4 warps, S read twice) 250; half of the weights by a
// cubic instead of the exponential unit 240.
//
// A hidden key's weight is an exact zero, but zero times an infinity or NaN among its values would
// still reach the row. A row that comes out non-finite is therefore computed again key by key
// (row_attention), which reads visible keys only, and its query from the tile in shared memory: outputs may
// be in place of the queries. What the copying and the multiplying thread do is in mc_window_roles.h.
#pragma once
#include "mc_window_roles.h"
#include "mc_window_row.cuh"

namespace mc {
namespace win {

constexpr int kTcThreads = 320;          // 8 softmax warps, 1 TMA warp, 1 MMA warp
constexpr int kTcKeys = 128;             // keys per tile
constexpr int kTcMaxDim = 128;
constexpr int kTcBlock = 128 * 128;      // 128 rows x 64 16-bit values
constexpr uint32_t kTcCols = 256;        // TMEM: S (P over it) | O

struct TcArgs {
  Args a;
  int tokens;          // TT
  int out_vec;         // output rows take 16-byte stores
};

constexpr size_t tc_smem(int dim) { return 1024 + 3 * (size_t)((dim + 63) / 64) * kTcBlock; }

template <class T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <class T>
__global__ void __launch_bounds__(kTcThreads, 2)
tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
          const __grid_constant__ CUtensorMap mv, const __grid_constant__ TcArgs args) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[8];
  __shared__ uint32_t tmem_slot;
  __shared__ float redo[4][kTcMaxDim];
  __shared__ float exchange[2][2][128];  // [tile parity][half][row]
  const Args& a = args.a;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int dim = a.dim, blocks = (dim + 63) / 64;
  uint8_t* sq = smem;
  uint8_t* sk = sq + blocks * kTcBlock;
  uint8_t* sv = sk + blocks * kTcBlock;
  uint64_t *q_full = bars, *k_full = bars + 1, *v_full = bars + 2, *s_full = bars + 3, *p_full = bars + 4,
           *o_full = bars + 5, *v_free = bars + 6;

  check_segments(a);
  const int tile_id = gridDim.x - 1 - blockIdx.x, hk = blockIdx.y, tt = args.tokens;
  const int b = a.q_start ? tile_segment(a.q_start, a.n_seg, tt, tile_id) : 0;
  const Segment seg = segment(a, b);
  const int first = (tile_id - (a.q_start ? a.q_start[b] / tt + b : 0)) * tt;  // first token in the segment
  if (first < 0 || first >= seg.nq) return;
  const int tokens = min(tt, seg.nq - first);
  const int pos0 = seg.nk - seg.nq + first, pos1 = pos0 + tokens - 1;  // positions of the first and last token
  // tiles of keys: the sinks' (below the window) and the window's
  const int win_lo = window_begin(a.window, pos0);
  const int win_tile = win_lo / kTcKeys;
  const int sink_tiles = pos1 < 0 ? 0 : min(win_tile, (min(a.sinks, win_lo) + kTcKeys - 1) / kTcKeys);
  const int n_tiles = pos1 < 0 ? 0 : sink_tiles + pos1 / kTcKeys - win_tile + 1;
  auto tile_key = [&](int i) { return (i < sink_tiles ? i : win_tile + i - sink_tiles) * kTcKeys; };

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(k_full, 1);
    mbar_init(v_full, 1);
    mbar_init(s_full, 1);
    mbar_init(p_full, 256);
    mbar_init(o_full, 1);
    mbar_init(v_free, 1);
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(&tmem_slot, kTcCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t t_s = tmem, t_o = tmem + 128;
  // rows [first, first + tokens) x group of the segment; the row of a thread
  const int my_row = threadIdx.x & 127, half = threadIdx.x >> 7;
  const int row_token = my_row / a.group, row_head = my_row - row_token * a.group;

  if (warp == 8) {
    if (lane == 0 && n_tiles > 0) {
      struct {
        const CUtensorMap *mq, *mk, *mv;
        uint8_t *sq, *sk, *sv;
        uint64_t *q_full, *k_full, *v_full, *s_full, *v_free;
        int blocks, q_bytes, q_head, q_row, hk, k0, win_tile, sink_tiles;
        __device__ int key(int i) const { return k0 + (i < sink_tiles ? i : win_tile + i - sink_tiles) * kTcKeys; }
        __device__ void copy_queries() {
          mbar_arrive_expect_tx(q_full, (uint32_t)q_bytes);
          for (int c = 0; c < blocks; ++c) tma_load_3d(sq + c * kTcBlock, mq, 64 * c, q_head, q_row, q_full);
        }
        __device__ void copy_keys(int i) {
          mbar_arrive_expect_tx(k_full, (uint32_t)(blocks * kTcBlock));
          for (int c = 0; c < blocks; ++c) tma_load_3d(sk + c * kTcBlock, mk, 64 * c, hk, key(i), k_full);
        }
        __device__ void copy_values(int i) {
          mbar_arrive_expect_tx(v_full, (uint32_t)(blocks * kTcBlock));
          for (int c = 0; c < blocks; ++c) tma_load_3d(sv + c * kTcBlock, mv, 64 * c, hk, key(i), v_full);
        }
        __device__ bool wait_scores(int phase) { return mbar_wait_or_abort(s_full, phase, kErrWaitEmpty); }
        __device__ bool wait_values_free(int phase) { return mbar_wait_or_abort(v_free, phase, kErrWaitEmpty); }
        __device__ void drain_queries(int phase) { mbar_wait(q_full, phase, kErrWaitFull); }
        __device__ void drain_keys(int phase) { mbar_wait(k_full, phase, kErrWaitFull); }
        __device__ void drain_values(int phase) { mbar_wait(v_full, phase, kErrWaitFull); }
      } copier{&mq, &mk, &mv, sq, sk, sv, q_full, k_full, v_full, s_full, v_free, blocks, blocks * tt * a.group * 128,
               hk * a.group, seg.q0 + first, hk, seg.k0, win_tile, sink_tiles};
      copy_tiles(copier, n_tiles);
    }
  } else if (warp == 9) {
    if (lane == 0 && n_tiles > 0) {
      struct {
        uint64_t *q_full, *k_full, *v_full, *s_full, *p_full, *o_full, *v_free;
        uint64_t dq, dk, dv;
        uint32_t t_s, t_o, id_s, id_o;
        int dim;
        __device__ void multiply_scores() {
          for (int k = 0; k < dim / 16; ++k) {
            const uint64_t off = (uint64_t)((k >> 2) * (kTcBlock >> 4) + (k & 3) * 2);
            mma_f16(t_s, dq + off, dk + off, id_s, k > 0);
          }
          mma_commit(s_full);
        }
        __device__ void multiply_values(int i) {
          tc_fence_after();
          for (int k = 0; k < kTcKeys / 16; ++k)
            mma_f16_ts(t_o, t_s + 8 * k, dv + (uint64_t)k * (2048 >> 4), id_o, i > 0 || k > 0);
        }
        __device__ void commit_values_free() { mma_commit(v_free); }
        __device__ void commit_outputs() { mma_commit(o_full); }
        __device__ bool wait_queries(int phase) { return mbar_wait_or_abort(q_full, phase, kErrWaitFull); }
        __device__ bool wait_keys(int phase) { return mbar_wait_or_abort(k_full, phase, kErrWaitFull); }
        __device__ bool wait_values(int phase) { return mbar_wait_or_abort(v_full, phase, kErrWaitFull); }
        __device__ bool wait_weights(int phase) { return mbar_wait_or_abort(p_full, phase, kErrWaitAccFree); }
        __device__ void drain_outputs(int phase) { mbar_wait(o_full, phase, kErrWaitAcc); }
      } multiplier{q_full, k_full, v_full, s_full, p_full, o_full, v_free,
                   smem_desc_sw128(sq), smem_desc_sw128(sk), smem_desc_sw128_mn(sv, kTcBlock), t_s, t_o,
                   idesc_f16(128, kTcKeys, !std::is_same<T, __half>::value, false),
                   idesc_f16(128, dim, !std::is_same<T, __half>::value, true), dim};
      multiply_tiles(multiplier, n_tiles);
    }
  } else {
    const int pos = pos0 + row_token;  // of this thread's row
    const bool real = row_token < tokens;
    const int lo = window_begin(a.window, pos);
    const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
    const int c0 = 64 * half;  // this thread's keys of a tile
    constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;
    auto meet = []() { asm volatile("bar.sync 1, 256;" ::: "memory"); };  // the softmax warps
    float top = -INFINITY;
    float2 total = make_float2(0.f, 0.f);
    const float2 scale2 = make_float2(a.scale, a.scale);
    bool ok = true;
    for (int i = 0; i < n_tiles; ++i) {
      const int key = tile_key(i) + c0;
      ok = __all_sync(~0u, mbar_wait_or_abort(s_full, i & 1, kErrWaitAcc));
      float s[64], m = -INFINITY;
      if (ok) {
        tc_fence_after();
        tmem_ld32(t_s + lane_off + c0, *reinterpret_cast<uint32_t(*)[32]>(s));
        tmem_ld32(t_s + lane_off + c0 + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
        tmem_wait_ld();
        // visible: key + c in [lo, pos] or below the sinks (which never lie past pos)
        const int c_lo = lo - key, c_hi = pos - key, c_sink = min(a.sinks, pos + 1) - key;
        if (!__all_sync(~0u, c_hi >= 63 && (c_lo <= 0 || c_sink >= 64))) {
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (!((c >= c_lo && c <= c_hi) || c < c_sink)) s[c] = -INFINITY;
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 64; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) m4[e] = kv::max3(m4[e], s[c + 2 * e], s[c + 2 * e + 1]);
        m = __fmul_rn(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), a.scale);
        exchange[i & 1][half][my_row] = m;
      }
      meet();  // every softmax warp takes every tile's turn, also after a wait that gave up
      // the two threads of a row, and so the warps that have the same rows, decide alike
      m = fmaxf(m, exchange[i & 1][1 - half][my_row]);
      if (ok && __any_sync(~0u, m > top + 8.f || (top == -INFINITY && m > top))) {
        const float raised = fmaxf(top, m);
        const float keep = top == -INFINITY ? 0.f : exp2f(__fsub_rn(top, raised));
        total = kv::mul2(total, keep);
        top = raised;
        if (i > 0) {
          for (int c = 16 * half; c < dim; c += 32) {
            uint32_t x[16];
            tmem_ld16(t_o + lane_off + c, x);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__fmul_rn(__uint_as_float(x[e]), keep));
            tmem_st16(t_o + lane_off + c, x);
          }
        }
      }
      if (ok) {
        const float shift = top == -INFINITY ? 0.f : top - kLift;
        const float2 shift2 = make_float2(-shift, -shift);
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 x = kv::fma2(make_float2(s[c + 2 * e], s[c + 2 * e + 1]), scale2, shift2);
            const float2 y = make_float2(kv::exp2_fast(x.x), kv::exp2_fast(x.y));
            total = kv::add2(total, y);
            p[e] = pack16<T>(y.x, y.y);
          }
          // P's columns lie over scores that both threads of the row have read: they have met since
          tmem_st16(t_s + lane_off + (c0 + c) / 2, p);
        }
        tmem_wait_st();
        tc_fence_before();
      }
      mbar_arrive(p_full);
    }
    // ---- the output row: each thread every other 16 dimensions of it
    if (n_tiles > 0) ok = __all_sync(~0u, ok && mbar_wait_or_abort(o_full, 0, kErrWaitAcc));
    meet();
    exchange[0][half][my_row] = __fadd_rn(total.x, total.y);
    meet();
    const float sum = __fadd_rn(exchange[0][0][my_row], exchange[0][1][my_row]);
    float bad = 0.f;
    if (ok) {
      tc_fence_after();
      const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.0f, sum);
      const int row = seg.q0 + first + row_token, h = hk * a.group + row_head;
      T* out = static_cast<T*>(a.out.p) + row * a.out.row + h * a.out.head;
      for (int c = 16 * half; c < dim; c += 32) {
        uint32_t x[16];
        if (n_tiles > 0) {
          tmem_ld16(t_o + lane_off + c, x);
          tmem_wait_ld();
        }
        uint32_t y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float v0 = __uint_as_float(x[2 * e]), v1 = __uint_as_float(x[2 * e + 1]);
          if (n_tiles == 0) v0 = v1 = 0.f;
          bad = __fmaf_rn(v0, 0.f, __fmaf_rn(v1, 0.f, bad));  // NaN once a value is not finite
          y[e] = pack16<T>(__fmul_rn(v0, inv), __fmul_rn(v1, inv));
        }
        if (real && args.out_vec) {
          *reinterpret_cast<uint4*>(out + c) = make_uint4(y[0], y[1], y[2], y[3]);
          *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(y[4], y[5], y[6], y[7]);
        } else if (real) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const T* pair = reinterpret_cast<const T*>(&y[e]);
            out[c + 2 * e] = pair[0];
            out[c + 2 * e + 1] = pair[1];
          }
        }
      }
      bad = __fmaf_rn(sum, 0.f, bad);
    }
    exchange[1][half][my_row] = bad;
    meet();  // also orders the row's stores before those of a second computation
    if (ok && half == 0) {
      uint32_t again = __ballot_sync(~0u, real && !(exchange[1][0][my_row] == 0.f && exchange[1][1][my_row] == 0.f));
      // the queries from their tile: outputs may be in place of them. The copy has long landed; this wait is
      // for its bytes to be seen by this warp.
      if (again && !__all_sync(~0u, mbar_wait_or_abort(q_full, 0, kErrWaitFull))) again = 0;
      while (again) {
        const int l = __ffs(again) - 1, r = 32 * warp + l;
        again &= again - 1;
        auto query = [&](int d) {
          return *reinterpret_cast<const T*>(sq + (d >> 6) * kTcBlock + 128 * r + ((((d >> 3) & 7) ^ (r & 7)) << 4) + 2 * (d & 7));
        };
        row_attention<T>(a, seg.q0 + first + r / a.group, hk * a.group + r % a.group, seg.k0, pos0 + r / a.group, redo[warp], query);
        __syncwarp();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, kTcCols);
}

}  // namespace win
}  // namespace mc
