// Kernels of the quantised key/value cache (mc_kv.cuh): quantising rows as they are written,
// reading them back, and one query token's attention over a session's cached positions.
#include <algorithm>
#include <climits>
#include <cmath>
#include <mutex>
#include <new>
#include <set>
#include <type_traits>
#include <utility>

#include "../../include/mignon_cuda.h"
#include "mc_host.h"
#include "mc_kv.cuh"
#include "mc_kv_attend.cuh"

namespace mc {
namespace kv {

constexpr int kCacheThreads = 256;

// ------------------------------------------------------------------------------------------------
// Write and read
//
// Both move a row's codes between its dtype and the interleaved layout. A segment's rows go four
// at a time: the rows of one group of slots (four consecutive slots, the first a multiple of
// four), eight lanes to a row, a lane eight consecutive dimensions of it (and the eight 64 further
// on). Then every access is a full word or vector: the keys' words of four rows are 16 consecutive
// bytes, and the values' words, which hold one dimension of four rows, are made by a byte
// transpose over the four rows' lanes (two shuffles); at the ends of a segment the values' bytes are
// written one by one. Rows whose slots do not follow their order in a group (past a ring's end that is
// not a multiple of four) and single tokens go one at a time by a whole warp.
//
// What bounds it: reading, memory (65,536 rows of 8 heads of 128 from 4 bits: 64 us, 0.81 of the copy rate);
// writing, instruction issue, 82 % busy at about seven instructions a value (80,000 such rows: 129 us, memory's
// share 64); single tokens, the latency of a warp's dependent loads and narrow stores (4096 of 4 heads of 32: 12.5 us
// to write, 9.3 to read). 48 registers for 40 warps an SM: 32 warps took a tenth longer, 24 a half.
// ------------------------------------------------------------------------------------------------
struct RowArgs {
  Cache c;
  Rows k, v;
  int n_rows, n_seg;
  const int *start, *sess, *pos0, *lens;
  int vec;         // rows are aligned for 16-byte accesses of eight elements
  int warp_heads;  // heads that a warp of segment_kernel takes one after the other
  float spread;    // segments per row, on average
};

// Where a row goes or comes from: its session and slot, slot -1 for none.
struct RowPlace {
  int session, slot;
};

// Row `row` of segment b, whose first row is `first` of `rows`.
template <bool WRITE>
__device__ __forceinline__ RowPlace place(const RowArgs& a, int b, int first, int rows, int row) {
  RowPlace w{a.sess ? a.sess[b] : b, -1};
  const int pos0 = a.pos0[b];
  if ((unsigned)w.session >= (unsigned)a.c.sessions || pos0 < 0 || pos0 > INT_MAX - rows) {
    atomicExch(a.c.error, 1);
    w.session = 0;
    return w;
  }
  const int pos = pos0 + (row - first);
  // writing a segment longer than the ring: only the positions that it leaves behind
  if (is_held(a.c, pos, WRITE ? pos0 + rows : a.lens[b])) w.slot = slot_of(a.c, pos);
  return w;
}

__device__ __forceinline__ int signed_nibble(uint32_t byte, int high) { return (int)(byte << (high ? 24 : 28)) >> 28; }

// One row by a warp: lanes own dimensions lane + 32u. `cs` holds kMaxDim codes of the warp's.
template <class T>
__device__ void write_row(const RowArgs& a, int row, int head, RowPlace w, int8_t* cs) {
  const int lane = threadIdx.x & 31, dim = a.c.dim, bits = a.c.bits, cb = a.c.cb;
  uint8_t* region = region_of(a.c, w.session, head);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const Rows& r = which ? a.v : a.k;
    const T* x = static_cast<const T*>(r.p) + row * r.row + head * r.head;
    float v[kMaxDim / 32];
    float hi = -INFINITY, lo = INFINITY;
#pragma unroll
    for (int u = 0; u < kMaxDim / 32; ++u) {
      const int d = lane + 32 * u;
      if (d >= dim) break;
      v[u] = to_float<T>(x[d]);
      hi = max_nan(hi, v[u]);
      lo = min_nan(lo, v[u]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      hi = max_nan(hi, __shfl_xor_sync(~0u, hi, o));
      lo = min_nan(lo, __shfl_xor_sync(~0u, lo, o));
    }
    const Quant q = quant_of(hi, lo, bits);
#pragma unroll
    for (int u = 0; u < kMaxDim / 32; ++u) {
      const int d = lane + 32 * u;
      if (d < dim) cs[d] = (int8_t)code_bits(q, v[u], bits);
    }
    __syncwarp();
    const int s = w.slot & 3;
    const int g = w.slot >> 2;
    if (which == 0) {
      uint32_t* out = keys_of(a.c, region, w.slot);
      for (int i = lane; i < cb / 4; i += 32) {
        uint32_t word = 0;
        for (int b = 0; b < 4; ++b)
          word |= (uint32_t)(bits == 4 ? (cs[8 * i + b] & 15) | ((cs[8 * i + 4 + b] & 15) << 4) : (uint8_t)cs[4 * i + b])
                  << (8 * b);
        out[4 * key_unit(i, g, cb, bits) + s] = word;
      }
    } else {
      uint8_t* out = reinterpret_cast<uint8_t*>(values_of(a.c, region, w.slot));
      const int ni = cb / 8;
      for (int j = lane; j < cb; j += 32) {
        const int n = j / ni, i = j % ni;
        out[4 * value_word(n, i, g, ni) + s] = (uint8_t)(bits == 4 ? (cs[16 * i + n] & 15) | ((cs[16 * i + 8 + n] & 15) << 4) : cs[8 * i + n]);
      }
    }
    if (lane == 0) *params_of(a.c, region, w.slot, which) = param_word(q);
    __syncwarp();
  }
}

template <class T>
__device__ void read_row(const RowArgs& a, int row, int head, RowPlace w) {
  const int lane = threadIdx.x & 31, dim = a.c.dim, bits = a.c.bits, cb = a.c.cb;
  const bool held = w.slot >= 0;
  const int slot = held ? w.slot : 0, s = slot & 3;
  uint8_t* region = region_of(a.c, w.session, head);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const Rows& r = which ? a.v : a.k;
    T* y = static_cast<T*>(r.p) + row * r.row + head * r.head;
    const uint8_t* codes = reinterpret_cast<const uint8_t*>(which ? values_of(a.c, region, slot) : keys_of(a.c, region, slot));
    const uint32_t param = held ? *params_of(a.c, region, slot, which) : 0;
    const float scale = param_scale(param), center = param_center(param);
    for (int d = lane; d < dim; d += 32) {
      float m = 0.f;
      if (held) {
        uint32_t byte;
        if (which == 0) {
          byte = codes[16 * key_unit(bits == 4 ? d / 8 : d / 4, slot >> 2, cb, bits) + 4 * s + d % 4];
        } else {
          byte = codes[4 * value_word(d % 8, bits == 4 ? d / 16 : d / 8, slot >> 2, cb / 8) + s];
        }
        m = bits == 4 ? (float)(2 * signed_nibble(byte, (d >> (which ? 3 : 2)) & 1) + 1) : (float)(int8_t)byte;
      }
      y[d] = from_float<T>(held ? __fmaf_rn(scale, m, center) : 0.f);
    }
  }
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8], bool vec) {
  if (vec) {
    alignas(16) T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_float<T>(x[i]);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_float<T>(x[i]);
  }
}

// 4 x 4 bytes transposed over the four rows' lanes (s = lane / 8): lane s gives the bytes n of its
// row and gets the bytes of dimension n = s, row 0's lowest. Its own inverse.
__device__ __forceinline__ uint32_t transpose_bytes(uint32_t x, int s) {
  uint32_t y = __shfl_xor_sync(~0u, x, 8);
  x = s & 1 ? __byte_perm(y, x, 0x7351) : __byte_perm(x, y, 0x6240);  // rows 2t, 2t + 1 of n = s % 2 and s % 2 + 2
  y = __shfl_xor_sync(~0u, x, 16);
  return s & 2 ? __byte_perm(y, x, 0x7632) : __byte_perm(x, y, 0x5410);
}

// Where a lane's words of a group of slots are, from the start of its block: the same for every head.
// Lane (s, c): row s, chunks of eight dimensions c and c + 8 (u). Keys: 4 bits one word a chunk, 8 bits two;
// values: likewise, after the transpose.
template <int BITS>
struct LaneWords {
  static constexpr int W = BITS / 4;
  int key[2][W], value[2][W];
  __device__ __forceinline__ LaneWords(int slot0, int cb) {
    const int lane = threadIdx.x & 31, s = lane >> 3, c = lane & 7, g = slot0 >> 2, ni = cb / 8;
    const int kbase = ((slot0 & 31) >> 2) * cb, vbase = kBlockSlots * (cb + 4) / 4 + ((slot0 & 31) >> 3) * 2 * cb;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int chunk = c + 8 * u;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        key[u][w] = kbase + 4 * key_unit(W * chunk + w, g, cb, BITS) + s;
        value[u][w] = vbase + (BITS == 4 ? value_word(4 * (chunk & 1) + s, chunk >> 1, g, ni) : value_word(4 * w + s, chunk, g, ni));
      }
    }
  }
};

// The words of scale and center of slot0's keys, from the start of its block (the values': kBlockSlots
// (cb + 4) bytes on).
__device__ __forceinline__ int param_word_at(int slot0, int cb) { return kBlockSlots * cb / 4 + (slot0 & 31); }

// Eight consecutive elements as they are in memory.
template <class T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
      alignas(16) T e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(e)[i];
    }
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float<T>(e[i]);
  }
};

// The extremes of a row held by eight lanes (NaN once an element is). 16-bit elements are compared in
// pairs, as they are.
template <class T>
__device__ __forceinline__ void row_extremes(const Raw8<T> (&raw)[2], const bool (&in)[2], float& hi, float& lo) {
  if constexpr (sizeof(T) == 4) {
    hi = -INFINITY, lo = INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (in[u]) {
        float x[8];
        raw[u].get(x);
#pragma unroll
        for (int e = 0; e < 8; ++e) hi = max_nan(hi, x[e]), lo = min_nan(lo, x[e]);
      }
#pragma unroll
    for (int o = 1; o <= 4; o <<= 1) {
      hi = max_nan(hi, __shfl_xor_sync(~0u, hi, o));
      lo = min_nan(lo, __shfl_xor_sync(~0u, lo, o));
    }
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 h, l;
    h.x = h.y = from_float<T>(-INFINITY);
    l.x = l.y = from_float<T>(INFINITY);
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (in[u]) {
        const T2* e = reinterpret_cast<const T2*>(raw[u].w);
#pragma unroll
        for (int i = 0; i < 4; ++i) h = __hmax2_nan(h, e[i]), l = __hmin2_nan(l, e[i]);
      }
    T2 both;  // the maximum of the elements and that of their negatives
    both.x = __hmax_nan(h.x, h.y);
    both.y = __hneg(__hmin_nan(l.x, l.y));
#pragma unroll
    for (int o = 1; o <= 4; o <<= 1) {
      const uint32_t other = __shfl_xor_sync(~0u, *reinterpret_cast<const uint32_t*>(&both), o);
      both = __hmax2_nan(both, *reinterpret_cast<const T2*>(&other));
    }
    hi = to_float<T>(both.x);
    lo = -to_float<T>(both.y);
  }
}

// The rows of one group of slots, heads [h0, h1): lane (s, c) has the row of slot0 + s, if that is `live`.
template <class T, int BITS>
__device__ void write_group(const RowArgs& a, int row, bool live, int h0, int h1, int session, int slot0) {
  const int lane = threadIdx.x & 31, s = lane >> 3, c0 = lane & 7, chunks = a.c.dim / 8, cb = a.c.cb;
  const LaneWords<BITS> at(slot0, cb);
  const int param_at = param_word_at(slot0, cb) + s;
  uint32_t* block = reinterpret_cast<uint32_t*>(region_of(a.c, session, h0) + (long long)(slot0 >> 5) * block_bytes(cb));
  const T* rows[2] = {static_cast<const T*>(a.k.p) + row * a.k.row + h0 * a.k.head + 8 * c0,
                      static_cast<const T*>(a.v.p) + row * a.v.row + h0 * a.v.head + 8 * c0};
  const bool in[2] = {c0 < chunks, c0 + 8 < chunks};
  const unsigned rows_live = __ballot_sync(~0u, live);  // a row's eight lanes alike
  // a word of values, one byte a row: whole, or the bytes of the rows there are
  auto store_values = [&](uint32_t* at_word, uint32_t word) {
    if (rows_live == ~0u) {
      *at_word = word;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (rows_live >> (8 * r) & 1) reinterpret_cast<uint8_t*>(at_word)[r] = (uint8_t)(word >> (8 * r));
    }
  };
  for (int h = h0; h < h1; ++h) {
    Raw8<T> raw[2][2];
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (in[u] && live) raw[which][u].load(rows[which] + 64 * u, a.vec);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float hi, lo;
      row_extremes<T>(raw[which], in, hi, lo);
      const Quant q = quant_of(hi, lo, BITS);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (8 * u >= chunks) break;  // uniform
        uint32_t code[8];
        float x[8];
        raw[which][u].get(x);
        code_bits8<BITS>(q, x, code);
        const uint32_t b0 = pack_low_bytes(code[0], code[1], code[2], code[3]);
        const uint32_t b1 = pack_low_bytes(code[4], code[5], code[6], code[7]);
        if (which == 0) {
          if constexpr (BITS == 4) {
            if (in[u] && live) block[at.key[u][0]] = (b0 & 0x0F0F0F0Fu) | ((b1 << 4) & 0xF0F0F0F0u);
          } else if (in[u] && live) {
            block[at.key[u][0]] = b0;
            block[at.key[u][BITS / 4 - 1]] = b1;
          }
        } else if constexpr (BITS == 4) {
          // even chunks (low nibbles) keep dimensions n = 0..3 of the pair, odd ones (high) n = 4..7
          const bool odd = c0 & 1;
          const uint32_t got = __shfl_xor_sync(~0u, odd ? b0 : b1, 1);
          const uint32_t low = odd ? got : b0, high = odd ? b1 : got;
          const uint32_t word = transpose_bytes((low & 0x0F0F0F0Fu) | ((high << 4) & 0xF0F0F0F0u), s);
          if (in[u]) store_values(block + at.value[u][0], word);
        } else {
          const uint32_t w0 = transpose_bytes(b0, s), w1 = transpose_bytes(b1, s);
          if (in[u]) {
            store_values(block + at.value[u][0], w0);
            store_values(block + at.value[u][BITS / 4 - 1], w1);
          }
        }
      }
      if (c0 == 0 && live) block[param_at + (which ? kBlockSlots * (cb + 4) / 4 : 0)] = param_word(q);
      rows[which] += which ? a.v.head : a.k.head;
    }
    block += a.c.region / 4;
  }
}

// Four codes as they are in bytes biased by 128: 2^23 + byte is a float whose low byte it is.
__device__ __forceinline__ void decode4(float* x, uint32_t biased, float2 scale, float2 center) {
#pragma unroll
  for (int e = 0; e < 4; e += 2) {
    const float2 f = make_float2(__uint_as_float(__byte_perm(biased, 0x4B000000u, 0x7440 + e)),
                                 __uint_as_float(__byte_perm(biased, 0x4B000000u, 0x7441 + e)));
    const float2 y = fma2(scale, add2(f, make_float2(-8388736.0f, -8388736.0f)), center);
    x[e] = y.x, x[e + 1] = y.y;
  }
}

// As write_group; a row that is `mine` but not live comes back as zeros.
template <class T, int BITS>
__device__ void read_group(const RowArgs& a, int row, bool mine, bool live, int h0, int h1, int session, int slot0) {
  constexpr int W = BITS / 4;
  const int lane = threadIdx.x & 31, s = lane >> 3, c0 = lane & 7, chunks = a.c.dim / 8, cb = a.c.cb;
  const LaneWords<BITS> at(slot0, cb);
  const int param_at = param_word_at(slot0, cb) + s;
  const uint32_t* block = reinterpret_cast<const uint32_t*>(region_of(a.c, session, h0) + (long long)(slot0 >> 5) * block_bytes(cb));
  T* rows[2] = {static_cast<T*>(a.k.p) + row * a.k.row + h0 * a.k.head + 8 * c0,
                static_cast<T*>(a.v.p) + row * a.v.row + h0 * a.v.head + 8 * c0};
  const bool in[2] = {c0 < chunks, c0 + 8 < chunks};
  // a head's words, loaded while the head before it is decoded
  uint32_t w[2][2][W] = {}, param[2], w_next[2][2][W] = {}, param_next[2];
  auto load = [&](const uint32_t* from, uint32_t (&words)[2][2][W], uint32_t (&params)[2]) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (in[u]) {
#pragma unroll
          for (int i = 0; i < W; ++i) words[which][u][i] = __ldg(from + (which ? at.value[u][i] : at.key[u][i]));
        }
      params[which] = __ldg(from + param_at + (which ? kBlockSlots * (cb + 4) / 4 : 0));
    }
  };
  load(block, w_next, param_next);
  for (int h = h0; h < h1; ++h) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      param[which] = param_next[which];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < W; ++i) w[which][u][i] = w_next[which][u][i];
    }
    block += a.c.region / 4;
    if (h + 1 < h1) load(block, w_next, param_next);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      // nibbles come as bytes 16c + 8 = 8m, so their scale is an eighth
      const float scale = __fmul_rn(param_scale(param[which]), BITS == 4 ? 0.125f : 1.0f), center = param_center(param[which]);
      const float2 scale2 = make_float2(scale, scale), center2 = make_float2(center, center);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (8 * u >= chunks) break;  // uniform
        uint32_t b0, b1;
        if constexpr (BITS == 4) {
          const uint32_t word = w[which][u][0];
          if (which == 0) {
            b0 = low_codes(word), b1 = high_codes(word);
          } else {
            const uint32_t mine = transpose_bytes(word, s), other = __shfl_xor_sync(~0u, mine, 1);
            b0 = c0 & 1 ? high_codes(other) : low_codes(mine);
            b1 = c0 & 1 ? high_codes(mine) : low_codes(other);
          }
        } else {
          b0 = which ? transpose_bytes(w[which][u][0], s) : w[which][u][0];
          b1 = which ? transpose_bytes(w[which][u][W - 1], s) : w[which][u][W - 1];
        }
        float y[8];
        decode4(y, b0 ^ 0x80808080u, scale2, center2);
        decode4(y + 4, b1 ^ 0x80808080u, scale2, center2);
        if (!live) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = 0.f;
        }
        if (in[u] && mine) store8<T>(rows[which] + 64 * u, y, a.vec);
      }
      rows[which] += which ? a.v.head : a.k.head;
    }
  }
}

// Reports segments that do not fit the rows there are (a start below zero, past the rows or below the one
// before it), of which nothing is moved; by the grid's warps together.
__device__ __forceinline__ void check_starts(const RowArgs& a, unsigned item, unsigned warps) {
  for (long long b = 32ll * item + (threadIdx.x & 31); b < a.n_seg; b += 32ll * warps) {
    const int first = a.start[b], end = a.start[b + 1];
    if (first < 0 || end < first || end > a.n_rows) atomicExch(a.c.error, 1);
  }
}

// One warp per group of slots and a.warp_heads heads of the segments. Segment b's groups have numbers
// from start[b] / 4 + 2b on: room for its rows / 4 + 2, and it has no more whatever its first slot.
template <class T, bool WRITE>
__global__ void __launch_bounds__(kCacheThreads, WRITE ? (sizeof(T) == 4 ? 4 : 5) : 5) segment_kernel(const __grid_constant__ RowArgs a) {
  __shared__ int8_t codes[WRITE ? kCacheThreads / 32 : 1][kMaxDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned item = blockIdx.x * (kCacheThreads / 32) + warp;  // fewer than 2^31
  const unsigned parts = (unsigned)(a.c.heads + a.warp_heads - 1) / a.warp_heads, group = item / parts;
  const int h0 = (int)(item - group * parts) * a.warp_heads, h1 = min(h0 + a.warp_heads, a.c.heads);
  check_starts(a, item, gridDim.x * (kCacheThreads / 32));
  if constexpr (!WRITE) {  // rows before the first segment and after the last that fit come back as zeros
    int lo = a.start[0], hi = a.start[a.n_seg];
    if (lo < 0) lo = a.start[last_at_most(a.n_seg, [&](int i) { return a.start[i] < 0; }) + 1];
    if (hi > a.n_rows) {
      const int b = last_at_most(a.n_seg, [&](int i) { return a.start[i] < a.n_rows; });
      if (a.start[b + 1] > a.n_rows) hi = a.start[b];
    }
    lo = max(0, min(lo, a.n_rows)), hi = max(lo, min(hi, a.n_rows));
    for (long long e = item; e < (long long)(lo + a.n_rows - hi) * a.c.heads; e += (long long)gridDim.x * (kCacheThreads / 32)) {
      const int i = (int)(e / a.c.heads);
      read_row<T>(a, i < lo ? i : hi + i - lo, (int)(e % a.c.heads), RowPlace{0, -1});
    }
  }
  const int b = last_at_most(a.n_seg, [&](int i) { return (a.start[i] >> 2) + 2ll * i <= (long long)group; });
  const int first = a.start[b], rows = a.start[b + 1] - first;
  const long long at = (long long)group - ((first >> 2) + 2ll * b);
  if (rows <= 0 || first < 0 || rows > a.n_rows - first || at < 0) return;
  const int offset = a.pos0[b] >= 0 ? slot_of(a.c, a.pos0[b]) & 3 : 0;  // of the segment's first row in its group
  // lane 8s + c asks for the row of the group's slot s
  const int s = lane >> 3;
  const long long i = 4 * at - offset + s;
  const bool mine = i >= 0 && i < rows;
  const unsigned any = __ballot_sync(~0u, mine);
  if (!any) return;
  const int row = mine ? first + (int)i : first;
  const RowPlace p = place<WRITE>(a, b, first, rows, mine ? row : first);
  const int slot = mine ? p.slot : -1;
  const unsigned live = __ballot_sync(~0u, slot >= 0);
  const int slot0 = live ? __shfl_sync(~0u, slot, __ffs(live) - 1) & ~3 : 0;
  if (__all_sync(~0u, slot < 0 || slot == slot0 + s)) {
    if (WRITE && !live) return;
    if (a.c.bits == 4) {
      if constexpr (WRITE) write_group<T, 4>(a, row, slot >= 0, h0, h1, p.session, slot0);
      else read_group<T, 4>(a, row, mine, slot >= 0, h0, h1, p.session, slot0);
    } else {
      if constexpr (WRITE) write_group<T, 8>(a, row, slot >= 0, h0, h1, p.session, slot0);
      else read_group<T, 8>(a, row, mine, slot >= 0, h0, h1, p.session, slot0);
    }
    return;
  }
  for (int r = 0; r < 4; ++r) {
    if (!(any >> (8 * r) & 1)) continue;
    const RowPlace q{p.session, __shfl_sync(~0u, slot, 8 * r)};
    const int at_row = __shfl_sync(~0u, row, 8 * r);
    for (int h = h0; h < h1; ++h) {
      if constexpr (WRITE) {
        if (q.slot >= 0) write_row<T>(a, at_row, h, q, codes[warp]);
      } else {
        read_row<T>(a, at_row, h, q);
      }
    }
  }
}

// One warp per (row, head): rows that are a segment of their own.
template <class T, bool WRITE>
__global__ void __launch_bounds__(kCacheThreads) single_kernel(const __grid_constant__ RowArgs a) {
  __shared__ int8_t codes[WRITE ? kCacheThreads / 32 : 1][kMaxDim];
  const int warp = threadIdx.x >> 5;
  const unsigned item = blockIdx.x * (kCacheThreads / 32) + warp;  // fewer than 2^31
  const int row = (int)(item / a.c.heads), head = (int)(item - (unsigned)row * a.c.heads);
  if (a.start) check_starts(a, item, gridDim.x * (kCacheThreads / 32));
  if (row >= a.n_rows) return;
  RowPlace w{0, -1};
  if (!a.start) {
    w = place<WRITE>(a, row, row, 1, row);
  } else if (a.n_seg > 0 && row >= a.start[0] && row < a.start[a.n_seg]) {
    // where an even spread has the row (decode steps), else by search
    int b = min((int)((float)row * a.spread), a.n_seg - 1);
    if (a.start[b] > row || a.start[b + 1] <= row) b = last_at_most(a.n_seg, [&](int i) { return a.start[i] <= row; });
    const int first = a.start[b], rows = a.start[b + 1] - first;
    if (first >= 0 && row - first < rows && rows <= a.n_rows - first) w = place<WRITE>(a, b, first, rows, row);
  }
  if constexpr (WRITE) {
    if (w.slot >= 0) write_row<T>(a, row, head, w, codes[warp]);
  } else {
    read_row<T>(a, row, head, w);
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
  bool own = false;          // whether the memory is the library's
  int* arrived = nullptr;
  float* partial = nullptr;
  int n_sm = 0;
};

namespace mc {
namespace kv {

// Lets a kernel use `bytes` of dynamic shared memory on the current device, once for each. 48 KB need no
// leave, but what the kernels have besides (at most 8 KB) counts too.
static cudaError_t allow_smem(const void* f, int device, int bytes) {
  if (bytes <= 40 * 1024) return cudaSuccess;
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  std::lock_guard<std::mutex> lock(mu);
  if (done.count({f, device})) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.insert({f, device});
  return e;
}

static bool rows_ok(const mc_rows* r) { return r && r->data; }
static Rows rows_of(const mc_rows* r) { return Rows{r->data, (long long)r->row_stride, (long long)r->head_stride}; }

template <bool SEGMENTS, class T>
static void (*row_kernel_of(bool write))(RowArgs) {
  if constexpr (SEGMENTS) return write ? segment_kernel<T, true> : segment_kernel<T, false>;
  else return write ? single_kernel<T, true> : single_kernel<T, false>;
}
template <bool SEGMENTS>
static void (*row_variant(int dtype, bool write))(RowArgs) {
  return dtype == kF32   ? row_kernel_of<SEGMENTS, float>(write)
         : dtype == kF16 ? row_kernel_of<SEGMENTS, __half>(write)
                         : row_kernel_of<SEGMENTS, __nv_bfloat16>(write);
}

static int row_launch(const char* name, bool write, mc_kv* kv, const mc_rows* k, const mc_rows* v, int dtype, int n_rows,
                      const int32_t* start, const int32_t* sess, const int32_t* pos0, const int32_t* lens, int n_seg,
                      cudaStream_t stream) {
  clear_error();
  if (!kv || !k || !v) return set_error(kInvalidArgument, std::string(name) + ": null argument");
  if (dtype < kF32 || dtype > kBF16) return set_error(kInvalidArgument, std::string(name) + ": unknown dtype");
  if (n_rows < 0 || n_seg < 0 || (!start && n_rows != n_seg))
    return set_error(kInvalidArgument, std::string(name) + ": negative counts, or rows without row_start that are not one per segment");
  if (n_rows == 0 || (write && n_seg == 0)) return kOk;
  if (!k->data || !v->data || (n_seg > 0 && (!pos0 || (!write && !lens)))) return set_error(kInvalidArgument, std::string(name) + ": null argument");
  DeviceRestore restore_device;
  MC_CUDA(cudaSetDevice(kv->device));
  const int size = dtype == kF32 ? 4 : 2;
  auto aligned = [&](const mc_rows* r) {  // for the 16-byte accesses of eight elements
    return reinterpret_cast<uintptr_t>(r->data) % 16 == 0 && r->row_stride * size % 16 == 0 && r->head_stride * size % 16 == 0;
  };
  // Groups of slots pay once segments have more than a row: write and read of 8192 segments, 8 heads of 64,
  // in us by groups and row by row: 1 row a segment 102, 98; 1.5 rows 117, 182; 5 rows 172, 516.
  // (rows of no segment at all are read, as zeros, row by row)
  const bool groups = start && n_rows > n_seg && n_seg > 0;
  long long warps = (long long)n_rows * kv->c.heads;
  int warp_heads = 1;
  if (groups) {
    // heads a warp goes through with one group's addresses: as many as leave every SM its 32 warps twice
    const long long n = n_rows / 4 + 2ll * n_seg;
    while (2 * warp_heads <= kv->c.heads && warp_heads < (write ? 2 : 4) && n * kv->c.heads / (2 * warp_heads) >= 128ll * kv->n_sm) warp_heads *= 2;
    warps = n * ((kv->c.heads + warp_heads - 1) / warp_heads);
  }
  const RowArgs a{kv->c, rows_of(k), rows_of(v), n_rows, n_seg, start, sess, pos0, lens, aligned(k) && aligned(v), warp_heads,
                  (float)n_seg / (float)n_rows};
  const long long blocks = (warps + kCacheThreads / 32 - 1) / (kCacheThreads / 32);
  if (warps > INT_MAX) return set_error(kInvalidArgument, std::string(name) + ": too many rows");
  auto f = groups ? row_variant<true>(dtype, write) : row_variant<false>(dtype, write);
  f<<<(unsigned)blocks, kCacheThreads, 0, stream>>>(a);
  MC_CUDA(cudaGetLastError());
  return kOk;
}

}  // namespace kv
}  // namespace mc

namespace mc {
namespace kv {

// The cache of a spec, without its memory, and the bytes it needs: `head` of workspace, then the regions.
static int layout(const char* name, const mc_kv_spec* spec, Cache* c, size_t* head, size_t* bytes) {
  const std::string who = std::string(name) + ": ";
  if (!spec) return set_error(kInvalidArgument, who + "null argument");
  const mc_kv_spec& s = *spec;
  if (s.sessions < 1 || s.heads < 1 || s.slots < 1)
    return set_error(kInvalidArgument, who + "sessions, heads and slots must be positive");
  if (s.head_dim < 16 || s.head_dim > kMaxDim || s.head_dim % 16)
    return set_error(kInvalidArgument, who + "head_dim must be a multiple of 16 from 16 to 128");
  if (s.bits != 4 && s.bits != 8) return set_error(kInvalidArgument, who + "bits must be 4 or 8");
  if (s.sinks < 0 || s.sinks >= s.slots) return set_error(kInvalidArgument, who + "sinks must be in [0, slots)");
  if (s.slots > (1 << 30)) return set_error(kInvalidArgument, who + "slots above 2^30");
  *c = Cache{};
  c->sessions = s.sessions;
  c->heads = s.heads;
  c->dim = s.head_dim;
  c->bits = s.bits;
  c->slots = s.slots;
  c->sinks = s.sinks;
  c->ring = s.slots - s.sinks;
  c->cap = (s.slots + 63) / 64 * 64;
  c->cb = s.head_dim * s.bits / 8;
  c->region = (long long)(c->cap / kBlockSlots) * block_bytes(c->cb);
  // the workspace of mc_kv_attend_dev is part of the cache, so that no call allocates
  *head = 256 + kMaxPartials * (sizeof(int) + kAttendRows * (2 + s.head_dim) * sizeof(float));
  const double need = (double)c->region * s.sessions * s.heads + (double)*head;
  if (need > 9e18) return set_error(kOutOfMemory, who + "a cache of " + std::to_string(need) + " bytes");
  *bytes = (size_t)c->region * s.sessions * s.heads + *head;
  return kOk;
}

}  // namespace kv
}  // namespace mc

extern "C" int mc_kv_bytes(const mc_kv_spec* spec, size_t* bytes) {
  using namespace mc;
  clear_error();
  kv::Cache c;
  size_t head = 0;
  if (!bytes) return set_error(kInvalidArgument, "mc_kv_bytes: null argument");
  return kv::layout("mc_kv_bytes", spec, &c, &head, bytes);
}

extern "C" int mc_kv_open(int device, const mc_kv_spec* spec, void* memory, void* stream, mc_kv** out) {
  using namespace mc;
  clear_error();
  if (!out) return set_error(kInvalidArgument, "mc_kv_open: null argument");
  *out = nullptr;
  kv::Cache c;
  size_t head = 0, bytes = 0;
  const int st = kv::layout("mc_kv_open", spec, &c, &head, &bytes);
  if (st != kOk) return st;
  if (reinterpret_cast<uintptr_t>(memory) % 256) return set_error(kInvalidArgument, "mc_kv_open: memory must be 256-byte aligned");
  DeviceRestore restore_device;
  MC_CUDA(cudaSetDevice(device));
  int n_sm = 0;
  MC_CUDA(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, device));
  mc_kv* kv = new (std::nothrow) mc_kv;
  if (!kv) return set_error(kOutOfMemory, "mc_kv_open: out of host memory");
  void* mem = memory;
  if (!mem && cudaMalloc(&mem, bytes) != cudaSuccess) {
    (void)cudaGetLastError();
    delete kv;
    return set_error(kOutOfMemory, "mc_kv_open: no room for a cache of " + std::to_string(bytes) + " bytes");
  }
  const cudaError_t e = cudaMemsetAsync(mem, 0, bytes, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) {
    if (!memory) cudaFree(mem);
    delete kv;
    return set_error(kCudaError, std::string("mc_kv_open: cudaMemsetAsync: ") + cudaGetErrorString(e));
  }
  c.error = static_cast<int*>(mem);
  c.base = static_cast<uint8_t*>(mem) + head;  // a multiple of 256
  kv->device = device;
  kv->c = c;
  kv->mem = mem;
  kv->own = !memory;
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
  cudaError_t e = cudaSuccess;
  if (kv->own) {
    DeviceRestore restore_device;
    cudaSetDevice(kv->device);
    e = cudaFree(kv->mem);  // waits for the device's work
  }
  delete kv;
  if (e != cudaSuccess) return set_error(kCudaError, std::string("mc_kv_close: ") + cudaGetErrorString(e));
  return kOk;
}

namespace mc {
namespace kv {

// Reads and clears the current device's error word of this unit's kernels, whose work is done. While it is set, waits
// that take long give up early.
static int take_timeout() {
  int code = 0;
  MC_CUDA(cudaMemcpyFromSymbol(&code, g_device_error, sizeof(int)));
  if (!code) return kOk;
  const int zero = 0;
  MC_CUDA(cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int)));
  MC_CUDA(cudaDeviceSynchronize());
  return set_error(kDeviceTimeout, "device wait gave up (code " + std::to_string(code) + "); the kernel returned without finishing its work");
}

// As the engine's, for this unit's error word, which stays set.
__global__ void selftest_wait_kernel() {
  __shared__ uint64_t bar;
  if (threadIdx.x != 0) return;
  mbar_init(&bar, 1);
  fence_barrier_init();
  mbar_wait(&bar, 0, kErrWaitFull);  // phase 0 never completes
}

}  // namespace kv
}  // namespace mc

extern "C" int mc_selftest_kv_wait_timeout(int device) {
  using namespace mc;
  clear_error();
  DeviceRestore restore_device;
  MC_CUDA(cudaSetDevice(device));
  kv::selftest_wait_kernel<<<1, 32>>>();
  MC_CUDA(cudaGetLastError());
  MC_CUDA(cudaDeviceSynchronize());
  return kOk;
}

extern "C" int mc_kv_error(mc_kv* kv) {
  using namespace mc;
  clear_error();
  if (!kv) return set_error(kInvalidArgument, "mc_kv_error: null cache");
  DeviceRestore restore_device;
  MC_CUDA(cudaSetDevice(kv->device));
  MC_CUDA(cudaDeviceSynchronize());
  const int st = kv::take_timeout();
  if (st != kOk) return st;
  int code = 0;
  MC_CUDA(cudaMemcpy(&code, kv->c.error, sizeof(int), cudaMemcpyDeviceToHost));
  if (!code) return kOk;
  MC_CUDA(cudaMemset(kv->c.error, 0, sizeof(int)));
  MC_CUDA(cudaDeviceSynchronize());  // before what other streams do next
  return set_error(kInvalidArgument, "mc_kv: a session, a position or a segment was out of range; its rows were skipped");
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

namespace mc {
namespace kv {

// CTAs that an item's visible slots are split over (0: none, a warp to an item), for `warps` resident
// warps. A warp costs about as much as 160 slots on top of those it reads (start, query planes, joining);
// up to three waves count whole. Both sides measured, us, 8 heads of 64 in 8 bits, 1024 slots: 16 sessions
// 29 with a warp to an item, 12 split; 64: 31, 27; 200: 41, 46; 300 (one item more than a wave): 79, 64;
// 256 slots: 64 sessions 12, 10; 200: 17, 24.
static int attend_pieces(long long items, long long slots, long long warps) {
  auto cost = [&](long long n, double read) {
    const double waves = (double)n / warps;
    return (waves <= 3 ? std::ceil(waves) : waves) * (160 + read);
  };
  int best = 0;
  double least = cost(items, (double)slots);
  const long long most = std::min<long long>({kMaxPieces, kMaxPartials / items, (slots + 127) / 128});
  for (int p = 1; p <= std::max(1ll, most); ++p) {
    const double c = cost(items * kAttendWarps * p, (double)slots / (kAttendWarps * p));
    if (c < least) best = p, least = c;
  }
  return best;
}

}  // namespace kv
}  // namespace mc

extern "C" int mc_kv_attend_dev(mc_kv* kv, const mc_rows* q, const mc_rows* out, int dtype, int q_heads,
                                const int32_t* sessions, const int32_t* lens, int n, int window, float scale,
                                void* stream) {
  using namespace mc;
  using namespace mc::kv;
  clear_error();
  if (!kv || !q || !out) return set_error(kInvalidArgument, "mc_kv_attend_dev: null argument");
  if (dtype < kF32 || dtype > kBF16) return set_error(kInvalidArgument, "mc_kv_attend_dev: unknown dtype");
  if (n < 0 || window < 0) return set_error(kInvalidArgument, "mc_kv_attend_dev: n and window must not be negative");
  if (q_heads < 1 || q_heads % kv->c.heads)
    return set_error(kInvalidArgument, "mc_kv_attend_dev: q_heads must be a multiple of the cache's heads");
  if (!(scale > 0.f) || !std::isfinite(scale)) return set_error(kInvalidArgument, "mc_kv_attend_dev: scale must be positive");
  if (n == 0) return kOk;
  if (!q->data || !out->data || !lens) return set_error(kInvalidArgument, "mc_kv_attend_dev: null argument");
  DeviceRestore restore_device;
  MC_CUDA(cudaSetDevice(kv->device));
  const Cache& c = kv->c;
  const int group = q_heads / c.heads, row_groups = (group + kAttendRows - 1) / kAttendRows;
  const long long items = (long long)n * c.heads * row_groups;
  const AttendVariant f = attend_variant(c.bits, c.dim, dtype == kF32 ? 3 : 2, group);
  const long long ctas = (long long)f.ctas * kv->n_sm;
  const int pieces = attend_pieces(items, window > 0 ? std::min<long long>(c.slots, (long long)window + c.sinks) : c.slots, ctas * kAttendWarps);
  const int size = dtype == kF32 ? 4 : 2;
  auto aligned = [&](const mc_rows* r) {
    return reinterpret_cast<uintptr_t>(r->data) % 16 == 0 && r->row_stride * size % 16 == 0 && r->head_stride * size % 16 == 0;
  };
  const AttendArgs a{c, rows_of(q), rows_of(out), n, q_heads, group, row_groups, window, dtype, aligned(q) && aligned(out),
                     pieces, sessions, lens, scale * 1.4426950408889634f, kv->partial, kv->arrived};
  if (items > INT_MAX) return set_error(kInvalidArgument, "mc_kv_attend_dev: too many rows");
  const long long blocks = pieces ? items : std::min<long long>((items + kAttendWarps - 1) / kAttendWarps, ctas);
  MC_CUDA(allow_smem(reinterpret_cast<const void*>(f.f), kv->device, f.smem));
  f.f<<<dim3((unsigned)blocks, std::max(1, pieces)), kAttendWarps * 32, f.smem, static_cast<cudaStream_t>(stream)>>>(a);
  MC_CUDA(cudaGetLastError());
  return kOk;
}
