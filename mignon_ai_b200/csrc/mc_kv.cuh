// The quantised key/value cache: its layout in memory, its quantiser and the positions it holds.
//
// A cache has `slots` places per session. Position p of a session lies at slot p while p < sinks
// (the first positions are never overwritten) and at sinks + (p - sinks) % (slots - sinks) after
// that: a ring behind pinned places. Every (session, head) owns one region of cap / 32 blocks (cap =
// slots rounded up to 64), a block being all there is of 32 slots, so that one copy fetches its keys or its values:
//
//   keys' codes | keys' scales and centers | values' codes | values' scales and centers
//
// Codes of consecutive slots are interleaved, so that a 16-byte load gives a lane words of several of
// them, in the order in which the operands of an 8-bit m16n8k32 MMA want them (cb code bytes per slot):
//
//   keys    four slots at a time: the group's 16-byte unit of word w holds that word of its slots,
//           one after the other. 8 bits: word w is dimensions 4w..4w+3. 4 bits: byte b of word w is
//           dimensions 8w + b (low) and 8w + 4 + b (high). The contraction runs along the dimensions:
//           a word is an operand.
//   values  eight slots at a time (two groups u): word n * 2ni + u * ni + i is dimension 8i + n
//           (8 bits, ni = dim / 8), or 16i + n (low) and 16i + 8 + n (high) (4 bits, ni = dim / 16), of
//           the group's four slots, slot s in byte s % 4. The contraction runs along the slots.
//
// Within a group or pair the 16-byte units are permuted (key_unit, value_word) such that the eight
// lanes that load together, two groups by four units of keys, or two n by the four pairs of
// a block of values, meet eight different shared-memory banks of 16 bytes.
//
// A slot's scale and center are one word: scale in the low half, center in the high (bfloat16).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mc_sm100.cuh"

namespace mc {
namespace kv {

enum Dtype : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

constexpr int kMaxDim = 128;

// Rows [row][head][dim] with element strides; the dimensions of a row are contiguous.
struct Rows {
  void* p;
  long long row, head;
};

struct Cache {
  int sessions, heads, dim, bits, slots, sinks, ring, cap;
  int cb;              // code bytes of one slot's keys (and of its values): dim * bits / 8
  long long region;    // bytes of one (session, head)
  uint8_t* base;       // [session][head] regions
  int* error;          // set when an index was out of range (that access is skipped)
};

__device__ __forceinline__ uint8_t* region_of(const Cache& c, int session, int head) {
  return c.base + ((long long)session * c.heads + head) * c.region;
}
constexpr int kBlockSlots = 32;
__host__ __device__ constexpr int block_bytes(int cb) { return kBlockSlots * (2 * cb + 8); }

// The 16-byte unit of a group of four slots that holds word w of their keys (g: the group's number).
__host__ __device__ __forceinline__ constexpr int key_unit(int w, int g, int cb, int bits) {
  return bits == 8 ? w ^ (g & 1) : cb % 32 == 0 ? w ^ ((g & 1) << 2) : w;
}
// The word of a pair of groups that holds value word (n, i) of group g; ni words per n and group.
__host__ __device__ __forceinline__ constexpr int value_swizzle(int n, int pair, int ni) {
  return ni == 2   ? 2 * (pair & 3)
         : ni == 4 ? (pair & 1) | ((pair & 2) << 1)
         : ni == 8 ? pair & 3
         : ni == 16 ? (pair & 3) | ((n & 1) << 2)
                    : 0;
}
__host__ __device__ __forceinline__ constexpr int value_word(int n, int i, int g, int ni) {
  const int at = (2 * n + (g & 1)) * ni + i;
  return at ^ (value_swizzle(n, g >> 1, ni) << 2);
}

// The words of slot s's group of four keys, those of its pair of groups of values, and the words of
// scale and center from slot s on, in a region.
__device__ __forceinline__ uint32_t* keys_of(const Cache& c, uint8_t* region, int s) {
  return reinterpret_cast<uint32_t*>(region + (long long)(s >> 5) * block_bytes(c.cb)) + ((s & 31) >> 2) * c.cb;
}
__device__ __forceinline__ uint32_t* values_of(const Cache& c, uint8_t* region, int s) {
  return reinterpret_cast<uint32_t*>(region + (long long)(s >> 5) * block_bytes(c.cb) + kBlockSlots * (c.cb + 4)) +
         ((s & 31) >> 3) * 2 * c.cb;
}
__device__ __forceinline__ uint32_t* params_of(const Cache& c, uint8_t* region, int s, bool values) {
  return reinterpret_cast<uint32_t*>(region + (long long)(s >> 5) * block_bytes(c.cb) + kBlockSlots * c.cb +
                                     (values ? kBlockSlots * (c.cb + 4) : 0)) +
         (s & 31);
}

__device__ __forceinline__ int slot_of(const Cache& c, int pos) {
  return pos < c.sinks ? pos : c.sinks + (pos - c.sinks) % c.ring;
}

// Whether a session of `len` positions still holds position pos.
__device__ __forceinline__ bool is_held(const Cache& c, int pos, int len) {
  return pos >= 0 && pos < len && (pos < c.sinks || pos >= len - c.ring);
}

template <class T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

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
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2_down(float2 a, float b) {  // rounded down
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tadd.rm.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b));
  return d;
}

// The quantiser of one row x of one head, from its extremes:
//   center = bf16(hi / 2 + lo / 2), half = max(hi - center, center - lo),
//   scale  = half / (15 or 127), rounded up to bfloat16 so that the codes reach both extremes
//            (0 where half is below 2^-100: the row then reads back as its center),
//   m      = the odd integer of [-15, 15] (4 bits) or the integer of [-127, 127] (8 bits) next to
//            (x - center) / scale.
// The row reads back as center + scale * m. The products scale * m are exact in float32 (8 by at
// most 8 bits), so a fused and a separate multiply-add give the same value. A row that is not all
// finite, or whose center or scale leaves bfloat16's range, reads back as NaN (scale and
// center NaN).
struct Quant {
  float scale, center, inv;
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// hi and lo by max_nan and min_nan: either is not finite once an element is not.
__device__ __forceinline__ Quant quant_of(float hi, float lo, int bits) {
  Quant q;
  q.center = __bfloat162float(__float2bfloat16_rn(__fadd_rn(__fmul_rn(0.5f, hi), __fmul_rn(0.5f, lo))));
  const float half = fmaxf(__fsub_rn(hi, q.center), __fsub_rn(q.center, lo));
  const float step = __fmul_rn(half, bits == 4 ? 1.0f / 15.0f : 1.0f / 127.0f);
  q.scale = __uint_as_float((__float_as_uint(step) + 0xFFFFu) & 0xFFFF0000u);
  if (half < 0x1p-100f) q.scale = 0.f;
  q.inv = q.scale > 0.f ? __fdiv_rn(1.0f, q.scale) : 0.f;
  if (!(fabsf(hi) < INFINITY) || !(fabsf(lo) < INFINITY) || !(fabsf(q.center) < INFINITY) || !(q.scale < INFINITY)) {
    q.scale = q.center = __int_as_float(0x7FFF0000);
    q.inv = 0.f;
  }
  return q;
}

__device__ __forceinline__ uint32_t param_word(const Quant& q) {
  return (__float_as_uint(q.scale) >> 16) | (__float_as_uint(q.center) & 0xFFFF0000u);
}
__device__ __forceinline__ float param_scale(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float param_center(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// The code of x in the low bits of a word: 4 bits: c = floor(t / 2) of t = (x - center) / scale, m = 2c + 1
// (a nibble in two's complement); 8 bits: m = t rounded to the nearest integer, ties to even. |t| stays below 16
// or 127.5, so adding 1.5 * 2^24 rounded down (whose float spacing is 2), or 1.5 * 2^23, leaves them there.
__device__ __forceinline__ uint32_t code_bits(const Quant& q, float x, int bits) {
  const float t = __fmul_rn(__fsub_rn(x, q.center), q.inv);
  return __float_as_uint(bits == 4 ? __fadd_rd(t, 25165824.0f) : __fadd_rn(t, 12582912.0f));
}

// A word of nibbles c (two's complement) as bytes 16c + 8 = 8m: the low and the high nibbles.
__device__ __forceinline__ uint32_t low_codes(uint32_t w) { return ((w << 4) & 0xF0F0F0F0u) | 0x08080808u; }
__device__ __forceinline__ uint32_t high_codes(uint32_t w) { return (w & 0xF0F0F0F0u) | 0x08080808u; }

// Eight codes at once (as code_bits).
template <int BITS>
__device__ __forceinline__ void code_bits8(const Quant& q, const float (&x)[8], uint32_t (&code)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 d = add2(make_float2(x[e], x[e + 1]), make_float2(-q.center, -q.center));
    const float2 t = mul2(d, q.inv);
    if constexpr (BITS == 4) {
      const float2 y = add2_down(t, 25165824.0f);
      code[e] = __float_as_uint(y.x);
      code[e + 1] = __float_as_uint(y.y);
    } else {  // one by one: a packed product and sum, both to nearest, came out fused, rounded once
      code[e] = __float_as_uint(__fadd_rn(t.x, 12582912.0f));
      code[e + 1] = __float_as_uint(__fadd_rn(t.y, 12582912.0f));
    }
  }
}

// The last i of [0, n) for which `at_most` holds, by a whole warp with 32 probes a round (0 if it
// holds nowhere; it must not hold again after it failed).
template <class F>
__device__ __forceinline__ int last_at_most(int n, F at_most) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const bool below = at < hi && (lane == 0 || at_most(at));
    lo += (31 - __clz(__ballot_sync(~0u, below))) * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

}  // namespace kv
}  // namespace mc
