// The 8-bit form of activations and weights: e4m3 values, every 32 of a row under one power-of-two scale, which is the form that the
// matrix instructions with scales read.
//
//   data    e4m3 [rows, cols], contiguous; cols a multiple of 32
//   scales  [ceil(cols / 128), rows, 4]: byte (t, r, q) belongs to columns 128 t + 32 q .. + 31 of row r and stands for 2^(byte - 127); bytes past the last
//           column are 0.  So the scales that a tile of rows needs for 128 of contraction lie side by side, four bytes a row.
//
// A block's scale is the smallest 2^e (e >= -127) for which its largest |value| / 2^e is at most 448, the largest e4m3 value: nothing saturates, and
// dividing by it is exact.  Values of a block whose largest is 2^-118 or more are off by at most 2^-4 of themselves, or by 2^-10 * 2^e where they lie under
// 2^-6 * 2^e.  A block that holds an infinity or a NaN becomes NaN as a whole (scale byte 255): an overflow shows in whatever is made of it.
#pragma once
#include "common.h"

namespace pico {
namespace {

constexpr int kBlock = 32, kGroup = 128;   // values under one scale; columns whose four scales lie side by side

template <int kControl>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {   // (0 from lanes that are off)
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kControl, 0xf, 0xf, true));
}
// the largest of L neighbouring lanes (4 or 8), in all of them
template <int L>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  static_assert(L == 4 || L == 8);
  v = max(v, dpp<0xb1>(v));    // lane ^ 1
  v = max(v, dpp<0x4e>(v));    // lane ^ 2
  if constexpr (L == 8) v = max(v, dpp<0x141>(v));   // 7 - lane of eight
  return v;
}
// The scale of a block whose largest |value| has these bits.  An infinity's bits and a NaN's are larger than any finite value's.  448 is 1.75 * 2^8: a
// mantissa over 1.75 takes the next power of two (what is added, a quarter of a mantissa less its last bit, carries then).
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest) {
  const int e = static_cast<int>((largest + 0x1fffffu) >> 23) - 8;
  return largest >= 0x7f800000u ? 255u : static_cast<uint32_t>(max(e, 0));
}
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fc00000u : (254u - byte) << 23); }

// V values of a block that 32 / V neighbouring lanes hold, as codes, and the block's scale byte.  All lanes of a block have to be on.
template <int V>
struct Codes {
  uint32_t word[V / 4];
  uint32_t scale;
};
template <int V>
__device__ __forceinline__ Codes<V> encode(const float (&v)[V]) {
  uint32_t largest = 0;
#pragma unroll
  for (int e = 0; e < V; ++e) largest = max(largest, __float_as_uint(v[e]) & 0x7fffffffu);
  Codes<V> c;
  c.scale = scale_byte(lanes_max<kBlock / V>(largest));
  const float inverse = inverse_scale(c.scale);
#pragma unroll
  for (int w = 0; w < V / 4; ++w) {
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * w] * inverse, v[4 * w + 1] * inverse, 0, false);
    c.word[w] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * w + 2] * inverse, v[4 * w + 3] * inverse, low, true));
  }
  return c;
}
// The four scales of the 128 columns that 128 / V lanes hold, in all of them; `lane` counts from a group's first on.
template <int V>
__device__ __forceinline__ uint32_t four_scales(uint32_t byte, int lane) {
  uint32_t v = byte << (lane / (kBlock / V) % 4 * 8);
  if constexpr (V == 8) {
    v |= dpp<0x124>(v);   // 4 lanes round 16
    v |= dpp<0x128>(v);   // 8 lanes round 16
  } else {
    v |= dpp<0x128>(v);
    v |= __shfl_xor(v, 16, kWave);
  }
  return v;
}
template <int V>
__device__ __forceinline__ void decode(const uint32_t (&word)[V / 4], uint32_t byte, float (&v)[V]) {
  const int e = static_cast<int>(byte) - 127;
#pragma unroll
  for (int w = 0; w < V / 4; ++w) {
    const int codes = byte == 255u ? 0x7f7f7f7f : static_cast<int>(word[w]);   // (NaN, whatever codes a block of it has)
    const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false), high = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
    v[4 * w] = __builtin_amdgcn_ldexpf(low[0], e);
    v[4 * w + 1] = __builtin_amdgcn_ldexpf(low[1], e);
    v[4 * w + 2] = __builtin_amdgcn_ldexpf(high[0], e);
    v[4 * w + 3] = __builtin_amdgcn_ldexpf(high[1], e);
  }
}
// V codes at p, V bytes apart from any other thread's
template <int V>
__device__ __forceinline__ void store_codes(uint8_t* p, const uint32_t (&word)[V / 4]) {
  if constexpr (V == 8) *reinterpret_cast<u32x2*>(p) = u32x2{word[0], word[1]};
  else *reinterpret_cast<uint32_t*>(p) = word[0];
}
template <int V>
__device__ __forceinline__ void load_codes(const uint8_t* p, uint32_t (&word)[V / 4]) {
  if constexpr (V == 8) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    word[0] = v[0];
    word[1] = v[1];
  } else {
    word[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// What an entry point checks of one operand; PICO_OK or the failure.
inline int check_mx8(const char* fn, const char* what, const pico_mx8* t) {
  if (!t || !t->data || !t->scales) return fail(PICO_ERR_NULL, "%s: %s needs its data and its scales", fn, what);
  if (!aligned16(t->data) || (reinterpret_cast<uintptr_t>(t->scales) & 3u))
    return fail(PICO_ERR_ALIGN, "%s: %s must have 16-byte aligned data and 4-byte aligned scales", fn, what);
  return PICO_OK;
}
// A launch has under 2^32 threads, in workgroups of 256, and up to 32 lanes walk a group of 128 columns: 2^24 - 1 workgroups of 8 groups.
constexpr int64_t kMostGroups = (int64_t{1} << 27) - 8;
inline int check_mx8_shape(const char* fn, int64_t rows, int64_t cols) {
  if (rows < 0 || cols < kBlock || cols % kBlock != 0 || cols > (int64_t{1} << 30) || rows > kMostGroups / ((cols + kGroup - 1) / kGroup))
    return fail(PICO_ERR_SHAPE, "%s: rows=%lld cols=%lld (cols must be a multiple of %d, rows times groups of %d columns at most 2^27 - 8)", fn, (long long)rows, (long long)cols,
                kBlock, kGroup);
  return PICO_OK;
}

}  // namespace
}  // namespace pico
