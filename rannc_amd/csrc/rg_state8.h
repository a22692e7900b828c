// Device side of optimizer states in 8 bits, shared by the step and by the two conversions.
//
// A tensor's state is cut into blocks of 256 consecutive elements; a block keeps its largest magnitude s (fp32) and, for
// every element x, the e4m3 number that y = 256 x / s is rounded to.  256 is a power of two, so the element that sets s
// is stored and read back exactly and the factor s / 256 loses no bit; the numbers between it and e4m3's largest (448)
// stay unused, which costs no precision (relative steps are the same in every octave) and under one of its 18 octaves of range.
// A second moment is stored as its square root r: half the range in the exponent, and the step needs r anyway.
#pragma once

#include "rg_device.h"

namespace rg {
namespace {

constexpr uint32_t kState8TinyBits = (127u - 100u) << 23;   // 2^-100: below it 256 / s would come near overflow
constexpr float kState8MinRoot = 0.001953125f;              // 2^-9, e4m3's smallest number

// The additive recurrence that dithers a step's rounding: fractions 1/g, 1/g^2, 1/g^3 (g the real root of x^4 = x + 1) in
// 32 bits, one for the element's place in its tensor and one per moment for the step count.  Rounding with such a number
// instead of 1/2 leaves the first moment and the root right on average each time: beta2 = 0.999 moves a root by less than 0.1 % a
// step, e4m3's neighbours are 6-12 % apart, and a root rounded to nearest would stay where it is until a gradient of eight
// times its size came along, following nothing but its block's scale meanwhile.
// Over a run the second moment is not right on average: the next step squares the root, so a rounding's variance - the root's
// movement times the neighbours' distance q - is added to it and forgotten at beta2's rate.  It ends up too large by the factor
// 1 + q / (2 r) D, D = E|g^2 / v - 1| (0.97 for normal gradients, at most 2), and a root is off by sqrt(q / (4 r) D) rms.  For
// 1/16 <= q / r <= 1/8 and normal gradients that is 3-6 % and 12-17 %; over 4,000 steps at beta2 = 0.999 they came out as 4.4 % and 15.3 %.
constexpr uint32_t kDitherPlace = 0xD1B54A33u, kDitherFirst = 0xABC98389u, kDitherRoot = 0x8CB92BA7u;

__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The largest of two numbers per lane, both at once: lanes 0-31 get the largest `a`, lanes 32-63 the largest `b` (all 64
// lanes active).  The halves trade places (a's upper for b's lower), then the two rows of 16 lanes of each half, then
// rotations within a row: 9 instructions, where two reductions of 64 lanes one after the other take 16 and more.  On magnitudes'
// bits the order is that of the numbers with infinity above them and NaN above that, so neither is lost on the way.
template <int N> __device__ __forceinline__ uint32_t max_row_ror(uint32_t x) {
  const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + N, 0xf, 0xf, true);
  return x > y ? x : y;
}
__device__ __forceinline__ uint32_t half_max(uint32_t a, uint32_t b) {
  const u32x2 halves = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(a, b, false, false));
  uint32_t x = halves.x > halves.y ? halves.x : halves.y;
  const u32x2 rows = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(x, x, false, false));
  x = rows.x > rows.y ? rows.x : rows.y;
  x = max_row_ror<1>(x);
  x = max_row_ror<2>(x);
  x = max_row_ror<4>(x);
  return max_row_ror<8>(x);
}
__device__ __forceinline__ float read_lane_f32(float x, int lane) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), lane));
}

// What a block stores as its scale, and the factor that takes its elements to e4m3's range (inv == 0: every code of the
// block is zero).  `max_bits` may belong to elements that are carried times 1 / shift, a power of two.
struct BlockScale {
  float s, inv;
};
__device__ __forceinline__ BlockScale block_scale(uint32_t max_bits, float shift) {
  const float top = __uint_as_float(max_bits), s = top * shift;
  const bool number = max_bits < 0x7f800000u, holds = number && s >= __uint_as_float(kState8TinyBits);
  BlockScale out;
  out.s = holds ? s : number ? 0.0f : __uint_as_float(0x7fc00000u);
  // 256 / top correctly rounded, so that top * inv rounds to 256 at most.  (1 / top, taken first, is subnormal from 2^126 on.)
  out.inv = holds ? 1.0f / (top * 0.00390625f) : 0.0f;
  return out;
}

// Four elements of a block to their codes, to nearest (ties to even) or dithered by four numbers of 32 bits, of which the
// conversion uses the upper 20: it adds them below the last kept bit and cuts (also where e4m3 is subnormal).
__device__ __forceinline__ uint32_t encode_nearest(const float (&y)[4]) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  return (uint32_t)w;
}
__device__ __forceinline__ uint32_t encode_dithered(const float (&y)[4], uint32_t u) {
  int w = __builtin_amdgcn_cvt_sr_fp8_f32(y[0], u, 0, 0);
  w = __builtin_amdgcn_cvt_sr_fp8_f32(y[1], u + kDitherPlace, w, 1);
  w = __builtin_amdgcn_cvt_sr_fp8_f32(y[2], u + 2u * kDitherPlace, w, 2);
  w = __builtin_amdgcn_cvt_sr_fp8_f32(y[3], u + 3u * kDitherPlace, w, 3);
  return (uint32_t)w;
}
// Four codes to values; k = s / 256.
__device__ __forceinline__ void decode(uint32_t w, float k, float (&x)[4]) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = lo.x * k;
  x[1] = lo.y * k;
  x[2] = hi.x * k;
  x[3] = hi.y * k;
}

// One dword of codes per lane.
template <bool NT> __device__ __forceinline__ uint32_t ld_codes(const char* p) {
  const RG_GLOBAL uint32_t* g = (const RG_GLOBAL uint32_t*)p;
  return NT ? __builtin_nontemporal_load(g) : *g;
}
template <bool NT> __device__ __forceinline__ void st_codes(char* p, uint32_t w) {
  RG_GLOBAL uint32_t* g = (RG_GLOBAL uint32_t*)p;
  if (NT) __builtin_nontemporal_store(w, g);
  else *g = w;
}
// A block's scale, the same address for all lanes: through a pointer of the global address space it becomes a scalar load, through
// a generic one a FLAT load, whose wait drains every load in flight.  The step takes the same time either way.  (A scale is read
// before its block's wavefront, and no other, writes it; the scalar cache starts empty in every launch.)
__device__ __forceinline__ float load_scale(const float* p) { return *(const RG_GLOBAL float*)p; }
__device__ __forceinline__ uint32_t load_u8(const char* p) { return (uint32_t)*(const RG_GLOBAL unsigned char*)p; }

}  // namespace
}  // namespace rg
