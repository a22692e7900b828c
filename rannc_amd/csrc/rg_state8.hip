// Optimizer states in 8 bits: the Adam step that keeps both moments that way, and the conversions between 8 and 32 bits.
// All of it is bound by HBM.  Figures in this file: MI355X, BERT-large's 391 tensors (335,141,888 elements) unless others are named.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "rg_host.h"
#include "rg_internal.h"
#include "rg_state8.h"

namespace rg {
namespace {

constexpr int kLaneElems = 4;      // elements of a block one lane holds: 64 lanes, 256 elements
// The step: 2 wavefronts, a block each.  It lives from wavefronts in flight: 858 us with all 16 workgroups a compute unit holds,
// 896 / 1,015 / 1,090 us with 13 / 10 / 8.  64 threads 860-885 us, 256 threads 872 us; over bare arrays two or four blocks a
// wavefront, their loads up front, are 3-6 % slower than one.
constexpr int kAdam8Threads = 128, kAdam8TileElems = 512;
// The conversions: 2 wavefronts, two blocks each, 4 KiB of values in two accesses a lane.  Reading back 254 us; over bare arrays
// 247 us this way, 293-301 us with one block a wavefront, 283-311 us with four.
constexpr int kConvThreads = 128, kConvTileElems = 1024;
constexpr int64_t kState8ChunkElems = 8192;      // elements of a full record of a conversion's table

template <int DT> __device__ __forceinline__ float load_one(const char* p) { return __uint_as_float(load_u32(p)); }
template <> __device__ __forceinline__ float load_one<RG_F16>(const char* p) {
  return f16_to_f32(__builtin_bit_cast(_Float16, (unsigned short)load_u16(p)));
}
template <> __device__ __forceinline__ float load_one<RG_BF16>(const char* p) { return bf16_bits_to_f32(load_u16(p)); }

// Four elements of a lane, of which `n` exist (the rest read as zeros).
template <int DT, bool NT> __device__ __forceinline__ void load4(const char* p, int n, float (&f)[4]) {
  if (n >= 4) {
    Codec<DT, 4>::unpack(Mem<DT, 4, NT>::load(p), f);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = j < n ? load_one<DT>(p + (size_t)j * ElemSize<DT>::value) : 0.0f;
}
template <int DT, bool NT> __device__ __forceinline__ void store4(char* p, int n, const float (&f)[4]) {
  if (n >= 4) {
    Mem<DT, 4, NT>::store(p, Codec<DT, 4>::pack(f));
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < n) store1<DT>(p + (size_t)j * ElemSize<DT>::value, f[j]);
}
template <bool NT> __device__ __forceinline__ uint32_t load_codes4(const char* p, int n) {
  if (n >= 4) return ld_codes<NT>(p);
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < n) w |= load_u8(p + j) << (8 * j);
  return w;
}
template <bool NT> __device__ __forceinline__ void store_codes4(char* p, int n, uint32_t w) {
  if (n >= 4) {
    st_codes<NT>(p, w);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < n) store_u8(p + j, (w >> (8 * j)) & 0xffu);
}

// Hand-out order of a launch's tiles: workgroups are dealt to the eight XCDs in turn, and runs of consecutive tiles go to
// one of them (an incomplete last round keeps its order).  The step, BERT-large in bf16 / 621 M elements in fp16 / 934 ResNet tensors in
// fp32, by run: 16: 909 / 1,716 / 604 us, 64: 884 / 1,666 / 581, 128: 864 / 1,655 / 585, 224: 860 / 1,630 / 590,
// 448: 867 / 1,621 / 592.  From 128 to 448 each stays within 2 % of its best; 224 and 448 have the least sum, and 224 keeps the order
// of shorter tables.  The conversions over bare arrays: reading back 259 us in turn and 247 in runs of 64; quantizing does not care (263
// and 262) and takes the same run.
constexpr unsigned kXcdRun = 224;
constexpr unsigned kConvXcdRun = 64;
template <unsigned RUN> __device__ __forceinline__ unsigned tile_of_block() {
  const unsigned b = blockIdx.x, round = b / (8u * RUN) * (8u * RUN);
  if (round + 8u * RUN > gridDim.x) return b;
  const unsigned in = b - round;
  return round + (in % 8u) * RUN + in / 8u;
}

// Stores of a wavefront's lanes side by side at `base` (the same for all lanes): streaming ones as raw buffer stores with
// the policy "sc1 nt".  Against "nt" alone: reading back over bare arrays 247 and 276 us, the step no different; "sc1" alone costs the step 5 %.
constexpr int kStreamAux = 18;
template <bool NT> __device__ __forceinline__ void put16(char* base, uint32_t off, u32x4 v) {
  if (NT) __builtin_amdgcn_raw_buffer_store_b128(v, __builtin_amdgcn_make_buffer_rsrc(base, 0, -1, 0x00020000), off, 0, kStreamAux);
  else st16<false>(base + off, v);
}
template <bool NT> __device__ __forceinline__ void put8(char* base, uint32_t off, u32x2 v) {
  if (NT) __builtin_amdgcn_raw_buffer_store_b64(v, __builtin_amdgcn_make_buffer_rsrc(base, 0, -1, 0x00020000), off, 0, kStreamAux);
  else st8<false>(base + off, v);
}
template <bool NT> __device__ __forceinline__ void put4(char* base, uint32_t off, uint32_t v) {
  if (NT) __builtin_amdgcn_raw_buffer_store_b32(v, __builtin_amdgcn_make_buffer_rsrc(base, 0, -1, 0x00020000), off, 0, kStreamAux);
  else st_codes<false>(base + off, v);
}
template <int DT, bool NT> __device__ __forceinline__ void put_raw(char* base, int lane, const Raw<DT, 4>& r) {
  if constexpr (DT == RG_F32) put16<NT>(base, (uint32_t)lane * 16u, r.v);
  else put8<NT>(base, (uint32_t)lane * 8u, r.v);
}

__device__ __forceinline__ float maximum_abs3(float a, float b, float c) {   // NaN if any is
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(__builtin_fabsf(a), __builtin_fabsf(b)), __builtin_fabsf(c));
}

// Square root in five instructions (the compiler's own takes 15), correctly rounded, for 2^-100 <= x < infinity; NaN for anything smaller than 2^-126 (zero too) and for
// infinity.  The estimate x * rsq(x) is off by at most a few units; its residual x - s^2 is exact in one fma, and s +
// residual / (2 s) then rounds as the root itself does: tests/test_gpu_state8_magnitudes.py compares every number of the
// range with the root in float64.
__device__ __forceinline__ float sqrt_normal(float x) {
  const float y = __builtin_amdgcn_rsqf(x);
  const float s = x * y;
  return __builtin_fmaf(__builtin_fmaf(-s, s, x), 0.5f * y, s);
}

__device__ __forceinline__ float minimum3(float a, float b, float c) {       // NaN if any is
  return __builtin_elementwise_minimum(__builtin_elementwise_minimum(a, b), c);
}

// Squares are carried times 2^50 and roots times 2^25, so that every square that fp32 holds lies in sqrt_normal's range
// (a product's factor is moved instead of the product, which costs nothing and changes no rounding).  The square of a root
// that is held in 8 bits (2^-117 at the least) may still lie below it: quick roots under 2^-50 are not used.
constexpr float kRootShift = 33554432.0f, kSquareShift = 1125899906842624.0f;
constexpr float kLeastQuickSquare = 7.888609052210118e-31f, kLeastQuickRoot = 8.881784197001252e-16f;    // 2^-100, 2^-50

// The root times 2^25 for any magnitudes: q is the old root times 2^25.  Every product is rounded as if exponents had no end:
// what leaves fp32's range times 2^50 is worked out times 1 or times 2^200.
__device__ __forceinline__ float root_of_any(float q, float g, float beta2, float one_minus_beta2) {
  const float square = beta2 * (q * q) + ((one_minus_beta2 * kSquareShift) * g) * g;
  if (square < kLeastQuickSquare) {
    const float old = fminf(q, 67108864.0f) * 137438953472.0f;            // 2^37; the minimum is q, unless beta2 is 0
    const float grad = g * 1.2676506002282294e30f;                        // 2^100
    return sqrtf((beta2 * 7.555786372591432e22f) * (old * old) + (one_minus_beta2 * grad) * grad) * 2.6469779601696886e-23f;   // 2^76, 2^-75
  }
  if (square < __builtin_inff()) return sqrtf(square);
  const float old = q * (1.0f / kRootShift);
  return sqrtf(beta2 * (old * old) + (one_minus_beta2 * g) * g) * kRootShift;
}

// One block of 256 elements (fewer at a tensor's end) by one wavefront, four per lane:
//   m = beta1 m + (1 - beta1) g,  v = beta2 r^2 + (1 - beta2) g^2,  r = sqrt(v),  p -= step_size m / (r / bias2_sqrt + eps)
// and m and r back to codes by their new largest magnitudes.  Every operation that a code depends on is rounded by itself,
// so the codes are those of the same formulas written in elementary fp32 operations; the parameter's quotient is not
// (a reciprocal of 1 unit).  About 52 vector instructions an element: 858-870 us for 5.38 GB (6.2-6.3 TB/s), and the same in builds
// without the square root, the encoding or the reduction: HBM with six streams read and written bounds it (838-852 us for those
// streams over bare arrays without a table).  Those figures are for tensors that begin at multiples of 256 elements.  A block lies
// where its tensor puts it, so on others the parameter's and copy's accesses straddle lines: 1,097 us with tensors 16 elements further on,
// 1,200 us with tensors 1 or 3 elements further on.
template <int G, int C, bool NT, bool FULL>
__device__ __forceinline__ void adam8_block(const Opt8ChunkRec& r, int start, int lane, const Adam8Const& c, float coef,
                                            uint32_t step) {
  constexpr int CD = C >= 0 ? C : RG_F32;
  constexpr int GS = ElemSize<G>::value, CS = ElemSize<CD>::value;
  const int block = start / kState8Block;
  const int n = FULL ? kLaneElems : r.len - start - lane * kLaneElems;       // <= 0: this lane has no element
  char* pp = reinterpret_cast<char*>(r.param) + (size_t)start * 4;
  const char* gp = reinterpret_cast<const char*>(r.grad) + (size_t)start * GS;
  char* c1 = reinterpret_cast<char*>(r.codes1) + start;
  char* c2 = reinterpret_cast<char*>(r.codes2) + start;
  char* cp = reinterpret_cast<char*>(r.copy) + (size_t)start * CS;
  float p[4], g[4], m[4], q[4];
  load4<RG_F32, NT>(pp + lane * 16, n, p);
  load4<G, NT>(gp + lane * (4 * GS), n, g);
  const uint32_t w1 = load_codes4<NT>(c1 + lane * 4, n), w2 = load_codes4<NT>(c2 + lane * 4, n);
  const float s1_old = load_scale(r.scales1 + block), s2_old = load_scale(r.scales2 + block);
  decode(w1, s1_old * 0.00390625f, m);                                       // s / 256
  decode(w2, s2_old * (0.00390625f * kRootShift), q);
#pragma unroll
  for (int j = 0; j < 4; ++j) {        // x * 1 is x: no branch needed
    g[j] = g[j] * c.grad_scale;
    g[j] = g[j] * coef;
    p[j] = p[j] * c.param_mul;
  }
  if (c.weight_decay != 0.0f) {
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = g[j] + c.weight_decay * p[j];
  }
  float root[4];
  const float one_minus_beta2 = c.one_minus_beta2 * kSquareShift;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = c.beta1 * m[j] + c.one_minus_beta1 * g[j];
    root[j] = sqrt_normal(c.beta2 * (q[j] * q[j]) + (one_minus_beta2 * g[j]) * g[j]);
  }
  float top2 = __builtin_elementwise_maximum(maximum_abs3(root[0], root[1], root[2]), root[3]);
  const float low2 = __builtin_elementwise_minimum(minimum3(root[0], root[1], root[2]), root[3]);
  const bool plain = __builtin_amdgcn_ballot_w64(!(low2 >= kLeastQuickRoot)) == 0;
  if (!plain) {      // some second moment is zero, very small or not a number: the roots one by one
    top2 = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      root[j] = root_of_any(q[j], g[j], c.beta2, c.one_minus_beta2);
      top2 = __builtin_elementwise_maximum(top2, __builtin_fabsf(root[j]));
    }
  }
  const float top1 = __builtin_elementwise_maximum(maximum_abs3(m[0], m[1], m[2]), __builtin_fabsf(m[3]));
  const float inv_bias = c.inv_bias2_sqrt * (1.0f / kRootShift);
  if (plain) {       // the denominators are normal numbers: a reciprocal (1 unit) in place of the division
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = p[j] + (c.neg_step_size * m[j]) * __builtin_amdgcn_rcpf(root[j] * inv_bias + c.eps);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = p[j] + (c.neg_step_size * m[j]) / (root[j] * inv_bias + c.eps);
  }
  if (FULL) put_raw<RG_F32, NT>(pp, lane, Codec<RG_F32, 4>::pack(p));
  else store4<RG_F32, NT>(pp + lane * 16, n, p);
  if constexpr (C >= 0) {
    if (FULL) put_raw<CD, NT>(cp, lane, Codec<CD, 4>::pack(p));
    else store4<CD, NT>(cp + lane * (4 * CS), n, p);
  }

  // Both moments' largest at once: the lower half of the wavefront ends up with the first's, the upper with the root's.
  const BlockScale s = block_scale(half_max(magnitude_bits(top1), magnitude_bits(top2)), lane < 32 ? 1.0f : 1.0f / kRootShift);
  const float inv1 = read_lane_f32(s.inv, 0), inv2 = read_lane_f32(s.inv, 32);
  if ((lane & 31) == 0) store1<RG_F32>(reinterpret_cast<char*>((lane == 0 ? r.scales1 : r.scales2) + block), s.s);

  const uint32_t place = (r.first + (uint32_t)start) * kDitherPlace, u = (uint32_t)lane * (kLaneElems * kDitherPlace);
  uint32_t o1 = 0, o2 = 0;
  if (inv1 != 0.0f) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = m[j] * inv1;
    o1 = encode_dithered(y, u + (place + step * kDitherFirst));
  }
  if (inv2 != 0.0f) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = fmaxf(root[j] * inv2, kState8MinRoot);
    if (!plain) {
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = root[j] > 0.0f ? y[j] : 0.0f;
    }
    o2 = encode_dithered(y, u + (place + step * kDitherRoot));
  }
  if (FULL) {
    put4<NT>(c1, (uint32_t)lane * 4u, o1);
    put4<NT>(c2, (uint32_t)lane * 4u, o2);
  } else {
    store_codes4<NT>(c1 + lane * 4, n, o1);
    store_codes4<NT>(c2 + lane * 4, n, o2);
  }
}

template <bool NT>
__global__ __launch_bounds__(kAdam8Threads) void adam8_kernel(Adam8Args a) {
  float coef = 1.0f;
  if (a.gate != nullptr) {
    if (a.gate->skipped != 0) return;
    coef = a.gate->coef;
  }
  if (a.grad_scale_dev != nullptr) a.c.grad_scale = a.grad_scale_sign * *a.grad_scale_dev;
  uint32_t step = a.step;
  if (a.clock != nullptr) {      // written by adam_clock_kernel earlier on the same stream
    step = (uint32_t)a.clock->step;
    a.c.neg_step_size = a.clock->neg_step_size;
    a.c.inv_bias2_sqrt = 1.0f / a.clock->bias2_sqrt;
  }
  constexpr unsigned kTiles = (unsigned)(kOpt8ChunkElems / kAdam8TileElems);
  const unsigned t = tile_of_block<kXcdRun>();
  const Opt8ChunkRec r = a.chunks[t / kTiles];
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64u)), lane = (int)(threadIdx.x % 64u);
  const int start = (int)(t % kTiles) * kAdam8TileElems + wave * kState8Block;
  if (start >= r.len) return;
  const bool full = r.len - start >= kState8Block;
  const int copy_kind = r.copy ? r.copy_dtype : -1;
#define RG_ADAM8(G, C)                                                    \
  if (r.grad_dtype == G && copy_kind == C) {                              \
    if (full) adam8_block<G, C, NT, true>(r, start, lane, a.c, coef, step); \
    else adam8_block<G, C, NT, false>(r, start, lane, a.c, coef, step);   \
    return;                                                               \
  }
  RG_ADAM8(RG_F32, -1)
  RG_ADAM8(RG_F32, RG_BF16)
  RG_ADAM8(RG_F32, RG_F16)
  RG_ADAM8(RG_F32, RG_F32)
  RG_ADAM8(RG_BF16, -1)
  RG_ADAM8(RG_BF16, RG_BF16)
  RG_ADAM8(RG_BF16, RG_F16)
  RG_ADAM8(RG_BF16, RG_F32)
  RG_ADAM8(RG_F16, -1)
  RG_ADAM8(RG_F16, RG_F16)
  RG_ADAM8(RG_F16, RG_BF16)
  RG_ADAM8(RG_F16, RG_F32)
#undef RG_ADAM8
}

// ---------------------------------------------------------------- conversions

// One row of a conversion's work table: a run of whole blocks of one tensor (the last may be shorter).
struct State8Rec {
  void* codes;
  float* scales;
  float* values;
  int32_t len;
  int32_t root;
};
static_assert(sizeof(State8Rec) == 32, "conversion record must stay 32 bytes");

// The magnitudes to be stored: the values, or their roots (times kRootShift).  `plain`: no root is zero or not a number.
template <bool ROOT> __device__ __forceinline__ bool stored_form(float (&x)[4], float& top) {
  if (!ROOT) {
    top = __builtin_elementwise_maximum(maximum_abs3(x[0], x[1], x[2]), __builtin_fabsf(x[3]));
    return true;
  }
  float r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = sqrt_normal(x[j] * kSquareShift);
  top = __builtin_elementwise_maximum(maximum_abs3(r[0], r[1], r[2]), r[3]);
  const bool plain = __builtin_amdgcn_ballot_w64(top != top) == 0;
  if (!plain) {
    top = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r[j] = sqrtf(x[j]) * kRootShift;
      top = __builtin_elementwise_maximum(top, __builtin_fabsf(r[j]));
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = r[j];
  return plain;
}
template <bool ROOT> __device__ __forceinline__ uint32_t nearest_codes(const float (&x)[4], float inv, bool plain) {
  if (inv == 0.0f) return 0;
  float y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[j] = x[j] * inv;
    if (ROOT) {
      y[j] = fmaxf(y[j], kState8MinRoot);
      if (!plain) y[j] = x[j] > 0.0f ? y[j] : 0.0f;
    }
  }
  return encode_nearest(y);
}

// Two consecutive blocks by one wavefront (the second may be missing, either may end early), so that one reduction
// finds both largest magnitudes.  261 us for 1.68 GB (6.4 TB/s; 257-262 us over bare arrays).
template <bool ROOT, bool NT, bool FULL>
__device__ __forceinline__ void quantize_pair(const State8Rec& r, int start, int lane) {
  const char* vp = reinterpret_cast<const char*>(r.values) + (size_t)start * 4;
  char* cp = reinterpret_cast<char*>(r.codes) + start;
  const int na = FULL ? kLaneElems : r.len - start - lane * kLaneElems, nb = FULL ? kLaneElems : na - kState8Block;
  float a[4], b[4], top_a, top_b;
  load4<RG_F32, NT>(vp + lane * 16, na, a);
  load4<RG_F32, NT>(vp + (kState8Block * 4 + lane * 16), nb, b);
  const bool plain_a = stored_form<ROOT>(a, top_a), plain_b = stored_form<ROOT>(b, top_b);
  const BlockScale s = block_scale(half_max(magnitude_bits(top_a), magnitude_bits(top_b)), ROOT ? 1.0f / kRootShift : 1.0f);
  const uint32_t wa = nearest_codes<ROOT>(a, read_lane_f32(s.inv, 0), plain_a);
  const uint32_t wb = nearest_codes<ROOT>(b, read_lane_f32(s.inv, 32), plain_b);
  if (FULL) {
    put4<NT>(cp, (uint32_t)lane * 4u, wa);
    put4<NT>(cp, (uint32_t)lane * 4u + kState8Block, wb);
  } else {
    store_codes4<NT>(cp + lane * 4, na, wa);
    store_codes4<NT>(cp + (kState8Block + lane * 4), nb, wb);
  }
  const int block = start / kState8Block + (lane >> 5);
  if ((lane & 31) == 0 && block * kState8Block < r.len) store1<RG_F32>(reinterpret_cast<char*>(r.scales + block), s.s);
}

// Back to fp32, two blocks a wavefront with both loads first: 253 us for 1.68 GB (6.6 TB/s), four fifths of it written.  (Block
// after block in one wavefront, each store behind its own load: 379 us.  Values that begin 1 or 3 elements off a multiple of 256: 352 us,
// 16 elements off: 254 us; quantizing takes the same time at any place.)
template <bool ROOT, bool NT, bool FULL>
__device__ __forceinline__ void dequantize_pair(const State8Rec& r, int start, int lane) {
  char* vp = reinterpret_cast<char*>(r.values) + (size_t)start * 4;
  const char* cp = reinterpret_cast<const char*>(r.codes) + start;
  const int na = FULL ? kLaneElems : r.len - start - lane * kLaneElems, nb = FULL ? kLaneElems : na - kState8Block;
  const uint32_t wa = load_codes4<NT>(cp + lane * 4, na), wb = load_codes4<NT>(cp + (kState8Block + lane * 4), nb);
  const int block = start / kState8Block;
  const bool second = FULL || r.len - start > kState8Block;
  const float sa = load_scale(r.scales + block), sb = second ? load_scale(r.scales + block + 1) : 0.0f;
  float a[4], b[4];
  decode(wa, sa * 0.00390625f, a);
  decode(wb, sb * 0.00390625f, b);
  if (ROOT) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = a[j] * a[j];
      b[j] = b[j] * b[j];
    }
  }
  if (FULL) {
    put16<NT>(vp, (uint32_t)lane * 16u, Codec<RG_F32, 4>::pack(a).v);
    put16<NT>(vp, (uint32_t)lane * 16u + kState8Block * 4, Codec<RG_F32, 4>::pack(b).v);
  } else {
    store4<RG_F32, NT>(vp + lane * 16, na, a);
    store4<RG_F32, NT>(vp + (kState8Block * 4 + lane * 16), nb, b);
  }
}

template <bool WRITE_CODES, bool NT>
__global__ __launch_bounds__(kConvThreads) void state8_kernel(const State8Rec* recs) {
  constexpr unsigned kTiles = (unsigned)(kState8ChunkElems / kConvTileElems);
  const unsigned t = tile_of_block<kConvXcdRun>();
  const State8Rec r = recs[t / kTiles];
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64u)), lane = (int)(threadIdx.x % 64u);
  const int start = (int)(t % kTiles) * kConvTileElems + wave * (2 * kState8Block);
  if (start >= r.len) return;
  const bool full = r.len - start >= 2 * kState8Block;
#define RG_CONVERT(ROOT, FULL)                                        \
  if ((r.root != 0) == ROOT && full == FULL) {                        \
    if (WRITE_CODES) quantize_pair<ROOT, NT, FULL>(r, start, lane);   \
    else dequantize_pair<ROOT, NT, FULL>(r, start, lane);             \
    return;                                                           \
  }
  RG_CONVERT(false, true)
  RG_CONVERT(true, true)
  RG_CONVERT(false, false)
  RG_CONVERT(true, false)
#undef RG_CONVERT
}

}  // namespace

// A launch holds fewer than 2^32 threads: larger tables take several.
constexpr int64_t kMaxBlocks = (int64_t)1 << 24;
template <typename F> static hipError_t launch_in_parts(int64_t n_chunks, int64_t tiles_per_chunk, const F& launch) {
  const int64_t most = kMaxBlocks / tiles_per_chunk;
  for (int64_t at = 0; at < n_chunks; at += most) {
    launch(at, (unsigned)(std::min(most, n_chunks - at) * tiles_per_chunk));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_adam8(const Adam8Args& args, int64_t n_chunks, bool streaming, hipStream_t stream) {
  return launch_in_parts(n_chunks, kOpt8ChunkElems / kAdam8TileElems, [&](int64_t at, unsigned blocks) {
    Adam8Args a = args;
    a.chunks += at;
    if (streaming) hipLaunchKernelGGL((adam8_kernel<true>), dim3(blocks), dim3(kAdam8Threads), 0, stream, a);
    else hipLaunchKernelGGL((adam8_kernel<false>), dim3(blocks), dim3(kAdam8Threads), 0, stream, a);
  });
}

}  // namespace rg

using namespace rg;

struct rg_state8 {
  int device = 0;
  int64_t n_chunks = 0;
  int64_t total_numel = 0;
  State8Rec* d_recs = nullptr;
};

RG_API int64_t rg_state8_num_scales(int64_t numel) { return numel < 0 ? -1 : (numel + kState8Block - 1) / kState8Block; }

RG_API int rg_state8_create(rg_state8** out, int device, int n, void* const* codes, float* const* scales, float* const* values,
                            const int64_t* numel, const int* root) {
  if (out == nullptr || n < 0 ||
      (n > 0 && (codes == nullptr || scales == nullptr || values == nullptr || numel == nullptr || root == nullptr))) {
    set_error("rg_state8_create: bad arguments");
    return RG_EINVAL;
  }
  *out = nullptr;
  int64_t chunks = 0, total = 0;
  for (int i = 0; i < n; ++i) {
    if (numel[i] < 0 || numel[i] > kMaxTensorElems) {
      set_error("rg_state8_create: tensor %d has %lld elements", i, (long long)numel[i]);
      return RG_EINVAL;
    }
    if (numel[i] == 0) continue;
    if (codes[i] == nullptr || scales[i] == nullptr || values[i] == nullptr) {
      set_error("rg_state8_create: tensor %d lacks its codes, scales or values", i);
      return RG_EINVAL;
    }
    int rc = check_pointer(codes[i], 4, "codes", i);
    if (rc == RG_OK) rc = check_pointer(scales[i], 4, "scales", i);
    if (rc == RG_OK) rc = check_pointer(values[i], 4, "values", i);
    if (rc != RG_OK) return rc;
    chunks += (numel[i] + kState8ChunkElems - 1) / kState8ChunkElems;
    total += numel[i];
  }
  rg_state8* t = new (std::nothrow) rg_state8;
  if (t == nullptr) {
    set_error("rg_state8_create: out of host memory");
    return RG_ENOMEM;
  }
  t->device = device;
  t->n_chunks = chunks;
  t->total_numel = total;
  if (chunks > 0) {
    State8Rec* recs = new (std::nothrow) State8Rec[(size_t)chunks];
    if (recs == nullptr) {
      delete t;
      set_error("rg_state8_create: out of host memory");
      return RG_ENOMEM;
    }
    int64_t c = 0;
    for (int i = 0; i < n; ++i) {
      for (int64_t start = 0; start < numel[i]; start += kState8ChunkElems, ++c) {
        State8Rec& r = recs[c];
        r.codes = static_cast<char*>(codes[i]) + start;
        r.scales = scales[i] + start / kState8Block;
        r.values = values[i] + start;
        r.len = (int32_t)std::min(numel[i] - start, kState8ChunkElems);
        r.root = root[i] ? 1 : 0;
      }
    }
    DeviceGuard guard(device);
    hipError_t e = hipMalloc(reinterpret_cast<void**>(&t->d_recs), (size_t)chunks * sizeof(State8Rec));
    if (e == hipSuccess) e = hipMemcpy(t->d_recs, recs, (size_t)chunks * sizeof(State8Rec), hipMemcpyHostToDevice);
    delete[] recs;
    if (e != hipSuccess) {
      const int code = hip_fail(e, "rg_state8_create");
      (void)rg_state8_destroy(t);
      return e == hipErrorOutOfMemory ? RG_ENOMEM : code;
    }
  }
  *out = t;
  return RG_OK;
}

RG_API int rg_state8_destroy(rg_state8* t) {
  if (t == nullptr) return RG_OK;
  DeviceGuard guard(t->device);
  if (t->d_recs) (void)hipFree(t->d_recs);
  delete t;
  return RG_OK;
}

static int launch_state8(const rg_state8* t, bool write_codes, void* stream, const char* op) {
  if (t == nullptr) {
    set_error("%s: null table", op);
    return RG_EINVAL;
  }
  if (t->n_chunks == 0) return RG_OK;
  DeviceGuard guard(t->device);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool nt = streams(t->total_numel * 5);
  RG_HIP(launch_in_parts(t->n_chunks, kState8ChunkElems / kConvTileElems, [&](int64_t at, unsigned blocks) {
    const dim3 grid(blocks), block(kConvThreads);
    const State8Rec* recs = t->d_recs + at;
    if (write_codes && nt) hipLaunchKernelGGL((state8_kernel<true, true>), grid, block, 0, s, recs);
    else if (write_codes) hipLaunchKernelGGL((state8_kernel<true, false>), grid, block, 0, s, recs);
    else if (nt) hipLaunchKernelGGL((state8_kernel<false, true>), grid, block, 0, s, recs);
    else hipLaunchKernelGGL((state8_kernel<false, false>), grid, block, 0, s, recs);
  }));
  return RG_OK;
}

RG_API int rg_state8_quantize(rg_state8* t, void* stream) { return launch_state8(t, true, stream, "rg_state8_quantize"); }
RG_API int rg_state8_dequantize(rg_state8* t, void* stream) { return launch_state8(t, false, stream, "rg_state8_dequantize"); }
