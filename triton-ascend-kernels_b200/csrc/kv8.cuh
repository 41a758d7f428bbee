// Shared definitions of the 8-bit KV cache kernels: the cache's description,
// code <-> value conversion, and the bounded page lookup.
//
// A cache holds K and V rows as 8-bit codes [num_blocks, Hkv, block_size, D]
// with one fp32 scale per (page, KV head, group of `group` rows): an element's
// value is code * scale.  Codes are int8 (|code| <= 127) or e4m3.
#pragma once

#include <cuda_fp8.h>

#include "../../include/tak_attention.h"
#include "common.cuh"
#include "kernels.h"

namespace tak {

enum Kv8Code : int { kI8 = 0, kE4M3 = 1 };

// K or V plane of a cache (codes and scales), as the kernels see it.
struct Kv8Plane {
  uint8_t* code;
  int64_t sc[4];
  float* scale;
  int64_t ss[3];
};

// Division of x < 2^31 by an invariant divisor (Granlund and Montgomery, 1994): with
// 2^l the least power of two that is at least d and mul = floor(2^(31 + l) / d) + 1,
// the quotient is x * mul >> (31 + l).  mul 0 stands for d = 1.
struct Kv8Div {
  uint32_t mul, shift;
  __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return mul ? __umulhi(x, mul) >> shift : x; }
};
inline Kv8Div kv8_div_by(uint32_t d) {
  if (d <= 1) return {0, 0};
  uint32_t l = 1;
  while ((uint64_t{1} << l) < d) ++l;
  return {static_cast<uint32_t>((uint64_t{1} << (31 + l)) / d + 1), l - 1};
}

struct Kv8View {
  Kv8Plane plane[2];  // K, V
  const int32_t* block_tables;
  int64_t sbt[2];
  int Hkv, P, D, group, num_seqs, max_blocks;
  int64_t num_blocks;
  int64_t max_rows;  // max_blocks * P, at most 2^31 - 2^16
  Kv8Div by_P, by_group;
};

// Page holding row r of sequence s, or -1 when the row lies past the
// sequence's block-table row or the table names a page outside the cache.
__device__ __forceinline__ int64_t kv8_page(const Kv8View& c, int s, int64_t r) {
  if (r < 0 || r >= c.max_rows) return -1;
  const int64_t page = c.block_tables[s * c.sbt[0] + static_cast<int64_t>(c.by_P(static_cast<uint32_t>(r))) * c.sbt[1]];
  return (page >= 0 && page < c.num_blocks) ? page : -1;
}
__device__ __forceinline__ uint8_t* kv8_row(const Kv8Plane& p, int64_t page, int h, int row) {
  return p.code + page * p.sc[0] + h * p.sc[1] + row * p.sc[2];
}
__device__ __forceinline__ float* kv8_scale(const Kv8Plane& p, int64_t page, int h, int g) {
  return p.scale + page * p.ss[0] + h * p.ss[1] + g * p.ss[2];
}

template <int CODE> struct Kv8;
template <> struct Kv8<kI8> {
  static constexpr float kInvMax = 1.0f / 127.0f;
  static __device__ __forceinline__ float dec(uint8_t c) { return static_cast<float>(static_cast<int8_t>(c)); }
  // round to nearest even, as rintf; NaN and out-of-range products cannot
  // reach it from a finite scale (|x| <= amax), the clamp keeps -128 out
  static __device__ __forceinline__ uint8_t enc(float x) {
    const int v = __float2int_rn(x);
    return static_cast<uint8_t>(static_cast<int8_t>(max(-127, min(127, v))));
  }
};
template <> struct Kv8<kE4M3> {
  static constexpr float kInvMax = 1.0f / 448.0f;
  static __device__ __forceinline__ float dec(uint8_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(c), __NV_E4M3)));
  }
  static __device__ __forceinline__ uint8_t enc(float x) {
    return static_cast<uint8_t>(__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3));
  }
};

// Magnitudes are compared as the bits of |x| (ordered as the floats are), so
// infinities and NaN come out largest and are never lost in a maximum.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr uint32_t kInfBits = 0x7f800000u;
constexpr float kTinyAmax = 7.8886090522101180541e-31f;  // 2^-100

// Scale of a group whose largest magnitude has the bits `amax`: amax / QMAX
// (as a product with the rounded reciprocal); 0 below 2^-100, where 1 / scale
// would leave fp32's range; NaN when the group holds an infinity or a NaN, so
// that its rows read back as NaN instead of as wrong finite values.
template <int CODE>
__device__ __forceinline__ float kv8_scale_of(uint32_t amax) {
  if (amax >= kInfBits) return __uint_as_float(0x7fffffffu);
  const float a = __uint_as_float(amax);
  return a < kTinyAmax ? 0.f : a * Kv8<CODE>::kInvMax;
}
// maximum of two non-negative scales that keeps a NaN
__device__ __forceinline__ float kv8_scale_max(float a, float b) {
  return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
}

// Four codes at once, the same roundings as dec and enc one by one.
// int8 -> fp32: the byte with its sign bit flipped, as the mantissa's low byte of
// 2^23, less 2^23 + 128.  fp32 -> int8: adding 1.5 * 2^23 rounds to nearest even
// and leaves the two's complement in the low byte; a group's own scale keeps |f|
// within 127 (1 + 2^-22), so nothing has to be clamped.
// (Two fp32 operations at a time where both halves take the same one.)
__device__ __forceinline__ void add2(float& a, float& b, float c) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(c));
}
__device__ __forceinline__ void mul2(float& a, float& b, float c) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(c));
}
template <int CODE> __device__ __forceinline__ void kv8_dec4(uint32_t q, float* f) {
  if (CODE == kI8) {
    const uint32_t x = q ^ 0x80808080u;
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = __uint_as_float(__byte_perm(x, 0x4b000000u, 0x7540 + k));
    add2(f[0], f[1], -8388736.f);
    add2(f[2], f[3], -8388736.f);
  } else {
    const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(q & 0xffffu), __NV_E4M3)));
    const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(q >> 16), __NV_E4M3)));
    f[0] = a.x;
    f[1] = a.y;
    f[2] = b.x;
    f[3] = b.y;
  }
}
template <int CODE> __device__ __forceinline__ uint32_t kv8_enc4(const float* f) {
  if (CODE == kI8) {
    float g[4] = {f[0], f[1], f[2], f[3]};
    add2(g[0], g[1], 12582912.f);
    add2(g[2], g[3], 12582912.f);
    const uint32_t u[4] = {__float_as_uint(g[0]), __float_as_uint(g[1]), __float_as_uint(g[2]), __float_as_uint(g[3])};
    return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
  }
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
template <int CODE> __device__ __forceinline__ uint32_t kv8_rescale4(uint32_t q, float ratio) {
  float f[4];
  kv8_dec4<CODE>(q, f);
  if (CODE == kI8) {  // one by one: a packed product before the packed sum is fused with it, and rounds once
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = __fmul_rn(f[k], ratio);
  } else {
    mul2(f[0], f[1], ratio);
    mul2(f[2], f[3], ratio);
  }
  return kv8_enc4<CODE>(f);
}

struct Kv8AttnArgs {
  const void* q; int64_t sq[4];       // [B, Lq, H, D]
  const int32_t* context_lens;
  void* out; int64_t so[4];
  float* lse;                         // [B, Lq, H] contiguous, may be null
  float* weights; int64_t sw[3];      // [B, Hkv, W], may be null
  int64_t weights_width;
  int H, Lq;
  float scale, softcap;
  int dtype, code_type;
  void* workspace; int64_t workspace_bytes;
  int force_generic;
};
int kv8_write_launch(const Kv8View& c, int code_type, const void* k, const int64_t* sk, const void* v,
                     const int64_t* sv, const int32_t* start_lens, const int32_t* cu, int64_t total, int dtype,
                     cudaStream_t st);
int kv8_read_launch(const Kv8View& c, int code_type, const int32_t* cu, const int32_t* start_lens, int64_t total,
                    void* k, const int64_t* sk, void* v, const int64_t* sv, int dtype, cudaStream_t st);
int kv8_evict_launch(const Kv8View& c, int code_type, const int32_t* context_lens, float* weights,
                     const int64_t* sw, int64_t width, int64_t budget, int64_t recent, int32_t* kept,
                     int32_t* new_lens, cudaStream_t st);
int64_t kv8_attention_ws_bytes(const Kv8View& c, const Kv8AttnArgs& a);
int kv8_attention_launch(const Kv8View& c, const Kv8AttnArgs& a, cudaStream_t st);

// dispatch on the element type of 16 / 32-bit tensors and on the code type
#define TAK_BY_DTYPE(dtype, ...)                                        \
  do {                                                                  \
    if ((dtype) == kBF16) { using T = __nv_bfloat16; __VA_ARGS__; }     \
    else if ((dtype) == kF16) { using T = __half; __VA_ARGS__; }        \
    else { using T = float; __VA_ARGS__; }                              \
  } while (0)
#define TAK_BY_CODE(code, ...)                                          \
  do {                                                                  \
    if ((code) == kI8) { constexpr int CODE = kI8; __VA_ARGS__; }       \
    else { constexpr int CODE = kE4M3; __VA_ARGS__; }                   \
  } while (0)

}  // namespace tak
