// The 8-bit form of a matrix (lf_float8_matrix): codes in rows of whole 16-byte groups, and for every 128 consecutive channels of
// a row (of a weight: 128 x 128 elements) one power of two.
//
// amax = the largest finite magnitude of the block = m 2^p, 1 <= m < 2.  The largest finite code is 1.75 2^8 (e4m3) or 1.75 2^15 (e5m2), so
// the least power of two that brings amax to it is 2^(p - 8), or 2^(p - 7) where m > 1.75: the exponent field of amax less 8, plus a
// carry out of the mantissa.  It is kept as that biased byte, at least 1 (2^-126, the least normal number).  Scaling by it
// rounds nothing, so a code is one rounding of the value, and a decoded value (at most four significant bits) is exact in float32 and bf16.
//
// Exponent bytes lie as the tensor cores read them as scales: [512 channels][128 rows] tiles of 512 bytes, in a tile
// [row % 32][row / 32][block % 4].
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "common.cuh"

// Checks that several entry points share (float8.cu).
lf_status lf_float8_check_rows(lf_context* ctx, const char* what, int64_t rows, int channels, int dtype);
lf_status lf_float8_check(lf_context* ctx, const char* what, const lf_float8_matrix& m, int64_t rows, int channels);
lf_status lf_float8_done(lf_context* ctx, lf_result* r, int launches);

namespace f8 {

constexpr int kBlock = 128;      // channels that share an exponent

__host__ __device__ inline int64_t pitch(int channels) { return (channels + 15) & ~15; }
__host__ __device__ inline int blocks(int channels) { return (channels + kBlock - 1) / kBlock; }
__host__ __device__ inline int64_t row_tiles(int64_t rows) { return (rows + 127) >> 7; }
__host__ __device__ inline int64_t exponent_bytes(int64_t rows, int channels) { return (int64_t)((blocks(channels) + 3) / 4) * row_tiles(rows) * 512; }
// `tiles` = row_tiles(rows)
__device__ __forceinline__ int64_t exponent_at(int64_t row, int block, int64_t tiles) {
  return ((block >> 2) * tiles + (row >> 7)) * 512 + ((row & 31) << 4) + (((row >> 5) & 3) << 2) + (block & 3);
}

// Limit exponent of a format: 8 (e4m3) or 15 (e5m2).
__host__ __device__ constexpr int limit(int format) { return format == LF_FLOAT8_E4M3 ? 8 : 15; }
// From the bits of a finite amax.
__device__ __forceinline__ int exponent_byte(uint32_t amax, int format) {
  return max(1, (int)((amax + 0x1fffffu) >> 23) - limit(format));
}
// 2^(127 - s) and 2^(s - 127), 1 <= s <= 254
__device__ __forceinline__ float down(int s) { return __int_as_float((254 - s) << 23); }
__device__ __forceinline__ float up(int s) { return __int_as_float(s << 23); }

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
constexpr uint32_t kInfinity = 0x7f800000u;

// Two codes, x in the low byte.  `scaled` values are within the format's range (or not finite: see code_special).
__device__ __forceinline__ uint32_t code2(float x, float y, int format) {
  return __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, format == LF_FLOAT8_E4M3 ? __NV_E4M3 : __NV_E5M2);
}
// One code of a value that may be infinite: e4m3 has no infinity, so that it becomes NaN and is not lost in a finite code.
__device__ __forceinline__ uint32_t code_special(float v, int format) {
  const uint32_t sign = __float_as_uint(v) >> 24 & 0x80u;
  if (magnitude(v) > kInfinity) return format == LF_FLOAT8_E4M3 ? 0x7fu : 0x7eu;
  if (magnitude(v) == kInfinity) return sign | (format == LF_FLOAT8_E4M3 ? 0x7fu : 0x7cu);
  return code2(v, 0.f, format) & 0xffu;
}
__device__ __forceinline__ float2 decode2(uint32_t two, int format) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, format == LF_FLOAT8_E4M3 ? __NV_E4M3 : __NV_E5M2);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Eight codes -> eight values times `factor`
__device__ __forceinline__ void decode8(uint2 codes, float factor, int format, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 d = decode2((i < 2 ? codes.x : codes.y) >> (16 * (i & 1)) & 0xffffu, format);
    v[2 * i] = d.x * factor;
    v[2 * i + 1] = d.y * factor;
  }
}

// Eight neighbouring values of a row as one lane of a group of LANES <= 16 (a whole block's, or all of a narrower row's) holds them: the
// block's exponent byte, and the lane's codes.  All lanes of the warp call it.
template <int LANES>
__device__ __forceinline__ int encode8(const float (&v)[8], int format, uint2& codes) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, magnitude(v[i]));
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (__any_sync(0xffffffffu, most >= kInfinity)) {      // values that are not finite have no say in the scale
    uint32_t finite = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) finite = max(finite, magnitude(v[i]) < kInfinity ? magnitude(v[i]) : 0u);
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) finite = max(finite, __shfl_xor_sync(0xffffffffu, finite, o));
    const int s = exponent_byte(finite, format);
    const float f = down(s);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2] |= code_special(v[i] * f, format) << (8 * (i & 3));
    codes = make_uint2(w[0], w[1]);
    return s;
  }
  const int s = exponent_byte(most, format);
  const float f = down(s);
  codes.x = code2(v[0] * f, v[1] * f, format) | code2(v[2] * f, v[3] * f, format) << 16;
  codes.y = code2(v[4] * f, v[5] * f, format) | code2(v[6] * f, v[7] * f, format) << 16;
  return s;
}

// Eight neighbouring elements of a row: `vector` - the address is a multiple of their bytes (or of 16) and all eight exist; else the
// first `count`, zeros behind them.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int count, bool vector, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, int count, bool vector, float (&v)[8]) {
  if (vector && count >= 8) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < count ? p[i] : 0.f;
  }
}
template <>
__device__ __forceinline__ void load8<bf16>(const bf16* p, int count, bool vector, float (&v)[8]) {
  if (vector && count >= 8) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < count ? __bfloat162float(p[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int count, bool vector, const float (&v)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* p, int count, bool vector, const float (&v)[8]) {
  if (vector && count >= 8) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < count) p[i] = v[i];
  }
}
template <>
__device__ __forceinline__ void store8<bf16>(bf16* p, int count, bool vector, const float (&v)[8]) {
  if (vector && count >= 8) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < count) p[i] = __float2bfloat16_rn(v[i]);
  }
}

// A matrix as the kernels take it.
struct Matrix {
  uint8_t* codes;
  uint8_t* exponents;
  int64_t rows, tiles, pitch;
  int channels, format;
};
static inline Matrix matrix(const lf_float8_matrix& m) {
  return {(uint8_t*)m.codes, (uint8_t*)m.exponents, m.rows, row_tiles(m.rows), pitch(m.channels), m.channels, m.format};
}
// Codes and exponent of eight channels from `first`, all of which lie in the row's pitch; lanes whose `lead` is set write the exponent.
__device__ __forceinline__ void put8(const Matrix& m, int64_t row, int first, uint2 codes, int s, bool lead) {
  if (first < m.pitch) *reinterpret_cast<uint2*>(m.codes + row * m.pitch + first) = codes;
  if (lead) {
    // a row of one block writes its whole word: the words of a tile fill its sectors
    uint8_t* e = m.exponents + exponent_at(row, first / kBlock, m.tiles);
    if (m.channels <= kBlock) *reinterpret_cast<uint32_t*>(e) = 0x01010100u | (uint32_t)s;
    else *e = (uint8_t)s;
  }
}

}  // namespace f8
