// The 8-bit form of a matrix (lf_float8_matrix): codes in rows of whole 16-byte groups, and for every 128 consecutive channels of
// a row (of a weight: 128 x 128 elements) one power of two.
//
// amax = the largest finite magnitude of the block = m 2^p, 1 <= m < 2.  The largest finite code is 1.75 2^8 (e4m3) or 1.75 2^15 (e5m2), so
// the least power of two that brings amax to it is 2^(p - 8), or 2^(p - 7) where m > 1.75: the exponent field of amax less 8, plus a
// carry out of the mantissa.  It is kept as that biased byte, at least 1 (2^-126, the least normal number).  Scaling by it
// rounds nothing, so a code is one rounding of the value, and a decoded value (at most four significant bits) is exact in float32, and in bf16 down to its least step 2^-133 (powers
// of two below 2^-124, e5m2 2^-117, have codes beneath it).
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
// A result's memory is apart from an operand's: its first blocks store while others still read.
lf_status lf_float8_apart(lf_context* ctx, const char* what, const void* out, uint64_t bytes, const void* operand, uint64_t operand_bytes);
lf_status lf_float8_apart(lf_context* ctx, const char* what, const void* out, uint64_t bytes, const lf_float8_matrix& operand);
lf_status lf_float8_done(lf_context* ctx, lf_result* r, int launches);

namespace f8 {

constexpr int kBlock = 128;      // channels that share an exponent

__host__ __device__ inline int64_t pitch(int channels) { return ((int64_t)channels + 15) & ~(int64_t)15; }
__host__ __device__ inline int blocks(int channels) { return (int)(((uint32_t)channels + (kBlock - 1)) / kBlock); }
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

constexpr float kInfinity = __builtin_huge_valf();

// Formats are template arguments where codes are made and read, behind one branch for many codes: chosen code by code they cost both conversions.
// Two codes, x in the low byte.  `scaled` values are within the format's range (or not finite: see code_special).
template <int FORMAT>
__device__ __forceinline__ uint32_t code2(float x, float y) {
  return __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, FORMAT == LF_FLOAT8_E4M3 ? __NV_E4M3 : __NV_E5M2);
}
// One code of a value that may be infinite: e4m3 has no infinity, so that it becomes NaN and is not lost in a finite code.
template <int FORMAT>
__device__ __forceinline__ uint32_t code_special(float v) {
  if (fabsf(v) == kInfinity) return (__float_as_uint(v) >> 24 & 0x80u) | (FORMAT == LF_FLOAT8_E4M3 ? 0x7fu : 0x7cu);
  return code2<FORMAT>(v, 0.f) & 0xffu;
}
template <int FORMAT>
__device__ __forceinline__ uint32_t half2_of(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, FORMAT == LF_FLOAT8_E4M3 ? __NV_E4M3 : __NV_E5M2);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <int FORMAT>
__device__ __forceinline__ float2 decode2(uint32_t two) {
  const uint32_t h = half2_of<FORMAT>(two);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// A lane's share of a row is sixteen neighbouring channels, as eight pairs for the two-at-once float32 instructions: eight lanes hold a
// block.  (Eight channels a lane: the shuffles of a block's maximum and of a row's sums cost twice as much an element, and codes leave
// in pieces of eight bytes; LayerNorm + checkpoint of 147456 x 128 took 42 us then, its backward pass 48, encoding 1 Mi x 128 121.)
constexpr int kShare = 16;
struct Share { float2 v[kShare / 2]; };

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 y;
  asm("{\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%2, %3};\n\t"
      "mov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 a, a, b;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "=f"(y.x), "=f"(y.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return y;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// What a lane loads of a row, still as it lies in memory.
template <typename T>
struct Raw { uint32_t w[kShare * sizeof(T) / 4]; };

// How rows can be accessed: 32 bytes at a time, 16, or element by element.
enum { kElements = 0, kSixteen = 1, kThirtyTwo = 2 };
static inline int row_access(const void* p, int c, int dtype) {
  const int64_t bytes = (int64_t)c * (dtype == LF_DTYPE_BF16 ? 2 : 4);
  return ((uintptr_t)p & 31) == 0 && bytes % 32 == 0 ? kThirtyTwo : ((uintptr_t)p & 15) == 0 && bytes % 16 == 0 ? kSixteen : kElements;
}

// Rows that no 16-byte access divides go through shared memory: neighbouring lanes load neighbouring elements, and each takes its sixteen from there when
// it needs them (lane by lane, sixteen elements each, a warp's load touches sixteen lines instead of one).  A warp's room, in float32; every
// 32 elements are followed by four of padding, so that eight lanes' 16-byte pieces lie in different banks.
constexpr int kRoom = 32 * kShare / 32 * 36;
__device__ __forceinline__ int room_at(int e) { return e + (e >> 5) * 4; }

// The lane's part of a row (p: its first channel, `left` channels from there to the row's end; channels behind it read as zero, as
// does a row that is not `live`).  LANES neighbouring lanes have neighbouring parts.  All lanes of a warp call these three.
template <typename T, int LANES>
__device__ __forceinline__ void load16(Raw<T>& r, const T* p, int left, bool live, int access) {
  constexpr int kWords = kShare * sizeof(T) / 4;
  const int count = live ? left : 0;
  if (access == kElements) {      // element j * LANES + lane of the group's
    const int lane = threadIdx.x % LANES, all = live ? left + lane * kShare : 0;
    const T* from = p - lane * kShare;
    if (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < kShare; ++j) r.w[j % kWords] = j * LANES + lane < all ? reinterpret_cast<const uint32_t*>(from)[j * LANES + lane] : 0u;
    } else {
#pragma unroll
      for (int j = 0; j < kShare; j += 2)
        r.w[j / 2] = (j * LANES + lane < all ? (uint32_t)reinterpret_cast<const uint16_t*>(from)[j * LANES + lane] : 0u) |
                     ((j + 1) * LANES + lane < all ? (uint32_t)reinterpret_cast<const uint16_t*>(from)[(j + 1) * LANES + lane] << 16 : 0u);
    }
  } else if (count >= kShare && access == kThirtyTwo) {
#pragma unroll
    for (int i = 0; i < kWords; i += 8)
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(r.w[i]), "=r"(r.w[i + 1]), "=r"(r.w[i + 2]), "=r"(r.w[i + 3]), "=r"(r.w[i + 4]), "=r"(r.w[i + 5]), "=r"(r.w[i + 6]), "=r"(r.w[i + 7])
                   : "l"(reinterpret_cast<const uint32_t*>(p) + i)
                   : "memory");
  } else {      // rows are whole 16-byte pieces
    constexpr int kPiece = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (i / 4 * kPiece < count) u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
      r.w[i] = u.x; r.w[i + 1] = u.y; r.w[i + 2] = u.z; r.w[i + 3] = u.w;
    }
  }
}
template <typename T>
__device__ __forceinline__ Share unpack_in_order(const Raw<T>& r) {
  constexpr int kWords = kShare * sizeof(T) / 4;
  Share s;
#pragma unroll
  for (int i = 0; i < kShare / 2; ++i) {
    if (sizeof(T) == 4) s.v[i] = make_float2(__uint_as_float(r.w[(2 * i) % kWords]), __uint_as_float(r.w[(2 * i + 1) % kWords]));
    else s.v[i] = make_float2(__uint_as_float(r.w[i] << 16), __uint_as_float(r.w[i] & 0xffff0000u));
  }
  return s;
}
template <typename T, int LANES>
__device__ __forceinline__ Share unpack(const Raw<T>& r, int access, float* room) {
  const Share s = unpack_in_order(r);
  if (access != kElements) return s;
  // (LANES <= 32 divides 32, and so do the groups' parts of the room)
  const int lane = threadIdx.x % LANES, base = (threadIdx.x & 31) / LANES * LANES * kShare;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < kShare; ++j) room[room_at(base + j * LANES + lane)] = j & 1 ? s.v[j / 2].y : s.v[j / 2].x;
  __syncwarp();
  Share t;
#pragma unroll
  for (int i = 0; i < kShare; i += 4) {
    const float4 f = *reinterpret_cast<const float4*>(&room[room_at(base + lane * kShare + i)]);
    t.v[i / 2] = make_float2(f.x, f.y);
    t.v[i / 2 + 1] = make_float2(f.z, f.w);
  }
  return t;
}
template <typename T, int LANES>
__device__ __forceinline__ void store16(T* p, int left, bool live, int access, const Share& s, float* room) {
  constexpr int kWords = kShare * sizeof(T) / 4;
  const int count = live ? left : 0;
  if (access == kElements) {
    const int lane = threadIdx.x % LANES, base = (threadIdx.x & 31) / LANES * LANES * kShare, all = live ? left + lane * kShare : 0;
    T* to = p - lane * kShare;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kShare; i += 4)
      *reinterpret_cast<float4*>(&room[room_at(base + lane * kShare + i)]) = make_float4(s.v[i / 2].x, s.v[i / 2].y, s.v[i / 2 + 1].x, s.v[i / 2 + 1].y);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kShare; ++j) {
      const float v = room[room_at(base + j * LANES + lane)];
      if (j * LANES + lane < all) {
        if (sizeof(T) == 4) reinterpret_cast<float*>(to)[j * LANES + lane] = v;
        else reinterpret_cast<bf16*>(to)[j * LANES + lane] = __float2bfloat16_rn(v);
      }
    }
    return;
  }
  uint32_t w[kWords];
#pragma unroll
  for (int i = 0; i < kShare / 2; ++i) {
    if (sizeof(T) == 4) { w[(2 * i) % kWords] = __float_as_uint(s.v[i].x); w[(2 * i + 1) % kWords] = __float_as_uint(s.v[i].y); }
    else {
      const __nv_bfloat162 t = __floats2bfloat162_rn(s.v[i].x, s.v[i].y);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
  }
  if (count >= kShare && access == kThirtyTwo) {
#pragma unroll
    for (int i = 0; i < kWords; i += 8)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<uint32_t*>(p) + i), "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]),
                   "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7])
                   : "memory");
  } else {
    constexpr int kPiece = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < kWords; i += 4)
      if (i / 4 * kPiece < count) *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(p) + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  }
}

// A lane's sixteen codes -> values, without their power of two
template <int FORMAT>
__device__ __forceinline__ Share decode16_as(uint4 codes) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
  Share s;
#pragma unroll
  for (int i = 0; i < kShare / 2; ++i) s.v[i] = decode2<FORMAT>(w[i >> 1] >> (16 * (i & 1)) & 0xffffu);
  return s;
}
__device__ __forceinline__ Share decode16(uint4 codes, int format) {
  return format == LF_FLOAT8_E4M3 ? decode16_as<LF_FLOAT8_E4M3>(codes) : decode16_as<LF_FLOAT8_E5M2>(codes);
}

// A lane's codes of x over the power of two of the byte s; `special`: infinities may be among the values.
template <int FORMAT>
__device__ __forceinline__ uint4 code16_as(const Share& x, int s, bool special) {
  const float2 f = both(down(s));
  uint32_t w[4];
  if (special) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = code_special<FORMAT>(x.v[2 * i].x * f.x) | code_special<FORMAT>(x.v[2 * i].y * f.x) << 8 | code_special<FORMAT>(x.v[2 * i + 1].x * f.x) << 16 |
             code_special<FORMAT>(x.v[2 * i + 1].y * f.x) << 24;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = mul2(x.v[2 * i], f), b = mul2(x.v[2 * i + 1], f);
      w[i] = code2<FORMAT>(a.x, a.y) | code2<FORMAT>(b.x, b.y) << 16;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 code16(const Share& x, int s, int format, bool special) {
  return format == LF_FLOAT8_E4M3 ? code16_as<LF_FLOAT8_E4M3>(x, s, special) : code16_as<LF_FLOAT8_E5M2>(x, s, special);
}
// The largest magnitude of a lane's values, NaN left out; of its finite ones.
__device__ __forceinline__ float most_of(const Share& x) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < kShare / 2; ++i) most = fmaxf(most, fmaxf(fabsf(x.v[i].x), fabsf(x.v[i].y)));
  return most;
}
__device__ __forceinline__ float most_finite_of(const Share& x) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < kShare / 2; ++i) {
    if (fabsf(x.v[i].x) < kInfinity) most = fmaxf(most, fabsf(x.v[i].x));
    if (fabsf(x.v[i].y) < kInfinity) most = fmaxf(most, fabsf(x.v[i].y));
  }
  return most;
}

// The exponent byte of the block that LANES neighbouring lanes hold (eight lanes, or all of a narrower row's), and the lane's codes.  All lanes of
// the warp call it.
template <int LANES>
__device__ __forceinline__ int encode16(const Share& x, int format, uint4& codes) {
  float most = most_of(x);
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  const bool special = __any_sync(0xffffffffu, most == kInfinity);
  if (special) {
    most = most_finite_of(x);
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  const int s = exponent_byte(__float_as_uint(most), format);
  codes = code16(x, s, format, special);
  return s;
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
// A lane's codes (its channels from `first` on) and, from the lane that leads its block, the exponent.
__device__ __forceinline__ void put16(const Matrix& m, int64_t row, int first, uint4 codes, int s) {
  if (first >= m.channels) return;
  *reinterpret_cast<uint4*>(m.codes + row * m.pitch + first) = codes;
  if ((first & (kBlock - 1)) == 0) {
    uint8_t* e = m.exponents + exponent_at(row, first / kBlock, m.tiles);
    if (m.channels <= kBlock) *reinterpret_cast<uint32_t*>(e) = 0x01010100u | (uint32_t)s;      // the only block of the row: its whole word
    else *e = (uint8_t)s;
  }
}

}  // namespace f8
