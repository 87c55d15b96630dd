// The weights' gradient of a projection from the 8-bit form of its input: dW[n][k] = sum over rows m of dy[m][n] x8[m][k], and
// dbias[n] = sum of dy[m][n], float32.
//
// The sum runs over the rows, whose exponents differ, so the exponent has to be in the operand: codes become bf16 values on the way to
// shared memory (exactly: four significant bits times a power of two), and tcgen05.mma of kind f16 multiplies them with dy, which is bf16
// or comes from codes the same way.  Both operands lie with the summed index outside (MN-major), as they are in memory; nothing is transposed.
// The column sums of dy are added up by two warps of the first column tile's blocks, from the operand in shared memory.  (By the converting warps: 262144 x 128 -> 512
// 66 -> 88 us, from codes 78 -> 175.)
//
// The tensor core's additions to an accumulator truncate: their error grows with how many there are (one for 16 rows).  So all of the 512 columns of tensor
// memory are accumulators that take steps in turn (two of 256 channels, or four of 128, for one block of outputs), added up in registers at the end, and
// a split has 4096 rows at most (more only beyond 65535 such splits).
//
// Products are dW's n x k in tiles of 128 x 256 or 256 x 256 over all rows; there are few tiles and many rows, so the rows are split over as many
// blocks as the GPU has room for, each writes its float32 partial tile, and a second kernel adds them in order.
//
// What bounds it beside the loads is shared memory: of a step of 64 rows and 128 outputs, 128 KB pass through it (codes in and out, operands in, both operands
// to the tensor core), 1000 cycles for 512 of products.  Two blocks of 128 outputs share x's conversion and operand: 96 KB a block.  65536 x 512 -> 128: 17.5 to
// 20 us and 7 to join; 262144 x 128 -> 512: 67 (87 with one block); 4096 x 4096 -> 4096: 145 (216), 950 TFLOP/s.
#include <cuda.h>

#include <algorithm>

#include "float8.cuh"
#include "tc05.cuh"
#include "tc_kernels.cuh"

namespace tc {

using namespace tc05;

lf_status make_map_bytes(lf_context* ctx, CUtensorMap* map, const void* base, uint64_t width, uint64_t rows, uint64_t pitch, uint32_t box_rows);
lf_status make_map_rows(lf_context* ctx, CUtensorMap* map, const void* base, bool f32, uint64_t width, uint64_t rows, uint32_t box_rows, bool narrow = false);
lf_status make_map_f32_any(lf_context* ctx, CUtensorMap* map, const void* base, const uint64_t (&dims)[3], const uint64_t (&strides)[2], const uint32_t (&box)[3]);

constexpr int WG_BN = 128, WG_BK = 256, WG_ROWS = 64;      // outputs of a block (a tile has one or two), channels, rows of a step
constexpr int WG_A_BYTES = WG_BN * WG_ROWS * 2, WG_B_BYTES = WG_BK * WG_ROWS * 2;
constexpr int WG_CODES = WG_BK * WG_ROWS, WG_DY_CODES = WG_BN * WG_ROWS;
constexpr int WG_OPERANDS = 2;                             // converted steps
constexpr int WG_CONVERT = 16;                             // warps that convert, and store the tile
constexpr int WG_SUMS = 2;                                 // warps that add up dy's columns
constexpr int WG_THREADS = 64 + 32 * (WG_CONVERT + WG_SUMS);
constexpr int WG_EXPONENTS = 2 * 512;
// [dy: a ring of bf16 operands, or two that are converted and a ring of its codes][ring of x's codes][x's operands][exponents]
template <int NB>
struct GradientShape {
  static constexpr int a_bytes = NB * WG_A_BYTES, dy_codes = NB * WG_DY_CODES;
  static constexpr int ring = NB == 1 ? 4 : 3, ring_codes = NB == 1 ? 4 : 2;      // steps on their way from memory; of a dy in codes
  static constexpr int dy = ring * a_bytes;
  static constexpr int smem = dy + ring * (WG_CODES + WG_EXPONENTS) + WG_OPERANDS * WG_B_BYTES + 256 + 1024;
  static_assert(WG_OPERANDS * a_bytes + ring_codes * dy_codes <= dy && WG_CONVERT * 8192 <= dy + ring * WG_CODES, "");
};

struct GradientParams {
  int m, n, k;
  int steps, per_split;          // steps of 64 rows in all, and of a split
  const bf16* dy;
  f8::Matrix dy8, x;
  float* out;                    // [split][n][ld] partial tiles, or dW itself
  float* bias;                   // [split][n]
  int64_t ld, split_stride, bias_stride;
  int vector_out;
  Status* status;
};

__device__ __forceinline__ uint32_t bf16x2_bits(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Sixteen neighbouring codes of one row -> two 16-byte pieces of bf16.
template <int FORMAT>
__device__ __forceinline__ void convert16_as(uint4 codes, int s, uint4 (&out)[2]) {
  const f8::Share v = f8::decode16_as<FORMAT>(codes);
  const float2 factor = f8::both(f8::up(s));
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 t = f8::mul2(v.v[i], factor);
    o[i] = bf16x2_bits(t.x, t.y);
  }
  out[0] = make_uint4(o[0], o[1], o[2], o[3]);
  out[1] = make_uint4(o[4], o[5], o[6], o[7]);
}
__device__ __forceinline__ void convert16(uint4 codes, int s, int format, uint4 (&out)[2]) {
  if (format == LF_FLOAT8_E4M3) convert16_as<LF_FLOAT8_E4M3>(codes, s, out); else convert16_as<LF_FLOAT8_E5M2>(codes, s, out);
}

// Sixteen neighbouring elements from `first` on of a bf16 tensor of `all`, wherever they start: the aligned 8-byte words that they lie in, and element by element (`count` of
// them) where those would reach beyond the tensor's ends.  (By elements alone a warp's load touched 32 sectors: 65536 x 256 -> 1283 took 164 us,
// now 99, and 100000 x 300 -> 300 152, now 93.)
__device__ __forceinline__ void fetch_unaligned(uint2 (&raw)[5], const bf16* tensor, int64_t all, int64_t first, int count) {
#pragma unroll
  for (int i = 0; i < 5; ++i) raw[i] = make_uint2(0, 0);
  if (count <= 0) return;
  const uintptr_t base = reinterpret_cast<uintptr_t>(tensor), at = base + 2 * first, from = at & ~(uintptr_t)7;
  if (from >= base && from + 40 <= base + 2 * all) {
#pragma unroll
    for (int i = 0; i < 5; ++i) raw[i] = *reinterpret_cast<const uint2*>(from + 8 * i);
  } else {
    const int skip = (int)(at - from) / 2;
    auto half = [&](int h) { return h >= skip && h < skip + count ? (uint32_t)*reinterpret_cast<const uint16_t*>(from + 2 * h) : 0u; };
#pragma unroll
    for (int i = 0; i < 5; ++i) raw[i] = make_uint2(half(4 * i) | half(4 * i + 1) << 16, half(4 * i + 2) | half(4 * i + 3) << 16);
  }
}
// The elements in their places, zeros from `count` on.
__device__ __forceinline__ void place_unaligned(const uint2 (&raw)[5], const bf16* tensor, int64_t first, int count, uint4 (&out)[2]) {
  const uint32_t off = ((uint32_t)reinterpret_cast<uintptr_t>(tensor) + 2 * (uint32_t)first) & 7;      // bytes in front of the first
  uint32_t w[9], o[8];
#pragma unroll
  for (int i = 0; i < 9; ++i) {
    const uint32_t near = i & 1 ? raw[i / 2].y : raw[i / 2].x, next = i & 1 ? raw[i / 2 + 1].x : raw[i / 2].y;
    w[i] = off & 4 ? next : near;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = __funnelshift_r(w[i], w[i + 1], (off & 2) * 8);
  if (count < 16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 2 * i + 1 < count ? o[i] : 2 * i < count ? o[i] & 0xffffu : 0u;
  }
  out[0] = make_uint4(o[0], o[1], o[2], o[3]);
  out[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

// The place of a piece of eight columns in an MN-major operand: blocks of 64 columns, rows of 128 bytes, 128-byte swizzle.
__device__ __forceinline__ uint32_t piece_at(int row, int piece) { return (piece >> 3) * (WG_ROWS * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4); }

// Warp roles: 0 = loads (dy, x's codes, the exponents that belong to them), 1 = MMA issuer (owns TMEM), 2..17 = conversion, then the tile's stores, 18 and 19 =
// dy's sums.
// MODE: how dy comes, by TMA (0), as bf16 rows that no 16-byte access divides (1), as codes (2).
template <int NB, int MODE>
__global__ void __launch_bounds__(WG_THREADS, 1)
float8_gradient_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapO,
                       const GradientParams p) {
  using S = GradientShape<NB>;
  constexpr int WG_RING = S::ring;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* dy_s = align_shared(smem_raw);
  uint8_t* dy_codes = dy_s + WG_OPERANDS * S::a_bytes;
  uint8_t* x_codes = dy_s + S::dy;
  uint8_t* x_s = x_codes + WG_RING * WG_CODES;
  uint8_t* exponents = x_s + WG_OPERANDS * WG_B_BYTES;
  const int ring = MODE == 2 ? S::ring_codes : S::ring;
  uint64_t* loaded = reinterpret_cast<uint64_t*>(exponents + WG_RING * WG_EXPONENTS);      // [RING] codes, exponents and a bf16 dy are here
  uint64_t* taken = loaded + WG_RING;                              // [RING] their codes are read (and a bf16 dy multiplied)
  uint64_t* full = taken + WG_RING;                                // [OPERANDS]
  uint64_t* empty = full + WG_OPERANDS;
  uint64_t* done = empty + WG_OPERANDS;                            // every product, and every step's sums
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.y * (NB * WG_BN), k0 = blockIdx.x * WG_BK, split = blockIdx.z;
  const int first = split * p.per_split, last = min(first + p.per_split, p.steps);
  const int columns = min(WG_BK, p.k - k0);
  const int groups = (columns + 63) / 64;                   // 64-channel blocks of x that exist
  const bool sums = blockIdx.x == 0 && p.bias;              // dy's, too
  const int wide = columns > 128 ? 256 : 128, accumulators = 512 / (NB * wide);

  if (threadIdx.x == 0) {
    for (int s = 0; s < WG_RING; ++s) { mbar_init(&loaded[s], 1); mbar_init(&taken[s], WG_CONVERT + (MODE == 0 ? 1 + (sums ? WG_SUMS : 0) : 0)); }
    for (int s = 0; s < WG_OPERANDS; ++s) { mbar_init(&full[s], WG_CONVERT); mbar_init(&empty[s], 1 + (MODE != 0 && sums ? WG_SUMS : 0)); }
    mbar_init(done, 1 + (sums ? WG_SUMS : 0));
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  lf_chain();

  if (warp == 0) {
    if (lane == 0) {
      if (MODE != 1) prefetch_tensormap(&mapA);
      prefetch_tensormap(&mapX);
      const uint32_t x_boxes = columns > 128 ? 2 : 1;
      const uint32_t bytes = x_boxes * (WG_CODES / 2) + 512 + (MODE == 0 ? S::a_bytes : MODE == 2 ? S::dy_codes + 512 : 0);
      const uint8_t* ex = p.x.exponents + (int64_t)(k0 >> 9) * p.x.tiles * 512;
      const uint8_t* ey = p.dy8.exponents + (int64_t)(n0 >> 9) * p.dy8.tiles * 512;
      int stage = 0; uint32_t phase = 0;
      for (int t = first; t < last; ++t) {
        if (!mbar_wait(&taken[stage], phase ^ 1, abort_flag, p.status, 131)) break;
        uint64_t* bar = &loaded[stage];
        mbar_expect_tx(bar, bytes);
        for (uint32_t i = 0; i < x_boxes; ++i) tma_load_3d(x_codes + stage * WG_CODES + i * (WG_CODES / 2), &mapX, bar, k0 + i * 128, t * WG_ROWS, 0);
        bulk_load(exponents + stage * WG_EXPONENTS, ex + (int64_t)(t >> 1) * 512, 512, bar);
        if (MODE == 0) {
#pragma unroll
          for (int i = 0; i < 2 * NB; ++i) tma_load_3d(dy_s + stage * S::a_bytes + i * (WG_A_BYTES / 2), &mapA, bar, n0 + 64 * i, t * WG_ROWS, 0);
        } else if (MODE == 2) {
#pragma unroll
          for (int i = 0; i < NB; ++i) tma_load_3d(dy_codes + stage * S::dy_codes + i * WG_DY_CODES, &mapA, bar, n0 + 128 * i, t * WG_ROWS, 0);
          bulk_load(exponents + stage * WG_EXPONENTS + 512, ey + (int64_t)(t >> 1) * 512, 512, bar);
        }
        if (++stage == ring) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // (the whole warp walks and waits, so that what the instructions take stays in uniform registers; one lane issues)
    int slot = 0, stage = 0, acc = 0; uint32_t phase = 0, ring_phase = 0;
    constexpr uint32_t both = (1u << 7) | (1u << 10);      // bf16 operands
    const uint32_t idesc = make_idesc_f16(WG_BN, groups * 64, 1, 1) | both;
    const uint64_t a_first = make_smem_desc(smem_u32(dy_s), WG_ROWS * 128, 1024), b_first = make_smem_desc(smem_u32(x_s), WG_ROWS * 128, 1024);
    for (int t = first; t < last; ++t) {
      // (an expired wait ends the loop for all lanes alike)
      if (!__all_sync(0xffffffffu, mbar_wait(&full[slot], phase, abort_flag, p.status, 132))) break;
      if (MODE == 0 && !__all_sync(0xffffffffu, mbar_wait(&loaded[stage], ring_phase, abort_flag, p.status, 136))) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t a = a_first + (uint32_t)((MODE == 0 ? stage : slot) * (S::a_bytes >> 4)), b = b_first + (uint32_t)(slot * (WG_B_BYTES >> 4));
#pragma unroll
        for (int kk = 0; kk < WG_ROWS / 16; ++kk) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            umma_f16(tmem_base + (acc * NB + nb) * wide, a + kk * 128 + nb * (WG_A_BYTES >> 4), b + kk * 128, idesc, (t - first >= accumulators || kk != 0) ? 1u : 0u);
        }
        umma_commit(&empty[slot]);
        if (MODE == 0) umma_commit(&taken[stage]);
        if (t + 1 == last) umma_commit(done);
      }
      __syncwarp();
      if (++acc == accumulators) acc = 0;
      if (++slot == WG_OPERANDS) { slot = 0; phase ^= 1; }
      if (++stage == ring) { stage = 0; ring_phase ^= 1; }
    }
  } else if (warp >= 2 + WG_CONVERT) {
    // A warp has NB blocks of 64 outputs: eight columns a lane, every fourth row.
    if (sums) {
      const int w = warp - 2 - WG_CONVERT, piece = lane & 7, r0 = lane >> 3;
      float2 total[NB][4];
#pragma unroll
      for (int i = 0; i < NB * 4; ++i) total[i / 4][i % 4] = make_float2(0.f, 0.f);
      int slot = 0, stage = 0; uint32_t phase = 0, ring_phase = 0;
      for (int t = first; t < last; ++t) {
        const bool here = MODE == 0 ? mbar_wait(&loaded[stage], ring_phase, abort_flag, p.status, 137) : mbar_wait(&full[slot], phase, abort_flag, p.status, 138);
        if (!__all_sync(0xffffffffu, here)) break;
        const uint8_t* sA = dy_s + (MODE == 0 ? stage : slot) * S::a_bytes;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll 8
          for (int r = r0; r < WG_ROWS; r += 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(sA + piece_at(r, (w * NB + b) * 8 + piece));
            const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) total[b][i] = add2(total[b][i], make_float2(__uint_as_float(v[i] << 16), __uint_as_float(v[i] & 0xffff0000u)));
          }
        __syncwarp();
        if (lane == 0) mbar_arrive(MODE == 0 ? &taken[stage] : &empty[slot]);
        if (++slot == WG_OPERANDS) { slot = 0; phase ^= 1; }
        if (++stage == ring) { stage = 0; ring_phase ^= 1; }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(done);      // (the last steps' slots are not filled again: nothing else waits for these reads of them)
#pragma unroll
      for (int i = 0; i < NB * 4; ++i) {
        float2 v = total[i / 4][i % 4];
#pragma unroll
        for (int o = 8; o < 32; o *= 2) { v.x += __shfl_xor_sync(0xffffffffu, v.x, o); v.y += __shfl_xor_sync(0xffffffffu, v.y, o); }
        const int n = n0 + (w * NB + i / 4) * 64 + piece * 8 + i % 4 * 2;
        float* to = p.bias + split * p.bias_stride + n;
        if (r0 == 0 && n < p.n) to[0] = v.x;
        if (r0 == 0 && n + 1 < p.n) to[1] = v.y;
      }
    }
  } else {
    // Rows of a step: x has 16 pieces of 16 channels, dy 8 of 16 outputs; neighbouring lanes take neighbouring pieces of a row.
    const int thread = threadIdx.x - 64;
    constexpr int kUnits = WG_ROWS * 16 / (32 * WG_CONVERT);      // of x a thread
    const int xp = thread & 15, xr = thread >> 4;                 // piece, first row (rows xr + 32 u)
    constexpr int kPerRow = 8 * NB, kStep = 32 * WG_CONVERT / kPerRow;      // of dy: NB units a thread, rows yr + kStep u
    const int yp = thread % kPerRow, yr = thread / kPerRow;
    const int ych = n0 + yp * 16;
    const int x_block = (k0 >> 7 & 3) + (xp >> 3), y_block = (n0 >> 7 & 3) + (yp >> 3);
    const bool x_any = xp < groups * 4, x_here = xp * 16 < (columns > 128 ? 256 : 128);
    // MODE 1: the next step's units, each as the five 8-byte words that its sixteen elements lie in
    uint2 ahead[MODE == 1 ? NB : 1][5];
    auto fetch = [&](int t) {
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        const int64_t row = (int64_t)t * WG_ROWS + yr + kStep * u;
        fetch_unaligned(ahead[u], p.dy, (int64_t)p.m * p.n, row * p.n + ych, row < p.m ? min(16, p.n - ych) : 0);
      }
    };
    int slot = 0, stage = 0; uint32_t phase = 0, ring_phase = 0;
    bool ok = true;
    if (MODE == 1) fetch(first);
    for (int t = first; t < last; ++t) {
      if (!__all_sync(0xffffffffu, mbar_wait(&loaded[stage], ring_phase, abort_flag, p.status, 135))) { ok = false; break; }
      uint4 codes[kUnits], dy_unit[NB][2];
      int s[kUnits], sy[NB];
      const uint8_t* e = exponents + stage * WG_EXPONENTS + (t & 1) * 8;      // (rows 64 .. 127 of a tile: words 2 and 3)
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {      // row xr + 32 u of the step
        codes[u] = make_uint4(0, 0, 0, 0);
        if (x_here) codes[u] = *reinterpret_cast<const uint4*>(x_codes + stage * WG_CODES + (xp >> 3) * (WG_CODES / 2) + swizzle128_offset(xr + 32 * u, xp & 7));
        s[u] = t * WG_ROWS + xr + 32 * u < p.m ? e[xr * 16 + u * 4 + x_block] : 1;      // (bytes behind the last row are of no account)
      }
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        const int r = yr + kStep * u;
        if (MODE == 2) {
          dy_unit[u][0] = *reinterpret_cast<const uint4*>(dy_codes + stage * S::dy_codes + (yp >> 3) * WG_DY_CODES + swizzle128_offset(r, yp & 7));
          sy[u] = t * WG_ROWS + r < p.m ? e[512 + (r & 31) * 16 + (r >> 5) * 4 + y_block] : 1;
        } else if (MODE == 1) {
          const int64_t row = (int64_t)t * WG_ROWS + r;
          place_unaligned(ahead[u], p.dy, row * p.n + ych, row < p.m ? min(16, p.n - ych) : 0, dy_unit[u]);
        }
      }
      if (MODE == 1 && t + 1 < last) fetch(t + 1);
      __syncwarp();
      if (lane == 0) mbar_arrive(&taken[stage]);      // the codes are in registers
      if (!__all_sync(0xffffffffu, mbar_wait(&empty[slot], phase ^ 1, abort_flag, p.status, 133))) { ok = false; break; }
      uint8_t* sA = dy_s + slot * S::a_bytes;
      uint8_t* sB = x_s + slot * WG_B_BYTES;
      // (odd blocks of 64 columns store their second piece first: eight lanes then fill eight different 16-byte columns of the banks)
      if (x_any) {
        const int swap = xp >> 2 & 1;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          uint4 v[2];
          convert16(codes[u], s[u], p.x.format, v);
          const int row = xr + 32 * u;
          *reinterpret_cast<uint4*>(sB + piece_at(row, xp * 2 + swap)) = swap ? v[1] : v[0];
          *reinterpret_cast<uint4*>(sB + piece_at(row, xp * 2 + 1 - swap)) = swap ? v[0] : v[1];
        }
      }
      if (MODE != 0) {
        const int swap = yp >> 2 & 1;
#pragma unroll
        for (int u = 0; u < NB; ++u) {
          uint4 v[2] = {dy_unit[u][0], dy_unit[u][1]};
          if (MODE == 2) convert16(dy_unit[u][0], sy[u], p.dy8.format, v);
          const int row = yr + kStep * u;
          *reinterpret_cast<uint4*>(sA + piece_at(row, yp * 2 + swap)) = swap ? v[1] : v[0];
          *reinterpret_cast<uint4*>(sA + piece_at(row, yp * 2 + 1 - swap)) = swap ? v[0] : v[1];
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[slot]);
      if (++slot == WG_OPERANDS) { slot = 0; phase ^= 1; }
      if (++stage == ring) { stage = 0; ring_phase ^= 1; }
    }
    // The tile: 16 warps, 64 columns of a lane quadrant each.
    ok = ok && __all_sync(0xffffffffu, mbar_wait(done, 0, abort_flag, p.status, 134));
    tc_fence_after();
    if (ok) {
      const int q = warp & 3, part = (warp - 2) >> 2, col0 = k0 + part * 64;
      uint8_t* tiles = dy_s + (warp - 2) * 8192;      // (every product is done and dy's columns are added up: the rings of dy and of x's codes are free)
      float* out = p.out + split * p.split_stride;
      const int used = min(accumulators, last - first);
#pragma unroll 1
      for (int nb = 0; nb < NB; ++nb) {
        const int row0 = n0 + nb * WG_BN + q * 32;
        const uint32_t d = tmem_base + ((uint32_t)(q * 32) << 16) + nb * wide + part * 64;
        if (row0 < p.n && col0 < p.k) {
          uint32_t r[2][32];
          tmem_ld32(d, r[0]);
          tmem_ld32(d + 32, r[1]);
          if (lane == 0) bulk_wait_read();      // the copies of the block before have read the staging rows
          __syncwarp();
          tmem_ld_wait();
          tie32(r[0]);
          tie32(r[1]);
          for (int i = 1; i < used; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint32_t more[32];
              tmem_ld32(d + i * NB * wide + half * 32, more);
              tmem_ld_wait();
              tie32(more);
#pragma unroll
              for (int c = 0; c < 32; ++c) r[half][c] = __float_as_uint(__uint_as_float(r[half][c]) + __uint_as_float(more[c]));
            }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int c0 = col0 + half * 32;
            if (c0 >= p.k) break;
            uint8_t* tile = tiles + half * 4096;
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<uint4*>(tile + swizzle128_offset(lane, c)) = make_uint4(r[half][c * 4], r[half][c * 4 + 1], r[half][c * 4 + 2], r[half][c * 4 + 3]);
            if (p.vector_out) {
              fence_async_smem();
              __syncwarp();
              if (lane == 0) { tma_store_3d(&mapO, tile, c0, row0, split); bulk_commit(); }
            } else {
              __syncwarp();
              const int rows = min(32, p.n - row0);
              for (int row = 0; row < rows; ++row)
                if (c0 + lane < p.k) out[(int64_t)(row0 + row) * p.ld + c0 + lane] = *reinterpret_cast<const float*>(tile + swizzle128_offset(row, lane >> 2) + (lane & 3) * 4);
              __syncwarp();
            }
          }
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    tc_fence_before();
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) drain_after_abort();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, 512); }
}

// dW and dbias from the splits' partial tiles, added in a fixed order: four neighbouring columns a thread, STRANDS threads of a block share the splits, eight
// loads in flight each.
template <int STRANDS>
__global__ void __launch_bounds__(256)
gradient_join_kernel(const float* partial, int ld, int64_t split_stride, int splits, int n, int k, int direct, float* out, const float* bias_partial,
                     float* bias) {
  constexpr int kColumns = 256 / STRANDS;
  __shared__ float4 s[STRANDS][kColumns];
  const int lane = threadIdx.x % kColumns, strand = threadIdx.x / kColumns;
  lf_chain();
  const uint32_t per_row = ld / 4;
  const int64_t at = (int64_t)blockIdx.x * kColumns + lane;
  const int64_t row = at / per_row;
  const int col = (int)(at - row * per_row) * 4;
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
  if (row < n) {
    const float4* from = reinterpret_cast<const float4*>(partial + row * ld + col);
    for (int i = strand; i < splits; i += 8 * STRANDS) {
      float4 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i + j * STRANDS < splits ? from[(i + j * STRANDS) * (split_stride / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 8; ++j) { t.x += v[j].x; t.y += v[j].y; t.z += v[j].z; t.w += v[j].w; }
    }
  }
  if (STRANDS > 1) {
    s[strand][lane] = t;
    __syncthreads();
    if (strand == 0) {
#pragma unroll
      for (int i = 1; i < STRANDS; ++i) { t.x += s[i][lane].x; t.y += s[i][lane].y; t.z += s[i][lane].z; t.w += s[i][lane].w; }
    }
  }
  if (strand == 0 && row < n) {
    float* to = out + row * k + col;
    if (direct) *reinterpret_cast<float4*>(to) = t;      // whole, aligned rows
    else {
      to[0] = t.x;      // (the row's last group may be in part behind its end)
      if (col + 1 < k) to[1] = t.y;
      if (col + 2 < k) to[2] = t.z;
      if (col + 3 < k) to[3] = t.w;
    }
  }
  const int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (b < n && bias) {
    float u = 0.f;
#pragma unroll 8
    for (int i = 0; i < splits; ++i) u += bias_partial[(int64_t)i * n + b];
    bias[b] = u;
  }
}

// f(NB, MODE as types)
template <typename F>
static void gradient_forms(int blocks, int mode, F f) {
  auto with = [&](auto nb) {
    if (mode == 0) f(nb, std::integral_constant<int, 0>{});
    else if (mode == 1) f(nb, std::integral_constant<int, 1>{});
    else f(nb, std::integral_constant<int, 2>{});
  };
  if (blocks == 1) with(std::integral_constant<int, 1>{}); else with(std::integral_constant<int, 2>{});
}

void configure_float8_gradient() {
  for (int i = 0; i < 6; ++i)
    gradient_forms(1 + i / 3, i % 3, [](auto nb, auto mode) {
      constexpr int NB = decltype(nb)::value;
      cudaFuncSetAttribute(float8_gradient_kernel<NB, decltype(mode)::value>, cudaFuncAttributeMaxDynamicSharedMemorySize, GradientShape<NB>::smem);
    });
}

// Blocks of outputs of a tile: two where there are two and work enough that sharing x's conversion pays (2^31 multiplications; 12000 x 128 -> 512 takes 14.2 us with
// one block and 17.0 with two, 12000 x 100 -> 2000 26.1 and 22.4).  Beside more than 128 channels they leave room for one accumulator: from 2^32 on, some 20 us.
static int gradient_blocks(int64_t m, int n, int k) { return n > WG_BN && (double)m * n * k >= (k <= 128 ? 2147483648.0 : 4294967296.0) ? 2 : 1; }

// Blocks of rows: as many as the GPU has multiprocessors for beside the tiles, with four steps of 64 rows each at least - and 64 at most: the tensor core's
// additions truncate, and 65536 x 1024 x 1024 with values of one sign was 3.5e-5 off in sums of 16384 rows (4.8e-6 in 4096).
static void gradient_plan(const lf_context* ctx, int64_t m, int n, int k, int& steps, int& splits, int& per_split) {
  constexpr int kMostSteps = 64, kMostSplits = 65535;      // (of the grid; beyond 64 * 65535 steps splits are longer)
  const int outputs = WG_BN * gradient_blocks(m, n, k);
  const int64_t tiles = (int64_t)((n + outputs - 1) / outputs) * ((k + WG_BK - 1) / WG_BK);
  steps = (int)((m + WG_ROWS - 1) / WG_ROWS);
  const int want = std::max(1, std::min((int)(ctx->sm_count / tiles), steps / 4)), least = (steps + kMostSplits - 1) / kMostSplits, most = std::max(kMostSteps, least);
  per_split = (steps + want - 1) / want;
  if (per_split > most) {      // whole turns of the blocks
    const int turns = (per_split + most - 1) / most;
    per_split = std::max(least, (steps + want * turns - 1) / (want * turns));
  }
  splits = (steps + per_split - 1) / per_split;
}
static int64_t partial_ld(int k) { return (k + 3) / 4 * 4; }
constexpr int kMostChannels = 1 << 22;      // of either side; blocks of 128 outputs then number 32768

}  // namespace tc

using namespace f8;

extern "C" {

uint64_t lf_float8_weight_gradient_workspace(const lf_context* ctx, int64_t rows, int32_t channels, int32_t out_channels) {
  if (!ctx || rows <= 0 || rows > 0x7fffff00 || channels <= 0 || out_channels <= 0 || channels > tc::kMostChannels || out_channels > tc::kMostChannels) return 0;
  int steps, splits, per_split;
  tc::gradient_plan(ctx, rows, out_channels, channels, steps, splits, per_split);
  return splits == 1 ? 0 : (uint64_t)splits * out_channels * (tc::partial_ld(channels) + 1) * sizeof(float);
}

lf_status lf_float8_weight_gradient_run(lf_context* ctx, const lf_float8_weight_gradient_desc* d, lf_result* r) {
  if (!ctx) return LF_ERR_ARGUMENT;
  if (!d || (!d->gradient && !d->encoded_gradient.codes) || !d->weight_gradient) return lf_fail(ctx, LF_ERR_ARGUMENT, "float8 weight gradient: null argument");
  if (d->gradient && d->encoded_gradient.codes) return lf_fail(ctx, LF_ERR_ARGUMENT, "float8 weight gradient: a gradient or an encoded one, not both");
  const lf_float8_matrix& x = d->activations;
  LF_TRY(lf_float8_check_rows(ctx, "float8 weight gradient", x.rows, x.channels, LF_DTYPE_BF16));
  LF_TRY(lf_float8_check_rows(ctx, "float8 weight gradient", x.rows, d->out_channels, LF_DTYPE_BF16));
  if (d->out_channels > tc::kMostChannels || x.channels > tc::kMostChannels) return lf_fail(ctx, LF_ERR_UNSUPPORTED, "float8 weight gradient: %d x %d are too many channels", d->out_channels, x.channels);
  LF_TRY(lf_float8_check(ctx, "float8 weight gradient, activations", x, x.rows, x.channels));
  if (d->encoded_gradient.codes) LF_TRY(lf_float8_check(ctx, "float8 weight gradient, gradient", d->encoded_gradient, x.rows, d->out_channels));
  const uint64_t need = lf_float8_weight_gradient_workspace(ctx, x.rows, x.channels, d->out_channels);
  if (need && (!d->workspace || d->workspace_bytes < need || !lf_aligned16(d->workspace)))
    return lf_fail(ctx, LF_ERR_ARGUMENT, "float8 weight gradient: a workspace of %llu bytes on a 16-byte boundary is needed", (unsigned long long)need);
  const lf_device_guard device(ctx);
  tc::GradientParams p{};
  p.m = (int)x.rows; p.n = d->out_channels; p.k = x.channels;
  int splits;
  tc::gradient_plan(ctx, x.rows, p.n, p.k, p.steps, splits, p.per_split);
  p.x = matrix(x);
  int mode;
  CUtensorMap ma{}, mx{}, mo{};
  LF_TRY(tc::make_map_bytes(ctx, &mx, p.x.codes, p.k, p.m, p.x.pitch, tc::WG_ROWS));
  if (d->encoded_gradient.codes) {
    mode = 2;
    p.dy8 = matrix(d->encoded_gradient);
    LF_TRY(tc::make_map_bytes(ctx, &ma, p.dy8.codes, p.n, p.m, p.dy8.pitch, tc::WG_ROWS));
  }
  else {
    p.dy = (const bf16*)d->gradient;
    mode = lf_aligned16(p.dy) && p.n % 8 == 0 ? 0 : 1;
    if (mode == 0) LF_TRY(tc::make_map_rows(ctx, &ma, p.dy, false, p.n, p.m, tc::WG_ROWS));
  }
  const bool direct = splits == 1;
  p.out = direct ? d->weight_gradient : (float*)d->workspace;
  p.ld = direct ? p.k : tc::partial_ld(p.k);
  p.split_stride = direct ? 0 : (int64_t)p.n * p.ld;
  float* bias_partial = direct ? nullptr : p.out + (int64_t)splits * p.split_stride;
  p.bias = direct ? d->bias_gradient : bias_partial;
  p.bias_stride = p.n;
  p.vector_out = lf_aligned16(p.out) && p.ld % 4 == 0;
  if (p.vector_out)
    LF_TRY(tc::make_map_f32_any(ctx, &mo, p.out, {(uint64_t)p.k, (uint64_t)p.n, (uint64_t)splits}, {(uint64_t)p.ld * 4, (uint64_t)p.ld * 4 * p.n}, {32, 32, 1}));
  p.status = (tc05::Status*)ctx->tc_status;
  lf_prof_begin(ctx, LF_KERNEL_TRIANGLE_CONTRACT);
  const int blocks = tc::gradient_blocks(x.rows, p.n, p.k), outputs = tc::WG_BN * blocks;
  const dim3 grid((p.k + tc::WG_BK - 1) / tc::WG_BK, (p.n + outputs - 1) / outputs, splits);
  tc::gradient_forms(blocks, mode, [&](auto nb, auto how) {
    constexpr int NB = decltype(nb)::value;
    lf_launch(ctx, tc::float8_gradient_kernel<NB, decltype(how)::value>, grid, tc::WG_THREADS, tc::GradientShape<NB>::smem, ma, mx, mo, p);
  });
  lf_prof_end(ctx);
  ctx->launches++;
  if (!direct) {
    lf_prof_begin(ctx, LF_KERNEL_ELEMENTWISE);
    const int64_t fours = (int64_t)p.n * (p.ld / 4);
    const int whole = p.ld == p.k && lf_aligned16(d->weight_gradient);
    auto join = [&](auto kernel, int per_block) {      // (as many blocks as the bias needs, where the rows are short)
      lf_launch(ctx, kernel, std::max(lf_ceil_div(fours, per_block), lf_ceil_div(p.n, 256)), 256, 0, p.out, (int)p.ld, p.split_stride, splits, p.n, p.k, whole,
                d->weight_gradient, bias_partial, d->bias_gradient);
    };
    if (splits > 8) join(tc::gradient_join_kernel<8>, 32); else join(tc::gradient_join_kernel<1>, 256);
    lf_prof_end(ctx);
    ctx->launches++;
  }
  return lf_float8_done(ctx, r, direct ? 1 : 2);
}

}  // extern "C"
