// The weights' gradient of a projection from the 8-bit form of its input: dW[n][k] = sum over rows m of dy[m][n] x8[m][k], and
// dbias[n] = sum of dy[m][n], float32.
//
// The sum runs over the rows, whose exponents differ, so the exponent has to be in the operand: codes become bf16 values on the way to
// shared memory (exactly: four significant bits times a power of two), and tcgen05.mma of kind f16 multiplies them with dy, which is bf16
// or comes from codes the same way.  Both operands lie with the summed index outside (MN-major), as they are in memory; nothing is transposed.
// The column sums of dy are one more product, with a tile of ones of 16 columns, on the blocks of the first column tile.
//
// Products are dW's n x k in tiles of 128 x 256 over all rows; there are few tiles and many rows, so the rows are split over as many
// blocks as the GPU has room for, each writes its float32 partial tile, and a second kernel adds them in order.
#include <cuda.h>

#include <algorithm>

#include "float8.cuh"
#include "tc05.cuh"
#include "tc_kernels.cuh"

namespace tc {

using namespace tc05;

lf_status make_map_rows(lf_context* ctx, CUtensorMap* map, const void* base, bool f32, uint64_t width, uint64_t rows, uint32_t box_rows);
lf_status make_map_f32_any(lf_context* ctx, CUtensorMap* map, const void* base, const uint64_t (&dims)[3], const uint64_t (&strides)[2], const uint32_t (&box)[3]);

constexpr int WG_BN = 128, WG_BK = 256, WG_ROWS = 64;      // outputs, channels, rows of a step
constexpr int WG_A_BYTES = WG_BN * WG_ROWS * 2, WG_B_BYTES = WG_BK * WG_ROWS * 2, WG_STAGE = WG_A_BYTES + WG_B_BYTES, WG_STAGES = 3;
constexpr int WG_CONVERT = 16;                             // warps that convert, and store the tile
constexpr int WG_THREADS = 64 + 32 * WG_CONVERT;
constexpr int WG_SMEM = WG_STAGES * WG_STAGE + WG_CONVERT * 4096 + 512 + 256 + 1024;

struct GradientParams {
  int m, n, k;
  int steps, per_split;          // steps of 64 rows in all, and of a split
  int dy_mode;                   // 0: by TMA, 1: bf16 rows that no 16-byte access divides, 2: codes
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
__device__ __forceinline__ void convert16(uint4 codes, int s, int format, uint4 (&out)[2]) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t o[8];
  const float factor = f8::up(s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = f8::decode2(w[i >> 1] >> (16 * (i & 1)) & 0xffffu, format);
    o[i] = bf16x2_bits(v.x * factor, v.y * factor);
  }
  out[0] = make_uint4(o[0], o[1], o[2], o[3]);
  out[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

// The place of a piece of eight columns in an MN-major operand: blocks of 64 columns, rows of 128 bytes, 128-byte swizzle.
__device__ __forceinline__ uint32_t piece_at(int row, int piece) { return (piece >> 3) * (WG_ROWS * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4); }

__global__ void __launch_bounds__(WG_THREADS, 1)
float8_gradient_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapO, const GradientParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_shared(smem_raw);
  uint8_t* out_stage = smem + WG_STAGES * WG_STAGE;
  uint8_t* ones = out_stage + WG_CONVERT * 4096;
  uint64_t* full = reinterpret_cast<uint64_t*>(ones + 512);
  uint64_t* empty = full + WG_STAGES;
  uint64_t* done = empty + WG_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.y * WG_BN, k0 = blockIdx.x * WG_BK, split = blockIdx.z;
  const int first = split * p.per_split, last = min(first + p.per_split, p.steps);
  const int columns = min(WG_BK, p.k - k0);
  const int groups = (columns + 63) / 64;                   // 64-channel blocks of x that exist
  const bool sums = blockIdx.x == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < WG_STAGES; ++s) { mbar_init(&full[s], WG_CONVERT + (p.dy_mode == 0)); mbar_init(&empty[s], 1); }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x < 128) reinterpret_cast<uint32_t*>(ones)[threadIdx.x] = 0x3f803f80u;
  fence_async_smem();
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  lf_chain();

  if (warp == 0) {
    if (lane == 0 && p.dy_mode == 0) {
      prefetch_tensormap(&mapA);
      int stage = 0; uint32_t phase = 0;
      for (int t = first; t < last; ++t) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, p.status, 131)) break;
        uint8_t* sA = smem + stage * WG_STAGE;
        mbar_expect_tx(&full[stage], WG_A_BYTES);
        tma_load_3d(sA, &mapA, &full[stage], n0, t * WG_ROWS, 0);
        tma_load_3d(sA + WG_A_BYTES / 2, &mapA, &full[stage], n0 + 64, t * WG_ROWS, 0);
        if (++stage == WG_STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0; uint32_t phase = 0;
      bool ok = true;
      constexpr uint32_t both = (1u << 7) | (1u << 10);      // bf16 operands
      const uint32_t idesc = make_idesc_f16(WG_BN, groups * 64, 1, 1) | both, idesc_ones = make_idesc_f16(WG_BN, 16, 1, 0) | both;
      const uint64_t ones_desc = make_smem_desc_plain(smem_u32(ones), 128, 256);
      for (int t = first; t < last; ++t) {
        if (!mbar_wait(&full[stage], phase, abort_flag, p.status, 132)) { ok = false; break; }
        tc_fence_after();
        const uint32_t a0 = smem_u32(smem + stage * WG_STAGE), b0 = a0 + WG_A_BYTES;
#pragma unroll
        for (int kk = 0; kk < WG_ROWS / 16; ++kk) {
          const uint64_t a = make_smem_desc(a0 + kk * 2048, WG_ROWS * 128, 1024);
          umma_f16(tmem_base, a, make_smem_desc(b0 + kk * 2048, WG_ROWS * 128, 1024), idesc, (t != first || kk != 0) ? 1u : 0u);
          if (sums) umma_f16(tmem_base + WG_BK, a, ones_desc, idesc_ones, (t != first || kk != 0) ? 1u : 0u);
        }
        umma_commit(&empty[stage]);
        if (++stage == WG_STAGES) { stage = 0; phase ^= 1; }
      }
      if (ok) umma_commit(done);
    }
  } else {
    // Rows of a step: x has 16 pieces of 16 channels, dy 8 of 16 outputs; neighbouring lanes take neighbouring pieces of a row.
    const int thread = threadIdx.x - 64;
    constexpr int kUnits = WG_ROWS * 16 / (32 * WG_CONVERT);      // of x a thread
    const int xp = thread & 15, xr = thread >> 4;                 // piece, first row (rows xr + 32 u)
    const int yp = thread & 7, yr = thread >> 3;                  // of dy, one unit a thread
    const int xch = k0 + xp * 16, ych = n0 + yp * 16;
    const bool x_any = xch < p.x.pitch && xp < groups * 4, y_any = ych < p.n;
    const int64_t xblock = xch / f8::kBlock, yblock = ych / f8::kBlock;
    uint4 xc[kUnits], yc[2];
    int xs[kUnits], ys = 1;
    auto fetch = [&](int t) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int64_t row = (int64_t)t * WG_ROWS + xr + 32 * u;
        xc[u] = make_uint4(0, 0, 0, 0);
        xs[u] = 1;
        if (x_any && row < p.m) {
          xc[u] = *reinterpret_cast<const uint4*>(p.x.codes + row * p.x.pitch + xch);
          xs[u] = p.x.exponents[f8::exponent_at(row, (int)xblock, p.x.tiles)];
        }
      }
      if (p.dy_mode != 0) {
        const int64_t row = (int64_t)t * WG_ROWS + yr;
        yc[0] = yc[1] = make_uint4(0, 0, 0, 0);
        if (y_any && row < p.m) {
          if (p.dy_mode == 2) {
            yc[0] = *reinterpret_cast<const uint4*>(p.dy8.codes + row * p.dy8.pitch + ych);
            ys = p.dy8.exponents[f8::exponent_at(row, (int)yblock, p.dy8.tiles)];
          } else {
            const uint16_t* from = reinterpret_cast<const uint16_t*>(p.dy) + row * p.n + ych;
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              o[i] = (ych + 2 * i < p.n ? (uint32_t)from[2 * i] : 0u) | (ych + 2 * i + 1 < p.n ? (uint32_t)from[2 * i + 1] << 16 : 0u);
            yc[0] = make_uint4(o[0], o[1], o[2], o[3]);
            yc[1] = make_uint4(o[4], o[5], o[6], o[7]);
          }
        }
      }
    };
    int stage = 0; uint32_t phase = 0;
    bool ok = true;
    fetch(first);
    for (int t = first; t < last; ++t) {
      if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, p.status, 133)) { ok = false; break; }
      uint8_t* sA = smem + stage * WG_STAGE;
      uint8_t* sB = sA + WG_A_BYTES;
      uint4 codes[kUnits], other[2] = {yc[0], yc[1]};
      int s[kUnits];
      const int sy = ys;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) { codes[u] = xc[u]; s[u] = xs[u]; }
      if (t + 1 < last) fetch(t + 1);
      // (odd blocks of 64 columns store their second piece first: eight lanes then fill eight different 16-byte columns of the banks)
      if (xp < groups * 4) {
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
      if (p.dy_mode != 0) {
        uint4 v[2] = {other[0], other[1]};
        if (p.dy_mode == 2) convert16(other[0], sy, p.dy8.format, v);
        const int swap = yp >> 2 & 1;
        *reinterpret_cast<uint4*>(sA + piece_at(yr, yp * 2 + swap)) = swap ? v[1] : v[0];
        *reinterpret_cast<uint4*>(sA + piece_at(yr, yp * 2 + 1 - swap)) = swap ? v[0] : v[1];
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[stage]);
      if (++stage == WG_STAGES) { stage = 0; phase ^= 1; }
    }
    // The tile: 16 warps, 64 columns of a lane quadrant each.
    ok = ok && mbar_wait(done, 0, abort_flag, p.status, 134);
    tc_fence_after();
    if (ok) {
      const int q = warp & 3, part = (warp - 2) >> 2, row0 = n0 + q * 32, col0 = k0 + part * 64;
      uint8_t* tile = out_stage + (warp - 2) * 4096;
      float* out = p.out + split * p.split_stride;
      if (row0 < p.n && col0 < p.k) {
        uint32_t r[2][32];
        const uint32_t d = tmem_base + ((uint32_t)(q * 32) << 16) + part * 64;
        tmem_ld32(d, r[0]);
        tmem_ld32(d + 32, r[1]);
        tmem_ld_wait();
        tie32(r[0]);
        tie32(r[1]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int c0 = col0 + half * 32;
          if (c0 >= p.k) break;
          if (lane == 0) bulk_wait_read();
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<uint4*>(tile + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(r[half][c * 4], r[half][c * 4 + 1], r[half][c * 4 + 2], r[half][c * 4 + 3]);
          if (p.vector_out) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) { tma_store_3d(&mapO, tile, c0, row0, split); bulk_commit(); }
          } else {
            __syncwarp();
            const int rows = min(32, p.n - row0);
            for (int row = 0; row < rows; ++row)
              if (c0 + lane < p.k) out[(int64_t)(row0 + row) * p.ld + c0 + lane] = *reinterpret_cast<const float*>(tile + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4);
            __syncwarp();
          }
        }
      }
      if (sums && part == 0) {
        uint32_t r[8];
        tmem_ld8(tmem_base + ((uint32_t)(q * 32) << 16) + WG_BK, r);
        tmem_ld_wait();
        if (p.bias && row0 + lane < p.n) p.bias[split * p.bias_stride + row0 + lane] = __uint_as_float(r[0]);
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

// dW and dbias from the splits' partial tiles, added in order.
__global__ void __launch_bounds__(256)
gradient_join_kernel(const float* partial, int64_t ld, int64_t split_stride, int splits, int n, int k, float* out, const float* bias_partial, float* bias) {
  lf_chain();
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, total = (int64_t)n * k;
  if (at < total) {
    const int64_t row = at / k;
    const float* from = partial + row * ld + (at - row * k);
    float t = 0.f;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) t += from[s * split_stride];
    out[at] = t;
  }
  if (at < n && bias) {
    float t = 0.f;
    for (int s = 0; s < splits; ++s) t += bias_partial[(int64_t)s * n + at];
    bias[at] = t;
  }
}

void configure_float8_gradient() { cudaFuncSetAttribute(float8_gradient_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, WG_SMEM); }

// Blocks of rows: as many as the GPU has multiprocessors for beside the tiles, and four steps of 64 rows each at least.
static void gradient_plan(const lf_context* ctx, int64_t m, int n, int k, int& steps, int& splits, int& per_split) {
  const int tiles = ((n + WG_BN - 1) / WG_BN) * ((k + WG_BK - 1) / WG_BK);
  steps = (int)((m + WG_ROWS - 1) / WG_ROWS);
  const int want = std::max(1, std::min(ctx->sm_count / tiles, steps / 4));
  per_split = (steps + want - 1) / want;
  splits = (steps + per_split - 1) / per_split;
}
static int64_t partial_ld(int k) { return (k + 3) / 4 * 4; }

}  // namespace tc

using namespace f8;

extern "C" {

uint64_t lf_float8_weight_gradient_workspace(const lf_context* ctx, int64_t rows, int32_t channels, int32_t out_channels) {
  if (!ctx || rows <= 0 || rows > 0x7fffffff || channels <= 0 || out_channels <= 0) return 0;
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
  if (d->out_channels > (1 << 22) || x.channels > (1 << 22)) return lf_fail(ctx, LF_ERR_UNSUPPORTED, "float8 weight gradient: %d x %d are too many channels", d->out_channels, x.channels);
  LF_TRY(lf_float8_check(ctx, "float8 weight gradient, activations", x, x.rows, x.channels));
  if (d->encoded_gradient.codes) LF_TRY(lf_float8_check(ctx, "float8 weight gradient, gradient", d->encoded_gradient, x.rows, d->out_channels));
  const uint64_t need = lf_float8_weight_gradient_workspace(ctx, x.rows, x.channels, d->out_channels);
  if (need && (!d->workspace || d->workspace_bytes < need || !lf_aligned16(d->workspace)))
    return lf_fail(ctx, LF_ERR_ARGUMENT, "float8 weight gradient: a workspace of %llu bytes on a 16-byte boundary is needed", (unsigned long long)need);
  LF_CUDA(ctx, cudaSetDevice(ctx->device));
  tc::GradientParams p{};
  p.m = (int)x.rows; p.n = d->out_channels; p.k = x.channels;
  int splits;
  tc::gradient_plan(ctx, x.rows, p.n, p.k, p.steps, splits, p.per_split);
  p.x = matrix(x);
  CUtensorMap ma{}, mo{};
  if (d->encoded_gradient.codes) { p.dy_mode = 2; p.dy8 = matrix(d->encoded_gradient); }
  else {
    p.dy = (const bf16*)d->gradient;
    p.dy_mode = lf_aligned16(p.dy) && p.n % 8 == 0 ? 0 : 1;
    if (p.dy_mode == 0) LF_TRY(tc::make_map_rows(ctx, &ma, p.dy, false, p.n, p.m, tc::WG_ROWS));
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
  lf_launch(ctx, tc::float8_gradient_kernel, dim3((p.k + tc::WG_BK - 1) / tc::WG_BK, (p.n + tc::WG_BN - 1) / tc::WG_BN, splits), tc::WG_THREADS, tc::WG_SMEM, ma, mo, p);
  lf_prof_end(ctx);
  ctx->launches++;
  if (!direct) {
    lf_prof_begin(ctx, LF_KERNEL_ELEMENTWISE);
    lf_launch(ctx, tc::gradient_join_kernel, lf_ceil_div((int64_t)p.n * p.k, 256), 256, 0, p.out, p.ld, p.split_stride, splits, p.n, p.k, d->weight_gradient, bias_partial,
              d->bias_gradient);
    lf_prof_end(ctx);
    ctx->launches++;
  }
  return lf_float8_done(ctx, r, direct ? 1 : 2);
}

}  // extern "C"
