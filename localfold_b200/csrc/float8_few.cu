// The projection on 8-bit operands for few rows (single tokens): the weights are all that is read, so their way from memory is what counts.
//
// A block has 16 outputs over all channels, its warps every eighth block of 128 channels each, so that many short streams of weights are in
// flight at once.  Codes become fp16 in registers (exactly) and mma.sync multiplies 16 outputs by 8 rows, 16 channels at a time; the order of channels
// within 64 is permuted alike in both operands, so that a lane's share is 16 neighbouring codes.  The sum of a block of 128 channels is scaled by its
// two powers of two and added in float32; the warps' sums meet in shared memory.  The rows are encoded by every block (they
// are few), so that one launch does it all: 4 x 1536 -> 384 takes 4.1 us, and took 2.2 for the encoder and 6.7 for the tiled kernel.
#include "float8.cuh"
#include "tc_kernels.cuh"

namespace tc {

using namespace f8;

constexpr int FEW_WARPS = 8, FEW_OUT = 16;

struct FewParams {
  int rows, n, k, out_f32, access;
  const void* source;          // null: x has the codes
  Matrix x, w;                 // (x.codes null: not kept)
  const float* bias;
  void* out;
};

__device__ __forceinline__ void mma_16x8x16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// total + c 2^(s - 254), s the sum of the two powers' bytes.  By halves of the power: the rows' whole power may take c out of float32's range where the
// weights' brings it back.
__device__ __forceinline__ float scaled_sum(float total, float c, int s) { return fmaf(c * up(s >> 1), up(s - (s >> 1)), total); }

// EIGHTS: 8 or 16 rows; FORMAT of x (weights are e4m3).  Shared memory: the rows' codes, rows of `room` bytes, then their exponents [row][block].
template <typename T, int EIGHTS, int FORMAT>
__global__ void __launch_bounds__(FEW_WARPS * 32)
float8_few_kernel(const FewParams p) {
  constexpr int kRows = EIGHTS * 8;
  extern __shared__ __align__(16) uint8_t few_smem[];
  __shared__ __align__(16) float rooms[FEW_WARPS][kRoom];
  __shared__ float sums[FEW_WARPS][FEW_OUT][kRows + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nblk = blocks(p.k), room = nblk * kBlock + 64;      // (two rows' 64 bytes lie in different banks)
  uint8_t* codes_s = few_smem;
  uint8_t* exp_s = few_smem + kRows * room;
  const int n0 = blockIdx.x * FEW_OUT;
  lf_chain();

  // the rows' codes: a block of 128 channels per eight lanes
  const int units = kRows * nblk, l8 = threadIdx.x & 7;
  for (int u0 = 0; u0 < units; u0 += FEW_WARPS * 4) {      // (the same number of turns for every lane)
    const int u = u0 + (threadIdx.x >> 3), row = u / nblk, block = u - row * nblk, first = block * kBlock + l8 * kShare;
    const bool live = u < units && row < p.rows;
    uint4 codes = make_uint4(0, 0, 0, 0);
    int s = 1;
    if (p.source) {
      Raw<T> raw;
      load16<T, 8>(raw, static_cast<const T*>(p.source) + (int64_t)row * p.k + first, p.k - first, live, p.access);
      s = encode16<8>(unpack<T, 8>(raw, p.access, rooms[warp]), FORMAT, codes);
      if (live && p.x.codes && blockIdx.x == 0) put16(p.x, row, first, codes, s);
    } else if (live) {
      if (first < p.k) codes = *reinterpret_cast<const uint4*>(p.x.codes + row * p.x.pitch + first);
      s = p.x.exponents[exponent_at(row, block, p.x.tiles)];
    }
    if (u < units) {
      *reinterpret_cast<uint4*>(codes_s + row * room + first) = codes;
      if (l8 == 0) exp_s[row * nblk + block] = (uint8_t)s;
    }
  }
  __syncthreads();

  const int g = lane >> 2, t = lane & 3;
  const int64_t r0 = n0 + g, r1 = r0 + 8;
  float total[EIGHTS][4];
#pragma unroll
  for (int e = 0; e < EIGHTS; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) total[e][i] = 0.f;
  constexpr int kAhead = 2;      // blocks whose weights are in flight
  uint4 w[kAhead][2][2];         // [block][half of its channels][output row]
  int sw[kAhead][2];
  auto fetch = [&](int slot, int block) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = block * kBlock + h * 64 + t * 16;
      w[slot][h][0] = w[slot][h][1] = make_uint4(0, 0, 0, 0);
      if (c < p.k) {      // (the last group of sixteen lies in the row's pitch, zeros behind its end)
        if (r0 < p.n) w[slot][h][0] = *reinterpret_cast<const uint4*>(p.w.codes + r0 * p.w.pitch + c);
        if (r1 < p.n) w[slot][h][1] = *reinterpret_cast<const uint4*>(p.w.codes + r1 * p.w.pitch + c);
      }
    }
    sw[slot][0] = r0 < p.n ? p.w.exponents[exponent_at(r0, block, p.w.tiles)] : 1;
    sw[slot][1] = r1 < p.n ? p.w.exponents[exponent_at(r1, block, p.w.tiles)] : 1;
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (warp + i * FEW_WARPS < nblk) fetch(i, warp + i * FEW_WARPS);
  for (int base = warp; base < nblk; base += FEW_WARPS * kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int block = base + i * FEW_WARPS;
      if (block < nblk) {
        float c[EIGHTS][4];
#pragma unroll
        for (int e = 0; e < EIGHTS; ++e)
#pragma unroll
          for (int j = 0; j < 4; ++j) c[e][j] = 0.f;
        const int w0_power = sw[i][0], w1_power = sw[i][1];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 x[EIGHTS];
#pragma unroll
          for (int e = 0; e < EIGHTS; ++e) x[e] = *reinterpret_cast<const uint4*>(codes_s + (e * 8 + g) * room + block * kBlock + h * 64 + t * 16);
          const uint32_t w0[4] = {w[i][h][0].x, w[i][h][0].y, w[i][h][0].z, w[i][h][0].w}, w1[4] = {w[i][h][1].x, w[i][h][1].y, w[i][h][1].z, w[i][h][1].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {      // four codes a lane are 16 channels of the product
            const uint32_t a[4] = {half2_of<LF_FLOAT8_E4M3>(w0[j] & 0xffffu), half2_of<LF_FLOAT8_E4M3>(w1[j] & 0xffffu), half2_of<LF_FLOAT8_E4M3>(w0[j] >> 16),
                                   half2_of<LF_FLOAT8_E4M3>(w1[j] >> 16)};
#pragma unroll
            for (int e = 0; e < EIGHTS; ++e) {
              const uint32_t xw = j == 0 ? x[e].x : j == 1 ? x[e].y : j == 2 ? x[e].z : x[e].w;
              mma_16x8x16(c[e], a, half2_of<FORMAT>(xw & 0xffffu), half2_of<FORMAT>(xw >> 16));
            }
          }
        }
        if (block + FEW_WARPS * kAhead < nblk) fetch(i, block + FEW_WARPS * kAhead);
#pragma unroll
        for (int e = 0; e < EIGHTS; ++e) {
          const int x0_power = exp_s[(e * 8 + 2 * t) * nblk + block], x1_power = exp_s[(e * 8 + 2 * t + 1) * nblk + block];
          total[e][0] = scaled_sum(total[e][0], c[e][0], x0_power + w0_power);
          total[e][1] = scaled_sum(total[e][1], c[e][1], x1_power + w0_power);
          total[e][2] = scaled_sum(total[e][2], c[e][2], x0_power + w1_power);
          total[e][3] = scaled_sum(total[e][3], c[e][3], x1_power + w1_power);
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < EIGHTS; ++e) {
    sums[warp][g][e * 8 + 2 * t] = total[e][0];
    sums[warp][g][e * 8 + 2 * t + 1] = total[e][1];
    sums[warp][g + 8][e * 8 + 2 * t] = total[e][2];
    sums[warp][g + 8][e * 8 + 2 * t + 1] = total[e][3];
  }
  __syncthreads();
  const int o = threadIdx.x & 15, row = threadIdx.x >> 4;
  if (row < p.rows && row < kRows && n0 + o < p.n) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < FEW_WARPS; ++i) v += sums[i][o][row];
    if (p.bias) v += p.bias[n0 + o];
    const int64_t at = (int64_t)row * p.n + n0 + o;
    if (p.out_f32) static_cast<float*>(p.out)[at] = v;
    else static_cast<bf16*>(p.out)[at] = __float2bfloat16_rn(v);
  }
}

static int few_smem_bytes(int rows8, int k) { return rows8 * 8 * (blocks(k) * kBlock + 64 + blocks(k)); }

// Rows that the kernel takes: sixteen, and what their codes may have of shared memory.
bool float8_few_takes(int64_t rows, int k) { return rows <= 16 && k <= 4096; }

// f(T, EIGHTS, FORMAT as types)
template <typename F>
static void few_forms(int dtype, int eights, int format, F f) {
  auto with = [&](auto t, auto e) {
    if (format == LF_FLOAT8_E4M3) f(t, e, std::integral_constant<int, LF_FLOAT8_E4M3>{}); else f(t, e, std::integral_constant<int, LF_FLOAT8_E5M2>{});
  };
  auto typed = [&](auto t) { if (eights == 1) with(t, std::integral_constant<int, 1>{}); else with(t, std::integral_constant<int, 2>{}); };
  if (dtype == LF_DTYPE_BF16) typed(bf16{}); else typed(float{});
}

void configure_float8_few() {
  for (int i = 0; i < 8; ++i)
    few_forms(i & 1, 1 + (i >> 1 & 1), i >> 2, [](auto t, auto e, auto f) {
      cudaFuncSetAttribute(float8_few_kernel<decltype(t), decltype(e)::value, decltype(f)::value>, cudaFuncAttributeMaxDynamicSharedMemorySize, few_smem_bytes(2, 4096));
    });
}

// out = x . w^T + bias; `source` (dtype) or x's codes; x.codes, where set beside a source, receive its 8-bit form.
lf_status float8_few(lf_context* ctx, const void* source, int dtype, const Matrix& x, const Matrix& w, const float* bias, void* out, int out_dtype) {
  FewParams p{};
  p.rows = (int)x.rows; p.n = (int)w.rows; p.k = x.channels; p.out_f32 = out_dtype == LF_DTYPE_F32;
  p.source = source; p.access = source ? row_access(source, x.channels, dtype) : 0;
  p.x = x; p.w = w; p.bias = bias; p.out = out;
  const int eights = p.rows > 8 ? 2 : 1;
  lf_prof_begin(ctx, LF_KERNEL_SIMT);
  few_forms(dtype, eights, x.format, [&](auto t, auto e, auto f) {
    lf_launch(ctx, float8_few_kernel<decltype(t), decltype(e)::value, decltype(f)::value>, lf_ceil_div(p.n, FEW_OUT), FEW_WARPS * 32, few_smem_bytes(eights, p.k), p);
  });
  lf_prof_end(ctx);
  ctx->launches++;
  return LF_OK;
}

}  // namespace tc
