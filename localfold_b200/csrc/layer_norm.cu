// LayerNorm as an operator of its own, forward and backward (the pair stack's own norms are fused into the kernels that read them).
//
//   forward   y = (x - mean) rstd g + b, mean and rstd over the c channels of a row in float32, in two passes over registers
//   backward  u = (x - mean) rstd, h = dy g:  dx = rstd (h - mean(h) - u mean(h u)), dg = sum over rows of dy u, db = sum of dy
//
// Both read and write each element once, so memory bounds them.  A group of G lanes holds a row in registers, eight neighbouring
// channels a lane and step: 16 lanes a block of 128 channels, so that the row can leave in its 8-bit form (float8.cuh) or come back
// from it in the same pass.  Blocks stay and walk over the rows, the weights in registers; a lane always has the same channels, so
// dg and db add up in its registers and every block leaves one row of sums, which a second, small kernel adds in a fixed order.
#include "float8.cuh"

namespace lnorm {

using namespace f8;

constexpr int kThreads = 256;

struct Forward {
  int64_t rows;
  int c, vector_in, vector_out;
  float epsilon;
  const void* x;
  const float *scale, *offset;
  void* y;                       // or null
  float *mean, *inverse;         // or null
  Matrix kept, encoded;          // codes null: none
};

struct Backward {
  int64_t rows;
  int c, vector_dy, vector_x, vector_dx;
  const void *dy, *x;            // x null: `kept`
  Matrix kept;
  const float *mean, *inverse, *scale;
  void* dx;
  float* partial;                // [blocks][2][c]
};

// Sum over the G lanes of a row; G = kThreads: the whole block, through two rows of slots in turn.
template <int G>
__device__ __forceinline__ float group_sum(float v, float* slots, int& turn) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (G > 32) {
    float* s = slots + (turn++ & 1) * (kThreads / 32);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) v += s[w];
  }
  return v;
}

template <typename T, int G, int NV, int R>
__global__ void __launch_bounds__(kThreads)
forward_kernel(const Forward a) {
  __shared__ float slots[2 * kThreads / 32];
  constexpr int kGroups = kThreads / G;
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  int turn = 0;
  lf_chain();
  float scale[NV][8], offset[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int first = (v * G + lane) * 8;
    load8(a.scale + first, a.c - first, false, scale[v]);
    load8(a.offset + first, a.c - first, false, offset[v]);
  }
  const float over = 1.0f / (float)a.c;
  // (the trip count is the same for every lane of a block)
  for (int64_t base = (int64_t)blockIdx.x * kGroups * R; base < a.rows; base += (int64_t)gridDim.x * kGroups * R) {
    float x[R][NV][8];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kGroups + group;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int first = (v * G + lane) * 8;
        load8(static_cast<const T*>(a.x) + row * a.c + first, row < a.rows ? a.c - first : 0, a.vector_in, x[r][v]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kGroups + group;
      const bool live = row < a.rows;
      if (a.kept.codes) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int first = (v * G + lane) * 8;
          uint2 codes;
          const int s = encode8<(G < 16 ? G : 16)>(x[r][v], a.kept.format, codes);
          if (live) put8(a.kept, row, first, codes, s, (first & 127) == 0 && first < a.c);
        }
      }
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += x[r][v][i];
      const float mean = group_sum<G>(sum, slots, turn) * over;
      sum = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[r][v][i] -= mean;
          if ((v * G + lane) * 8 + i < a.c) sum = fmaf(x[r][v][i], x[r][v][i], sum);
        }
      const float inverse = 1.0f / sqrtf(fmaf(group_sum<G>(sum, slots, turn), over, a.epsilon));
      if (a.mean && live && lane == 0) { a.mean[row] = mean; a.inverse[row] = inverse; }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int first = (v * G + lane) * 8;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = fmaf(x[r][v][i] * inverse, scale[v][i], offset[v][i]);
        if (a.y && live) store8(static_cast<T*>(a.y) + row * a.c + first, a.c - first, a.vector_out, y);
        if (a.encoded.codes) {
#pragma unroll
          for (int i = 0; i < 8; ++i) if (first + i >= a.c) y[i] = 0.f;
          uint2 codes;
          const int s = encode8<(G < 16 ? G : 16)>(y, a.encoded.format, codes);
          if (live) put8(a.encoded, row, first, codes, s, (first & 127) == 0 && first < a.c);
        }
      }
    }
  }
}

template <typename T, int G, int NV, int R>
__global__ void __launch_bounds__(kThreads)
backward_kernel(const Backward a) {
  constexpr int kGroups = kThreads / G;
  __shared__ float slots[2 * kThreads / 32];
  __shared__ float sums[kGroups > 1 ? kThreads * NV * 8 : 1];
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  int turn = 0;
  lf_chain();
  float scale[NV][8], dg[NV][8], db[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int first = (v * G + lane) * 8;
    load8(a.scale + first, a.c - first, false, scale[v]);
#pragma unroll
    for (int i = 0; i < 8; ++i) dg[v][i] = db[v][i] = 0.f;
  }
  const float over = 1.0f / (float)a.c;
  for (int64_t base = (int64_t)blockIdx.x * kGroups * R; base < a.rows; base += (int64_t)gridDim.x * kGroups * R) {
    float dy[R][NV][8], u[R][NV][8], mean[R], inverse[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kGroups + group;
      const bool live = row < a.rows;
      mean[r] = live ? a.mean[row] : 0.f;
      inverse[r] = live ? a.inverse[row] : 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int first = (v * G + lane) * 8, count = live ? a.c - first : 0;
        load8(static_cast<const T*>(a.dy) + row * a.c + first, count, a.vector_dy, dy[r][v]);
        if (a.x) load8(static_cast<const T*>(a.x) + row * a.c + first, count, a.vector_x, u[r][v]);
        else {
          uint2 codes = make_uint2(0, 0);
          float factor = 0.f;
          if (count > 0) {
            codes = *reinterpret_cast<const uint2*>(a.kept.codes + row * a.kept.pitch + first);
            factor = up(a.kept.exponents[exponent_at(row, first / kBlock, a.kept.tiles)]);
          }
          decode8(codes, factor, a.kept.format, u[r][v]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kGroups + group;
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          u[r][v][i] = (u[r][v][i] - mean[r]) * inverse[r];
          const float h = dy[r][v][i] * scale[v][i];
          dg[v][i] = fmaf(dy[r][v][i], u[r][v][i], dg[v][i]);
          db[v][i] += dy[r][v][i];
          s1 += h;
          s2 = fmaf(h, u[r][v][i], s2);
        }
      s1 = group_sum<G>(s1, slots, turn) * over;
      s2 = group_sum<G>(s2, slots, turn) * over;
      if (row < a.rows) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int first = (v * G + lane) * 8;
          float dx[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) dx[i] = inverse[r] * (fmaf(dy[r][v][i], scale[v][i], -s1) - u[r][v][i] * s2);
          store8(static_cast<T*>(a.dx) + row * a.c + first, a.c - first, a.vector_dx, dx);
        }
      }
    }
  }
  // this block's row of sums
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = a.partial + ((int64_t)blockIdx.x * 2 + which) * a.c;
    if (kGroups == 1) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int first = (v * G + lane) * 8;
        store8(out + first, a.c - first, false, which ? db[v] : dg[v]);
      }
    } else {
      __syncthreads();
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[group * (G * NV * 8) + (v * G + lane) * 8 + i] = which ? db[v][i] : dg[v][i];
      __syncthreads();
      for (int col = threadIdx.x; col < a.c; col += kThreads) {
        float t = 0.f;
#pragma unroll 8
        for (int g = 0; g < kGroups; ++g) t += sums[g * (G * NV * 8) + col];
        out[col] = t;
      }
    }
  }
}

// Column sums of the blocks' rows, in the same order every time: 32 columns a block, 16 strands of rows, then the strands.
__global__ void __launch_bounds__(512)
join_kernel(const float* partial, int count, int c, float* dg, float* db) {
  __shared__ float s[16][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  lf_chain();
  float t = 0.f;
  if (col < c)
    for (int i = strand; i < count; i += 16) t += partial[((int64_t)i * 2 + blockIdx.y) * c + col];
  s[strand][lane] = t;
  __syncthreads();
  if (strand == 0 && col < c) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += s[i][lane];
    (blockIdx.y ? db : dg)[col] = t;
  }
}

// Blocks that stay on the GPU, and no more than there are rows for.
static int grid_of(const lf_context* ctx, int64_t rows, int per_block, int per_sm) {
  const int64_t need = (rows + per_block - 1) / per_block, most = (int64_t)ctx->sm_count * per_sm;
  return (int)(need < most ? need : most);
}

// Lanes of a row, steps of eight channels a lane, rows in flight: by the width alone.
//   f(G, NV, R) with the constants as types
template <typename F>
static auto by_width(int c, F f) {
#define LF_NORM_FORM(G, NV, R) f(std::integral_constant<int, G>{}, std::integral_constant<int, NV>{}, std::integral_constant<int, R>{})
  if (c <= 64) return LF_NORM_FORM(8, 1, 2);
  if (c <= 128) return LF_NORM_FORM(16, 1, 2);
  if (c <= 256) return LF_NORM_FORM(32, 1, 2);
  if (c <= 512) return LF_NORM_FORM(32, 2, 1);
  if (c <= 1024) return LF_NORM_FORM(32, 4, 1);
  if (c <= 2048) return LF_NORM_FORM(kThreads, 1, 1);
  if (c <= 4096) return LF_NORM_FORM(kThreads, 2, 1);
  return LF_NORM_FORM(kThreads, 4, 1);
#undef LF_NORM_FORM
}

constexpr int kMostChannels = 8192, kPerSm = 4;

template <typename T>
static void launch_forward(lf_context* ctx, const Forward& a) {
  by_width(a.c, [&](auto g, auto nv, auto r) {
    constexpr int G = decltype(g)::value, NV = decltype(nv)::value, R = decltype(r)::value;
    lf_launch(ctx, forward_kernel<T, G, NV, R>, grid_of(ctx, a.rows, kThreads / G * R, kPerSm), kThreads, 0, a);
  });
}

static int backward_blocks(const lf_context* ctx, int64_t rows, int c) {
  return by_width(c, [&](auto g, auto, auto r) { return grid_of(ctx, rows, kThreads / decltype(g)::value * decltype(r)::value, kPerSm); });
}

template <typename T>
static void launch_backward(lf_context* ctx, const Backward& a, int blocks) {
  by_width(a.c, [&](auto g, auto nv, auto r) {
    lf_launch(ctx, backward_kernel<T, decltype(g)::value, decltype(nv)::value, decltype(r)::value>, blocks, kThreads, 0, a);
  });
}

static bool vector_rows(const void* p, int c, int dtype) { return lf_aligned16(p) && c % (dtype == LF_DTYPE_BF16 ? 8 : 4) == 0; }

}  // namespace lnorm

using namespace lnorm;

extern "C" {

lf_status lf_layer_norm_run(lf_context* ctx, const lf_layer_norm_desc* d, lf_result* r) {
  if (!ctx) return LF_ERR_ARGUMENT;
  if (!d || !d->activations || !d->scale || !d->offset) return lf_fail(ctx, LF_ERR_ARGUMENT, "layer norm: null argument");
  if (!d->out && !d->encoded.codes) return lf_fail(ctx, LF_ERR_ARGUMENT, "layer norm: neither an output nor an encoded output");
  if (!d->mean != !d->inverse_deviation) return lf_fail(ctx, LF_ERR_ARGUMENT, "layer norm: mean and inverse_deviation come together");
  LF_TRY(lf_float8_check_rows(ctx, "layer norm", d->rows, d->channels, d->act_dtype));
  if (d->channels > kMostChannels) return lf_fail(ctx, LF_ERR_UNSUPPORTED, "layer norm of %d channels: at most %d", d->channels, kMostChannels);
  if (d->variance != LF_VARIANCE_TWO_PASS && d->variance != LF_VARIANCE_FAST) return lf_fail(ctx, LF_ERR_ARGUMENT, "unknown variance %d", d->variance);
  if (!(d->epsilon > 0.f) || !(d->epsilon < INFINITY)) return lf_fail(ctx, LF_ERR_SHAPE, "epsilon must be finite and positive; received %g", d->epsilon);
  for (const lf_float8_matrix* m : {&d->checkpoint, &d->encoded})
    if (m->codes) LF_TRY(lf_float8_check(ctx, "layer norm", *m, d->rows, d->channels));
  LF_CUDA(ctx, cudaSetDevice(ctx->device));
  Forward a{};
  a.rows = d->rows; a.c = d->channels; a.epsilon = d->epsilon;
  a.vector_in = vector_rows(d->activations, a.c, d->act_dtype);
  a.vector_out = vector_rows(d->out, a.c, d->act_dtype);
  a.x = d->activations; a.scale = d->scale; a.offset = d->offset; a.y = d->out; a.mean = d->mean; a.inverse = d->inverse_deviation;
  if (d->checkpoint.codes) a.kept = matrix(d->checkpoint);
  if (d->encoded.codes) a.encoded = matrix(d->encoded);
  lf_prof_begin(ctx, LF_KERNEL_ELEMENTWISE);
  if (d->act_dtype == LF_DTYPE_BF16) launch_forward<bf16>(ctx, a); else launch_forward<float>(ctx, a);
  lf_prof_end(ctx);
  ctx->launches++;
  return lf_float8_done(ctx, r, 1);
}

uint64_t lf_layer_norm_backward_workspace(const lf_context* ctx, int64_t rows, int32_t channels) {
  if (!ctx || rows <= 0 || channels <= 0 || channels > kMostChannels) return 0;
  return (uint64_t)backward_blocks(ctx, rows, channels) * 2 * channels * sizeof(float);
}

lf_status lf_layer_norm_backward_run(lf_context* ctx, const lf_layer_norm_backward_desc* d, lf_result* r) {
  if (!ctx) return LF_ERR_ARGUMENT;
  if (!d || !d->gradient || (!d->activations && !d->checkpoint.codes) || !d->mean || !d->inverse_deviation || !d->scale || !d->out ||
      !d->scale_gradient || !d->offset_gradient || !d->workspace)
    return lf_fail(ctx, LF_ERR_ARGUMENT, "layer norm backward: null argument");
  if (d->activations && d->checkpoint.codes) return lf_fail(ctx, LF_ERR_ARGUMENT, "layer norm backward: activations or a checkpoint, not both");
  LF_TRY(lf_float8_check_rows(ctx, "layer norm backward", d->rows, d->channels, d->act_dtype));
  if (d->channels > kMostChannels) return lf_fail(ctx, LF_ERR_UNSUPPORTED, "layer norm of %d channels: at most %d", d->channels, kMostChannels);
  if (d->checkpoint.codes) LF_TRY(lf_float8_check(ctx, "layer norm backward", d->checkpoint, d->rows, d->channels));
  const uint64_t need = lf_layer_norm_backward_workspace(ctx, d->rows, d->channels);
  if (d->workspace_bytes < need || !lf_aligned16(d->workspace))
    return lf_fail(ctx, LF_ERR_ARGUMENT, "layer norm backward: a workspace of %llu bytes on a 16-byte boundary is needed", (unsigned long long)need);
  LF_CUDA(ctx, cudaSetDevice(ctx->device));
  Backward a{};
  a.rows = d->rows; a.c = d->channels;
  a.vector_dy = vector_rows(d->gradient, a.c, d->act_dtype);
  a.vector_x = vector_rows(d->activations, a.c, d->act_dtype);
  a.vector_dx = vector_rows(d->out, a.c, d->act_dtype);
  a.dy = d->gradient; a.x = d->activations; a.mean = d->mean; a.inverse = d->inverse_deviation; a.scale = d->scale; a.dx = d->out;
  if (d->checkpoint.codes) a.kept = matrix(d->checkpoint);
  a.partial = (float*)d->workspace;
  const int blocks = backward_blocks(ctx, a.rows, a.c);
  lf_prof_begin(ctx, LF_KERNEL_ELEMENTWISE);
  if (d->act_dtype == LF_DTYPE_BF16) launch_backward<bf16>(ctx, a, blocks); else launch_backward<float>(ctx, a, blocks);
  lf_prof_end(ctx);
  lf_prof_begin(ctx, LF_KERNEL_ELEMENTWISE);
  lf_launch(ctx, join_kernel, dim3(lf_ceil_div(a.c, 32), 2), 512, 0, a.partial, blocks, a.c, d->scale_gradient, d->offset_gradient);
  lf_prof_end(ctx);
  ctx->launches += 2;
  return lf_float8_done(ctx, r, 2);
}

}  // extern "C"
