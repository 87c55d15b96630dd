// LayerNorm as an operator of its own, forward and backward (the pair stack's own norms are fused into the kernels that read them).
//
//   forward   y = (x - mean) rstd g + b, mean and rstd over the c channels of a row in float32, in two passes over registers
//   backward  u = (x - mean) rstd, h = dy g:  dx = rstd (h - mean(h) - u mean(h u)), dg = sum over rows of dy u, db = sum of dy
//
// Both read and write each element once, so memory bounds them - as long as the instructions an element costs stay few: a lane has sixteen
// neighbouring channels of a row, so that the shuffles of the sums are shared by sixteen elements, arithmetic goes two float32 at a time,
// and eight lanes are a block of the 8-bit form (float8.cuh), which leaves or comes back in the same pass.  G lanes hold a row in registers.
// Blocks stay and walk over the rows, the next row's loads in flight under the present one's arithmetic and the weights in registers; a lane always
// has the same channels, so dg and db add up in its registers and every block leaves one row of sums, which a second, small kernel
// adds in a fixed order.  205824 x 64 in float32: forward 18.2 us, 5.8 TB/s; 147456 x 128 in bf16 with an e4m3 checkpoint: forward 19.1, backward 21.5 and 3.4
// to join, 5.0 and 4.4 TB/s (copies of such sizes reach 5.7).
#include <algorithm>

#include "float8.cuh"
#include "tc05.cuh"

namespace lnorm {

using namespace f8;
using tc05::add2;
using tc05::fma2;

struct Forward {
  int64_t rows;
  int c, access_in, access_out, access_weights;
  float epsilon;
  const void* x;
  const float *scale, *offset;
  void* y;                       // or null
  float *mean, *inverse;         // or null
  Matrix kept, encoded;          // codes null: none
};

struct Backward {
  int64_t rows;
  int c, access_dy, access_x, access_dx, access_weights;
  const void *dy, *x;            // x null: `kept`
  Matrix kept;
  const float *mean, *inverse, *scale;
  void* dx;
  float *partial_g, *partial_b;  // [blocks][2][c] and its second rows; of one block the gradients themselves
};

__host__ __device__ constexpr int threads_of(int G) { return G <= 256 ? 256 : G; }
__host__ __device__ constexpr int blocks_of(int G) { return 512 / threads_of(G); }      // a multiprocessor's
// (rows in 16 bits leave the forward pass registers for three blocks: 147456 x 128 with a checkpoint 19.7 -> 19.1 us; float32 is slower so, 205824 x 64
// 18.3 -> 19.4)
template <typename T>
__host__ __device__ constexpr int forward_blocks_of(int G) { return sizeof(T) == 2 && threads_of(G) == 256 ? 3 : blocks_of(G); }

// Two sums over the G lanes of a row.  Wider than a warp: through two sets of slots in turn, with a barrier for the group's warps alone (which
// all make the same number of calls).
template <int G>
__device__ __forceinline__ float2 group_sum(float2 v, float2* slots, int& turn) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (G > 32) {
    constexpr int kWarps = threads_of(G) / 32, kOwn = G > 32 ? G / 32 : 1;
    const int warp = threadIdx.x >> 5, group = warp / kOwn;
    float2* s = slots + (turn++ & 1) * kWarps;
    if ((threadIdx.x & 31) == 0) s[warp] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(G > 32 ? G : 32) : "memory");
    v = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kOwn; ++w) { v.x += s[group * kOwn + w].x; v.y += s[group * kOwn + w].y; }
  }
  return v;
}

template <int LANES>
__device__ __forceinline__ Share load_weights(const float* p, int left, int access, float* room) {
  Raw<float> r;
  load16<float, LANES>(r, p, left, true, access);
  return unpack<float, LANES>(r, access, room);
}

template <typename T, int G>
__global__ void __launch_bounds__(threads_of(G), forward_blocks_of<T>(G))
forward_kernel(const Forward a) {
  constexpr int kGroups = threads_of(G) / G, kLanes = G < 8 ? G : 8, kWarp = G < 32 ? G : 32;
  __shared__ __align__(16) float rooms[threads_of(G) / 32][kRoom];
  float* room = rooms[threadIdx.x >> 5];
  __shared__ float2 slots[2 * threads_of(G) / 32];
  const int lane = threadIdx.x % G, group = threadIdx.x / G, first = lane * kShare, left = a.c - first;
  int turn = 0;
  lf_chain();
  const int64_t step = (int64_t)gridDim.x * kGroups;
  int64_t row = (int64_t)blockIdx.x * kGroups + group;
  Raw<T> raw;
  load16<T, kWarp>(raw, static_cast<const T*>(a.x) + row * a.c + first, left, row < a.rows, a.access_in);
  const Share scale = load_weights<kWarp>(a.scale + first, left, a.access_weights, room), offset = load_weights<kWarp>(a.offset + first, left, a.access_weights, room);
  const float over = 1.0f / (float)a.c;
  // (the trip count is the same for every lane of a block)
  for (int64_t base = (int64_t)blockIdx.x * kGroups; base < a.rows; base += step, row += step) {
    const bool live = row < a.rows;
    Share x = unpack<T, kWarp>(raw, a.access_in, room);
    load16<T, kWarp>(raw, static_cast<const T*>(a.x) + (row + step) * a.c + first, left, row + step < a.rows, a.access_in);
    if (a.kept.codes) {
      uint4 codes;
      const int s = encode16<kLanes>(x, a.kept.format, codes);
      if (live) put16(a.kept, row, first, codes, s);
    }
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kShare / 2; ++i) sum = add2(sum, x.v[i]);
    const float mean = group_sum<G>(make_float2(sum.x + sum.y, 0.f), slots, turn).x * over;
    sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kShare / 2; ++i) {
      x.v[i] = add2(x.v[i], both(-mean));
      if (left < kShare) {      // channels behind the last have no deviation
        if (2 * i >= left) x.v[i].x = 0.f;
        if (2 * i + 1 >= left) x.v[i].y = 0.f;
      }
      sum = fma2(x.v[i], x.v[i], sum);
    }
    const float inverse = 1.0f / sqrtf(fmaf(group_sum<G>(make_float2(sum.x + sum.y, 0.f), slots, turn).x, over, a.epsilon));
    if (a.mean && live && lane == 0) { a.mean[row] = mean; a.inverse[row] = inverse; }
#pragma unroll
    for (int i = 0; i < kShare / 2; ++i) x.v[i] = fma2(mul2(x.v[i], both(inverse)), scale.v[i], offset.v[i]);
    if (a.y) store16<T, kWarp>(static_cast<T*>(a.y) + row * a.c + first, left, live, a.access_out, x, room);
    if (a.encoded.codes) {
      if (left < kShare) {      // (0 * inverse is no zero in a row whose statistics are no numbers)
#pragma unroll
        for (int i = 0; i < kShare / 2; ++i) {
          if (2 * i >= left) x.v[i].x = 0.f;
          if (2 * i + 1 >= left) x.v[i].y = 0.f;
        }
      }
      uint4 codes;
      const int s = encode16<kLanes>(x, a.encoded.format, codes);
      if (live) put16(a.encoded, row, first, codes, s);
    }
  }
}

template <typename T, int G, bool KEPT>
__global__ void __launch_bounds__(threads_of(G), blocks_of(G))
backward_kernel(const Backward a) {
  constexpr int kThreads = threads_of(G), kGroups = kThreads / G, kWarp = G < 32 ? G : 32;
  __shared__ __align__(16) float rooms[kThreads / 32][kRoom];
  float* room = rooms[threadIdx.x >> 5];
  __shared__ float2 slots[2 * kThreads / 32];
  __shared__ float sums[kGroups > 1 ? kThreads * kShare : 1];
  const int lane = threadIdx.x % G, group = threadIdx.x / G, first = lane * kShare, left = a.c - first;
  int turn = 0;
  lf_chain();
  const int64_t step = (int64_t)gridDim.x * kGroups;
  int64_t row = (int64_t)blockIdx.x * kGroups + group;
  Raw<T> raw_dy, raw_x;
  uint4 codes;
  int power = 1;      // (a byte as it is loaded: what has to wait for it waits when the row's turn comes)
  float mean, inverse;
  auto fetch = [&](int64_t r) {      // (a row that does not exist is all zeros)
    const bool live = r < a.rows;
    load16<T, kWarp>(raw_dy, static_cast<const T*>(a.dy) + r * a.c + first, left, live, a.access_dy);
    codes = make_uint4(0, 0, 0, 0);
    if (!KEPT) load16<T, kWarp>(raw_x, static_cast<const T*>(a.x) + r * a.c + first, left, live, a.access_x);
    else if (live && left > 0) {
      codes = *reinterpret_cast<const uint4*>(a.kept.codes + r * a.kept.pitch + first);
      power = a.kept.exponents[exponent_at(r, first / kBlock, a.kept.tiles)];
    }
    mean = live ? a.mean[r] : 0.f;
    inverse = live ? a.inverse[r] : 0.f;
  };
  fetch(row);
  const Share scale = load_weights<kWarp>(a.scale + first, left, a.access_weights, room);
  Share dg, db;
#pragma unroll
  for (int i = 0; i < kShare / 2; ++i) dg.v[i] = db.v[i] = make_float2(0.f, 0.f);
  const float over = 1.0f / (float)a.c;
  for (int64_t base = (int64_t)blockIdx.x * kGroups; base < a.rows; base += step, row += step) {
    const Share dy = unpack<T, kWarp>(raw_dy, a.access_dy, room);
    Share u = KEPT ? decode16(codes, a.kept.format) : unpack<T, kWarp>(raw_x, a.access_x, room);
    const float inv = inverse;
    // (x - mean) rstd; of codes by one multiply-add, their power of two with rstd
    const float2 by = both(KEPT ? up(power) * inv : inv), from = both(KEPT ? -mean * inv : -mean);
#pragma unroll
    for (int i = 0; i < kShare / 2; ++i) u.v[i] = KEPT ? fma2(u.v[i], by, from) : mul2(add2(u.v[i], from), by);
    fetch(row + step);
    float2 s1 = make_float2(0.f, 0.f), s2 = s1;
#pragma unroll
    for (int i = 0; i < kShare / 2; ++i) {
      const float2 h = mul2(dy.v[i], scale.v[i]);
      dg.v[i] = fma2(dy.v[i], u.v[i], dg.v[i]);
      db.v[i] = add2(db.v[i], dy.v[i]);
      s1 = add2(s1, h);
      s2 = fma2(h, u.v[i], s2);
    }
    const float2 s = group_sum<G>(make_float2(s1.x + s1.y, s2.x + s2.y), slots, turn);
    const float2 t1 = both(-s.x * over * inv), t2 = both(-s.y * over * inv);
#pragma unroll
    for (int i = 0; i < kShare / 2; ++i) u.v[i] = fma2(u.v[i], t2, fma2(mul2(dy.v[i], scale.v[i]), both(inv), t1));
    store16<T, kWarp>(static_cast<T*>(a.dx) + row * a.c + first, left, row < a.rows, a.access_dx, u, room);
  }
  // this block's row of sums
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = (which ? a.partial_b : a.partial_g) + (int64_t)blockIdx.x * 2 * a.c;
    if (kGroups == 1) store16<float, kWarp>(out + first, left, true, kElements, which ? db : dg, room);
    else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kShare / 2; ++i) *reinterpret_cast<float2*>(&sums[threadIdx.x * kShare + 2 * i]) = which ? db.v[i] : dg.v[i];
      __syncthreads();
      for (int col = threadIdx.x; col < a.c; col += kThreads) {
        float t = 0.f;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) t += sums[g * (G * kShare) + col];
        out[col] = t;
      }
    }
  }
}

// Column sums of the blocks' rows, in the same order every time: 32 columns a block, 32 strands of rows with eight loads in flight each, then
// the strands.
__global__ void __launch_bounds__(1024)
join_kernel(const float* partial, int count, int c, float* dg, float* db) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  lf_chain();
  float t = 0.f;
  if (col < c) {
    const float* from = partial + (int64_t)blockIdx.y * c + col;
    for (int i = strand; i < count; i += 256) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = i + 32 * k < count ? from[(int64_t)(i + 32 * k) * 2 * c] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) t += v[k];
    }
  }
  s[strand][lane] = t;
  __syncthreads();
  t = s[lane][strand];      // (a column's strands are a warp's lanes)
#pragma unroll
  for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (lane == 0 && blockIdx.x * 32 + strand < c) (blockIdx.y ? db : dg)[blockIdx.x * 32 + strand] = t;
}

// Blocks that stay on the GPU, and no more than there are rows for.
static int grid_of(const lf_context* ctx, int64_t rows, int per_block, int per_sm) {
  const int64_t need = (rows + per_block - 1) / per_block, most = (int64_t)ctx->sm_count * per_sm;
  return (int)(need < most ? need : most);
}

constexpr int kMostChannels = 8192;

// f(lanes of a row as a type), by the width alone
template <typename F>
static auto by_width(int c, F f) {
  if (c <= 64) return f(std::integral_constant<int, 4>{});
  if (c <= 128) return f(std::integral_constant<int, 8>{});
  if (c <= 256) return f(std::integral_constant<int, 16>{});
  if (c <= 512) return f(std::integral_constant<int, 32>{});
  if (c <= 1024) return f(std::integral_constant<int, 64>{});
  if (c <= 2048) return f(std::integral_constant<int, 128>{});
  if (c <= 4096) return f(std::integral_constant<int, 256>{});
  return f(std::integral_constant<int, 512>{});
}

// Few rows take one block, whose sums are the gradients: three more turns of it cost less than the launch that joins blocks.
static int backward_blocks(const lf_context* ctx, int64_t rows, int c) {
  return by_width(c, [&](auto g) {
    constexpr int G = decltype(g)::value, kGroups = threads_of(G) / G;
    return rows <= 4 * kGroups ? 1 : grid_of(ctx, rows, kGroups, blocks_of(G));
  });
}

template <typename T>
static void launch_forward(lf_context* ctx, const Forward& a) {
  by_width(a.c, [&](auto g) {
    constexpr int G = decltype(g)::value;
    lf_launch(ctx, forward_kernel<T, G>, grid_of(ctx, a.rows, threads_of(G) / G, forward_blocks_of<T>(G)), threads_of(G), 0, a);
  });
}

template <typename T>
static void launch_backward(lf_context* ctx, const Backward& a, int blocks) {
  by_width(a.c, [&](auto g) {
    constexpr int G = decltype(g)::value;
    if (a.x) lf_launch(ctx, backward_kernel<T, G, false>, blocks, threads_of(G), 0, a);
    else lf_launch(ctx, backward_kernel<T, G, true>, blocks, threads_of(G), 0, a);
  });
}

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
  const uint64_t bytes = (uint64_t)d->rows * d->channels * (d->act_dtype == LF_DTYPE_BF16 ? 2 : 4);
  if (d->out && d->out != d->activations) LF_TRY(lf_float8_apart(ctx, "layer norm", d->out, bytes, d->activations, bytes));
  for (const float* operand : {d->scale, d->offset}) LF_TRY(lf_float8_apart(ctx, "layer norm", d->out, bytes, operand, (uint64_t)d->channels * 4));
  const lf_device_guard device(ctx);
  Forward a{};
  a.rows = d->rows; a.c = d->channels; a.epsilon = d->epsilon;
  a.access_in = row_access(d->activations, a.c, d->act_dtype);
  a.access_out = row_access(d->out, a.c, d->act_dtype);
  a.access_weights = std::min(row_access(d->scale, a.c, LF_DTYPE_F32), row_access(d->offset, a.c, LF_DTYPE_F32));
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
  const int blocks = backward_blocks(ctx, rows, channels);
  return blocks == 1 ? 0 : (uint64_t)blocks * 2 * channels * sizeof(float);
}

lf_status lf_layer_norm_backward_run(lf_context* ctx, const lf_layer_norm_backward_desc* d, lf_result* r) {
  if (!ctx) return LF_ERR_ARGUMENT;
  if (!d || !d->gradient || (!d->activations && !d->checkpoint.codes) || !d->mean || !d->inverse_deviation || !d->scale || !d->out ||
      !d->scale_gradient || !d->offset_gradient)
    return lf_fail(ctx, LF_ERR_ARGUMENT, "layer norm backward: null argument");
  if (d->activations && d->checkpoint.codes) return lf_fail(ctx, LF_ERR_ARGUMENT, "layer norm backward: activations or a checkpoint, not both");
  LF_TRY(lf_float8_check_rows(ctx, "layer norm backward", d->rows, d->channels, d->act_dtype));
  if (d->channels > kMostChannels) return lf_fail(ctx, LF_ERR_UNSUPPORTED, "layer norm of %d channels: at most %d", d->channels, kMostChannels);
  if (d->checkpoint.codes) LF_TRY(lf_float8_check(ctx, "layer norm backward", d->checkpoint, d->rows, d->channels));
  const uint64_t bytes = (uint64_t)d->rows * d->channels * (d->act_dtype == LF_DTYPE_BF16 ? 2 : 4);
  for (const void* operand : {d->gradient, d->activations})      // (a row is read by the lanes that store it, before they do)
    if (operand && d->out != operand) LF_TRY(lf_float8_apart(ctx, "layer norm backward", d->out, bytes, operand, bytes));
  LF_TRY(lf_float8_apart(ctx, "layer norm backward", d->out, bytes, d->checkpoint));
  for (const float* operand : {d->mean, d->inverse_deviation}) LF_TRY(lf_float8_apart(ctx, "layer norm backward", d->out, bytes, operand, (uint64_t)d->rows * 4));
  LF_TRY(lf_float8_apart(ctx, "layer norm backward", d->out, bytes, d->scale, (uint64_t)d->channels * 4));
  const uint64_t need = lf_layer_norm_backward_workspace(ctx, d->rows, d->channels);
  if (need && (!d->workspace || d->workspace_bytes < need || !lf_aligned16(d->workspace)))
    return lf_fail(ctx, LF_ERR_ARGUMENT, "layer norm backward: a workspace of %llu bytes on a 16-byte boundary is needed", (unsigned long long)need);
  const lf_device_guard device(ctx);
  Backward a{};
  a.rows = d->rows; a.c = d->channels;
  a.access_dy = row_access(d->gradient, a.c, d->act_dtype);
  a.access_x = row_access(d->activations, a.c, d->act_dtype);
  a.access_dx = row_access(d->out, a.c, d->act_dtype);
  a.access_weights = row_access(d->scale, a.c, LF_DTYPE_F32);
  a.dy = d->gradient; a.x = d->activations; a.mean = d->mean; a.inverse = d->inverse_deviation; a.scale = d->scale; a.dx = d->out;
  if (d->checkpoint.codes) a.kept = matrix(d->checkpoint);
  const int blocks = backward_blocks(ctx, a.rows, a.c);
  a.partial_g = blocks == 1 ? d->scale_gradient : (float*)d->workspace;
  a.partial_b = blocks == 1 ? d->offset_gradient : a.partial_g + a.c;
  lf_prof_begin(ctx, LF_KERNEL_ELEMENTWISE);
  if (d->act_dtype == LF_DTYPE_BF16) launch_backward<bf16>(ctx, a, blocks); else launch_backward<float>(ctx, a, blocks);
  lf_prof_end(ctx);
  ctx->launches++;
  if (blocks == 1) return lf_float8_done(ctx, r, 1);
  lf_prof_begin(ctx, LF_KERNEL_ELEMENTWISE);
  lf_launch(ctx, join_kernel, dim3(lf_ceil_div(a.c, 32), 2), 1024, 0, a.partial_g, blocks, a.c, d->scale_gradient, d->offset_gradient);
  lf_prof_end(ctx);
  ctx->launches++;
  return lf_float8_done(ctx, r, 2);
}

}  // extern "C"
